// Index arithmetic of the paged key-value cache and of the attention's work split: plain integer code shared by the device
// kernels, the host launchers and a CPU test.
#pragma once
#include <stddef.h>
#include <stdint.h>

#if defined(__CUDACC__)
#define FERRIC_KV_HD __host__ __device__ __forceinline__
#else
#define FERRIC_KV_HD inline
#endif

namespace ferric {

// Keys and values of one layer: [n_pages][heads][page][dim] each, pages `page_stride` elements apart.
struct KvCacheView {
    void* k = nullptr;
    void* v = nullptr;
    long long page_stride = 0;
    int n_pages = 0, page_shift = 0, heads = 0, dim = 0;
    int bf16 = 0;                    // 1: bf16, 0: f16
};
// The batch: table[seq][cols] page numbers, lengths (new tokens included), first token row of each sequence (null: token
// row i is the one new token of sequence i); `tokens` rows of activations in all.
struct KvSeqsView {
    const int* table = nullptr;
    long long table_stride = 0;
    const int* lens = nullptr;
    const int* starts = nullptr;
    int cols = 0, seqs = 0, tokens = 0;
};
struct RopeView {
    const double* turns = nullptr;   // [rotary / 2] turns per position
    int rotary = 0;                  // leading elements of a head that are rotated; 0: none
    int interleaved = 0;             // 1: pairs (2i, 2i + 1), 0: pairs (i, i + rotary / 2)
};

FERRIC_KV_HD int kv_min(int a, int b) { return a < b ? a : b; }
FERRIC_KV_HD int kv_max(int a, int b) { return a > b ? a : b; }

// The new tokens of sequence i: activation rows [first, first + n), the last of them at position len - 1.
struct KvSpan {
    int first, n, len;
    // position of new token j; a length shorter than the new tokens puts the first of them below 0, where nothing is
    FERRIC_KV_HD int pos(int j) const { return (int)((long long)len - n + j < INT32_MIN ? INT32_MIN : (long long)len - n + j); }
};
FERRIC_KV_HD KvSpan kv_span(const KvSeqsView& s, int i)
{
    KvSpan r;
    if (s.starts) {
        // starts that do not ascend, or reach past the activations, yield empty spans, never a row outside them
        const int a = kv_max(0, s.starts[i]), b = kv_min(s.tokens, s.starts[i + 1]);
        r.first = a;
        r.n = b > a ? b - a : 0;
    } else {
        r.first = i;
        r.n = 1;
    }
    r.len = s.lens[i];
    return r;
}
// The sequence whose span holds activation row t, or -1 (rows before the first start and behind the last one).
FERRIC_KV_HD int kv_seq_of(const KvSeqsView& s, int t)
{
    if (!s.starts) return t < s.seqs ? t : -1;
    if (t < s.starts[0] || t >= s.starts[s.seqs]) return -1;
    int lo = 0, hi = s.seqs;   // starts[lo] <= t < starts[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s.starts[mid] <= t) lo = mid;
        else hi = mid;
    }
    return lo;
}
// The cache page of column `col` of sequence `seq`, or -1 where the table has none.
FERRIC_KV_HD int kv_page(const KvCacheView& c, const KvSeqsView& s, int seq, int col)
{
    if (col < 0 || col >= s.cols) return -1;
    const int page = s.table[(long long)seq * s.table_stride + col];
    return (unsigned)page < (unsigned)c.n_pages ? page : -1;
}
// First element of (page of position `pos`, head h, slot of `pos`), or -1 where there is no page.  64-bit: a cache passes
// 2^31 elements at 4 GB.
FERRIC_KV_HD long long kv_offset(const KvCacheView& c, const KvSeqsView& s, int seq, int h, int pos)
{
    const int page = pos < 0 ? -1 : kv_page(c, s, seq, pos >> c.page_shift);
    if (page < 0) return -1;
    return (long long)page * c.page_stride + (((long long)h << c.page_shift) + (pos & ((1 << c.page_shift) - 1))) * c.dim;
}
// Keys a token at position `pos` sees: [lo, hi).  The table's capacity (at most kKvMaxPositions) bounds hi; a window of w keys
// bounds lo.
constexpr long long kKvMaxPositions = 1ll << 30;
FERRIC_KV_HD int kv_seen_lo(int pos, int window) { return window > 0 && pos >= window ? pos - window + 1 : 0; }
FERRIC_KV_HD int kv_seen_hi(const KvCacheView& c, const KvSeqsView& s, int pos)
{
    const long long cap = (long long)s.cols << c.page_shift, h = pos < 0 ? 0 : (long long)pos + 1;
    return (int)(h < cap ? h : cap);
}

// ---- the attention's work split ---------------------------------------------------------------------------------------
// The query rows of a sequence and key-value head are its (token, query head of the group) pairs, token-major; a block is
// `rb` of them, against key tiles of kAttendTile positions.  All tiles of all blocks -- sequence by sequence, head by head,
// block by block -- form one line that is cut evenly over the CTAs, wherever blocks begin and end: the lengths decide on the
// device, so a captured launch stays balanced when they change.
constexpr int kAttendTile = 64;
struct AttendBlock {
    int r0, rows;      // query rows [r0, r0 + rows) of the sequence
    int j0, j1;        // new tokens of the first and the last row
    int lo, hi;        // keys that any of the rows sees
    int t0, tiles;     // key tiles [t0, t0 + tiles); a block that sees nothing has one, with every key masked
};
FERRIC_KV_HD int attend_blocks(const KvSpan& p, int group, int rb) { return (p.n * group + rb - 1) / rb; }
FERRIC_KV_HD AttendBlock attend_block(const KvCacheView& c, const KvSeqsView& s, const KvSpan& p, int group, int rb, int window, int b)
{
    AttendBlock k;
    k.r0 = b * rb;
    k.rows = kv_min(p.n * group - k.r0, rb);
    k.j0 = k.r0 / group;
    k.j1 = (k.r0 + k.rows - 1) / group;
    k.lo = kv_seen_lo(p.pos(k.j0), window);
    k.hi = kv_seen_hi(c, s, p.pos(k.j1));
    k.t0 = k.lo / kAttendTile;
    k.tiles = (k.hi + kAttendTile - 1) / kAttendTile - k.t0;
    if (k.hi <= k.lo) {
        k.lo = k.hi = k.t0 = 0;
        k.tiles = 1;
    }
    return k;
}
// Tiles of one head of a sequence.
FERRIC_KV_HD long long attend_seq_tiles(const KvCacheView& c, const KvSeqsView& s, const KvSpan& p, int group, int rb, int window)
{
    const int nb = attend_blocks(p, group, rb);
    if (nb == 0) return 0;
    if (p.n == 1) return (long long)nb * attend_block(c, s, p, group, rb, window, 0).tiles;
    long long t = 0;
    for (int b = 0; b < nb; b++) t += attend_block(c, s, p, group, rb, window, b).tiles;
    return t;
}
// 64-bit quotient; nearly always both fit 32 bits, where the division costs a fraction
FERRIC_KV_HD long long attend_div(long long a, long long b)
{
    return ((a | b) >> 32) == 0 ? (long long)((unsigned)a / (unsigned)b) : a / b;
}
// `total` tiles over `parts` CTAs: part i starts at attend_cut(i), and tile x is attend_part_of(x)'s.
FERRIC_KV_HD long long attend_cut(long long total, int parts, int i)
{
    const long long q = attend_div(total, parts), r = total - q * parts;
    return i * q + (i < r ? i : r);
}
FERRIC_KV_HD int attend_part_of(long long total, int parts, long long x)
{
    const long long q = attend_div(total, parts), r = total - q * parts;
    return (int)(x < r * (q + 1) ? attend_div(x, q + 1) : r + attend_div(x - r * (q + 1), q));
}

}  // namespace ferric
