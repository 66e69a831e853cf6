// Host-side C shim over ferric_b200/csrc/kv_index.h so the CPU tests can drive the very index functions the device kernels
// use (compiled with g++, no CUDA needed).
#include "../../ferric_b200/csrc/kv_index.h"

using namespace ferric;

static KvSeqsView seqs(const int* table, long long stride, int cols, const int* lens, const int* starts, int n, int tokens)
{
    KvSeqsView s;
    s.table = table;
    s.table_stride = stride;
    s.cols = cols;
    s.lens = lens;
    s.starts = starts;
    s.seqs = n;
    s.tokens = tokens;
    return s;
}

extern "C" {
void shim_span(const int* lens, const int* starts, int n, int tokens, int i, int* first_n_pos0_poslast)
{
    const KvSpan p = kv_span(seqs(nullptr, 0, 0, lens, starts, n, tokens), i);
    first_n_pos0_poslast[0] = p.first;
    first_n_pos0_poslast[1] = p.n;
    first_n_pos0_poslast[2] = p.pos(0);
    first_n_pos0_poslast[3] = p.pos(p.n - 1);
}
int shim_seq_of(const int* starts, int n, int tokens, int t) { return kv_seq_of(seqs(nullptr, 0, 0, nullptr, starts, n, tokens), t); }
long long shim_offset(int n_pages, int heads, int page_shift, int dim, long long page_stride, const int* table, long long stride, int cols,
                      int n, int seq, int h, int pos)
{
    KvCacheView c;
    c.n_pages = n_pages;
    c.heads = heads;
    c.page_shift = page_shift;
    c.dim = dim;
    c.page_stride = page_stride;
    return kv_offset(c, seqs(table, stride, cols, nullptr, nullptr, n, n), seq, h, pos);
}
void shim_seen(int page_shift, int cols, int pos, int window, int* lo_hi)
{
    KvCacheView c;
    c.page_shift = page_shift;
    lo_hi[0] = kv_seen_lo(pos, window);
    lo_hi[1] = kv_seen_hi(c, seqs(nullptr, 0, cols, nullptr, nullptr, 0, 0), pos);
}
// blocks of one sequence: out[b] = {r0, rows, j0, j1, lo, hi, t0, tiles}; returns their number
int shim_blocks(int page_shift, int cols, int first, int n, int len, int group, int rb, int window, int* out, int cap, long long* tiles)
{
    KvCacheView c;
    c.page_shift = page_shift;
    const KvSeqsView s = seqs(nullptr, 0, cols, nullptr, nullptr, 1, first + n);
    KvSpan p;
    p.first = first;
    p.n = n;
    p.len = len;
    const int nb = attend_blocks(p, group, rb);
    for (int b = 0; b < nb && b < cap; b++) {
        const AttendBlock k = attend_block(c, s, p, group, rb, window, b);
        const int v[8] = {k.r0, k.rows, k.j0, k.j1, k.lo, k.hi, k.t0, k.tiles};
        for (int i = 0; i < 8; i++) out[8 * b + i] = v[i];
    }
    *tiles = attend_seq_tiles(c, s, p, group, rb, window);
    return nb;
}
long long shim_cut(long long total, int parts, int i) { return attend_cut(total, parts, i); }
int shim_part_of(long long total, int parts, long long x) { return attend_part_of(total, parts, x); }
}
