// Attention of the new tokens over the paged key-value cache:
//   out[t, h] = sum_k softmax_k(scale * R(pos_t) q[t, h] . k) v      over the keys token t sees,
// in one pass over the keys (running maximum m and sum l in f32; the output rescaled by 2^(m_old - m_new) when the maximum
// grows; scores in log2 units, so that the exponential is ex2).
#include <string.h>

#include <type_traits>

#include "kv.cuh"
#include "tc_common.cuh"

namespace ferric {

int* gemm_status_word();   // device address of the status word shared with the tensor-core products (kernels_gemm.cu)

// ---------------------------------------------------------------------------------------------------------------------
// attend_split_kernel: few query rows against many keys, kept to f32 accuracy.
//
// 64 sequences over 0.7k-8k keys (40 over 8 heads x 128, f16): 194 us a call = 6.1 TB/s (190 in a captured graph); on a bf16 cache
// 229 in a graph: three parts of q and the sums pass the 168 registers that two CTAs per SM leave, and spill (288 bytes stored, 624
// loaded).  One over 131000 (bf16): 114 us = 4.7 TB/s, of which the stream itself takes about 80.  Bound by the cache's bytes from
// HBM (2 * 2 * head_dim per key and head; at 5 query heads per key-value head that is 5 multiply-adds per byte).  So: one CTA
// reads a tile of 64 keys once for all query heads of its key-value head, tiles travel
// by TMA into a ring filled by a warp of its own, and the line of all tiles is cut evenly over the resident CTAs
// (kv_index.h); a block that several CTAs share leaves pieces (m, l, unnormalised output) in the workspace, which the CTA
// that finishes last joins, in piece order whoever that is, so the same call gives the same bits.
//
// The products run on mma.sync m16n8k16: decode has 1 to 8 query rows per key-value head, and its 16-row operand has room
// for the q of 8 rows twice.  The cache's elements are 16-bit already; q and the weights p are f32, and rounding them to 16
// bits would put up to 2^-8 of error where the o product takes f32 -- so they are split into 16-bit parts that add up to (almost)
// the f32 value: two f16 parts (22 bits), the first in rows 0-7 and the second in rows 8-15 of one MMA, or three bf16 parts
// (24 bits), the third in a second MMA.  A row's two halves meet in one thread's registers (rows g and g + 8).  f16 parts
// are scaled away from f16's lower end first: q by a power of two per row, p by 2^14.
template <typename T, int D, int WM>
struct SplitCfg {
    static constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
    static constexpr int kWarps = WM == 8 ? 8 : 4;       // consumer warps: WM row tiles of 8 x kWN runs of keys
    static constexpr int kWN = kWarps / WM;
    static constexpr int kRows = 8 * WM;
    static constexpr int kKeys = kAttendTile / kWN;      // keys of a tile one warp works on
    static constexpr int kThreads = 32 * (kWarps + 1);
    static constexpr int kStageBytes = 2 * kAttendTile * D * 2;
    static constexpr bool kQSmem = D == 256;             // 96 registers of q and 128 of output do not fit one thread
    static constexpr int kQBytes = kQSmem ? WM * (D / 16) * 32 * (kBf16 ? 24 : 16) : 0;
    static constexpr int kPitch = D + 8;                 // floats of a row of q, or of results done again: D sums, m, l
    // warps that hand their results over in one round of the merge
    static constexpr int kMerge = kWN == 1 ? 0 : (D == 256 && WM == 1) ? 1 : kWarps / 2;
    static constexpr int kSlot = 8 * D + 32;
    static constexpr int kBufFloats = kMerge * kSlot > kRows * kPitch ? kMerge * kSlot : kRows * kPitch;   // merge; results done again
    // the widest tiles at head_dim 256 keep q and the results in one place: the next block's q comes when this one is done
    static constexpr bool kOneBuf = D == 256 && WM == 4;
    static constexpr int kFixed = 1024 + kQBytes + (kOneBuf ? 0 : kRows * kPitch * 4) + kBufFloats * 4 + 512;
    // Two CTAs per SM where registers and shared memory allow: one CTA's set-up and join hide under the other's stream.
    static constexpr int kMinCtas = (D == 256 || WM == 8) ? 1 : 2;
    static constexpr int kSmemMax = kMinCtas == 2 ? 113 * 1024 : 227 * 1024;
    static constexpr int kStagesFit = (kSmemMax - kFixed) / kStageBytes;
    static constexpr int kStages = kStagesFit > 8 ? 8 : kStagesFit;
    static constexpr int kSmem = kFixed + kStages * kStageBytes;
    static constexpr int kTileFloats = 8 * D + 16;       // a row tile of a piece
    static constexpr int kPieceFloats = WM * kTileFloats;
    static_assert(kStages >= 2, "a ring of two stages at least");
};
constexpr float kPShiftF16 = 14.0f;   // p in f16 parts is scaled by 2^14: parts stay normal down to 2^-28

struct SplitWork {
    float* pieces;       // [CTA][2][piece]
    unsigned* tickets;   // [CTA], zero between launches
    int* status;
    int min_tiles;       // tiles per CTA at least, while there are few ..
    int min_parts;       // .. but as many CTAs as there are (sequence, head) pairs to do side by side
    unsigned long long group_recip;   // ceil(2^32 / group)
};
struct SplitBars {
    uint64_t full[8], empty[8], q_full, q_empty;
    unsigned valid[8];           // per stage: which of the tile's pages exist
    long long warp_sum[16];
    long long item_start;
    int seq, last;
    int tainted;                 // bit 0: a value that is not finite; bit 1: weights that are NaN (bf16)
    int inf_count, inf_key[32];  // infinite keys
    volatile int abort;          // a wait ran out
};
static_assert(sizeof(SplitBars) <= 512, "SplitCfg::kFixed has 512 bytes for it");

__device__ __forceinline__ float ex2f(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// hi + lo, where an infinite or NaN lo does not count: the first part of q decides on an infinite key.
__device__ __forceinline__ float add_finite(float hi, float lo)
{
    asm("min.xorsign.abs.f32 %0, %0, %1;" : "+f"(lo) : "f"(3.4028235e38f));
    return hi + lo;
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <bool BF16>
__device__ __forceinline__ void mma_kv(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    if constexpr (BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        mma_16816(c, a0, a1, a2, a3, b0, b1);
}
// (x, y) as NL pairs of 16-bit parts, largest first.
template <bool BF16>
__device__ __forceinline__ void split_pair(float x, float y, uint32_t& p0, uint32_t& p1, uint32_t& p2)
{
    if constexpr (BF16) {
        __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        p0 = *reinterpret_cast<uint32_t*>(&h);
        x -= __uint_as_float(p0 << 16);
        y -= __uint_as_float(p0 & 0xffff0000u);
        h = __floats2bfloat162_rn(x, y);
        p1 = *reinterpret_cast<uint32_t*>(&h);
        x -= __uint_as_float(p1 << 16);
        y -= __uint_as_float(p1 & 0xffff0000u);
        h = __floats2bfloat162_rn(x, y);
        p2 = *reinterpret_cast<uint32_t*>(&h);
    } else {
        __half2 h = __floats2half2_rn(x, y);
        p0 = h2_as_u32(h);
        const float2 f = __half22float2(h);
        h = __floats2half2_rn(x - f.x, y - f.y);
        p1 = h2_as_u32(h);
        p2 = 0;
    }
}
template <bool BF16>
__device__ __forceinline__ uint32_t not_finite2(uint32_t w)   // non-zero if either 16-bit element is an infinity or NaN
{
    constexpr uint32_t e = BF16 ? 0x7f80u : 0x7c00u;
    return ((w & e) == e) | ((w & (e << 16)) == (e << 16));
}

template <typename T, int D, int WM>
__global__ void __launch_bounds__(SplitCfg<T, D, WM>::kThreads, SplitCfg<T, D, WM>::kMinCtas)
attend_split_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, KvCacheView c, KvSeqsView s,
                    RopeView rope, AttendArgs a, SplitWork wk)
{
    using C = SplitCfg<T, D, WM>;
    constexpr bool BF = C::kBf16;
    constexpr int KS = D / 16, NT = D / 8, WN = C::kWN, RB = C::kRows;
    constexpr float kShift = BF ? 0.0f : kPShiftF16;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t* qfrag = ring + C::kStages * C::kStageBytes;
    float* qrow = reinterpret_cast<float*>(qfrag + C::kQBytes);   // the block's q rows, rotated in place
    float* buf = C::kOneBuf ? qrow : qrow + C::kRows * C::kPitch;
    SplitBars* bar = reinterpret_cast<SplitBars*>(buf + C::kBufFloats);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int group = a.heads / c.heads;

    if (tid == 0) {
        for (int i = 0; i < C::kStages; i++) {
            mbar_init(&bar->full[i], 1);
            mbar_init(&bar->empty[i], C::kWarps);
        }
        mbar_init(&bar->q_full, 1);
        mbar_init(&bar->q_empty, C::kWarps);
        bar->tainted = bar->abort = bar->inf_count = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    pdl_launch_dependents();
    // this thread's pair of elements of a q row and its frequency (immutable: read before the wait)
    constexpr int kPairs = D / 2, kCons = 32 * C::kWarps;
    const int pair = tid % kPairs;
    const bool rot = 2 * pair < rope.rotary;
    const int e0 = rot && !rope.interleaved ? pair : 2 * pair, e1 = rot && !rope.interleaved ? pair + (rope.rotary >> 1) : 2 * pair + 1;
    const double turns = rot ? rope.turns[pair] : 0.0;
    pdl_wait();

    // ---- this CTA's run of tiles: the batch's total, then the sequence in which the run starts
    constexpr int kScan = C::kThreads;
    auto seq_tiles = [&](int i) -> long long {
        return i < s.seqs ? attend_seq_tiles(c, s, kv_span(s, i), group, RB, a.window) * c.heads : 0;
    };
    // inclusive sum over the block's threads; `all` is the sum over all of them
    auto block_incl = [&](long long v, long long* all) {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long u = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += u;
        }
        if (lane == 31) bar->warp_sum[warp] = v;
        __syncthreads();
        long long before = 0, sum = 0;
#pragma unroll
        for (int w = 0; w < C::kWarps + 1; w++) {
            if (w == warp) before = sum;
            sum += bar->warp_sum[w];
        }
        *all = sum;
        return v + before;
    };
    long long total = 0, mine = 0, incl = 0;
    for (int i0 = 0; i0 < s.seqs; i0 += kScan) {
        if (i0) __syncthreads();
        long long all;
        mine = seq_tiles(i0 + tid);
        incl = block_incl(mine, &all);
        total += all;
    }
    if (total == 0) return;
    long long want = (total + wk.min_tiles - 1) / wk.min_tiles;
    if (want < wk.min_parts) want = wk.min_parts < total ? wk.min_parts : total;
    const int parts = (int)(want < (long long)gridDim.x ? want : (long long)gridDim.x);
    if ((int)blockIdx.x >= parts) return;
    const long long x0 = attend_cut(total, parts, blockIdx.x), x1 = attend_cut(total, parts, blockIdx.x + 1);
    {
        long long base = 0;
        for (int i0 = 0; i0 < s.seqs; i0 += kScan) {
            long long all = 0;
            if (s.seqs > kScan) {             // (the one chunk of a smaller batch is still in registers)
                __syncthreads();
                mine = seq_tiles(i0 + tid);
                incl = block_incl(mine, &all);
            }
            if (x0 >= base + incl - mine && x0 < base + incl) {
                bar->seq = i0 + tid;
                bar->item_start = base + incl - mine;
            }
            base += all;
        }
        __syncthreads();
    }
    int seq = bar->seq;
    long long item = bar->item_start;         // line position of the current block's first tile
    KvSpan span = kv_span(s, seq);
    int head = 0, blk = 0;
    {
        const long long per_head = attend_seq_tiles(c, s, span, group, RB, a.window);
        head = (int)(attend_div(x0 - item, per_head));
        item += head * per_head;
    }
    int nblk = attend_blocks(span, group, RB);
    AttendBlock b = attend_block(c, s, span, group, RB, a.window, blk);
    while (x0 >= item + b.tiles) {
        item += b.tiles;
        b = attend_block(c, s, span, group, RB, a.window, ++blk);
    }
    auto advance = [&]() {                    // to the next block on the line
        item += b.tiles;
        if (item >= x1) return;
        if (++blk == nblk) {
            blk = 0;
            if (++head == c.heads) {
                head = 0;
                do span = kv_span(s, ++seq);
                while (span.n == 0);
                nblk = attend_blocks(span, group, RB);
            }
        }
        b = attend_block(c, s, span, group, RB, a.window, blk);
    };
    // query row r of the block is (new token, query head of the group); rem0 + r < group + 64, so the reciprocal is exact
    auto token_of = [&](int r) { return b.j0 + (int)(((unsigned)(b.r0 - b.j0 * group + r) * wk.group_recip) >> 32); };
    auto head_of = [&](int r) { return b.r0 + r - token_of(r) * group; };
    bool dead = false;                        // a wait ran out: wait for nothing more, finish the launch
    auto wait = [&](uint64_t* which, uint32_t parity, int code) {
        if (dead || mbar_wait(which, parity)) return;
        dead = true;
        bar->abort = code;
        if (wk.status) atomicExch(wk.status, code);
    };
    auto let_copies_land = [&] {              // .. before the CTA's memory goes away
        if (!bar->abort) return;
        for (int i = 0; i < 200; i++) __nanosleep(1000);
    };

    if (warp == C::kWarps) {
        // ---- producer: pages to tensor-map coordinates, lane = copy (a box of 64 dimensions x up to 64 rows of one page)
        const int box = kv_min(kAttendTile, 1 << c.page_shift), pp = kAttendTile / box;
        const int copies = pp * (D / 64) * 2;
        const int piece = lane % pp, half = (lane / pp) % (D / 64), which = lane / (pp * (D / 64));
        int n = 0, nq = 0;
        for (; item < x1; advance()) {
            const int ta = item < x0 ? (int)(x0 - item) : 0, tb = item + b.tiles > x1 ? (int)(x1 - item) : b.tiles;
            // the block's q rows come before its tiles, so that they are not queued behind a ring full of them
            if (nq > 0) wait(&bar->q_empty, (nq - 1) & 1, 42);
            if (__any_sync(0xffffffffu, dead)) break;   // its place may still be in use
            nq++;
            if (lane == 0) mbar_expect_tx(&bar->q_full, (uint32_t)b.rows * D * 4);
            __syncwarp();
            for (int r = lane; r < b.rows; r += 32) {
                const int j = token_of(r), h = head * group + head_of(r);
                bulk_g2s(qrow + r * C::kPitch, a.q + (size_t)(span.first + j) * a.ldq + (size_t)h * D, D * 4, &bar->q_full);
            }
            for (int t = ta; t < tb; t++, n++) {
                const int st = n % C::kStages;
                const int pos = (b.t0 + t) * kAttendTile + piece * box;
                const int page = kv_page(c, s, seq, pos >> c.page_shift);
                const unsigned have = __ballot_sync(0xffffffffu, page >= 0);
                if (n >= C::kStages) wait(&bar->empty[st], ((n / C::kStages) & 1) ^ 1, 40);
                if (__any_sync(0xffffffffu, dead)) break;
                if (lane == 0) {
                    bar->valid[st] = have & ((1u << pp) - 1u);
                    mbar_expect_tx(&bar->full[st], C::kStageBytes);
                }
                __syncwarp();
                if (lane < copies) {
                    uint8_t* dst = ring + st * C::kStageBytes + which * (C::kStageBytes / 2) + half * (kAttendTile * 128) + piece * box * 128;
                    // an absent page: a coordinate behind the last one, which the copy fills with zeros
                    tma_load_4d(dst, which ? &vmap : &kmap, half * 64, pos & ((1 << c.page_shift) - 1), head, page >= 0 ? page : max(1, c.n_pages),
                                &bar->full[st]);
                }
            }
        }
        let_copies_land();
        return;
    }

    // ---- consumers
    const int wm = warp % WM, kn = warp / WM, g = lane >> 2, t4 = lane & 3;
    const uint32_t ring_addr = smem_u32(ring);
    const uint32_t k_lane = (uint32_t)((kn * C::kKeys + ((lane >> 4) & 1) * 8 + (lane & 7)) * 128);
    const uint32_t v_lane = (uint32_t)((kn * C::kKeys + ((lane >> 3) & 1) * 8 + (lane & 7)) * 128);
    const int box_shift = kv_min(6, c.page_shift);
    int n = 0, nq = 0;
    for (; item < x1; advance()) {
        const int ta = item < x0 ? (int)(x0 - item) : 0, tb = item + b.tiles > x1 ? (int)(x1 - item) : b.tiles;

        // q of the block's rows, rotated and scaled to log2 units in place; a pair of elements per thread and row, its angle
        // kept while the token stays the same (the query heads of a group)
        wait(&bar->q_full, nq & 1, 43);
        nq++;
        {
            constexpr int kStep = kCons / kPairs;
            const float scale = a.scale * kLog2e;
            int jt = -1;
            float cs = 1.0f, sn = 0.0f;
#pragma unroll 4
            for (int r = tid / kPairs; r < RB; r += kStep) {
                float* q = qrow + r * C::kPitch;
                const int j = token_of(r);
                if (rot && j != jt && r < b.rows) rope_cos_sin(turns, span.pos(j), &cs, &sn);
                jt = j;
                const float x = q[e0], y = q[e1];
                q[e0] = fmaf(-y, sn, x * cs) * scale;
                q[e1] = fmaf(y, cs, x * sn) * scale;
            }
        }
        named_bar_sync(1, kCons);
        // parts of q as MMA operands; lane (g, t): row g of the warp's tile, elements 16 ks + 2 t + {0, 1, 8, 9}
        float unscale = 1.0f;
        uint32_t qa[C::kQSmem ? 1 : KS][4], qb[C::kQSmem || !BF ? 1 : KS][2];
        {
            const float* q = qrow + (wm * 8 + g) * C::kPitch;
            float qscale = 1.0f;
            if (!BF) {
                float mx = 0.0f;
                for (int e = t4; e < D; e += 4) mx = fmaxf(mx, fabsf(q[e]));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                f16_row_scale(mx, &qscale, &unscale);
            }
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                const float2 u = *reinterpret_cast<const float2*>(q + 16 * ks + 2 * t4), w = *reinterpret_cast<const float2*>(q + 16 * ks + 2 * t4 + 8);
                uint32_t f[4], e0, e1;
                split_pair<BF>(u.x * qscale, u.y * qscale, f[0], f[1], e0);
                split_pair<BF>(w.x * qscale, w.y * qscale, f[2], f[3], e1);
                if constexpr (C::kQSmem) {
                    if (kn == 0) {
                        *reinterpret_cast<uint4*>(qfrag + ((wm * KS + ks) * 32 + lane) * 16) = make_uint4(f[0], f[1], f[2], f[3]);
                        if (BF) *reinterpret_cast<uint2*>(qfrag + WM * KS * 512 + ((wm * KS + ks) * 32 + lane) * 8) = make_uint2(e0, e1);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 4; i++) qa[ks][i] = f[i];
                    if constexpr (BF) {
                        qb[ks][0] = e0;
                        qb[ks][1] = e1;
                    }
                }
            }
        }
        auto q_done = [&] {   // the next block's q may land (by the async proxy, behind this thread's own writes)
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar->q_empty);
        };
        if constexpr (!C::kOneBuf) q_done();
        if constexpr (C::kQSmem) named_bar_sync(1, kCons);

        // keys this thread's row sees, and those that every row of the block sees
        const int my_r = wm * 8 + g, my_j = token_of(my_r);
        const int lo_r = my_r < b.rows ? kv_seen_lo(span.pos(my_j), a.window) : 0;
        const int hi_r = my_r < b.rows ? kv_seen_hi(c, s, span.pos(my_j)) : 0;
        const int lo_all = kv_seen_lo(span.pos(b.j1), a.window), hi_all = kv_seen_hi(c, s, span.pos(b.j0));

        float m = -INFINITY, l = 0.0f, o[NT][4];
#pragma unroll
        for (int i = 0; i < NT; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;

        auto tile_pass = [&](auto masked_c, int tile, uint32_t kbase, uint32_t vbase, unsigned valid) {
            constexpr bool MASKED = decltype(masked_c)::value;
            float sc[C::kKeys / 8][4];
#pragma unroll
            for (int i = 0; i < C::kKeys / 8; i++) sc[i][0] = sc[i][1] = sc[i][2] = sc[i][3] = 0.0f;
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                uint32_t A[4];
                [[maybe_unused]] uint32_t E[2];
                if constexpr (C::kQSmem) {
                    const uint4 f = *reinterpret_cast<const uint4*>(qfrag + ((wm * KS + ks) * 32 + lane) * 16);
                    A[0] = f.x, A[1] = f.y, A[2] = f.z, A[3] = f.w;
                    if constexpr (BF) {
                        const uint2 e = *reinterpret_cast<const uint2*>(qfrag + WM * KS * 512 + ((wm * KS + ks) * 32 + lane) * 8);
                        E[0] = e.x, E[1] = e.y;
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 4; i++) A[i] = qa[ks][i];
                    if constexpr (BF) E[0] = qb[ks][0], E[1] = qb[ks][1];
                }
                const uint32_t chunk = (uint32_t)(((2 * ks + ((lane >> 3) & 1)) & 7) ^ (lane & 7)) << 4;
#pragma unroll
                for (int np = 0; np < C::kKeys / 16; np++) {
                    uint32_t kf[4];
                    ldsm4(kf, kbase + k_lane + (ks >> 2) * (kAttendTile * 128) + np * (16 * 128) + chunk);
                    mma_kv<BF>(sc[2 * np], A[0], A[1], A[2], A[3], kf[0], kf[1]);
                    mma_kv<BF>(sc[2 * np + 1], A[0], A[1], A[2], A[3], kf[2], kf[3]);
                    if constexpr (BF) {
                        mma_kv<BF>(sc[2 * np], 0u, E[0], 0u, E[1], kf[0], kf[1]);
                        mma_kv<BF>(sc[2 * np + 1], 0u, E[0], 0u, E[1], kf[2], kf[3]);
                    }
                }
            }
            // scores: the two halves of a row are in this thread
            const int key0 = tile * kAttendTile + kn * C::kKeys + 2 * t4;
            float mx = -INFINITY;
#pragma unroll
            for (int i = 0; i < C::kKeys / 8; i++) {
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    // (in bf16 the zeros beside the third part have been multiplied by the key too)
                    float v = BF ? sc[i][e] + sc[i][e + 2] : add_finite(sc[i][e], sc[i][e + 2]);
                    if (!BF) v *= unscale;
                    if (MASKED) {
                        const int key = key0 + 8 * i + e;
                        const bool page = (valid >> ((kn * C::kKeys + 8 * i) >> box_shift)) & 1u;
                        if (!(key >= lo_r && key < hi_r && page)) v = -INFINITY;
                    }
                    sc[i][e] = v;
                    mx = fmaxf(mx, v);
                }
            }
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2)) - kShift;
            if (__any_sync(0xffffffffu, mx > m)) {
                const float mn = fmaxf(m, mx), fix = ex2f(m - (mn == -INFINITY ? 0.0f : mn));
                m = mn;
                l *= fix;
#pragma unroll
                for (int i = 0; i < NT; i++)
#pragma unroll
                    for (int e = 0; e < 4; e++) o[i][e] *= fix;
            }
            const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll
            for (int kk = 0; kk < C::kKeys / 16; kk++) {
                float p[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    p[e] = ex2f(sc[2 * kk + (e >> 1)][e & 1] - base);
                    l += p[e];
                }
                uint32_t P[4], E[2];
                split_pair<BF>(p[0], p[1], P[0], P[1], E[0]);
                split_pair<BF>(p[2], p[3], P[2], P[3], E[1]);
                uint32_t z0 = 0xffffffffu, z1 = 0xffffffffu;
                if (MASKED) {   // values no row of the block sees are taken as 0, whatever the cache holds there
                    const int key = key0 + 16 * kk;
                    const bool page = (valid >> ((kn * C::kKeys + 16 * kk) >> box_shift)) & 1u;
                    auto in = [&](int k) { return page && k >= b.lo && k < b.hi; };
                    z0 = (in(key) ? 0x0000ffffu : 0u) | (in(key + 1) ? 0xffff0000u : 0u);
                    z1 = (in(key + 8) ? 0x0000ffffu : 0u) | (in(key + 9) ? 0xffff0000u : 0u);
                }
                uint32_t odd = 0;
#pragma unroll
                for (int np = 0; np < NT / 2; np++) {
                    uint32_t vf[4];
                    const uint32_t chunk = (uint32_t)(((2 * np + (lane >> 4)) & 7) ^ (lane & 7)) << 4;
                    ldsm4t(vf, vbase + v_lane + (np >> 2) * (kAttendTile * 128) + kk * (16 * 128) + chunk);
                    if (MASKED) {
                        vf[0] &= z0, vf[1] &= z1, vf[2] &= z0, vf[3] &= z1;
                        odd |= not_finite2<BF>(vf[0]) | not_finite2<BF>(vf[1]) | not_finite2<BF>(vf[2]) | not_finite2<BF>(vf[3]);
                    }
                    mma_kv<BF>(o[2 * np], P[0], P[1], P[2], P[3], vf[0], vf[1]);
                    mma_kv<BF>(o[2 * np + 1], P[0], P[1], P[2], P[3], vf[2], vf[3]);
                    if constexpr (BF) {
                        mma_kv<BF>(o[2 * np], 0u, E[0], 0u, E[1], vf[0], vf[1]);
                        mma_kv<BF>(o[2 * np + 1], 0u, E[0], 0u, E[1], vf[2], vf[3]);
                    }
                }
                if (MASKED && odd && b.j0 != b.j1) atomicOr(&bar->tainted, 1);
            }
        };

        for (int t = ta; t < tb; t++, n++) {
            const int st = n % C::kStages, tile = b.t0 + t;
            wait(&bar->full[st], (n / C::kStages) & 1, 41);
            const uint32_t kbase = ring_addr + st * C::kStageBytes, vbase = kbase + C::kStageBytes / 2;
            const unsigned valid = bar->valid[st];
            const int pp = kAttendTile >> box_shift;
            if (tile * kAttendTile >= lo_all && (tile + 1) * kAttendTile <= hi_all && valid == (1u << pp) - 1u)
                tile_pass(std::false_type(), tile, kbase, vbase, valid);
            else
                tile_pass(std::true_type(), tile, kbase, vbase, valid);
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar->empty[st]);
        }

        // the row's halves and the quad's sums together
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        if (BF && l != l && my_r < b.rows) atomicOr(&bar->tainted, 2);
        float2 oo[NT];
#pragma unroll
        for (int i = 0; i < NT; i++) oo[i] = make_float2(o[i][0] + o[i][2], o[i][1] + o[i][3]);

        // the warps that share rows: pairwise through `buf`, in a fixed order
        named_bar_sync(1, kCons);
        const int tainted = bar->tainted;
        auto give = [&](float* slot) {
#pragma unroll
            for (int i = 0; i < NT; i++) *reinterpret_cast<float2*>(slot + i * 64 + lane * 2) = oo[i];
            if (t4 == 0) *reinterpret_cast<float2*>(slot + 8 * D + 2 * g) = make_float2(m, l);
        };
        auto take = [&](const float* slot) {
            const float2 ml = *reinterpret_cast<const float2*>(slot + 8 * D + 2 * g);
            const float mn = fmaxf(m, ml.x), base = mn == -INFINITY ? 0.0f : mn;
            const float f0 = ex2f(m - base), f1 = ex2f(ml.x - base);
            l = l * f0 + ml.y * f1;
            m = mn;
#pragma unroll
            for (int i = 0; i < NT; i++) {
                const float2 w = *reinterpret_cast<const float2*>(slot + i * 64 + lane * 2);
                oo[i].x = oo[i].x * f0 + w.x * f1;
                oo[i].y = oo[i].y * f0 + w.y * f1;
            }
        };
        if constexpr (C::kMerge == 1) {           // one warp at a time, where the buffer holds no more
#pragma unroll
            for (int w = 1; w < WN; w++) {
                if (kn == w) give(buf);
                named_bar_sync(1, kCons);
                if (kn == 0) take(buf);
                if (w + 1 < WN) named_bar_sync(1, kCons);
            }
        } else {
#pragma unroll
            for (int half = WN / 2; half > 0; half >>= 1) {
                float* slot = buf + ((kn % half) * WM + wm) * C::kSlot;
                if (kn >= half && kn < 2 * half) give(slot);
                named_bar_sync(1, kCons);
                if (kn < half) take(slot);
                if (half > 1) named_bar_sync(1, kCons);
            }
        }

        // now the kn == 0 warps hold their tile's rows: lane (g, t) elements 8 i + 2 t + {0, 1} of row g
        if (tainted) {
            // A value that some rows of the block see and others do not is not finite: weight 0 does not hide it in a matrix
            // product.  The rows again, one by one and key by key, over this CTA's tiles of the block.  Or weights are NaN: the rows
            // that infinite keys spoilt, if there are any.
            if (tainted == 2)
                list_infinite_keys<T, D>(c, s, seq, head, kv_max(b.lo, (b.t0 + ta) * kAttendTile), kv_min(b.hi, (b.t0 + tb) * kAttendTile), warp,
                                         C::kWarps, lane, &bar->inf_count, bar->inf_key, 32);
            named_bar_sync(1, kCons);
            const int infs = bar->inf_count;
            if ((tainted & 1) || infs > 0) {
                for (int r = warp; r < b.rows; r += C::kWarps) {
                    float* q = buf + r * C::kPitch;   // the row's q, then its results
                    const int j = token_of(r), h = head * group + head_of(r), pos = span.pos(j);
                    const int lo = kv_seen_lo(pos, a.window), hi = kv_seen_hi(c, s, pos);
                    const float* src = a.q + (size_t)(span.first + j) * a.ldq + (size_t)h * D;
                    __syncwarp();
                    for (int e = lane; e < D; e += 32) q[e] = rope_element(rope, src, e, pos) * (a.scale * kLog2e);
                    __syncwarp();
                    const bool again = (tainted & 1) || infinite_keys_weigh_nothing<T, D>(c, s, seq, head, q, lo, hi, infs, bar->inf_key, lane);
                    if (lane == 0) q[D + 2] = again ? 1.0f : 0.0f;
                    if (!again) continue;
                    float pm, pl, acc[D / 32];
                    attend_row_plain<T, D>(c, s, seq, head, q, kv_max(lo, (b.t0 + ta) * kAttendTile), kv_min(hi, (b.t0 + tb) * kAttendTile), lane, &pm,
                                           &pl, acc);
                    __syncwarp();
#pragma unroll
                    for (int e = 0; e < D / 32; e++) q[lane + 32 * e] = acc[e];
                    if (lane == 0) *reinterpret_cast<float2*>(q + D) = make_float2(pm, pl);
                }
            }
            named_bar_sync(1, kCons);
            if (tid == 0) bar->tainted = bar->inf_count = 0;
            const float* row = buf + (wm * 8 + g) * C::kPitch;
            if (((tainted & 1) || infs > 0) && my_r < b.rows && row[D + 2] != 0.0f) {
#pragma unroll
                for (int i = 0; i < NT; i++) oo[i] = *reinterpret_cast<const float2*>(row + 8 * i + 2 * t4);
                m = row[D];
                l = row[D + 1];
            }
        }

        auto out_at = [&](int r, int e) {   // element e of row r of the block
            return (size_t)(span.first + token_of(r)) * a.ldo + (size_t)(head * group + head_of(r)) * D + e;
        };
        if (ta == 0 && tb == b.tiles) {
            if (kn == 0 && my_r < b.rows) {
                const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                const size_t at = out_at(my_r, 2 * t4);
#pragma unroll
                for (int i = 0; i < NT; i++) {
                    const float2 v = make_float2(oo[i].x * inv, oo[i].y * inv);
                    if (a.out_bf16)
                        *reinterpret_cast<__nv_bfloat162*>(reinterpret_cast<__nv_bfloat16*>(a.out) + at + 8 * i) = __floats2bfloat162_rn(v.x, v.y);
                    else
                        *reinterpret_cast<float2*>(reinterpret_cast<float*>(a.out) + at + 8 * i) = v;
                }
            }
            if constexpr (C::kOneBuf) {
                named_bar_sync(1, kCons);
                q_done();
            }
            continue;
        }
        // A piece, in the lanes' order: per row tile [i][lane] pairs, then m and l of its rows.  A CTA has at most two: one of a
        // block begun before its run (slot 0), one of a block that goes on behind it (slot 1); the block's ticket belongs to the
        // CTA it begins in.
        const int c0 = attend_part_of(total, parts, item), c1 = attend_part_of(total, parts, item + b.tiles - 1), np = c1 - c0 + 1;
        auto piece_of = [&](int p) { return wk.pieces + ((size_t)(c0 + p) * 2 + (p == 0 ? 1 : 0)) * C::kPieceFloats; };
        if (kn == 0) {
            float* dst = piece_of((int)blockIdx.x - c0) + wm * C::kTileFloats;
#pragma unroll
            for (int i = 0; i < NT; i++) *reinterpret_cast<float2*>(dst + i * 64 + lane * 2) = oo[i];
            if (t4 == 0) *reinterpret_cast<float2*>(dst + 8 * D + 2 * g) = make_float2(m, l);
        }
        named_bar_sync(1, kCons);
        if (tid == 0) {
            unsigned before;
            asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(wk.tickets + c0) : "memory");
            bar->last = before == (unsigned)(np - 1);
            if (bar->last) wk.tickets[c0] = 0;
        }
        named_bar_sync(1, kCons);
        if constexpr (C::kOneBuf) q_done();
        if (!bar->last) continue;
        // The join: out = sum_i 2^(m_i - m) O_i / sum_i 2^(m_i - m) l_i, pieces in order, rescaled as the maximum grows.  A thread
        // takes four elements of a row at a time and asks for eight pieces' (m, l) and elements at once: it is trips to L2 that
        // the join consists of.
        constexpr int NV = RB * D / 4 / kCons, kAtOnce = 8, kPair = NV >= 2 ? 2 : 1;
#pragma unroll 1
        for (int v0 = 0; v0 < NV; v0 += kPair) {
            float4 acc[kPair];
            float M[kPair], L[kPair];
            size_t o_at[kPair], ml_at[kPair];
#pragma unroll
            for (int v = 0; v < kPair; v++) {
                const int i = tid + (v0 + v) * kCons, tile = i / (2 * D), at = i % (2 * D);
                o_at[v] = (size_t)tile * C::kTileFloats + 4 * at;
                ml_at[v] = (size_t)tile * C::kTileFloats + 8 * D + ((at & 15) & ~1);
                acc[v] = make_float4(0.f, 0.f, 0.f, 0.f);
                M[v] = -INFINITY;
                L[v] = 0.0f;
            }
#pragma unroll 1
            for (int p = 0; p < np; p += kAtOnce) {
                float4 w[kPair][kAtOnce];
                float2 x[kPair][kAtOnce];
#pragma unroll
                for (int k = 0; k < kAtOnce; k++) {
                    const float* piece = piece_of(kv_min(p + k, np - 1));
#pragma unroll
                    for (int v = 0; v < kPair; v++) {
                        x[v][k] = __ldcg(reinterpret_cast<const float2*>(piece + ml_at[v]));
                        w[v][k] = __ldcg(reinterpret_cast<const float4*>(piece + o_at[v]));
                    }
                }
#pragma unroll
                for (int v = 0; v < kPair; v++) {
                    float mn = M[v];
#pragma unroll
                    for (int k = 0; k < kAtOnce; k++) mn = fmaxf(mn, x[v][k].x);      // (the last piece again past the end)
                    const float base = mn == -INFINITY ? 0.0f : mn, fix = ex2f(M[v] - base);
                    M[v] = mn;
                    acc[v].x *= fix, acc[v].y *= fix, acc[v].z *= fix, acc[v].w *= fix;
                    L[v] *= fix;
#pragma unroll
                    for (int k = 0; k < kAtOnce; k++) {
                        if (p + k < np) {
                            const float f = ex2f(x[v][k].x - base);
                            L[v] = fmaf(x[v][k].y, f, L[v]);
                            acc[v].x = fmaf(w[v][k].x, f, acc[v].x);
                            acc[v].y = fmaf(w[v][k].y, f, acc[v].y);
                            acc[v].z = fmaf(w[v][k].z, f, acc[v].z);
                            acc[v].w = fmaf(w[v][k].w, f, acc[v].w);
                        }
                    }
                }
            }
#pragma unroll
            for (int v = 0; v < kPair; v++) {
                const int i = tid + (v0 + v) * kCons, at = i % (2 * D), r = i / (2 * D) * 8 + (at & 15) / 2, e = (at >> 4) * 8 + (at & 1) * 4;
                if (r >= b.rows) continue;
                const float inv = L[v] == 0.0f ? 0.0f : 1.0f / L[v];
                const size_t at_out = out_at(r, e);
                if (a.out_bf16) {
                    const __nv_bfloat162 y = __floats2bfloat162_rn(acc[v].x * inv, acc[v].y * inv), z = __floats2bfloat162_rn(acc[v].z * inv, acc[v].w * inv);
                    *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(a.out) + at_out) =
                        make_uint2(*reinterpret_cast<const uint32_t*>(&y), *reinterpret_cast<const uint32_t*>(&z));
                } else {
                    *reinterpret_cast<float4*>(reinterpret_cast<float*>(a.out) + at_out) =
                        make_float4(acc[v].x * inv, acc[v].y * inv, acc[v].z * inv, acc[v].w * inv);
                }
            }
        }
    }
    let_copies_land();
}

// ---------------------------------------------------------------------------------------------------------------------
namespace {
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_tiled_fn()
{
    static EncodeTiledFn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<EncodeTiledFn>(p);
    }();
    return fn;
}

}  // namespace

// [n_pages][heads][page][dim], read in boxes of 64 elements x up to 64 rows of a page (128-byte swizzle).
int32_t encode_cache(CUtensorMap* map, const KvCacheView& c, void* base, const void* stand_in)
{
    EncodeTiledFn enc = encode_tiled_fn();
    if (!enc) {
        set_last_error("the CUDA driver does not export cuTensorMapEncodeTiled");
        return kErrCuda;
    }
    const cuuint64_t page = (cuuint64_t)1 << c.page_shift;
    // a cache without pages: a map of one page that no copy reaches (absent pages have coordinate 1)
    const cuuint64_t dims[4] = {(cuuint64_t)c.dim, page, (cuuint64_t)c.heads, (cuuint64_t)(c.n_pages > 0 ? c.n_pages : 1)};
    const cuuint64_t strides[3] = {(cuuint64_t)c.dim * 2, page * c.dim * 2, (cuuint64_t)c.page_stride * 2};
    const cuuint32_t box[4] = {64, (cuuint32_t)(page < kAttendTile ? page : kAttendTile), 1, 1}, estr[4] = {1, 1, 1, 1};
    const CUresult r = enc(map, c.bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                           c.n_pages > 0 ? base : const_cast<void*>(stand_in), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        set_last_error("cuTensorMapEncodeTiled (cache) failed with code %d", (int)r);
        return kErrCuda;
    }
    return kOk;
}

namespace {
// Two tiles a CTA at least: joining a block of two tiles costs more than its second tile (1 x 100 keys, 40 over 8 heads:
// 12.3 us on sixteen CTAs and eight joins, 8.4 us on eight).
constexpr int kSplitMinTiles = 2;
constexpr size_t kTicketBytes = 8192;   // the split kernel's [2 x SMs], then the prompt kernel's [SMs]

template <typename T, int D, int WM>
size_t split_ws_floats(int sm_count)
{
    return (size_t)sm_count * SplitCfg<T, D, WM>::kMinCtas * 2 * SplitCfg<T, D, WM>::kPieceFloats;
}

template <typename T, int D, int WM>
int32_t launch_split(cudaStream_t st, const KvCacheView& c, const KvSeqsView& s, const RopeView& r, const AttendArgs& a, void* ws,
                     const GemvTuning& tune)
{
    using C = SplitCfg<T, D, WM>;
    static bool attr_done[64] = {};
    int dev = 0;
    FERRIC_CUDA_TRY(cudaGetDevice(&dev));
    if (dev >= 64 || !attr_done[dev]) {
        FERRIC_CUDA_TRY(cudaFuncSetAttribute(attend_split_kernel<T, D, WM>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
        if (dev < 64) attr_done[dev] = true;
    }
    CUtensorMap kmap, vmap;
    int32_t rc;
    if ((rc = encode_cache(&kmap, c, c.k, a.q)) != kOk || (rc = encode_cache(&vmap, c, c.v, a.q)) != kOk) return rc;
    SplitWork wk;
    wk.tickets = reinterpret_cast<unsigned*>(ws);
    wk.pieces = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(ws) + kTicketBytes);
    wk.status = gemm_status_word();
    wk.min_tiles = kSplitMinTiles;
    wk.min_parts = (int)((long long)s.seqs * c.heads < 4096 ? (long long)s.seqs * c.heads : 4096);
    wk.group_recip = (0x100000000ull + (unsigned)(a.heads / c.heads) - 1) / (unsigned)(a.heads / c.heads);
    FERRIC_CUDA_TRY(launch_kernel(attend_split_kernel<T, D, WM>, dim3((unsigned)(tune.sm_count * C::kMinCtas)), dim3(C::kThreads), C::kSmem, st,
                                  tune.pdl, kmap, vmap, c, s, r, a, wk));
    return kOk;
}

template <typename T, int D>
int32_t launch_attend_td(cudaStream_t st, const KvCacheView& c, const KvSeqsView& s, const RopeView& r, const AttendArgs& a, void* ws,
                         const GemvTuning& tune)
{
    // Row tiles of a block: as many as the average sequence's query rows fill.  More would leave MMAs empty and take the keys'
    // share of the warps; fewer would read the keys again for every block.
    const long long rows = ((long long)s.tokens + s.seqs - 1) / s.seqs * (a.heads / c.heads);
    if (rows <= 8) return launch_split<T, D, 1>(st, c, s, r, a, ws, tune);
    if (rows <= 16) return launch_split<T, D, 2>(st, c, s, r, a, ws, tune);
    if (rows <= 32 || D == 256) return launch_split<T, D, 4>(st, c, s, r, a, ws, tune);
    return launch_split<T, D, D == 256 ? 4 : 8>(st, c, s, r, a, ws, tune);
}
}  // namespace

size_t attend_ws_bytes(int sm_count)
{
    const size_t f[] = {split_ws_floats<__half, 64, 8>(sm_count), split_ws_floats<__half, 64, 4>(sm_count), split_ws_floats<__half, 128, 8>(sm_count),
                        split_ws_floats<__half, 128, 4>(sm_count), split_ws_floats<__half, 256, 4>(sm_count)};
    size_t most = 0;
    for (size_t x : f) most = x > most ? x : most;
    const size_t split = most * sizeof(float), prompt = attend_prompt_ws_bytes(sm_count);
    return kTicketBytes + (split > prompt ? split : prompt);
}
size_t attend_ticket_bytes() { return kTicketBytes; }

int32_t launch_attend(cudaStream_t st, const KvCacheView& c, const KvSeqsView& s, const RopeView& r, const AttendArgs& a, void* ws,
                      const GemvTuning& tune, int* launches)
{
    *launches = 1;
    if (attend_prompt_eligible(c, s, a)) return launch_attend_prompt(st, c, s, r, a, ws, kTicketBytes, tune);
    switch (c.dim) {
    case 64: return c.bf16 ? launch_attend_td<__nv_bfloat16, 64>(st, c, s, r, a, ws, tune) : launch_attend_td<__half, 64>(st, c, s, r, a, ws, tune);
    case 128: return c.bf16 ? launch_attend_td<__nv_bfloat16, 128>(st, c, s, r, a, ws, tune) : launch_attend_td<__half, 128>(st, c, s, r, a, ws, tune);
    default: return c.bf16 ? launch_attend_td<__nv_bfloat16, 256>(st, c, s, r, a, ws, tune) : launch_attend_td<__half, 256>(st, c, s, r, a, ws, tune);
    }
}

}  // namespace ferric
