// attend_prompt_kernel: attention of many new tokens (prompts and chunks of them), result in bf16, on tcgen05.
//
// A prompt of 4096 (40 over 8 heads x 128, bf16): 288 us a call = 597 TFLOP/s (267 in a captured graph); chunks of three prompts
// (f16): 227 us = 834 TFLOP/s (208).  At head_dim 256 a prompt of 4096 (16 over 4 heads) takes 254 us in bf16, 202 in f16 (graph).
// Bound by the tensor cores (4 head_dim flop per visible pair and query head), short of it by a block's set-up and end and, in
// bf16, by a ring of three stages.  A CTA takes 256 query rows (head_dim 256:
// 128) of one key-value head -- (token, query head of the group) pairs, so that all heads of the group share the keys it
// reads -- and walks the keys they see in tiles.  Per tile and 128 rows, a "unit": S = Q K^T into tensor memory; one thread
// per row takes the softmax step in registers and writes the weights back over S as 16-bit values; O += P V with P read
// straight from tensor memory and V from shared memory as it lies (rows = keys: the MMA takes it transposed).  There are two
// S buffers, one per row tile, or alternating over the keys where one row tile fills tensor memory: while one unit is with
// its softmax warps the other one's products run.
//
// The maximum of a row only has to keep 2^(s - m) in range, so it moves -- and O is rescaled, a round trip through registers
// -- only when the new one exceeds the old one by more than 2^kSlack; the division by the sum makes up for the rest.
//
// Rounding: the weights are rounded once to the cache's type (they multiply its values on the tensor cores; up to 2^-8 of
// a weight in bf16, as much as the result's own rounding), summed in f32 before that.  q is rounded to f16 for an f16 cache, each
// row scaled by a power of two first (undone on its scores, in the subtraction of the maximum); for a bf16 cache it is split into
// two bf16 parts, since one alone would move every score by up to 2^-8 of its terms.
#include <string.h>

#include <type_traits>

#include "kv.cuh"
#include "tc_common.cuh"

namespace ferric {

int* gemm_status_word();   // device address of the status word shared with the tensor-core products (kernels_gemm.cu)
int32_t encode_cache(CUtensorMap* map, const KvCacheView& c, void* base, const void* stand_in);   // kernels_attend.cu

struct PromptBars {
    uint64_t full[8], empty[8];
    uint64_t s_full[2], p_full[2], pv_done[2], turn[2];
    uint32_t tmem;
    int tainted, last;    // tainted: bit 0 a value that is not finite, bit 1 weights that are NaN
    volatile int abort;   // a wait ran out
    int inf_count, inf_key[32];
};
template <typename T, int D>
struct PromptCfg {
    static constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
    static constexpr int kParts = kBf16 ? 2 : 1;           // 16-bit parts of q
    static constexpr int kTilesQ = D == 256 ? 1 : 2;       // row tiles of 128
    static constexpr int kRows = 128 * kTilesQ;
    static constexpr int kKeys = D == 256 ? 64 : 128;      // keys of a tile
    static constexpr int kSoftWarps = 4 * kTilesQ;
    // Issuing threads: the MMA queue is shallow, so a thread's barrier waits and commits (about 1000 cycles a unit, beside 58
    // for each of its 16 or 24 MMAs) leave the tensor pipe idle.  One thread per row tile, in turns: one waits and commits
    // while the other issues.  (Without turns the two tiles fall into step, products and softmax no longer overlap.)
    static constexpr int kMmaWarps = kTilesQ;
    // Two row tiles make three warpgroups of 168 registers a thread; the softmax's 128 scores a row want more, the issuing and
    // loading warps less, so they trade (2 x 128 x 208 + 128 x 88 = 384 x 168).
    static constexpr bool kTrade = kTilesQ == 2;
    static constexpr int kThreads = kTrade ? 384 : 32 * (kSoftWarps + kMmaWarps + 1);
    static constexpr int kQBytes = kTilesQ * kParts * 128 * D * 2;
    static constexpr int kStageBytes = kKeys * D * 2;      // a tile of K or of V
    static constexpr int kBarBytes = 512;
    static constexpr int kScaleBytes = kBf16 ? 0 : kRows * 4;   // f16: what undoes each row's scaling
    static constexpr int kFixed = 1024 + kBarBytes + kScaleBytes + kQBytes;
    static constexpr int kStagesFit = (232448 - kFixed) / kStageBytes;
    static constexpr int kStages = kStagesFit > 8 ? 8 : kStagesFit;
    static constexpr int kSmem = kFixed + kStages * kStageBytes;
    static constexpr int kOCol = 2 * kKeys;                // tensor memory: S0 | S1 | O (one per row tile)
    static constexpr int kPieceFloats = kRows * (D + 2);   // of a block whose keys several CTAs share: [D / 4][row][4], then m, l
    static_assert(sizeof(PromptBars) <= kBarBytes, "barriers");
    static_assert(kStages >= 3 && kOCol + kTilesQ * D <= 512, "shared and tensor memory");
};
constexpr float kSlack = 6.0f;         // log2 units
constexpr float kPromptShiftF16 = 8.0f;   // f16 weights are scaled by 2^8: at most 2^14 with the slack, normal down to 2^-22

// Few blocks against many keys (a chunk of a prompt on a long cache) would leave most SMs idle: `splits` CTAs then share a
// block's keys, each leaving a piece, and the last one joins them in order.
struct PromptWork {
    float* pieces;       // [block][split][piece]
    unsigned* tickets;   // [block], zero between launches
    int* status;
    int splits;
};
constexpr int kPromptMinTiles = 4;     // per CTA: less is lost in its set-up
constexpr int kPromptMaxSplits = 8;

// B operand whose rows are the summation index (V as it lies, [key][64 elements] swizzled rows): 8-row groups 1024 bytes
// apart, runs of 64 elements `run` bytes apart.
__device__ __forceinline__ uint64_t umma_desc_rows(uint32_t saddr, uint32_t run)
{
    uint64_t d = 0;
    d |= (uint64_t)((saddr & 0x3FFFF) >> 4);
    d |= (uint64_t)(run >> 4) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
__host__ __device__ constexpr uint32_t attend_idesc(bool bf16, int n, bool b_rows)
{
    const uint32_t ty = bf16 ? 1u : 0u;
    return (1u << 4) | (ty << 7) | (ty << 10) | ((b_rows ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}
// D += A B with A (16-bit pairs, lane = row) in tensor memory.
__device__ __forceinline__ void umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate)
{
    asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p; }" ::"r"(tmem_d), "r"(tmem_a),
                 "l"(bdesc), "r"(idesc), "r"(accumulate)
                 : "memory");
}
__device__ __forceinline__ void tmem_ld32_nowait(uint32_t taddr, uint32_t* v)
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
          "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]),
          "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]),
          "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* v)
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
        "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]),
        "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]),
        "r"(v[31])
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* v)
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr), "r"(v[0]),
                 "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]),
                 "r"(v[13]), "r"(v[14]), "r"(v[15])
                 : "memory");
}
// The loads issued before are complete; their registers must not be used earlier, which the empty statements pin down.
template <int N>
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&v)[N])
{
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; i++) asm volatile("" : "+r"(v[i]));
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float x, float y)
{
    if constexpr (BF16) {
        __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        return *reinterpret_cast<uint32_t*>(&h);
    } else {
        return h2_as_u32(__floats2half2_rn(x, y));
    }
}
__device__ __forceinline__ float ex2_approx(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint64_t pack_f32x2(float lo, float hi)
{
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void unpack_f32x2(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t fma_f32x2(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add_f32x2(uint64_t a, uint64_t b)
{
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

template <int N>
__device__ __forceinline__ void regs_more()
{
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_fewer()
{
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

template <typename T, int D>
__global__ void __launch_bounds__(PromptCfg<T, D>::kThreads, 1)
attend_prompt_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, KvCacheView c, KvSeqsView s,
                     RopeView rope, AttendArgs a, PromptWork wk)
{
    using C = PromptCfg<T, D>;
    constexpr bool BF = C::kBf16;
    constexpr int NX = C::kTilesQ, KT = C::kKeys, PRE = 2 / NX, H = D / 64;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t* qs = smem;                              // [tile][part][D / 64][128 rows][128 bytes]
    uint8_t* ring = smem + C::kQBytes;               // [stage][D / 64][KT rows][128 bytes]
    PromptBars* bar = reinterpret_cast<PromptBars*>(ring + C::kStages * C::kStageBytes);
    [[maybe_unused]] float* row_scale = reinterpret_cast<float*>(ring + C::kStages * C::kStageBytes + C::kBarBytes);   // f16: [row]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int group = a.heads / c.heads;

    pdl_launch_dependents();
    pdl_wait();

    // ---- this CTA's block: the heads' blocks side by side, each sequence's longest first, so that short ones fill up the end
    const int head = (int)(blockIdx.x % (unsigned)c.heads);
    int seq = -1, blk = (int)(blockIdx.x / (unsigned)c.heads);
    for (int i0 = 0; i0 < s.seqs; i0 += 32) {   // 32 sequences at a time, every warp for itself
        const int mine = i0 + lane < s.seqs ? attend_blocks(kv_span(s, i0 + lane), group, C::kRows) : 0;
        int incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        const unsigned past = __ballot_sync(0xffffffffu, blk < incl);
        if (past) {
            const int at = __ffs(past) - 1;
            seq = i0 + at;
            blk -= __shfl_sync(0xffffffffu, incl - mine, at);
            break;
        }
        blk -= __shfl_sync(0xffffffffu, incl, 31);
    }
    if (seq < 0) return;
    const KvSpan span = kv_span(s, seq);
    const int nb = attend_blocks(span, group, C::kRows);
    const AttendBlock b = attend_block(c, s, span, group, C::kRows, a.window, nb - 1 - blk);
    const int first_tile = b.lo / KT, all_tiles = kv_max(1, (b.hi + KT - 1) / KT - first_tile);
    const int parts = kv_max(1, kv_min(wk.splits, all_tiles / kPromptMinTiles)), part = (int)blockIdx.y;
    if (part >= parts) return;
    const int t0 = first_tile + all_tiles * part / parts, tiles = first_tile + all_tiles * (part + 1) / parts - t0;
    float4* piece = reinterpret_cast<float4*>(wk.pieces + ((size_t)blockIdx.x * wk.splits + part) * C::kPieceFloats);

    if (warp == C::kSoftWarps) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bar->tmem)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    if (tid == 0) {
        for (int i = 0; i < C::kStages; i++) {
            mbar_init(&bar->full[i], 1);
            mbar_init(&bar->empty[i], C::kMmaWarps);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&bar->s_full[i], 1);
            mbar_init(&bar->p_full[i], 4);
            mbar_init(&bar->pv_done[i], 1);
            mbar_init(&bar->turn[i], 1);
        }
        bar->tainted = bar->abort = bar->inf_count = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // Q: rotated, scaled to log2 units, in 16-bit parts, K-major with a 128-byte swizzle.  A thread takes one token's 16
    // elements of two runs of eight (as in the append), its eight angles serving the token's heads.
    if (warp < C::kSoftWarps) {
        constexpr int kUnits = D / 16;
        const int items = (b.j1 - b.j0 + 1) * kUnits;
        const float scale = a.scale * kLog2e;
        for (int it = tid; it < items; it += 32 * C::kSoftWarps) {
            const int u = it % kUnits, j = b.j0 + it / kUnits, pos = span.pos(j);
            const bool rot = u * 16 < rope.rotary;
            const int ea = rot && !rope.interleaved ? 8 * u : 16 * u;
            const int eb = rot && !rope.interleaved ? (rope.rotary >> 1) + 8 * u : 16 * u + 8;
            float cs[8], sn[8];
            if (rot) {
#pragma unroll
                for (int i = 0; i < 8; i++) rope_cos_sin(rope.turns[8 * u + i], pos, &cs[i], &sn[i]);
            }
            const int g0 = kv_max(0, b.r0 - j * group), g1 = kv_min(group, b.r0 + b.rows - j * group);
            // four heads' loads in flight at a time: a block starts with little else to do
            constexpr int kAhead = 4;
            for (int g4 = g0; g4 < g1; g4 += kAhead) {
                float x[kAhead][16];
#pragma unroll
                for (int i = 0; i < kAhead; i++) {
                    const float* q = a.q + (size_t)(span.first + j) * a.ldq + (size_t)(head * group + kv_min(g4 + i, g1 - 1)) * D;
                    *reinterpret_cast<float4*>(x[i]) = ld_act(reinterpret_cast<const float4*>(q + ea));
                    *reinterpret_cast<float4*>(x[i] + 4) = ld_act(reinterpret_cast<const float4*>(q + ea + 4));
                    *reinterpret_cast<float4*>(x[i] + 8) = ld_act(reinterpret_cast<const float4*>(q + eb));
                    *reinterpret_cast<float4*>(x[i] + 12) = ld_act(reinterpret_cast<const float4*>(q + eb + 4));
                }
#pragma unroll
                for (int i = 0; i < kAhead; i++) {
                    if (g4 + i >= g1) break;
                    if (rot) rope_rotate16(x[i], cs, sn, rope.interleaved);
                    const int row = j * group + g4 + i - b.r0, tile = row >> 7, rr = row & 127;
                    uint8_t* base = qs + tile * (C::kParts * 128 * D * 2) + rr * 128;
#pragma unroll
                    for (int e = 0; e < 16; e++) x[i][e] *= scale;
                    if constexpr (!BF) {   // the row's largest magnitude: its units are in kUnits neighbouring lanes
                        float mx = 0.0f, up, down;
#pragma unroll
                        for (int e = 0; e < 16; e++) mx = fmaxf(mx, fabsf(x[i][e]));
#pragma unroll
                        for (int o = 1; o < kUnits; o <<= 1)
                            mx = fmaxf(mx, __shfl_xor_sync(((1u << kUnits) - 1u) << (lane & ~(kUnits - 1)), mx, o));
                        f16_row_scale(mx, &up, &down);
#pragma unroll
                        for (int e = 0; e < 16; e++) x[i][e] *= up;
                        if (u == 0) row_scale[row] = down;
                    }
#pragma unroll
                    for (int part = 0; part < C::kParts; part++) {
                        uint32_t w[8];
#pragma unroll
                        for (int e = 0; e < 8; e++) {
                            w[e] = pack2<BF>(x[i][2 * e], x[i][2 * e + 1]);
                            if (BF) {
                                x[i][2 * e] -= __uint_as_float(w[e] << 16);
                                x[i][2 * e + 1] -= __uint_as_float(w[e] & 0xffff0000u);
                            }
                        }
                        uint8_t* p = base + part * (128 * D * 2);
                        const int ca = ea >> 3, cb = eb >> 3;
                        *reinterpret_cast<uint4*>(p + (ca >> 3) * (128 * 128) + (((ca & 7) ^ (rr & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
                        *reinterpret_cast<uint4*>(p + (cb >> 3) * (128 * 128) + (((cb & 7) ^ (rr & 7)) << 4)) = make_uint4(w[4], w[5], w[6], w[7]);
                    }
                }
            }
        }
        // rows the block does not have
        if constexpr (!BF) {
            for (int i = b.rows + tid; i < C::kRows; i += 32 * C::kSoftWarps) row_scale[i] = 1.0f;
        }
        for (int i = tid + b.rows * (D / 8); i < C::kRows * (D / 8); i += 32 * C::kSoftWarps) {
            const int row = i / (D / 8), ch = i % (D / 8);
#pragma unroll
            for (int part = 0; part < C::kParts; part++)
                *reinterpret_cast<uint4*>(qs + (row >> 7) * (C::kParts * 128 * D * 2) + part * (128 * D * 2) + (ch >> 3) * (128 * 128) + (row & 127) * 128 +
                                          ((ch & 7) << 4)) = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async();
    }
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = bar->tmem;
    bool dead = false;                        // a wait ran out: wait for nothing more, finish the launch
    auto wait = [&](uint64_t* which, uint32_t parity, int code) {
        if (dead || mbar_wait(which, parity)) return;
        dead = true;
        bar->abort = code;
        if (wk.status) atomicExch(wk.status, code);
    };
    // keys every row of the block sees: tiles inside need no mask
    const int lo_all = kv_seen_lo(span.pos(b.j1), a.window), hi_all = kv_seen_hi(c, s, span.pos(b.j0));

    if (warp >= C::kSoftWarps) {
    if constexpr (C::kTrade) regs_fewer<88>();
    if (warp == C::kSoftWarps + C::kMmaWarps) {
        // ---- loader: K0 (.. K1), then V_j and K_{j + PRE} in turn, the order in which the products first use them
        const int box = kv_min(kAttendTile, 1 << c.page_shift), pp = KT / box, copies = pp * H;
        const int piece = lane % pp, half = (lane / pp) % H;
        int n = 0;
        auto load = [&](const CUtensorMap* map, int j) {
            const int st = n % C::kStages, pos = (t0 + j) * KT + piece * box;
            const int page = kv_page(c, s, seq, pos >> c.page_shift);
            if (n >= C::kStages) wait(&bar->empty[st], ((n / C::kStages) & 1) ^ 1, 50);
            n++;
            if (__any_sync(0xffffffffu, dead)) return;   // its place may still be in use
            if (lane == 0) mbar_expect_tx(&bar->full[st], C::kStageBytes);
            __syncwarp();
            if (lane < copies)
                tma_load_4d(ring + st * C::kStageBytes + half * (KT * 128) + piece * box * 128, map, half * 64, pos & ((1 << c.page_shift) - 1), head,
                            page >= 0 ? page : max(1, c.n_pages), &bar->full[st]);
        };
        for (int j = 0; j < kv_min(PRE, tiles); j++) load(&kmap, j);
        for (int j = 0; j < tiles; j++) {
            const int mine = n;
            load(&vmap, j);
            if (j + PRE < tiles) load(&kmap, j + PRE);
            // A tile that some rows see and others do not: an infinity or NaN among its values would reach all of them through
            // the product.  Such a block is done again key by key (below); the tile cannot be refilled before this warp says so.
            const int k0 = (t0 + j) * KT;
            if (b.j0 != b.j1 && (k0 < lo_all || k0 + KT > hi_all)) {
                const int st = mine % C::kStages;
                wait(&bar->full[st], (mine / C::kStages) & 1, 51);
                bool odd = false;
                for (int i = lane; i < KT * (D / 8); i += 32) {
                    const int row = (i >> 3) % KT, hf = i / (8 * KT);
                    const uint4 w = *reinterpret_cast<const uint4*>(ring + st * C::kStageBytes + hf * (KT * 128) + row * 128 + ((i & 7) << 4));
                    constexpr uint32_t e = BF ? 0x7f80u : 0x7c00u;
                    auto bad = [&](uint32_t v) { return (v & e) == e || (v & (e << 16)) == (e << 16); };
                    if (k0 + row >= b.lo && k0 + row < b.hi) odd |= bad(w.x) || bad(w.y) || bad(w.z) || bad(w.w);
                }
                if (odd) atomicOr(&bar->tainted, 1);
                __syncwarp();
            }
        }
    } else if (warp < C::kSoftWarps + C::kMmaWarps) {
        // ---- products of one row tile: unit j is key tile j.  Its S buffer is the tile's own, or, where one tile fills tensor
        // memory, they alternate; PRE units are issued ahead.  Ring positions: K_j and V_j in the loader's order.
        const int x = warp - C::kSoftWarps;
        const uint32_t qbase = smem_u32(qs), rbase = smem_u32(ring);
        constexpr uint32_t id_s = attend_idesc(BF, KT, false), id_o = attend_idesc(BF, D, true);
        int n = 0;                            // ring position
        auto buffer = [&](int j) { return (j * NX + x) & 1; };
        auto next_stage = [&](int code) {     // the next tile of the ring, landed
            const int st = n % C::kStages;
            wait(&bar->full[st], (n / C::kStages) & 1, code);
            n++;
            return st;
        };
        // MMAs are issued in blocks, tile 0's and tile 1's in turn; block i of tile 0 follows block i - 1 of tile 1
        int block = 0;
        auto my_turn = [&] {
            if (NX == 2 && (x == 1 || block > 0)) wait(&bar->turn[x], (x == 1 ? block : block - 1) & 1, 58);
            block++;
            tc_fence_after();
        };
        auto pass_turn = [&] {
            if (NX == 2 && lane == 0) mbar_arrive(&bar->turn[x ^ 1]);
        };
        auto mma_s = [&](int j, int st) {
            const uint32_t kb = umma_desc_lo(rbase + st * C::kStageBytes);
#pragma unroll
            for (int part = 0; part < C::kParts; part++) {
                const uint32_t qb = umma_desc_lo(qbase + (x * C::kParts + part) * (128 * D * 2));
#pragma unroll
                for (int ks = 0; ks < D / 16; ks++)
                    umma_f16_lo(tmem + buffer(j) * KT, qb + (ks >> 2) * (128 * 128 / 16) + (ks & 3) * 2, kb + (ks >> 2) * (KT * 128 / 16) + (ks & 3) * 2,
                                id_s, part > 0 || ks > 0);
            }
        };
        for (int j = 0; j < kv_min(PRE, tiles); j++) {
            const int st = next_stage(52);
            my_turn();
            if (lane == 0 && !dead) {
                mma_s(j, st);
                umma_commit(&bar->s_full[buffer(j)]);
                umma_commit(&bar->empty[st]);
            }
            pass_turn();
            __syncwarp();
        }
        for (int j = 0; j < tiles; j++) {
            const int sv = next_stage(53);
            // keys outside what any row sees have weight 0; their values must not be infinities or NaN
            const int k0 = (t0 + j) * KT, z0 = kv_max(0, b.lo - k0), z1 = kv_min(KT, b.hi - k0);
            if (z0 > 0 || z1 < KT) {
                for (int i = lane; i < KT * (D / 8); i += 32) {
                    const int row = (i >> 3) % KT, hf = i / (8 * KT);
                    if (row < z0 || row >= z1)
                        *reinterpret_cast<uint4*>(ring + sv * C::kStageBytes + hf * (KT * 128) + row * 128 + ((i & 7) << 4)) = make_uint4(0, 0, 0, 0);
                }
                fence_proxy_async();
                __syncwarp();
            }
            const bool more = j + PRE < tiles;
            const int sk = more ? next_stage(52) : 0;
            wait(&bar->p_full[buffer(j)], ((j * NX + x) >> 1) & 1, 54);
            my_turn();
            if (lane == 0 && !dead) {
                const uint64_t vd = umma_desc_rows(rbase + sv * C::kStageBytes, KT * 128);
#pragma unroll
                for (int kk = 0; kk < KT / 16; kk++)
                    umma_ts(tmem + C::kOCol + x * D, tmem + buffer(j) * KT + kk * 8, vd + kk * (2048 / 16), id_o, j > 0 || kk > 0);
                umma_commit(&bar->empty[sv]);   // before S: the tile after next is waiting for this stage
                if (more) mma_s(j + PRE, sk);
            }
            pass_turn();
            if (lane == 0 && !dead) {
                if (more) {
                    umma_commit(&bar->s_full[buffer(j + PRE)]);
                    umma_commit(&bar->empty[sk]);
                }
                if (PRE == 2 || !more) umma_commit(&bar->pv_done[x]);
            }
            __syncwarp();
        }
    }
    // Back to the launch's split, one warpgroup at a time and only when all of its warps are here: a warp without a role that
    // asked for its registers back early would take what the softmax is waiting for.
    if constexpr (C::kTrade) {
        named_bar_sync(1, 128);
        regs_more<168>();
    }
    } else {
        // ---- softmax: thread = row
        if constexpr (C::kTrade) regs_more<208>();
        const int x = warp >> 2, row = x * 128 + (warp & 3) * 32 + lane, r = b.r0 + row;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const int j_tok = r / group;
        const bool have = row < b.rows;
        const int lo_r = have ? kv_seen_lo(span.pos(j_tok), a.window) : 0, hi_r = have ? kv_seen_hi(c, s, span.pos(j_tok)) : 0;
        const int run = kv_min(KT == 128 ? 7 : 6, c.page_shift), pages = KT >> run;
        constexpr float kShift = BF ? 0.0f : kPromptShiftF16;
        const float undo = BF ? 1.0f : row_scale[row];
        const uint64_t undo2 = pack_f32x2(undo, undo);
        float m = -INFINITY, l = 0.0f;      // weights are 2^(s - m)
        for (int j = 0; j < tiles; j++) {
            const int u = j * NX + x, sb = u & 1, k0 = (t0 + j) * KT;
            const unsigned valid = __ballot_sync(0xffffffffu, lane < pages && kv_page(c, s, seq, (k0 + (lane << run)) >> c.page_shift) >= 0);
            wait(&bar->s_full[sb], (u >> 1) & 1, 55);
            tc_fence_after();
            const uint32_t s_col = tmem + lanes + sb * KT;
            const bool masked = k0 < lo_all || k0 + KT > hi_all || valid != (1u << pages) - 1u;
            auto mask = [&](uint32_t* w, int i0, int count) {   // scores of keys this row does not see
#pragma unroll
                for (int i = 0; i < count; i++) {
                    const int key = k0 + i0 + i;
                    const bool page = (valid >> ((i0 + i) >> run)) & 1u;
                    if (!(key >= lo_r && key < hi_r && page)) w[i] = 0xff800000u;   // -inf
                }
            };
            uint32_t w[KT];
#pragma unroll
            for (int i = 0; i < KT / 32; i++) tmem_ld32_nowait(s_col + 32 * i, w + 32 * i);
            tmem_wait_ld(w);
            if (masked) mask(w, 0, KT);
            float mq[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int i = 0; i < KT; i += 2)
                asm("max.f32 %0, %0, %1, %2;" : "+f"(mq[(i >> 1) & 3]) : "f"(__uint_as_float(w[i])), "f"(__uint_as_float(w[i + 1])));
            const float mx = fmaxf(fmaxf(mq[0], mq[1]), fmaxf(mq[2], mq[3])) * undo - kShift;
            // O may be touched once the unit before has been added.  Where S runs one unit ahead, S itself says so: its commit
            // covers what the thread issued before.  Where it runs two ahead, pv_done does.  A parity only tells neighbouring
            // phases apart, so every phase of that is waited for once, in order, and before this unit's weights are handed
            // over: its own products cannot have completed by then, and no wait finds the barrier more than one phase away.
            bool summed = PRE == 1 || j == 0;
            auto wait_summed = [&] {
                if (!summed) wait(&bar->pv_done[x], (j - 1) & 1, 56);
                summed = true;
            };
            const bool move = mx > m + kSlack || (m == -INFINITY && mx > m);
            if (__any_sync(0xffffffffu, move)) {
                const float mn = move ? mx : m, fix = move ? ex2_approx(m - mn) : 1.0f;
                m = mn;
                l *= fix;
                if (j > 0) {
                    wait_summed();
                    tc_fence_after();
#pragma unroll 1
                    for (int i = 0; i < D / 32; i++) {
                        uint32_t v[32];
                        tmem_ld32_nowait(tmem + lanes + C::kOCol + x * D + 32 * i, v);
                        tmem_wait_ld(v);
#pragma unroll
                        for (int e = 0; e < 32; e++) v[e] = __float_as_uint(__uint_as_float(v[e]) * fix);
                        tmem_st32(tmem + lanes + C::kOCol + x * D + 32 * i, v);
                    }
                }
            }
            const float base = m == -INFINITY ? 0.0f : m;
            const uint64_t minus = pack_f32x2(-base, -base);
            uint64_t sum[2] = {0, 0};
#pragma unroll
            for (int i = 0; i < KT / 2; i++) {
                const uint64_t s2 = pack_f32x2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
                const uint64_t x = BF ? add_f32x2(s2, minus) : fma_f32x2(s2, undo2, minus);
                float p0, p1;
                unpack_f32x2(x, p0, p1);
                p0 = ex2_approx(p0);
                p1 = ex2_approx(p1);
                sum[i & 1] = add_f32x2(sum[i & 1], pack_f32x2(p0, p1));
                w[i] = pack2<BF>(p0, p1);
                if (i % 16 == 15) tmem_st16(s_col + (i - 15), w + (i - 15));
            }
            {
                float a0, a1;
                unpack_f32x2(add_f32x2(sum[0], sum[1]), a0, a1);
                l += a0 + a1;
            }
            tmem_wait_st();
            wait_summed();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar->p_full[sb]);
        }
        wait(&bar->pv_done[x], PRE == 2 ? (tiles - 1) & 1 : 0, 57);
        tc_fence_after();
        // an infinite key: q's parts (or an element rounded to 0) make inf - inf or 0 inf of what may be a score of -inf (see below)
        if (have && l != l) atomicOr(&bar->tainted, 2);
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        // The result goes through the tile's place of Q, done with since its last S: written row by row as tensor memory
        // holds it (16-byte chunks, permuted so that eight rows do not meet in a bank), stored row-contiguously.
        uint8_t* stage = qs + x * (C::kParts * 128 * D * 2) + (warp & 3) * 32 * (D * 2);
#pragma unroll 1
        for (int i = 0; i < D / 32; i++) {
            uint32_t v[32];
            tmem_ld32_nowait(tmem + lanes + C::kOCol + x * D + 32 * i, v);
            tmem_wait_ld(v);
            if (parts > 1) {
#pragma unroll
                for (int e = 0; e < 8; e++)
                    piece[(size_t)(8 * i + e) * C::kRows + row] = make_float4(__uint_as_float(v[4 * e]), __uint_as_float(v[4 * e + 1]),
                                                                             __uint_as_float(v[4 * e + 2]), __uint_as_float(v[4 * e + 3]));
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    uint32_t y[4];
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        y[k] = pack2<true>(__uint_as_float(v[8 * e + 2 * k]) * inv, __uint_as_float(v[8 * e + 2 * k + 1]) * inv);
                    *reinterpret_cast<uint4*>(stage + lane * (D * 2) + (((4 * i + e) ^ (lane & 7)) << 4)) = make_uint4(y[0], y[1], y[2], y[3]);
                }
            }
        }
        if (parts == 1) {
            __syncwarp();
            unsigned long long mine = 0;      // where this lane's row goes
            if (have)
                mine = reinterpret_cast<unsigned long long>(reinterpret_cast<__nv_bfloat16*>(a.out) + (size_t)(span.first + j_tok) * a.ldo +
                                                            (size_t)(head * group + r % group) * D);
            constexpr int kLanes = D / 8;     // of a row
#pragma unroll 4
            for (int i = 0; i < kLanes; i++) {
                const int rr = i * (32 / kLanes) + lane / kLanes, ch = lane % kLanes;
                const unsigned long long to = __shfl_sync(0xffffffffu, mine, rr);
                if (to) *reinterpret_cast<uint4*>(to + 16 * ch) = *reinterpret_cast<const uint4*>(stage + rr * (D * 2) + ((ch ^ (rr & 7)) << 4));
            }
        }
        if (parts > 1) reinterpret_cast<float2*>(piece + (size_t)(D / 4) * C::kRows)[row] = make_float2(m, l);
        tc_fence_before();
        if constexpr (C::kTrade) {
            named_bar_sync(2 + x, 128);
            regs_fewer<168>();
        }
    }
    __syncthreads();
    if (bar->abort) {
        for (int i = 0; i < 200; i++) __nanosleep(1000);   // let copies and products still in flight finish
        __syncthreads();
    }
    if (warp == C::kSoftWarps)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    const int tainted = bar->tainted;
    if (tainted == 2) {   // NaN is right, unless infinite keys made it where their scores are -inf
        list_infinite_keys<T, D>(c, s, seq, head, kv_max(b.lo, t0 * KT), kv_min(b.hi, (t0 + tiles) * KT), warp, C::kThreads / 32, lane, &bar->inf_count,
                                 bar->inf_key, 32);
        __syncthreads();
    }
    const int infs = bar->inf_count;
    if ((tainted & 1) || infs > 0) {
        // the rows one by one, key by key (what was stored above is overwritten)
        float* q = reinterpret_cast<float*>(qs) + warp * D;
        for (int row = warp; row < b.rows; row += C::kThreads / 32) {
            const int j = (b.r0 + row) / group, h = head * group + (b.r0 + row) % group, pos = span.pos(j);
            const float* src = a.q + (size_t)(span.first + j) * a.ldq + (size_t)h * D;
            __syncwarp();
            for (int e = lane; e < D; e += 32) q[e] = rope_element(rope, src, e, pos) * (a.scale * kLog2e);
            __syncwarp();
            const int lo = kv_seen_lo(pos, a.window), hi = kv_seen_hi(c, s, pos);
            if (!(tainted & 1) && !infinite_keys_weigh_nothing<T, D>(c, s, seq, head, q, lo, hi, infs, bar->inf_key, lane)) continue;
            float m, l, acc[D / 32];
            attend_row_plain<T, D>(c, s, seq, head, q, kv_max(lo, t0 * KT), kv_min(hi, (t0 + tiles) * KT), lane, &m, &l, acc);
            if (parts > 1) {
#pragma unroll
                for (int e = 0; e < D / 32; e++) {
                    const int at = lane + 32 * e;
                    reinterpret_cast<float*>(piece + (size_t)(at / 4) * C::kRows + row)[at & 3] = acc[e];
                }
                if (lane == 0) reinterpret_cast<float2*>(piece + (size_t)(D / 4) * C::kRows)[row] = make_float2(m, l);
            } else {
                const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(a.out) + (size_t)(span.first + j) * a.ldo + (size_t)h * D;
#pragma unroll
                for (int e = 0; e < D / 32; e++) out[lane + 32 * e] = __float2bfloat16_rn(acc[e] * inv);
            }
        }
    }
    if (parts == 1) return;
    // ---- the join, by the CTA that finishes last: out = sum_i 2^(m_i - m) O_i / sum_i 2^(m_i - m) l_i, thread = row
    __syncthreads();
    if (tid == 0) {
        unsigned before;
        asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(wk.tickets + blockIdx.x) : "memory");
        bar->last = before == (unsigned)(parts - 1);
        if (bar->last) wk.tickets[blockIdx.x] = 0;
    }
    __syncthreads();
    if (!bar->last || tid >= b.rows) return;
    const float4* p0 = reinterpret_cast<const float4*>(wk.pieces + (size_t)blockIdx.x * wk.splits * C::kPieceFloats) + tid;
    float f[kPromptMaxSplits], mx = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kPromptMaxSplits; i++) {
        const float2 ml = i < parts ? __ldcg(reinterpret_cast<const float2*>(p0 - tid + (size_t)i * (C::kPieceFloats / 4) + (size_t)(D / 4) * C::kRows) + tid)
                                    : make_float2(-INFINITY, 0.0f);
        f[i] = ml.x;
        mx = fmaxf(mx, ml.x);
    }
    const float base = mx == -INFINITY ? 0.0f : mx;
#pragma unroll
    for (int i = 0; i < kPromptMaxSplits; i++) {
        f[i] = ex2_approx(f[i] - base);
        if (i < parts)
            sum = fmaf(__ldcg(reinterpret_cast<const float2*>(p0 - tid + (size_t)i * (C::kPieceFloats / 4) + (size_t)(D / 4) * C::kRows) + tid).y, f[i], sum);
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    const int r = b.r0 + tid;
    __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(a.out) + (size_t)(span.first + r / group) * a.ldo + (size_t)(head * group + r % group) * D;
#pragma unroll 2
    for (int e = 0; e < D / 4; e++) {
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int i = 0; i < kPromptMaxSplits; i++) {
            if (i < parts) {
                const float4 v = __ldcg(p0 + (size_t)i * (C::kPieceFloats / 4) + (size_t)e * C::kRows);
                acc.x = fmaf(v.x, f[i], acc.x);
                acc.y = fmaf(v.y, f[i], acc.y);
                acc.z = fmaf(v.z, f[i], acc.z);
                acc.w = fmaf(v.w, f[i], acc.w);
            }
        }
        *reinterpret_cast<uint2*>(out + 4 * e) = make_uint2(pack2<true>(acc.x * inv, acc.y * inv), pack2<true>(acc.z * inv, acc.w * inv));
    }
}

namespace {
template <typename T, int D>
int32_t launch_prompt(cudaStream_t st, const KvCacheView& c, const KvSeqsView& s, const RopeView& r, const AttendArgs& a, void* ws, size_t ticket_bytes,
                      const GemvTuning& tune)
{
    using C = PromptCfg<T, D>;
    static bool attr_done[64] = {};
    int dev = 0;
    FERRIC_CUDA_TRY(cudaGetDevice(&dev));
    if (dev >= 64 || !attr_done[dev]) {
        FERRIC_CUDA_TRY(cudaFuncSetAttribute(attend_prompt_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
        if (dev < 64) attr_done[dev] = true;
    }
    CUtensorMap kmap, vmap;
    int32_t rc;
    if ((rc = encode_cache(&kmap, c, c.k, a.q)) != kOk || (rc = encode_cache(&vmap, c, c.v, a.q)) != kOk) return rc;
    // the batch's spans are on the device: as many blocks as any could make, those behind the last return at once
    const long long blocks = ((long long)s.tokens * (a.heads / c.heads)) / C::kRows + s.seqs;
    if (blocks * c.heads > INT32_MAX) {
        set_last_error("%d tokens x %d heads is more than one launch covers", s.tokens, a.heads);
        return kErrShape;
    }
    // a block's keys are shared only as far as its CTAs then fit the device at once (one per SM)
    PromptWork wk;
    wk.splits = (int)(tune.sm_count / (blocks * c.heads));
    wk.splits = wk.splits < 1 ? 1 : (wk.splits > kPromptMaxSplits ? kPromptMaxSplits : wk.splits);
    wk.tickets = reinterpret_cast<unsigned*>(reinterpret_cast<uint8_t*>(ws) + ticket_bytes / 2);   // (the first half is the split kernel's)
    wk.pieces = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(ws) + ticket_bytes);
    wk.status = gemm_status_word();
    FERRIC_CUDA_TRY(launch_kernel(attend_prompt_kernel<T, D>, dim3((unsigned)(blocks * c.heads), (unsigned)wk.splits), dim3(C::kThreads), C::kSmem, st, tune.pdl,
                                  kmap, vmap, c, s, r, a, wk));
    return kOk;
}
}  // namespace

// Above 32 query rows a sequence and key-value head the tensor cores' tiles of 128 rows win, or cost little, although most of one is
// empty; where a result is wanted in f32, the split kernel runs.  Measured in a graph, this kernel / the split kernel, us:
//                                       8 sequences x 2000 keys            48 sequences x 2000 keys
//   40 over 8 heads x 128, bf16    30 rows 54 / 57    40 rows 54 / 85     30: 185 / 209   40: 186 / 375
//   40 over 8 heads x 128, f16             50 / 39             50 / 56         162 / 119        162 / 213
//   16 over 2 heads x 256, bf16    32 rows 51 / 65    40 rows 51 / 61     32:  70 / 130   40:  70 / 210
//   16 over 2 heads x 256, f16             49 / 52             49 / 45          53 /  84         54 / 136
//   32 over 8 heads x 64, bf16     32 rows 36 / 30    40 rows 36 / 41     32: 141 /  94   40: 141 / 163
//   32 over 8 heads x 64, f16              35 / 25             35 / 33         132 /  65        132 / 113
// The rows are the batch's average, so what runs for a sequence, and how its weights are rounded, depends on the others.
bool attend_prompt_eligible(const KvCacheView& c, const KvSeqsView& s, const AttendArgs& a)
{
    return a.out_bf16 && ((long long)s.tokens + s.seqs - 1) / s.seqs * (a.heads / c.heads) > 32;
}
size_t attend_prompt_ws_bytes(int sm_count)
{
    const size_t most = PromptCfg<__half, 256>::kPieceFloats > PromptCfg<__half, 128>::kPieceFloats ? PromptCfg<__half, 256>::kPieceFloats
                                                                                                  : PromptCfg<__half, 128>::kPieceFloats;
    return (size_t)sm_count * most * sizeof(float);
}
int32_t launch_attend_prompt(cudaStream_t st, const KvCacheView& c, const KvSeqsView& s, const RopeView& r, const AttendArgs& a, void* ws, size_t ticket_bytes,
                             const GemvTuning& tune)
{
    switch (c.dim) {
    case 64: return c.bf16 ? launch_prompt<__nv_bfloat16, 64>(st, c, s, r, a, ws, ticket_bytes, tune) : launch_prompt<__half, 64>(st, c, s, r, a, ws, ticket_bytes, tune);
    case 128: return c.bf16 ? launch_prompt<__nv_bfloat16, 128>(st, c, s, r, a, ws, ticket_bytes, tune) : launch_prompt<__half, 128>(st, c, s, r, a, ws, ticket_bytes, tune);
    default: return c.bf16 ? launch_prompt<__nv_bfloat16, 256>(st, c, s, r, a, ws, ticket_bytes, tune) : launch_prompt<__half, 256>(st, c, s, r, a, ws, ticket_bytes, tune);
    }
}

}  // namespace ferric
