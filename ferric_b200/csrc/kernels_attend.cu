// Attention of the new tokens over the paged key-value cache:
//   out[t, h] = sum_k softmax_k(scale * R(pos_t) q[t, h] . k) v      over the keys token t sees,
// with the softmax taken in one pass over the keys (running maximum m and sum l in f32; the output rescaled by
// 2^(m_old - m_new) when the maximum grows; scores in log2 units, so that the exponential is ex2).
#include "kv.cuh"

namespace ferric {

// One warp per (token, head).
template <typename T, int D>
__global__ void __launch_bounds__(128) attend_plain_kernel(KvCacheView c, KvSeqsView s, RopeView r, AttendArgs a)
{
    __shared__ float qs[4][D];
    pdl_launch_dependents();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long row = (long long)blockIdx.x * 4 + warp;
    if (row >= (long long)s.tokens * a.heads) return;
    const int t = (int)(row / a.heads), h = (int)(row % a.heads);
    const int seq = kv_seq_of(s, t);
    if (seq < 0) return;
    const KvSpan sp = kv_span(s, seq);
    const int pos = sp.pos(t - sp.first);
    const float* q = a.q + (size_t)t * a.ldq + (size_t)h * D;
    const float scale = a.scale * kLog2e;
    for (int e = lane; e < D; e += 32) qs[warp][e] = rope_element(r, q, e, pos) * scale;
    __syncwarp();
    float m, l, acc[D / 32];
    const int lo = kv_seen_lo(pos, a.window), hi = kv_seen_hi(c, s, pos);
    attend_row_plain<T, D>(c, s, seq, h / (a.heads / c.heads), qs[warp], lo, hi, lane, &m, &l, acc);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;   // a token that sees no key: zeros
#pragma unroll
    for (int e = 0; e < D / 32; e++) {
        const size_t o = (size_t)t * a.ldo + (size_t)h * D + lane + 32 * e;
        if (a.out_bf16) reinterpret_cast<__nv_bfloat16*>(a.out)[o] = __float2bfloat16_rn(acc[e] * inv);
        else reinterpret_cast<float*>(a.out)[o] = acc[e] * inv;
    }
}

template <typename T, int D>
static int32_t launch_attend_td(cudaStream_t st, const KvCacheView& c, const KvSeqsView& s, const RopeView& r, const AttendArgs& a,
                                const GemvTuning& tune, int* launches)
{
    const long long blocks = ((long long)s.tokens * a.heads + 3) / 4;
    if (blocks > INT32_MAX) {
        set_last_error("%d tokens x %d heads is more than one launch covers", s.tokens, a.heads);
        return kErrShape;
    }
    FERRIC_CUDA_TRY(launch_kernel(attend_plain_kernel<T, D>, dim3((unsigned)blocks), dim3(128), 0, st, tune.pdl, c, s, r, a));
    *launches = 1;
    return kOk;
}

int32_t launch_attend(cudaStream_t st, const KvCacheView& c, const KvSeqsView& s, const RopeView& r, const AttendArgs& a,
                      const GemvTuning& tune, int* launches)
{
    switch (c.dim) {
    case 64: return c.bf16 ? launch_attend_td<__nv_bfloat16, 64>(st, c, s, r, a, tune, launches) : launch_attend_td<__half, 64>(st, c, s, r, a, tune, launches);
    case 128: return c.bf16 ? launch_attend_td<__nv_bfloat16, 128>(st, c, s, r, a, tune, launches) : launch_attend_td<__half, 128>(st, c, s, r, a, tune, launches);
    default: return c.bf16 ? launch_attend_td<__nv_bfloat16, 256>(st, c, s, r, a, tune, launches) : launch_attend_td<__half, 256>(st, c, s, r, a, tune, launches);
    }
}

}  // namespace ferric
