// Appending to the paged key-value cache: the new tokens' keys are rotated to their positions and both are rounded to the
// cache's 16-bit type on the way in, straight from the q|k|v product's f32 result.
#include "kv.cuh"

namespace ferric {

// k' = R(pos) k, v' = v, one rounding each (the cache's type is the user's choice; the rotation itself is in f32 with its
// angle in 64 bits).  Bound by HBM for many tokens (8 bytes read and 4 written per element of k and v) and by the launch
// and one chain of loads (lengths -> page -> row) for few.  A thread takes 16 elements of a head: a rotated unit is eight
// pairs -- two runs of eight elements half the rotated width apart, or one run of sixteen for adjacent pairs -- so reads are
// two or four float4 and writes are 16 bytes, and its eight angles serve `h_per` heads.  A token row outside every
// sequence, or a position without a page, writes nothing.
template <typename T>
__global__ void __launch_bounds__(256) kv_append_kernel(KvCacheView c, KvSeqsView s, RopeView r, const float* __restrict__ k, size_t ldk,
                                                        const float* __restrict__ v, size_t ldv, int units, int h_slots, int h_per)
{
    pdl_launch_dependents();
    pdl_wait();
    const long long item = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    const int u = (int)(item % units);
    const long long rest = item / units;
    const int hs = (int)(rest % h_slots);
    const long long tl = rest / h_slots;
    if (tl >= s.tokens) return;
    const int t = (int)tl;
    const int seq = kv_seq_of(s, t);
    if (seq < 0) return;
    const KvSpan sp = kv_span(s, seq);
    const int pos = sp.pos(t - sp.first);
    const long long off0 = kv_offset(c, s, seq, 0, pos);
    if (off0 < 0) return;
    const bool rot = u * 16 < r.rotary;
    // elements of the two runs of eight
    const int ea = rot && !r.interleaved ? 8 * u : 16 * u;
    const int eb = rot && !r.interleaved ? (r.rotary >> 1) + 8 * u : 16 * u + 8;
    float cs[8], sn[8];
    if (rot) {
#pragma unroll
        for (int i = 0; i < 8; i++) rope_cos_sin(r.turns[8 * u + i], pos, &cs[i], &sn[i]);
    }
    const long long head_step = (long long)c.dim << c.page_shift;
    T* kc = reinterpret_cast<T*>(c.k);
    T* vc = reinterpret_cast<T*>(c.v);
    for (int i = 0; i < h_per; i++) {
        const int h = hs + i * h_slots;
        if (h >= c.heads) break;
        const float* kr = k + (size_t)t * ldk + (size_t)h * c.dim;
        const float* vr = v + (size_t)t * ldv + (size_t)h * c.dim + 16 * u;
        float a[16], w[16];
        *reinterpret_cast<float4*>(a) = ld_act(reinterpret_cast<const float4*>(kr + ea));
        *reinterpret_cast<float4*>(a + 4) = ld_act(reinterpret_cast<const float4*>(kr + ea + 4));
        *reinterpret_cast<float4*>(a + 8) = ld_act(reinterpret_cast<const float4*>(kr + eb));
        *reinterpret_cast<float4*>(a + 12) = ld_act(reinterpret_cast<const float4*>(kr + eb + 4));
#pragma unroll
        for (int e = 0; e < 4; e++) *reinterpret_cast<float4*>(w + 4 * e) = ld_act(reinterpret_cast<const float4*>(vr + 4 * e));
        if (rot) rope_rotate16(a, cs, sn, r.interleaved);
        T ko[16], vo[16];
#pragma unroll
        for (int e = 0; e < 16; e++) {
            kv_from_float(a[e], &ko[e]);
            kv_from_float(w[e], &vo[e]);
        }
        const long long off = off0 + h * head_step;
        *reinterpret_cast<uint4*>(kc + off + ea) = *reinterpret_cast<const uint4*>(ko);
        *reinterpret_cast<uint4*>(kc + off + eb) = *reinterpret_cast<const uint4*>(ko + 8);
        *reinterpret_cast<uint4*>(vc + off + 16 * u) = *reinterpret_cast<const uint4*>(vo);
        *reinterpret_cast<uint4*>(vc + off + 16 * u + 8) = *reinterpret_cast<const uint4*>(vo + 8);
    }
}

int32_t launch_kv_append(cudaStream_t st, const KvCacheView& c, const KvSeqsView& s, const RopeView& r, const float* k, size_t ldk,
                         const float* v, size_t ldv, const GemvTuning& tune)
{
    const int units = c.dim / 16;
    const int h_per = 1, h_slots = c.heads;
    const long long items = (long long)s.tokens * h_slots * units;
    const long long blocks = (items + 255) / 256;
    if (blocks > INT32_MAX) {
        set_last_error("%d tokens x %d heads is more than one launch covers", s.tokens, c.heads);
        return kErrShape;
    }
    auto* fn = c.bf16 ? kv_append_kernel<__nv_bfloat16> : kv_append_kernel<__half>;
    FERRIC_CUDA_TRY(launch_kernel(fn, dim3((unsigned)blocks), dim3(256), 0, st, tune.pdl, c, s, r, k, ldk, v, ldv, units, h_slots, h_per));
    return kOk;
}

}  // namespace ferric
