// Appending to the paged key-value cache: the new tokens' keys are rotated to their positions and both are rounded to the
// cache's 16-bit type on the way in, straight from the q|k|v product's f32 result.
#include "kv.cuh"

namespace ferric {

// k' = R(pos) k, v' = v, one rounding each (the cache's type is the user's choice; the rotation itself is in f32 with its
// angle in 64 bits).  Bound by HBM for many tokens (8 bytes read and 4 written per element of k and v) and by the launch
// and one chain of loads (lengths -> page) for few.  A thread takes 16 elements of HP heads, k and v: a rotated unit is eight
// pairs -- two runs of eight elements half the rotated width apart, or one run of sixteen for adjacent pairs -- so reads are
// float4, writes are 16 bytes, and the unit's eight angles serve all of its heads.  The rows are requested before the
// lengths and pages are looked up: nothing about where they go decides what is read.  16384 tokens x 8 heads x 128: 36 us =
// 5.6 TB/s; one token 2.3 us on the device.  A token row outside every sequence,
// or a position without a page, writes nothing.
template <typename T, int HP>
__global__ void __launch_bounds__(256) kv_append_kernel(KvCacheView c, KvSeqsView s, RopeView r, const float* __restrict__ k, size_t ldk,
                                                        const float* __restrict__ v, size_t ldv, int unit_shift)
{
    pdl_launch_dependents();
    const unsigned item = blockIdx.x * blockDim.x + threadIdx.x;
    const int u = (int)(item & ((1u << unit_shift) - 1u)), t = (int)(item >> unit_shift), h0 = blockIdx.y * HP;
    const bool rot = u * 16 < r.rotary;
    // elements of the two runs of eight
    const int ea = rot && !r.interleaved ? 8 * u : 16 * u;
    const int eb = rot && !r.interleaved ? (r.rotary >> 1) + 8 * u : 16 * u + 8;
    pdl_wait();
    if (t >= s.tokens) return;
    float a[HP][16], w[HP][16];
#pragma unroll
    for (int i = 0; i < HP; i++) {
        const int h = kv_min(h0 + i, c.heads - 1);
        const float* kr = k + (size_t)t * ldk + (size_t)h * c.dim;
        const float* vr = v + (size_t)t * ldv + (size_t)h * c.dim + 16 * u;
        *reinterpret_cast<float4*>(a[i]) = ld_act(reinterpret_cast<const float4*>(kr + ea));
        *reinterpret_cast<float4*>(a[i] + 4) = ld_act(reinterpret_cast<const float4*>(kr + ea + 4));
        *reinterpret_cast<float4*>(a[i] + 8) = ld_act(reinterpret_cast<const float4*>(kr + eb));
        *reinterpret_cast<float4*>(a[i] + 12) = ld_act(reinterpret_cast<const float4*>(kr + eb + 4));
#pragma unroll
        for (int e = 0; e < 4; e++) *reinterpret_cast<float4*>(w[i] + 4 * e) = ld_act(reinterpret_cast<const float4*>(vr + 4 * e));
    }
    const int seq = kv_seq_of(s, t);
    if (seq < 0) return;
    const KvSpan sp = kv_span(s, seq);
    const int pos = sp.pos(t - sp.first);
    const long long off0 = kv_offset(c, s, seq, 0, pos);
    if (off0 < 0) return;
    if (rot) {
        float cs[8], sn[8];
#pragma unroll
        for (int i = 0; i < 8; i++) rope_cos_sin(r.turns[8 * u + i], pos, &cs[i], &sn[i]);
#pragma unroll
        for (int i = 0; i < HP; i++) rope_rotate16(a[i], cs, sn, r.interleaved);
    }
    const long long head_step = (long long)c.dim << c.page_shift;
    T* kc = reinterpret_cast<T*>(c.k);
    T* vc = reinterpret_cast<T*>(c.v);
#pragma unroll
    for (int i = 0; i < HP; i++) {
        if (h0 + i >= c.heads) break;
        T ko[16], vo[16];
#pragma unroll
        for (int e = 0; e < 16; e++) {
            kv_from_float(a[i][e], &ko[e]);
            kv_from_float(w[i][e], &vo[e]);
        }
        const long long off = off0 + (h0 + i) * head_step;
        *reinterpret_cast<uint4*>(kc + off + ea) = *reinterpret_cast<const uint4*>(ko);
        *reinterpret_cast<uint4*>(kc + off + eb) = *reinterpret_cast<const uint4*>(ko + 8);
        *reinterpret_cast<uint4*>(vc + off + 16 * u) = *reinterpret_cast<const uint4*>(vo);
        *reinterpret_cast<uint4*>(vc + off + 16 * u + 8) = *reinterpret_cast<const uint4*>(vo + 8);
    }
}

int32_t launch_kv_append(cudaStream_t st, const KvCacheView& c, const KvSeqsView& s, const RopeView& r, const float* k, size_t ldk,
                         const float* v, size_t ldv, const GemvTuning& tune)
{
    const int unit_shift = c.dim == 64 ? 2 : (c.dim == 128 ? 3 : 4);
    const long long items = (long long)s.tokens << unit_shift;
    if (items > INT32_MAX) {
        set_last_error("%d tokens are more than one append covers", s.tokens);
        return kErrShape;
    }
    // Two heads a thread halve the angles' arithmetic, once there are threads enough to fill the device's memory pipes.
    const bool two = items * c.heads >= (long long)tune.sm_count * 2048 && c.heads > 1;
    const int threads = items >= 256 ? 256 : 32 * ((int)(items + 31) / 32);
    auto* fn = c.bf16 ? (two ? kv_append_kernel<__nv_bfloat16, 2> : kv_append_kernel<__nv_bfloat16, 1>)
                      : (two ? kv_append_kernel<__half, 2> : kv_append_kernel<__half, 1>);
    FERRIC_CUDA_TRY(launch_kernel(fn, dim3((unsigned)((items + threads - 1) / threads), (unsigned)(two ? (c.heads + 1) / 2 : c.heads)),
                                  dim3((unsigned)threads), 0, st, tune.pdl, c, s, r, k, ldk, v, ldv, unit_shift));
    return kOk;
}

}  // namespace ferric
