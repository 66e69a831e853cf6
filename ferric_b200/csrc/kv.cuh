// What the kernels over the paged key-value cache share: the views they are given, the position rotation and the plain
// evaluation of one query row.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "common.cuh"
#include "kernels.h"

namespace ferric {

// cos and sin of pos * frequency.  The frequencies are held in turns per position in 64 bits: a float product is off by
// 2^-24 of the whole angle, which at position 10^5 is 6e-3 rad; here the whole turns are dropped in 64 bits and the
// rest, at most half a turn, is rounded to a float once.
__device__ __forceinline__ void rope_cos_sin(double turns_per_pos, int pos, float* c, float* s)
{
    const double t = (double)pos * turns_per_pos;
    sincospif(2.0f * (float)(t - rint(t)), s, c);
}
// Rotation partner of element e of a head and where their pair sits among the frequencies; e >= rotary: not rotated.
__device__ __forceinline__ float rope_element(const RopeView& r, const float* x, int e, int pos)
{
    if (e >= r.rotary) return x[e];
    float c, s;
    if (r.interleaved) {
        rope_cos_sin(r.turns[e >> 1], pos, &c, &s);
        return (e & 1) ? fmaf(x[e - 1], s, x[e] * c) : fmaf(-x[e + 1], s, x[e] * c);
    }
    const int half = r.rotary >> 1;
    rope_cos_sin(r.turns[e < half ? e : e - half], pos, &c, &s);
    return e < half ? fmaf(-x[e + half], s, x[e] * c) : fmaf(x[e - half], s, x[e] * c);
}

// Eight pairs at once: the two runs of eight elements x[0..8) and x[8..16) (pairs across the runs), or sixteen adjacent ones.
__device__ __forceinline__ void rope_rotate16(float (&x)[16], const float (&cs)[8], const float (&sn)[8], int interleaved)
{
    if (interleaved) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float a = x[2 * e], b = x[2 * e + 1];
            x[2 * e] = fmaf(-b, sn[e], a * cs[e]);
            x[2 * e + 1] = fmaf(b, cs[e], a * sn[e]);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float a = x[e], b = x[e + 8];
            x[e] = fmaf(-b, sn[e], a * cs[e]);
            x[e + 8] = fmaf(b, cs[e], a * sn[e]);
        }
    }
}

__device__ __forceinline__ float kv_to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float kv_to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void kv_from_float(float v, __half* o) { *o = __float2half_rn(v); }
__device__ __forceinline__ void kv_from_float(float v, __nv_bfloat16* o) { *o = __float2bfloat16_rn(v); }

constexpr float kLog2e = 1.4426950408889634f;

// The power of two that brings a row of q (in log2 units, largest magnitude `mx`) to f16's upper end, and its inverse: any finite
// row fits f16 and keeps the type's 11 bits down to 2^-25 of its largest element, and undoing it on the scores is exact.
__device__ __forceinline__ void f16_row_scale(float mx, float* up, float* down)
{
    // mx < 2^e, from its exponent bits; rows of less than 2^-100 keep that scaling, and one with an infinity stays infinite
    const int e = max((int)(__float_as_uint(mx) >> 23) - 126, -100);
    *up = __uint_as_float((unsigned)(127 + 11 - e) << 23);
    *down = __uint_as_float((unsigned)(127 - 11 + e) << 23);
}

// One query row against keys [lo, hi) of one sequence and head, by one warp, in f32: the definition, key by key.  `q` is
// the rotated row times scale * log2(e), in shared memory.  Lane = key for the scores, lane = dimension for the sums, so a
// masked or absent key is never multiplied by anything.  Leaves the running maximum (log2 units), the sum and the
// unnormalised output (element lane + 32 e).
template <typename T, int D>
__device__ __forceinline__ void attend_row_plain(const KvCacheView& c, const KvSeqsView& s, int seq, int h, const float* q, int lo, int hi,
                                                 int lane, float* m_out, float* l_out, float (&acc)[D / 32])
{
    const T* K = reinterpret_cast<const T*>(c.k);
    const T* V = reinterpret_cast<const T*>(c.v);
    float m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int e = 0; e < D / 32; e++) acc[e] = 0.0f;
    for (int k0 = lo; k0 < hi; k0 += 32) {
        const int key = k0 + lane;
        const long long off = key < hi ? kv_offset(c, s, seq, h, key) : -1;
        float dot = -INFINITY;
        if (off >= 0) {
            dot = 0.0f;
            for (int d = 0; d < D; d += 8) {
                const uint4 w = *reinterpret_cast<const uint4*>(K + off + d);
                const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
                for (int i = 0; i < 8; i++) dot = fmaf(q[d + i], kv_to_float(e[i]), dot);
            }
        }
        float mx = dot;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        mx = fmaxf(mx, m);
        const float base = mx == -INFINITY ? 0.0f : mx;   // nothing seen yet: every term below is 0
        const float fix = exp2f(m - base);
        const float p = off >= 0 ? exp2f(dot - base) : 0.0f;
        l = l * fix + p;
        m = mx;
#pragma unroll
        for (int e = 0; e < D / 32; e++) acc[e] *= fix;
        const unsigned have = __ballot_sync(0xffffffffu, off >= 0);
        for (int i = 0; i < 32; i++) {
            if (!((have >> i) & 1u)) continue;
            const float pi = __shfl_sync(0xffffffffu, p, i);
            const long long oi = __shfl_sync(0xffffffffu, off, i);
#pragma unroll
            for (int e = 0; e < D / 32; e++) acc[e] = fmaf(pi, kv_to_float(V[oi + lane + 32 * e]), acc[e]);
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    *m_out = m;
    *l_out = l;
}

// An infinite key makes inf - inf or 0 inf of q in parts where the score of q itself may be -inf, a weight of 0.  Kernels that see it
// only by a row's weights being NaN look for such keys then, and evaluate again the rows whose scores it spoilt; a NaN key, or one
// with a score of +inf, has NaN for its result as it is.
//
// Keys in [lo, hi) of one sequence and head that hold an infinity: this warp's share (`warps` warps in all) is counted in *n and the
// first `cap` of all are listed.
template <typename T, int D>
__device__ __forceinline__ void list_infinite_keys(const KvCacheView& c, const KvSeqsView& s, int seq, int h, int lo, int hi, int warp, int warps,
                                                   int lane, int* n, int* list, int cap)
{
    constexpr int kLanes = D / 8, kAtOnce = 32 / kLanes;   // of a key; keys a warp reads at once
    constexpr unsigned kAll = kLanes == 32 ? 0xffffffffu : (1u << (kLanes & 31)) - 1u;
    const T* K = reinterpret_cast<const T*>(c.k);
    for (int k0 = lo + warp * kAtOnce; k0 < hi; k0 += warps * kAtOnce) {
        const int key = k0 + lane / kLanes;
        const long long off = key < hi ? kv_offset(c, s, seq, h, key) : -1;
        bool found = false;
        if (off >= 0) {
            const uint4 w = *reinterpret_cast<const uint4*>(K + off + lane % kLanes * 8);
            const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
            for (int i = 0; i < 8; i++) found |= fabsf(kv_to_float(e[i])) == INFINITY;
        }
        const unsigned any = __ballot_sync(0xffffffffu, found);
        if (lane % kLanes == 0 && ((any >> lane) & kAll)) {
            const int at = atomicAdd(n, 1);
            if (at < cap) list[at] = key;
        }
    }
}

// Whether a row of NaN weights, with its `q` (as for attend_row_plain) in shared memory, is to be evaluated again: it sees one of the
// `n` infinite keys (of which 32 are listed), and every one that it sees has a score of -inf.  Otherwise NaN is its result.
template <typename T, int D>
__device__ __forceinline__ bool infinite_keys_weigh_nothing(const KvCacheView& c, const KvSeqsView& s, int seq, int h, const float* q, int lo, int hi,
                                                            int n, const int* list, int lane)
{
    bool sees = n > 32;
    for (int i = 0; i < kv_min(n, 32); i++) {
        const int key = list[i];
        if (key < lo || key >= hi) continue;
        const T* k = reinterpret_cast<const T*>(c.k) + kv_offset(c, s, seq, h, key);
        float dot = 0.0f;
        for (int e = lane; e < D; e += 32) dot = fmaf(q[e], kv_to_float(k[e]), dot);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
        if (!(dot == -INFINITY)) return false;
        sees = true;
    }
    return sees;
}

}  // namespace ferric
