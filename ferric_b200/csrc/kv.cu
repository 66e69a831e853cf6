// C ABI of the paged key-value cache and the attention over it: argument checks, handles, the workspace.
#include <math.h>
#include <string.h>

#include <new>

#include "../../include/ferric_cuda.h"
#include "common.cuh"
#include "handles.h"
#include "kernels.h"

using namespace ferric;

namespace {

bool misaligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) != 0; }

int32_t cache_view(const ferric_kv_cache* c, KvCacheView* v)
{
    if (!c) {
        set_last_error("NULL cache");
        return kErrInvalidArg;
    }
    if (c->ggml_type != FERRIC_GGML_F16 && c->ggml_type != FERRIC_GGML_BF16) {
        set_last_error("a key-value cache is f16 or bf16, not ggml type %u", c->ggml_type);
        return kErrUnsupportedType;
    }
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) {
        set_last_error("head_dim %zu: 64, 128 and 256 are supported", c->head_dim);
        return kErrShape;
    }
    int shift = 4;
    while (shift <= 8 && ((size_t)1 << shift) != c->page_size) shift++;
    if (shift > 8) {
        set_last_error("page_size %zu: 16, 32, 64, 128 and 256 are supported", c->page_size);
        return kErrShape;
    }
    if (c->n_heads == 0 || c->n_heads > 4096) {
        set_last_error("%zu key-value heads", c->n_heads);
        return kErrShape;
    }
    const size_t dense = c->n_heads * c->page_size * c->head_dim;
    const size_t stride = c->page_stride ? c->page_stride : dense;
    size_t total;
    if (c->n_pages > (size_t)INT32_MAX || __builtin_mul_overflow(c->n_pages, stride, &total) || total > (size_t)INT64_MAX / 2) {
        set_last_error("%zu pages of %zu elements are more than this backend indexes", c->n_pages, stride);
        return kErrShape;
    }
    if (stride < dense || stride % 8 != 0) {
        set_last_error("page_stride %zu must cover a page (%zu elements) and be a multiple of 8", stride, dense);
        return kErrShape;
    }
    if (c->n_pages > 0 && (!c->k_dev || !c->v_dev)) {
        set_last_error("NULL cache memory");
        return kErrInvalidArg;
    }
    if (misaligned(c->k_dev, 16) || misaligned(c->v_dev, 16)) {
        set_last_error("cache memory must be 16-byte aligned");
        return kErrInvalidArg;
    }
    v->k = c->k_dev;
    v->v = c->v_dev;
    v->page_stride = (long long)stride;
    v->n_pages = (int)c->n_pages;
    v->page_shift = shift;
    v->heads = (int)c->n_heads;
    v->dim = (int)c->head_dim;
    v->bf16 = c->ggml_type == FERRIC_GGML_BF16 ? 1 : 0;
    return kOk;
}

int32_t seqs_view(const ferric_kv_seqs* q, const KvCacheView& c, size_t n_tokens, KvSeqsView* v)
{
    if (!q) {
        set_last_error("NULL sequence table");
        return kErrInvalidArg;
    }
    const size_t stride = q->table_stride ? q->table_stride : q->max_pages;
    if (q->n_seqs > (1u << 20) || q->max_pages > (size_t)INT32_MAX || n_tokens > (size_t)INT32_MAX || stride > (size_t)INT32_MAX) {
        set_last_error("%zu sequences x %zu pages, %zu tokens are more than this backend indexes", q->n_seqs, q->max_pages, n_tokens);
        return kErrShape;
    }
    if ((long long)q->max_pages << c.page_shift > kKvMaxPositions) {
        set_last_error("%zu pages of %d positions are more than this backend indexes (2^30 positions)", q->max_pages, 1 << c.page_shift);
        return kErrShape;
    }
    if (stride < q->max_pages) {
        set_last_error("table_stride %zu is shorter than max_pages %zu", stride, q->max_pages);
        return kErrShape;
    }
    if (!q->starts_dev && n_tokens != q->n_seqs) {
        set_last_error("without starts there is one token per sequence: %zu tokens, %zu sequences", n_tokens, q->n_seqs);
        return kErrShape;
    }
    if (q->n_seqs > 0 && (!q->lens_dev || (q->max_pages > 0 && !q->page_table_dev))) {
        set_last_error("NULL lengths or page table");
        return kErrInvalidArg;
    }
    if (misaligned(q->lens_dev, 4) || misaligned(q->page_table_dev, 4) || misaligned(q->starts_dev, 4)) {
        set_last_error("sequence tables must be 4-byte aligned");
        return kErrInvalidArg;
    }
    v->table = q->page_table_dev;
    v->table_stride = (long long)stride;
    v->cols = (int)q->max_pages;
    v->lens = q->lens_dev;
    v->starts = q->starts_dev;
    v->seqs = (int)q->n_seqs;
    v->tokens = (int)n_tokens;
    return kOk;
}

// The context comes last of all checks, so that what else is wrong with a call can be seen without a device.
int32_t rope_view(const ferric_cuda_ctx* ctx, const ferric_rope* r, size_t head_dim, RopeView* v)
{
    if (!ctx) {
        set_last_error("NULL context");
        return kErrInvalidArg;
    }
    if (!r) return kOk;
    if (r->device != ctx->device) {
        set_last_error("rotation lives on device %d, context on device %d", r->device, ctx->device);
        return kErrInvalidArg;
    }
    if ((size_t)r->rotary > head_dim) {
        set_last_error("rotation of %d elements, heads have %zu", r->rotary, head_dim);
        return kErrShape;
    }
    v->turns = r->turns;
    v->rotary = r->rotary;
    v->interleaved = r->interleaved;
    return kOk;
}

// An f32 activation matrix [n, cols] with a row stride; 0 = dense.
int32_t check_rows(const char* what, const float* p, size_t n, size_t cols, size_t* ld)
{
    if (*ld == 0) *ld = cols;
    if (*ld < cols || (*ld & 3) || *ld > (size_t)INT64_MAX / 4 / (n ? n : 1)) {
        set_last_error("row stride %zu of %s must cover its %zu columns and be a multiple of 4", *ld, what, cols);
        return kErrShape;
    }
    if (n > 0 && !p) {
        set_last_error("NULL %s", what);
        return kErrInvalidArg;
    }
    if (misaligned(p, 16)) {
        set_last_error("%s must be 16-byte aligned", what);
        return kErrInvalidArg;
    }
    return kOk;
}

// Whether n rows of `a_bytes` every `a_pitch` share memory with n rows of `b_bytes` every `b_pitch` (columns of one wider matrix
// do not; other interleavings count as sharing).
bool rows_overlap(const void* a, size_t a_pitch, size_t a_bytes, const void* b, size_t b_pitch, size_t b_bytes, size_t n)
{
    const uintptr_t a0 = reinterpret_cast<uintptr_t>(a), a1 = a0 + (n - 1) * a_pitch + a_bytes;
    const uintptr_t b0 = reinterpret_cast<uintptr_t>(b), b1 = b0 + (n - 1) * b_pitch + b_bytes;
    if (a1 <= b0 || b1 <= a0) return false;
    if (a_pitch != b_pitch) return true;
    const uintptr_t d = b0 >= a0 ? (b0 - a0) % a_pitch : (a_pitch - (a0 - b0) % a_pitch) % a_pitch;   // b's columns from a's first
    return d < a_bytes || d + b_bytes > a_pitch;
}

}  // namespace

extern "C" {

int32_t ferric_cuda_rope_create(ferric_cuda_ctx* ctx, size_t rotary, double base, const double* inv_freq, int32_t interleaved,
                                ferric_rope** out)
{
    if (!ctx || !out) {
        set_last_error("NULL context or output pointer");
        return kErrInvalidArg;
    }
    *out = nullptr;
    if (rotary == 0 || rotary % 16 != 0 || rotary > 256) {
        set_last_error("rotary %zu must be a multiple of 16, at most 256", rotary);
        return kErrShape;
    }
    if (!inv_freq && !(base > 0.0 && base < INFINITY)) {
        set_last_error("base %g must be positive and finite", base);
        return kErrInvalidArg;
    }
    double turns[128];
    for (size_t i = 0; i < rotary / 2; i++) {
        const double f = inv_freq ? inv_freq[i] : pow(base, -2.0 * (double)i / (double)rotary);
        if (!isfinite(f)) {
            set_last_error("frequency %zu is not finite", i);
            return kErrInvalidArg;
        }
        turns[i] = f / (2.0 * M_PI);
    }
    DeviceGuard guard(ctx->device);
    if (!guard.ok) return cuda_fail(cudaGetLastError(), "cudaSetDevice");
    cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
    FERRIC_CUDA_TRY(cudaStreamIsCapturing(ctx->stream, &cap));
    if (cap != cudaStreamCaptureStatusNone) {
        set_last_error("a rotation allocates and synchronises: create it before capturing");
        return kErrInvalidArg;
    }
    ferric_rope* r = new (std::nothrow) ferric_rope;
    if (!r) return kErrOom;
    r->device = ctx->device;
    r->rotary = (int)rotary;
    r->interleaved = interleaved != 0;
    cudaError_t e = cudaMalloc(reinterpret_cast<void**>(&r->turns), sizeof(double) * (rotary / 2));
    // The copy is waited for on its stream: cudaMemcpy from pageable memory may return with the transfer to the device still
    // to come, and the streams that use the rotation are not ordered behind it.
    if (e == cudaSuccess) e = cudaMemcpyAsync(r->turns, turns, sizeof(double) * (rotary / 2), cudaMemcpyHostToDevice, ctx->stream);
    if (e == cudaSuccess) e = cudaStreamSynchronize(ctx->stream);
    if (e != cudaSuccess) {
        if (r->turns) cudaFree(r->turns);
        delete r;
        return cuda_fail(e, "rope_create");
    }
    *out = r;
    return kOk;
}

void ferric_cuda_rope_free(ferric_rope* r)
{
    if (!r) return;
    DeviceGuard guard(r->device);
    cudaFree(r->turns);
    delete r;
}

int32_t ferric_cuda_kv_append(ferric_cuda_ctx* ctx, const ferric_kv_cache* cache, const ferric_kv_seqs* seqs, const ferric_rope* rope,
                              const float* k_dev, size_t ldk, const float* v_dev, size_t ldv, size_t n_tokens)
{
    KvCacheView c;
    KvSeqsView s;
    RopeView r;
    int32_t rc;
    if ((rc = cache_view(cache, &c)) != kOk || (rc = seqs_view(seqs, c, n_tokens, &s)) != kOk) return rc;
    const size_t cols = cache->n_heads * cache->head_dim;
    if ((rc = check_rows("k", k_dev, n_tokens, cols, &ldk)) != kOk || (rc = check_rows("v", v_dev, n_tokens, cols, &ldv)) != kOk) return rc;
    if ((rc = rope_view(ctx, rope, cache->head_dim, &r)) != kOk) return rc;
    if (n_tokens == 0 || s.seqs == 0 || s.cols == 0 || c.n_pages == 0) return kOk;
    DeviceGuard guard(ctx->device);
    if (!guard.ok) return cuda_fail(cudaGetLastError(), "cudaSetDevice");
    rc = launch_kv_append(ctx->stream, c, s, r, k_dev, ldk, v_dev, ldv, ctx->tune);
    if (rc == kOk) ctx->launches++;
    return rc;
}

int32_t ferric_cuda_attend_reserve(ferric_cuda_ctx* ctx)
{
    if (!ctx) {
        set_last_error("NULL context");
        return kErrInvalidArg;
    }
    if (ctx->attend_ws) return kOk;
    DeviceGuard guard(ctx->device);
    if (!guard.ok) return cuda_fail(cudaGetLastError(), "cudaSetDevice");
    cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
    FERRIC_CUDA_TRY(cudaStreamIsCapturing(ctx->stream, &cap));
    if (cap != cudaStreamCaptureStatusNone) {
        set_last_error("the attention's workspace is not allocated yet: call ferric_cuda_attend_reserve (or attend once) before capturing");
        return kErrInvalidArg;
    }
    if (!ctx->attend_event) FERRIC_CUDA_TRY(cudaEventCreateWithFlags(&ctx->attend_event, cudaEventDisableTiming));
    void* ws = nullptr;
    FERRIC_CUDA_TRY(cudaMalloc(&ws, attend_ws_bytes(ctx->tune.sm_count)));
    cudaError_t e = cudaMemsetAsync(ws, 0, attend_ticket_bytes(), ctx->stream);
    if (e == cudaSuccess) e = cudaStreamSynchronize(ctx->stream);
    if (e != cudaSuccess) {
        cudaFree(ws);
        return cuda_fail(e, "attend_reserve");
    }
    ctx->attend_ws = ws;
    return kOk;
}

int32_t ferric_cuda_kv_attend(ferric_cuda_ctx* ctx, const ferric_kv_cache* cache, const ferric_kv_seqs* seqs, const ferric_rope* rope,
                              const float* q_dev, size_t ldq, size_t n_tokens, size_t n_q_heads, float scale, size_t window,
                              void* out_dev, uint32_t out_type, size_t ldo)
{
    KvCacheView c;
    KvSeqsView s;
    RopeView r;
    AttendArgs a;
    int32_t rc;
    if ((rc = cache_view(cache, &c)) != kOk || (rc = seqs_view(seqs, c, n_tokens, &s)) != kOk) return rc;
    if (n_q_heads == 0 || n_q_heads % cache->n_heads != 0 || n_q_heads > 16384) {
        set_last_error("%zu query heads over %zu key-value heads", n_q_heads, cache->n_heads);
        return kErrShape;
    }
    const size_t cols = n_q_heads * cache->head_dim;
    if ((rc = check_rows("q", q_dev, n_tokens, cols, &ldq)) != kOk) return rc;
    if (out_type != FERRIC_GGML_F32 && out_type != FERRIC_GGML_BF16) {
        set_last_error("the result is f32 or bf16, not ggml type %u", out_type);
        return kErrUnsupportedType;
    }
    const size_t out_size = out_type == FERRIC_GGML_F32 ? 4 : 2;
    if (ldo == 0) ldo = cols;
    if (ldo < cols || (ldo * out_size) % 16 != 0 || ldo > (size_t)INT64_MAX / 4 / (n_tokens ? n_tokens : 1)) {
        set_last_error("row stride %zu of the result must cover its %zu columns and be a multiple of 16 bytes", ldo, cols);
        return kErrShape;
    }
    if (n_tokens > 0 && !out_dev) {
        set_last_error("NULL result");
        return kErrInvalidArg;
    }
    if (misaligned(out_dev, 16)) {
        set_last_error("the result must be 16-byte aligned");
        return kErrInvalidArg;
    }
    if (n_tokens > 0 && rows_overlap(q_dev, ldq * 4, cols * 4, out_dev, ldo * out_size, cols * out_size, n_tokens)) {
        set_last_error("the result overlaps q, which other rows still need");
        return kErrInvalidArg;
    }
    if (!isfinite(scale)) {
        set_last_error("scale %g is not finite", (double)scale);
        return kErrInvalidArg;
    }
    if ((rc = rope_view(ctx, rope, cache->head_dim, &r)) != kOk) return rc;
    if (n_tokens == 0 || s.seqs == 0) return kOk;
    a.q = q_dev;
    a.ldq = ldq;
    a.out = out_dev;
    a.ldo = ldo;
    a.out_bf16 = out_type == FERRIC_GGML_BF16;
    a.heads = (int)n_q_heads;
    a.scale = scale == 0.0f ? 1.0f / sqrtf((float)cache->head_dim) : scale;
    a.window = window > (size_t)INT32_MAX ? 0 : (int)window;   // a window past every position hides nothing
    DeviceGuard guard(ctx->device);
    if (!guard.ok) return cuda_fail(cudaGetLastError(), "cudaSetDevice");
    if ((rc = ferric_cuda_attend_reserve(ctx)) != kOk) return rc;
    int launched = 0;
    rc = launch_attend(ctx->stream, c, s, r, a, ctx->attend_ws, ctx->tune, &launched);
    if (rc == kOk) {
        ctx->launches += launched;
        ctx->attend_used = true;
    }
    return rc;
}

}  // extern "C"
