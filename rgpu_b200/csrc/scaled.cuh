// Handles of the block-scaled matrices: what rt_mx4_* and rt_fp8_* share.
#pragma once

#include <algorithm>
#include <climits>
#include <new>

#include "internal.h"

namespace rt {

inline int check_scaled_extents(const char* what, int64_t rows, int64_t k) {
    RT_CHECK(rows >= 0 && k >= 0, "%s: negative extent %lld x %lld", what, (long long)rows, (long long)k);
    // box coordinates and the block count of a row are 32-bit
    RT_CHECK(rows <= INT_MAX - 256 && k <= INT_MAX - 256, "%s: extent above 2^31 - 257: %lld x %lld", what,
             (long long)rows, (long long)k);
    return RT_OK;
}

// A matrix of zeros: codes of cb bytes and scales of sb in one allocation.
template <typename Q>
int scaled_zeros(rt_ctx* ctx, int64_t rows, int64_t k, size_t cb, size_t sb, int (*encode_maps)(Q*), Q** out) {
    const size_t scales_at = (cb + 511) / 512 * 512;
    RT_CUDA(cudaSetDevice(ctx->device));
    void* p = nullptr;
    cudaError_t e = cudaMalloc(&p, std::max<size_t>(scales_at + sb, 16));
    if (e != cudaSuccess)
        return fail(RT_ERR_OOM, "cudaMalloc(%zu) failed: %s", scales_at + sb, cudaGetErrorString(e));
    e = cudaMemsetAsync(p, 0, std::max<size_t>(scales_at + sb, 16), ctx->stream);
    if (e != cudaSuccess) {
        cudaFree(p);
        return fail(RT_ERR_CUDA, "cudaMemsetAsync failed: %s", cudaGetErrorString(e));
    }
    Q* q = new (std::nothrow) Q;
    if (!q) {
        cudaFree(p);
        return fail(RT_ERR_OOM, "out of host memory");
    }
    q->ctx = ctx;
    q->codes = static_cast<uint8_t*>(p);
    q->scales = q->codes + scales_at;
    q->rows = rows;
    q->k = k;
    q->owned = true;
    const int s = encode_maps(q);
    if (s != RT_OK) {
        cudaFree(p);
        delete q;
        return s;
    }
    *out = q;
    return RT_OK;
}

// A view of caller memory.
template <typename Q>
int scaled_wrap(const char* what, rt_ctx* ctx, void* codes, void* scales, int64_t rows, int64_t k,
                int (*encode_maps)(Q*), Q** out) {
    RT_CHECK((codes && scales) || rows == 0 || k == 0, "%s: codes or scales is NULL", what);
    RT_CHECK(((reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(scales)) & 15) == 0,
             "%s: codes and scales must be 16-byte aligned", what);
    Q* q = new (std::nothrow) Q;
    if (!q) return fail(RT_ERR_OOM, "%s: out of host memory", what);
    q->ctx = ctx;
    q->codes = static_cast<uint8_t*>(codes);
    q->scales = static_cast<uint8_t*>(scales);
    q->rows = rows;
    q->k = k;
    const int s = encode_maps(q);
    if (s != RT_OK) {
        delete q;
        return s;
    }
    *out = q;
    return RT_OK;
}

template <typename Q>
int scaled_free(Q* q) {
    if (!q) return RT_OK;
    if (q->owned) {
        cudaSetDevice(q->ctx->device);
        cudaStreamSynchronize(q->ctx->stream);
        cudaFree(q->codes);
    }
    delete q;
    return RT_OK;
}

// The checks of C = A B^T + bias.
template <typename Q>
int check_scaled_matmul(const char* what, const rt_ctx* ctx, const Q* a, const Q* b, const rt_tensor* c,
                        const rt_tensor* bias) {
    RT_CHECK(ctx && a && b && c, "%s: bad arguments", what);
    RT_CHECK(a->ctx == ctx && b->ctx == ctx && c->ctx == ctx && (!bias || bias->ctx == ctx),
             "tensor belongs to another context");
    RT_CHECK(c->dtype == RT_F32 || c->dtype == RT_BF16, "%s: C must be f32 or bf16", what);
    RT_CHECK(a->k == b->k, "%s: A is %lldx%lld, B %lldx%lld: the second extents differ", what, (long long)a->rows,
             (long long)a->k, (long long)b->rows, (long long)b->k);
    RT_CHECK(c->rows == a->rows && c->cols == b->rows, "%s: C is %lldx%lld, not %lldx%lld", what, (long long)c->rows,
             (long long)c->cols, (long long)a->rows, (long long)b->rows);
    if (bias) {
        RT_CHECK(bias->dtype == RT_F32, "%s: bias must be f32", what);
        RT_CHECK(bias->rows == 1 && bias->cols == b->rows, "%s: bias is %lldx%lld, not 1x%lld", what,
                 (long long)bias->rows, (long long)bias->cols, (long long)b->rows);
    }
    return RT_OK;
}

}  // namespace rt
