// Microscaled 4-bit matrices: handles, quantisation and dequantisation.
#include <algorithm>
#include <climits>
#include <new>

#include "mx4.cuh"

namespace rt {
namespace {

using namespace mx4;

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

// One thread per block of 32 elements, and per block that only pads the last
// scale tile (its scale byte becomes 0).
template <typename T>
__global__ void quantize_kernel(const T* __restrict__ src, int64_t row_stride, int64_t k_stride, int64_t rows,
                                int64_t k, int64_t blocks, int64_t groups, uint8_t* __restrict__ codes,
                                uint8_t* __restrict__ scales) {
    const int64_t total = rows * groups * 4;
    for (int64_t idx = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; idx < total;
         idx += (int64_t)gridDim.x * blockDim.x) {
        const int64_t row = idx / (groups * 4), b = idx % (groups * 4);
        uint32_t byte = 0;
        if (b < blocks) {
            const T* x = src + row * row_stride + b * 32 * k_stride;
            const int cnt = (int)min((int64_t)32, k - b * 32);
            uint32_t amax = 0;
            for (int i = 0; i < cnt; ++i) amax = max(amax, __float_as_uint(to_f32<T>(x[i * k_stride])) & 0x7fffffffu);
            byte = scale_byte(amax);
            const float inv = inv_scale(byte);
            uint8_t* out = codes + row * blocks * 16 + b * 16;
            for (int i = 0; i < 32; i += 2) {
                const float lo = i < cnt && byte != kNanScale ? to_f32<T>(x[i * k_stride]) * inv : 0.0f;
                const float hi = i + 1 < cnt && byte != kNanScale ? to_f32<T>(x[(i + 1) * k_stride]) * inv : 0.0f;
                out[i / 2] = (uint8_t)encode2(lo, hi);
            }
        }
        scales[scale_offset(row, b, groups)] = (uint8_t)byte;
    }
}

template <typename T>
__global__ void dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int64_t rows,
                                  int64_t k, int64_t blocks, int64_t groups, T* __restrict__ dst, int64_t ld) {
    const int64_t total = rows * k;
    for (int64_t idx = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; idx < total;
         idx += (int64_t)gridDim.x * blockDim.x) {
        const int64_t row = idx / k, j = idx % k;
        const uint32_t two = codes[row * blocks * 16 + (j >> 1)];
        const float v = decode((j & 1) ? two >> 4 : two & 15u) * scale_value(scales[scale_offset(row, j >> 5, groups)]);
        if constexpr (sizeof(T) == 2)
            dst[row * ld + j] = __float2bfloat16_rn(v);
        else
            dst[row * ld + j] = v;
    }
}

int check_extents(int64_t rows, int64_t k) {
    RT_CHECK(rows >= 0 && k >= 0, "mx4: negative extent %lld x %lld", (long long)rows, (long long)k);
    // box coordinates and the block count of a row are 32-bit
    RT_CHECK(rows <= INT_MAX - 256 && k <= INT_MAX - 256, "mx4: extent above 2^31 - 257: %lld x %lld", (long long)rows,
             (long long)k);
    return RT_OK;
}

int grid_for(const rt_ctx* ctx, int64_t items, int threads) {
    const int64_t want = (items + threads - 1) / threads;
    return (int)std::max<int64_t>(1, std::min<int64_t>(want, (int64_t)ctx->sm_count * 16));
}

}  // namespace
}  // namespace rt

using namespace rt;

extern "C" {

int64_t rt_mx4_code_bytes(int64_t rows, int64_t k) {
    if (check_extents(rows, k) != RT_OK) return -1;
    return rows * ((k + 31) / 32) * 16;
}

int64_t rt_mx4_scale_bytes(int64_t rows, int64_t k) {
    if (check_extents(rows, k) != RT_OK) return -1;
    return (rows + 127) / 128 * ((k + 127) / 128) * 512;
}

int rt_mx4_zeros(rt_ctx* ctx, int64_t rows, int64_t k, rt_mx4** out) {
    RT_CHECK(ctx && out, "rt_mx4_zeros: bad arguments");
    *out = nullptr;
    RT_TRY(check_extents(rows, k));
    const size_t cb = (size_t)rt_mx4_code_bytes(rows, k), sb = (size_t)rt_mx4_scale_bytes(rows, k);
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
    rt_mx4* q = new (std::nothrow) rt_mx4;
    if (!q) {
        cudaFree(p);
        return fail(RT_ERR_OOM, "rt_mx4_zeros: out of host memory");
    }
    q->ctx = ctx;
    q->codes = static_cast<uint8_t*>(p);
    q->scales = q->codes + scales_at;
    q->rows = rows;
    q->k = k;
    q->owned = true;
    *out = q;
    return RT_OK;
}

int rt_mx4_wrap(rt_ctx* ctx, void* codes, void* scales, int64_t rows, int64_t k, rt_mx4** out) {
    RT_CHECK(ctx && out, "rt_mx4_wrap: bad arguments");
    *out = nullptr;
    RT_TRY(check_extents(rows, k));
    RT_CHECK((codes && scales) || rows == 0 || k == 0, "rt_mx4_wrap: codes or scales is NULL");
    RT_CHECK(((reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(scales)) & 15) == 0,
             "rt_mx4_wrap: codes and scales must be 16-byte aligned");
    rt_mx4* q = new (std::nothrow) rt_mx4;
    if (!q) return fail(RT_ERR_OOM, "rt_mx4_wrap: out of host memory");
    q->ctx = ctx;
    q->codes = static_cast<uint8_t*>(codes);
    q->scales = static_cast<uint8_t*>(scales);
    q->rows = rows;
    q->k = k;
    *out = q;
    return RT_OK;
}

int rt_mx4_free(rt_mx4* q) {
    if (!q) return RT_OK;
    if (q->owned) {
        cudaSetDevice(q->ctx->device);
        cudaStreamSynchronize(q->ctx->stream);
        cudaFree(q->codes);
    }
    delete q;
    return RT_OK;
}

int rt_mx4_dims(const rt_mx4* q, int64_t* rows, int64_t* k) {
    RT_CHECK(q, "mx4 matrix is NULL");
    if (rows) *rows = q->rows;
    if (k) *k = q->k;
    return RT_OK;
}

void* rt_mx4_codes(const rt_mx4* q) { return q ? q->codes : nullptr; }
void* rt_mx4_scales(const rt_mx4* q) { return q ? q->scales : nullptr; }

int rt_mx4_quantize(rt_ctx* ctx, const rt_tensor* src, int axis, rt_mx4* dst) {
    RT_CHECK(ctx && src && dst, "rt_mx4_quantize: bad arguments");
    RT_CHECK(axis == 0 || axis == 1, "rt_mx4_quantize: axis must be 0 or 1 (got %d)", axis);
    RT_CHECK(src->dtype == RT_F32 || src->dtype == RT_BF16, "rt_mx4_quantize: src must be f32 or bf16");
    const int64_t rows = axis == 1 ? src->rows : src->cols, k = axis == 1 ? src->cols : src->rows;
    RT_CHECK(rows == dst->rows && k == dst->k, "rt_mx4_quantize: src is %lldx%lld along the blocks, dst %lldx%lld",
             (long long)rows, (long long)k, (long long)dst->rows, (long long)dst->k);
    if (rows == 0 || k == 0) return RT_OK;
    const int64_t rs = axis == 1 ? src->ld : 1, ks = axis == 1 ? 1 : src->ld;
    const int grid = grid_for(ctx, rows * dst->groups() * 4, 256);
    if (src->dtype == RT_BF16)
        quantize_kernel<<<grid, 256, 0, ctx->stream>>>(static_cast<const __nv_bfloat16*>(src->ptr), rs, ks, rows, k,
                                                       dst->blocks(), dst->groups(), dst->codes, dst->scales);
    else
        quantize_kernel<<<grid, 256, 0, ctx->stream>>>(static_cast<const float*>(src->ptr), rs, ks, rows, k,
                                                       dst->blocks(), dst->groups(), dst->codes, dst->scales);
    RT_CUDA(cudaGetLastError());
    count_launch(ctx);
    return RT_OK;
}

int rt_mx4_dequantize(rt_ctx* ctx, const rt_mx4* q, rt_tensor* dst) {
    RT_CHECK(ctx && q && dst, "rt_mx4_dequantize: bad arguments");
    RT_CHECK(dst->dtype == RT_F32 || dst->dtype == RT_BF16, "rt_mx4_dequantize: dst must be f32 or bf16");
    RT_CHECK(q->rows == dst->rows && q->k == dst->cols, "rt_mx4_dequantize: q is %lldx%lld, dst %lldx%lld",
             (long long)q->rows, (long long)q->k, (long long)dst->rows, (long long)dst->cols);
    if (q->rows == 0 || q->k == 0) return RT_OK;
    const int grid = grid_for(ctx, q->rows * q->k, 256);
    if (dst->dtype == RT_BF16)
        dequantize_kernel<<<grid, 256, 0, ctx->stream>>>(q->codes, q->scales, q->rows, q->k, q->blocks(), q->groups(),
                                                         static_cast<__nv_bfloat16*>(dst->ptr), dst->ld);
    else
        dequantize_kernel<<<grid, 256, 0, ctx->stream>>>(q->codes, q->scales, q->rows, q->k, q->blocks(), q->groups(),
                                                         static_cast<float*>(dst->ptr), dst->ld);
    RT_CUDA(cudaGetLastError());
    count_launch(ctx);
    return RT_OK;
}

int rt_mx4_matmul(rt_ctx* ctx, const rt_mx4* a, const rt_mx4* b, rt_tensor* c, const rt_tensor* bias, int relu) {
    RT_CHECK(ctx && a && b && c, "rt_mx4_matmul: bad arguments");
    RT_CHECK(c->dtype == RT_F32 || c->dtype == RT_BF16, "rt_mx4_matmul: C must be f32 or bf16");
    RT_CHECK(a->k == b->k, "rt_mx4_matmul: A is %lldx%lld, B %lldx%lld: the second extents differ", (long long)a->rows,
             (long long)a->k, (long long)b->rows, (long long)b->k);
    RT_CHECK(c->rows == a->rows && c->cols == b->rows, "rt_mx4_matmul: C is %lldx%lld, not %lldx%lld",
             (long long)c->rows, (long long)c->cols, (long long)a->rows, (long long)b->rows);
    if (bias) {
        RT_CHECK(bias->dtype == RT_F32, "rt_mx4_matmul: bias must be f32");
        RT_CHECK(bias->rows == 1 && bias->cols == b->rows, "rt_mx4_matmul: bias is %lldx%lld, not 1x%lld",
                 (long long)bias->rows, (long long)bias->cols, (long long)b->rows);
    }
    if (c->rows == 0 || c->cols == 0) return RT_OK;
    return launch_gemm_mx4(ctx, *a, *b, *c, bias ? static_cast<const float*>(bias->ptr) : nullptr, relu != 0,
                           ctx->stream);
}

}  // extern "C"
