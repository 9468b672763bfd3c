// Microscaled 4-bit matrices: handles, quantisation and dequantisation.
#include <algorithm>
#include <climits>
#include <new>

#include <cuda_fp16.h>

#include "mx4.cuh"

namespace rt {
namespace {

using namespace mx4;

// Every kernel here launches as a programmatic dependent of the one before it on
// the stream (launch_k), and waits for it before touching memory.

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

// Eight elements of a row from p (those at `left` and after read as 0), as f32.
// VEC: p is 16-byte aligned.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* p, int64_t left, float (&v)[8]) {
    if (VEC && left >= 8) {
        if constexpr (sizeof(T) == 2) {
            const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[2 * i] = __uint_as_float(w[i] << 16);
                v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            }
        } else {
            const float4 x = __ldg(reinterpret_cast<const float4*>(p)), y = __ldg(reinterpret_cast<const float4*>(p) + 1);
            v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
            v[4] = y.x, v[5] = y.y, v[6] = y.z, v[7] = y.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < left ? to_f32<T>(p[i]) : 0.0f;
    }
}

template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* p, int64_t left, const float (&v)[8]) {
    if (VEC && left >= 8) {
        if constexpr (sizeof(T) == 2) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t*>(&h);
            }
            *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
            *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
            *(reinterpret_cast<float4*>(p) + 1) = make_float4(v[4], v[5], v[6], v[7]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < left) {
                if constexpr (sizeof(T) == 2)
                    p[i] = __float2bfloat16_rn(v[i]);
                else
                    p[i] = v[i];
            }
    }
}

// Blocks along a row.  A warp takes 256 elements (two scale groups) of the four
// rows r, r + 32, r + 64, r + 96 of a 128-row tile: the scales of these rows lie
// side by side, 16 bytes for a group, and every lane has four independent reads
// of 16 (f32: 32) bytes under way.  A lane encodes 8 elements of each row to 4
// bytes; the four lanes of a block find its largest magnitude by shuffles.
// HBM-bound: 2 (f32: 4) bytes in and 17/32 out per element.
struct Tasks {
    int64_t total;   // warps' worth of work
    int64_t chunks;  // of 256 elements along k
    int rcount;      // rows r of a tile: 32, or fewer where the matrix has fewer
};

__device__ __forceinline__ void task_at(const Tasks& w, int64_t i, int64_t& chunk, int64_t& row) {
    chunk = i % w.chunks;
    const int64_t q = i / w.chunks;
    row = q / w.rcount * 128 + q % w.rcount;
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const T* __restrict__ src, int64_t ld, int64_t rows,
                                                            int64_t k, Tasks w, int64_t blocks, int64_t groups,
                                                            uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31;
    for (int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); i < w.total; i += (int64_t)gridDim.x * 8) {
        int64_t chunk, row;
        task_at(w, i, chunk, row);
        const int64_t j = chunk * 256 + lane * 8;
        float v[4][8];
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (row + 32 * q < rows)
                load8<T, VEC>(src + (row + 32 * q) * ld + j, k - j, v[q]);
            else
#pragma unroll
                for (int e = 0; e < 8; ++e) v[q][e] = 0.0f;
        uint32_t word[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            uint32_t amax = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) amax = max(amax, __float_as_uint(v[q][e]) & 0x7fffffffu);
            amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            const uint32_t byte = scale_byte(amax);
            const float inv = inv_scale(byte);
            uint32_t c = 0;
#pragma unroll
            for (int e = 0; e < 8; e += 2) c |= encode2(v[q][e] * inv, v[q][e + 1] * inv) << (4 * e);
            if (byte == kNanScale) c = 0;
            if (row + 32 * q < rows && j < blocks * 32)
                *reinterpret_cast<uint32_t*>(codes + (row + 32 * q) * blocks * 16 + (j >> 1)) = c;
            // the bytes of a group's four blocks into its first lane
            word[q] = byte | __shfl_down_sync(0xffffffffu, byte, 4) << 8;
            word[q] |= __shfl_down_sync(0xffffffffu, word[q], 8) << 16;
        }
        const int64_t group = chunk * 2 + (lane >> 4);
        if ((lane & 15) == 0 && group < groups)
            *reinterpret_cast<uint4*>(scales + ((row >> 7) * groups + group) * 512 + (row & 31) * 16) =
                make_uint4(word[0], word[1], word[2], word[3]);
    }
}

// Blocks down a column, laid out transposed.  A CTA takes one scale tile: 128
// columns of src by 128 of its rows.  A thread holds the 32 elements of a block of
// one column (bf16: of two neighbouring columns), a warp reads 128 bytes of a row
// of src at a time, 32 rows under way.  The tile's scales meet in shared memory
// and leave as 512 contiguous bytes.  HBM-bound by the reads.
template <typename T, bool PAIR>
__global__ void __launch_bounds__(256) quantize_columns_kernel(const T* __restrict__ src, int64_t ld, int64_t rows,
                                                               int64_t k, int64_t blocks, int64_t groups,
                                                               uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    __shared__ uint32_t tile[128];
    pdl_wait();
    pdl_launch_dependents();
    constexpr int W = PAIR ? 2 : 1;  // columns of a thread
    const int64_t group = blockIdx.x % groups, col0 = blockIdx.x / groups * 128;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint8_t* bytes = reinterpret_cast<uint8_t*>(tile);
    // PAIR: warps 0-1 take the 128 columns of block 0, 2-3 of block 1, ...; else
    // warps 0-3 take blocks 0 and 1, warps 4-7 blocks 2 and 3
    constexpr int WARPS = 4 / W;
    const int c = (warp % WARPS) * 32 * W + lane * W;
#pragma unroll
    for (int rep = 0; rep < 2 / W; ++rep) {
        const int b = PAIR ? warp / 2 : warp / 4 * 2 + rep;
        const int64_t block = group * 4 + b, k0 = block * 32, col = col0 + c;
        float v[W][32];
        const T* p = src + k0 * ld + col;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            if constexpr (PAIR) {
                uint32_t u = 0;
                if (k0 + i < k && col < rows) {
                    if (col + 1 < rows)
                        u = __ldg(reinterpret_cast<const uint32_t*>(p + i * ld));
                    else
                        u = *reinterpret_cast<const uint16_t*>(p + i * ld);
                }
                v[0][i] = __uint_as_float(u << 16);
                v[1][i] = __uint_as_float(u & 0xffff0000u);
            } else {
                v[0][i] = k0 + i < k && col < rows ? to_f32<T>(p[i * ld]) : 0.0f;
            }
        }
#pragma unroll
        for (int x = 0; x < W; ++x) {
            uint32_t amax = 0;
#pragma unroll
            for (int i = 0; i < 32; ++i) amax = max(amax, __float_as_uint(v[x][i]) & 0x7fffffffu);
            const uint32_t byte = scale_byte(amax);
            const float inv = inv_scale(byte);
            uint32_t out[4] = {0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < 32; i += 2) out[i / 8] |= encode2(v[x][i] * inv, v[x][i + 1] * inv) << (4 * (i % 8));
            if (byte == kNanScale) out[0] = out[1] = out[2] = out[3] = 0;
            if (block < blocks && col + x < rows)
                *reinterpret_cast<uint4*>(codes + (col + x) * blocks * 16 + block * 16) =
                    make_uint4(out[0], out[1], out[2], out[3]);
            const int r = c + x;  // row of the tile
            bytes[(r & 31) * 16 + (r >> 5) * 4 + b] = (uint8_t)byte;
        }
    }
    __syncthreads();
    if (threadIdx.x < 128)
        reinterpret_cast<uint32_t*>(scales + (col0 / 128 * groups + group) * 512)[threadIdx.x] = tile[threadIdx.x];
}

// 8 codes (element i in bits 4i) to f32.
__device__ __forceinline__ void decode8(uint32_t c, float scale, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t h;  // two halves
        asm("{\n\t.reg .b8 b;\n\tcvt.u8.u32 b, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, b;\n\t}" : "=r"(h) : "r"((c >> (8 * i)) & 255u));
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
        v[2 * i] = f.x * scale;
        v[2 * i + 1] = f.y * scale;
    }
}

// The same tasks as quantize_rows_kernel, the other way.  bf16 holds every value
// exactly: two significant bits, exponents 2^-128 to 2^130 (an overflow is the
// same infinity in f32).  HBM-bound: 17/32 bytes in, 2 (f32: 4) out per element.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) dequantize_kernel(const uint8_t* __restrict__ codes,
                                                         const uint8_t* __restrict__ scales, int64_t rows, int64_t k,
                                                         Tasks w, int64_t blocks, int64_t groups, T* __restrict__ dst,
                                                         int64_t ld) {
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31;
    for (int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); i < w.total; i += (int64_t)gridDim.x * 8) {
        int64_t chunk, row;
        task_at(w, i, chunk, row);
        const int64_t j = chunk * 256 + lane * 8;
        if (j >= k) continue;
        const uint4 s = __ldg(reinterpret_cast<const uint4*>(scales + ((row >> 7) * groups + (j >> 7)) * 512 + (row & 31) * 16));
        const uint32_t word[4] = {s.x, s.y, s.z, s.w};
        uint32_t c[4];
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (row + 32 * q < rows)
                c[q] = __ldg(reinterpret_cast<const uint32_t*>(codes + (row + 32 * q) * blocks * 16 + (j >> 1)));
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (row + 32 * q < rows) {
                float v[8];
                decode8(c[q], scale_value((word[q] >> (8 * ((j >> 5) & 3))) & 255u), v);
                store8<T, VEC>(dst + (row + 32 * q) * ld + j, k - j, v);
            }
    }
}

// CTAs for `items` of `per_cta` each: all of them, or as many as the kernels' loops
// share out evenly enough.
int grid_for(const rt_ctx* ctx, int64_t items, int per_cta) {
    const int64_t want = (items + per_cta - 1) / per_cta;
    return (int)std::max<int64_t>(1, std::min<int64_t>(want, (int64_t)ctx->sm_count * 64));
}

Tasks tasks_for(int64_t rows, int64_t k) {
    Tasks w;
    w.chunks = (k + 255) / 256;
    w.rcount = (int)std::min<int64_t>(rows, 32);
    w.total = w.chunks * w.rcount * ((rows + 127) / 128);
    return w;
}

bool aligned16(const rt_tensor* t) {
    return ((reinterpret_cast<uintptr_t>(t->ptr) | (uintptr_t)(t->ld * dtype_size(t->dtype))) & 15) == 0;
}

template <typename T>
int launch_quantize(rt_ctx* ctx, const rt_tensor* src, int axis, rt_mx4* q) {
    const T* p = static_cast<const T*>(src->ptr);
    if (axis == 1) {
        const Tasks w = tasks_for(q->rows, q->k);
        const int grid = grid_for(ctx, w.total, 8);
        auto* kernel = aligned16(src) ? quantize_rows_kernel<T, true> : quantize_rows_kernel<T, false>;
        RT_CUDA(launch_k(ctx->pdl, kernel, grid, 256, 0, ctx->stream, p, src->ld, q->rows, q->k, w, q->blocks(),
                         q->groups(), q->codes, q->scales));
    } else {
        const int64_t grid = q->groups() * ((q->rows + 127) / 128);
        RT_CHECK(grid <= INT_MAX, "rt_mx4_quantize: src is too large");
        auto* kernel = quantize_columns_kernel<T, false>;
        if constexpr (sizeof(T) == 2)
            if ((reinterpret_cast<uintptr_t>(p) & 3) == 0 && src->ld % 2 == 0) kernel = quantize_columns_kernel<T, true>;
        RT_CUDA(launch_k(ctx->pdl, kernel, (unsigned)grid, 256, 0, ctx->stream, p, src->ld, q->rows, q->k, q->blocks(),
                         q->groups(), q->codes, q->scales));
    }
    count_launch(ctx);
    return RT_OK;
}

template <typename T>
int launch_dequantize(rt_ctx* ctx, const rt_mx4* q, rt_tensor* dst) {
    const Tasks w = tasks_for(q->rows, q->k);
    const int grid = grid_for(ctx, w.total, 8);
    auto* kernel = aligned16(dst) ? dequantize_kernel<T, true> : dequantize_kernel<T, false>;
    RT_CUDA(launch_k(ctx->pdl, kernel, grid, 256, 0, ctx->stream, q->codes, q->scales, q->rows, q->k, w, q->blocks(),
                     q->groups(), static_cast<T*>(dst->ptr), dst->ld));
    count_launch(ctx);
    return RT_OK;
}

int check_extents(int64_t rows, int64_t k) {
    RT_CHECK(rows >= 0 && k >= 0, "mx4: negative extent %lld x %lld", (long long)rows, (long long)k);
    // box coordinates and the block count of a row are 32-bit
    RT_CHECK(rows <= INT_MAX - 256 && k <= INT_MAX - 256, "mx4: extent above 2^31 - 257: %lld x %lld", (long long)rows,
             (long long)k);
    return RT_OK;
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
    RT_CUDA(cudaSetDevice(ctx->device));
    return src->dtype == RT_BF16 ? launch_quantize<__nv_bfloat16>(ctx, src, axis, dst)
                                 : launch_quantize<float>(ctx, src, axis, dst);
}

int rt_mx4_dequantize(rt_ctx* ctx, const rt_mx4* q, rt_tensor* dst) {
    RT_CHECK(ctx && q && dst, "rt_mx4_dequantize: bad arguments");
    RT_CHECK(dst->dtype == RT_F32 || dst->dtype == RT_BF16, "rt_mx4_dequantize: dst must be f32 or bf16");
    RT_CHECK(q->rows == dst->rows && q->k == dst->cols, "rt_mx4_dequantize: q is %lldx%lld, dst %lldx%lld",
             (long long)q->rows, (long long)q->k, (long long)dst->rows, (long long)dst->cols);
    if (q->rows == 0 || q->k == 0) return RT_OK;
    RT_CUDA(cudaSetDevice(ctx->device));
    return dst->dtype == RT_BF16 ? launch_dequantize<__nv_bfloat16>(ctx, q, dst) : launch_dequantize<float>(ctx, q, dst);
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
