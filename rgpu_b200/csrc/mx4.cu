// Microscaled 4-bit matrices: handles, quantisation and dequantisation.
#include "mx4.cuh"
#include "row_piece.cuh"
#include "scaled.cuh"

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

// Codes of the piece's elements 8 i .. 8 i + 7.
template <typename T>
__device__ __forceinline__ uint32_t encode(const Piece<T>& x, int i, float inv) {
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = x.value(i * 8 + e);
    return encode8(v, inv);
}

// Blocks along a row.  A warp takes 512 (f32: 256) elements of the four rows r,
// r + 32, r + 64, r + 96 of a 128-row tile: the scales of these rows lie side by
// side, 16 bytes for a group, and every lane has four 32-byte reads under way.  Few
// lanes to a block keep the instructions per element low enough for HBM to be the
// bound: 2 (f32: 4) bytes in and 17/32 out per element.  8192 x 8192 bf16: 30 us,
// 5.7 TB/s.
template <typename T, int V>
__global__ void __launch_bounds__(256, V ? 4 : 3) quantize_rows_kernel(const T* src, int64_t ld, int64_t rows,
                                                               int64_t k, Rows w, int64_t blocks, int64_t groups,
                                                               uint8_t* codes,
                                                               uint8_t* scales) {
    using P = Piece<T>;
    constexpr int PER_BLOCK = 32 / P::E, PER_GROUP = 128 / P::E;  // lanes that share a block, a scale group
    __shared__ __align__(16) uint32_t boxes[V ? 1 : 8][256];
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31;
    const int64_t row_bytes = blocks * 16;
    const Place at(w);
    for (int64_t set = at.set; set < w.sets; set += at.set_step)
        for (int chunk = at.chunk; chunk < w.chunks; chunk += at.chunk_step) {
            const int64_t row = set_row(w, set), j0 = (int64_t)chunk * P::WARP, j = j0 + lane * P::E;
            const int live = (int)min((int64_t)4, (rows - row + 31) >> 5);  // rows of the set that there are
            const T* p = src + row * ld + j0;
            P x[4];
            if constexpr (V == 0) {
                typename P::Words r[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) r[q] = P::fetch_any(p + q * (32 * ld), q < live ? k - j0 : 0, lane);
#pragma unroll
                for (int q = 0; q < 4; ++q) x[q].deal_any(r[q], P::between(p + q * (32 * ld)), boxes[threadIdx.x >> 5], lane);
            } else {
#pragma unroll
                for (int q = 0; q < 4; ++q) x[q].template load<V>(p + q * (32 * ld) + lane * P::E, q < live ? k - j : 0);
            }
            uint32_t word[4];
            uint8_t* out = codes + row * row_bytes + (j >> 1);
            const bool inside = j < blocks * 32;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                uint32_t amax = x[q].amax();
#pragma unroll
                for (int o = 1; o < PER_BLOCK; o *= 2) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
                const uint32_t byte = scale_byte(amax);
                const float inv = inv_scale(byte);
                const bool nan = byte == kNanScale;
                if (q < live && inside) {
                    if constexpr (sizeof(T) == 2)
                        *reinterpret_cast<uint2*>(out + q * (32 * row_bytes)) =
                            make_uint2(nan ? 0u : encode(x[q], 0, inv), nan ? 0u : encode(x[q], 1, inv));
                    else
                        *reinterpret_cast<uint32_t*>(out + q * (32 * row_bytes)) = nan ? 0u : encode(x[q], 0, inv);
                }
                // the bytes of a group's four blocks into its first lane
                word[q] = byte | __shfl_down_sync(0xffffffffu, byte, PER_BLOCK) << 8;
                word[q] |= __shfl_down_sync(0xffffffffu, word[q], 2 * PER_BLOCK) << 16;
            }
            const int64_t group = j >> 7;
            if (lane % PER_GROUP == 0 && group < groups)
                *reinterpret_cast<uint4*>(scales + ((row >> 7) * groups + group) * 512 + (row & 31) * 16) =
                    make_uint4(word[0], word[1], word[2], word[3]);
        }
}

// Blocks down a column, laid out transposed.  A CTA takes one scale tile: 128
// columns of src by 128 of its rows.  A thread holds the 32 elements of a block of
// one column (bf16: of two neighbouring columns), a warp reads 128 bytes of a row
// of src at a time, 32 rows under way.  The tile's scales meet in shared memory
// and leave as 512 contiguous bytes.  4096 x 8192 f32 in 32 to 34 us and bf16 in 22,
// where their bytes take 23 and 13 at the rate of a copy: bound by the 32 scattered
// rows of a warp's reads, not by HBM.
template <typename T, bool PAIR>
__global__ void __launch_bounds__(256) quantize_columns_kernel(const T* src, int64_t ld, int64_t rows,
                                                               int64_t k, int64_t blocks, int64_t groups,
                                                               uint8_t* codes, uint8_t* scales) {
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
                        u = *reinterpret_cast<const uint32_t*>(p + i * ld);
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
            uint32_t out[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float e[8];
#pragma unroll
                for (int y = 0; y < 8; ++y) e[y] = v[x][i * 8 + y];
                out[i] = encode8(e, inv);
            }
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

// Codes to values.  The bits s e e m of a code, put where bf16 has its sign, its
// lowest exponent bits and its first mantissa bit, are the value times 2^-126
// (bf16's subnormals hold 0.5 too); two exact products with powers of two make up
// for that and the scale.
struct Unit {
    uint32_t a, b;  // f32 patterns, a b = 2^126 scale: 2^(byte - 1) up to 2^127, and the rest
    __device__ __forceinline__ explicit Unit(uint32_t byte) {
        a = byte == kNanScale ? 0x7fc00000u : min(byte + 126u, 254u) << 23;
        b = (byte > 128u ? byte - 1u : 127u) << 23;
    }
};

__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
    const __nv_bfloat162 r = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}

// The rows of quantize_rows_kernel, the other way.  bf16 holds every value exactly:
// two significant bits, exponents 2^-128 to 2^129 (past 2^128 the same infinity as
// in f32).  HBM-bound: 17/32 bytes in, 2 (f32: 4) out per element.  8192 x 8192
// bf16: 28 us, 6.0 TB/s.
template <typename T, int V>
__global__ void __launch_bounds__(256) dequantize_kernel(const uint8_t* codes,
                                                         const uint8_t* scales, int64_t rows, int64_t k,
                                                         Rows w, int64_t blocks, int64_t groups, T* dst,
                                                         int64_t ld) {
    using P = Piece<T>;
    __shared__ __align__(16) uint32_t boxes[V ? 1 : 8][256];
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31;
    const int64_t row_bytes = blocks * 16;
    const Place at(w);
    for (int64_t set = at.set; set < w.sets; set += at.set_step)
        for (int chunk = at.chunk; chunk < w.chunks; chunk += at.chunk_step) {
            const int64_t row = set_row(w, set), j0 = (int64_t)chunk * P::WARP, j = j0 + lane * P::E;
            if (V ? j >= k : j0 >= k) continue;
            const bool inside = j < blocks * 32;
            const int live = (int)min((int64_t)4, (rows - row + 31) >> 5);
            const uint4 s = !inside ? make_uint4(0, 0, 0, 0) : *reinterpret_cast<const uint4*>(scales + ((row >> 7) * groups + (j >> 7)) * 512 + (row & 31) * 16);
            const uint32_t word[4] = {s.x, s.y, s.z, s.w};
            const uint8_t* in = codes + row * row_bytes + (j >> 1);
            uint32_t c[4][P::E / 8];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                c[q][0] = c[q][P::E / 8 - 1] = 0;
                if (q < live && inside) {
                    if constexpr (sizeof(T) == 2) {
                        const uint2 two = *reinterpret_cast<const uint2*>(in + q * (32 * row_bytes));
                        c[q][0] = two.x;
                        c[q][P::E / 8 - 1] = two.y;
                    } else {
                        c[q][0] = *reinterpret_cast<const uint32_t*>(in + q * (32 * row_bytes));
                    }
                }
            }
            const int shift = (int)(j >> 5 & 3) * 8;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                if (q >= live) break;
                const Unit u((word[q] >> shift) & 255u);
                P x;
#pragma unroll
                for (int i = 0; i < P::E / 2; ++i) {
                    // two codes to two bf16 patterns
                    const uint32_t two = c[q][i / 4] >> (8 * (i & 3)) & 255u, y = two | two << 12;
                    const uint32_t h = (y & 0x00070007u) << 6 | (y & 0x00080008u) << 12;
                    if constexpr (sizeof(T) == 2) {
                        x.w[i] = mul_bf16x2(mul_bf16x2(h, u.a | u.a >> 16), u.b | u.b >> 16);
                    } else {
                        x.w[2 * i] = __float_as_uint(__uint_as_float(h << 16) * __uint_as_float(u.a) * __uint_as_float(u.b));
                        x.w[2 * i + 1] = __float_as_uint(__uint_as_float(h & 0xffff0000u) * __uint_as_float(u.a) * __uint_as_float(u.b));
                    }
                }
                if constexpr (V == 0)
                    x.store_any(dst + (row + 32 * q) * ld + j0, k - j0, boxes[threadIdx.x >> 5], lane);
                else
                    x.template store<V>(dst + (row + 32 * q) * ld + j, k - j);
            }
        }
}

template <typename T>
int launch_quantize(rt_ctx* ctx, const rt_tensor* src, int axis, rt_mx4* q) {
    const T* p = static_cast<const T*>(src->ptr);
    if (axis == 1) {
        dim3 grid;
        const Rows w = rows_for(ctx, q->rows, q->k, Piece<T>::WARP, &grid);
        const int v = access_of(src);
        auto* kernel = v == 32 ? quantize_rows_kernel<T, 32> : v == 16 ? quantize_rows_kernel<T, 16> : quantize_rows_kernel<T, 0>;
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
    dim3 grid;
    const Rows w = rows_for(ctx, q->rows, q->k, Piece<T>::WARP, &grid);
    const int v = access_of(dst);
    auto* kernel = v == 32 ? dequantize_kernel<T, 32> : v == 16 ? dequantize_kernel<T, 16> : dequantize_kernel<T, 0>;
    RT_CUDA(launch_k(ctx->pdl, kernel, grid, 256, 0, ctx->stream, q->codes, q->scales, q->rows, q->k, w, q->blocks(),
                     q->groups(), static_cast<T*>(dst->ptr), dst->ld));
    count_launch(ctx);
    return RT_OK;
}

int check_extents(int64_t rows, int64_t k) { return check_scaled_extents("mx4", rows, k); }

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
    return scaled_zeros(ctx, rows, k, (size_t)rt_mx4_code_bytes(rows, k), (size_t)rt_mx4_scale_bytes(rows, k),
                        mx4_encode_maps, out);
}

int rt_mx4_wrap(rt_ctx* ctx, void* codes, void* scales, int64_t rows, int64_t k, rt_mx4** out) {
    RT_CHECK(ctx && out, "rt_mx4_wrap: bad arguments");
    *out = nullptr;
    RT_TRY(check_extents(rows, k));
    return scaled_wrap("rt_mx4_wrap", ctx, codes, scales, rows, k, mx4_encode_maps, out);
}

int rt_mx4_free(rt_mx4* q) { return scaled_free(q); }

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
    RT_CHECK(src->ctx == ctx && dst->ctx == ctx, "tensor belongs to another context");
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
    RT_CHECK(q->ctx == ctx && dst->ctx == ctx, "tensor belongs to another context");
    RT_CHECK(dst->dtype == RT_F32 || dst->dtype == RT_BF16, "rt_mx4_dequantize: dst must be f32 or bf16");
    RT_CHECK(q->rows == dst->rows && q->k == dst->cols, "rt_mx4_dequantize: q is %lldx%lld, dst %lldx%lld",
             (long long)q->rows, (long long)q->k, (long long)dst->rows, (long long)dst->cols);
    if (q->rows == 0 || q->k == 0) return RT_OK;
    RT_CUDA(cudaSetDevice(ctx->device));
    return dst->dtype == RT_BF16 ? launch_dequantize<__nv_bfloat16>(ctx, q, dst) : launch_dequantize<float>(ctx, q, dst);
}

int rt_mx4_matmul(rt_ctx* ctx, const rt_mx4* a, const rt_mx4* b, rt_tensor* c, const rt_tensor* bias, int relu) {
    RT_TRY(check_scaled_matmul("rt_mx4_matmul", ctx, a, b, c, bias));
    if (c->rows == 0 || c->cols == 0) return RT_OK;
    return launch_gemm_mx4(ctx, *a, *b, *c, bias ? static_cast<const float*>(bias->ptr) : nullptr, relu != 0,
                           ctx->stream);
}

}  // extern "C"
