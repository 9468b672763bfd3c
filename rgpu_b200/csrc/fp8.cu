// Matrices in 8-bit floating point (E4M3) with a power-of-two scale for each block of
// 128: handles, quantisation and dequantisation.
//
// A block's scale is the least power of two 2^e, e >= -127, with amax <= 448 * 2^e (448 is
// the largest element), so nothing saturates; x / 2^e is exact but for underflow far
// below the smallest element, then rounded to nearest even.  A power of two, not amax /
// 448, because the tensor cores multiply it in while they sum: no accumulator has to
// leave TMEM every 128 of k.  It leaves up to a factor of two of the range unused.
#include "row_piece.cuh"
#include "scaled.cuh"

namespace rt {
namespace {

constexpr uint32_t kNanScale = 255;

// Every kernel here launches as a programmatic dependent of the one before it on
// the stream (launch_k), and waits for it before touching memory.

// Scale byte of a block from the bit pattern of its largest magnitude: 448 is 1.75 *
// 2^8, so the exponent field less 8, one more where the mantissa is above 0.75 (adding
// 0x1FFFFF then carries into the field), at least 0 (2^-127).  An infinity or a NaN takes
// the NaN scale.
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax_bits) {
    if (amax_bits >= 0x7f800000u) return kNanScale;
    const int field = (int)((amax_bits + 0x1FFFFFu) >> 23) - 8;
    return field > 0 ? (uint32_t)field : 0u;
}
// 2^(127 - byte): scale_byte gives at most 247, so a normal number (the NaN scale's is not used).
__device__ __forceinline__ float inv_scale(uint32_t byte) { return __uint_as_float((254u - min(byte, 253u)) << 23); }
// 2^(byte - 127), subnormal for byte 0; NaN for 255.
__device__ __forceinline__ float scale_of(uint32_t byte) {
    return __uint_as_float(byte == kNanScale ? 0x7fc00000u : byte ? byte << 23 : 0x00400000u);
}

// Four elements, each times inv, to E4M3 (element i in bits 8 i).
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d, float inv) {
    uint32_t r;
    asm("{\n\t.reg .b16 x, y;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 x, %2, %1;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 y, %4, %3;\n\t"
        "mov.b32 %0, {x, y};\n\t}"
        : "=r"(r)
        : "f"(a * inv), "f"(b * inv), "f"(c * inv), "f"(d * inv));
    return r;
}
// Two E4M3 codes (the low 16 bits) to floats; every one is a half too.
__device__ __forceinline__ float2 decode2(uint32_t codes) {
    uint32_t h;
    asm("{\n\t.reg .b16 x;\n\tcvt.u16.u32 x, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, x;\n\t}" : "=r"(h) : "r"(codes));
    float2 v;
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.f32.f16 %0, a;\n\tcvt.f32.f16 %1, b;\n\t}"
        : "=f"(v.x), "=f"(v.y)
        : "r"(h));
    return v;
}

// Blocks along a row; the warps' order is row_piece.cuh's.  A warp's piece of a row is
// four blocks (f32: two), eight (sixteen) lanes to a block.  HBM-bound: 2 (f32: 4) bytes in,
// 129/128 out per element; 8192 x 8192 bf16 30 us, 6.7 TB/s.
template <typename T, int V>
__global__ void __launch_bounds__(256, V ? 4 : 3) quantize_rows_kernel(const T* src, int64_t ld,
                                                                       int64_t rows, int64_t k, Rows w,
                                                                       int64_t row_bytes, int64_t groups,
                                                                       uint8_t* codes,
                                                                       uint8_t* scales) {
    using P = Piece<T>;
    constexpr int PER_BLOCK = 128 / P::E;
    __shared__ __align__(16) uint32_t boxes[V ? 1 : 8][256];
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31;
    const Place at(w);
    for (int64_t set = at.set; set < w.sets; set += at.set_step)
        for (int chunk = at.chunk; chunk < w.chunks; chunk += at.chunk_step) {
            const int64_t row = set_row(w, set), j0 = (int64_t)chunk * P::WARP, j = j0 + lane * P::E;
            const int live = (int)min((int64_t)4, (rows - row + 31) >> 5);  // rows of the set that there are
            if (live <= 0) continue;
            const T* p = src + row * ld + j0;
            P x[4];
            if constexpr (V == 0) {
                typename P::Words r[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) r[q] = P::fetch_any(p + q * (32 * ld), q < live ? k - j0 : 0, lane);
#pragma unroll
                for (int q = 0; q < 4; ++q) x[q].deal_any(r[q], P::between(p + q * (32 * ld)), boxes[threadIdx.x >> 5], lane);
            } else {
                // V: rows are whole pieces; in place of a row or a piece that is not there another is read
                const T* at = src + row * ld + (j < k ? j : 0);
#pragma unroll
                for (int q = 0; q < 4; ++q) x[q].template load_whole<V>(at + min(q, live - 1) * (32 * ld));
                if (j >= k)
#pragma unroll
                    for (int q = 0; q < 4; ++q)
#pragma unroll
                        for (int i = 0; i < 8; ++i) x[q].w[i] = 0;
            }
            uint32_t word[4];
            uint8_t* out = codes + row * row_bytes + j;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                uint32_t amax = x[q].amax();
#pragma unroll
                for (int o = 1; o < PER_BLOCK; o *= 2) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
                const uint32_t byte = scale_byte(amax);
                const float inv = inv_scale(byte);
                const bool nan = byte == kNanScale;
                uint32_t c[P::E / 4];
#pragma unroll
                for (int i = 0; i < P::E / 4; ++i)
                    c[i] = nan ? 0u : encode4(x[q].value(4 * i), x[q].value(4 * i + 1), x[q].value(4 * i + 2), x[q].value(4 * i + 3), inv);
                if (q < live && j < row_bytes) {
                    if constexpr (P::E == 16)
                        *reinterpret_cast<uint4*>(out + q * (32 * row_bytes)) = make_uint4(c[0], c[1], c[2], c[3]);
                    else
                        *reinterpret_cast<uint2*>(out + q * (32 * row_bytes)) = make_uint2(c[0], c[1]);
                }
                // the bytes of the piece's blocks into its first lane
                word[q] = byte | __shfl_down_sync(0xffffffffu, byte, PER_BLOCK % 32) << 8;
                if constexpr (P::E == 16) word[q] |= __shfl_down_sync(0xffffffffu, word[q], 16) << 16;
            }
            if (lane == 0) {
                uint8_t* to = scales + ((row >> 7) * groups + (j0 >> 9)) * 512 + (row & 31) * 16;
                if constexpr (P::E == 16)
                    *reinterpret_cast<uint4*>(to) = make_uint4(word[0], word[1], word[2], word[3]);
                else
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        *reinterpret_cast<uint16_t*>(to + q * 4 + (j0 >> 7 & 2)) = (uint16_t)word[q];
            }
        }
}

// Blocks down a column, laid out transposed.  A CTA takes 128 columns of src by one block
// of 128 of its rows.  A thread holds 32 rows of one column (bf16: of two neighbouring
// ones), all its reads under way at once, a warp 128 bytes of a row each; the maxima of a
// column's four threads meet in shared memory.  A thread's 32 codes of a column are one
// sector of the output (WIDE: and one store, where the output's rows are so aligned).
// 4096 x 8192 f32: 31 us, 5.4 TB/s; with 64 rows a thread and a condition on each load 39.
template <typename T, bool PAIR, bool WIDE>
__global__ void __launch_bounds__(PAIR ? 256 : 512) quantize_columns_kernel(
    const T* src, int64_t ld, int64_t rows, int64_t k, int64_t blocks, int64_t row_bytes, int64_t groups,
    uint8_t* codes, uint8_t* scales) {
    constexpr int W = PAIR ? 2 : 1, N = 32, SHARES = 128 / N;  // columns, rows of a thread; threads to a column
    __shared__ uint32_t maxima[SHARES][128];
    pdl_wait();
    pdl_launch_dependents();
    const int64_t block = blockIdx.x % blocks, col0 = blockIdx.x / blocks * 128;
    const int share = threadIdx.x / (128 / W), c = threadIdx.x % (128 / W) * W;
    const int64_t k0 = block * 128 + share * N, col = col0 + c;
    float v[W][N];
    const T* p = src + k0 * ld + col;
    const int live = (int)max((int64_t)0, min((int64_t)N, k - k0));
    if (live == N && col + W <= rows) {  // without conditions on each: all loads are issued, then waited for
        uint32_t u[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if constexpr (PAIR || sizeof(T) == 4) u[i] = *reinterpret_cast<const uint32_t*>(p + i * ld);
            else u[i] = *reinterpret_cast<const uint16_t*>(p + i * ld);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            v[0][i] = __uint_as_float(sizeof(T) == 4 ? u[i] : u[i] << 16);
            if constexpr (PAIR) v[1][i] = __uint_as_float(u[i] & 0xffff0000u);
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int x = 0; x < W; ++x) {
                v[x][i] = 0.0f;
                if (i < live && col + x < rows) {
                    if constexpr (sizeof(T) == 2) v[x][i] = __bfloat162float(p[i * ld + x]);
                    else v[x][i] = p[i * ld + x];
                }
            }
    }
#pragma unroll
    for (int x = 0; x < W; ++x) {
        uint32_t amax = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) amax = max(amax, __float_as_uint(v[x][i]) & 0x7fffffffu);
        maxima[share][c + x] = amax;
    }
    __syncthreads();
#pragma unroll
    for (int x = 0; x < W; ++x) {
        if (col + x >= rows) break;
        uint32_t amax = 0;
#pragma unroll
        for (int s = 0; s < SHARES; ++s) amax = max(amax, maxima[s][c + x]);
        const uint32_t byte = scale_byte(amax);
        const float inv = inv_scale(byte);
        uint32_t e[N / 4];
#pragma unroll
        for (int y = 0; y < N / 4; ++y) {
            const float* u = &v[x][4 * y];
            e[y] = byte == kNanScale ? 0u : encode4(u[0], u[1], u[2], u[3], inv);
        }
        uint8_t* out = codes + (col + x) * row_bytes + k0;
        if constexpr (WIDE) {
            if (k0 < row_bytes)
                asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(out), "r"(e[0]), "r"(e[1]),
                             "r"(e[2]), "r"(e[3]), "r"(e[4]), "r"(e[5]), "r"(e[6]), "r"(e[7])
                             : "memory");
        } else {
#pragma unroll
            for (int i = 0; i < N; i += 16)
                if (k0 + i < row_bytes)
                    *reinterpret_cast<uint4*>(out + i) = make_uint4(e[i / 4], e[i / 4 + 1], e[i / 4 + 2], e[i / 4 + 3]);
        }
        if (share == 0) {
            const int r = c + x;  // row of the scale tile
            scales[(col0 / 128 * groups + (block >> 2)) * 512 + (r & 31) * 16 + (r >> 5) * 4 + (block & 3)] = (uint8_t)byte;
        }
    }
}

// The rows of quantize_rows_kernel, the other way.  f32 holds every value exactly; bf16 all
// from 2^-130 on, those below it are rounded to multiples of 2^-133.  8192 x 8192 bf16: 29 us, 6.9 TB/s.
template <typename T, int V>
__global__ void __launch_bounds__(256) dequantize_kernel(const uint8_t* codes,
                                                         const uint8_t* scales, int64_t rows, int64_t k,
                                                         Rows w, int64_t row_bytes, int64_t groups, T* dst,
                                                         int64_t ld) {
    using P = Piece<T>;
    __shared__ __align__(16) uint32_t boxes[V ? 1 : 8][256];
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31;
    const Place at(w);
    for (int64_t set = at.set; set < w.sets; set += at.set_step)
        for (int chunk = at.chunk; chunk < w.chunks; chunk += at.chunk_step) {
            const int64_t row = set_row(w, set), j0 = (int64_t)chunk * P::WARP, j = j0 + lane * P::E;
            if (V ? j >= k : j0 >= k) continue;
            const int live = (int)min((int64_t)4, (rows - row + 31) >> 5);
            if (live <= 0) continue;
            const uint4 s = *reinterpret_cast<const uint4*>(scales + ((row >> 7) * groups + (j0 >> 9)) * 512 + (row & 31) * 16);
            const uint32_t word[4] = {s.x, s.y, s.z, s.w};
            // without a branch (Piece::load_whole): another piece or row in place of one that is not there
            const uint8_t* in = codes + row * row_bytes + (j < k ? j : j0);
            uint32_t c[4][P::E / 4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const uint8_t* at = in + min(q, live - 1) * (32 * row_bytes);
                if constexpr (P::E == 16) {
                    const uint4 four = *reinterpret_cast<const uint4*>(at);
                    c[q][0] = four.x, c[q][1] = four.y, c[q][2] = four.z, c[q][3] = four.w;
                } else {
                    const uint2 two = *reinterpret_cast<const uint2*>(at);
                    c[q][0] = two.x, c[q][1] = two.y;
                }
            }
            const int shift = (int)(j >> 7 & 3) * 8;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                if (q >= live) break;
                const float unit = scale_of((word[q] >> shift) & 255u);
                P x;
#pragma unroll
                for (int i = 0; i < P::E / 2; ++i) {
                    const float2 v = decode2(c[q][i / 2] >> (16 * (i & 1)));
                    if constexpr (sizeof(T) == 2) {
                        const __nv_bfloat162 h = __floats2bfloat162_rn(v.x * unit, v.y * unit);
                        x.w[i] = *reinterpret_cast<const uint32_t*>(&h);
                    } else {
                        x.w[2 * i] = __float_as_uint(v.x * unit);
                        x.w[2 * i + 1] = __float_as_uint(v.y * unit);
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
int launch_quantize(rt_ctx* ctx, const rt_tensor* src, int axis, rt_fp8* q) {
    const T* p = static_cast<const T*>(src->ptr);
    if (axis == 1) {
        dim3 grid;
        const Rows w = rows_for(ctx, q->rows, q->k, Piece<T>::WARP, &grid);
        const int v = q->k % Piece<T>::E ? 0 : access_of(src);
        auto* kernel = v == 32 ? quantize_rows_kernel<T, 32> : v == 16 ? quantize_rows_kernel<T, 16> : quantize_rows_kernel<T, 0>;
        RT_CUDA(launch_k(ctx->pdl, kernel, grid, 256, 0, ctx->stream, p, src->ld, q->rows, q->k, w, q->row_bytes(),
                         q->groups(), q->codes, q->scales));
    } else {
        const int64_t grid = q->blocks() * ((q->rows + 127) / 128);
        RT_CHECK(grid <= INT_MAX, "rt_fp8_quantize: src is too large");
        const bool wide = ((reinterpret_cast<uintptr_t>(q->codes) | (uintptr_t)q->row_bytes()) & 31) == 0;
        auto* kernel = wide ? quantize_columns_kernel<T, false, true> : quantize_columns_kernel<T, false, false>;
        int threads = 512;
        if constexpr (sizeof(T) == 2)
            if ((reinterpret_cast<uintptr_t>(p) & 3) == 0 && src->ld % 2 == 0) {
                kernel = wide ? quantize_columns_kernel<T, true, true> : quantize_columns_kernel<T, true, false>;
                threads = 256;
            }
        RT_CUDA(launch_k(ctx->pdl, kernel, (unsigned)grid, threads, 0, ctx->stream, p, src->ld, q->rows, q->k, q->blocks(),
                         q->row_bytes(), q->groups(), q->codes, q->scales));
    }
    count_launch(ctx);
    return RT_OK;
}

template <typename T>
int launch_dequantize(rt_ctx* ctx, const rt_fp8* q, rt_tensor* dst) {
    dim3 grid;
    const Rows w = rows_for(ctx, q->rows, q->k, Piece<T>::WARP, &grid);
    const int v = access_of(dst);
    auto* kernel = v == 32 ? dequantize_kernel<T, 32> : v == 16 ? dequantize_kernel<T, 16> : dequantize_kernel<T, 0>;
    RT_CUDA(launch_k(ctx->pdl, kernel, grid, 256, 0, ctx->stream, q->codes, q->scales, q->rows, q->k, w, q->row_bytes(),
                     q->groups(), static_cast<T*>(dst->ptr), dst->ld));
    count_launch(ctx);
    return RT_OK;
}

int check_extents(int64_t rows, int64_t k) { return check_scaled_extents("fp8", rows, k); }

}  // namespace
}  // namespace rt

using namespace rt;

extern "C" {

int64_t rt_fp8_code_bytes(int64_t rows, int64_t k) {
    if (check_extents(rows, k) != RT_OK) return -1;
    return rows * ((k + 15) / 16) * 16;
}

int64_t rt_fp8_scale_bytes(int64_t rows, int64_t k) {
    if (check_extents(rows, k) != RT_OK) return -1;
    return (rows + 127) / 128 * ((k + 511) / 512) * 512;
}

int rt_fp8_zeros(rt_ctx* ctx, int64_t rows, int64_t k, rt_fp8** out) {
    RT_CHECK(ctx && out, "rt_fp8_zeros: bad arguments");
    *out = nullptr;
    RT_TRY(check_extents(rows, k));
    return scaled_zeros(ctx, rows, k, (size_t)rt_fp8_code_bytes(rows, k), (size_t)rt_fp8_scale_bytes(rows, k),
                        fp8_encode_maps, out);
}

int rt_fp8_wrap(rt_ctx* ctx, void* codes, void* scales, int64_t rows, int64_t k, rt_fp8** out) {
    RT_CHECK(ctx && out, "rt_fp8_wrap: bad arguments");
    *out = nullptr;
    RT_TRY(check_extents(rows, k));
    return scaled_wrap("rt_fp8_wrap", ctx, codes, scales, rows, k, fp8_encode_maps, out);
}

int rt_fp8_free(rt_fp8* q) { return scaled_free(q); }

int rt_fp8_dims(const rt_fp8* q, int64_t* rows, int64_t* k) {
    RT_CHECK(q, "fp8 matrix is NULL");
    if (rows) *rows = q->rows;
    if (k) *k = q->k;
    return RT_OK;
}

void* rt_fp8_codes(const rt_fp8* q) { return q ? q->codes : nullptr; }
void* rt_fp8_scales(const rt_fp8* q) { return q ? q->scales : nullptr; }

int rt_fp8_quantize(rt_ctx* ctx, const rt_tensor* src, int axis, rt_fp8* dst) {
    RT_CHECK(ctx && src && dst, "rt_fp8_quantize: bad arguments");
    RT_CHECK(src->ctx == ctx && dst->ctx == ctx, "tensor belongs to another context");
    RT_CHECK(axis == 0 || axis == 1, "rt_fp8_quantize: axis must be 0 or 1 (got %d)", axis);
    RT_CHECK(src->dtype == RT_F32 || src->dtype == RT_BF16, "rt_fp8_quantize: src must be f32 or bf16");
    const int64_t rows = axis == 1 ? src->rows : src->cols, k = axis == 1 ? src->cols : src->rows;
    RT_CHECK(rows == dst->rows && k == dst->k, "rt_fp8_quantize: src is %lldx%lld along the blocks, dst %lldx%lld",
             (long long)rows, (long long)k, (long long)dst->rows, (long long)dst->k);
    if (rows == 0 || k == 0) return RT_OK;
    RT_CUDA(cudaSetDevice(ctx->device));
    return src->dtype == RT_BF16 ? launch_quantize<__nv_bfloat16>(ctx, src, axis, dst)
                                 : launch_quantize<float>(ctx, src, axis, dst);
}

int rt_fp8_dequantize(rt_ctx* ctx, const rt_fp8* q, rt_tensor* dst) {
    RT_CHECK(ctx && q && dst, "rt_fp8_dequantize: bad arguments");
    RT_CHECK(q->ctx == ctx && dst->ctx == ctx, "tensor belongs to another context");
    RT_CHECK(dst->dtype == RT_F32 || dst->dtype == RT_BF16, "rt_fp8_dequantize: dst must be f32 or bf16");
    RT_CHECK(q->rows == dst->rows && q->k == dst->cols, "rt_fp8_dequantize: q is %lldx%lld, dst %lldx%lld",
             (long long)q->rows, (long long)q->k, (long long)dst->rows, (long long)dst->cols);
    if (q->rows == 0 || q->k == 0) return RT_OK;
    RT_CUDA(cudaSetDevice(ctx->device));
    return dst->dtype == RT_BF16 ? launch_dequantize<__nv_bfloat16>(ctx, q, dst) : launch_dequantize<float>(ctx, q, dst);
}

int rt_fp8_matmul(rt_ctx* ctx, const rt_fp8* a, const rt_fp8* b, rt_tensor* c, const rt_tensor* bias, int relu) {
    RT_TRY(check_scaled_matmul("rt_fp8_matmul", ctx, a, b, c, bias));
    if (c->rows == 0 || c->cols == 0) return RT_OK;
    return launch_gemm_fp8(ctx, *a, *b, *c, bias ? static_cast<const float*>(bias->ptr) : nullptr, relu != 0,
                           ctx->stream);
}

}  // extern "C"
