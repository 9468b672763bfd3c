// Dropout from a counter-based generator; the mask is computed where it is used and
// never stored.
//
//   y[i,j] = add[i,j] + keep[i,j] x[i,j] / (1 - p),   dx = keep dy / (1 - p)
//
// keep[i,j] is a function of (seed, site, step, row i, column j) alone, so the backward
// pass is the same call on the gradient, and a row's mask does not depend on the batch
// that it is in, on strides or on the grid.  The generator is Philox4x32 with ten rounds
// (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011): key
// the seed, counter (j / 8, row, step, site).  Its 128 bits serve eight elements, 16 bits
// each: p is taken to the nearest 2^-16, and 1 - p in the scale is that of the rounded p,
// so the expectation is exact.  32 bits an element would double the rounds, whose
// integer products then take longer than HBM.
#include <climits>

#include "row_piece.cuh"

namespace rt {
namespace {

struct DropoutParams {
    int64_t rows, cols;
    uint32_t key0, key1, step, site, first_row;
    const uint32_t* step_at;  // added to step; may be null
    uint32_t drop;            // kept where the 16 bits are at least this
    float scale;
    int chunks, along;        // warps' pieces of a row; log2 of the warps of a CTA that lie along a row
};

// The 128 bits of eight columns, two elements a word.
__device__ __forceinline__ uint4 philox(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, uint32_t k0, uint32_t k1) {
#pragma unroll
    for (int i = 0; i < 10; ++i) {
        const uint64_t p = (uint64_t)c0 * 0xD2511F53u, q = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(q >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)q;
        c2 = (uint32_t)(p >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)p;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return make_uint4(c0, c1, c2, c3);
}

__device__ __forceinline__ uint32_t pack(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// A warp takes a piece of a row, a lane 16 (f32: 8) neighbouring elements: whole groups of
// eight, so no two lanes compute the same numbers.  8192 x 8192 bf16 with a sum: 60 to 63 us,
// 6.4 TB/s and more; two rows a warp were 9 % slower, four 5 %, for fewer warps then fit an SM, and what hides a
// warp's ten rounds is the reads of others.
// Elements that are dropped are chosen away, not multiplied by zero: an infinity or a
// NaN there does not come through.  x and add are read before y is written, by the
// same warp, so y may be either.  V: bytes that the rows, which are whole pieces, are
// aligned to, 32 or 16; 0: any rows.
template <typename T, int V, bool ADD>
__global__ void __launch_bounds__(256) dropout_kernel(const T* x, int64_t ldx, const T* add, int64_t lda, T* y,
                                                      int64_t ldy, DropoutParams p) {
    using P = Piece<T>;
    __shared__ __align__(16) uint32_t boxes[V ? 1 : 8][256];
    pdl_wait();
    pdl_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t* box = boxes[V ? 0 : warp];
    const uint32_t step = p.step + (p.step_at ? *p.step_at : 0u);
    const int64_t row = ((int64_t)blockIdx.x << (3 - p.along)) + (warp >> p.along);
    if (row >= p.rows) return;
    x += row * ldx;
    if (ADD) add += row * lda;
    y += row * ldy;
    for (int chunk = (blockIdx.y << p.along) + (warp & ((1 << p.along) - 1)); chunk < p.chunks; chunk += gridDim.y << p.along) {
        const int64_t j0 = (int64_t)chunk * P::WARP, j = j0 + lane * P::E;
        P v, a;
        if constexpr (V == 0) {
            const auto r = P::fetch_any(x + j0, p.cols - j0, lane);
            if (ADD) {
                const auto s = P::fetch_any(add + j0, p.cols - j0, lane);
                a.deal_any(s, P::between(add + j0), box, lane);
            }
            v.deal_any(r, P::between(x + j0), box, lane);
        } else {
            if (j >= p.cols) break;
            v.template load_whole<V>(x + j);
            if (ADD) a.template load_whole<V>(add + j);
        }
#pragma unroll
        for (int g = 0; g < P::E / 8; ++g) {
            const uint4 r = philox((uint32_t)(j >> 3) + g, p.first_row + (uint32_t)row, step, p.site, p.key0, p.key1);
            const uint32_t bits[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int e = g * 8 + i * 2;
                float lo = (bits[i] & 0xffffu) >= p.drop ? __fmul_rn(v.value(e), p.scale) : 0.0f;
                float hi = (bits[i] >> 16) >= p.drop ? __fmul_rn(v.value(e + 1), p.scale) : 0.0f;
                if (ADD) {
                    lo = __fadd_rn(a.value(e), lo);
                    hi = __fadd_rn(a.value(e + 1), hi);
                }
                if constexpr (sizeof(T) == 2) {
                    v.w[e / 2] = pack(lo, hi);
                } else {
                    v.w[e] = __float_as_uint(lo);
                    v.w[e + 1] = __float_as_uint(hi);
                }
            }
        }
        if constexpr (V == 0)
            v.store_any(y + j0, p.cols - j0, box, lane);
        else
            v.template store<V>(y + j, P::E);
    }
}

template <typename T, int V>
int launch(rt_ctx* ctx, dim3 grid, const rt_tensor* x, const rt_tensor* add, rt_tensor* y, const DropoutParams& p) {
    const T *px = static_cast<const T*>(x->ptr), *pa = add ? static_cast<const T*>(add->ptr) : nullptr;
    auto* kernel = add ? dropout_kernel<T, V, true> : dropout_kernel<T, V, false>;
    RT_CUDA(launch_k(ctx->pdl, kernel, grid, 256, 0, ctx->stream, px, x->ld, pa, add ? add->ld : 0, static_cast<T*>(y->ptr),
                     y->ld, p));
    count_launch(ctx);
    return RT_OK;
}

template <typename T>
int launch_dropout(rt_ctx* ctx, const rt_tensor* x, const rt_tensor* add, rt_tensor* y, DropoutParams p) {
    p.chunks = (int)((p.cols + Piece<T>::WARP - 1) / Piece<T>::WARP);
    for (p.along = 0; p.along < 3 && p.chunks % (2 << p.along) == 0;) ++p.along;
    const int64_t groups = (p.rows + (8 >> p.along) - 1) >> (3 - p.along);
    RT_CHECK(groups <= INT_MAX, "rt_dropout: %lld rows are too many", (long long)p.rows);
    const dim3 grid((unsigned)groups, (unsigned)std::min(p.chunks >> p.along, 65535));
    int v = std::min(access_of(x), access_of(y));
    if (add) v = std::min(v, access_of(add));
    if (p.cols % Piece<T>::E) v = 0;
    if (v == 32) return launch<T, 32>(ctx, grid, x, add, y, p);
    if (v == 16) return launch<T, 16>(ctx, grid, x, add, y, p);
    return launch<T, 0>(ctx, grid, x, add, y, p);
}

}  // namespace
}  // namespace rt

using namespace rt;

extern "C" int rt_dropout(rt_ctx* ctx, const rt_tensor* x, const rt_tensor* add, rt_tensor* y, const rt_dropout_mask* mask) {
    RT_CHECK(ctx && x && y && mask, "rt_dropout: bad arguments");
    RT_CHECK(x->ctx == ctx && y->ctx == ctx && (!add || add->ctx == ctx) && (!mask->step_at || mask->step_at->ctx == ctx),
             "tensor belongs to another context");
    RT_CHECK(x->dtype == RT_F32 || x->dtype == RT_BF16, "rt_dropout: x must be f32 or bf16");
    RT_CHECK(y->dtype == x->dtype && (!add || add->dtype == x->dtype), "rt_dropout: x, add and y must have one type");
    RT_CHECK(y->rows == x->rows && y->cols == x->cols, "rt_dropout: x is %lldx%lld, y %lldx%lld", (long long)x->rows,
             (long long)x->cols, (long long)y->rows, (long long)y->cols);
    RT_CHECK(!add || (add->rows == x->rows && add->cols == x->cols), "rt_dropout: x is %lldx%lld, add %lldx%lld",
             (long long)x->rows, (long long)x->cols, (long long)(add ? add->rows : 0), (long long)(add ? add->cols : 0));
    RT_CHECK(mask->p >= 0.0 && mask->p <= 1.0, "rt_dropout: p must be in [0, 1] (got %g)", mask->p);
    RT_CHECK(mask->first_row >= 0 && mask->first_row <= (int64_t)1 << 32 && x->rows <= ((int64_t)1 << 32) - mask->first_row,
             "rt_dropout: %lld rows from row %lld on are not within 2^32", (long long)x->rows, (long long)mask->first_row);
    RT_CHECK(x->cols <= (int64_t)1 << 34, "rt_dropout: %lld columns are over 2^34", (long long)x->cols);
    const rt_tensor* s = mask->step_at;
    RT_CHECK(!s || (s->dtype == RT_U32 && s->rows * s->cols == 1), "rt_dropout: step_at must be one u32");
    if (x->rows == 0 || x->cols == 0) return RT_OK;
    DropoutParams p{};
    p.rows = x->rows;
    p.cols = x->cols;
    p.key0 = (uint32_t)mask->seed;
    p.key1 = (uint32_t)(mask->seed >> 32);
    p.step = mask->step;
    p.site = mask->site;
    p.first_row = (uint32_t)mask->first_row;
    p.step_at = s ? static_cast<const uint32_t*>(s->ptr) : nullptr;
    // half way between two multiples of 2^-16: to the even one
    p.drop = (uint32_t)__builtin_nearbyint(mask->p * 65536.0);
    p.scale = p.drop < 65536u ? (float)(65536.0 / (65536.0 - p.drop)) : 0.0f;
    RT_CUDA(cudaSetDevice(ctx->device));
    return x->dtype == RT_BF16 ? launch_dropout<__nv_bfloat16>(ctx, x, add, y, p)
                               : launch_dropout<float>(ctx, x, add, y, p);
}
