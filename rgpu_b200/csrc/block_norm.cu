// The row-wise work between two blocks of a residual stream: the norm after a
// block, its gate and residual scale, the residual sum and the norm before the
// next block (rt_block_forward), and their gradients (rt_block_backward).
//
//   u = N_post(y),  z = r + s (g . u),  h = N_pre(z)
//
// Backward, with x^ = (x - mu) rho, rho = 1 / sqrt(mean((x - mu)^2) + eps):
//   N^T(d) = rho (a - [layer] mean(a) - x^ mean(a x^)),   a = d gamma
//   dr = dz + N_pre^T(dh),  du = s g dr,  dy = N_post^T(du)
//   dgamma_pre = sum_rows dh z^,  dbeta_pre = sum_rows dh
// and, with w = dr (times g where the gate differs from row to row), the sums over
// rows A = sum w y^ and B = sum w give every other vector:
//   dgamma_post = s g A,  dbeta_post = s g B,  dgate = s (gamma_post A + beta_post B)
// (g = 1 where w holds it; the [1,1] gate's gradient sums dgate over columns).
#include <algorithm>
#include <initializer_list>

#include "landing.cuh"
#include "mx4.cuh"
#include "tc_common.cuh"

namespace rt {
namespace {

// Every kernel here launches as a programmatic dependent of the one before it on
// the stream (launch_k), and waits for it before touching global memory.

enum GateMode : int { GATE_NONE = 0, GATE_ONE = 1, GATE_ROW = 2, GATE_COLUMN = 3, GATE_FULL = 4 };

// Stride of a vector of partial sums: whole eights.
__host__ __device__ constexpr int64_t columns(int64_t n) { return (n + 7) & ~int64_t(7); }

struct NormP {
    int kind;
    float eps;
    const float* gamma;
    const float* beta;
};

struct BlockP {
    const void *r, *y;
    int64_t ldr, ldy;
    NormP post, pre;
    int gate_mode;
    const void* gate;  // f32, or y's type under GATE_FULL
    int64_t ldg;       // row stride of a column or full gate
    float scale;
    void *z, *h;
    int64_t ldz, ldh;
    uint8_t *codes, *scales;
    int64_t m, n;
};

struct GradP {
    const void *dz, *dh;
    int64_t lddz, lddh;
    void *dr, *dy;
    int64_t lddr, lddy;
    void* dgate;       // column and full gates (y's type under GATE_FULL)
    int64_t lddg;
    float* partials;   // [parts][4][columns(n)]: A, B, sum dh z^, sum dh of each CTA's rows
    int sums;          // bit i: sum i is wanted
};

template <typename T>
__device__ __forceinline__ float ld(const void* p, int64_t i) {
    if constexpr (sizeof(T) == 2)
        return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
    else
        return static_cast<const float*>(p)[i];
}
template <typename T>
__device__ __forceinline__ void st(void* p, int64_t i, float v) {
    if constexpr (sizeof(T) == 2)
        static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
    else
        static_cast<float*>(p)[i] = v;
}
template <typename T>
__device__ __forceinline__ float as_stored(float v) {
    if constexpr (sizeof(T) == 2)
        return __bfloat162float(__float2bfloat16_rn(v));
    else
        return v;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

struct Stat {
    float mu, rho;
};

__device__ __forceinline__ float gamma_at(const NormP& p, int64_t j) { return p.gamma ? p.gamma[j] : 1.0f; }

// ------------------------------------------------------------- rows of any width
// For rows that the kernels below do not hold (over 16384 wide): a CTA of 1024 threads per row, which
// it reads once per pass, four elements a thread at a time, all of their reads under
// way together.
constexpr int kWide = 1024;

// Sum over the CTA, to every thread, in a fixed order; `red` holds 32 floats.
__device__ __forceinline__ float wide_sum(float v, float* red) {
    v = warp_sum(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    return warp_sum(red[threadIdx.x & 31]);
}

// The thread's four elements of a pass's turn at `base`: of a row, of a vector (or
// what stands for it), of the gate.
template <typename T>
__device__ __forceinline__ void row4(const void* x, int64_t at, int64_t base, int64_t n, float (&v)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t j = base + i * kWide + threadIdx.x;
        v[i] = j < n ? ld<T>(x, at + j) : 0.0f;
    }
}
__device__ __forceinline__ void vector4(const float* x, float other, int64_t base, int64_t n, float (&v)[4], int stride = 1) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t j = base + i * kWide + threadIdx.x;
        v[i] = x && j < n ? x[j * stride] : other;
    }
}
template <typename T>
__device__ __forceinline__ void gate4(const BlockP& p, int64_t row, int64_t base, int64_t n, float (&v)[4]) {
    if (p.gate_mode == GATE_FULL)
        row4<T>(p.gate, row * p.ldg, base, n, v);
    else
        vector4(p.gate_mode == GATE_NONE ? nullptr
                                         : static_cast<const float*>(p.gate) + (p.gate_mode == GATE_COLUMN ? row * p.ldg : 0),
                1.0f, base, n, v, p.gate_mode == GATE_ROW ? 1 : 0);
}

// Mean (layer) and reciprocal deviation of a row; x(base, v) gives four elements,
// zeros past the end.
template <typename F>
__device__ __forceinline__ Stat row_stat(const NormP& p, int64_t n, float* red, F x) {
    Stat s{0.0f, 1.0f};
    if (p.kind == RT_NORM_NONE) return s;
    if (p.kind == RT_NORM_LAYER) {
        float t = 0.0f;
        for (int64_t base = 0; base < n; base += 4 * kWide) {
            float v[4];
            x(base, v);
            t += (v[0] + v[1]) + (v[2] + v[3]);
        }
        s.mu = wide_sum(t, red) / (float)n;
    }
    float t = 0.0f;
    for (int64_t base = 0; base < n; base += 4 * kWide) {
        float v[4];
        x(base, v);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float d = base + i * kWide + threadIdx.x < n ? v[i] - s.mu : 0.0f;
            t += d * d;
        }
    }
    s.rho = rsqrtf(wide_sum(t, red) / (float)n + p.eps);
    return s;
}

// One block of 32 in 4 bits by a whole warp, a lane's element h at j.
__device__ __forceinline__ void store_block(const BlockP& p, int64_t row, int64_t j, int64_t blocks, int64_t groups, float h) {
    const int lane = threadIdx.x & 31;
    const uint32_t amax = __reduce_max_sync(0xffffffffu, __float_as_uint(h) & 0x7fffffffu);
    const uint32_t byte = mx4::scale_byte(amax);
    const float q = byte == mx4::kNanScale ? 0.0f : h * mx4::inv_scale(byte);
    const float next = __shfl_down_sync(0xffffffffu, q, 1);
    if ((lane & 1) == 0) p.codes[row * blocks * 16 + (j >> 1)] = (uint8_t)mx4::encode2(q, next);
    if (lane == 0) {
        p.scales[mx4::scale_offset(row, j >> 5, groups)] = (uint8_t)byte;
        if ((j >> 5) == blocks - 1)
            for (int64_t b = blocks; b < groups * 4; ++b) p.scales[mx4::scale_offset(row, b, groups)] = 0;
    }
}

template <typename T>
__global__ void __launch_bounds__(kWide) forward_kernel(BlockP p) {
    __shared__ float red[32];
    pdl_wait();
    pdl_launch_dependents();
    const int64_t n = p.n, blocks = (n + 31) / 32, groups = (blocks + 3) / 4;
    for (int64_t row = blockIdx.x; row < p.m; row += gridDim.x) {
        Stat sy{0.0f, 1.0f};
        if (p.y) sy = row_stat(p.post, n, red, [&](int64_t base, float (&v)[4]) { row4<T>(p.y, row * p.ldy, base, n, v); });
        auto z4 = [&](int64_t base, float (&z)[4]) {
            row4<T>(p.r, row * p.ldr, base, n, z);
            if (!p.y) return;
            float y[4], gamma[4], beta[4], gate[4];
            row4<T>(p.y, row * p.ldy, base, n, y);
            vector4(p.post.gamma, 1.0f, base, n, gamma);
            vector4(p.post.beta, 0.0f, base, n, beta);
            gate4<T>(p, row, base, n, gate);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (base + i * kWide + threadIdx.x < n)
                    z[i] += p.scale * gate[i] * ((y[i] - sy.mu) * sy.rho * gamma[i] + beta[i]);
        };
        const Stat sz = row_stat(p.pre, n, red, z4);
        for (int64_t base = 0; base < n; base += 4 * kWide) {
            float z[4], gamma[4], beta[4];
            z4(base, z);
            vector4(p.pre.gamma, 1.0f, base, n, gamma);
            vector4(p.pre.beta, 0.0f, base, n, beta);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int64_t j = base + i * kWide + threadIdx.x;
                const float h = j < n ? (z[i] - sz.mu) * sz.rho * gamma[i] + beta[i] : 0.0f;
                if (j < n && p.z) st<T>(p.z, row * p.ldz + j, z[i]);
                if (j < n && p.h) st<T>(p.h, row * p.ldh + j, h);
                if (p.codes && (j & ~int64_t(31)) < n) store_block(p, row, j, blocks, groups, as_stored<T>(h));
            }
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(kWide) backward_kernel(BlockP p, GradP g) {
    __shared__ float red[32];
    pdl_wait();
    pdl_launch_dependents();
    const int64_t n = p.n;
    const int64_t cols = columns(n);
    float* acc = g.partials ? g.partials + (int64_t)blockIdx.x * 4 * cols : nullptr;
    if (acc)
        for (int64_t i = threadIdx.x; i < 4 * cols; i += kWide)
            if ((g.sums >> (i / cols)) & 1) acc[i] = 0.0f;
    __syncthreads();
    const float inv_n = 1.0f / (float)n;
    const bool own_gate = p.gate_mode >= GATE_COLUMN;
    for (int64_t row = blockIdx.x; row < p.m; row += gridDim.x) {
        auto z4 = [&](int64_t base, float (&v)[4]) { row4<T>(p.z, row * p.ldz, base, n, v); };
        auto y4 = [&](int64_t base, float (&v)[4]) { row4<T>(p.y, row * p.ldy, base, n, v); };
        const Stat sz = row_stat(p.pre, n, red, z4);
        Stat sy{0.0f, 1.0f};
        if (p.y) sy = row_stat(p.post, n, red, y4);
        // means of a and a z^ of the norm before the next block
        float a0 = 0.0f, a1 = 0.0f;
        if (g.dh && p.pre.kind != RT_NORM_NONE) {
            for (int64_t base = 0; base < n; base += 4 * kWide) {
                float z[4], d[4], gamma[4];
                z4(base, z);
                row4<T>(g.dh, row * g.lddh, base, n, d);
                vector4(p.pre.gamma, 1.0f, base, n, gamma);
#pragma unroll
                for (int i = 0; i < 4; ++i) {  // d is zero past the row's end
                    a0 += d[i] * gamma[i];
                    a1 += d[i] * gamma[i] * ((z[i] - sz.mu) * sz.rho);
                }
            }
            a0 = p.pre.kind == RT_NORM_LAYER ? wide_sum(a0, red) * inv_n : 0.0f;
            a1 = wide_sum(a1, red) * inv_n;
        }
        // four elements of dr; dh and z^ beside it
        auto dr4 = [&](int64_t base, float (&dr)[4], float (&d)[4], float (&hat)[4]) {
#pragma unroll
            for (int i = 0; i < 4; ++i) dr[i] = d[i] = hat[i] = 0.0f;
            float gamma[4];
            if (g.dz) row4<T>(g.dz, row * g.lddz, base, n, dr);
            if (!g.dh) return;
            row4<T>(g.dh, row * g.lddh, base, n, d);
            // without a norm z has no part in dr: an infinity in it would be a NaN times a1 = 0
            if (p.pre.kind != RT_NORM_NONE) z4(base, hat);
            vector4(p.pre.gamma, 1.0f, base, n, gamma);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                hat[i] = (hat[i] - sz.mu) * sz.rho;
                if (base + i * kWide + threadIdx.x < n) dr[i] += (d[i] * gamma[i] - a0 - hat[i] * a1) * sz.rho;
            }
        };
        float b0 = 0.0f, b1 = 0.0f;
        const bool normed = p.post.kind != RT_NORM_NONE;  // else y has no part in dy
        if (p.y) {
            float gsum = 0.0f;
            for (int64_t base = 0; base < n; base += 4 * kWide) {
                float dr[4], d[4], hat[4], y[4], gate[4], gamma[4], beta[4];
                dr4(base, dr, d, hat);
                y4(base, y);
                gate4<T>(p, row, base, n, gate);
                vector4(p.post.gamma, 1.0f, base, n, gamma);
                vector4(p.post.beta, 0.0f, base, n, beta);
#pragma unroll
                for (int i = 0; i < 4; ++i) {  // dr is zero past the row's end
                    const float dt = p.scale * dr[i], yh = (y[i] - sy.mu) * sy.rho, b = dt * gate[i] * gamma[i];
                    b0 += b;
                    b1 += b * yh;
                    gsum += dt * (yh * gamma[i] + beta[i]);
                }
            }
            b0 = p.post.kind == RT_NORM_LAYER ? wide_sum(b0, red) * inv_n : 0.0f;
            b1 = p.post.kind != RT_NORM_NONE ? wide_sum(b1, red) * inv_n : 0.0f;
            if (g.dgate && p.gate_mode == GATE_COLUMN) {
                gsum = wide_sum(gsum, red);
                if (threadIdx.x == 0) static_cast<float*>(g.dgate)[row * g.lddg] = gsum;
            }
        }
        for (int64_t base = 0; base < n; base += 4 * kWide) {
            float dr[4], d[4], hat[4], y[4], gate[4], gamma[4], beta[4], sum[4][4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if ((g.sums >> k) & 1) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int64_t j = base + i * kWide + threadIdx.x;
                        sum[k][i] = j < n ? acc[k * cols + j] : 0.0f;
                    }
                }
            dr4(base, dr, d, hat);
            if (p.y) {
                y4(base, y);
                gate4<T>(p, row, base, n, gate);
                vector4(p.post.gamma, 1.0f, base, n, gamma);
                vector4(p.post.beta, 0.0f, base, n, beta);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int64_t j = base + i * kWide + threadIdx.x;
                if (j >= n) continue;
                if (p.y) {
                    const float dt = p.scale * dr[i], yh = (y[i] - sy.mu) * sy.rho, b = dt * gate[i] * gamma[i];
                    if (g.dy) st<T>(g.dy, row * g.lddy + j, (b - b0 - (normed ? yh : 0.0f) * b1) * sy.rho);
                    if (g.dgate && p.gate_mode == GATE_FULL)
                        st<T>(g.dgate, row * g.lddg + j, dt * (yh * gamma[i] + beta[i]));
                    const float w = own_gate ? dr[i] * gate[i] : dr[i];
                    if (g.sums & 1) acc[j] = sum[0][i] + w * yh;
                    if (g.sums & 2) acc[cols + j] = sum[1][i] + w;
                }
                if (g.dh) {
                    if (g.sums & 4) acc[2 * cols + j] = sum[2][i] + d[i] * hat[i];
                    if (g.sums & 8) acc[3 * cols + j] = sum[3][i] + d[i];
                }
                if (g.dr) st<T>(g.dr, row * g.lddr + j, dr[i]);
            }
        }
    }
}

// ------------------------------------------------------- rows in registers
// Eight elements as they are stored: 16 bytes of bf16, 32 of f32.
template <typename T>
struct Raw8 {
    uint4 u[sizeof(T) / 2];
};
template <typename T>
__device__ __forceinline__ Raw8<T> zero8() {
    Raw8<T> r;
#pragma unroll
    for (auto& x : r.u) x = make_uint4(0, 0, 0, 0);
    return r;
}
template <typename T>
__device__ __forceinline__ Raw8<T> load_raw8(const void* base, int64_t at) {
    const uint4* p = reinterpret_cast<const uint4*>(static_cast<const T*>(base) + at);
    Raw8<T> r;
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.u[i] = p[i];
    return r;
}
template <typename T>
__device__ __forceinline__ void unpack8(const Raw8<T>& r, float (&v)[8]) {
    if constexpr (sizeof(T) == 2) {
        const uint32_t w[4] = {r.u[0].x, r.u[0].y, r.u[0].z, r.u[0].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    } else {
        const uint32_t w[8] = {r.u[0].x, r.u[0].y, r.u[0].z, r.u[0].w, r.u[1].x, r.u[1].y, r.u[1].z, r.u[1].w};
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
    }
}
template <typename T>
__device__ __forceinline__ void store8(void* base, int64_t at, const float (&v)[8]) {
    uint4* p = reinterpret_cast<uint4*>(static_cast<T*>(base) + at);
    uint32_t w[8];
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
        p[0] = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(v[i]);
        p[0] = make_uint4(w[0], w[1], w[2], w[3]);
        p[1] = make_uint4(w[4], w[5], w[6], w[7]);
    }
}
// v = p[at..], or `other` where there is no vector.
__device__ __forceinline__ void vector8(const float* p, int64_t at, float other, float (&v)[8]) {
    if (p) {
        const float4 a = *reinterpret_cast<const float4*>(p + at), b = reinterpret_cast<const float4*>(p + at)[1];
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
        v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = other;
    }
}

// Sum over the TPR threads of a row, to each of them, in a fixed order.  `red`
// holds 2 x 32 floats of the row; `turn` alternates between the halves, so one
// barrier a sum is enough.  Rows of more than a warp in a CTA of several rows
// share the CTA's barrier: all rows make the same sums.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* red, int& turn) {
    v = warp_sum(v);
    if constexpr (TPR > 32) {
        constexpr int W = TPR / 32;
        float* half = red + turn * 32;
        turn ^= 1;
        if ((threadIdx.x & 31) == 0) half[(threadIdx.x % TPR) >> 5] = v;
        __syncthreads();
        v = (threadIdx.x & 31) < W ? half[threadIdx.x & 31] : 0.0f;
#pragma unroll
        for (int o = W / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        v = __shfl_sync(0xffffffffu, v, 0);
    }
    return v;
}

// Mean and reciprocal deviation of a row held 8 C elements a thread.  (rsqrtf, here
// and below, is within 2 units in the last place: sums of hundreds of rounded terms
// precede it.)
template <int TPR, int C>
__device__ __forceinline__ Stat stat_of(const NormP& p, const float (&x)[C][8], const bool (&has)[C], float inv_n,
                                        float* red, int& turn) {
    Stat s{0.0f, 1.0f};
    if (p.kind == RT_NORM_NONE) return s;
    if (p.kind == RT_NORM_LAYER) {
        float t = 0.0f;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) t += x[c][i];  // zeros where the row has ended
        s.mu = row_sum<TPR>(t, red, turn) * inv_n;
    }
    float t = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c)
        if (has[c])
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float d = x[c][i] - s.mu;
                t += d * d;
            }
    s.rho = rsqrtf(row_sum<TPR>(t, red, turn) * inv_n + p.eps);
    return s;
}

// Eight elements of h, stored and in 4 bits; called by whole warps, `has` where
// the eight lie in the row (which `live` says exists).
template <typename T>
__device__ __forceinline__ void store_h(const BlockP& p, int64_t row, int j, bool live, bool has, float (&h)[8]) {
    if (p.h && has) store8<T>(p.h, row * p.ldh + j, h);
    if (!p.codes) return;
    const int blocks = (int)((p.n + 31) / 32), groups = (blocks + 3) / 4;
    // four neighbouring lanes hold a block of 32
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        h[i] = has ? as_stored<T>(h[i]) : 0.0f;
        amax = max(amax, __float_as_uint(h[i]) & 0x7fffffffu);
    }
    amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    const uint32_t byte = mx4::scale_byte(amax);
    const float inv = mx4::inv_scale(byte);
    uint32_t code = mx4::encode8(h, inv);
    if (byte == mx4::kNanScale) code = 0;
    if (live && j < blocks * 32) *reinterpret_cast<uint32_t*>(p.codes + row * blocks * 16 + (j >> 1)) = code;
    // the scales of a group's four blocks as one word
    uint32_t word = byte | __shfl_down_sync(0xffffffffu, byte, 4) << 8;
    word |= __shfl_down_sync(0xffffffffu, word, 8) << 16;
    if (live && (threadIdx.x & 15) == 0 && j < groups * 128)
        *reinterpret_cast<uint32_t*>(p.scales + mx4::scale_offset(row, j >> 5, groups)) = word;
}

// One pass: a row lies in the registers of TPR threads, 8 neighbouring elements
// in each of C turns, so y and r are read once, z and h written once and the
// sums of a norm are taken twice over the same registers (mean, then the centred
// squares).  HBM-bound: 4 elements moved for each of the row; few rows are bound by
// the launch (one of 8192 bf16: 4 to 5 us in a stream of launches).  Needs 16-byte
// aligned rows and whole eights (n % 8 = 0); a CTA holds ROWS = max(1, 128 / TPR)
// rows.
constexpr int cta_threads(int tpr) { return tpr < 128 ? 128 : tpr; }

template <typename T, int TPR, int C>
__global__ void __launch_bounds__(cta_threads(TPR)) forward_rows_kernel(BlockP p) {
    constexpr int ROWS = cta_threads(TPR) / TPR;
    pdl_wait();
    pdl_launch_dependents();
    __shared__ float red_all[ROWS][64];
    float* red = red_all[threadIdx.x / TPR];
    int turn = 0;
    const int t = threadIdx.x % TPR;
    const int n = (int)p.n;
    const float inv_n = 1.0f / (float)n;
    const int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / TPR;
    const bool live = row < p.m;
    bool has[C];
    float z[C][8];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        has[c] = live && (c * TPR + t) * 8 < n;
        const Raw8<T> raw = has[c] ? load_raw8<T>(p.r, row * p.ldr + (c * TPR + t) * 8) : zero8<T>();
        unpack8<T>(raw, z[c]);
    }
    if (p.y) {
        float y[C][8];
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const Raw8<T> raw = has[c] ? load_raw8<T>(p.y, row * p.ldy + (c * TPR + t) * 8) : zero8<T>();
            unpack8<T>(raw, y[c]);
        }
        const Stat s = stat_of<TPR, C>(p.post, y, has, inv_n, red, turn);
        const float one = p.gate_mode == GATE_ONE              ? *static_cast<const float*>(p.gate)
                          : p.gate_mode == GATE_COLUMN && live ? static_cast<const float*>(p.gate)[row * p.ldg]
                                                               : 1.0f;
#pragma unroll
        for (int c = 0; c < C; ++c)
            if (has[c]) {
                const int j = (c * TPR + t) * 8;
                float gamma[8], beta[8], gate[8];
                vector8(p.post.gamma, j, 1.0f, gamma);
                vector8(p.post.beta, j, 0.0f, beta);
                if (p.gate_mode == GATE_FULL)
                    unpack8<T>(load_raw8<T>(p.gate, row * p.ldg + j), gate);
                else
                    vector8(p.gate_mode == GATE_ROW ? static_cast<const float*>(p.gate) : nullptr, j, one, gate);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float u = (y[c][i] - s.mu) * s.rho * gamma[i] + beta[i];
                    z[c][i] += p.scale * gate[i] * u;
                }
            }
    }
    const Stat s = stat_of<TPR, C>(p.pre, z, has, inv_n, red, turn);
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int j = (c * TPR + t) * 8;
        if (has[c]) {
            if (p.z) store8<T>(p.z, row * p.ldz + j, z[c]);
            float gamma[8], beta[8];
            vector8(p.pre.gamma, j, 1.0f, gamma);
            vector8(p.pre.beta, j, 0.0f, beta);
#pragma unroll
            for (int i = 0; i < 8; ++i) z[c][i] = (z[c][i] - s.mu) * s.rho * gamma[i] + beta[i];
        }
        store_h<T>(p, row, j, live, has[c], z[c]);
    }
}

// ---------------------------------------------------- rows of any alignment
// The same for rows that are not 16-byte aligned or whole eights (an odd width): a
// thread holds every S-th element, so a warp's 2- or 4-byte accesses are always
// neighbours.  E elements a thread; WARP: a warp to a row (four to a CTA), else a
// CTA, of as many warps as the row needs.
__device__ __forceinline__ float cta_sum(float v, float* red, int& turn) {
    v = warp_sum(v);
    const int lane = threadIdx.x & 31;
    float* half = red + turn * 32;
    turn ^= 1;
    if (lane == 0) half[threadIdx.x >> 5] = v;
    __syncthreads();
    return warp_sum(lane < (int)(blockDim.x >> 5) ? half[lane] : 0.0f);
}

template <typename T, bool WARP, int E>
__global__ void __launch_bounds__(WARP ? 128 : 1024) forward_strided_kernel(BlockP p) {
    pdl_wait();
    pdl_launch_dependents();
    __shared__ float red[64];
    int turn = 0;
    const int S = WARP ? 32 : (int)blockDim.x, t = WARP ? threadIdx.x & 31 : threadIdx.x;
    const int n = (int)p.n;
    const float inv_n = 1.0f / (float)n;
    const int64_t row = WARP ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5) : blockIdx.x;
    if (row >= p.m) return;  // a whole warp, and rows of a warp share no barrier
    auto sum = [&](float v) { return WARP ? warp_sum(v) : cta_sum(v, red, turn); };
    auto load = [&](auto x, float other, float (&v)[E]) {
#pragma unroll
        for (int i = 0; i < E; ++i) v[i] = i * S + t < n ? x(i * S + t) : other;
    };
    auto stat = [&](const NormP& norm, const float (&x)[E]) {
        Stat s{0.0f, 1.0f};
        if (norm.kind == RT_NORM_NONE) return s;
        float v = 0.0f;
        if (norm.kind == RT_NORM_LAYER) {
#pragma unroll
            for (int i = 0; i < E; ++i) v += x[i];
            s.mu = sum(v) * inv_n;
            v = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const float d = i * S + t < n ? x[i] - s.mu : 0.0f;
            v += d * d;
        }
        s.rho = rsqrtf(sum(v) * inv_n + norm.eps);
        return s;
    };
    // x = x^ gamma + beta
    auto scale = [&](const Stat& s, const float (&gamma)[E], const float* beta, float (&x)[E]) {
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] = (x[i] - s.mu) * s.rho * gamma[i];
        if (beta) {
            float w[E];
            load([&](int j) { return beta[j]; }, 0.0f, w);
#pragma unroll
            for (int i = 0; i < E; ++i) x[i] += w[i];
        }
    };
    // the vectors are on their way while the sums are taken; one choice for all of a
    // thread's elements, so that their reads are under way together
    auto vector = [&](const float* x, int stride, float (&v)[E]) {
        if (x)
            load([&](int j) { return x[(int64_t)j * stride]; }, 0.0f, v);
        else
#pragma unroll
            for (int i = 0; i < E; ++i) v[i] = 1.0f;
    };
    float z[E], gamma[E];
    load([&](int j) { return ld<T>(p.r, row * p.ldr + j); }, 0.0f, z);
    if (p.y) {
        float y[E], gate[E];
        load([&](int j) { return ld<T>(p.y, row * p.ldy + j); }, 0.0f, y);
        vector(p.post.gamma, 1, gamma);
        if (p.gate_mode == GATE_FULL)
            load([&](int j) { return ld<T>(p.gate, row * p.ldg + j); }, 0.0f, gate);
        else
            vector(p.gate_mode == GATE_NONE ? nullptr
                                            : static_cast<const float*>(p.gate) + (p.gate_mode == GATE_COLUMN ? row * p.ldg : 0),
                   p.gate_mode == GATE_ROW ? 1 : 0, gate);
        scale(stat(p.post, y), gamma, p.post.beta, y);
#pragma unroll
        for (int i = 0; i < E; ++i) z[i] += i * S + t < n ? p.scale * gate[i] * y[i] : 0.0f;
    }
    vector(p.pre.gamma, 1, gamma);
    const Stat s = stat(p.pre, z);
    if (p.z)
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (i * S + t < n) st<T>(p.z, row * p.ldz + i * S + t, z[i]);
    scale(s, gamma, p.pre.beta, z);
    if (p.h)
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (i * S + t < n) st<T>(p.h, row * p.ldh + i * S + t, z[i]);
    if (!p.codes) return;
    const int blocks = (n + 31) / 32, groups = (blocks + 3) / 4;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const int j = i * S + t;  // a warp holds one block of 32
        if (i * S + (t & ~31) < n) store_block(p, row, j, blocks, groups, j < n ? as_stored<T>(z[i]) : 0.0f);
    }
}

// ------------------------------------------------------ rows through a ring
// For many rows: one CTA of 1024 threads (backward: 512, for the registers that its
// sums over rows take) to an SM, its groups of TPR threads each take a row at a
// time.  The rows arrive by bulk copies into a ring of slots, so
// the next rows are on their way while this one is summed, however few registers
// that leaves; the vectors (gamma, beta and a gate of one row, folded together
// where they meet) lie in shared memory once, in f32.
constexpr int kRingThreads = 1024;
constexpr int kRingSmem = 227 * 1024;
// a group's sums [2][warps of its cluster, 32 at least][4], its barriers (up to eight),
// the abort flag and where each group gave up
constexpr int sum_floats(int cluster) { return cluster > 2 ? 128 * cluster : 256; }
constexpr int ring_scratch(int groups, int cluster) { return groups * (sum_floats(cluster) * 4 + 64 + 4) + 16; }

struct RingP {
    int depth;         // slots of a group
    int slot_bytes;    // the row of each tensor
    int vectors;       // f32 vectors in shared memory
    int smem;          // bytes in all: what they leave is L1
    int* err;
};

// Warp sums of four values by halves: each exchange hands over the values that
// the other half of the lanes goes on with, 6 shuffles in all and not 20.  Lane l
// returns the sum of value l >> 3.
__device__ __forceinline__ float warp_sum4(float v0, float v1, float v2, float v3) {
    const int lane = threadIdx.x & 31;
    const bool hi = lane & 16;
    float a = (hi ? v2 : v0) + __shfl_xor_sync(0xffffffffu, hi ? v0 : v2, 16);
    float b = (hi ? v3 : v1) + __shfl_xor_sync(0xffffffffu, hi ? v1 : v3, 16);
    const bool odd = lane & 8;
    a = (odd ? b : a) + __shfl_xor_sync(0xffffffffu, odd ? a : b, 8);
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
    return a;
}

// The threads of a row: TPR of a CTA, or (CL > 1) the CTAs of a cluster, each with its
// share of the columns.
template <int THREADS, int TPR, int CL = 1>
struct Group {
    static_assert(CL == 1 || TPR == THREADS, "a cluster's row takes whole CTAs");
    static constexpr int COUNT = THREADS / TPR, W = TPR / 32, HALF = sum_floats(CL) / 2;
    int index, t;    // of the group in its CTA, of the thread in its group
    float* red;      // [2][warps][4]
    int turn = 0;
    int rank = 0;        // of the CTA in its cluster
    uint32_t there = 0;  // CL > 1: red of the CTA that this lane hands its warp's sums to

    __device__ __forceinline__ void join_cluster() {
        if constexpr (CL > 1) {
            uint32_t at = tc::smem_u32(red);
            asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(at), "r"(threadIdx.x & (CL - 1)));
            sync_row();  // every CTA runs before it is written to
        }
    }
    // Waits for all that take the row; what they handed over is then here.
    __device__ __forceinline__ void sync_row() const {
        if constexpr (CL > 1)
            asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        else
            sync();
    }
    // A value of the warp to every CTA of the row: called by CL neighbouring lanes.
    __device__ __forceinline__ void hand(int at, float v) const {
        if constexpr (CL > 1)
            asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(there + (uint32_t)(turn * HALF + at) * 4), "f"(v) : "memory");
        else
            red[turn * HALF + at] = v;
    }
    __device__ __forceinline__ void sync() const {
        if constexpr (TPR == 32)
            __syncwarp();
        else if constexpr (TPR == THREADS)
            __syncthreads();
        else
            asm volatile("bar.sync %0, %1;" ::"r"(1 + index), "n"(TPR) : "memory");
    }
    // Sums over the group, to every thread, in a fixed order; one barrier.
    __device__ __forceinline__ void sum(float& v) {
        v = warp_sum(v);
        if constexpr (TPR == 32) {
            __syncwarp();
        } else {
            const int lane = threadIdx.x & 31;
            const float* half = red + turn * HALF;
            if (lane < CL) hand(rank * W + (t >> 5), v);
            turn ^= 1;
            sync_row();
            v = half[lane % (W * CL)];
            if constexpr (W * CL > 32) v += half[lane + 32];
#pragma unroll
            for (int o = (W * CL > 32 ? 32 : W * CL) / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        }
    }
    template <int K>
    __device__ __forceinline__ void sum(float (&v)[K]) {
        static_assert(K == 3 || K == 4, "three or four sums at a time");
        float a = warp_sum4(v[0], v[1], v[2], K == 4 ? v[K - 1] : 0.0f);
        const int lane = threadIdx.x & 31;
        if constexpr (TPR == 32) {
            __syncwarp();
        } else {
            const float* half = red + turn * HALF;
            if ((lane & 7) < CL) hand((rank * W + (t >> 5)) * 4 + (lane >> 3), a);
            turn ^= 1;
            sync_row();
            float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (lane < W * CL) x = *reinterpret_cast<const float4*>(half + lane * 4);
            if constexpr (W * CL > 32) {
                const float4 y = *reinterpret_cast<const float4*>(half + (lane + 32) * 4);
                x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
            }
            a = warp_sum4(x.x, x.y, x.z, K == 4 ? x.w : 0.0f);
        }
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = __shfl_sync(0xffffffffu, a, k * 8);
    }
};

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
                 "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}

// A wait that gave up leaves its slot and phase for the end of the kernel, where
// the thread that issues (it issues no more) waits, again with a limit, for the
// copies on their way.  That wait inside the loop took backward_pipe_kernel from
// 144 to 158 us at 8192x8192, although no call reached it.
__device__ __forceinline__ void gave_up(const RingP& r, volatile int* abort_flag, int group, int slot, uint32_t phase) {
    *abort_flag = 1;
    tc::record_error(r.err, DEV_TIMEOUT_ROWS, (int)blockIdx.x);
    if (group >= 0) abort_flag[1 + group] = slot * 2 + (int)phase;
}
__device__ __noinline__ void land_copies(uint32_t full, int depth, int count, int at) {
    volatile int never = 0;
    land_ring(depth, count, at >> 1, at & 1, [&](int slot, uint32_t phase) { tc::mbar_wait(full + slot * 8, phase, &never); });
}

// Shared memory of a ring kernel: vectors, slots, sums, barriers.
struct RingSmem {
    float* vec;
    uint8_t* slots;
    float* red;
    uint64_t* full;
};
__device__ __forceinline__ RingSmem ring_smem(uint8_t* smem, const RingP& r, int n, int groups, int cluster = 1) {
    RingSmem s;
    s.vec = reinterpret_cast<float*>(smem);
    s.slots = smem + (size_t)r.vectors * n * 4;
    s.red = reinterpret_cast<float*>(s.slots + (size_t)groups * r.depth * r.slot_bytes);
    s.full = reinterpret_cast<uint64_t*>(s.red + groups * sum_floats(cluster));
    return s;
}

// Pairs of f32 in one 64-bit register and Blackwell's packed arithmetic on them:
// the ring kernels would otherwise be bound by instructions, not by HBM.
using f2 = unsigned long long;
__device__ __forceinline__ f2 pack2(float a, float b) {
    f2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 unpack2(f2 a) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a));
    return r;
}
__device__ __forceinline__ f2 splat2(float a) { return pack2(a, a); }
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
    f2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
    f2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
    f2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float both(f2 a) {
    const float2 x = unpack2(a);
    return x.x + x.y;
}

// Eight elements as pairs: of a register's worth of bf16, of a slot's row, of a
// vector in shared memory.
__device__ __forceinline__ void pairs8(const Raw8<float>& r, f2 (&v)[4]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        v[2 * i] = pack2(__uint_as_float(r.u[i].x), __uint_as_float(r.u[i].y));
        v[2 * i + 1] = pack2(__uint_as_float(r.u[i].z), __uint_as_float(r.u[i].w));
    }
}
__device__ __forceinline__ void pairs8(const Raw8<__nv_bfloat16>& r, f2 (&v)[4]) {
    const uint32_t w[4] = {r.u[0].x, r.u[0].y, r.u[0].z, r.u[0].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = pack2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
}
template <typename T>
__device__ __forceinline__ void slot8(const uint8_t* row, int j, f2 (&v)[4]) {
    const uint4* p = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(row) + j);
    Raw8<T> raw;
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) raw.u[i] = p[i];
    pairs8(raw, v);
}
__device__ __forceinline__ void vec8(const float* p, int j, f2 (&v)[4]) {
    const ulonglong2 a = *reinterpret_cast<const ulonglong2*>(p + j), b = *reinterpret_cast<const ulonglong2*>(p + j + 4);
    v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
}
__device__ __forceinline__ void floats8(const f2 (&v)[4], float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 a = unpack2(v[i]);
        x[2 * i] = a.x;
        x[2 * i + 1] = a.y;
    }
}
// The pair with what lies past a row's end as zeros: `left` elements are in it.
__device__ __forceinline__ f2 keep2(f2 v, int left) {
    return left >= 2 ? v : left == 1 ? v & 0xffffffffull : 0ull;
}
template <typename T>
__device__ __forceinline__ void store8(void* base, int64_t at, const f2 (&v)[4]) {
    float x[8];
    floats8(v, x);
    store8<T>(base, at, x);
}

// The gate where it is the same for every row (1 where it is not).
__device__ __forceinline__ float shared_gate(const BlockP& p, int j) {
    return p.gate_mode == GATE_ONE   ? *static_cast<const float*>(p.gate)
           : p.gate_mode == GATE_ROW ? static_cast<const float*>(p.gate)[j]
                                     : 1.0f;
}

// Forward.  Slots hold r and y; vectors P = s g gamma_post, Q = s g beta_post (g
// where all rows share it), gamma_pre, beta_pre, those that there are (mask 1 2 4
// 8).  8192 x 8192 bf16, RMS norms and a gate: 94 to 101 us, 5.3 to 5.7 TB/s, HBM-bound (a
// device copy reaches 6.55); forward_rows_kernel, whose reads wait behind each row's
// sums, took 241.
// FULL: with layer norms, betas and gates that rows do not share; else RMS norms
// and shared gates alone.
template <typename T, int TPR, int C, bool FULL>
__global__ void __launch_bounds__(kRingThreads, 1) forward_ring_kernel(BlockP p, RingP r, int mask) {
    extern __shared__ __align__(128) uint8_t smem[];
    using G = Group<kRingThreads, TPR>;
    const int n = (int)p.n;
    const RingSmem sm = ring_smem(smem, r, n, G::COUNT);
    G g;
    g.index = threadIdx.x / TPR;
    g.t = threadIdx.x % TPR;
    g.red = sm.red + g.index * 256;
    uint8_t* slots = sm.slots + (size_t)g.index * r.depth * r.slot_bytes;
    const uint32_t full = tc::smem_u32(sm.full + g.index * r.depth);
    const uint32_t row_bytes = (uint32_t)n * sizeof(T);
    const int64_t step = (int64_t)gridDim.x * G::COUNT, first = (int64_t)blockIdx.x * G::COUNT + g.index;
    volatile int* abort_flag = reinterpret_cast<volatile int*>(sm.full + G::COUNT * r.depth);

    if (threadIdx.x == 0) {
        for (int i = 0; i < G::COUNT * r.depth; ++i) tc::mbar_init(tc::smem_u32(sm.full + i), 1);
        *abort_flag = 0;
        tc::fence_barrier_init();
    }
    pdl_wait();
    pdl_launch_dependents();
    float *vp = sm.vec, *vq = vp + (mask & 1 ? n : 0), *v2 = vq + (mask & 2 ? n : 0), *vb = v2 + (mask & 4 ? n : 0);
    for (int j = threadIdx.x; j < n; j += kRingThreads) {
        const float sg = p.scale * shared_gate(p, j);
        if (mask & 1) vp[j] = sg * (p.post.gamma ? p.post.gamma[j] : 1.0f);
        if (mask & 2) vq[j] = sg * p.post.beta[j];
        if (mask & 4) v2[j] = p.pre.gamma[j];
        if (mask & 8) vb[j] = p.pre.beta[j];
    }
    __syncthreads();
    bool ok = true;  // this thread's waits so far
    auto issue = [&](int64_t row, int slot) {
        const uint32_t bar = full + slot * 8, dst = tc::smem_u32(slots + (size_t)slot * r.slot_bytes);
        tc::mbar_expect_tx(bar, (uint32_t)r.slot_bytes);
        bulk_load(dst, static_cast<const T*>(p.r) + row * p.ldr, row_bytes, bar);
        if (p.y) bulk_load(dst + row_bytes, static_cast<const T*>(p.y) + row * p.ldy, row_bytes, bar);
    };
    if (g.t == 0)
        for (int d = 0; d < r.depth && first + d * step < p.m; ++d) issue(first + d * step, d);
    const float inv_n = 1.0f / (float)n;
    int slot = 0;
    uint32_t phase = 0;
    bool has[C];
#pragma unroll
    for (int c = 0; c < C; ++c) has[c] = (c * TPR + g.t) * 8 < n;
    for (int64_t row = first; row < p.m; row += step) {
        if (!tc::mbar_wait(full + slot * 8, phase, abort_flag)) {
            if (ok) gave_up(r, abort_flag, g.t == 0 ? g.index : -1, slot, phase);
            ok = false;
        }
        const uint8_t* at = slots + (size_t)slot * r.slot_bytes;
        f2 z[C][4];
#pragma unroll
        for (int c = 0; c < C; ++c) {
#pragma unroll
            for (int i = 0; i < 4; ++i) z[c][i] = 0;
            if (has[c]) slot8<T>(at, (c * TPR + g.t) * 8, z[c]);
        }
        if (p.y) {
            const uint8_t* ay = at + row_bytes;
            Stat s{0.0f, 1.0f};
            if (FULL && p.post.kind == RT_NORM_LAYER) {
                f2 v2x = 0;
#pragma unroll
                for (int c = 0; c < C; ++c)
                    if (has[c]) {
                        f2 y[4];
                        slot8<T>(ay, (c * TPR + g.t) * 8, y);
#pragma unroll
                        for (int i = 0; i < 4; ++i) v2x = add2(v2x, y[i]);
                    }
                float v = both(v2x);
                g.sum(v);
                s.mu = v * inv_n;
            }
            const f2 less_mu = splat2(-s.mu);
            if (p.post.kind != RT_NORM_NONE) {
                f2 v2x = 0;
#pragma unroll
                for (int c = 0; c < C; ++c)
                    if (has[c]) {
                        f2 y[4];
                        slot8<T>(ay, (c * TPR + g.t) * 8, y);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            if (FULL) y[i] = add2(y[i], less_mu);
                            v2x = fma2(y[i], y[i], v2x);
                        }
                    }
                float v = both(v2x);
                g.sum(v);
                s.rho = rsqrtf(v * inv_n + p.post.eps);
            }
            const f2 rho = splat2(mask & 1 ? s.rho : s.rho * p.scale);
#pragma unroll
            for (int c = 0; c < C; ++c)
                if (has[c]) {
                    const int j = (c * TPR + g.t) * 8;
                    f2 y[4], w[4];
                    slot8<T>(ay, j, y);
                    if (FULL)
#pragma unroll
                        for (int i = 0; i < 4; ++i) y[i] = add2(y[i], less_mu);
                    if (mask & 1) {
                        vec8(vp, j, w);
#pragma unroll
                        for (int i = 0; i < 4; ++i) y[i] = mul2(y[i], w[i]);
                    }
                    if (!FULL) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) z[c][i] = fma2(y[i], rho, z[c][i]);
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i) y[i] = mul2(y[i], rho);
                        if (mask & 2) {
                            vec8(vq, j, w);
#pragma unroll
                            for (int i = 0; i < 4; ++i) y[i] = add2(y[i], w[i]);
                        }
                        if (p.gate_mode == GATE_COLUMN) {
                            const f2 one = splat2(static_cast<const float*>(p.gate)[row * p.ldg]);
#pragma unroll
                            for (int i = 0; i < 4; ++i) y[i] = mul2(y[i], one);
                        } else if (p.gate_mode == GATE_FULL) {
                            slot8<T>(reinterpret_cast<const uint8_t*>(static_cast<const T*>(p.gate) + row * p.ldg), j, w);
#pragma unroll
                            for (int i = 0; i < 4; ++i) y[i] = mul2(y[i], w[i]);
                        }
#pragma unroll
                        for (int i = 0; i < 4; ++i) z[c][i] = add2(z[c][i], y[i]);
                    }
                }
        }
        // z is complete: its slot is free once the whole group is past the next barrier
        Stat s{0.0f, 1.0f};
        bool freed = false;
        auto refill = [&] {
            freed = true;
            if (g.t == 0 && ok && row + r.depth * step < p.m) issue(row + r.depth * step, slot);
        };
        if (FULL && p.pre.kind == RT_NORM_LAYER) {
            f2 v2x = 0;
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) v2x = add2(v2x, z[c][i]);
            float v = both(v2x);
            g.sum(v);
            refill();
            s.mu = v * inv_n;
        }
        const f2 less_mu = splat2(-s.mu);
        if (p.pre.kind != RT_NORM_NONE) {
            f2 v2x = 0;
#pragma unroll
            for (int c = 0; c < C; ++c)
                if (has[c])
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const f2 d = FULL ? add2(z[c][i], less_mu) : z[c][i];
                        v2x = fma2(d, d, v2x);
                    }
            float v = both(v2x);
            g.sum(v);
            if (!freed) refill();
            s.rho = rsqrtf(v * inv_n + p.pre.eps);
        }
        if (!freed) {
            g.sync();
            refill();
        }
        const f2 rho = splat2(s.rho);
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int j = (c * TPR + g.t) * 8;
            if (has[c]) {
                if (p.z) store8<T>(p.z, row * p.ldz + j, z[c]);
                f2 w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) z[c][i] = mul2(FULL ? add2(z[c][i], less_mu) : z[c][i], rho);
                if (mask & 4) {
                    vec8(v2, j, w);
#pragma unroll
                    for (int i = 0; i < 4; ++i) z[c][i] = mul2(z[c][i], w[i]);
                }
                if (FULL && (mask & 8)) {
                    vec8(vb, j, w);
#pragma unroll
                    for (int i = 0; i < 4; ++i) z[c][i] = add2(z[c][i], w[i]);
                }
            }
            float h[8];
            floats8(z[c], h);
            store_h<T>(p, row, j, true, has[c], h);
        }
        if (++slot == r.depth) {
            slot = 0;
            phase ^= 1;
        }
    }
    if (!ok && g.t == 0) land_copies(full, r.depth, r.depth, abort_flag[1 + g.index]);
}

// Backward.  Slots hold z and those of y, dz and dh that there are; vectors
// gamma_pre, P = s gamma_post (times g where all rows share it) and, for the
// gradient of a gate that rows do not share, s beta_post (mask 1 2 4).  A thread
// keeps the sums over rows of its eight columns in registers (FULL: those of the
// betas too); the groups' sums are joined in shared memory in order, one partial
// a CTA, and column_kernel adds the partials in order.
constexpr int kBackThreads = 512;

// Columns of each CTA of a cluster of CL (the last may have fewer): whole eights.
template <int CL>
__device__ __host__ __forceinline__ int share_of(int64_t n) {
    return CL == 1 ? (int)n : (int)columns((n + CL - 1) / CL);
}

// The sums of one kind of the groups that had a row, added in order through acc [n], to the partial
// `part` of rows of n columns, from column col0 on.
template <typename G, int C>
__device__ __forceinline__ void join_sums(const G& g, const GradP& q, float* acc, int groups, int64_t n, int part, int col0, int which,
                                          const f2 (&sums)[C][4], const int (&j)[C], const bool (&has)[C]) {
    if (!((q.sums >> which) & 1)) return;
    for (int k = 0; k < groups; ++k) {
        if (g.index == k)
#pragma unroll
            for (int c = 0; c < C; ++c)
                if (has[c]) {
                    f2* a = reinterpret_cast<f2*>(acc + j[c]);
                    f2 x[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[i] = k > 0 ? add2(a[i], sums[c][i]) : sums[c][i];
                    if (k == groups - 1)
                        a = reinterpret_cast<f2*>(q.partials + ((int64_t)part * 4 + which) * columns(n) + col0 + j[c]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) a[i] = x[i];
                }
        if (groups > 1) __syncthreads();
    }
}

// C: eights of a thread.  With the betas' sums a thread of sixteen columns spills
// (and with all of shared memory taken, spills go to L2), so FULL takes eight: 2047 x 1000 f32 layer norms, full gate: 26 to 29 us with the sums
// over columns behind it, 15 more with C = 2; bound by the latency of a row's barriers
// among 16 warps (3.5 rows a group).
//
// BULK: rows arrive by bulk copies, which want 16-byte aligned rows of whole eights.
// Else the group copies a row's tensors into its one slot itself, neighbouring
// elements by neighbouring threads, a row ending in zeros up to whole eights, and
// its results out of it likewise; groups of a CTA hide each other's waits.
//
// CL: CTAs of the cluster that shares a row, an equal share of its columns each.
template <typename T, int TPR, int C, bool FULL, bool BULK, int CL>
__global__ void __launch_bounds__(kBackThreads, 1) backward_ring_kernel(BlockP p, GradP q, RingP r, int mask) {
    extern __shared__ __align__(128) uint8_t smem[];
    using G = Group<kBackThreads, TPR, CL>;
    const int width = share_of<CL>(p.n), cols = (int)columns(width);
    const RingSmem sm = ring_smem(smem, r, cols, G::COUNT, CL);
    G g;
    g.index = threadIdx.x / TPR;
    g.t = threadIdx.x % TPR;
    g.red = sm.red + g.index * 256;
    g.join_cluster();
    // the CTA's columns: n from col0 on
    const int col0 = CL > 1 ? g.rank * width : 0, n = CL > 1 ? min(width, (int)p.n - col0) : (int)p.n;
    const int part = blockIdx.x / CL;
    uint8_t* slots = sm.slots + (size_t)g.index * r.depth * r.slot_bytes;
    const uint32_t full = tc::smem_u32(sm.full + g.index * r.depth);
    const uint32_t row_bytes = (uint32_t)(CL > 1 && BULK ? n : cols) * sizeof(T);
    // rows go to the thread blocks in turn, then to their groups: few rows spread over the device
    const int64_t parts = gridDim.x / CL, step = parts * G::COUNT, first = g.index * parts + part;
    const bool own_gate = FULL && (p.gate_mode == GATE_COLUMN || p.gate_mode == GATE_FULL);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(sm.full + G::COUNT * r.depth);

    if (threadIdx.x == 0) {
        for (int i = 0; i < G::COUNT * r.depth; ++i) tc::mbar_init(tc::smem_u32(sm.full + i), 1);
        *abort_flag = 0;
        tc::fence_barrier_init();
    }
    pdl_wait();
    pdl_launch_dependents();
    float *v2 = sm.vec, *vp = v2 + (mask & 1 ? cols : 0), *vb = vp + (mask & 2 ? cols : 0);
    for (int j = threadIdx.x; j < cols; j += kBackThreads) {
        const bool in = (BULK && CL == 1) || j < n;
        const int at = col0 + j;
        if (mask & 1) v2[j] = in ? p.pre.gamma[at] : 0.0f;
        if (mask & 2) vp[j] = in ? p.scale * shared_gate(p, at) * (p.post.gamma ? p.post.gamma[at] : 1.0f) : 0.0f;
        if (mask & 4) vb[j] = in ? p.scale * p.post.beta[at] : 0.0f;
    }
    __syncthreads();
    // the slot's rows: z, then y, dz, dh; not BULK: all of them, and a gate's
    const uint32_t at_y = row_bytes, at_dz = at_y + (p.y || !BULK ? row_bytes : 0),
                   at_dh = at_dz + (q.dz || !BULK ? row_bytes : 0), at_gate = at_dh + row_bytes;
    const uint32_t tensors = 1 + (p.y ? 1 : 0) + (q.dz ? 1 : 0) + (q.dh ? 1 : 0);
    bool ok = true;  // this thread's waits so far
    auto issue = [&](int64_t row, int slot) {
        const uint32_t bar = full + slot * 8, dst = tc::smem_u32(slots + (size_t)slot * r.slot_bytes);
        tc::mbar_expect_tx(bar, CL > 1 ? tensors * row_bytes : (uint32_t)r.slot_bytes);
        bulk_load(dst, static_cast<const T*>(p.z) + row * p.ldz + col0, row_bytes, bar);
        if (p.y) bulk_load(dst + at_y, static_cast<const T*>(p.y) + row * p.ldy + col0, row_bytes, bar);
        if (q.dz) bulk_load(dst + at_dz, static_cast<const T*>(q.dz) + row * q.lddz + col0, row_bytes, bar);
        if (q.dh) bulk_load(dst + at_dh, static_cast<const T*>(q.dh) + row * q.lddh + col0, row_bytes, bar);
    };
    // a row into the slot, or out of it, by the group (not BULK)
    // (every read of a row before its first write: the compiler cannot tell them apart)
    auto take_row = [&](const void* from, int64_t stride, int64_t row, T (&v)[8 * C]) {
        const T* x = static_cast<const T*>(from) + row * stride + col0 + g.t;
#pragma unroll
        for (int i = 0; i < 8 * C; ++i) v[i] = i * TPR + g.t < n ? x[i * TPR] : T(0.0f);
    };
    auto put_slot = [&](uint32_t to, const T (&v)[8 * C]) {
        T* d = reinterpret_cast<T*>(slots + to) + g.t;
#pragma unroll
        for (int i = 0; i < 8 * C; ++i)
            if (i * TPR + g.t < cols) d[i * TPR] = v[i];
    };
    auto copy_out = [&](void* to, int64_t stride, int64_t row, uint32_t from) {
        const T* x = reinterpret_cast<const T*>(slots + from) + g.t;
        T* d = static_cast<T*>(to) + row * stride + col0 + g.t;
        T v[8 * C];
#pragma unroll
        for (int i = 0; i < 8 * C; ++i) v[i] = i * TPR + g.t < n ? x[i * TPR] : T(0.0f);
#pragma unroll
        for (int i = 0; i < 8 * C; ++i)
            if (i * TPR + g.t < n) d[i * TPR] = v[i];
    };
    if (BULK && g.t == 0)
        for (int d = 0; d < r.depth && first + d * step < p.m; ++d) issue(first + d * step, d);
    const float inv_n = 1.0f / (float)p.n;
    int j[C];
    bool has[C];
    f2 sum_a[C][4], sum_b[FULL ? C : 1][4], sum_c[C][4], sum_d[FULL ? C : 1][4];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        j[c] = (c * TPR + g.t) * 8;
        has[c] = j[c] < n;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            sum_a[c][i] = sum_c[c][i] = 0;
            if constexpr (FULL) sum_b[c][i] = sum_d[c][i] = 0;
        }
    }
    int slot = 0;
    uint32_t phase = 0;
    const bool back = q.dh && p.pre.kind != RT_NORM_NONE;
    for (int64_t row = first; row < p.m; row += step) {
        if constexpr (BULK) {
            if (!tc::mbar_wait(full + slot * 8, phase, abort_flag)) {
                if (ok) gave_up(r, abort_flag, g.t == 0 ? g.index : -1, slot, phase);
                ok = false;
            }
        } else {
            T a[8 * C], b[8 * C];
            take_row(p.z, p.ldz, row, a);
            if (p.y) take_row(p.y, p.ldy, row, b);
            put_slot(0, a);
            if (p.y) put_slot(at_y, b);
            if (q.dz) take_row(q.dz, q.lddz, row, a);
            if (q.dh) take_row(q.dh, q.lddh, row, b);
            if (q.dz) put_slot(at_dz, a);
            if (q.dh) put_slot(at_dh, b);
            if (p.gate_mode == GATE_FULL) {
                take_row(p.gate, p.ldg, row, a);
                put_slot(at_gate, a);
            }
            g.sync();
        }
        const uint8_t* at = slots + (size_t)slot * r.slot_bytes;
        Raw8<T> own[FULL ? C : 1];  // a full gate's row: under way while the sums are taken
        if constexpr (FULL)
            if (p.gate_mode == GATE_FULL)
#pragma unroll
                for (int c = 0; c < C; ++c)
                    own[c] = !has[c] ? zero8<T>() : BULK ? load_raw8<T>(p.gate, row * p.ldg + col0 + j[c]) : load_raw8<T>(at + at_gate, j[c]);
        // sums of both norms: means first where there is a layer norm, then the
        // centred squares and a (z - mu)
        Stat sz{0.0f, 1.0f}, sy{0.0f, 1.0f};
        float a0 = 0.0f, a1 = 0.0f;
        if (FULL && (p.pre.kind == RT_NORM_LAYER || p.post.kind == RT_NORM_LAYER)) {
            f2 sums[3] = {0, 0, 0};
#pragma unroll
            for (int c = 0; c < C; ++c)
                if (has[c]) {
                    f2 x[4], w[4];
                    if (p.pre.kind == RT_NORM_LAYER) {
                        slot8<T>(at, j[c], x);
#pragma unroll
                        for (int i = 0; i < 4; ++i) sums[0] = add2(sums[0], x[i]);
                        if (back) {
                            slot8<T>(at + at_dh, j[c], x);
                            if (mask & 1) {
                                vec8(v2, j[c], w);
#pragma unroll
                                for (int i = 0; i < 4; ++i) x[i] = mul2(x[i], w[i]);
                            }
#pragma unroll
                            for (int i = 0; i < 4; ++i) sums[1] = add2(sums[1], x[i]);
                        }
                    }
                    if (p.post.kind == RT_NORM_LAYER) {
                        slot8<T>(at + at_y, j[c], x);
#pragma unroll
                        for (int i = 0; i < 4; ++i) sums[2] = add2(sums[2], x[i]);
                    }
                }
            float v[3] = {both(sums[0]), both(sums[1]), both(sums[2])};
            g.sum(v);
            sz.mu = v[0] * inv_n;
            a0 = v[1] * inv_n;
            sy.mu = v[2] * inv_n;
        }
        const f2 less_z = splat2(-sz.mu), less_y = splat2(-sy.mu);
        if (p.pre.kind != RT_NORM_NONE || p.post.kind != RT_NORM_NONE) {
            f2 sums[3] = {0, 0, 0};
#pragma unroll
            for (int c = 0; c < C; ++c)
                if (has[c]) {
                    f2 x[4];
                    if (p.pre.kind != RT_NORM_NONE) {
                        slot8<T>(at, j[c], x);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            if (FULL) x[i] = add2(x[i], less_z);
                            if (!BULK) x[i] = keep2(x[i], n - j[c] - 2 * i);
                            sums[0] = fma2(x[i], x[i], sums[0]);
                        }
                        if (back) {
                            f2 d[4], w[4];
                            slot8<T>(at + at_dh, j[c], d);
                            if (mask & 1) {
                                vec8(v2, j[c], w);
#pragma unroll
                                for (int i = 0; i < 4; ++i) d[i] = mul2(d[i], w[i]);
                            }
#pragma unroll
                            for (int i = 0; i < 4; ++i) sums[1] = fma2(d[i], x[i], sums[1]);
                        }
                    }
                    if (p.post.kind != RT_NORM_NONE) {
                        slot8<T>(at + at_y, j[c], x);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            if (FULL) x[i] = add2(x[i], less_y);
                            if (!BULK) x[i] = keep2(x[i], n - j[c] - 2 * i);
                            sums[2] = fma2(x[i], x[i], sums[2]);
                        }
                    }
                }
            float v[3] = {both(sums[0]), both(sums[1]), both(sums[2])};
            g.sum(v);
            if (p.pre.kind != RT_NORM_NONE) sz.rho = rsqrtf(v[0] * inv_n + p.pre.eps);
            if (p.post.kind != RT_NORM_NONE) sy.rho = rsqrtf(v[2] * inv_n + p.post.eps);
            a1 = v[1] * inv_n * sz.rho;  // mean of a z^
        }
        // dr and the sums over rows of dh; then b = s g gamma_post dr and its sums
        f2 b[C][4], hat[C][4];
        f2 sums[3] = {0, 0, 0};
#pragma unroll
        for (int c = 0; c < C; ++c) {
            if (!has[c]) continue;
            f2 dr[4], w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) dr[i] = 0;
            if (q.dz) slot8<T>(at + at_dz, j[c], dr);
            if (q.dh) {
                f2 d[4], h[4];
                const f2 rho = splat2(sz.rho), less_a0 = splat2(-a0), less_a1 = splat2(-a1);
                slot8<T>(at + at_dh, j[c], d);
                // without a norm z has no part in dr: an infinity in it would be a NaN times a1 = 0
                if (back) slot8<T>(at, j[c], h);
                else h[0] = h[1] = h[2] = h[3] = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    h[i] = mul2(FULL ? add2(h[i], less_z) : h[i], rho);
                    sum_c[c][i] = fma2(d[i], h[i], sum_c[c][i]);
                    if constexpr (FULL) sum_d[c][i] = add2(sum_d[c][i], d[i]);
                }
                if (mask & 1) {
                    vec8(v2, j[c], w);
#pragma unroll
                    for (int i = 0; i < 4; ++i) d[i] = mul2(d[i], w[i]);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (FULL) d[i] = add2(d[i], less_a0);
                    dr[i] = fma2(fma2(h[i], less_a1, d[i]), rho, dr[i]);
                    if (!BULK) dr[i] = keep2(dr[i], n - j[c] - 2 * i);
                }
            }
            if (!BULK) store8<T>(slots, at_dz / sizeof(T) + j[c], dr);
            else if (q.dr) store8<T>(q.dr, row * q.lddr + col0 + j[c], dr);
            if (!p.y) continue;
            const f2 rho = splat2(sy.rho);
            slot8<T>(at + at_y, j[c], hat[c]);
#pragma unroll
            for (int i = 0; i < 4; ++i) hat[c][i] = mul2(FULL ? add2(hat[c][i], less_y) : hat[c][i], rho);
            if (mask & 2) {
                vec8(vp, j[c], w);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = splat2(p.scale);
            }
            if constexpr (FULL) if (own_gate) {
                // s u dr is the gate's gradient, and g dr takes the place of dr
                f2 u[4], gate[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) u[i] = mul2(hat[c][i], w[i]);
                if (mask & 4) {
                    vec8(vb, j[c], gate);
#pragma unroll
                    for (int i = 0; i < 4; ++i) u[i] = add2(u[i], gate[i]);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    u[i] = mul2(u[i], dr[i]);
                    sums[2] = add2(sums[2], u[i]);
                }
                if (p.gate_mode == GATE_FULL) {
                    pairs8(own[c], gate);
                    if (!BULK) store8<T>(slots, at_gate / sizeof(T) + j[c], u);
                    else if (q.dgate) store8<T>(q.dgate, row * q.lddg + col0 + j[c], u);
                } else {
                    const f2 one = splat2(static_cast<const float*>(p.gate)[row * p.ldg]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) gate[i] = one;
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) dr[i] = mul2(dr[i], gate[i]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                sum_a[c][i] = fma2(dr[i], hat[c][i], sum_a[c][i]);
                if constexpr (FULL) sum_b[c][i] = add2(sum_b[c][i], dr[i]);
                b[c][i] = mul2(dr[i], w[i]);
                if (FULL) sums[0] = add2(sums[0], b[c][i]);
                sums[1] = fma2(b[c][i], hat[c][i], sums[1]);
            }
        }
        // likewise y, which has no part in dy without a norm
        const bool normed = p.post.kind != RT_NORM_NONE;
        if (!normed)
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) hat[c][i] = 0;
        float b0 = 0.0f, b1 = both(sums[1]);
        if (!p.y) {
            g.sync();
        } else if constexpr (FULL) {
            float v[3] = {both(sums[0]), b1, both(sums[2])};
            g.sum(v);
            b0 = p.post.kind == RT_NORM_LAYER ? -v[0] * inv_n : 0.0f;
            b1 = v[1];
            if (g.t == 0 && g.rank == 0 && q.dgate && p.gate_mode == GATE_COLUMN) static_cast<float*>(q.dgate)[row * q.lddg] = v[2];
        } else {
            g.sum(b1);
        }
        // every thread of the group has read the slot: all of it before the last barrier
        if (BULK && g.t == 0 && ok && row + r.depth * step < p.m) issue(row + r.depth * step, slot);
        if (q.dy) {
            const f2 rho = splat2(sy.rho), add = splat2(b0), less_b1 = splat2(normed ? -b1 * inv_n : 0.0f);
#pragma unroll
            for (int c = 0; c < C; ++c)
                if (has[c]) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (FULL) b[c][i] = add2(b[c][i], add);
                        b[c][i] = mul2(fma2(hat[c][i], less_b1, b[c][i]), rho);
                    }
                    if (BULK) store8<T>(q.dy, row * q.lddy + col0 + j[c], b[c]);
                    else store8<T>(slots, at_y / sizeof(T) + j[c], b[c]);
                }
        }
        if constexpr (!BULK) {
            g.sync();
            if (q.dr) copy_out(q.dr, q.lddr, row, at_dz);
            if (q.dy) copy_out(q.dy, q.lddy, row, at_y);
            if (q.dgate && p.gate_mode == GATE_FULL) copy_out(q.dgate, q.lddg, row, at_gate);
            g.sync();
            continue;
        }
        if (++slot == r.depth) {
            slot = 0;
            phase ^= 1;
        }
    }
    if (BULK && !ok && g.t == 0) land_copies(full, r.depth, r.depth, abort_flag[1 + g.index]);
    if (!q.partials) return;
    __syncthreads();  // the slots are all read
    float* acc = reinterpret_cast<float*>(sm.slots);
    const int groups = (int)min((p.m - part + parts - 1) / parts, (int64_t)G::COUNT);  // that had a row
    join_sums<G>(g, q, acc, groups, p.n, part, col0, 0, sum_a, j, has);
    join_sums<G>(g, q, acc, groups, p.n, part, col0, 2, sum_c, j, has);
    if constexpr (FULL) {
        join_sums<G>(g, q, acc, groups, p.n, part, col0, 1, sum_b, j, has);
        join_sums<G>(g, q, acc, groups, p.n, part, col0, 3, sum_d, j, has);
    }
}

// Backward for the common training step, bf16 rows between two RMS norms with
// dz, dh and y all there: rows overlap, so each costs one barrier.  While row i's
// dr is computed and summed against y^ its successor's three sums are taken, and
// all four are joined at once.  z, y and dh of a row are read into registers when
// its sums are taken and their slots are then free; dz has slots of its own.
// 8192 x 8192: 143 to 156 us, 10 of them column_kernel; the kernel above, whose
// barriers come one after another, took 195.
template <int TPR, int CL>
__global__ void __launch_bounds__(kBackThreads, 1) backward_pipe_kernel(BlockP p, GradP q, RingP r) {
    using T = __nv_bfloat16;
    extern __shared__ __align__(128) uint8_t smem[];
    using G = Group<kBackThreads, TPR, CL>;
    constexpr int C = 2;
    const int width = share_of<CL>(p.n), depth = r.depth;
    const RingSmem sm = ring_smem(smem, r, width, G::COUNT, CL);
    G g;
    g.index = threadIdx.x / TPR;
    g.t = threadIdx.x % TPR;
    g.red = sm.red + g.index * 256;
    g.join_cluster();
    // the CTA's columns: n from col0 on
    const int col0 = CL > 1 ? g.rank * width : 0, n = CL > 1 ? min(width, (int)p.n - col0) : (int)p.n;
    const int part = blockIdx.x / CL;
    // slots: [depth] of z, y, dh, then [depth] of dz; barriers likewise
    uint8_t* slots = sm.slots + (size_t)g.index * depth * r.slot_bytes;
    const uint32_t row_bytes = (uint32_t)n * sizeof(T);
    uint8_t* slots_dz = slots + (size_t)depth * 3 * row_bytes;
    const uint32_t full = tc::smem_u32(sm.full + g.index * 2 * depth), full_dz = full + depth * 8;
    // rows go to the thread blocks in turn, then to their groups: few rows spread over the device
    const int64_t parts = gridDim.x / CL, step = parts * G::COUNT, first = g.index * parts + part;
    volatile int* abort_flag = reinterpret_cast<volatile int*>(sm.full + G::COUNT * 2 * depth);

    if (threadIdx.x == 0) {
        for (int i = 0; i < G::COUNT * 2 * depth; ++i) tc::mbar_init(tc::smem_u32(sm.full + i), 1);
        *abort_flag = 0;
        tc::fence_barrier_init();
    }
    pdl_wait();
    pdl_launch_dependents();
    float *v2 = sm.vec, *vp = v2 + n;
    for (int j = threadIdx.x; j < n; j += kBackThreads) {
        const int at = col0 + j;
        v2[j] = p.pre.gamma ? p.pre.gamma[at] : 1.0f;
        vp[j] = p.scale * shared_gate(p, at) * (p.post.gamma ? p.post.gamma[at] : 1.0f);
    }
    __syncthreads();
    bool ok = true;  // this thread's waits so far
    auto issue = [&](int64_t row, int slot) {
        const uint32_t bar = full + slot * 8, dst = tc::smem_u32(slots + (size_t)slot * 3 * row_bytes);
        tc::mbar_expect_tx(bar, 3 * row_bytes);
        bulk_load(dst, static_cast<const T*>(p.z) + row * p.ldz + col0, row_bytes, bar);
        bulk_load(dst + row_bytes, static_cast<const T*>(p.y) + row * p.ldy + col0, row_bytes, bar);
        bulk_load(dst + 2 * row_bytes, static_cast<const T*>(q.dh) + row * q.lddh + col0, row_bytes, bar);
    };
    auto issue_dz = [&](int64_t row, int slot) {
        const uint32_t bar = full_dz + slot * 8;
        tc::mbar_expect_tx(bar, row_bytes);
        bulk_load(tc::smem_u32(slots_dz + (size_t)slot * row_bytes), static_cast<const T*>(q.dz) + row * q.lddz + col0, row_bytes, bar);
    };
    if (g.t == 0)
        for (int d = 0; d < depth && first + d * step < p.m; ++d) {
            issue(first + d * step, d);
            issue_dz(first + d * step, d);
        }
    // the wait for `slot` of either ring; dz's ring is at most one slot behind
    auto wait = [&](uint32_t ring, int slot, uint32_t phase) {
        if (!tc::mbar_wait(ring + slot * 8, phase, abort_flag)) {
            if (ok) gave_up(r, abort_flag, g.t == 0 ? g.index : -1, slot, phase);
            ok = false;
        }
    };
    const float inv_n = 1.0f / (float)p.n;
    int j[C];
    bool has[C];
    f2 sum_a[C][4], sum_c[C][4];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        j[c] = (c * TPR + g.t) * 8;
        has[c] = j[c] < n;
#pragma unroll
        for (int i = 0; i < 4; ++i) sum_a[c][i] = sum_c[c][i] = 0;
    }
    Raw8<T> rz[C], ry[C], rd[C];
    // z, y and dh of the row in `slot`, and what they add to z^2, gamma_pre dh z, y^2
    auto take = [&](int slot, float (&v)[3]) {
        const uint8_t* at = slots + (size_t)slot * 3 * row_bytes;
        f2 sums[3] = {0, 0, 0};
#pragma unroll
        for (int c = 0; c < C; ++c) {
            if (!has[c]) continue;
            rz[c] = load_raw8<T>(at, j[c]);
            ry[c] = load_raw8<T>(at + row_bytes, j[c]);
            rd[c] = load_raw8<T>(at + 2 * row_bytes, j[c]);
            f2 x[4], d[4], w[4];
            pairs8(rz[c], x);
            pairs8(rd[c], d);
            vec8(v2, j[c], w);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                sums[0] = fma2(x[i], x[i], sums[0]);
                sums[1] = fma2(mul2(d[i], w[i]), x[i], sums[1]);
            }
            pairs8(ry[c], x);
#pragma unroll
            for (int i = 0; i < 4; ++i) sums[2] = fma2(x[i], x[i], sums[2]);
        }
#pragma unroll
        for (int k = 0; k < 3; ++k) v[k] = both(sums[k]);
    };
    float rho_z = 0.0f, rho_y = 0.0f, a1 = 0.0f;
    auto stats = [&](float z2, float az, float y2) {
        rho_z = rsqrtf(z2 * inv_n + p.pre.eps);
        rho_y = rsqrtf(y2 * inv_n + p.post.eps);
        a1 = az * inv_n * rho_z;
    };
    int slot = 0;
    uint32_t phase = 0;
    if (first < p.m) {
        wait(full, 0, 0);
        float v[3];
        take(0, v);
        g.sum(v);
        stats(v[0], v[1], v[2]);
        if (g.t == 0 && ok && first + depth * step < p.m) issue(first + depth * step, 0);
    }
    for (int64_t row = first; row < p.m; row += step) {
        wait(full_dz, slot, phase);
        const uint8_t* at = slots_dz + (size_t)slot * row_bytes;
        f2 b[C][4], hat[C][4];
        f2 sum_b = 0;
        const f2 rz2 = splat2(rho_z), ry2 = splat2(rho_y), less_a1 = splat2(-a1);
#pragma unroll
        for (int c = 0; c < C; ++c) {
            if (!has[c]) continue;
            f2 dr[4], d[4], h[4], w[4];
            slot8<T>(at, j[c], dr);
            pairs8(rd[c], d);
            pairs8(rz[c], h);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                h[i] = mul2(h[i], rz2);
                sum_c[c][i] = fma2(d[i], h[i], sum_c[c][i]);
            }
            vec8(v2, j[c], w);
#pragma unroll
            for (int i = 0; i < 4; ++i) dr[i] = fma2(fma2(h[i], less_a1, mul2(d[i], w[i])), rz2, dr[i]);
            if (q.dr) store8<T>(q.dr, row * q.lddr + col0 + j[c], dr);
            pairs8(ry[c], hat[c]);
            vec8(vp, j[c], w);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                hat[c][i] = mul2(hat[c][i], ry2);
                sum_a[c][i] = fma2(dr[i], hat[c][i], sum_a[c][i]);
                b[c][i] = mul2(dr[i], w[i]);
                sum_b = fma2(b[c][i], hat[c][i], sum_b);
            }
        }
        const int next = slot + 1 == depth ? 0 : slot + 1;
        const uint32_t next_phase = next ? phase : phase ^ 1;
        const bool more = row + step < p.m;
        float t[3] = {0.0f, 0.0f, 0.0f};
        if (more) {
            wait(full, next, next_phase);
            take(next, t);
        }
        float v[4] = {t[0], t[1], t[2], both(sum_b)};
        g.sum(v);
        if (g.t == 0 && ok) {
            if (row + depth * step < p.m) issue_dz(row + depth * step, slot);
            if (row + (depth + 1) * step < p.m) issue(row + (depth + 1) * step, next);
        }
        if (q.dy) {
            const f2 less_b1 = splat2(-v[3] * inv_n);
#pragma unroll
            for (int c = 0; c < C; ++c)
                if (has[c]) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) b[c][i] = mul2(fma2(hat[c][i], less_b1, b[c][i]), ry2);
                    store8<T>(q.dy, row * q.lddy + col0 + j[c], b[c]);
                }
        }
        stats(v[0], v[1], v[2]);
        slot = next;
        phase = next_phase;
    }
    if (!ok && g.t == 0) {
        // a wait for dz that gave up: z's ring is one use further, its slot already filled again
        land_copies(full, depth, depth + 1, abort_flag[1 + g.index]);
        land_copies(full_dz, depth, depth, abort_flag[1 + g.index]);
    }
    if (!q.partials) return;
    __syncthreads();  // the slots are all read
    float* acc = reinterpret_cast<float*>(sm.slots);
    const int groups = (int)min((p.m - part + parts - 1) / parts, (int64_t)G::COUNT);  // that had a row
    join_sums<G>(g, q, acc, groups, p.n, part, col0, 0, sum_a, j, has);
    join_sums<G>(g, q, acc, groups, p.n, part, col0, 2, sum_c, j, has);
}

struct ReduceP {
    const float* partials;
    int parts, sums;
    int64_t n;
    int gate_mode;
    const float* gate;
    float scale;
    const float *gamma, *beta;  // of the norm after the block
    float *dgamma_post, *dbeta_post, *dgamma_pre, *dbeta_pre, *dgate;
    float* gate_row;  // [n]: a [1,1] gate's gradient by column
};

// Column sums of the partials and the vectors they give.  All latency: a CTA takes
// COLS columns, Q = 32 / COLS lanes of each of its warps every (Q WARPS)th part, all
// reads under way together; the lanes' and then the warps' sums are added in order.
// Eight columns (a sector) up to 4096 wide: 148 parts of 1000 columns 3 us behind the
// kernel before it, where 32 columns and reads one after another took 10.  Wider, 32
// columns keep the CTAs to one wave.
template <int COLS>
__global__ void __launch_bounds__(COLS * 16 + 512) column_kernel(ReduceP p) {
    constexpr int WARPS = COLS / 2 + 16, Q = 32 / COLS, STEP = WARPS * Q, U = 160 / STEP;
    __shared__ float sums[WARPS][4 * COLS];
    __shared__ float totals[4 * COLS];
    pdl_wait();
    pdl_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, column = lane % COLS;
    const int64_t j = (int64_t)blockIdx.x * COLS + column, stride = columns(p.n);
    float s[4] = {};
    for (int i0 = warp * Q + lane / COLS; i0 < p.parts; i0 += U * STEP) {
        float x[U][4];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int v = 0; v < 4; ++v)
                x[u][v] = j < p.n && i0 + u * STEP < p.parts && ((p.sums >> v) & 1)
                              ? p.partials[((int64_t)(i0 + u * STEP) * 4 + v) * stride + j]
                              : 0.0f;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int v = 0; v < 4; ++v) s[v] += x[u][v];
    }
#pragma unroll
    for (int v = 0; v < 4; ++v) {
#pragma unroll
        for (int o = COLS; o < 32; o *= 2) s[v] += __shfl_xor_sync(0xffffffffu, s[v], o);
        if (lane < COLS) sums[warp][v * COLS + column] = s[v];
    }
    __syncthreads();
    if (threadIdx.x < 4 * COLS) {
        float total = 0.0f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) total += sums[w][threadIdx.x];
        totals[threadIdx.x] = total;
    }
    __syncthreads();
    if (threadIdx.x >= COLS || j >= p.n) return;
#pragma unroll
    for (int v = 0; v < 4; ++v) s[v] = totals[v * COLS + column];
    s[0] *= p.scale;
    s[1] *= p.scale;
    const float g = p.gate_mode == GATE_ONE ? p.gate[0] : p.gate_mode == GATE_ROW ? p.gate[j] : 1.0f;
    if (p.dgamma_post) p.dgamma_post[j] = s[0] * g;
    if (p.dbeta_post) p.dbeta_post[j] = s[1] * g;
    if (p.dgamma_pre) p.dgamma_pre[j] = s[2];
    if (p.dbeta_pre) p.dbeta_pre[j] = s[3];
    const float dg = (p.gamma ? p.gamma[j] : 1.0f) * s[0] + (p.beta ? p.beta[j] * s[1] : 0.0f);
    if (p.gate_row) p.gate_row[j] = dg;
    else if (p.dgate) p.dgate[j] = dg;
}

__global__ void __launch_bounds__(kWide) gate_one_kernel(const float* row, int64_t n, float* out) {
    __shared__ float red[32];
    pdl_wait();
    pdl_launch_dependents();
    float s = 0.0f;
    for (int64_t j = threadIdx.x; j < n; j += kWide) s += row[j];
    s = wide_sum(s, red);
    if (threadIdx.x == 0) out[0] = s;
}

// --------------------------------------------------------------- host side
int check_ctx(const rt_ctx* ctx, std::initializer_list<const rt_tensor*> ts) {
    for (const rt_tensor* t : ts) RT_CHECK(!t || t->ctx == ctx, "tensor belongs to another context");
    return RT_OK;
}

int check_like(const char* what, const rt_tensor* t, const rt_tensor* r) {
    RT_CHECK(t->dtype == r->dtype, "%s must have r's type", what);
    RT_CHECK(t->rows == r->rows && t->cols == r->cols, "%s is %lldx%lld, not %lldx%lld", what, (long long)t->rows,
             (long long)t->cols, (long long)r->rows, (long long)r->cols);
    return RT_OK;
}

int check_vector(const char* what, const rt_tensor* t, int64_t n) {
    RT_CHECK(t->dtype == RT_F32, "%s must be f32", what);
    RT_CHECK(t->rows == 1 && t->cols == n, "%s is %lldx%lld, not 1x%lld", what, (long long)t->rows, (long long)t->cols,
             (long long)n);
    return RT_OK;
}

int check_norm(const char* what, const rt_norm& p, int64_t n, NormP* out) {
    RT_CHECK(p.kind == RT_NORM_NONE || p.kind == RT_NORM_RMS || p.kind == RT_NORM_LAYER, "%s: unknown norm %d", what,
             (int)p.kind);
    RT_CHECK(p.kind != RT_NORM_NONE || (!p.gamma && !p.beta), "%s: no norm, but gamma or beta", what);
    RT_CHECK(p.kind == RT_NORM_NONE || p.eps >= 0.0f, "%s: eps must be >= 0", what);
    if (p.gamma) RT_TRY(check_vector("gamma", p.gamma, n));
    if (p.beta) RT_TRY(check_vector("beta", p.beta, n));
    *out = NormP{(int)p.kind, p.eps, p.gamma ? static_cast<const float*>(p.gamma->ptr) : nullptr,
                 p.beta ? static_cast<const float*>(p.beta->ptr) : nullptr};
    return RT_OK;
}

// The gate's form from its shape: [1,1], then the full one where the type says
// so, [1,n], [m,1].
int check_gate(const char* what, const rt_tensor* t, const rt_tensor* r, int* mode) {
    if (t->rows == r->rows && t->cols == r->cols && t->dtype == r->dtype && !(t->rows == 1 && t->dtype == RT_F32) &&
        !(t->cols == 1 && t->dtype == RT_F32)) {
        *mode = GATE_FULL;
        return RT_OK;
    }
    RT_CHECK(t->dtype == RT_F32, "%s: a broadcast gate must be f32, a full one of y's type and shape", what);
    if (t->rows == 1 && t->cols == 1)
        *mode = GATE_ONE;
    else if (t->rows == 1 && t->cols == r->cols)
        *mode = GATE_ROW;
    else if (t->rows == r->rows && t->cols == 1)
        *mode = GATE_COLUMN;
    else
        return fail(RT_ERR_INVALID, "%s is %lldx%lld: it must be 1x1, 1x%lld, %lldx1 or %lldx%lld", what,
                    (long long)t->rows, (long long)t->cols, (long long)r->cols, (long long)r->rows, (long long)r->rows,
                    (long long)r->cols);
    return RT_OK;
}

// What forward and backward share; `r` is the tensor that gives shape and type.
int block_params(const rt_block_args* a, const rt_tensor* r, BlockP* p) {
    RT_CHECK(r->dtype == RT_F32 || r->dtype == RT_BF16, "the residual stream must be f32 or bf16");
    p->m = r->rows;
    p->n = r->cols;
    if (a->y) {
        RT_TRY(check_like("y", a->y, r));
        p->y = a->y->ptr;
        p->ldy = a->y->ld;
    } else {
        RT_CHECK(a->post.kind == RT_NORM_NONE && !a->gate, "a norm after the block or a gate, but no y");
    }
    RT_TRY(check_norm("post", a->post, p->n, &p->post));
    RT_TRY(check_norm("pre", a->pre, p->n, &p->pre));
    p->scale = a->scale;
    p->gate_mode = GATE_NONE;
    if (a->gate) {
        RT_TRY(check_gate("gate", a->gate, r, &p->gate_mode));
        p->gate = a->gate->ptr;
        p->ldg = a->gate->ld;
    }
    return RT_OK;
}

bool aligned16(const void* p, int64_t ld, size_t es) {
    return ((reinterpret_cast<uintptr_t>(p) | (uintptr_t)(ld * (int64_t)es)) & 15) == 0;
}

// Whether the kernels that hold rows in registers apply: whole eights of 16-byte
// aligned rows, and 16-byte aligned vectors.
bool rows_aligned(const BlockP& p, size_t es) {
    return p.n % 8 == 0 && aligned16(p.r, p.ldr, es) && aligned16(p.y, p.ldy, es) && aligned16(p.z, p.ldz, es) &&
           aligned16(p.h, p.ldh, es) && aligned16(p.post.gamma, 0, 4) && aligned16(p.post.beta, 0, 4) &&
           aligned16(p.pre.gamma, 0, 4) && aligned16(p.pre.beta, 0, 4) &&
           (p.gate_mode == GATE_FULL ? aligned16(p.gate, p.ldg, es) : p.gate_mode != GATE_ROW || aligned16(p.gate, 0, 4));
}

template <typename T, int TPR, int C = 1>
cudaError_t launch_forward_rows(bool pdl, const BlockP& p, cudaStream_t st) {
    constexpr int threads = cta_threads(TPR), rows = threads / TPR;
    return launch_k(pdl, forward_rows_kernel<T, TPR, C>, (unsigned)((p.m + rows - 1) / rows), threads, 0, st, p);
}

// Fills in the ring's shape, of at most `most` slots a group; false where not even
// one fits.
bool plan_ring(RingP* r, int64_t n, int groups, int tensors, size_t es, int vectors, int most = 4, int cluster = 1) {
    r->slot_bytes = (int)(tensors * n * (int64_t)es);
    r->vectors = vectors;
    const int64_t room = kRingSmem - ring_scratch(groups, cluster) - (int64_t)vectors * n * 4;
    r->depth = (int)std::min<int64_t>(most, room / ((int64_t)groups * r->slot_bytes));
    r->smem = (int)(kRingSmem - room) + groups * r->depth * r->slot_bytes;
    return r->depth >= 1;
}

template <typename T, int TPR, int C>
int launch_forward_ring(rt_ctx* ctx, const BlockP& p, RingP r, int mask, cudaStream_t st) {
    constexpr int groups = kRingThreads / TPR;
    const int64_t ctas = std::min<int64_t>(ctx->sm_count, (p.m + groups - 1) / groups);
    const bool full = p.post.kind == RT_NORM_LAYER || p.pre.kind == RT_NORM_LAYER || (mask & 10) ||
                      p.gate_mode == GATE_COLUMN || p.gate_mode == GATE_FULL;
    auto* kernel = full ? forward_ring_kernel<T, TPR, C, true> : forward_ring_kernel<T, TPR, C, false>;
    RT_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingSmem));
    RT_CUDA(launch_k(ctx->pdl, kernel, (unsigned)ctas, kRingThreads, r.smem, st, p, r, mask));
    return RT_OK;
}

// The ring's kernel where there are rows enough for it: true if it was launched.
template <typename T>
int forward_ring(rt_ctx* ctx, const BlockP& p, cudaStream_t st, bool* done) {
    *done = false;
    if (!rows_aligned(p, sizeof(T)) || p.n > 8192) return RT_OK;
    const bool shared = p.gate_mode == GATE_ONE || p.gate_mode == GATE_ROW;
    const int mask = (p.y && (p.post.gamma || shared) ? 1 : 0) | (p.post.beta ? 2 : 0) | (p.pre.gamma ? 4 : 0) |
                     (p.pre.beta ? 8 : 0);
    const int tpr = p.n <= 512 ? 32 : p.n <= 2048 ? 128 : p.n <= 4096 ? 256 : 512;
    if (p.m < (int64_t)2 * ctx->sm_count * (kRingThreads / tpr)) return RT_OK;
    RingP r{};
    r.err = ctx->dev_err;
    if (!plan_ring(&r, p.n, kRingThreads / tpr, p.y ? 2 : 1, sizeof(T), __builtin_popcount(mask))) return RT_OK;
    *done = true;
    if (tpr == 32) return launch_forward_ring<T, 32, 2>(ctx, p, r, mask, st);
    if (tpr == 128) return launch_forward_ring<T, 128, 2>(ctx, p, r, mask, st);
    if (tpr == 256) return launch_forward_ring<T, 256, 2>(ctx, p, r, mask, st);
    return launch_forward_ring<T, 512, 2>(ctx, p, r, mask, st);
}

template <typename T, int TPR, int C, bool FULL, bool BULK, int CL = 1>
int launch_backward_ring(rt_ctx* ctx, const BlockP& p, const GradP& q, const RingP& r, int mask, int parts, cudaStream_t st) {
    auto* kernel = backward_ring_kernel<T, TPR, C, FULL, BULK, CL>;
    RT_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingSmem));
    RT_CUDA(launch_cluster(CL, ctx->pdl, kernel, (unsigned)(parts * CL), kBackThreads, r.smem, st, p, q, r, mask));
    return RT_OK;
}

template <int TPR, int CL = 1>
int launch_backward_pipe(bool pdl, const BlockP& p, const GradP& q, const RingP& r, int parts, cudaStream_t st) {
    auto* kernel = backward_pipe_kernel<TPR, CL>;
    RT_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingSmem));
    RT_CUDA(launch_cluster(CL, pdl, kernel, (unsigned)(parts * CL), kBackThreads, r.smem, st, p, q, r));
    return RT_OK;
}

template <typename T, bool BULK>
int launch_backward_full(rt_ctx* ctx, const BlockP& p, const GradP& q, const RingP& r, int mask, int tpr, int cluster, int parts,
                         cudaStream_t st) {
    if (cluster == 4) return launch_backward_ring<T, 512, 1, true, BULK, 4>(ctx, p, q, r, mask, parts, st);
    if (cluster == 2) return launch_backward_ring<T, 512, 1, true, BULK, 2>(ctx, p, q, r, mask, parts, st);
    switch (tpr) {
        case 32: return launch_backward_ring<T, 32, 1, true, BULK>(ctx, p, q, r, mask, parts, st);
        case 64: return launch_backward_ring<T, 64, 1, true, BULK>(ctx, p, q, r, mask, parts, st);
        case 128: return launch_backward_ring<T, 128, 1, true, BULK>(ctx, p, q, r, mask, parts, st);
        case 256: return launch_backward_ring<T, 256, 1, true, BULK>(ctx, p, q, r, mask, parts, st);
        default: return launch_backward_ring<T, 512, 1, true, BULK>(ctx, p, q, r, mask, parts, st);
    }
}

// Rings that take a row by four CTAs: how many such clusters the device runs at once
// (what it is divided into decides that, so it is asked, once).
int ring_clusters(rt_ctx* ctx, int cluster, int* count) {
    *count = ctx->sm_count / cluster;
    if (cluster <= 2) return RT_OK;
    if (ctx->ring_clusters4 == 0) {
        auto* kernel = backward_ring_kernel<float, kBackThreads, 1, true, true, 4>;
        RT_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingSmem));
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = 4 * *count;
        cfg.blockDim = kBackThreads;
        cfg.dynamicSmemBytes = kRingSmem;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim = {4, 1, 1};
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        RT_CUDA(cudaOccupancyMaxActiveClusters(&ctx->ring_clusters4, kernel, &cfg));
        RT_CHECK(ctx->ring_clusters4 > 0, "no cluster of four thread blocks fits the device");
    }
    *count = std::min(*count, ctx->ring_clusters4);
    return RT_OK;
}

// The backward pass through the ring, up to 16384 wide.  *parts is then the number of
// partials.  A CTA takes 8192 columns, 4096 with all features (which want registers):
// wider rows are shared by a cluster.  1000 x 16384 bf16 RMS 61 to 69 us so, layer norms with
// a full gate 164 to 173, against 301 and 416 by the kernel for any width; 4096 x 4099 with
// all features 403 to 423 against 540 by one CTA whose threads spill.  Unaligned rows up to
// 4096 wide take the full kernel without its features: eight columns a thread, 4000 x
// 1001 bf16 RMS 32 to 37 us.
template <typename T>
int backward_ring(rt_ctx* ctx, const BlockP& p, const GradP& q, cudaStream_t st, int* parts, bool* done) {
    *done = false;
    const size_t es = sizeof(T);
    if (p.n > 16384 || p.m == 0 || !aligned16(q.partials, 0, 4)) return RT_OK;
    const bool bulk = rows_aligned(p, es) && aligned16(q.dz, q.lddz, es) && aligned16(q.dh, q.lddh, es) &&
                      aligned16(q.dr, q.lddr, es) && aligned16(q.dy, q.lddy, es) &&
                      (p.gate_mode != GATE_FULL || aligned16(q.dgate, q.lddg, es));
    const bool shared = p.gate_mode == GATE_ONE || p.gate_mode == GATE_ROW;
    const int mask = (p.pre.gamma ? 1 : 0) | (p.post.gamma || (p.y && shared) ? 2 : 0) |
                     (p.post.beta && q.dgate && !shared ? 4 : 0);
    const bool full = (!bulk && p.n <= 4096) || p.post.kind == RT_NORM_LAYER || p.pre.kind == RT_NORM_LAYER || (q.sums & 10) ||
                      p.gate_mode == GATE_COLUMN || p.gate_mode == GATE_FULL;
    const int eights = full ? 1 : 2;
    int tpr = 32, cluster = 1;
    while (tpr < kBackThreads && tpr * eights * 8 < p.n) tpr *= 2;
    while (cluster * tpr * eights * 8 < p.n) cluster *= 2;
    const int groups = kBackThreads / tpr;
    const int64_t width = columns((p.n + cluster - 1) / cluster);
    RingP r{};
    r.err = ctx->dev_err;
    const int tensors = bulk ? 1 + (p.y ? 1 : 0) + (q.dz ? 1 : 0) + (q.dh ? 1 : 0) : p.gate_mode == GATE_FULL ? 5 : 4;
    if (!plan_ring(&r, width, groups, tensors, es, __builtin_popcount(mask), bulk ? 4 : 1, cluster)) return RT_OK;
    *done = true;
    int clusters = 0;
    RT_TRY(ring_clusters(ctx, cluster, &clusters));
    *parts = (int)std::min<int64_t>(clusters, p.m);
    if constexpr (sizeof(T) == 2) {
        RingP two{};
        two.err = ctx->dev_err;
        if (bulk && !full && p.post.kind == RT_NORM_RMS && p.pre.kind == RT_NORM_RMS && q.dz && q.dh &&
            plan_ring(&two, width, groups, 4, es, 2, 4, cluster) && two.depth >= 2) {
            if (cluster == 2) return launch_backward_pipe<512, 2>(ctx->pdl, p, q, two, *parts, st);
            switch (tpr) {
                case 32: return launch_backward_pipe<32>(ctx->pdl, p, q, two, *parts, st);
                case 64: return launch_backward_pipe<64>(ctx->pdl, p, q, two, *parts, st);
                case 128: return launch_backward_pipe<128>(ctx->pdl, p, q, two, *parts, st);
                case 256: return launch_backward_pipe<256>(ctx->pdl, p, q, two, *parts, st);
                default: return launch_backward_pipe<512>(ctx->pdl, p, q, two, *parts, st);
            }
        }
    }
    if (!full && !bulk)
        return cluster == 2 ? launch_backward_ring<T, 512, 2, false, false, 2>(ctx, p, q, r, mask, *parts, st)
                            : launch_backward_ring<T, 512, 2, false, false>(ctx, p, q, r, mask, *parts, st);
    if (!full) {
        if (cluster == 2) return launch_backward_ring<T, 512, 2, false, true, 2>(ctx, p, q, r, mask, *parts, st);
        switch (tpr) {
            case 32: return launch_backward_ring<T, 32, 2, false, true>(ctx, p, q, r, mask, *parts, st);
            case 64: return launch_backward_ring<T, 64, 2, false, true>(ctx, p, q, r, mask, *parts, st);
            case 128: return launch_backward_ring<T, 128, 2, false, true>(ctx, p, q, r, mask, *parts, st);
            case 256: return launch_backward_ring<T, 256, 2, false, true>(ctx, p, q, r, mask, *parts, st);
            default: return launch_backward_ring<T, 512, 2, false, true>(ctx, p, q, r, mask, *parts, st);
        }
    }
    return bulk ? launch_backward_full<T, true>(ctx, p, q, r, mask, tpr, cluster, *parts, st)
                : launch_backward_full<T, false>(ctx, p, q, r, mask, tpr, cluster, *parts, st);
}

// Up to 16384 wide: the fewest threads that hold a row eight elements each (the
// widest rows, sixteen).
template <typename T>
int forward_rows(rt_ctx* ctx, const BlockP& p, cudaStream_t st, bool* done) {
    *done = false;
    if (!rows_aligned(p, sizeof(T)) || p.n > 16384 || p.m > INT32_MAX) return RT_OK;
    *done = true;
    const bool pdl = ctx->pdl;
    RT_CUDA(p.n <= 256    ? (launch_forward_rows<T, 32>(pdl, p, st))
            : p.n <= 512  ? (launch_forward_rows<T, 64>(pdl, p, st))
            : p.n <= 1024 ? (launch_forward_rows<T, 128>(pdl, p, st))
            : p.n <= 2048 ? (launch_forward_rows<T, 256>(pdl, p, st))
            : p.n <= 4096 ? (launch_forward_rows<T, 512>(pdl, p, st))
            : p.n <= 8192 ? (launch_forward_rows<T, 1024>(pdl, p, st))
                          : (launch_forward_rows<T, 1024, 2>(pdl, p, st)));
    return RT_OK;
}

template <typename T>
int forward_strided(rt_ctx* ctx, const BlockP& p, cudaStream_t st, bool* done) {
    *done = false;
    if (p.n > 16384 || p.m > INT32_MAX) return RT_OK;
    *done = true;
    if (p.n <= 256) {
        RT_CUDA(launch_k(ctx->pdl, forward_strided_kernel<T, true, 8>, (unsigned)((p.m + 3) / 4), 128, 0, st, p));
    } else if (p.n <= 8192) {
        RT_CUDA(launch_k(ctx->pdl, forward_strided_kernel<T, false, 8>, (unsigned)p.m, (unsigned)((p.n + 255) / 256 * 32), 0, st, p));
    } else {
        RT_CUDA(launch_k(ctx->pdl, forward_strided_kernel<T, false, 16>, (unsigned)p.m, (unsigned)((p.n + 511) / 512 * 32), 0, st, p));
    }
    return RT_OK;
}

// The forward pass on the kernel that fits it.
template <typename T>
int forward_any(rt_ctx* ctx, const BlockP& p, cudaStream_t st) {
    bool done = false;
    RT_TRY(forward_ring<T>(ctx, p, st, &done));
    if (!done) RT_TRY(forward_rows<T>(ctx, p, st, &done));
    if (!done) RT_TRY(forward_strided<T>(ctx, p, st, &done));
    if (!done)
        RT_CUDA(launch_k(ctx->pdl, forward_kernel<T>, (unsigned)std::min<int64_t>(p.m, (int64_t)ctx->sm_count * 8), kWide, 0,
                         st, p));
    count_launch(ctx);
    return RT_OK;
}

int parts_for(const rt_ctx* ctx, int64_t m) { return (int)std::max<int64_t>(1, std::min<int64_t>(m, ctx->sm_count)); }

}  // namespace
}  // namespace rt

using namespace rt;

extern "C" {

int rt_block_forward(rt_ctx* ctx, const rt_block_args* a) {
    RT_CHECK(ctx && a && a->r, "rt_block_forward: bad arguments");
    RT_TRY(check_ctx(ctx, {a->r, a->y, a->gate, a->z, a->h, a->post.gamma, a->post.beta, a->pre.gamma, a->pre.beta}));
    RT_CHECK(!a->hq || a->hq->ctx == ctx, "tensor belongs to another context");
    BlockP p{};
    RT_TRY(block_params(a, a->r, &p));
    p.r = a->r->ptr;
    p.ldr = a->r->ld;
    RT_CHECK(a->z || a->h || a->hq, "rt_block_forward: no output");
    if (a->z) {
        RT_TRY(check_like("z", a->z, a->r));
        p.z = a->z->ptr;
        p.ldz = a->z->ld;
    }
    if (a->h) {
        RT_TRY(check_like("h", a->h, a->r));
        p.h = a->h->ptr;
        p.ldh = a->h->ld;
    }
    if (a->hq) {
        RT_CHECK(a->hq->rows == p.m && a->hq->k == p.n, "hq is %lldx%lld, not %lldx%lld", (long long)a->hq->rows,
                 (long long)a->hq->k, (long long)p.m, (long long)p.n);
        p.codes = a->hq->codes;
        p.scales = a->hq->scales;
    }
    if (p.m == 0 || p.n == 0) return RT_OK;
    RT_CUDA(cudaSetDevice(ctx->device));
    return a->r->dtype == RT_BF16 ? forward_any<__nv_bfloat16>(ctx, p, ctx->stream) : forward_any<float>(ctx, p, ctx->stream);
}

int64_t rt_block_backward_workspace(rt_ctx* ctx, int64_t m, int64_t n) {
    if (!ctx || m < 0 || n < 0) {
        set_error("rt_block_backward_workspace: bad arguments");
        return -1;
    }
    return ((int64_t)parts_for(ctx, m) * 4 + 1) * columns(n);
}

int rt_block_backward(rt_ctx* ctx, const rt_block_args* a, const rt_block_grads* g) {
    RT_CHECK(ctx && a && g, "rt_block_backward: bad arguments");
    RT_TRY(check_ctx(ctx, {a->r, a->y, a->gate, a->z, a->post.gamma, a->post.beta, a->pre.gamma, a->pre.beta, g->dz, g->dh,
                           g->dr, g->dy, g->dgamma_post, g->dbeta_post, g->dgamma_pre, g->dbeta_pre, g->dgate, g->work}));
    const rt_tensor* z = a->z ? a->z : a->r;
    RT_CHECK(z && (a->z || !a->y), "rt_block_backward: z is needed where there is a y");
    BlockP p{};
    RT_TRY(block_params(a, z, &p));
    p.z = const_cast<void*>(static_cast<const void*>(z->ptr));
    p.ldz = z->ld;
    GradP q{};
    RT_CHECK(g->dz || g->dh, "rt_block_backward: neither dz nor dh");
    const struct {
        const char* name;
        const rt_tensor* t;
        const void** ptr;
        int64_t* ld;
    } full[] = {{"dz", g->dz, &q.dz, &q.lddz},
                {"dh", g->dh, &q.dh, &q.lddh},
                {"dr", g->dr, const_cast<const void**>(&q.dr), &q.lddr},
                {"dy", g->dy, const_cast<const void**>(&q.dy), &q.lddy}};
    for (const auto& f : full)
        if (f.t) {
            RT_TRY(check_like(f.name, f.t, z));
            *f.ptr = f.t->ptr;
            *f.ld = f.t->ld;
        }
    RT_CHECK(a->y || (!g->dy && !g->dgamma_post && !g->dbeta_post && !g->dgate), "gradients of a block that has no y");
    RT_CHECK((a->post.kind != RT_NORM_NONE || (!g->dgamma_post && !g->dbeta_post)) &&
                 (a->pre.kind != RT_NORM_NONE || (!g->dgamma_pre && !g->dbeta_pre)),
             "dgamma or dbeta of a norm that is not there");
    RT_CHECK(g->dh || (!g->dgamma_pre && !g->dbeta_pre), "dgamma_pre or dbeta_pre without dh");
    ReduceP c{};
    const struct {
        const char* name;
        const rt_tensor* t;
        float** ptr;
    } vec[] = {{"dgamma_post", g->dgamma_post, &c.dgamma_post},
               {"dbeta_post", g->dbeta_post, &c.dbeta_post},
               {"dgamma_pre", g->dgamma_pre, &c.dgamma_pre},
               {"dbeta_pre", g->dbeta_pre, &c.dbeta_pre}};
    for (const auto& v : vec)
        if (v.t) {
            RT_TRY(check_vector(v.name, v.t, p.n));
            *v.ptr = static_cast<float*>(v.t->ptr);
        }
    bool gate_sums = false;
    if (g->dgate) {
        RT_CHECK(a->gate, "dgate without a gate");
        RT_CHECK(g->dgate->dtype == a->gate->dtype && g->dgate->rows == a->gate->rows &&
                     g->dgate->cols == a->gate->cols,
                 "dgate must have the gate's type and shape");
        if (p.gate_mode == GATE_COLUMN || p.gate_mode == GATE_FULL) {
            q.dgate = g->dgate->ptr;
            q.lddg = g->dgate->ld;
        } else {
            gate_sums = true;
            c.dgate = static_cast<float*>(g->dgate->ptr);
        }
    }
    q.sums = (g->dgamma_post || gate_sums ? 1 : 0) | (g->dbeta_post || (gate_sums && p.post.beta) ? 2 : 0) |
             (g->dgamma_pre ? 4 : 0) | (g->dbeta_pre ? 8 : 0);
    if (p.n == 0) {  // sums over no columns
        if (g->dgate && p.m > 0 && (p.gate_mode == GATE_ONE || p.gate_mode == GATE_COLUMN)) {
            RT_CUDA(cudaSetDevice(ctx->device));
            RT_CUDA(cudaMemset2DAsync(g->dgate->ptr, (size_t)g->dgate->ld * 4, 0, 4, (size_t)g->dgate->rows, ctx->stream));
        }
        return RT_OK;
    }
    int parts = parts_for(ctx, p.m);
    if (q.sums) {
        RT_CHECK(g->work && g->work->dtype == RT_F32 && g->work->rows == 1 &&
                     g->work->cols >= rt_block_backward_workspace(ctx, p.m, p.n),
                 "rt_block_backward: work must be %lld f32 in one row",
                 (long long)rt_block_backward_workspace(ctx, p.m, p.n));
        q.partials = static_cast<float*>(g->work->ptr);
    }
    RT_CUDA(cudaSetDevice(ctx->device));
    bool done = false;
    RT_TRY(z->dtype == RT_BF16 ? backward_ring<__nv_bfloat16>(ctx, p, q, ctx->stream, &parts, &done)
                               : backward_ring<float>(ctx, p, q, ctx->stream, &parts, &done));
    // wider rows; and without rows the sums over rows are zero: the partials of one CTA
    if (!done)
        RT_CUDA(launch_k(ctx->pdl, z->dtype == RT_BF16 ? backward_kernel<__nv_bfloat16> : backward_kernel<float>, parts, kWide, 0,
                         ctx->stream, p, q));
    count_launch(ctx);
    if (!q.sums) return RT_OK;
    c.partials = q.partials;
    c.parts = parts;
    c.sums = q.sums;
    c.n = p.n;
    c.gate_mode = p.gate_mode;
    c.gate = static_cast<const float*>(p.gate);
    c.scale = p.scale;
    c.gamma = p.post.gamma;
    c.beta = p.post.beta;
    if (gate_sums && p.gate_mode == GATE_ONE) c.gate_row = q.partials + (int64_t)parts_for(ctx, p.m) * 4 * columns(p.n);
    if (p.n <= 4096) {
        RT_CUDA(launch_k(ctx->pdl, column_kernel<8>, (unsigned)((p.n + 7) / 8), 640, 0, ctx->stream, c));
    } else {
        RT_CUDA(launch_k(ctx->pdl, column_kernel<32>, (unsigned)((p.n + 31) / 32), 1024, 0, ctx->stream, c));
    }
    count_launch(ctx);
    if (c.gate_row) {
        RT_CUDA(launch_k(ctx->pdl, gate_one_kernel, 1, kWide, 0, ctx->stream, c.gate_row, p.n, c.dgate));
        count_launch(ctx);
    }
    return RT_OK;
}

}  // extern "C"
