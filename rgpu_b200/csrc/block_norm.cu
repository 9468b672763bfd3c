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
// and, with w = s dr (times g where the gate differs from row to row), the sums
// over rows A = sum w y^ and B = sum w give every other vector:
//   dgamma_post = g A,  dbeta_post = g B,  dgate = gamma_post A + beta_post B
// (g = 1 where w holds it; the [1,1] gate's gradient sums dgate over columns).
#include <algorithm>

#include "mx4.cuh"

namespace rt {
namespace {

enum GateMode : int { GATE_NONE = 0, GATE_ONE = 1, GATE_ROW = 2, GATE_COLUMN = 3, GATE_FULL = 4 };

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
    float* partials;   // [parts][4][n]: A, B, sum dh z^, sum dh of each CTA's rows
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

// Sum over the 256 threads of a block, to every thread, in a fixed order.
__device__ __forceinline__ float block_sum(float v, float* red) {
    v = warp_sum(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += red[i];
    return s;
}

struct Stat {
    float mu, rho;
};

// Mean (layer) and reciprocal deviation of a row, x(j) its elements.
template <typename F>
__device__ __forceinline__ Stat row_stat(const NormP& p, int64_t n, float* red, F x) {
    Stat s{0.0f, 1.0f};
    if (p.kind == RT_NORM_NONE) return s;
    if (p.kind == RT_NORM_LAYER) {
        float t = 0.0f;
        for (int64_t j = threadIdx.x; j < n; j += 256) t += x(j);
        s.mu = block_sum(t, red) / (float)n;
    }
    float t = 0.0f;
    for (int64_t j = threadIdx.x; j < n; j += 256) {
        const float d = x(j) - s.mu;
        t += d * d;
    }
    s.rho = 1.0f / sqrtf(block_sum(t, red) / (float)n + p.eps);
    return s;
}

__device__ __forceinline__ float gamma_at(const NormP& p, int64_t j) { return p.gamma ? p.gamma[j] : 1.0f; }
__device__ __forceinline__ float beta_at(const NormP& p, int64_t j) { return p.beta ? p.beta[j] : 0.0f; }

template <typename T>
__device__ __forceinline__ float gate_at(const BlockP& p, int64_t row, int64_t j) {
    switch (p.gate_mode) {
        case GATE_ONE: return static_cast<const float*>(p.gate)[0];
        case GATE_ROW: return static_cast<const float*>(p.gate)[j];
        case GATE_COLUMN: return static_cast<const float*>(p.gate)[row * p.ldg];
        case GATE_FULL: return ld<T>(p.gate, row * p.ldg + j);
        default: return 1.0f;
    }
}

// One CTA per row at a time, any width: the row is read once per pass.
template <typename T>
__global__ void __launch_bounds__(256) forward_kernel(BlockP p) {
    __shared__ float red[8];
    const int64_t n = p.n, blocks = (n + 31) / 32, groups = (blocks + 3) / 4;
    for (int64_t row = blockIdx.x; row < p.m; row += gridDim.x) {
        Stat sy{0.0f, 1.0f};
        if (p.y) sy = row_stat(p.post, n, red, [&](int64_t j) { return ld<T>(p.y, row * p.ldy + j); });
        auto z_at = [&](int64_t j) {
            float z = ld<T>(p.r, row * p.ldr + j);
            if (p.y) {
                const float u = (ld<T>(p.y, row * p.ldy + j) - sy.mu) * sy.rho * gamma_at(p.post, j) + beta_at(p.post, j);
                z += p.scale * gate_at<T>(p, row, j) * u;
            }
            return z;
        };
        const Stat sz = row_stat(p.pre, n, red, z_at);
        for (int64_t j = threadIdx.x; j < blocks * 32; j += 256) {
            float h = 0.0f;
            if (j < n) {
                const float z = z_at(j);
                h = (z - sz.mu) * sz.rho * gamma_at(p.pre, j) + beta_at(p.pre, j);
                if (p.z) st<T>(p.z, row * p.ldz + j, z);
                if (p.h) st<T>(p.h, row * p.ldh + j, h);
            }
            if (p.codes) {
                // a warp holds one block of 32
                h = as_stored<T>(h);
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
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(256) backward_kernel(BlockP p, GradP g) {
    __shared__ float red[8];
    const int64_t n = p.n;
    float* acc = g.partials ? g.partials + (int64_t)blockIdx.x * 4 * n : nullptr;
    if (acc)
        for (int64_t i = threadIdx.x; i < 4 * n; i += 256)
            if ((g.sums >> (i / n)) & 1) acc[i] = 0.0f;
    __syncthreads();
    const float inv_n = 1.0f / (float)n;
    for (int64_t row = blockIdx.x; row < p.m; row += gridDim.x) {
        auto z_at = [&](int64_t j) { return ld<T>(p.z, row * p.ldz + j); };
        auto y_at = [&](int64_t j) { return ld<T>(p.y, row * p.ldy + j); };
        const Stat sz = row_stat(p.pre, n, red, z_at);
        Stat sy{0.0f, 1.0f};
        if (p.y) sy = row_stat(p.post, n, red, y_at);
        // means of a and a z^ of the norm before the next block
        float a0 = 0.0f, a1 = 0.0f;
        if (g.dh && p.pre.kind != RT_NORM_NONE) {
            for (int64_t j = threadIdx.x; j < n; j += 256) {
                const float a = ld<T>(g.dh, row * g.lddh + j) * gamma_at(p.pre, j);
                a0 += a;
                a1 += a * (z_at(j) - sz.mu) * sz.rho;
            }
            a0 = p.pre.kind == RT_NORM_LAYER ? block_sum(a0, red) * inv_n : 0.0f;
            a1 = block_sum(a1, red) * inv_n;
        }
        auto dr_at = [&](int64_t j) {
            float d = g.dz ? ld<T>(g.dz, row * g.lddz + j) : 0.0f;
            if (g.dh) {
                const float a = ld<T>(g.dh, row * g.lddh + j) * gamma_at(p.pre, j);
                d += (a - a0 - (z_at(j) - sz.mu) * sz.rho * a1) * sz.rho;
            }
            return d;
        };
        float b0 = 0.0f, b1 = 0.0f, gsum = 0.0f;
        if (p.y) {
            for (int64_t j = threadIdx.x; j < n; j += 256) {
                const float dt = p.scale * dr_at(j), hat = (y_at(j) - sy.mu) * sy.rho;
                const float b = dt * gate_at<T>(p, row, j) * gamma_at(p.post, j);
                b0 += b;
                b1 += b * hat;
                gsum += dt * (hat * gamma_at(p.post, j) + beta_at(p.post, j));
            }
            b0 = p.post.kind == RT_NORM_LAYER ? block_sum(b0, red) * inv_n : 0.0f;
            b1 = p.post.kind != RT_NORM_NONE ? block_sum(b1, red) * inv_n : 0.0f;
            if (g.dgate && p.gate_mode == GATE_COLUMN) {
                gsum = block_sum(gsum, red);
                if (threadIdx.x == 0) static_cast<float*>(g.dgate)[row * g.lddg] = gsum;
            }
        }
        for (int64_t j = threadIdx.x; j < n; j += 256) {
            const float dr = dr_at(j);
            if (p.y) {
                const float dt = p.scale * dr, hat = (y_at(j) - sy.mu) * sy.rho, gt = gate_at<T>(p, row, j);
                const float b = dt * gt * gamma_at(p.post, j);
                if (g.dy) st<T>(g.dy, row * g.lddy + j, (b - b0 - hat * b1) * sy.rho);
                if (g.dgate && p.gate_mode == GATE_FULL)
                    st<T>(g.dgate, row * g.lddg + j, dt * (hat * gamma_at(p.post, j) + beta_at(p.post, j)));
                const float w = p.gate_mode >= GATE_COLUMN ? dt * gt : dt;
                if (g.sums & 1) acc[j] += w * hat;
                if (g.sums & 2) acc[n + j] += w;
            }
            if (g.dh) {
                const float dh = ld<T>(g.dh, row * g.lddh + j);
                if (g.sums & 4) acc[2 * n + j] += dh * (z_at(j) - sz.mu) * sz.rho;
                if (g.sums & 8) acc[3 * n + j] += dh;
            }
            if (g.dr) st<T>(g.dr, row * g.lddr + j, dr);
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
        const float4 a = __ldg(reinterpret_cast<const float4*>(p + at)), b = __ldg(reinterpret_cast<const float4*>(p + at) + 1);
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

// Mean and reciprocal deviation of a row held 8 C elements a thread.
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
    s.rho = 1.0f / sqrtf(row_sum<TPR>(t, red, turn) * inv_n + p.eps);
    return s;
}

// One pass: a row lies in the registers of TPR threads, 8 neighbouring elements
// in each of C turns, so y and r are read once, z and h written once and the
// sums of a norm are taken twice over the same registers (mean, then the centred
// squares).  HBM-bound: 4 elements moved for each of the row.  Needs 16-byte
// aligned rows and whole eights (n % 8 = 0); a CTA holds ROWS = max(1, 128 / TPR)
// rows.
constexpr int cta_threads(int tpr) { return tpr < 128 ? 128 : tpr; }

template <typename T, int TPR, int C>
__global__ void __launch_bounds__(cta_threads(TPR)) forward_rows_kernel(BlockP p) {
    constexpr int ROWS = cta_threads(TPR) / TPR;
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
        const float one = p.gate_mode == GATE_ONE              ? __ldg(static_cast<const float*>(p.gate))
                          : p.gate_mode == GATE_COLUMN && live ? __ldg(static_cast<const float*>(p.gate) + row * p.ldg)
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
    const int blocks = (n + 31) / 32, groups = (blocks + 3) / 4;
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
            if (p.h) store8<T>(p.h, row * p.ldh + j, z[c]);
        }
        if (p.codes) {
            // four neighbouring lanes hold a block of 32
            uint32_t amax = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                z[c][i] = has[c] ? as_stored<T>(z[c][i]) : 0.0f;
                amax = max(amax, __float_as_uint(z[c][i]) & 0x7fffffffu);
            }
            amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            const uint32_t byte = mx4::scale_byte(amax);
            const float inv = mx4::inv_scale(byte);
            uint32_t code = 0;
#pragma unroll
            for (int i = 0; i < 8; i += 2) code |= mx4::encode2(z[c][i] * inv, z[c][i + 1] * inv) << (4 * i);
            if (byte == mx4::kNanScale) code = 0;
            if (live && j < blocks * 32) *reinterpret_cast<uint32_t*>(p.codes + row * blocks * 16 + (j >> 1)) = code;
            // the scales of a group's four blocks as one word
            uint32_t word = byte | __shfl_down_sync(0xffffffffu, byte, 4) << 8;
            word |= __shfl_down_sync(0xffffffffu, word, 8) << 16;
            if (live && (threadIdx.x & 15) == 0 && j < groups * 128)
                *reinterpret_cast<uint32_t*>(p.scales + mx4::scale_offset(row, j >> 5, groups)) = word;
        }
    }
}

struct ReduceP {
    const float* partials;
    int parts, sums;
    int64_t n;
    int gate_mode;
    const float* gate;
    const float *gamma, *beta;  // of the norm after the block
    float *dgamma_post, *dbeta_post, *dgamma_pre, *dbeta_pre, *dgate;
    float* gate_row;  // [n]: a [1,1] gate's gradient by column
};

// Column sums of the partials, parts in order, and the vectors they give.
__global__ void __launch_bounds__(256) column_kernel(ReduceP p) {
    const int64_t j = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (j >= p.n) return;
    float s[4] = {};
    for (int i = 0; i < p.parts; ++i)
#pragma unroll
        for (int v = 0; v < 4; ++v)
            if ((p.sums >> v) & 1) s[v] += p.partials[((int64_t)i * 4 + v) * p.n + j];
    const float g = p.gate_mode == GATE_ONE ? p.gate[0] : p.gate_mode == GATE_ROW ? p.gate[j] : 1.0f;
    if (p.dgamma_post) p.dgamma_post[j] = s[0] * g;
    if (p.dbeta_post) p.dbeta_post[j] = s[1] * g;
    if (p.dgamma_pre) p.dgamma_pre[j] = s[2];
    if (p.dbeta_pre) p.dbeta_pre[j] = s[3];
    const float dg = (p.gamma ? p.gamma[j] : 1.0f) * s[0] + (p.beta ? p.beta[j] * s[1] : 0.0f);
    if (p.gate_row) p.gate_row[j] = dg;
    else if (p.dgate) p.dgate[j] = dg;
}

__global__ void __launch_bounds__(256) gate_one_kernel(const float* row, int64_t n, float* out) {
    __shared__ float red[8];
    float s = 0.0f;
    for (int64_t j = threadIdx.x; j < n; j += 256) s += row[j];
    s = block_sum(s, red);
    if (threadIdx.x == 0) out[0] = s;
}

// --------------------------------------------------------------- host side
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
void launch_forward_rows(const BlockP& p, cudaStream_t st) {
    constexpr int threads = cta_threads(TPR), rows = threads / TPR;
    forward_rows_kernel<T, TPR, C><<<(unsigned)((p.m + rows - 1) / rows), threads, 0, st>>>(p);
}

// Up to 16384 wide: the fewest threads that hold a row eight elements each (the
// widest rows, sixteen).
template <typename T>
bool forward_rows(const BlockP& p, cudaStream_t st) {
    if (!rows_aligned(p, sizeof(T)) || p.n > 16384 || p.m > INT32_MAX) return false;
    if (p.n <= 256) launch_forward_rows<T, 32>(p, st);
    else if (p.n <= 512) launch_forward_rows<T, 64>(p, st);
    else if (p.n <= 1024) launch_forward_rows<T, 128>(p, st);
    else if (p.n <= 2048) launch_forward_rows<T, 256>(p, st);
    else if (p.n <= 4096) launch_forward_rows<T, 512>(p, st);
    else if (p.n <= 8192) launch_forward_rows<T, 1024>(p, st);
    else launch_forward_rows<T, 1024, 2>(p, st);
    return true;
}

int parts_for(const rt_ctx* ctx, int64_t m) { return (int)std::max<int64_t>(1, std::min<int64_t>(m, ctx->sm_count)); }

}  // namespace
}  // namespace rt

using namespace rt;

extern "C" {

int rt_block_forward(rt_ctx* ctx, const rt_block_args* a) {
    RT_CHECK(ctx && a && a->r, "rt_block_forward: bad arguments");
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
    const int grid = (int)std::min<int64_t>(p.m, (int64_t)ctx->sm_count * 8);
    if (a->r->dtype == RT_BF16) {
        if (!forward_rows<__nv_bfloat16>(p, ctx->stream)) forward_kernel<__nv_bfloat16><<<grid, 256, 0, ctx->stream>>>(p);
    } else {
        if (!forward_rows<float>(p, ctx->stream)) forward_kernel<float><<<grid, 256, 0, ctx->stream>>>(p);
    }
    RT_CUDA(cudaGetLastError());
    count_launch(ctx);
    return RT_OK;
}

int64_t rt_block_backward_workspace(rt_ctx* ctx, int64_t m, int64_t n) {
    if (!ctx || m < 0 || n < 0) {
        set_error("rt_block_backward_workspace: bad arguments");
        return -1;
    }
    return (int64_t)parts_for(ctx, m) * 4 * n + n;
}

int rt_block_backward(rt_ctx* ctx, const rt_block_args* a, const rt_block_grads* g) {
    RT_CHECK(ctx && a && g, "rt_block_backward: bad arguments");
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
    if (p.n == 0) return RT_OK;
    const int parts = parts_for(ctx, p.m);
    if (q.sums) {
        RT_CHECK(g->work && g->work->dtype == RT_F32 && g->work->rows == 1 &&
                     g->work->cols >= rt_block_backward_workspace(ctx, p.m, p.n),
                 "rt_block_backward: work must be %lld f32 in one row",
                 (long long)rt_block_backward_workspace(ctx, p.m, p.n));
        q.partials = static_cast<float*>(g->work->ptr);
    }
    RT_CUDA(cudaSetDevice(ctx->device));
    // without rows the sums over rows are zero: the partials of one CTA
    if (z->dtype == RT_BF16)
        backward_kernel<__nv_bfloat16><<<parts, 256, 0, ctx->stream>>>(p, q);
    else
        backward_kernel<float><<<parts, 256, 0, ctx->stream>>>(p, q);
    RT_CUDA(cudaGetLastError());
    count_launch(ctx);
    if (!q.sums) return RT_OK;
    c.partials = q.partials;
    c.parts = parts;
    c.sums = q.sums;
    c.n = p.n;
    c.gate_mode = p.gate_mode;
    c.gate = static_cast<const float*>(p.gate);
    c.gamma = p.post.gamma;
    c.beta = p.post.beta;
    if (gate_sums && p.gate_mode == GATE_ONE) c.gate_row = q.partials + (int64_t)parts * 4 * p.n;
    column_kernel<<<(unsigned)((p.n + 255) / 256), 256, 0, ctx->stream>>>(c);
    RT_CUDA(cudaGetLastError());
    count_launch(ctx);
    if (c.gate_row) {
        gate_one_kernel<<<1, 256, 0, ctx->stream>>>(c.gate_row, p.n, c.dgate);
        RT_CUDA(cudaGetLastError());
        count_launch(ctx);
    }
    return RT_OK;
}

}  // extern "C"
