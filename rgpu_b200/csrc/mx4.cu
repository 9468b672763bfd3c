// Microscaled 4-bit matrices: handles, quantisation and dequantisation.
#include <algorithm>
#include <climits>
#include <new>

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

// A lane's piece of a row: 32 bytes, 16 bf16 or 8 f32.  V: bytes of an access, 32
// (one 256-bit access, Blackwell's widest) or 16 where the rows are so aligned.
// Else (0) a warp's accesses take neighbouring words, which change hands through its
// kilobyte of shared memory; an aligned row's last piece goes element by element.
template <typename T>
struct Piece {
    static constexpr int E = 32 / sizeof(T);         // elements
    static constexpr int PER_BLOCK = 32 / E;         // lanes that share a block
    static constexpr int PER_GROUP = 128 / E;        // and a scale group
    static constexpr int WARP = 32 * E;              // elements of a warp
    uint32_t w[8];

    template <int V>
    __device__ __forceinline__ void load(const T* p, int64_t left) {
        if (V == 32 && left >= E) {
            asm volatile("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                         : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                         : "l"(p));
        } else if (V == 16 && left >= E) {
            const uint4 a = __ldg(reinterpret_cast<const uint4*>(p)), b = __ldg(reinterpret_cast<const uint4*>(p) + 1);
            w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w;
            w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = 0;
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (e < left) {
                    if constexpr (sizeof(T) == 2)
                        w[e / 2] |= (uint32_t)__bfloat16_as_ushort(p[e]) << (16 * (e & 1));
                    else
                        w[e] = __float_as_uint(p[e]);
                }
        }
    }
    template <int V>
    __device__ __forceinline__ void store(T* p, int64_t left) const {
        if (V == 32 && left >= E) {
            asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
                         "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                         : "memory");
        } else if (V == 16 && left >= E) {
            reinterpret_cast<uint4*>(p)[0] = make_uint4(w[0], w[1], w[2], w[3]);
            reinterpret_cast<uint4*>(p)[1] = make_uint4(w[4], w[5], w[6], w[7]);
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (e < left) {
                    if constexpr (sizeof(T) == 2)
                        p[e] = __ushort_as_bfloat16((unsigned short)(w[e / 2] >> (16 * (e & 1))));
                    else
                        p[e] = __uint_as_float(w[e]);
                }
        }
    }
    // The warp's piece of an unaligned row of which `left` elements lie from p on, p and
    // left the warp's, not the lane's: read as words, then shared out through box, the
    // warp's 1 KB.  bf16 whose row starts between two words: pairs from element 1 on, and
    // element 0 by itself (`head`); a lane's words are then half a word off.
    struct Words {
        uint32_t v[8], head;
    };
    static __device__ __forceinline__ bool between(const T* p) { return sizeof(T) == 2 && (reinterpret_cast<uintptr_t>(p) & 2); }
    static __device__ __forceinline__ uint32_t half(const T* p) { return *reinterpret_cast<const unsigned short*>(p); }
    static __device__ __forceinline__ Words fetch_any(const T* p, int64_t left, int lane) {
        Words r;
        constexpr int N = 4 / sizeof(T);  // elements of a word
        const int odd = between(p);
        const uint32_t* words = reinterpret_cast<const uint32_t*>(p + odd);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int at = i * 32 + lane;
            const int64_t room = left - odd - at * N;
            r.v[i] = room >= N ? __ldg(words + at) : N == 2 && room == 1 ? half(p + odd + at * N) : 0u;
        }
        r.head = odd && lane == 0 && left > 0 ? half(p) << 16 : 0u;
        return r;
    }
    __device__ __forceinline__ void deal_any(const Words& r, bool odd, uint32_t* box, int lane) {
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; ++i) box[i * 32 + lane] = r.v[i];
        __syncwarp();
        const uint4 a = reinterpret_cast<const uint4*>(box)[lane * 2], b = reinterpret_cast<const uint4*>(box)[lane * 2 + 1];
        w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w;
        w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
        if (sizeof(T) == 2 && odd) {  // the same of the whole warp
            uint32_t before = __shfl_up_sync(0xffffffffu, w[7], 1);
            if (lane == 0) before = r.head;
#pragma unroll
            for (int i = 7; i >= 0; --i) w[i] = __funnelshift_l(i ? w[i - 1] : before, w[i], 16);
        }
    }
    __device__ __forceinline__ void store_any(T* p, int64_t left, uint32_t* box, int lane) const {
        constexpr int N = 4 / sizeof(T);
        const int odd = between(p);
        uint32_t s[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) s[i] = w[i];
        if (sizeof(T) == 2 && odd) {
            const uint32_t after = __shfl_down_sync(0xffffffffu, w[0], 1);
#pragma unroll
            for (int i = 0; i < 8; ++i) s[i] = __funnelshift_r(w[i], i < 7 ? w[i + 1] : after, 16);
            if (lane == 0 && left > 0) *reinterpret_cast<unsigned short*>(p) = (unsigned short)w[0];
        }
        __syncwarp();
        reinterpret_cast<uint4*>(box)[lane * 2] = make_uint4(s[0], s[1], s[2], s[3]);
        reinterpret_cast<uint4*>(box)[lane * 2 + 1] = make_uint4(s[4], s[5], s[6], s[7]);
        __syncwarp();
        uint32_t* words = reinterpret_cast<uint32_t*>(p + odd);
        const int64_t end = min(left, (int64_t)WARP) - odd;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int at = i * 32 + lane;
            const int64_t room = end - at * N;
            if (room >= N)
                words[at] = box[at];
            else if (N == 2 && room == 1)
                *reinterpret_cast<unsigned short*>(words + at) = (unsigned short)box[at];
        }
    }
    // Bit pattern (as f32) of the largest magnitude in the lane.
    __device__ __forceinline__ uint32_t amax() const {
        uint32_t m = 0;
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int i = 0; i < 8; ++i) asm("max.u16x2 %0, %0, %1;" : "+r"(m) : "r"(w[i] & 0x7fff7fffu));
            return max(m << 16, m & 0xffff0000u);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) m = max(m, w[i] & 0x7fffffffu);
            return m;
        }
    }
    // Codes of the elements 8 i .. 8 i + 7.
    __device__ __forceinline__ uint32_t encode(int i, float inv) const {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if constexpr (sizeof(T) == 2) {
                const uint32_t x = w[i * 4 + e / 2];
                v[e] = __uint_as_float(e & 1 ? x & 0xffff0000u : x << 16);
            } else {
                v[e] = __uint_as_float(w[e]);
            }
        }
        return encode8(v, inv);
    }
};

// Blocks along a row.  A warp takes 512 (f32: 256) elements of the four rows r,
// r + 32, r + 64, r + 96 of a 128-row tile: the scales of these rows lie side by
// side, 16 bytes for a group, and every lane has four 32-byte reads under way.  Few
// lanes to a block keep the instructions per element low enough for HBM to be the
// bound: 2 (f32: 4) bytes in and 17/32 out per element.  8192 x 8192 bf16: 30 us,
// 5.7 TB/s.
struct Rows {
    int64_t sets;  // sets of four rows
    int rcount;    // rows r of a tile: 32, or fewer where the matrix has fewer
    int chunks;    // warps' worth of elements along k
    int split;     // log2 of the warps of a CTA that lie along k; the others take other sets
};

// The warp's first chunk along k and first set, and the grid's strides.
struct Place {
    int chunk, chunk_step;
    int64_t set, set_step;
    __device__ __forceinline__ explicit Place(const Rows& w) {
        const int warp = threadIdx.x >> 5;
        chunk = ((int)blockIdx.x << w.split) + (warp & ((1 << w.split) - 1));
        chunk_step = (int)gridDim.x << w.split;
        set = ((int64_t)blockIdx.y << (3 - w.split)) + (warp >> w.split);
        set_step = (int64_t)gridDim.y << (3 - w.split);
    }
};
// First row of a set.
__device__ __forceinline__ int64_t set_row(const Rows& w, int64_t set) {
    return w.rcount == 32 ? (set >> 5) * 128 + (set & 31) : set;
}

template <typename T, int V>
__global__ void __launch_bounds__(256, V ? 4 : 3) quantize_rows_kernel(const T* __restrict__ src, int64_t ld, int64_t rows,
                                                               int64_t k, Rows w, int64_t blocks, int64_t groups,
                                                               uint8_t* __restrict__ codes,
                                                               uint8_t* __restrict__ scales) {
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
                for (int o = 1; o < P::PER_BLOCK; o *= 2) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
                const uint32_t byte = scale_byte(amax);
                const float inv = inv_scale(byte);
                const bool nan = byte == kNanScale;
                if (q < live && inside) {
                    if constexpr (sizeof(T) == 2)
                        *reinterpret_cast<uint2*>(out + q * (32 * row_bytes)) =
                            make_uint2(nan ? 0u : x[q].encode(0, inv), nan ? 0u : x[q].encode(1, inv));
                    else
                        *reinterpret_cast<uint32_t*>(out + q * (32 * row_bytes)) = nan ? 0u : x[q].encode(0, inv);
                }
                // the bytes of a group's four blocks into its first lane
                word[q] = byte | __shfl_down_sync(0xffffffffu, byte, P::PER_BLOCK) << 8;
                word[q] |= __shfl_down_sync(0xffffffffu, word[q], 2 * P::PER_BLOCK) << 16;
            }
            const int64_t group = j >> 7;
            if (lane % P::PER_GROUP == 0 && group < groups)
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
__global__ void __launch_bounds__(256) dequantize_kernel(const uint8_t* __restrict__ codes,
                                                         const uint8_t* __restrict__ scales, int64_t rows, int64_t k,
                                                         Rows w, int64_t blocks, int64_t groups, T* __restrict__ dst,
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
            const uint4 s = !inside ? make_uint4(0, 0, 0, 0) : __ldg(reinterpret_cast<const uint4*>(scales + ((row >> 7) * groups + (j >> 7)) * 512 + (row & 31) * 16));
            const uint32_t word[4] = {s.x, s.y, s.z, s.w};
            const uint8_t* in = codes + row * row_bytes + (j >> 1);
            uint32_t c[4][P::E / 8];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                c[q][0] = c[q][P::E / 8 - 1] = 0;
                if (q < live && inside) {
                    if constexpr (sizeof(T) == 2) {
                        const uint2 two = __ldg(reinterpret_cast<const uint2*>(in + q * (32 * row_bytes)));
                        c[q][0] = two.x;
                        c[q][P::E / 8 - 1] = two.y;
                    } else {
                        c[q][0] = __ldg(reinterpret_cast<const uint32_t*>(in + q * (32 * row_bytes)));
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

// Sets and chunks, and a grid that covers chunks before sets.
Rows rows_for(const rt_ctx* ctx, int64_t rows, int64_t k, int chunk, dim3* grid) {
    Rows w;
    w.rcount = (int)std::min<int64_t>(rows, 32);
    w.sets = w.rcount * ((rows + 127) / 128);
    w.chunks = (int)((k + chunk - 1) / chunk);
    w.split = w.chunks > 4 ? 3 : w.chunks > 2 ? 2 : w.chunks > 1 ? 1 : 0;
    const int64_t along = (w.chunks + (1 << w.split) - 1) >> w.split;
    const int64_t across = (w.sets + (8 >> w.split) - 1) >> (3 - w.split), limit = (int64_t)ctx->sm_count * 64;
    grid->x = (unsigned)std::min(along, limit);
    grid->y = (unsigned)std::min<int64_t>(std::min(across, std::max<int64_t>(1, limit / grid->x)), 65535);
    grid->z = 1;
    return w;
}

// Widest access that every row of t allows: 32, 16 or 0.
int access_of(const rt_tensor* t) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(t->ptr) | (uintptr_t)(t->ld * (int64_t)dtype_size(t->dtype));
    return (a & 31) == 0 ? 32 : (a & 15) == 0 ? 16 : 0;
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
    const int s = mx4_encode_maps(q);
    if (s != RT_OK) {
        cudaFree(p);
        delete q;
        return s;
    }
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
    const int s = mx4_encode_maps(q);
    if (s != RT_OK) {
        delete q;
        return s;
    }
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
    RT_CHECK(ctx && a && b && c, "rt_mx4_matmul: bad arguments");
    RT_CHECK(a->ctx == ctx && b->ctx == ctx && c->ctx == ctx && (!bias || bias->ctx == ctx),
             "tensor belongs to another context");
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
