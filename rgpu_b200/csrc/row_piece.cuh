// How the kernels that read or write matrices row by row reach their elements: a lane's
// 32 bytes whatever the rows' alignment, and the order in which warps take rows and
// pieces of them.
#pragma once

#include <algorithm>
#include <cstdint>

#include "internal.h"

namespace rt {

// A lane's piece of a row: 32 bytes, 16 bf16 or 8 f32.  V: bytes of an access, 32
// (one 256-bit access, Blackwell's widest) or 16 where the rows are so aligned.
// Else (0) a warp's accesses take neighbouring words, which change hands through its
// kilobyte of shared memory; an aligned row's last piece goes element by element.
template <typename T>
struct Piece {
    static constexpr int E = 32 / sizeof(T);         // elements
    static constexpr int WARP = 32 * E;              // elements of a warp
    uint32_t w[8];

    // All of the piece.  Without a branch, so that one load is not waited for before the next
    // is issued (dropout of 8192 x 8192 bf16 with a sum 59.9 us, with load below 60.9; without one 46.1 and 47.8).
    template <int V>
    __device__ __forceinline__ void load_whole(const T* p) {
        if constexpr (V == 32) {
            asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                         : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                         : "l"(p)
                         : "memory");
        } else {
            const uint4* at = reinterpret_cast<const uint4*>(p);
            const uint4 a = at[0], b = at[1];
            w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w;
            w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
        }
    }
    template <int V>
    __device__ __forceinline__ void load(const T* p, int64_t left) {
        if (V == 32 && left >= E) {
            load_whole<32>(p);
        } else if (V == 16 && left >= E) {
            load_whole<16>(p);
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
            r.v[i] = room >= N ? words[at] : N == 2 && room == 1 ? half(p + odd + at * N) : 0u;
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
    __device__ __forceinline__ float value(int e) const {
        if constexpr (sizeof(T) == 2)
            return __uint_as_float(e & 1 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
        else
            return __uint_as_float(w[e]);
    }
};

// A warp takes one piece a lane of the four rows r, r + 32, r + 64, r + 96 of a 128-row
// tile: every lane has four 32-byte reads under way, and the scales of these rows in a
// block-scaled matrix lie side by side.
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

// Sets and chunks, and a grid that covers chunks before sets.
inline Rows rows_for(const rt_ctx* ctx, int64_t rows, int64_t k, int chunk, dim3* grid) {
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
inline int access_of(const rt_tensor* t) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(t->ptr) | (uintptr_t)(t->ld * (int64_t)dtype_size(t->dtype));
    return (a & 31) == 0 ? 32 : (a & 15) == 0 ? 16 : 0;
}

}  // namespace rt
