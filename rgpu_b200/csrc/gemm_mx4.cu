// Product of two microscaled 4-bit matrices on the tensor cores,
// C[m,n] = A[m,k] B[n,k]^T + 1 bias (+ ReLU): tcgen05.mma kind::mxf4 with one
// E8M0 scale per 32 elements, f32 accumulators in TMEM.
//
// A's rows are called tokens here, T; B's rows are C's columns, W.
//
// A k stage is 256 elements: 128 bytes of codes per row (one 128-byte-swizzled
// TMA box) and two 512-byte scale tiles per 128 rows, in memory already in the
// order that tcgen05.cp spreads over TMEM (32 lanes x 4 columns, repeated in the
// four lane quadrants).  Each shared-memory stage has TMEM columns for its scales
// of its own, so the barrier that frees a stage frees its scales too.  A stage is
// four MMAs of 64 elements, two scales a row each.  Boxes past the matrices read
// zeros; MMAs wholly past k are not issued, and the last scale tile's bytes past
// k's blocks are not NaN, so they meet zero codes harmlessly.
#include <algorithm>

#include "landing.cuh"
#include "mx4.cuh"
#include "tc_common.cuh"

namespace rt {
namespace {

using namespace tc;

constexpr int kStageK = 256;          // elements of k in a stage
constexpr int kStageBlocks = kStageK / 32;
constexpr int kRowBytes = 128;        // codes of a row in a stage
constexpr int kWBytes = 128 * kRowBytes;
constexpr int kScaleTile = 512;       // scales of 128 rows x 4 blocks

struct Mx4Params {
    int64_t m, n;                     // C's extents
    int tiles_m, tiles_n;             // token tiles, column tiles
    int blocks;                       // blocks of 32 along k
    int stages, stages_per_split;     // k stages in all, and of one split
    void* c;
    int64_t ldc;
    int out_bf16;
    const float* bias;
    int relu;
    int access;                       // bytes that C's rows are aligned to (32, 16, 8, or 0 for less)
    int* err;
};

// kind::mxf4 instruction descriptor: E2M1 operands, both K-major, E8M0 scales;
// `half` selects the scale bytes 0-1 or 2-3 of each TMEM word for A and B.
__host__ __device__ constexpr uint32_t mx4_idesc(int m, int n, int half) {
    return (1u << 7)                         // A: E2M1
           | (1u << 10)                      // B: E2M1
           | ((uint32_t)(n >> 3) << 17)      // N / 8
           | (1u << 23)                      // scales: E8M0
           | ((uint32_t)(m >> 7) << 27)      // M / 128
           | ((uint32_t)(half * 2) << 29)    // A's scale bytes
           | ((uint32_t)(half * 2) << 4);    // B's scale bytes
}

template <int CG>
__device__ __forceinline__ void mma_mx4(uint32_t d, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t sfa,
                                        uint32_t sfb, uint32_t accumulate) {
    if constexpr (CG == 1)
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
            "l"(ad), "l"(bd), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
            "l"(ad), "l"(bd), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
            : "memory");
}

// Descriptor of a scale tile in shared memory: no swizzle, 8-row groups of
// 16-byte rows 128 bytes apart.
__device__ __forceinline__ uint64_t scale_desc(uint32_t smem) {
    return (uint64_t)((smem & 0x3FFFFu) >> 4) | ((uint64_t)1 << 16) | ((uint64_t)8 << 32) | ((uint64_t)1 << 46);
}

// One 512-byte scale tile from shared memory to four TMEM columns.
template <int CG>
__device__ __forceinline__ void copy_scales(uint32_t tmem, uint64_t desc) {
    if constexpr (CG == 1)
        asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
    else
        asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
}

// One lane of a converged warp.  The MMA warps run their loops with all lanes
// and issue from the elected one: descriptors and TMEM addresses then stay in
// uniform registers, where a lone diverged lane moves each into one for every
// instruction (measured at 8192^3: 120 clocks for each MMA issued, 335 more a
// stage, against 128 that the MMA takes).
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }

__device__ __forceinline__ uint32_t cta_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t in_cta(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}
__device__ __forceinline__ void sync_cluster() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__device__ __forceinline__ void tmem_ld_nowait(uint32_t taddr, float (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]),
          "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]),
          "=f"(r[16]), "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]),
          "=f"(r[24]), "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
        : "r"(taddr)
        : "memory");
}
// Waits for the loads above; naming the registers keeps their uses behind it.
__device__ __forceinline__ void tmem_ld_wait(float (&v)[4][32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int j = 0; j < 32; ++j) asm volatile("" : "+f"(v[c][j]));
}

// The larger of the two, a NaN if either is one: ReLU with floor 0, nothing with
// floor -infinity.
__device__ __forceinline__ float at_least(float v, float floor) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(v), "f"(floor));
    return r;
}

__device__ __forceinline__ void load_bias4(const Mx4Params& p, int64_t col, float (&bias)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) bias[i] = p.bias && col + i < p.n ? __ldg(p.bias + col + i) : 0.0f;
}

template <typename T>
__device__ __forceinline__ void store_one(T* c, float v) {
    if constexpr (sizeof(T) == 2)
        *c = __float2bfloat16_rn(v);
    else
        *c = v;
}

// Adds the splits' sums of a tile in order and stores C.  Each of the cluster's
// `splits` CTAs holds [token][128 columns] f32 at `sums` of its shared memory; the
// tokens are dealt out over the splits (this one is number `split`) and their warps.
// A lane takes four columns from `col` on; four tokens are under way at a time.
template <typename T>
__device__ __forceinline__ void add_splits(const Mx4Params& p, uint32_t sums, uint32_t splits, uint32_t split, int warp,
                                           int warps, int64_t row0, int count, int64_t col, const float (&bias)[4],
                                           int lane) {
    constexpr int U = 4;
    const float floor = p.relu ? 0.0f : -INFINITY;
    const int step = warps * (int)splits;
    int c = (int)split + warp * (int)splits;
    T* to = static_cast<T*>(p.c) + (row0 + c) * p.ldc + col;
    const int64_t ld = p.ldc * step;
    // four neighbouring elements of a row as one store, where they lie so in every row
    const bool whole = col + 3 < p.n && p.access >= 4 * (int)sizeof(T);
    const int left = (int)max((int64_t)0, min((int64_t)4, p.n - col));
    for (; c < count; c += U * step, to += U * ld) {
        float4 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 2
        for (uint32_t r = 0; r < splits; ++r) {
            const uint32_t at = in_cta(sums + lane * 16, r);
            float4 x[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (c + u * step < count) x[u] = ld_cluster4(at + (c + u * step) * 512);
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (c + u * step < count) {
                    v[u].x += x[u].x;
                    v[u].y += x[u].y;
                    v[u].z += x[u].z;
                    v[u].w += x[u].w;
                }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (c + u * step >= count) continue;
            T* at = to + u * ld;
            const float x[4] = {at_least(v[u].x + bias[0], floor), at_least(v[u].y + bias[1], floor),
                                at_least(v[u].z + bias[2], floor), at_least(v[u].w + bias[3], floor)};
            if (whole) {
                if constexpr (sizeof(T) == 2) {
                    const __nv_bfloat162 lo = __floats2bfloat162_rn(x[0], x[1]), hi = __floats2bfloat162_rn(x[2], x[3]);
                    *reinterpret_cast<uint2*>(at) =
                        make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
                } else {
                    *reinterpret_cast<float4*>(at) = make_float4(x[0], x[1], x[2], x[3]);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (i < left) store_one(at + i, x[i]);
            }
        }
    }
}

// ------------------------------------------------------------ one-CTA kernel
// For few tokens or little work.  The tensor cores compute C^T: 128 of W's rows are
// the MMA's M rows and TN tokens its N columns, so a CTA computes 128 columns of C
// for TN tokens over its share of k.  The CTAs of a cluster share one tile, split
// along k.  Their sums meet in shared memory and are added in rank order, tokens
// dealt out over the CTAs.  One token by 8192 x 8192: 9.6 us, 5.4 of them the
// weights' 36 MB at the rate of a copy, the others the launch and the join (8.2 with
// the weights in L2).  64 x 8192 x 4096: 6.9 to 7.1 us.  2047 x 1000 x 8192: 12.3 to 12.7 us,
// a stage 0.23 us for 35 KB, 19 TB/s from L2 to all SMs.
template <int TN>
struct Geo1 {
    static constexpr int T_BYTES = TN * kRowBytes;
    static constexpr int STAGE_BYTES = kWBytes + T_BYTES + 4 * kScaleTile;  // codes, two scale tiles of either side
    static constexpr int CTAS = TN > 64 ? 1 : 2;  // to an SM
    static constexpr int STAGES = CTAS > 1 ? 4 : 6;
    static constexpr int TMEM_COLS = 512 / CTAS;  // two accumulators of TN, and 16 of scales a stage
    static constexpr int SMEM = STAGES * STAGE_BYTES + 1024 + 256;
    static_assert(2 * TN + 16 * STAGES <= TMEM_COLS, "TMEM columns");
    static_assert(CTAS * SMEM <= 226 * 1024, "shared memory of an SM");
    static_assert(TN * 512 <= STAGES * STAGE_BYTES, "the split sums reuse the stages");
};

constexpr int kThreads1 = 224;  // warps: 0 TMA, 1 MMA, 2-5 epilogue (one TMEM lane quadrant each), 6 MMA

template <int TN>
__global__ void __launch_bounds__(kThreads1) mx4_kernel(const __grid_constant__ CUtensorMap map_w,
                                                        const __grid_constant__ CUtensorMap map_t,
                                                        const __grid_constant__ CUtensorMap map_sw,
                                                        const __grid_constant__ CUtensorMap map_st, Mx4Params p) {
    using G = Geo1<TN>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* smem_w = smem;
    uint8_t* smem_t = smem + G::STAGES * kWBytes;
    uint8_t* smem_s = smem_t + G::STAGES * G::T_BYTES;  // [stage][W 2 tiles, T 2 tiles]
    uint64_t* full = reinterpret_cast<uint64_t*>(smem_s + G::STAGES * 4 * kScaleTile);
    uint64_t* empty = full + G::STAGES;
    uint64_t* done = empty + G::STAGES;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    volatile int* issued_all = abort_flag + 1;

    const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
    const uint32_t rank = cta_rank(), ranks = cluster_size();
    const int tile = (int)(blockIdx.x / ranks);
    const int tm = tile % p.tiles_m, tn = tile / p.tiles_m;
    const int s0 = (int)rank * p.stages_per_split, s1 = min(p.stages, s0 + p.stages_per_split);

    if (threadIdx.x == 0) {
        for (int s = 0; s < G::STAGES; ++s) {
            mbar_init(smem_u32(&full[s]), 1);
            mbar_init(smem_u32(&empty[s]), 1);
        }
        mbar_init(smem_u32(done), 2);
        *abort_flag = 0;
        *issued_all = 0;
        fence_barrier_init();
        prefetch_tmap(&map_w);
        prefetch_tmap(&map_t);
        prefetch_tmap(&map_sw);
        prefetch_tmap(&map_st);
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "r"(G::TMEM_COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = uniform(*tmem_slot);
    // a programmatic dependent launch: the set-up above touched no global memory
    pdl_wait();
    pdl_launch_dependents();
    float bias[4];  // of the lane's columns of the epilogue
    load_bias4(p, (int64_t)tn * 128 + lane * 4, bias);

    if (warp == 0) {
        const uint32_t w0 = smem_u32(smem_w), t0 = smem_u32(smem_t), sc0 = smem_u32(smem_s);
        const uint32_t full0 = smem_u32(full), empty0 = smem_u32(empty);
        int slot = 0, phase = 1, issued = 0;
        bool ok = true;
        for (int s = s0; s < s1; ++s, ++issued) {
            ok = __all_sync(0xffffffffu, mbar_wait(empty0 + slot * 8, phase, abort_flag));
            if (!ok) break;
            if (elect_one()) {
                const uint32_t bar = full0 + slot * 8, ss = sc0 + slot * 4 * kScaleTile;
                mbar_expect_tx(bar, G::STAGE_BYTES);
                tma_load_2d(w0 + slot * kWBytes, &map_w, s * kRowBytes, tn * 128, bar);
                tma_load_2d(t0 + slot * G::T_BYTES, &map_t, s * kRowBytes, tm * TN, bar);
                tma_load_3d(ss, &map_sw, 0, s * 2, tn, bar);
                tma_load_3d(ss + 2 * kScaleTile, &map_st, 0, s * 2, tm * TN / 128, bar);
            }
            __syncwarp();
            if (++slot == G::STAGES) {
                slot = 0;
                phase ^= 1;
            }
        }
        if (elect_one()) {
            *issued_all = issued;
            if (!ok) {
                record_error(p.err, DEV_TIMEOUT_PRODUCER, blockIdx.x);
                *abort_flag = 1;
            }
        }
    } else if (warp == 1 || warp == 6) {
        // A stage's copies and MMAs take a warp 0.3 us to issue, more than they take to run:
        // two warps take every second stage, with an accumulator each (100 x 1000 x 4096: 6.7
        // us, with one 7.6).
        const int odd = warp == 6;
        const uint32_t token_col = (uint32_t)((tm * TN % 128) / 32);  // the tile's place in its 128-row scale tile
        const uint64_t w0 = smem_desc(smem_u32(smem_w), 16, 1024), t0 = smem_desc(smem_u32(smem_t), 16, 1024);
        const uint64_t sc0 = scale_desc(smem_u32(smem_s));
        const uint32_t cols0 = tmem + 2 * TN, sum = tmem + odd * TN;
        static_assert(G::STAGES % 2 == 0, "a warp's stages are every second slot");
        bool ok = true;
        int slot = odd, phase = 0;
        for (int s = s0 + odd; s < s1; s += 2) {
            ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&full[slot]), phase, abort_flag));
            if (!ok) break;
            tc_fence_after();
            const uint64_t w = w0 + slot * (kWBytes >> 4), t = t0 + slot * (G::T_BYTES >> 4);
            const uint64_t sc = sc0 + slot * (4 * kScaleTile >> 4);
            const uint32_t cols = cols0 + slot * 16;  // scales: W groups 0, 1, then T groups 0, 1
            const int steps = min(4, (p.blocks - s * kStageBlocks + 1) / 2);
            if (elect_one()) {
#pragma unroll
                for (int i = 0; i < 4; ++i) copy_scales<1>(cols + i * 4, sc + i * (kScaleTile >> 4));
#pragma unroll
                for (int kk = 0; kk < 4; ++kk)
                    if (kk < steps)
                        mma_mx4<1>(sum, w + kk * 2, t + kk * 2, mx4_idesc(128, TN, kk & 1), cols + (kk >> 1) * 4,
                                   cols + 8 + (kk >> 1) * 4 + token_col, (s > s0 + 1 || kk > 0) ? 1u : 0u);
                tc_commit(smem_u32(&empty[slot]));
            }
            __syncwarp();
            slot += 2;
            if (slot >= G::STAGES) {
                slot -= G::STAGES;
                phase ^= 1;
            }
        }
        if (elect_one()) {
            if (!ok) {
                record_error(p.err, DEV_TIMEOUT_MMA, blockIdx.x);
                *abort_flag = 1;
            }
            tc_commit(smem_u32(done));
        }
    } else {
        const int quad = warp & 3;
        const int count = (int)min((int64_t)TN, p.m - (int64_t)tm * TN);
        const bool got = mbar_wait(smem_u32(done), 0, abort_flag);
        if (!got && lane == 0) {
            record_error(p.err, DEV_TIMEOUT_EPILOGUE, blockIdx.x);
            *abort_flag = 1;
        }
        __syncwarp();
        tc_fence_after();
        float* sums = reinterpret_cast<float*>(smem) + quad * 32 + lane;  // [token][128 columns]; every stage has been read
        const bool two = s1 - s0 > 1;  // the second accumulator was written
        for (int c = 0; c < count && __all_sync(0xffffffffu, got); c += 32) {
            float v[32];
            tmem_ld_32x32(tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)c, v);
            if (two) {
                float u[32];
                tmem_ld_32x32(tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)(TN + c), u);
#pragma unroll
                for (int j = 0; j < 32; ++j) v[j] += u[j];
            }
#pragma unroll
            for (int j = 0; j < 32; ++j) sums[(c + j) * 128] = v[j];
        }
        tc_fence_before();
    }
    __syncwarp();
    // the splits' sums (or this CTA's own) to C: rows of it, four columns a lane
    if (ranks > 1)
        sync_cluster();
    else
        __syncthreads();
    {
        const int64_t row0 = (int64_t)tm * TN, col = (int64_t)tn * 128 + lane * 4;
        const int count = (int)min((int64_t)TN, p.m - row0);
        if (p.out_bf16)
            add_splits<__nv_bfloat16>(p, smem_u32(smem), ranks, rank, warp, kThreads1 / 32, row0, count, col, bias, lane);
        else
            add_splits<float>(p, smem_u32(smem), ranks, rank, warp, kThreads1 / 32, row0, count, col, bias, lane);
    }
    if (ranks > 1) sync_cluster();  // the sums are read before any CTA exits
    __syncthreads();
    if (*abort_flag && threadIdx.x == 0) {
        // copies and MMAs on their way use this CTA's memory: wait, again with a limit, for the last of them
        volatile int never = 0;
        for (int i = max(0, *issued_all - G::STAGES); i < *issued_all; ++i)
            mbar_wait(smem_u32(&full[i % G::STAGES]), (i / G::STAGES) & 1, &never);
        mbar_wait(smem_u32(done), 0, &never);
    }
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(G::TMEM_COLS) : "memory");
    }
}

// ----------------------------------------------------------- two-CTA kernel
// A cluster of two CTAs on a pair of SMs computes 256 tokens by 256 columns of C:
// each CTA holds the codes of 128 of the tokens and of 128 of the columns, the
// pair's MMAs (M = N = 256) read both, and each CTA's TMEM receives its 128 tokens
// for all 256 columns.  Half the bytes from L2 per MMA of a one-CTA tile: a stage is
// 35 KB per CTA for 4 x 128 clocks of MMA.  The scales of all 256 columns are
// needed by both CTAs, so each loads them itself.
//
// Here the tokens are the MMA's M rows, an accumulator lane is a row of C, and a
// thread holds 128 neighbouring elements of it: it stores them as 32-byte sectors,
// 256 bits an instruction, with nothing to wait for afterwards.  (Columns as lanes,
// staged through shared memory for TMA boxes, took 3.3 us a tile against the 2.3 us
// of MMAs that 2048 of k give it to hide in.)
//
// The f32 accumulator takes 256 of the 512 TMEM columns and the scales 24 a stage,
// which leaves no room for a second accumulator: instead the eight epilogue warps
// draw the finished tile into 128 registers a thread and hand the accumulator back
// at once (0.13 us), so the next tile's MMAs wait for that only, not for the stores.
// Persistent: tiles are dealt out round robin, the loads of the next tile run on
// while this one's epilogue stores.
//
// 8192^3, bf16 out: 184 us for a single launch, the tensor pipe 84 % busy; launched
// again and again 183 to 220 us, the clock held down by the 1 kW power limit (154 us
// on matrices of zeros, which draw less).
constexpr int kPairStages = 6;
constexpr int kPairStageBytes = 2 * kWBytes + 6 * kScaleTile;  // codes of T and W, two tiles of T's scales, four of W's
constexpr int kPairSmem = kPairStages * kPairStageBytes + 8 * 512 /* bias of each epilogue warp's columns */ + 256;
constexpr int kPairThreads = 320;  // warps: 0 TMA, 1 MMA (leader), 2-9 epilogue (two to a TMEM lane quadrant)
static_assert(kPairSmem <= 227 * 1024, "shared memory of a CTA");
static_assert(256 + 24 * kPairStages <= 512, "TMEM columns");

__device__ __forceinline__ void tma_pair_2d(uint32_t dst, const CUtensorMap* map, int32_t x, int32_t y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void tma_pair_3d(uint32_t dst, const CUtensorMap* map, int32_t x, int32_t y, int32_t z,
                                            uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void commit_pair(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// Counts bytes off a barrier of this CTA as a copy does that has landed.
__device__ __forceinline__ void complete_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void store_cluster(uint32_t addr, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

// Token tiles in groups of eight, the columns inside: the tiles in flight share operands in L2.
__device__ __forceinline__ void pair_tile(const Mx4Params& p, int t, int& tm, int& tn) {
    const int per = 8 * p.tiles_n, first = t / per * 8, rows = min(8, p.tiles_m - first), in = t % per;
    tm = first + in % rows;
    tn = in / rows;
}

// A 32 x 32 exchange over the warp: lane l's v[i] for lane i's v[l].
__device__ __forceinline__ void transpose32(float (&v)[32], int lane) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < 32; ++i)
            if (!(i & o)) {
                const bool hi = lane & o;
                const float other = __shfl_xor_sync(0xffffffffu, hi ? v[i] : v[i | o], o);
                if (hi)
                    v[i] = other;
                else
                    v[i | o] = other;
            }
}

// 32 rows of 128 columns of C whose rows are not 16-byte aligned: lanes and
// columns change places, so that a warp's 2- or 4-byte stores are neighbours.  The 128
// accumulators and the exchange do not fit 168 registers (some spill): 4096 x 4097 x
// 1024 bf16 36 us, where 4096 columns, aligned, take 18.  c: the first row's; rows, left: how many rows and columns there are from it on.
template <typename T>
__device__ __forceinline__ void store_columns(T* c, int64_t ldc, int64_t rows, int64_t left, const float* bias,
                                              float floor, int lane, float (&v)[4][32]) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        transpose32(v[k], lane);
        const float b = bias[k * 32 + lane];
        T* to = c + k * 32 + lane;
        if (k * 32 + lane < left)
#pragma unroll
            for (int i = 0; i < 32; ++i)
                if (i < rows) store_one(to + i * ldc, at_least(v[k][i] + b, floor));
    }
}

// 128 neighbouring elements of a row of C.  ACCESS: bytes that every 32 of them are
// aligned to (32 or 16; past the row's end element by element).
template <typename T, int ACCESS>
__device__ __forceinline__ void store_row(T* c, int64_t left, const float* bias, float floor, float (&v)[4][32]) {
    constexpr int E = ACCESS / (int)sizeof(T);  // elements of a store
#pragma unroll
    for (int k = 0; k < 128; k += E) {
        float x[E];
#pragma unroll
        for (int i = 0; i < E; i += 4) {
            const float4 b = *reinterpret_cast<const float4*>(bias + k + i);
            const float* y = &v[k / 32][k % 32 + i];
            x[i] = at_least(y[0] + b.x, floor), x[i + 1] = at_least(y[1] + b.y, floor);
            x[i + 2] = at_least(y[2] + b.z, floor), x[i + 3] = at_least(y[3] + b.w, floor);
        }
        if (left >= k + E) {
            uint32_t w[E * sizeof(T) / 4];
#pragma unroll
            for (int i = 0; i < (int)(E * sizeof(T) / 4); ++i) {
                if constexpr (sizeof(T) == 2) {
                    const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
                    w[i] = *reinterpret_cast<const uint32_t*>(&h);
                } else {
                    w[i] = __float_as_uint(x[i]);
                }
            }
            if constexpr (ACCESS == 32)
                asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(c + k), "r"(w[0]), "r"(w[1]),
                             "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                             : "memory");
            else
                *reinterpret_cast<uint4*>(c + k) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
#pragma unroll
            for (int i = 0; i < E; ++i)
                if (k + i < left) store_one(c + k + i, x[i]);
        }
    }
}

// ALIGNED: C's rows are 16-byte aligned.
template <bool ALIGNED>
__global__ void __launch_bounds__(kPairThreads, 1) mx4_pair_kernel(const __grid_constant__ CUtensorMap map_w,
                                                                   const __grid_constant__ CUtensorMap map_t,
                                                                   const __grid_constant__ CUtensorMap map_sw,
                                                                   const __grid_constant__ CUtensorMap map_st,
                                                                   Mx4Params p) {
    constexpr int S = kPairStages;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* smem_w = smem;
    uint8_t* smem_t = smem + S * kWBytes;
    uint8_t* smem_s = smem + 2 * S * kWBytes;  // [stage][T groups 0, 1; columns 0-127 groups 0, 1; columns 128-255]
    float* smem_bias = reinterpret_cast<float*>(smem_s + S * 6 * kScaleTile);  // [epilogue warp][128]
    uint64_t* full = reinterpret_cast<uint64_t*>(smem_bias + 8 * 128);  // leader: both CTAs' bytes of a stage
    uint64_t* empty = full + S;   // each CTA: stage read by the MMAs
    uint64_t* tfull = empty + S;  // each CTA: accumulator complete
    uint64_t* tempty = tfull + 1; // leader: accumulator drawn by both CTAs' epilogues
    uint64_t* drain = tempty + 1;
    uint64_t* told = drain + 1;   // leader: the peer's number of stages is there
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(told + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    volatile int* issued_all = abort_flag + 1;   // stages that this CTA issued, and
    volatile int* issued_peer = issued_all + 1;  // (leader) its peer

    const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
    const uint32_t rank = cta_rank();
    const int cluster = blockIdx.x >> 1, clusters = gridDim.x >> 1;
    const int tiles = p.tiles_m * p.tiles_n;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(smem_u32(&full[s]), 1);
            mbar_init(smem_u32(&empty[s]), 1);
        }
        mbar_init(smem_u32(tfull), 1);
        mbar_init(smem_u32(tempty), 16);  // epilogue warps of both CTAs
        mbar_init(smem_u32(drain), 1);
        mbar_init(smem_u32(told), 1);
        *abort_flag = 0;
        *issued_all = 0;
        fence_barrier_init();
        prefetch_tmap(&map_w);
        prefetch_tmap(&map_t);
        prefetch_tmap(&map_sw);
        prefetch_tmap(&map_st);
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    sync_cluster();
    tc_fence_after();
    const uint32_t tmem = uniform(*tmem_slot);
    pdl_wait();
    pdl_launch_dependents();
    auto raise_abort = [&](int code) {
        record_error(p.err, code, blockIdx.x);
        *abort_flag = 1;
        store_cluster(in_cta(smem_u32((const void*)abort_flag), rank ^ 1u), 1u);
    };

    if (warp == 0) {
        const uint32_t w0 = smem_u32(smem_w), t0 = smem_u32(smem_t), sc0 = smem_u32(smem_s);
        const uint32_t full0 = smem_u32(full), leader_full0 = in_cta(full0, 0), empty0 = smem_u32(empty);
        int slot = 0, phase = 1, issued = 0;
        bool ok = true;
        for (int t = cluster; t < tiles && ok; t += clusters) {
            int tm, tn;
            pair_tile(p, t, tm, tn);
            const int w_row = tn * 256 + (int)rank * 128, t_row = tm * 256 + (int)rank * 128;
            for (int s = 0; s < p.stages; ++s) {
                ok = __all_sync(0xffffffffu, mbar_wait(empty0 + slot * 8, phase, abort_flag));
                if (!ok) break;
                if (elect_one()) {
                    if (rank == 0) mbar_expect_tx(full0 + slot * 8, 2 * kPairStageBytes);
                    const uint32_t bar = leader_full0 + slot * 8, ss = sc0 + slot * 6 * kScaleTile;
                    tma_pair_2d(w0 + slot * kWBytes, &map_w, s * kRowBytes, w_row, bar);
                    tma_pair_2d(t0 + slot * kWBytes, &map_t, s * kRowBytes, t_row, bar);
                    tma_pair_3d(ss, &map_st, 0, s * 2, tm * 2 + (int)rank, bar);
                    tma_pair_3d(ss + 2 * kScaleTile, &map_sw, 0, s * 2, tn * 2, bar);
                }
                __syncwarp();
                ++issued;
                if (++slot == S) {
                    slot = 0;
                    phase ^= 1;
                }
            }
        }
        if (elect_one()) {
            *issued_all = issued;
            if (rank != 0) {
                store_cluster(in_cta(smem_u32((const void*)issued_peer), 0), (uint32_t)issued);
                arrive_cluster(in_cta(smem_u32(told), 0));
            }
            if (!ok) raise_abort(DEV_TIMEOUT_PRODUCER);
        }
    } else if (warp == 1 && rank == 0) {
        const uint64_t w0 = smem_desc(smem_u32(smem_w), 16, 1024), t0 = smem_desc(smem_u32(smem_t), 16, 1024);
        const uint64_t sc0 = scale_desc(smem_u32(smem_s));
        const uint32_t empty0 = smem_u32(empty), empty1 = in_cta(empty0, 1);
        const uint32_t tfull0 = smem_u32(tfull), tfull1 = in_cta(tfull0, 1);
        int slot = 0, phase = 0, done = 0;
        bool ok = true;
        for (int t = cluster; t < tiles && ok; t += clusters, ++done) {
            ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(tempty), (done & 1) ^ 1, abort_flag));
            if (!ok) break;
            tc_fence_after();
            for (int s = 0; s < p.stages; ++s) {
                ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&full[slot]), phase, abort_flag));
                if (!ok) break;
                tc_fence_after();
                const uint64_t wd = w0 + slot * (kWBytes >> 4), td = t0 + slot * (kWBytes >> 4);
                const uint64_t sc = sc0 + slot * (6 * kScaleTile >> 4);
                const uint32_t cols = tmem + 256 + slot * 24;  // T group 0, T group 1, W group 0 (8 wide), W group 1
                const int steps = min(4, (p.blocks - s * kStageBlocks + 1) / 2);
                if (elect_one()) {
#pragma unroll
                    for (int g = 0; g < 2; ++g) {
                        copy_scales<2>(cols + g * 4, sc + g * (kScaleTile >> 4));
                        copy_scales<2>(cols + 8 + g * 8, sc + (2 + g) * (kScaleTile >> 4));
                        copy_scales<2>(cols + 8 + g * 8 + 4, sc + (4 + g) * (kScaleTile >> 4));
                    }
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk)
                        if (kk < steps)
                            mma_mx4<2>(tmem, td + kk * 2, wd + kk * 2, mx4_idesc(256, 256, kk & 1),
                                       cols + (kk >> 1) * 4, cols + 8 + (kk >> 1) * 8, (s > 0 || kk > 0) ? 1u : 0u);
                    commit_pair(empty0 + slot * 8);
                    commit_pair(empty1 + slot * 8);
                }
                __syncwarp();
                if (++slot == S) {
                    slot = 0;
                    phase ^= 1;
                }
            }
            if (!ok) break;
            if (elect_one()) {
                commit_pair(tfull0);
                commit_pair(tfull1);
            }
            __syncwarp();
        }
        if (elect_one()) {
            if (!ok) raise_abort(DEV_TIMEOUT_MMA);
            commit_pair(smem_u32(drain));
            volatile int never = 0;  // a run that gave up waits for its MMAs too: they read both CTAs' memory
            mbar_wait(smem_u32(drain), 0, &never);
        }
    } else if (warp >= 2) {
        const int quad = warp & 3, half = (warp - 2) >> 2;  // lanes, columns
        float* bias = smem_bias + (warp - 2) * 128;
        int done = 0;
        bool ok = true;
        for (int t = cluster; t < tiles; t += clusters, ++done) {
            int tm, tn;
            pair_tile(p, t, tm, tn);
            const int64_t row = (int64_t)tm * 256 + rank * 128 + quad * 32 + lane, col0 = (int64_t)tn * 256 + half * 128;
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int64_t col = col0 + i * 32 + lane;
                bias[i * 32 + lane] = p.bias && col < p.n ? p.bias[col] : 0.0f;
            }
            __syncwarp();
            const bool got = mbar_wait(smem_u32(tfull), done & 1, abort_flag);
            if (!__all_sync(0xffffffffu, got)) {
                ok = false;
                break;
            }
            tc_fence_after();
            float v[4][32];
#pragma unroll
            for (int c = 0; c < 4; ++c)
                tmem_ld_nowait(tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)(half * 128 + c * 32), v[c]);
            tmem_ld_wait(v);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) arrive_cluster(in_cta(smem_u32(tempty), 0));
            const int64_t at = row * p.ldc + col0, left = p.n - col0, rows = p.m - row;
            const float floor = p.relu ? 0.0f : -INFINITY;
            if constexpr (!ALIGNED) {
                const int64_t first = at - lane * p.ldc;
                if (p.out_bf16)
                    store_columns(static_cast<__nv_bfloat16*>(p.c) + first, p.ldc, rows + lane, left, bias, floor, lane, v);
                else
                    store_columns(static_cast<float*>(p.c) + first, p.ldc, rows + lane, left, bias, floor, lane, v);
            } else if (rows > 0) {
                if (p.out_bf16) {
                    __nv_bfloat16* to = static_cast<__nv_bfloat16*>(p.c) + at;
                    if (p.access == 32) store_row<__nv_bfloat16, 32>(to, left, bias, floor, v);
                    else store_row<__nv_bfloat16, 16>(to, left, bias, floor, v);
                } else {
                    float* to = static_cast<float*>(p.c) + at;
                    if (p.access == 32) store_row<float, 32>(to, left, bias, floor, v);
                    else store_row<float, 16>(to, left, bias, floor, v);
                }
            }
        }
        if (!ok && lane == 0) raise_abort(DEV_TIMEOUT_EPILOGUE);
    }
    __syncwarp();
    __syncthreads();
    if (*abort_flag && rank == 0 && threadIdx.x == 0) {
        // the pair's copies complete on the leader's barriers
        volatile int never = 0;
        const bool both = mbar_wait(smem_u32(told), 0, &never);
        asm volatile("fence.acq_rel.cluster;" ::: "memory");
        land_pair(
            S, *issued_all, both ? *issued_peer : *issued_all,
            [&](int slot) { mbar_expect_tx(smem_u32(&full[slot]), kPairStageBytes); },
            [&](int slot) { complete_tx(smem_u32(&full[slot]), kPairStageBytes); },
            [&](int slot, uint32_t phase) { mbar_wait(smem_u32(&full[slot]), phase, &never); });
    }
    tc_fence_before();
    __syncthreads();
    sync_cluster();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

// C = bias (k = 0).
__global__ void bias_kernel(Mx4Params p) {
    pdl_wait();
    pdl_launch_dependents();
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < p.m * p.n; i += (int64_t)gridDim.x * blockDim.x)
    {
        const int64_t at = i / p.n * p.ldc + i % p.n;
        const float v = at_least(p.bias ? p.bias[i % p.n] : 0.0f, p.relu ? 0.0f : -INFINITY);
        if (p.out_bf16)
            store_one(static_cast<__nv_bfloat16*>(p.c) + at, v);
        else
            store_one(static_cast<float*>(p.c) + at, v);
    }
}

// ---------------------------------------------------------------- host side
int encode(CUtensorMap* map, CUtensorMapDataType type, int rank, const void* base, const cuuint64_t* dims,
           const cuuint64_t* strides, const cuuint32_t* box, CUtensorMapSwizzle swizzle) {
    EncodeTiledFn enc = encode_fn();
    if (!enc) return fail(RT_ERR_UNSUPPORTED, "cuTensorMapEncodeTiled is not available from the driver");
    const cuuint32_t ones[3] = {1, 1, 1};
    const CUresult r = enc(map, type, rank, const_cast<void*>(base), dims, strides, box, ones,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(RT_ERR_INVALID, "cuTensorMapEncodeTiled failed (%d)", (int)r);
    return RT_OK;
}

// Codes: rows of row_bytes bytes, box of `rows` x 128 bytes.
int map_codes(CUtensorMap* map, const rt_mx4& q, int rows) {
    const cuuint64_t dims[2] = {(cuuint64_t)q.row_bytes(), (cuuint64_t)q.rows};
    const cuuint64_t strides[1] = {(cuuint64_t)q.row_bytes()};
    const cuuint32_t box[2] = {kRowBytes, (cuuint32_t)rows};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, q.codes, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

// Scales: tiles of 128 words, [row tile][k group]; box of 2 k groups of `tiles` row tiles.
int map_scales(CUtensorMap* map, const rt_mx4& q, int tiles) {
    const cuuint64_t dims[3] = {128, (cuuint64_t)q.groups(), (cuuint64_t)((q.rows + 127) / 128)};
    const cuuint64_t strides[2] = {kScaleTile, (cuuint64_t)(q.groups() * kScaleTile)};
    const cuuint32_t box[3] = {128, 2, (cuuint32_t)tiles};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, q.scales, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE);
}

}  // namespace

int mx4_encode_maps(rt_mx4* q) {
    if (q->rows == 0 || q->k == 0) return RT_OK;
    for (int i = 0; i < 3; ++i) RT_TRY(map_codes(&q->maps.codes[i], *q, 32 << i));
    for (int i = 0; i < 2; ++i) RT_TRY(map_scales(&q->maps.scales[i], *q, 1 + i));
    return RT_OK;
}

namespace {

template <int TN>
int launch_one(rt_ctx* ctx, const rt_mx4& a, const rt_mx4& b, Mx4Params p, int splits, cudaStream_t stream) {
    using G = Geo1<TN>;
    const CUtensorMap &w = b.maps.codes[2], &t = a.maps.codes[TN / 64], &sw = b.maps.scales[0], &st = a.maps.scales[0];
    p.tiles_m = (int)((p.m + TN - 1) / TN);
    p.tiles_n = (int)((p.n + 127) / 128);
    const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n;
    p.stages_per_split = (p.stages + splits - 1) / splits;
    splits = (p.stages + p.stages_per_split - 1) / p.stages_per_split;
    RT_CHECK(tiles * splits <= INT32_MAX, "rt_mx4_matmul: C is too large");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(tiles * splits));
    cfg.blockDim = dim3(kThreads1);
    cfg.dynamicSmemBytes = G::SMEM;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = splits;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ctx->pdl ? 2 : 1;
    RT_CUDA(cudaLaunchKernelEx(&cfg, mx4_kernel<TN>, w, t, sw, st, p));
    count_launch(ctx);
    return RT_OK;
}

int launch_pair(rt_ctx* ctx, const rt_mx4& a, const rt_mx4& b, Mx4Params p, cudaStream_t stream) {
    const CUtensorMap &w = b.maps.codes[2], &t = a.maps.codes[2], &sw = b.maps.scales[1], &st = a.maps.scales[0];
    p.tiles_m = (int)((p.m + 255) / 256);
    p.tiles_n = (int)((p.n + 255) / 256);
    const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n;
    RT_CHECK(tiles <= INT32_MAX, "rt_mx4_matmul: C is too large");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(2 * std::min<int64_t>(tiles, ctx->sm_count / 2)));
    cfg.blockDim = dim3(kPairThreads);
    cfg.dynamicSmemBytes = kPairSmem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ctx->pdl ? 2 : 1;
    RT_CUDA(cudaLaunchKernelEx(&cfg, p.access >= 16 ? mx4_pair_kernel<true> : mx4_pair_kernel<false>, w, t, sw, st, p));
    count_launch(ctx);
    return RT_OK;
}

template <int TN>
int allow_smem() {
    RT_CUDA(cudaFuncSetAttribute(mx4_kernel<TN>, cudaFuncAttributeMaxDynamicSharedMemorySize, Geo1<TN>::SMEM));
    return RT_OK;
}

}  // namespace

int gemm_mx4_init() {
    RT_TRY(allow_smem<32>());
    RT_CUDA(cudaFuncSetAttribute(mx4_pair_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kPairSmem));
    RT_CUDA(cudaFuncSetAttribute(mx4_pair_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, kPairSmem));
    RT_TRY(allow_smem<64>());
    return allow_smem<128>();
}

int launch_gemm_mx4(rt_ctx* ctx, const rt_mx4& a, const rt_mx4& b, const rt_tensor& c, const float* bias, bool relu,
                    cudaStream_t stream) {
    Mx4Params p{};
    p.m = c.rows;
    p.n = c.cols;
    p.blocks = (int)a.blocks();
    p.stages = (int)((a.blocks() + kStageBlocks - 1) / kStageBlocks);
    p.c = c.ptr;
    p.ldc = c.ld;
    p.out_bf16 = c.dtype == RT_BF16;
    p.bias = bias;
    p.relu = relu;
    p.err = ctx->dev_err;
    const uintptr_t rows = reinterpret_cast<uintptr_t>(p.c) | (uintptr_t)(p.ldc * (p.out_bf16 ? 2 : 4));
    p.access = (rows & 31) == 0 ? 32 : (rows & 15) == 0 ? 16 : (rows & 7) == 0 ? 8 : 0;
    RT_CUDA(cudaSetDevice(ctx->device));
    if (p.blocks == 0) {
        RT_CUDA(launch_k(ctx->pdl, bias_kernel, ctx->sm_count * 4, 256, 0, stream, p));
        count_launch(ctx);
        return RT_OK;
    }
    // One-CTA tiles while they fit the device at once, two of 64 tokens to an SM (256 x
    // 8192 x 2048: 7.3 us against 8.4 with pairs), else pairs, which load half as much
    // per MMA (1024 x 4096 x 1024: 7.5 / 11.2; 2048^3: 8.7 / 13.6).  Where most SMs would
    // hold two, one of 128 tokens reads two thirds of the bytes, but has more to do after
    // its last stage: 2047 x 1000 x 8192, 32 stages, 12.3 us / 14.3; 512 x 4096 x 4096, 16
    // stages, 8.6 / 9.5; 256 x 8192 x 2048, 8 stages, 7.1 / 7.3; 2048 x 1024 x 1024, 4
    // stages, 6.2 / 5.8.
    const int tn = p.m <= 32 ? 32 : 64;
    const int64_t tiles = ((p.m + tn - 1) / tn) * ((p.n + 127) / 128), slots = 2 * (int64_t)ctx->sm_count;
    if (tiles > slots) return launch_pair(ctx, a, b, p, stream);
    if (tiles > ctx->sm_count && p.stages > 8 && ((p.m + 127) / 128) * ((p.n + 127) / 128) <= ctx->sm_count)
        return launch_one<128>(ctx, a, b, p, 1, stream);
    // Split k until a CTA has at most 8 stages, within those slots: joining the splits costs
    // about 2 us, and few tiles leave most SMs without work (16 x 1024 x 8192, 32 stages on 8
    // tiles: 5.9 us in four, 8.4 in one; 64 x 1000 x 8192: 7.3 / 9.7; 1024^3, 4 stages: 6.6 in
    // two, 4.9 in one).  With 64 tiles and more fewer splits would do (1 x 8192 x 8192: 8.2 in
    // four, 7.3 in two; 1024 x 1024 x 8192: 11.1 in two, 10.3 in one; both with the operands in
    // L2).
    int splits = 1;
    while (splits < 8 && p.stages > 8 * splits && tiles * splits * 2 <= slots) splits *= 2;
    if (tn == 32) return launch_one<32>(ctx, a, b, p, splits, stream);
    return launch_one<64>(ctx, a, b, p, splits, stream);
}

}  // namespace rt
