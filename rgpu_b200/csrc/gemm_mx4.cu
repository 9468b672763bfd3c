// Product of two block-scaled matrices on the tensor cores, C[m,n] = A[m,k] B[n,k]^T +
// 1 bias (+ ReLU), f32 accumulators in TMEM: microscaled 4-bit matrices (E2M1, an E8M0
// scale per 32 elements, tcgen05.mma kind::mxf4) and 8-bit ones (E4M3, an E8M0 scale per
// 128, kind::mxf8f6f4).  The formats share the kernels: a row is as many bytes a
// stage, only the scales' places differ.
//
// A's rows are called tokens here, T; B's rows are C's columns, W.
//
// A k stage is 128 bytes of codes per row (256 elements in 4 bits, 128 in 8; one
// 128-byte-swizzled TMA box) and its 512-byte scale tiles per 128 rows (two; one), in
// memory already in the
// order that tcgen05.cp spreads over TMEM (32 lanes x 4 columns, repeated in the
// four lane quadrants).  Each shared-memory stage has TMEM columns for its scales
// of its own, so the barrier that frees a stage frees its scales too.  A stage is
// four MMAs of 32 bytes a row.  Boxes past the matrices read
// zeros; MMAs wholly past k are not issued.  In 4 bits an MMA's second scale may lie
// past k's blocks: such bytes are not NaN, so they meet zero codes harmlessly.
#include <algorithm>

#include "landing.cuh"
#include "mx4.cuh"
#include "tc_common.cuh"

namespace rt {
namespace {

using namespace tc;

constexpr int kRowBytes = 128;        // codes of a row in a stage
constexpr int kStageSteps = 4;        // MMAs of a stage, 32 bytes of codes each
constexpr int kWBytes = 128 * kRowBytes;
constexpr int kScaleTile = 512;       // scales of 128 rows x 4 blocks

struct Mx4Params {
    int64_t m, n;                     // C's extents
    int tiles_m, tiles_n;             // token tiles, column tiles
    int steps;                        // MMAs along k
    int stages, stages_per_split;     // k stages in all, and of one split
    void* c;
    int64_t ldc;
    int out_bf16;
    const float* bias;
    int relu;
    int access;                       // bytes that C's rows are aligned to (32, 16, 8, or 0 for less)
    int* err;
};

// The two formats.  GROUPS: scale tiles of 128 rows that a stage needs; scale_group: the
// first of them along k; idesc: instruction descriptor of the stage's kk-th MMA (both
// operands K-major, E8M0 scales; bits 29 and 4 the first scale byte of each TMEM word for
// A and B), tile: the scale tile that it reads.

// kind::mxf4: E2M1 operands, 64 elements an MMA, two scales a row.
struct Mx4 {
    using Matrix = rt_mx4;
    static constexpr int GROUPS = 2;
    static int steps(const rt_mx4& q) { return (int)((q.blocks() + 1) / 2); }
    static __device__ __forceinline__ int scale_group(int stage) { return stage * 2; }
    static __device__ __forceinline__ constexpr int tile(int kk) { return kk >> 1; }
    static __device__ __forceinline__ constexpr uint32_t idesc(int m, int n, int kk, int /*stage*/) {
        return (1u << 7) | (1u << 10)            // A, B: E2M1
               | ((uint32_t)(n >> 3) << 17) | (1u << 23) | ((uint32_t)(m >> 7) << 27)
               | ((uint32_t)((kk & 1) * 2) << 29) | ((uint32_t)((kk & 1) * 2) << 4);
    }
};

// kind::mxf8f6f4: E4M3 operands, 32 elements an MMA, one scale a row.  The instruction
// takes a scale for every 32 elements; a block of 128 is one stage, whose four MMAs read
// the same byte, so a scale tile (four blocks) serves four stages and nothing is
// repeated in memory.  Each stage loads its tile again all the same: 512 bytes beside 16
// KB of codes.
struct Fp8 {
    using Matrix = rt_fp8;
    static constexpr int GROUPS = 1;
    static int steps(const rt_fp8& q) { return (int)((q.k + 31) / 32); }
    static __device__ __forceinline__ int scale_group(int stage) { return stage >> 2; }
    static __device__ __forceinline__ constexpr int tile(int) { return 0; }
    static __device__ __forceinline__ constexpr uint32_t idesc(int m, int n, int /*kk*/, int stage) {
        return ((uint32_t)(n >> 3) << 17) | (1u << 23) | ((uint32_t)(m >> 7) << 27)
               | ((uint32_t)(stage & 3) << 29) | ((uint32_t)(stage & 3) << 4);
    }
};

#define RT_SCALED_MMA(CG, KIND)                                                                                        \
    asm volatile("{\n\t.reg .pred p;\n\t"                                                                             \
                 "setp.ne.b32 p, %6, 0;\n\t"                                                                           \
                 "tcgen05.mma.cta_group::" CG ".kind::" KIND " [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),        \
                 "l"(ad), "l"(bd), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)                                     \
                 : "memory")

template <typename F, int CG>
__device__ __forceinline__ void mma_scaled(uint32_t d, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t sfa,
                                           uint32_t sfb, uint32_t accumulate) {
    if constexpr (F::GROUPS == 2) {
        if constexpr (CG == 1)
            RT_SCALED_MMA("1", "mxf4.block_scale.scale_vec::2X");
        else
            RT_SCALED_MMA("2", "mxf4.block_scale.scale_vec::2X");
    } else {
        if constexpr (CG == 1)
            RT_SCALED_MMA("1", "mxf8f6f4.block_scale.scale_vec::1X");
        else
            RT_SCALED_MMA("2", "mxf8f6f4.block_scale.scale_vec::1X");
    }
}
#undef RT_SCALED_MMA

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
    for (int i = 0; i < 4; ++i) bias[i] = p.bias && col + i < p.n ? p.bias[col + i] : 0.0f;
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
// a stage 0.23 us for 35 KB, 19 TB/s from L2 to all SMs.  In 8 bits one token by 8192 x 8192
// takes 15 us, 10.3 of them the weights' 68 MB.
template <typename F, int TN>
struct Geo1 {
    static constexpr int T_BYTES = TN * kRowBytes;
    static constexpr int S_BYTES = 2 * F::GROUPS * kScaleTile;
    static constexpr int STAGE_BYTES = kWBytes + T_BYTES + S_BYTES;  // codes, scale tiles of either side
    static constexpr int CTAS = TN > 64 ? 1 : 2;  // to an SM
    static constexpr int STAGES = CTAS > 1 ? 4 : 6;
    static constexpr int TMEM_COLS = 512 / CTAS;  // two accumulators of TN, and 16 of scales a stage
    static constexpr int SMEM = STAGES * STAGE_BYTES + 1024 + 256;
    static_assert(2 * TN + 16 * STAGES <= TMEM_COLS, "TMEM columns");
    static_assert(CTAS * SMEM <= 226 * 1024, "shared memory of an SM");
    static_assert(TN * 512 <= STAGES * STAGE_BYTES, "the split sums reuse the stages");
};

constexpr int kThreads1 = 224;  // warps: 0 TMA, 1 MMA, 2-5 epilogue (one TMEM lane quadrant each), 6 MMA

template <typename F, int TN>
__global__ void __launch_bounds__(kThreads1) mx4_kernel(const __grid_constant__ CUtensorMap map_w,
                                                        const __grid_constant__ CUtensorMap map_t,
                                                        const __grid_constant__ CUtensorMap map_sw,
                                                        const __grid_constant__ CUtensorMap map_st, Mx4Params p) {
    using G = Geo1<F, TN>;
    constexpr int NG = F::GROUPS;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* smem_w = smem;
    uint8_t* smem_t = smem + G::STAGES * kWBytes;
    uint8_t* smem_s = smem_t + G::STAGES * G::T_BYTES;  // [stage][W's NG tiles, T's]
    uint64_t* full = reinterpret_cast<uint64_t*>(smem_s + G::STAGES * G::S_BYTES);
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
                const uint32_t bar = full0 + slot * 8, ss = sc0 + slot * G::S_BYTES;
                mbar_expect_tx(bar, G::STAGE_BYTES);
                tma_load_2d(w0 + slot * kWBytes, &map_w, s * kRowBytes, tn * 128, bar);
                tma_load_2d(t0 + slot * G::T_BYTES, &map_t, s * kRowBytes, tm * TN, bar);
                tma_load_3d(ss, &map_sw, 0, F::scale_group(s), tn, bar);
                tma_load_3d(ss + NG * kScaleTile, &map_st, 0, F::scale_group(s), tm * TN / 128, bar);
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
            const uint64_t sc = sc0 + slot * (G::S_BYTES >> 4);
            const uint32_t cols = cols0 + slot * 16;  // scales: W's groups, then (at 8) T's
            const int steps = min(kStageSteps, p.steps - s * kStageSteps);
            if (elect_one()) {
#pragma unroll
                for (int i = 0; i < 2 * NG; ++i)
                    copy_scales<1>(cols + i / NG * 8 + i % NG * 4, sc + i * (kScaleTile >> 4));
#pragma unroll
                for (int kk = 0; kk < kStageSteps; ++kk)
                    if (kk < steps)
                        mma_scaled<F, 1>(sum, w + kk * 2, t + kk * 2, F::idesc(128, TN, kk, s), cols + F::tile(kk) * 4,
                                         cols + 8 + F::tile(kk) * 4 + token_col, (s > s0 + 1 || kk > 0) ? 1u : 0u);
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
// on matrices of zeros, which draw less).  In 8 bits, twice the stages: 340 us for a single
// launch, the tensor pipe 91 % busy, 429 to 443 again and again.
template <typename F>
constexpr int kPairStages = F::GROUPS == 1 ? 5 : 6;  // 8 bits: the sixth's room is the epilogue's
template <typename F>
constexpr int kPairStageBytes = 2 * kWBytes + 3 * F::GROUPS * kScaleTile;  // codes of T and W, a row tile of T's scales, two of W's
// Floats of an epilogue warp's stage, in 8 bits: 32 rows of 128 bytes, and 16 that turn the banks.
constexpr int kStageFloats = 32 * 36;
template <typename F>
constexpr int kStagesBytes = F::GROUPS == 1 ? 8 * kStageFloats * 4 : 0;
template <typename F>
constexpr int kPairSmem = kPairStages<F> * kPairStageBytes<F> + 8 * 512 /* bias of each epilogue warp's columns */ + kStagesBytes<F> + 256;
constexpr int kPairThreads = 320;  // warps: 0 TMA, 1 MMA (leader), 2-9 epilogue (two to a TMEM lane quadrant)
static_assert(kPairSmem<Mx4> <= 227 * 1024 && kPairSmem<Fp8> <= 227 * 1024, "shared memory of a CTA");
static_assert(256 + 24 * kPairStages<Mx4> <= 512, "TMEM columns");

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

// The same through the warp's stage in shared memory, 16 columns at a time: no exchange
// in registers.  4096 x 4097 x 1024 in 8 bits 31 us (f32 out 36; codes of zero), through the exchange above 36 (42).
template <typename T>
__device__ __forceinline__ void store_staged(T* c, int64_t ldc, int64_t rows, int64_t left, const float* bias, float floor,
                                             int lane, const float (&v)[32], float* stage) {
    const int col = lane & 15, first = lane >> 4;
#pragma unroll
    for (int h = 0; h < 32; h += 16) {
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 16; ++j) stage[lane * 17 + j] = v[h + j];
        __syncwarp();
        const float b = bias[h + col];
        T* to = c + h + col + first * ldc;
        const int end = h + col < left ? (int)min((int64_t)32, rows) : 0;
#pragma unroll 4
        for (int r = first; r < end; r += 2, to += 2 * ldc) store_one(to, at_least(stage[r * 17 + col] + b, floor));
    }
}

// N times 32 neighbouring elements of a row of C.  ACCESS: bytes that every 32 of them are
// aligned to (32 or 16; past the row's end element by element).
template <typename T, int ACCESS, int N>
__device__ __forceinline__ void store_row(T* c, int64_t left, const float* bias, float floor, float (&v)[N][32]) {
    constexpr int E = ACCESS / (int)sizeof(T);  // elements of a store
#pragma unroll
    for (int k = 0; k < 32 * N; k += E) {
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

// The same through the warp's stage: full lines of C, 128 bytes of a row, four rows an
// instruction.  The stores above touch 32 rows each.
// 4096 x 4096 x 1024, f32 out: 25 us, with them 29; 8192^3 432, 447 (pairs that split k, half
// of the columns a warp: 21.3, with them 20.6, so those keep them).  c: the
// warp's first row, rows and left: how many there are from there on.
template <typename T>
__device__ __forceinline__ void store_line(T* c, int64_t ldc, int64_t rows, int64_t left, const float* bias, float floor,
                                           int lane, const float (*v)[32], float* stage) {
    constexpr int E = 16 / (int)sizeof(T), V = 128 / (int)sizeof(T);  // elements of an access, of a line
    uint4* mine = reinterpret_cast<uint4*>(stage + lane * 36);
    __syncwarp();
#pragma unroll
    for (int k = 0; k < V; k += E) {
        float x[E];
#pragma unroll
        for (int i = 0; i < E; i += 4) {
            const float4 b = *reinterpret_cast<const float4*>(bias + k + i);
            const float* y = &v[(k + i) / 32][(k + i) % 32];
            x[i] = at_least(y[0] + b.x, floor), x[i + 1] = at_least(y[1] + b.y, floor);
            x[i + 2] = at_least(y[2] + b.z, floor), x[i + 3] = at_least(y[3] + b.w, floor);
        }
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 2) {
                const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t*>(&h);
            } else {
                w[i] = __float_as_uint(x[i]);
            }
        }
        mine[k / E] = make_uint4(w[0], w[1], w[2], w[3]);
    }
    __syncwarp();
    const int first = lane >> 3, at = (lane & 7) * E;
    const int end = (int)max((int64_t)0, min((int64_t)32, rows));
    T* to = c + first * ldc + at;
    if (left >= at + E) {
#pragma unroll 4
        for (int r = first; r < end; r += 4, to += 4 * ldc)
            *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(stage + r * 36 + (lane & 7) * 4);
    } else {
        for (int r = first; r < end; r += 4, to += 4 * ldc)
            for (int i = 0; i < E && at + i < left; ++i) to[i] = reinterpret_cast<const T*>(stage + r * 36)[at + i];
    }
}

template <typename T>
__device__ __forceinline__ void store_lines(T* c, int64_t ldc, int64_t rows, int64_t left, const float* bias, float floor,
                                            int lane, const float (&v)[4][32], float* stage) {
    constexpr int STEP = 4 / (int)sizeof(T);  // blocks of 32 columns in a line
#pragma unroll
    for (int k = 0; k < 4; k += STEP)
        store_line(c + k * 32, ldc, rows, left - k * 32, bias + k * 32, floor, lane, v + k, stage);
}

// A warp's 32 rows (lanes; `row` is the lane's) of N times 32 columns of C from `col` on, the
// way that fits C's alignment and the room for a stage.
template <typename F, typename T, bool ALIGNED, int N>
__device__ __forceinline__ void store_tile(const Mx4Params& p, int64_t row, int64_t col, const float* bias, float floor,
                                           int lane, float (&v)[N][32], float* stage) {
    T* to = static_cast<T*>(p.c) + row * p.ldc + col;
    const int64_t left = p.n - col, rows = p.m - row;
    if constexpr (ALIGNED) {
        if constexpr (F::GROUPS == 1 && N == 4) {
            store_lines(to - lane * p.ldc, p.ldc, rows + lane, left, bias, floor, lane, v, stage);
        } else if (rows > 0) {
            if (p.access == 32) store_row<T, 32>(to, left, bias, floor, v);
            else store_row<T, 16>(to, left, bias, floor, v);
        }
    } else if constexpr (F::GROUPS == 1) {
#pragma unroll
        for (int c = 0; c < N; ++c)
            store_staged(to - lane * p.ldc + c * 32, p.ldc, rows + lane, left - c * 32, bias + c * 32, floor, lane, v[c], stage);
    } else {
        store_columns(to - lane * p.ldc, p.ldc, rows + lane, left, bias, floor, lane, v);
    }
}

// ALIGNED: C's rows are 16-byte aligned.  SPLIT: a cluster is two pairs, which share one
// tile, each half of k.  Each leaves the sums of half of the columns (of every warp's 128, 64) in
// shared memory for the other and adds up the other half, about 2 us.  2047 x 1000 x 8192 in
// 8 bits, f32 out: 21 us, 32 stages of 0.29 us and 11 of launch, set-up, join and stores;
// 128-token tiles in one CTA 24.
template <typename F, bool ALIGNED, bool SPLIT>
__global__ void __launch_bounds__(kPairThreads, 1) mx4_pair_kernel(const __grid_constant__ CUtensorMap map_w,
                                                                   const __grid_constant__ CUtensorMap map_t,
                                                                   const __grid_constant__ CUtensorMap map_sw,
                                                                   const __grid_constant__ CUtensorMap map_st,
                                                                   Mx4Params p) {
    constexpr int S = kPairStages<F>, NG = F::GROUPS, S_BYTES = 3 * NG * kScaleTile;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* smem_w = smem;
    uint8_t* smem_t = smem + S * kWBytes;
    uint8_t* smem_s = smem + 2 * S * kWBytes;  // [stage][T's NG groups; those of columns 0-127; of columns 128-255]
    float* smem_bias = reinterpret_cast<float*>(smem_s + S * S_BYTES);  // [epilogue warp][128]
    float* stages = smem_bias + 8 * 128;  // [epilogue warp][kStageFloats], in 8 bits
    uint64_t* full = reinterpret_cast<uint64_t*>(stages + kStagesBytes<F> / 4);  // leader: both CTAs' bytes of a stage
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
    const uint32_t in_cluster = cta_rank(), rank = in_cluster & 1u, leader = in_cluster - rank;  // rank: in the pair
    constexpr int CTAS = SPLIT ? 4 : 2;  // of a cluster
    const int split = SPLIT ? (int)(in_cluster >> 1) : 0;
    const int cluster = blockIdx.x / CTAS, clusters = gridDim.x / CTAS;
    const int tiles = p.tiles_m * p.tiles_n;
    const int s0 = SPLIT ? split * p.stages_per_split : 0, s1 = SPLIT ? min(p.stages, s0 + p.stages_per_split) : p.stages;
    float* sums = reinterpret_cast<float*>(smem);

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
        store_cluster(in_cta(smem_u32((const void*)abort_flag), in_cluster ^ 1u), 1u);
    };

    float own[2][SPLIT ? 32 : 1];  // SPLIT: an epilogue thread's 64 sums
    if (warp == 0) {
        const uint32_t w0 = smem_u32(smem_w), t0 = smem_u32(smem_t), sc0 = smem_u32(smem_s);
        const uint32_t full0 = smem_u32(full), leader_full0 = in_cta(full0, leader), empty0 = smem_u32(empty);
        int slot = 0, phase = 1, issued = 0;
        bool ok = true;
        for (int t = cluster; t < tiles && ok; t += clusters) {
            int tm, tn;
            pair_tile(p, t, tm, tn);
            const int w_row = tn * 256 + (int)rank * 128, t_row = tm * 256 + (int)rank * 128;
            for (int s = s0; s < s1; ++s) {
                ok = __all_sync(0xffffffffu, mbar_wait(empty0 + slot * 8, phase, abort_flag));
                if (!ok) break;
                if (elect_one()) {
                    if (rank == 0) mbar_expect_tx(full0 + slot * 8, 2 * kPairStageBytes<F>);
                    const uint32_t bar = leader_full0 + slot * 8, ss = sc0 + slot * S_BYTES;
                    tma_pair_2d(w0 + slot * kWBytes, &map_w, s * kRowBytes, w_row, bar);
                    tma_pair_2d(t0 + slot * kWBytes, &map_t, s * kRowBytes, t_row, bar);
                    tma_pair_3d(ss, &map_st, 0, F::scale_group(s), tm * 2 + (int)rank, bar);
                    tma_pair_3d(ss + NG * kScaleTile, &map_sw, 0, F::scale_group(s), tn * 2, bar);
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
                store_cluster(in_cta(smem_u32((const void*)issued_peer), leader), (uint32_t)issued);
                arrive_cluster(in_cta(smem_u32(told), leader));
            }
            if (!ok) raise_abort(DEV_TIMEOUT_PRODUCER);
        }
    } else if (warp == 1 && rank == 0) {
        const uint64_t w0 = smem_desc(smem_u32(smem_w), 16, 1024), t0 = smem_desc(smem_u32(smem_t), 16, 1024);
        const uint64_t sc0 = scale_desc(smem_u32(smem_s));
        const uint32_t empty0 = smem_u32(empty), empty1 = in_cta(empty0, leader + 1);
        const uint32_t tfull0 = smem_u32(tfull), tfull1 = in_cta(tfull0, leader + 1);
        int slot = 0, phase = 0, done = 0;
        bool ok = true;
        for (int t = cluster; t < tiles && ok; t += clusters, ++done) {
            ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(tempty), (done & 1) ^ 1, abort_flag));
            if (!ok) break;
            tc_fence_after();
            for (int s = s0; s < s1; ++s) {
                ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&full[slot]), phase, abort_flag));
                if (!ok) break;
                tc_fence_after();
                const uint64_t wd = w0 + slot * (kWBytes >> 4), td = t0 + slot * (kWBytes >> 4);
                const uint64_t sc = sc0 + slot * (S_BYTES >> 4);
                const uint32_t cols = tmem + 256 + slot * 24;  // T's groups, then (at 8) W's, 8 wide each
                const int steps = min(kStageSteps, p.steps - s * kStageSteps);
                if (elect_one()) {
#pragma unroll
                    for (int g = 0; g < NG; ++g) {
                        copy_scales<2>(cols + g * 4, sc + g * (kScaleTile >> 4));
                        copy_scales<2>(cols + 8 + g * 8, sc + (NG + g) * (kScaleTile >> 4));
                        copy_scales<2>(cols + 8 + g * 8 + 4, sc + (2 * NG + g) * (kScaleTile >> 4));
                    }
#pragma unroll
                    for (int kk = 0; kk < kStageSteps; ++kk)
                        if (kk < steps)
                            mma_scaled<F, 2>(tmem, td + kk * 2, wd + kk * 2, F::idesc(256, 256, kk, s),
                                             cols + F::tile(kk) * 4, cols + 8 + F::tile(kk) * 8,
                                             (s > s0 || kk > 0) ? 1u : 0u);
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
        float *bias = smem_bias + (warp - 2) * 128, *stage = stages + (warp - 2) * kStageFloats;
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
            if (lane == 0) arrive_cluster(in_cta(smem_u32(tempty), leader));
            if constexpr (SPLIT) {
                // the other's 64 columns, [column][row]; every stage has been read
                float* to = sums + half * 64 * 128 + quad * 32 + lane;
#pragma unroll
                for (int j = 0; j < 64; ++j) {
                    to[j * 128] = split ? v[j / 32][j % 32] : v[2 + j / 32][j % 32];
                    if (!split) continue;
                    v[j / 32][j % 32] = v[2 + j / 32][j % 32];  // its own in front
                }
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                    for (int j = 0; j < 32; ++j) own[c][j] = v[c][j];
            } else {
                const float floor = p.relu ? 0.0f : -INFINITY;
                if (p.out_bf16) store_tile<F, __nv_bfloat16, ALIGNED>(p, row, col0, bias, floor, lane, v, stage);
                else store_tile<F, float, ALIGNED>(p, row, col0, bias, floor, lane, v, stage);
            }
        }
        if (!ok && lane == 0) raise_abort(DEV_TIMEOUT_EPILOGUE);
    }
    __syncwarp();
    if constexpr (SPLIT) {
        sync_cluster();
        if (warp >= 2) {
            const int quad = warp & 3, half = (warp - 2) >> 2;
            int tm, tn;
            pair_tile(p, cluster, tm, tn);
            const int64_t row = (int64_t)tm * 256 + rank * 128 + quad * 32 + lane, col0 = (int64_t)tn * 256 + half * 128 + split * 64;
            const float* bias = smem_bias + (warp - 2) * 128 + split * 64;
            float* stage = stages + (warp - 2) * kStageFloats;
            const float floor = p.relu ? 0.0f : -INFINITY;
            const uint32_t from = in_cta(smem_u32(sums + half * 64 * 128 + quad * 32 + lane), in_cluster ^ 2u);
            float y[2][32];
#pragma unroll
            for (int j = 0; j < 64; ++j)
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(y[j / 32][j % 32]) : "r"(from + j * 512) : "memory");
#pragma unroll
            for (int j = 0; j < 64; ++j) y[j / 32][j % 32] += own[j / 32][j % 32];
            if (p.out_bf16) store_tile<F, __nv_bfloat16, ALIGNED>(p, row, col0, bias, floor, lane, y, stage);
            else store_tile<F, float, ALIGNED>(p, row, col0, bias, floor, lane, y, stage);
        }
        __syncwarp();
    }
    __syncthreads();
    if (*abort_flag && rank == 0 && threadIdx.x == 0) {
        // the pair's copies complete on the leader's barriers
        volatile int never = 0;
        const bool both = mbar_wait(smem_u32(told), 0, &never);
        asm volatile("fence.acq_rel.cluster;" ::: "memory");
        land_pair(
            S, *issued_all, both ? *issued_peer : *issued_all,
            [&](int slot) { mbar_expect_tx(smem_u32(&full[slot]), kPairStageBytes<F>); },
            [&](int slot) { complete_tx(smem_u32(&full[slot]), kPairStageBytes<F>); },
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

// Codes: rows of `bytes` bytes, row_bytes apart; box of `rows` x 128 bytes.
int map_codes(CUtensorMap* map, const rt_scaled& q, int64_t bytes, int64_t row_bytes, int rows) {
    const cuuint64_t dims[2] = {(cuuint64_t)bytes, (cuuint64_t)q.rows};
    const cuuint64_t strides[1] = {(cuuint64_t)row_bytes};
    const cuuint32_t box[2] = {kRowBytes, (cuuint32_t)rows};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, q.codes, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

// Scales: tiles of 128 words, [row tile][k group]; box of `along` k groups of `tiles` row tiles.
int map_scales(CUtensorMap* map, const rt_scaled& q, int64_t groups, int along, int tiles) {
    const cuuint64_t dims[3] = {128, (cuuint64_t)groups, (cuuint64_t)((q.rows + 127) / 128)};
    const cuuint64_t strides[2] = {kScaleTile, (cuuint64_t)(groups * kScaleTile)};
    const cuuint32_t box[3] = {128, (cuuint32_t)along, (cuuint32_t)tiles};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, q.scales, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE);
}

int encode_maps(rt_scaled* q, int64_t bytes, int64_t row_bytes, int64_t groups, int along) {
    if (q->rows == 0 || q->k == 0) return RT_OK;
    for (int i = 0; i < 3; ++i) RT_TRY(map_codes(&q->maps.codes[i], *q, bytes, row_bytes, 32 << i));
    for (int i = 0; i < 2; ++i) RT_TRY(map_scales(&q->maps.scales[i], *q, groups, along, 1 + i));
    return RT_OK;
}

}  // namespace

int mx4_encode_maps(rt_mx4* q) { return encode_maps(q, q->row_bytes(), q->row_bytes(), q->groups(), Mx4::GROUPS); }
// The bytes between k and row_bytes lie outside the box: they read as zeros whatever they hold.
int fp8_encode_maps(rt_fp8* q) { return encode_maps(q, q->k, q->row_bytes(), q->groups(), Fp8::GROUPS); }

namespace {

template <typename F, int TN>
int launch_one(rt_ctx* ctx, const rt_scaled& a, const rt_scaled& b, Mx4Params p, int splits, cudaStream_t stream) {
    using G = Geo1<F, TN>;
    // A second tile's scales would begin at an odd TMEM column, which the MMA does not take (a
    // tile of 64 tokens has them at column 0 or 2).
    if (TN == 32) RT_CHECK(p.m <= 32, "block-scaled product: %lld tokens in a tile of 32", (long long)p.m);
    const CUtensorMap &w = b.maps.codes[2], &t = a.maps.codes[TN / 64], &sw = b.maps.scales[0], &st = a.maps.scales[0];
    p.tiles_m = (int)((p.m + TN - 1) / TN);
    p.tiles_n = (int)((p.n + 127) / 128);
    const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n;
    p.stages_per_split = (p.stages + splits - 1) / splits;
    splits = (p.stages + p.stages_per_split - 1) / p.stages_per_split;
    RT_CHECK(tiles * splits <= INT32_MAX, "block-scaled product: C is too large");
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
    RT_CUDA(cudaLaunchKernelEx(&cfg, mx4_kernel<F, TN>, w, t, sw, st, p));
    count_launch(ctx);
    return RT_OK;
}

template <typename F, bool SPLIT = false>
int launch_pair(rt_ctx* ctx, const rt_scaled& a, const rt_scaled& b, Mx4Params p, cudaStream_t stream) {
    const CUtensorMap &w = b.maps.codes[2], &t = a.maps.codes[2], &sw = b.maps.scales[1], &st = a.maps.scales[0];
    p.tiles_m = (int)((p.m + 255) / 256);
    p.tiles_n = (int)((p.n + 255) / 256);
    const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n;
    RT_CHECK(tiles <= INT32_MAX, "block-scaled product: C is too large");
    cudaLaunchConfig_t cfg = {};
    p.stages_per_split = (p.stages + 1) / 2;  // SPLIT: two stages or more
    // persistent, or a cluster for each tile
    cfg.gridDim = dim3((unsigned)(SPLIT ? 4 * tiles : 2 * std::min<int64_t>(tiles, ctx->sm_count / 2)));
    cfg.blockDim = dim3(kPairThreads);
    cfg.dynamicSmemBytes = kPairSmem<F>;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = SPLIT ? 4 : 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ctx->pdl ? 2 : 1;
    RT_CUDA(cudaLaunchKernelEx(&cfg, p.access >= 16 ? mx4_pair_kernel<F, true, SPLIT> : mx4_pair_kernel<F, false, SPLIT>, w, t, sw, st, p));
    count_launch(ctx);
    return RT_OK;
}

template <typename F, int TN>
int allow_smem() {
    RT_CUDA(cudaFuncSetAttribute(mx4_kernel<F, TN>, cudaFuncAttributeMaxDynamicSharedMemorySize, Geo1<F, TN>::SMEM));
    return RT_OK;
}

template <typename F>
int allow_all() {
    RT_TRY((allow_smem<F, 32>()));
    RT_TRY((allow_smem<F, 64>()));
    RT_TRY((allow_smem<F, 128>()));
    RT_CUDA(cudaFuncSetAttribute(mx4_pair_kernel<F, true, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, kPairSmem<F>));
    RT_CUDA(cudaFuncSetAttribute(mx4_pair_kernel<F, false, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, kPairSmem<F>));
    return RT_OK;
}

}  // namespace

int gemm_mx4_init() {
    RT_TRY(allow_all<Mx4>());
    RT_TRY(allow_all<Fp8>());
    RT_CUDA(cudaFuncSetAttribute(mx4_pair_kernel<Fp8, true, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kPairSmem<Fp8>));
    RT_CUDA(cudaFuncSetAttribute(mx4_pair_kernel<Fp8, false, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kPairSmem<Fp8>));
    return RT_OK;
}

namespace {

// The tiles of an 8-bit product of more than 32 tokens and at most two 64-token tiles to an
// SM (`tiles` of them).  A stage is half as deep as in 4 bits, so there are twice as many, and
// the rule is its own; bf16 out, us, operands in L2:
//  - two to an SM: 128-token tiles, one to an SM, from 9 stages on (512 x 4096 x 4096: 12.5, 64 tokens 14.4;
//    2048 x 1000 x 1024, 8 stages: 7.6 / 7.2); from 49 on pairs that split k (2048 x 1000 x 8192:
//    18.5 / 128 tokens 21.1; 512 x 4096 x 8192: 18.7 / 20.6; with 32 stages 13.3 / 11.7)
//  - fewer, but 32 or more of 128 tokens, and more than 32 stages: those, k split until every
//    SM has one (1024 x 1000 x 8192: 13.4 in two, 64 tokens in two 15.0; 256 x 1000 x 8192, 16 such tiles: 10.6 in four / 9.0)
//  - else 64 tokens, k split while a CTA has more than 8 stages and every SM at most one
//    CTA (256 x 4096 x 2048: 6.9 in one, 8.4 in two), two only above 24 stages (128 x 4096 x 8192: 14.2 in four, 16.4
//    in two); in eight only where that leaves half of the SMs idle (128 x 1000 x 8192: 8.6 in four, 9.9 in eight)
int launch_fp8(rt_ctx* ctx, const rt_scaled& a, const rt_scaled& b, const Mx4Params& p, int64_t tiles, cudaStream_t stream) {
    const int64_t sms = ctx->sm_count, tiles128 = ((p.m + 127) / 128) * ((p.n + 127) / 128);
    const int64_t pairs = ((p.m + 255) / 256) * ((p.n + 255) / 256);
    int splits = 1;
    if (tiles > sms) {
        if (p.stages > 48 && p.m >= 256 && pairs * 4 <= sms) return launch_pair<Fp8, true>(ctx, a, b, p, stream);
        if (p.stages > 8 && tiles128 <= sms) return launch_one<Fp8, 128>(ctx, a, b, p, 1, stream);
        return launch_one<Fp8, 64>(ctx, a, b, p, 1, stream);
    }
    if (p.m > 64 && p.stages > 32 && tiles128 >= 32) {
        while (splits < 4 && tiles128 * splits * 2 <= sms) splits *= 2;
        return launch_one<Fp8, 128>(ctx, a, b, p, splits, stream);
    }
    while (splits < 8 && p.stages > 8 * splits &&
           (tiles * splits * (splits == 4 ? 4 : 2) <= sms || (splits < 4 && p.stages > 24 * splits && tiles * splits <= sms)))
        splits *= 2;
    return launch_one<Fp8, 64>(ctx, a, b, p, splits, stream);
}

template <typename F>
int launch_product(rt_ctx* ctx, const typename F::Matrix& a, const typename F::Matrix& b, const rt_tensor& c,
                   const float* bias, bool relu, cudaStream_t stream) {
    Mx4Params p{};
    p.m = c.rows;
    p.n = c.cols;
    p.steps = F::steps(a);
    p.stages = (p.steps + kStageSteps - 1) / kStageSteps;
    p.c = c.ptr;
    p.ldc = c.ld;
    p.out_bf16 = c.dtype == RT_BF16;
    p.bias = bias;
    p.relu = relu;
    p.err = ctx->dev_err;
    const uintptr_t rows = reinterpret_cast<uintptr_t>(p.c) | (uintptr_t)(p.ldc * (p.out_bf16 ? 2 : 4));
    p.access = (rows & 31) == 0 ? 32 : (rows & 15) == 0 ? 16 : (rows & 7) == 0 ? 8 : 0;
    RT_CUDA(cudaSetDevice(ctx->device));
    if (p.steps == 0) {
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
    if (tiles > slots) return launch_pair<F>(ctx, a, b, p, stream);
    if constexpr (F::GROUPS == 1)
        if (tn == 64) return launch_fp8(ctx, a, b, p, tiles, stream);
    if (tiles > ctx->sm_count && p.stages > 8 && ((p.m + 127) / 128) * ((p.n + 127) / 128) <= ctx->sm_count)
        return launch_one<F, 128>(ctx, a, b, p, 1, stream);
    // Split k until a CTA has at most 8 stages, within those slots: joining the splits costs
    // about 2 us, and few tiles leave most SMs without work (16 x 1024 x 8192, 32 stages on 8
    // tiles: 5.9 us in four, 8.4 in one; 64 x 1000 x 8192: 7.3 / 9.7; 1024^3, 4 stages: 6.6 in
    // two, 4.9 in one).  With 64 tiles and more fewer splits would do (1 x 8192 x 8192: 8.2 in
    // four, 7.3 in two; 1024 x 1024 x 8192: 11.1 in two, 10.3 in one; both with the operands in
    // L2).  Products of up to 32 tokens in 8 bits, of twice as many stages, take the same rule; weights from HBM:
    // 1 x 8192 x 8192 14.9 in four, 16.7 in two, 20.5 in eight; 1 x 1000 x 8192 7.7 in eight, 9.0 in four; 8 x 16384 x 2048
    // 9.5 in two, 14.5 in four (4 bits: 10.1, 11.0, 16.4; 6.4, 6.6; 7.3, 12.4 and 6.5 in one).
    int splits = 1;
    while (splits < 8 && p.stages > 8 * splits && tiles * splits * 2 <= slots) splits *= 2;
    if (tn == 32) return launch_one<F, 32>(ctx, a, b, p, splits, stream);
    return launch_one<F, 64>(ctx, a, b, p, splits, stream);
}

}  // namespace

int launch_gemm_mx4(rt_ctx* ctx, const rt_mx4& a, const rt_mx4& b, const rt_tensor& c, const float* bias, bool relu,
                    cudaStream_t stream) {
    return launch_product<Mx4>(ctx, a, b, c, bias, relu, stream);
}

int launch_gemm_fp8(rt_ctx* ctx, const rt_fp8& a, const rt_fp8& b, const rt_tensor& c, const float* bias, bool relu,
                    cudaStream_t stream) {
    return launch_product<Fp8>(ctx, a, b, c, bias, relu, stream);
}

}  // namespace rt
