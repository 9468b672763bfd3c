// Embedding: rows of a table looked up by token and scaled, and the table's gradient.
//
//   y[i,:] = scale * E[tok_i,:]
//   dE[v,:] = scale * sum over i with tok_i = v, in ascending i, of dy[i,:]
//
// A token that is no row of the table (tok_i >= V) is padding: a row of zeros, no gradient.
//
// Backward.  The positions are sorted by token, stably, so that the rows of dy that a row
// of dE sums lie one after another and their order is fixed: no atomic adds floats, the
// same call gives the same bits.  Three ways by how many positions there are:
//  - up to kFew / 2, of narrow tables up to kFew, one launch (few_kernel): every CTA sorts the positions of its own rows
//  - up to kChunk * kMaxCluster the sort takes one cluster (cluster_sort_kernel)
//  - above, passes over launches (digit_*), each of which moves all positions: how often
//    the most frequent token occurs does not decide how evenly a pass is spread
// In the last two piece_kernel and row_kernel sum; the rows of tokens that do not occur are
// written beside the cluster's sort and beside the pieces.  65536 x 1024 bf16 rows of 50257
// tokens as frequent as words: 80 us, 52 of bytes; 2047 x 1000 f32 of 1000: 6.5 us.
//
// Each kernel waits (pdl_wait) for the one before it on the stream before it reads or writes
// anything: only that wait makes what earlier kernels wrote visible, those before the last one too.  Rows that did not
// wait for the pieces, of which they need none, took 6 us of these less.
#include <algorithm>
#include <climits>
#include <type_traits>

#include "internal.h"

namespace rt {
namespace {

constexpr int64_t kMaxWidth = 1 << 22;  // spans fit a grid's second extent

// A lane's N columns (4 or 8) of a warp's span of 32 N.  ACCESS: bytes that the rows are
// aligned to, 32 or 16: neighbouring columns, by accesses of that width; the row's length is
// then a multiple of N, so a lane has all of its columns or none.  0: anything else, a
// warp's accesses are neighbours, column lane + 32 i the lane's i-th.
template <int ACCESS, int N>
struct Columns {
    int64_t first, n;  // the lane's first column, the row's length
    bool on;           // it exists
    __device__ __forceinline__ Columns(int64_t span, int64_t n, int lane)
        : first(span * (32 * N) + lane * (ACCESS ? N : 1)), n(n), on(first < n) {
        if (ACCESS && !on) first = 0;  // reads without a condition; what it reads is not stored
    }
};

// The lane's elements of a row as they lie in memory, to be converted when they are used: a
// load is then not waited for before the next one is issued.
template <typename T, int ACCESS, int N>
struct Lane {
    using C = Columns<ACCESS, N>;
    static constexpr int WORDS = ACCESS ? N * sizeof(T) / 4 : N;
    static constexpr int WIDE = WORDS == 8 && ACCESS == 32 ? 8 : 4;  // words of an access
    uint32_t w[WORDS];

    __device__ __forceinline__ float value(int i) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
        else if constexpr (ACCESS == 0) return __uint_as_float(w[i] << 16);
        else return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    }
    __device__ __forceinline__ void load(const T* row, const C& c) {
        const T* p = row + c.first;
        if constexpr (ACCESS == 0) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                w[i] = 0;
                if (c.first + i * 32 < c.n) {
                    if constexpr (sizeof(T) == 2) w[i] = reinterpret_cast<const unsigned short*>(p)[i * 32];
                    else w[i] = reinterpret_cast<const uint32_t*>(p)[i * 32];
                }
            }
        } else if constexpr (WIDE == 8) {
            asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                         : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                         : "l"(p)
                         : "memory");
        } else {
#pragma unroll
            for (int i = 0; i < WORDS; i += 4) {
                const uint4* q = reinterpret_cast<const uint4*>(p) + i / 4;
                const uint4 u = *q;
                w[i] = u.x, w[i + 1] = u.y, w[i + 2] = u.z, w[i + 3] = u.w;
            }
        }
    }
    static __device__ __forceinline__ void store(T* row, const C& c, const float (&v)[N]) {
        T* p = row + c.first;
        if constexpr (ACCESS == 0) {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (c.first + i * 32 < c.n) {
                    if constexpr (sizeof(T) == 2) p[i * 32] = __float2bfloat16_rn(v[i]);
                    else p[i * 32] = v[i];
                }
        } else if (c.on) {
            uint32_t u[WORDS];
#pragma unroll
            for (int i = 0; i < WORDS; ++i) {
                if constexpr (sizeof(T) == 2) {
                    const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
                    u[i] = *reinterpret_cast<const uint32_t*>(&h);
                } else {
                    u[i] = __float_as_uint(v[i]);
                }
            }
            if constexpr (WIDE == 8)
                asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(u[0]), "r"(u[1]),
                             "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7])
                             : "memory");
            else
#pragma unroll
                for (int i = 0; i < WORDS; i += 4) reinterpret_cast<uint4*>(p)[i / 4] = make_uint4(u[i], u[i + 1], u[i + 2], u[i + 3]);
        }
    }
};

// A CTA's eight warps lie over groups of rows and spans of columns: 2^along of them beside one
// another, so that they read neighbouring parts of the same rows, gridDim.y such groups of
// spans.  Shifts only: a division for each warp's place cost as much as its work.
struct Lay {
    int along;
    dim3 grid;
    Lay(int64_t groups, int64_t spans) : along(0) {
        while (along < 3 && spans % (2 << along) == 0) ++along;
        grid = dim3((unsigned)((groups + (8 >> along) - 1) / (8 >> along)), (unsigned)(spans >> along));
    }
};
__device__ __forceinline__ int64_t lay_group(int along, unsigned block) {
    return ((int64_t)block << (3 - along)) + (threadIdx.x >> (5 + along));
}
__device__ __forceinline__ int64_t lay_span(int along) {
    return ((int64_t)blockIdx.y << along) + ((threadIdx.x >> 5) & ((1 << along) - 1));
}

// --------------------------------------------------------------------- forward
// A warp takes 256 columns of kRows positions, all their reads under way at once.
constexpr int kRows = 4, kLookup = 8;

template <typename TE, typename TY, int ACCESS>
__global__ void __launch_bounds__(256) lookup_kernel(const TE* table, int64_t lde, int64_t vocabulary,
                                                     const uint32_t* tokens, int64_t count, int64_t n,
                                                     int along, float scale, TY* y, int64_t ldy) {
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31;
    const int64_t i0 = lay_group(along, blockIdx.x) * kRows;
    const Columns<ACCESS, kLookup> c(lay_span(along), n, lane);
    const int live = (int)max((int64_t)0, min((int64_t)kRows, count - i0));
    Lane<TE, ACCESS, kLookup> e[kRows];
    bool there[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        const uint32_t token = r < live ? tokens[i0 + r] : 0u;
        there[r] = r < live && token < vocabulary;
        if (there[r]) e[r].load(table + token * lde, c);
    }
    TY* to = y + i0 * ldy;
#pragma unroll
    for (int r = 0; r < kRows; ++r, to += ldy) {
        if (r >= live) break;
        float v[kLookup];
#pragma unroll
        for (int i = 0; i < kLookup; ++i) v[i] = there[r] ? e[r].value(i) * scale : 0.0f;
        Lane<TY, ACCESS, kLookup>::store(to, c, v);
    }
}

// -------------------------------------------------------------------- backward
// The sort's arrays in the workspace, in 32-bit words.  A key is a token, or V for padding.
struct Sort {
    int64_t count, vocabulary;
    int beside;          // eighths of the rows of dE that get their zeros beside the cluster's sort
    int passes;          // by 8 bits of a key
    int ctas;            // of a pass over launches,
    int64_t span;        // and positions of a CTA
    int log_chunk;       // of the positions of a CTA of the cluster
    uint32_t* counts;    // [ctas][256]
    uint32_t* key;       // [count] between passes,
    uint32_t* place;     // [count] and their positions
    uint32_t* token;     // [count] sorted
    uint32_t* position;  // [count]
    uint32_t* start;     // [vocabulary + 1] first of each token in the sorted list
};

__device__ __forceinline__ uint32_t key_of(const Sort& s, const uint32_t* tokens, int64_t i) {
    return min(tokens[i], (uint32_t)s.vocabulary);
}

// cnt[digit] += how many lanes have it; returns the lane's rank: those of this warp before it.
__device__ __forceinline__ uint32_t count_rank(uint32_t* cnt, uint32_t digit, bool there, int lane) {
    const uint32_t same = __match_any_sync(0xffffffffu, there ? digit : 0xffffffffu);
    const int leader = __ffs(same) - 1;
    uint32_t before = 0;
    if (there && lane == leader) {
        before = cnt[digit];
        cnt[digit] = before + __popc(same);
    }
    __syncwarp();
    before = __shfl_sync(0xffffffffu, before, leader);
    return before + __popc(same & ((1u << lane) - 1));
}

// Each warp of a CTA owns neighbouring elements of [0, n) and goes over them in order, 32
// at a time: each(index, key, whether there is one).  Four keys are under way at once.
template <int WARPS, typename Key, typename Each>
__device__ __forceinline__ void in_order(int64_t n, int warp, int lane, Key key, Each each) {
    const int64_t share = (n + WARPS * 32 - 1) / (WARPS * 32) * 32;
    const int64_t begin = min(n, warp * share), end = min(n, begin + share);
    for (int64_t i = begin; i < end; i += 128) {
        uint32_t k[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) k[x] = i + x * 32 + lane < end ? key(i + x * 32 + lane) : 0u;
#pragma unroll
        for (int x = 0; x < 4; ++x)
            if (i + x * 32 < end) each(i + x * 32 + lane, k[x], i + x * 32 + lane < end);
    }
}

// A pass over launches: from the tokens themselves (keys null) or what the pass before
// left, to `to_key` and `to_place`.
struct Pass {
    const uint32_t *tokens, *keys, *places;
    uint32_t *to_key, *to_place;
    int shift;
    __device__ __forceinline__ uint32_t key(const Sort& s, int64_t i) const { return keys ? keys[i] : key_of(s, tokens, i); }
    __device__ __forceinline__ uint32_t place(int64_t i) const { return keys ? places[i] : (uint32_t)i; }
};

// How many positions of each CTA's span have each digit.
__global__ void __launch_bounds__(256) digit_count_kernel(Sort s, Pass p) {
    __shared__ uint32_t cnt[256];
    cnt[threadIdx.x] = 0;
    __syncthreads();
    pdl_wait();
    pdl_launch_dependents();
    const int64_t first = blockIdx.x * s.span, n = min(s.span, s.count - first);
#pragma unroll 4
    for (int64_t i = threadIdx.x; i < n; i += 256) atomicAdd(&cnt[p.key(s, first + i) >> p.shift & 255u], 1u);
    __syncthreads();
    s.counts[(int64_t)blockIdx.x * 256 + threadIdx.x] = cnt[threadIdx.x];
}

// Exclusive sums of v[0..bins) in place, by the whole CTA; sums holds a word a warp.
template <int WARPS>
__device__ __forceinline__ void exclusive(uint32_t* v, int bins, uint32_t* sums) {
    const int each = (bins + WARPS * 32 - 1) / (WARPS * 32), b = min(bins, (int)threadIdx.x * each), e = min(bins, b + each);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t own = 0;
    for (int i = b; i < e; ++i) own += v[i];
    uint32_t in = own;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const uint32_t x = __shfl_up_sync(0xffffffffu, in, o);
        if (lane >= o) in += x;
    }
    if (lane == 31) sums[warp] = in;
    __syncthreads();
    uint32_t run = in - own;
    for (int w = 0; w < warp; ++w) run += sums[w];
    for (int i = b; i < e; ++i) {
        const uint32_t x = v[i];
        v[i] = run;
        run += x;
    }
    __syncthreads();
}

// Moves the positions to their digits' places, in order.  A CTA adds up the CTAs' counts
// itself: with at most 256 of them that is cheaper than a launch that does it once.
__global__ void __launch_bounds__(1024) digit_deal_kernel(Sort s, Pass p) {
    constexpr int WARPS = 32, BINS = 256, PARTS = 4;
    __shared__ uint32_t cnt[WARPS][BINS];
    __shared__ uint32_t base[BINS], own[BINS], sums[WARPS];  // of the whole list; of the CTAs before this one
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, bin = threadIdx.x % BINS;
    for (int i = threadIdx.x; i < WARPS * BINS; i += 1024) cnt[0][i] = 0;
    if (threadIdx.x < BINS) base[bin] = own[bin] = 0;
    __syncthreads();
    pdl_wait();
    pdl_launch_dependents();
    {
        uint32_t all = 0, before = 0;
#pragma unroll 8
        for (int c = threadIdx.x / BINS; c < s.ctas; c += PARTS) {
            const uint32_t x = s.counts[(int64_t)c * BINS + bin];
            all += x;
            if (c < (int)blockIdx.x) before += x;
        }
        atomicAdd(&base[bin], all);
        atomicAdd(&own[bin], before);
    }
    const int64_t first = blockIdx.x * s.span, n = min(s.span, s.count - first);
    auto key = [&](int64_t i) { return p.key(s, first + i); };
    in_order<WARPS>(n, warp, lane, key, [&](int64_t, uint32_t k, bool there) { count_rank(cnt[warp], k >> p.shift & 255u, there, lane); });
    __syncthreads();
    exclusive<WARPS>(base, BINS, sums);
    if (threadIdx.x < BINS) {
        uint32_t run = base[bin] + own[bin];
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const uint32_t x = cnt[w][bin];
            cnt[w][bin] = run;
            run += x;
        }
    }
    __syncthreads();
    in_order<WARPS>(n, warp, lane, key, [&](int64_t i, uint32_t k, bool there) {
        const uint32_t to = count_rank(cnt[warp], k >> p.shift & 255u, there, lane);
        if (there) {
            p.to_key[to] = k;
            p.to_place[to] = p.place(first + i);
        }
    });
}

// Where each token starts in the sorted list: at the places where the key changes, for the
// tokens from the one after the last key to the new one.  Few by the thread that finds
// them, else by a warp, thousands by the CTA.
__global__ void __launch_bounds__(256) starts_kernel(Sort s) {
    __shared__ uint32_t list[257], found;
    if (threadIdx.x == 0) found = 0;
    __syncthreads();
    pdl_wait();
    pdl_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t first = (int64_t)blockIdx.x * 256, i = first + threadIdx.x;
    auto from = [&](int64_t at) { return at ? (int64_t)s.token[at - 1] + 1 : (int64_t)0; };
    auto upto = [&](int64_t at) { return at < s.count ? (int64_t)s.token[at] : s.vocabulary; };
    if (i < s.count) {
        const int64_t b = from(i), e = upto(i);
        if (e - b >= 8)
            list[atomicAdd(&found, 1u)] = threadIdx.x;
        else
            for (int64_t t = b; t <= e; ++t) s.start[t] = (uint32_t)i;
        if (i == s.count - 1) list[atomicAdd(&found, 1u)] = threadIdx.x + 1;  // the tokens behind the last
    }
    __syncthreads();
    for (int g = 0; g < (int)found; ++g) {
        const int64_t at = first + list[g], b = from(at), e = upto(at);
        if (e - b >= 4096)
            for (int64_t t = b + threadIdx.x; t <= e; t += 256) s.start[t] = (uint32_t)at;
        else if (g % 8 == warp)
            for (int64_t t = b + lane; t <= e; t += 32) s.start[t] = (uint32_t)at;
    }
}

// The whole sort in one launch where the positions fit the shared memory of one cluster:
// a CTA holds up to kChunk of them, and passes by 8 bits of the key, the low ones first, move
// them through distributed shared memory.  65536 positions of 50257 tokens: 26 us under a
// profiler, as long as the launches above, but on 16 SMs: the others have fill() meanwhile.
constexpr int kChunk = 4096, kMaxCluster = 16, kStride = 257;  // kStride: counters of a warp, off a bank each

struct ClusterSmem {
    uint2 item[kChunk];  // key, position
    uint32_t cnt[32 * kStride];
    uint32_t hist[256], base[256];
    uint32_t gaps;
};

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t in_cta(const void* p, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    return r;
}
__device__ __forceinline__ uint32_t ld_cluster(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void sync_cluster() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Rows whose tokens do not occur get zeros, by groups of kZeros of them: of eight groups the first `beside` beside
// the sort, the others beside the pieces.  Neighbouring tokens are about as frequent in many vocabularies, so
// neither has one end of the table.
constexpr int kZeros = 32;

// Those beside the sort.  CTA `part` of `parts` marks the tokens of its share of the rows by going over all positions
// itself, so it needs no sort.
constexpr int kMarks = 8192;  // rows at a time

template <int ACCESS>
__device__ __forceinline__ void fill(uint8_t* marks, const uint32_t* tokens, const Sort& s, float* out, int64_t ldo, int64_t n,
                                     uint32_t part, uint32_t parts) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t begin = s.vocabulary * part / parts, end = s.vocabulary * (part + 1) / parts;
    for (int64_t b = begin; b < end; b += kMarks) {
        const uint32_t rows = (uint32_t)min(end - b, (int64_t)kMarks);
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < rows; i += 1024) marks[i] = 0;
        __syncthreads();
        auto mark = [&](uint32_t token) {
            if (token - (uint32_t)b < rows) marks[token - (uint32_t)b] = 1;
        };
        const int64_t lead = min(s.count, (int64_t)((16 - (reinterpret_cast<uintptr_t>(tokens) & 15)) & 15) / 4);
        const int64_t quads = (s.count - lead) / 4;
        const uint4* four = reinterpret_cast<const uint4*>(tokens + lead);
#pragma unroll 8
        for (int64_t i = threadIdx.x; i < quads; i += 1024) {
            const uint4 t = four[i];
            mark(t.x), mark(t.y), mark(t.z), mark(t.w);
        }
        if (threadIdx.x < lead) mark(tokens[threadIdx.x]);
        if (threadIdx.x < s.count - lead - quads * 4) mark(tokens[lead + quads * 4 + threadIdx.x]);
        __syncthreads();
        const float zero[8] = {};
        for (uint32_t r = warp; r < rows; r += 32) {
            if (marks[r] || (int)((b + r) / kZeros % 8) >= s.beside) continue;
            float* row = out + (b + r) * ldo;
            for (int64_t j = 0; j * 256 < n; ++j) Lane<float, ACCESS, 8>::store(row, Columns<ACCESS, 8>(j, n, lane), zero);
        }
    }
}

// The grid's first cluster sorts; the others write zeros on SMs that it leaves idle.
template <int ACCESS>
__global__ void __launch_bounds__(1024) cluster_sort_kernel(Sort s, const uint32_t* tokens, float* out, int64_t ldo, int64_t n) {
    extern __shared__ __align__(16) uint8_t raw[];
    ClusterSmem& m = *reinterpret_cast<ClusterSmem*>(raw);
    pdl_wait();
    pdl_launch_dependents();
    if (blockIdx.x >= cluster_size()) {
        fill<ACCESS>(raw, tokens, s, out, ldo, n, blockIdx.x - cluster_size(), gridDim.x - cluster_size());
        return;
    }
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank(), ranks = cluster_size();
    const int chunk = 1 << s.log_chunk, share = chunk / 32;  // positions of a CTA, of a warp
    const int64_t first = (int64_t)rank * chunk;
    const int live = (int)max((int64_t)0, min((int64_t)chunk, s.count - first));  // positions of this CTA
    uint2 item[4];
    const int slot = warp * share + lane;  // of the thread's first item; the others 32 apart
    auto there = [&](int x) { return x * 32 < share && slot + x * 32 < live; };
#pragma unroll
    for (int x = 0; x < 4; ++x)
        if (there(x)) item[x] = make_uint2(key_of(s, tokens, first + slot + x * 32), (uint32_t)first + slot + x * 32);
    for (int pass = 0; pass < s.passes; ++pass) {
        const int shift = pass * 8;
        for (int i = threadIdx.x; i < 32 * kStride; i += 1024) m.cnt[i] = 0;
        if (pass)
#pragma unroll
            for (int x = 0; x < 4; ++x)
                if (there(x)) item[x] = m.item[slot + x * 32];
        __syncthreads();
        uint32_t before[4];  // of the item's digit: items before it in its warp
#pragma unroll
        for (int x = 0; x < 4; ++x)
            if (x * 32 < share) before[x] = count_rank(m.cnt + warp * kStride, item[x].x >> shift & 255u, there(x), lane);
        __syncthreads();
        // the warps' counters to exclusive sums over the warps: four threads a digit, eight warps each
        const int digit = threadIdx.x >> 2, part = threadIdx.x & 3;
        uint32_t c[8], own = 0;
#pragma unroll
        for (int w = 0; w < 8; ++w) {
            c[w] = m.cnt[(part * 8 + w) * kStride + digit];
            own += c[w];
        }
        uint32_t upto = own;
#pragma unroll
        for (int o = 1; o < 4; o *= 2) {
            const uint32_t x = __shfl_up_sync(0xffffffffu, upto, o);
            if (part >= o) upto += x;
        }
        if (part == 3) m.hist[digit] = upto;
        uint32_t run = upto - own;
#pragma unroll
        for (int w = 0; w < 8; ++w) {
            m.cnt[(part * 8 + w) * kStride + digit] = run;
            run += c[w];
        }
        sync_cluster();  // every CTA's items are in registers, its counts in hist
        uint32_t all = 0, earlier = 0;
#pragma unroll
        for (int i = 0; i < kMaxCluster / 4; ++i) {
            const uint32_t r = part + i * 4;
            const uint32_t x = r < ranks ? ld_cluster(in_cta(&m.hist[digit], r)) : 0u;
            all += x;
            if (r < rank) earlier += x;
        }
#pragma unroll
        for (int o = 1; o < 4; o *= 2) {
            all += __shfl_xor_sync(0xffffffffu, all, o);
            earlier += __shfl_xor_sync(0xffffffffu, earlier, o);
        }
        // exclusive sums over the digits: a warp has eight of them
        uint32_t in = part == 0 ? all : 0u;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const uint32_t x = __shfl_up_sync(0xffffffffu, in, o);
            if (lane >= o) in += x;
        }
        if (lane == 31) m.cnt[warp * kStride + 256] = in;  // the word between two warps' counters
        __syncthreads();
        uint32_t lower = 0;
        if (lane < warp) lower = m.cnt[lane * kStride + 256];
#pragma unroll
        for (int o = 16; o; o /= 2) lower += __shfl_xor_sync(0xffffffffu, lower, o);
        if (part == 0) m.base[digit] = lower + in - all + earlier;
        __syncthreads();
#pragma unroll
        for (int x = 0; x < 4; ++x)
            if (there(x)) {
                const uint32_t d = item[x].x >> shift & 255u, to = m.base[d] + m.cnt[warp * kStride + d] + before[x];
                const uint32_t at = in_cta(&m.item[to & (chunk - 1)], to >> s.log_chunk);
                asm volatile("st.shared::cluster.v2.u32 [%0], {%1, %2};" ::"r"(at), "r"(item[x].x), "r"(item[x].y) : "memory");
            }
        sync_cluster();
    }
    // sorted: token and position out; where tokens start from the places where the key changes
    if (threadIdx.x == 0) m.gaps = 0;
    const uint32_t previous = rank && live ? ld_cluster(in_cta(&m.item[chunk - 1], rank - 1)) : 0u;
    __syncthreads();
    uint32_t* list = m.cnt;  // places of wide gaps
    static_assert(32 * kStride >= kChunk + 1, "every place fits the list");
    for (int i = threadIdx.x; i < live; i += 1024) {
        const uint2 now = m.item[i];
        s.token[first + i] = now.x;
        s.position[first + i] = now.y;
        const int64_t from = first + i == 0 ? 0 : (int64_t)(i ? m.item[i - 1].x : previous) + 1;
        if ((int64_t)now.x - from >= 8)
            list[atomicAdd(&m.gaps, 1u)] = i;
        else
            for (int64_t t = from; t <= now.x; ++t) s.start[t] = (uint32_t)(first + i);
    }
    const bool last = live && first + live == s.count;
    if (last && threadIdx.x == 0) list[atomicAdd(&m.gaps, 1u)] = live;  // the tokens behind the last
    __syncthreads();
    const int gaps = (int)m.gaps;
    for (int g = warp; g < gaps; g += 32) {
        const int i = (int)list[g];
        const int64_t from = first + i == 0 ? 0 : (int64_t)(i ? m.item[i - 1].x : previous) + 1;
        const int64_t to = i < live ? (int64_t)m.item[i].x : s.vocabulary;
        for (int64_t t = from + lane; t <= to; t += 32) s.start[t] = (uint32_t)(first + i);
    }
    sync_cluster();  // a CTA's last item is read by the next one
}

// The sums.  A token that occurs at most kLight times is light: a warp takes 512 bytes' columns
// of `tokens` neighbouring rows of dE, whose positions lie one after another, and writes
// each row once.  The others are heavy: the sorted list is cut into pieces of kCut positions
// (fewer where there are few) whatever the tokens, a warp each; where a heavy run crosses pieces, each leaves a partial
// sum of it, and join() adds these in order.
constexpr int kCut = 64, kLight = 16;

// Columns of a lane: 16 bytes of dy.
template <typename T>
constexpr int kColumns = 16 / (int)sizeof(T);

struct Sums {
    int64_t count, vocabulary, n, spans, width;
    int64_t pieces;
    int beside;  // eighths of the rows that have their zeros, where they are absent; piece_kernel writes the others'
    int cut;  // positions of a piece: kCut, a half or a quarter
    const uint32_t* token;
    const uint32_t* position;
    const uint32_t* start;
    float* partial;  // [pieces][2][width]: the heavy run that began in an earlier piece, the one that began in this one
    float scale;
    int accumulate;
    float* out;
    int64_t ldo;
};

template <int ACCESS, int N>
__device__ __forceinline__ void emit(const Sums& s, uint32_t token, const Columns<ACCESS, N>& c, float (&v)[N]) {
    using L = Lane<float, ACCESS, N>;
    float* row = s.out + token * s.ldo;
    if (s.accumulate) {
        L old;
        old.load(row, c);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = old.value(i) + v[i] * s.scale;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] *= s.scale;
    }
    L::store(row, c, v);
}

// The zeros beside the pieces, a warp a part of a group's rows and a span.
constexpr int kZerosWarp = 8;

template <int ACCESS, int N>
__device__ __forceinline__ void zeros(const Sums& s, int64_t group, int64_t span) {
    const int lane = threadIdx.x & 31;
    constexpr int PARTS = kZeros / kZerosWarp;
    const uint32_t of = 8 - s.beside, at = (uint32_t)(group / PARTS);
    const int64_t t0 = ((int64_t)(at / of) * 8 + s.beside + at % of) * kZeros + group % PARTS * kZerosWarp;
    const Columns<ACCESS, N> c(span, s.n, lane);
    const bool there = lane < kZerosWarp && t0 + lane < s.vocabulary;
    const float zero[N] = {};
    for (uint32_t empty = __ballot_sync(0xffffffffu, there && s.start[t0 + lane] == s.start[t0 + lane + 1]); empty; empty &= empty - 1)
        Lane<float, ACCESS, N>::store(s.out + (t0 + __ffs(empty) - 1) * s.ldo, c, zero);
}

// Heavy runs, a warp a piece and span: their sums where they lie inside it, else partial ones.  The CTAs behind those
// of the pieces write zeros.
template <typename T, int ACCESS>
__global__ void __launch_bounds__(256) piece_kernel(Sums s, const T* dy, int64_t ldy, int along, int piece_blocks) {
    pdl_wait();
    pdl_launch_dependents();
    if ((int)blockIdx.x >= piece_blocks) {
        zeros<ACCESS, kColumns<T>>(s, lay_group(along, blockIdx.x - piece_blocks), lay_span(along));
        return;
    }
    constexpr int N = kColumns<T>, U = 8;  // U: rows of dy under way
    using L = Lane<T, ACCESS, N>;
    const int lane = threadIdx.x & 31;
    const Columns<ACCESS, N> c(lay_span(along), s.n, lane);
    const int64_t real = s.start[s.vocabulary];  // positions that hold a token
    const int64_t piece = lay_group(along, blockIdx.x), p0 = piece * s.cut;
    const int live = (int)max((int64_t)0, min((int64_t)s.cut, real - p0));
    uint32_t token[kCut / 32], row[kCut / 32], begin[kCut / 32], end[kCut / 32];
    uint64_t heavy = 0;  // a bit a position
#pragma unroll
    for (int h = 0; h < kCut / 32; ++h) {
        const bool there = h * 32 + lane < live;
        token[h] = there ? s.token[p0 + h * 32 + lane] : 0u;
        row[h] = there ? s.position[p0 + h * 32 + lane] : 0u;
        begin[h] = s.start[token[h]], end[h] = s.start[token[h] + 1];
        heavy |= (uint64_t)__ballot_sync(0xffffffffu, there && end[h] - begin[h] > kLight) << (32 * h);
    }
    if (!heavy) return;
    auto of = [&](const uint32_t (&v)[kCut / 32], int at) { return __shfl_sync(0xffffffffu, at < 32 ? v[0] : v[1], at & 31); };
    static_assert(kCut == 64, "two positions a lane");
    float sum[N] = {};
    int run = __ffsll((long long)heavy) - 1;  // a position of the run
    uint32_t run_token = of(token, run);
    auto flush = [&]() {
        const int64_t run0 = of(begin, run), run1 = of(end, run);
        if (run0 >= p0 && run1 <= p0 + s.cut)
            emit<ACCESS, N>(s, run_token, c, sum);
        else
            Lane<float, ACCESS, N>::store(s.partial + (piece * 2 + (run0 < p0 ? 0 : 1)) * s.width, c, sum);
    };
    while (heavy) {
        L v[U];
        int at[U];
#pragma unroll
        for (int x = 0; x < U; ++x) {
            at[x] = heavy ? __ffsll((long long)heavy) - 1 : -1;
            heavy &= heavy - 1;
            v[x].load(dy + of(row, max(at[x], 0)) * ldy, c);  // past the last one any row
        }
#pragma unroll
        for (int x = 0; x < U; ++x) {
            if (at[x] < 0) break;
            const uint32_t t = of(token, at[x]);
            if (t != run_token) {
                flush();
                run = at[x];
                run_token = t;
#pragma unroll
                for (int i = 0; i < N; ++i) sum[i] = 0.0f;
            }
#pragma unroll
            for (int i = 0; i < N; ++i) sum[i] += v[x].value(i);
        }
    }
    flush();
}

// Adds the partial sums of the heavy runs that begin in kJoin pieces: a run's second row
// there and the first rows of the pieces that follow. A warp takes a run that lies in
// kAlone pieces at most (17314 x 33 of 593, pieces of 64: 33 us; by the whole CTA, one after another, 38); longer
// ones are dealt out over the CTA's warps in order.
constexpr int kJoin = 8, kAlone = 16;
static_assert(kJoin == 8, "a warp each");

template <int ACCESS, int N>
__device__ __forceinline__ void join(const Sums& s, int64_t piece0, int64_t span) {
    using L = Lane<float, ACCESS, N>;
    __shared__ float part[8][32 * N];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t real = s.start[s.vocabulary];
    const Columns<ACCESS, N> c(span, s.n, lane);
    // every warp looks at the last position of each of the pieces
    const int64_t end = (piece0 + lane + 1) * s.cut;
    uint32_t token = 0;
    int64_t first = 0, next = 0;
    bool begins = lane < kJoin && end < real;
    if (begins) {
        token = s.token[end - 1];
        first = s.start[token], next = s.start[token + 1];
        begins = next > end && first >= end - s.cut && next - first > kLight;
    }
    const int pieces = begins ? (int)((next - 1) / s.cut - (piece0 + lane)) + 1 : 0;  // that the run lies in
    const uint32_t few = __ballot_sync(0xffffffffu, begins && pieces <= kAlone);
    float sum[N];
    auto add = [&](int64_t piece, int b, int e) {
#pragma unroll
        for (int i = 0; i < N; ++i) sum[i] = 0.0f;
        constexpr int U = 32 / N;  // partial sums under way
        for (int q = b; q < e; q += U) {
            L v[U];
#pragma unroll
            for (int x = 0; x < U; ++x) {
                const int at = min(q + x, e - 1);
                v[x].load(s.partial + ((piece + at) * 2 + (at == 0 ? 1 : 0)) * s.width, c);
            }
#pragma unroll
            for (int x = 0; x < U; ++x)
                if (q + x < e) {
#pragma unroll
                    for (int i = 0; i < N; ++i) sum[i] += v[x].value(i);
                }
        }
    };
    if (few >> warp & 1) {
        add(piece0 + warp, 0, __shfl_sync(0xffffffffu, pieces, warp));
        emit<ACCESS, N>(s, __shfl_sync(0xffffffffu, token, warp), c, sum);
    }
    for (uint32_t found = __ballot_sync(0xffffffffu, pieces > kAlone); found; found &= found - 1) {
        const int of = __ffs(found) - 1, count = __shfl_sync(0xffffffffu, pieces, of), each = (count + 7) / 8;
        const int b = min(count, warp * each);
        add(piece0 + of, b, min(count, b + each));
#pragma unroll
        for (int i = 0; i < N; ++i) part[warp][i * 32 + lane] = sum[i];
        __syncthreads();
        if (warp == 0) {
            const int used = (count + each - 1) / each;
            for (int w = 1; w < used; ++w)
#pragma unroll
                for (int i = 0; i < N; ++i) sum[i] += part[w][i * 32 + lane];
            emit<ACCESS, N>(s, __shfl_sync(0xffffffffu, token, of), c, sum);
        }
        __syncthreads();
    }
}

// Light tokens, a warp `tokens` (at most 31) rows of dE and a span; in the CTAs behind those, the joins.
template <typename T, int ACCESS>
__global__ void __launch_bounds__(256, 4) row_kernel(Sums s, const T* dy, int64_t ldy, int along, int tokens,
                                                     int row_blocks) {
    constexpr int N = kColumns<T>, U = 4;  // U: rows of dy under way
    using L = Lane<T, ACCESS, N>;
    pdl_wait();
    // Nothing lets the next kernel launch before this one's CTAs end: the sort of the next call
    // would take 16 SMs whole to wait there.
    if ((int)blockIdx.x >= row_blocks) {
        const unsigned q = blockIdx.x - row_blocks;  // 2^along neighbours take the spans of the same pieces
        join<ACCESS, N>(s, (int64_t)(q >> along) * kJoin, ((int64_t)blockIdx.y << along) + (q & ((1u << along) - 1)));
        return;
    }
    const int lane = threadIdx.x & 31;
    const Columns<ACCESS, N> c(lay_span(along), s.n, lane);
    const int64_t t0 = lay_group(along, blockIdx.x) * tokens;
    if (t0 >= s.vocabulary) return;
    const int64_t token = min(t0 + min(lane, tokens), s.vocabulary);
    const uint32_t first = s.start[token], next = __shfl_down_sync(0xffffffffu, first, 1);
    const uint32_t count = lane < tokens && token < s.vocabulary ? next - first : 0u;
    const uint32_t light = count <= kLight ? count : 0u;
    uint32_t upto = light;  // light positions of the rows up to the lane's
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const uint32_t x = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += x;
    }
    const uint32_t total = __shfl_sync(0xffffffffu, upto, 31);
    float sum[N] = {};
    int run = -1;
    for (uint32_t e0 = 0; e0 < total; e0 += 32) {
        // lane: the e-th light position, of row t0 + of: the first row with upto > e
        const uint32_t e = e0 + lane;
        int of = 0;
#pragma unroll
        for (int step = 16; step; step /= 2) {
            const uint32_t x = __shfl_sync(0xffffffffu, upto, of + step - 1);
            if (x <= e) of += step;
        }
        const uint32_t at = __shfl_sync(0xffffffffu, first, of) + e - (__shfl_sync(0xffffffffu, upto, of) - __shfl_sync(0xffffffffu, light, of));
        const uint32_t position = e < total ? s.position[at] : 0u;
        const int live = (int)min(32u, total - e0);
        for (int g = 0; g < live; g += U) {
            L v[U];
            int t[U];
#pragma unroll
            for (int x = 0; x < U; ++x) {
                t[x] = __shfl_sync(0xffffffffu, of, (g + x) & 31);
                v[x].load(dy + __shfl_sync(0xffffffffu, position, min(g + x, live - 1)) * ldy, c);
            }
#pragma unroll
            for (int x = 0; x < U; ++x) {
                if (g + x >= live) break;
                if (t[x] != run) {
                    if (run >= 0) emit<ACCESS, N>(s, (uint32_t)t0 + run, c, sum);
                    run = t[x];
#pragma unroll
                    for (int i = 0; i < N; ++i) sum[i] = 0.0f;
                }
#pragma unroll
                for (int i = 0; i < N; ++i) sum[i] += v[x].value(i);
            }
        }
    }
    if (run >= 0) emit<ACCESS, N>(s, (uint32_t)t0 + run, c, sum);
}

// Few positions: one launch.  A CTA takes `group` neighbouring rows of dE and a span of columns;
// it goes over all positions, sorts those of its rows in shared memory, and its warps take
// equal shares of them.  A run that crosses shares is joined through shared memory, in order.
constexpr int kFew = 8192, kGroup = 128;

template <typename T, int ACCESS, int WARPS>
__global__ void __launch_bounds__(32 * WARPS, 32 / WARPS) few_kernel(Sums s, const uint32_t* tokens, const T* dy,
                                                  int64_t ldy, int group) {
    constexpr int N = kColumns<T>;
    using L = Lane<T, ACCESS, N>;
    __shared__ uint32_t base[kGroup + 1], sums[WARPS];
    __shared__ uint32_t list[kFew];  // row << 16 | position, sorted
    __shared__ union {
        uint32_t cnt[WARPS][kGroup];
        float part[WARPS - 1][32 * N];  // of the run that began before a warp's share; the first has none
    } m;
    auto& cnt = m.cnt;
    auto& part = m.part;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int i = threadIdx.x; i < WARPS * kGroup; i += 32 * WARPS) cnt[0][i] = 0;
    __syncthreads();
    pdl_wait();
    pdl_launch_dependents();
    const int64_t t0 = (int64_t)blockIdx.x * group;
    const int rows = (int)min((int64_t)group, s.vocabulary - t0);
    const Columns<ACCESS, N> c(blockIdx.y, s.n, lane);
    auto key = [&](int64_t i) { return tokens[i] - (uint32_t)t0; };
    auto mine = [&](uint32_t k, bool there) { return there && k < (uint32_t)rows; };
    in_order<WARPS>(s.count, warp, lane, key, [&](int64_t, uint32_t k, bool there) {
        if (__ballot_sync(0xffffffffu, mine(k, there))) count_rank(cnt[warp], k, mine(k, there), lane);
    });
    __syncthreads();
    if (threadIdx.x <= kGroup) {
        uint32_t all = 0;
        if (threadIdx.x < kGroup)
#pragma unroll
            for (int w = 0; w < WARPS; ++w) all += cnt[w][threadIdx.x];
        base[threadIdx.x] = all;
    }
    __syncthreads();
    exclusive<WARPS>(base, kGroup + 1, sums);
    if (threadIdx.x < kGroup) {
        uint32_t run = base[threadIdx.x];
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const uint32_t x = cnt[w][threadIdx.x];
            cnt[w][threadIdx.x] = run;
            run += x;
        }
    }
    __syncthreads();
    in_order<WARPS>(s.count, warp, lane, key, [&](int64_t i, uint32_t k, bool there) {
        if (!__ballot_sync(0xffffffffu, mine(k, there))) return;
        const uint32_t to = count_rank(cnt[warp], k, mine(k, there), lane);
        if (mine(k, there)) list[to] = k << 16 | (uint32_t)i;
    });
    if (!s.accumulate) {
        const float zero[N] = {};
        for (int r = warp; r < rows; r += WARPS)
            if (base[r] == base[r + 1]) Lane<float, ACCESS, N>::store(s.out + (t0 + r) * s.ldo, c, zero);
    }
    __syncthreads();
    const int total = (int)base[kGroup], each = (total + WARPS - 1) / WARPS;
    const int begin = min(total, warp * each), end = min(total, begin + each);
    float sum[N] = {};
    int run = begin < end ? (int)(list[begin] >> 16) : -1;
    auto flush = [&]() {
        const int run0 = (int)base[run], run1 = (int)base[run + 1];
        if (run0 >= begin && run1 <= end) {
            emit<ACCESS, N>(s, (uint32_t)t0 + run, c, sum);
        } else if (run0 < begin) {
#pragma unroll
            for (int i = 0; i < N; ++i) part[warp - 1][i * 32 + lane] = sum[i];
        }
    };
    // U entries from e on, all of their rows of dy under way at once
    auto add = [&](int e, auto width) {
        constexpr int U = decltype(width)::value;
        L v[U];
        uint32_t entry[U];
#pragma unroll
        for (int x = 0; x < U; ++x) {
            entry[x] = list[min(e + x, end - 1)];
            v[x].load(dy + (entry[x] & 0xffffu) * ldy, c);
        }
#pragma unroll
        for (int x = 0; x < U; ++x) {
            if (e + x >= end) break;
            if ((int)(entry[x] >> 16) != run) {
                flush();
                run = (int)(entry[x] >> 16);
#pragma unroll
                for (int i = 0; i < N; ++i) sum[i] = 0.0f;
            }
#pragma unroll
            for (int i = 0; i < N; ++i) sum[i] += v[x].value(i);
        }
    };
    // Rows of dy under way: eight of aligned f32 (20 bytes spilled at the 64 registers that the SM's 32 warps have each),
    // else four.  Eight aligned bf16 rows spill 84 bytes (4096 x 1024 of 1000, as frequent as words: 15.9 us, four
    // 13.6), eight unaligned ones, a register an element, 328 (4096 x 1001: 38, four, which spill 64, 21.4).
    constexpr int MANY = ACCESS && sizeof(T) == 4 ? 8 : 4;
    int e = begin;
    for (; end - e >= MANY; e += MANY) add(e, std::integral_constant<int, MANY>());
    for (; e < end; e += 3) add(e, std::integral_constant<int, 3>());
    if (run >= 0) flush();
    __syncthreads();
    // the warp in whose share a run begins that goes on, its last one, adds it up
    if (run < 0 || (int)base[run + 1] <= end || (int)base[run] < begin) return;
    for (int w = warp + 1; w < WARPS && w * each < (int)base[run + 1]; ++w)
#pragma unroll
        for (int i = 0; i < N; ++i) sum[i] += part[w - 1][i * 32 + lane];
    emit<ACCESS, N>(s, (uint32_t)t0 + run, c, sum);
}

int bits_of(int64_t v) {
    int b = 0;
    while (v >> b) ++b;
    return b;
}

// Whether few_kernel takes them all: up to kFew / 2 positions always, up to kFew if the table is narrow and so
// short that the CTAs, of which each goes over all positions, fit the device at once, but not so short that a few
// of them have most of the positions (7424 x 128 of 1792: 8.9 us, with the cluster's sort 14.6; 8192 x 100 of 75000: 19 / 32;
// but as frequent as words 8192 x 64 of 1000: 18.2 / 16.5; of 256: 19.1 / 16.4; 8192 x 512 of 5000: 20.8 / 20.1; 8192 x 1024
// of 1000: 23.2 / 20.0).
bool is_few(int64_t count, int64_t vocabulary, int64_t n) {
    return count <= kFew / 2 ||
           (count <= kFew && n <= 256 && vocabulary >= 1000 && (vocabulary + kGroup - 1) / kGroup <= 4 * 148);
}

// The workspace's layout from its sizes; the words it needs.
int64_t lay_out(int64_t count, int64_t vocabulary, int64_t n, Sort* s, Sums* m) {
    s->passes = (std::max(1, bits_of(vocabulary)) + 7) / 8;
    s->count = count;
    s->vocabulary = vocabulary;
    // spans of at least 1024 positions: with more CTAs each would add up more counts
    s->ctas = (int)std::min<int64_t>(256, std::max<int64_t>(1, (count + 1023) / 1024));
    s->span = (count + s->ctas - 1) / s->ctas;
    // Shorter pieces while there are fewer than eight warps for each of the 148 SMs: a warp's reads of a piece wait for one another,
    // but a long run leaves more partial sums.  17314 x 33 of 593: 24 us with 16, 27 with 32, 33 with 64;
    // 65536 x 1024 of 50257: 88, 81 and 80.
    m->cut = kCut;
    while (m->cut > kCut / 4 && (count / m->cut) * ((n + 255) / 256) < 8 * 148) m->cut /= 2;
    m->pieces = (count + m->cut - 1) / m->cut;
    // all 16 CTAs before a CTA takes more than 1024: 16384 x 256 of 4000: 20 us, 4096 each 26; 10000 x 100
    // of 75000: 34 / 55; 32768 x 1024 of 50257: 66 / 69
    s->log_chunk = 10;
    while (s->log_chunk < 12 && count > kMaxCluster << s->log_chunk) ++s->log_chunk;
    m->width = (n + 7) / 8 * 8;
    auto words = [](int64_t v) { return (v + 31) / 32 * 32; };
    int64_t at = 0;
    uint32_t* base = s->counts;
    auto take = [&](int64_t v) {
        uint32_t* p = base + at;
        at += words(v);
        return p;
    };
    if (is_few(count, vocabulary, n)) return words(1);  // few_kernel needs none
    m->partial = reinterpret_cast<float*>(take(m->pieces * 2 * m->width));
    s->token = take(count);
    s->position = take(count);
    s->start = take(vocabulary + 1);
    if (count <= kChunk * kMaxCluster) return at;  // the rest of the sort happens in shared memory
    s->key = take(count);
    s->place = take(count);
    s->counts = take((int64_t)s->ctas * 256);
    return at;
}

int check_backward(int64_t count, int64_t vocabulary, int64_t n) {
    RT_CHECK(count >= 0 && vocabulary >= 0 && n >= 0, "embedding: negative extent");
    RT_CHECK(count <= INT_MAX, "embedding: %lld positions are over 2^31 - 1", (long long)count);
    RT_CHECK(vocabulary <= INT_MAX, "embedding: the gradient of %lld tokens is over 2^31 - 1", (long long)vocabulary);
    RT_CHECK(n <= kMaxWidth, "embedding: %lld columns are over 2^22", (long long)n);
    return RT_OK;
}

// Bytes that every row of t is aligned to, 32 or 16, if rows are whole columns of a lane (n); else 0.
int access_of(const rt_tensor* t, int n) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(t->ptr) | (uintptr_t)(t->ld * (int64_t)dtype_size(t->dtype));
    return t->cols % n ? 0 : (a & 31) == 0 ? 32 : (a & 15) == 0 ? 16 : 0;
}

template <typename TE, typename TY>
int launch_lookup(rt_ctx* ctx, const rt_tensor* table, const rt_tensor* tokens, float scale, rt_tensor* y) {
    const Lay lay((y->rows + kRows - 1) / kRows, (y->cols + 32 * kLookup - 1) / (32 * kLookup));
    const int access = std::min(access_of(table, kLookup), access_of(y, kLookup));
    auto* kernel = access == 32   ? lookup_kernel<TE, TY, 32>
                   : access == 16 ? lookup_kernel<TE, TY, 16>
                                  : lookup_kernel<TE, TY, 0>;
    RT_CUDA(launch_k(ctx->pdl, kernel, lay.grid, 256, 0, ctx->stream, static_cast<const TE*>(table->ptr), table->ld,
                     table->rows, static_cast<const uint32_t*>(tokens->ptr), y->rows, y->cols, lay.along, scale,
                     static_cast<TY*>(y->ptr), y->ld));
    count_launch(ctx);
    return RT_OK;
}

template <typename T, int ACCESS>
int launch_sums(rt_ctx* ctx, const rt_tensor* dy, Sums m) {
    constexpr int SPAN = 32 * kColumns<T>;
    m.spans = (m.n + SPAN - 1) / SPAN;
    // 16 rows a warp where that makes warps enough for every place on the device (65536 x 1024 of 50257:
    // 80 us, with 4 rows 88, with one 121); one, whose chain of reads is the shortest, where the device
    // holds most of the warps at once (7813 x 3979 of 430 bf16: 48 us, with 4 rows 56); else 4
    const int64_t sms = ctx->sm_count;
    const int tokens = m.vocabulary / 16 * m.spans >= sms * 32 ? 16 : m.vocabulary * m.spans < sms * 48 ? 1 : 4;
    const Lay pieces(m.pieces, m.spans), rows((m.vocabulary + tokens - 1) / tokens, m.spans);
    const T* p = static_cast<const T*>(dy->ptr);
    dim3 grid = pieces.grid;
    if (!m.accumulate && m.beside < 8) grid.x += Lay((m.vocabulary + 8 * kZeros - 1) / (8 * kZeros) * (8 - m.beside) * (kZeros / kZerosWarp), m.spans).grid.x;
    RT_CUDA(launch_k(ctx->pdl, piece_kernel<T, ACCESS>, grid, 256, 0, ctx->stream, m, p, dy->ld, pieces.along, (int)pieces.grid.x));
    grid = rows.grid;
    grid.x += (unsigned)((m.pieces + kJoin - 1) / kJoin) << rows.along;
    RT_CUDA(launch_k(ctx->pdl, row_kernel<T, ACCESS>, grid, 256, 0, ctx->stream, m, p, dy->ld, rows.along, tokens,
                     (int)rows.grid.x));
    count_launch(ctx, 2);
    return RT_OK;
}

template <typename T, int ACCESS>
int launch_few(rt_ctx* ctx, const rt_tensor* tokens, const rt_tensor* dy, const Sums& m) {
    constexpr int SPAN = 32 * kColumns<T>;
    const int64_t spans = (m.n + SPAN - 1) / SPAN;
    // So many rows a CTA that the CTAs fit the device at once, 32 warps to an SM: each goes over all positions.
    // 16 warps a CTA if such a number (at most kGroup) exists: they share a frequent token's positions
    // (2047 x 1000 of 1000: 6.7 us, with 8 warps 8.1; 4096 x 1024 of 1000, as frequent as words, bf16: 13.6 / 18.6);
    // else 8, which keep waiting less for one another (1024 x 1024 f32 of 50257: 41 us, with 16 57; 4096 x 1024 bf16: 52 / 53)
    auto ctas = [&](int group) { return (m.vocabulary + group - 1) / group * spans; };
    const bool wide = ctas(kGroup) <= 2 * (int64_t)ctx->sm_count;
    int group = 1;
    while (group < kGroup && ctas(group) > (wide ? 2 : 4) * (int64_t)ctx->sm_count) group *= 2;
    const dim3 grid((unsigned)((m.vocabulary + group - 1) / group), (unsigned)spans);
    RT_CUDA(launch_k(ctx->pdl, wide ? few_kernel<T, ACCESS, 16> : few_kernel<T, ACCESS, 8>, grid, wide ? 512 : 256, 0, ctx->stream, m,
                     static_cast<const uint32_t*>(tokens->ptr), static_cast<const T*>(dy->ptr), dy->ld, group));
    count_launch(ctx);
    return RT_OK;
}

// Rows of dy and dE aligned to 32 bytes, 16 or less; few: positions that one launch handles.
template <typename T>
int launch_sums(rt_ctx* ctx, const rt_tensor* tokens, const rt_tensor* dy, const rt_tensor* dtable, const Sums& m, bool few) {
    int access = std::min(access_of(dy, kColumns<T>), access_of(dtable, kColumns<T>));
    if (!few && (reinterpret_cast<uintptr_t>(m.partial) & 31)) access = std::min(access, 16);
    if (few)
        return access == 32   ? launch_few<T, 32>(ctx, tokens, dy, m)
               : access == 16 ? launch_few<T, 16>(ctx, tokens, dy, m)
                              : launch_few<T, 0>(ctx, tokens, dy, m);
    return access == 32   ? launch_sums<T, 32>(ctx, dy, m)
           : access == 16 ? launch_sums<T, 16>(ctx, dy, m)
                          : launch_sums<T, 0>(ctx, dy, m);
}

// The sort; in one cluster, the rows of dE that no token has beside it.
int launch_sort(rt_ctx* ctx, const uint32_t* t, Sort s, Sums* m, const rt_tensor* dtable) {
    const bool pdl = ctx->pdl;
    if (s.count <= kChunk * kMaxCluster) {
        int ranks = 1;
        while ((int64_t)ranks << s.log_chunk < s.count) ranks *= 2;
        const int access = access_of(dtable, 8);
        auto* kernel = access == 32 ? cluster_sort_kernel<32> : access == 16 ? cluster_sort_kernel<16> : cluster_sort_kernel<0>;
        // Beside the sort as many clusters as the device holds, a CTA with 16 rows or more: it goes over all tokens.
        // Both wait for the memory, so beside the sort lie as many rows as it has time for, the others beside the pieces:
        // half of them or more (8192 x 1024 of 50257: 49 us, all 52, none 59), and 32 MB with 1.5 KB a position (65536 x 1024
        // of 50257: 80 us, all 83, none 90; 65536 x 256 of 128256: 61, half 66, none 74).  Tables below 16 MB
        // have them all beside the pieces (17314 x 33 of 593: 23.4, beside the sort 24.2; 10000 x 100 of 75000,
        // 30 MB: 37.5 / 34.3).
        const int64_t bytes = s.vocabulary * m->n * 4;
        if (!m->accumulate && bytes >= 16 << 20)
            s.beside = (int)std::min<int64_t>(8, std::max<int64_t>(4, ((32 << 20) + s.count * 1536) * 8 / bytes));
        int64_t fills = s.beside ? std::min<int64_t>(ctx->sort_clusters[ranks == 16] - 1, s.vocabulary / (16 * ranks)) : 0;
        if (fills <= 0) fills = s.beside = 0;
        m->beside = s.beside;
        RT_CUDA(launch_cluster(ranks, pdl, kernel, (unsigned)((1 + fills) * ranks), 1024, sizeof(ClusterSmem), ctx->stream, s, t, m->out,
                               m->ldo, m->n));
        count_launch(ctx);
        return RT_OK;
    }
    Pass p{t, nullptr, nullptr, nullptr, nullptr, 0};
    for (int i = 0; i < s.passes; ++i, p.shift += 8) {
        const bool last = (s.passes - 1 - i) % 2 == 0;  // to the arrays that the last pass writes
        p.to_key = last ? s.token : s.key;
        p.to_place = last ? s.position : s.place;
        RT_CUDA(launch_k(pdl, digit_count_kernel, s.ctas, 256, 0, ctx->stream, s, p));
        RT_CUDA(launch_k(pdl, digit_deal_kernel, s.ctas, 1024, 0, ctx->stream, s, p));
        p.keys = p.to_key;
        p.places = p.to_place;
    }
    RT_CUDA(launch_k(pdl, starts_kernel, (unsigned)((s.count + 255) / 256), 256, 0, ctx->stream, s));
    count_launch(ctx, 2 * s.passes + 1);
    return RT_OK;
}

int check_tokens(const char* what, const rt_tensor* tokens, const rt_tensor* rows) {
    RT_CHECK(tokens->dtype == RT_U32 && (tokens->rows == 1 || tokens->cols == 1) &&
                 (tokens->rows == 1 || tokens->ld == 1),
             "%s: tokens must be a packed vector of u32", what);
    RT_CHECK(tokens->rows * tokens->cols == rows->rows, "%s: %lld tokens for %lld rows", what,
             (long long)(tokens->rows * tokens->cols), (long long)rows->rows);
    return RT_OK;
}

}  // namespace

template <int ACCESS>
int allow_sort() {
    RT_CUDA(cudaFuncSetAttribute(cluster_sort_kernel<ACCESS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(ClusterSmem)));
    RT_CUDA(cudaFuncSetAttribute(cluster_sort_kernel<ACCESS>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    return RT_OK;
}

int embedding_init(rt_ctx* ctx) {
    RT_TRY(allow_sort<0>());
    RT_TRY(allow_sort<16>());
    RT_TRY(allow_sort<32>());
    for (int i = 0; i < 2; ++i) {
        cudaLaunchConfig_t cfg = {};
        cudaLaunchAttribute attr;
        cfg.gridDim = dim3(1024);
        cfg.blockDim = dim3(1024);
        cfg.dynamicSmemBytes = sizeof(ClusterSmem);
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim = {8u << i, 1, 1};
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        RT_CUDA(cudaOccupancyMaxActiveClusters(&ctx->sort_clusters[i], cluster_sort_kernel<32>, &cfg));
    }
    return RT_OK;
}

}  // namespace rt

using namespace rt;

extern "C" {

int rt_embedding_forward(rt_ctx* ctx, const rt_tensor* table, const rt_tensor* tokens, float scale, rt_tensor* y) {
    RT_CHECK(ctx && table && tokens && y, "rt_embedding_forward: bad arguments");
    RT_CHECK(table->ctx == ctx && tokens->ctx == ctx && y->ctx == ctx, "tensor belongs to another context");
    RT_CHECK(table->dtype != RT_U32 && y->dtype != RT_U32, "rt_embedding_forward: table and y must be f32 or bf16");
    RT_CHECK(table->cols == y->cols, "rt_embedding_forward: table is %lldx%lld, y %lldx%lld", (long long)table->rows,
             (long long)table->cols, (long long)y->rows, (long long)y->cols);
    RT_TRY(check_tokens("rt_embedding_forward", tokens, y));
    RT_CHECK(y->cols <= kMaxWidth && y->rows <= (int64_t)1 << 32, "rt_embedding_forward: y %lldx%lld is over 2^32 x 2^22",
             (long long)y->rows, (long long)y->cols);
    if (y->rows == 0 || y->cols == 0) return RT_OK;
    RT_CUDA(cudaSetDevice(ctx->device));
    if (table->dtype == RT_BF16)
        return y->dtype == RT_BF16 ? launch_lookup<__nv_bfloat16, __nv_bfloat16>(ctx, table, tokens, scale, y)
                                   : launch_lookup<__nv_bfloat16, float>(ctx, table, tokens, scale, y);
    return y->dtype == RT_BF16 ? launch_lookup<float, __nv_bfloat16>(ctx, table, tokens, scale, y)
                               : launch_lookup<float, float>(ctx, table, tokens, scale, y);
}

int64_t rt_embedding_backward_workspace(int64_t count, int64_t vocabulary, int64_t n) {
    if (check_backward(count, vocabulary, n) != RT_OK) return -1;
    Sort s{};
    Sums m{};
    return lay_out(count, vocabulary, n, &s, &m);
}

int rt_embedding_backward(rt_ctx* ctx, const rt_tensor* tokens, const rt_tensor* dy, float scale, int accumulate,
                          rt_tensor* dtable, rt_tensor* work) {
    RT_CHECK(ctx && tokens && dy && dtable && work, "rt_embedding_backward: bad arguments");
    RT_CHECK(tokens->ctx == ctx && dy->ctx == ctx && dtable->ctx == ctx && work->ctx == ctx,
             "tensor belongs to another context");
    RT_CHECK(dy->dtype != RT_U32, "rt_embedding_backward: dy must be f32 or bf16");
    RT_CHECK(dtable->dtype == RT_F32, "rt_embedding_backward: dtable must be f32");
    RT_CHECK(dtable->cols == dy->cols, "rt_embedding_backward: dy is %lldx%lld, dtable %lldx%lld", (long long)dy->rows,
             (long long)dy->cols, (long long)dtable->rows, (long long)dtable->cols);
    RT_TRY(check_tokens("rt_embedding_backward", tokens, dy));
    RT_TRY(check_backward(dy->rows, dtable->rows, dy->cols));
    Sort s{};
    Sums m{};
    s.counts = static_cast<uint32_t*>(work->ptr);
    const int64_t need = lay_out(dy->rows, dtable->rows, dy->cols, &s, &m);
    RT_CHECK(work->dtype == RT_F32 && (work->rows <= 1 || work->ld == work->cols) && work->rows * work->cols >= need &&
                 (reinterpret_cast<uintptr_t>(work->ptr) & 15) == 0,
             "rt_embedding_backward: work must be %lld packed f32, 16-byte aligned", (long long)need);
    if (dtable->rows == 0 || dtable->cols == 0) return RT_OK;
    RT_CUDA(cudaSetDevice(ctx->device));
    m.count = s.count;
    m.vocabulary = s.vocabulary;
    m.n = dy->cols;
    m.token = s.token;
    m.position = s.position;
    m.start = s.start;
    m.scale = scale;
    m.accumulate = accumulate != 0;
    m.out = static_cast<float*>(dtable->ptr);
    m.ldo = dtable->ld;
    const bool few = is_few(s.count, s.vocabulary, m.n);
    if (!few) RT_TRY(launch_sort(ctx, static_cast<const uint32_t*>(tokens->ptr), s, &m, dtable));
    return dy->dtype == RT_BF16 ? launch_sums<__nv_bfloat16>(ctx, tokens, dy, dtable, m, few)
                                : launch_sums<float>(ctx, tokens, dy, dtable, m, few);
}

}  // extern "C"
