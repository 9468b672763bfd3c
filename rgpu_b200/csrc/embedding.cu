// Embedding: rows of a table looked up by token and scaled, and the table's gradient.
//
//   y[i,:] = scale * E[tok_i,:]
//   dE[v,:] = scale * sum over i with tok_i = v, in ascending i, of dy[i,:]
//
// A token that is no row of the table (tok_i >= V) is padding: a row of zeros, no gradient.
//
// Backward.  The positions are sorted by token, stably, so that the rows of dy that a row
// of dE sums lie one after another and their order is fixed: no atomic adds floats, the
// same call gives the same bits.  Keys have at most 21 bits, so one pass over the high bits
// deals the positions out to buckets and a CTA a bucket finishes by the low bits in
// shared memory.  The sorted list is cut into pieces of kCut positions whatever the
// tokens: how often the most frequent token occurs then does not decide how evenly the work is
// spread.  A run of one token inside a piece goes to dE at once; one that crosses
// pieces leaves a partial sum in each, which a second kernel adds in order.
#include <algorithm>
#include <climits>

#include "internal.h"

namespace rt {
namespace {

constexpr int kVec = 8;               // elements of a lane
constexpr int kSpan = 32 * kVec;      // and of a warp
constexpr int64_t kMaxVocabulary = (1 << 21) - 1;  // keys 0 .. V fit 21 bits

// A lane's eight neighbouring elements.  ALIGNED: by 16-byte accesses where all eight exist
// (rows on 16 bytes); else a warp's accesses are neighbours, element lane + 32 i the i-th.
template <typename T, bool ALIGNED>
struct Lane {
    static __device__ __forceinline__ int64_t at(int64_t j0, int i, int lane) {
        return ALIGNED ? j0 + lane * kVec + i : j0 + i * 32 + lane;
    }
    static __device__ __forceinline__ float one(const T* p) {
        if constexpr (sizeof(T) == 2) return __bfloat162float(*p);
        else return *p;
    }
    static __device__ __forceinline__ void put(T* p, float v) {
        if constexpr (sizeof(T) == 2) *p = __float2bfloat16_rn(v);
        else *p = v;
    }
    // of row p, from column j0 on, of n; NC: the kernel writes no row of p's matrix
    template <bool NC = true>
    static __device__ __forceinline__ void load(const T* p, int64_t j0, int64_t n, int lane, float (&v)[kVec]) {
        const int64_t j = j0 + lane * kVec;
        if (ALIGNED && j + kVec <= n) {
            if constexpr (sizeof(T) == 2) {
                const uint4 u = __ldg(reinterpret_cast<const uint4*>(p + j));
                const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            } else {
                const float4* f = reinterpret_cast<const float4*>(p + j);
                const float4 a = NC ? __ldg(f) : f[0], b = NC ? __ldg(f + 1) : f[1];
                v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < kVec; ++i) v[i] = at(j0, i, lane) < n ? one(p + at(j0, i, lane)) : 0.0f;
        }
    }
    static __device__ __forceinline__ void store(T* p, int64_t j0, int64_t n, int lane, const float (&v)[kVec]) {
        const int64_t j = j0 + lane * kVec;
        if (ALIGNED && j + kVec <= n) {
            if constexpr (sizeof(T) == 2) {
                uint32_t w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
                    w[i] = *reinterpret_cast<const uint32_t*>(&h);
                }
                *reinterpret_cast<uint4*>(p + j) = make_uint4(w[0], w[1], w[2], w[3]);
            } else {
                reinterpret_cast<float4*>(p + j)[0] = make_float4(v[0], v[1], v[2], v[3]);
                reinterpret_cast<float4*>(p + j)[1] = make_float4(v[4], v[5], v[6], v[7]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < kVec; ++i)
                if (at(j0, i, lane) < n) put(p + at(j0, i, lane), v[i]);
        }
    }
};

// --------------------------------------------------------------------- forward
// A warp takes kSpan columns of kRows positions, all their reads under way at once.
constexpr int kRows = 4;

template <typename TE, typename TY, bool ALIGNED>
__global__ void __launch_bounds__(256) lookup_kernel(const TE* __restrict__ table, int64_t lde, int64_t vocabulary,
                                                     const uint32_t* __restrict__ tokens, int64_t count, int64_t n,
                                                     int64_t spans, float scale, TY* __restrict__ y, int64_t ldy) {
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31;
    const int64_t units = (count + kRows - 1) / kRows * spans;
    for (int64_t u = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); u < units; u += (int64_t)gridDim.x * 8) {
        const int64_t i0 = u / spans * kRows, j0 = u % spans * kSpan;
        float v[kRows][kVec];
        bool there[kRows];
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            const uint32_t token = i0 + r < count ? __ldg(tokens + i0 + r) : 0u;
            there[r] = i0 + r < count && token < vocabulary;
            if (there[r]) Lane<TE, ALIGNED>::load(table + token * lde, j0, n, lane, v[r]);
        }
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            if (i0 + r >= count) break;
#pragma unroll
            for (int i = 0; i < kVec; ++i) v[r][i] = there[r] ? v[r][i] * scale : 0.0f;
            Lane<TY, ALIGNED>::store(y + (i0 + r) * ldy, j0, n, lane, v[r]);
        }
    }
}

// -------------------------------------------------------------------- backward
// The workspace, in 32-bit words.  B: CTAs of the first pass; bins: buckets; a run's
// partial sums: two rows of `width` floats (n rounded up to kVec) a piece.
struct Sort {
    int64_t count, vocabulary;
    int low, high;       // bits of a key: bucket high, order in it low
    int ctas;            // of the first pass
    int64_t span;        // positions of a CTA
    uint32_t* counts;    // [ctas][bins]
    uint32_t* bucket;    // [bins + 1] first position of each bucket
    uint32_t* key;       // [count] keys in bucket order
    uint32_t* place;     // [count] and their positions
    uint32_t* token;     // [count] sorted
    uint32_t* position;  // [count]
    uint32_t* start;     // [vocabulary + 1] first of each token in the sorted list
};

constexpr int kSortThreads = 256, kSortWarps = 8;
constexpr int kMaxHigh = 11, kMaxLow = 10;

__device__ __forceinline__ uint32_t key_of(const Sort& s, const uint32_t* tokens, int64_t i) {
    return min(__ldg(tokens + i), (uint32_t)s.vocabulary);
}

// Each warp of a CTA owns neighbouring elements of [first, first + n) and a row of
// counters; both passes below go over them 32 at a time, in order.
struct Share {
    int64_t begin, end;
    __device__ __forceinline__ Share(int64_t n, int warp) {
        const int64_t each = (n + kSortWarps * 32 - 1) / (kSortWarps * 32) * 32;
        begin = min(n, warp * each);
        end = min(n, begin + each);
    }
};

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

// How many positions of each CTA's span fall in each bucket.
__global__ void __launch_bounds__(kSortThreads) bucket_count_kernel(Sort s, const uint32_t* __restrict__ tokens) {
    extern __shared__ uint32_t cnt[];
    pdl_wait();
    pdl_launch_dependents();
    const int bins = 1 << s.high;
    for (int i = threadIdx.x; i < bins; i += kSortThreads) cnt[i] = 0;
    __syncthreads();
    const int64_t first = blockIdx.x * s.span, n = min(s.span, s.count - first);
    for (int64_t i = threadIdx.x; i < n; i += kSortThreads) atomicAdd(&cnt[key_of(s, tokens, first + i) >> s.low], 1u);
    __syncthreads();
    for (int i = threadIdx.x; i < bins; i += kSortThreads) s.counts[(int64_t)blockIdx.x * bins + i] = cnt[i];
}

// Exclusive sums of v[0..bins) in place, by the whole CTA (bins a multiple of nothing in particular).
__device__ __forceinline__ void exclusive(uint32_t* v, int bins, uint32_t* sums) {
    const int each = (bins + kSortThreads - 1) / kSortThreads, b = threadIdx.x * each, e = min(bins, b + each);
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

// Deals the positions out to their buckets, in order.  A CTA adds up the other CTAs'
// counts itself.
__global__ void __launch_bounds__(kSortThreads) bucket_deal_kernel(Sort s, const uint32_t* __restrict__ tokens) {
    extern __shared__ uint32_t shared[];
    const int bins = 1 << s.high;
    uint32_t* base = shared;              // [bins]
    uint32_t* cnt = shared + bins;        // [warps][bins]
    __shared__ uint32_t sums[kSortWarps];
    pdl_wait();
    pdl_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int b = threadIdx.x; b < bins; b += kSortThreads) {
        uint32_t all = 0, before = 0;
        for (int c = 0; c < s.ctas; ++c) {
            const uint32_t x = s.counts[(int64_t)c * bins + b];
            if (c < (int)blockIdx.x) before += x;
            all += x;
        }
        base[b] = all;
        cnt[b] = before;
#pragma unroll
        for (int w = 1; w < kSortWarps; ++w) cnt[w * bins + b] = 0;
    }
    __syncthreads();
    exclusive(base, bins, sums);
    for (int b = threadIdx.x; b < bins; b += kSortThreads) {
        if (blockIdx.x == 0) s.bucket[b] = base[b];
        base[b] += cnt[b];
        cnt[b] = 0;
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) s.bucket[bins] = (uint32_t)s.count;
    __syncthreads();
    const int64_t first = blockIdx.x * s.span, n = min(s.span, s.count - first);
    const Share own(n, warp);
    uint32_t* mine = cnt + warp * bins;
    for (int64_t i = own.begin; i < own.end; i += 32) {
        const bool there = i + lane < own.end;
        count_rank(mine, there ? key_of(s, tokens, first + i + lane) >> s.low : 0u, there, lane);
    }
    __syncthreads();
    for (int b = threadIdx.x; b < bins; b += kSortThreads) {
        uint32_t run = base[b];
#pragma unroll
        for (int w = 0; w < kSortWarps; ++w) {
            const uint32_t x = cnt[w * bins + b];
            cnt[w * bins + b] = run;
            run += x;
        }
    }
    __syncthreads();
    for (int64_t i = own.begin; i < own.end; i += 32) {
        const bool there = i + lane < own.end;
        const uint32_t key = there ? key_of(s, tokens, first + i + lane) : 0u;
        const uint32_t to = count_rank(mine, key >> s.low, there, lane);
        if (there) {
            s.key[to] = key;
            s.place[to] = (uint32_t)(first + i + lane);
        }
    }
}

// Sorts a bucket by the low bits and writes where each of its tokens starts.
__global__ void __launch_bounds__(kSortThreads) bucket_sort_kernel(Sort s) {
    extern __shared__ uint32_t shared[];
    const int bins = 1 << s.low;
    uint32_t* base = shared;        // [bins]
    uint32_t* cnt = shared + bins;  // [warps][bins]
    __shared__ uint32_t sums[kSortWarps];
    pdl_wait();
    pdl_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t first = s.bucket[blockIdx.x], n = s.bucket[blockIdx.x + 1] - first;
    for (int b = threadIdx.x; b < bins * kSortWarps; b += kSortThreads) cnt[b] = 0;
    __syncthreads();
    const Share own(n, warp);
    uint32_t* mine = cnt + warp * bins;
    const uint32_t mask = (uint32_t)bins - 1;
    for (int64_t i = own.begin; i < own.end; i += 32) {
        const bool there = i + lane < own.end;
        count_rank(mine, there ? s.key[first + i + lane] & mask : 0u, there, lane);
    }
    __syncthreads();
    for (int b = threadIdx.x; b < bins; b += kSortThreads) {
        uint32_t all = 0;
#pragma unroll
        for (int w = 0; w < kSortWarps; ++w) all += cnt[w * bins + b];
        base[b] = all;
    }
    __syncthreads();
    exclusive(base, bins, sums);
    for (int b = threadIdx.x; b < bins; b += kSortThreads) {
        uint32_t run = (uint32_t)first + base[b];
        const int64_t token = ((int64_t)blockIdx.x << s.low) + b;
        if (token <= s.vocabulary) s.start[token] = run;
#pragma unroll
        for (int w = 0; w < kSortWarps; ++w) {
            const uint32_t x = cnt[w * bins + b];
            cnt[w * bins + b] = run;
            run += x;
        }
    }
    __syncthreads();
    for (int64_t i = own.begin; i < own.end; i += 32) {
        const bool there = i + lane < own.end;
        const uint32_t key = there ? s.key[first + i + lane] : 0u, place = there ? s.place[first + i + lane] : 0u;
        const uint32_t to = count_rank(mine, key & mask, there, lane);
        if (there) {
            s.token[to] = key;
            s.position[to] = place;
        }
    }
}

// The sums.  A warp takes kSpan columns of a piece of kCut positions, or of 32 rows of dE
// that are looked over for tokens that do not occur.
constexpr int kCut = 64, kEmpty = 32;

struct Sums {
    int64_t count, vocabulary, n, spans, width;
    int64_t pieces;
    const uint32_t* token;
    const uint32_t* position;
    const uint32_t* start;
    float* partial;  // [pieces][2][width]: the run that began in an earlier piece, the one that goes on in the next
    float scale;
    int accumulate;
    float* out;
    int64_t ldo;
};

template <bool ALIGNED>
__device__ __forceinline__ void emit(const Sums& s, uint32_t token, int64_t j0, int lane, float (&v)[kVec]) {
    float* row = s.out + token * s.ldo;
    float old[kVec];
    if (s.accumulate) Lane<float, ALIGNED>::template load<false>(row, j0, s.n, lane, old);
#pragma unroll
    for (int i = 0; i < kVec; ++i) v[i] = s.accumulate ? old[i] + v[i] * s.scale : v[i] * s.scale;
    Lane<float, ALIGNED>::store(row, j0, s.n, lane, v);
}

template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(256) sum_kernel(Sums s, const T* __restrict__ dy, int64_t ldy, int64_t units,
                                                  int64_t piece_units) {
    pdl_wait();
    pdl_launch_dependents();
    constexpr int U = sizeof(T) == 2 ? 8 : 4;  // rows of dy under way
    const int lane = threadIdx.x & 31;
    const int64_t real = s.start[s.vocabulary];  // positions that hold a token
    for (int64_t u = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); u < units; u += (int64_t)gridDim.x * 8) {
        if (u >= piece_units) {
            const int64_t r0 = (u - piece_units) / s.spans * kEmpty, j0 = (u - piece_units) % s.spans * kSpan;
            const int64_t r = r0 + lane;
            uint32_t empty = __ballot_sync(0xffffffffu, r < s.vocabulary && s.start[r] == s.start[r + 1]);
            const float zero[kVec] = {};
            for (; empty; empty &= empty - 1)
                Lane<float, ALIGNED>::store(s.out + (r0 + __ffs(empty) - 1) * s.ldo, j0, s.n, lane, zero);
            continue;
        }
        const int64_t piece = u / s.spans, j0 = u % s.spans * kSpan, p0 = piece * kCut, p1 = min(real, p0 + kCut);
        if (p0 >= p1) continue;
        const uint32_t before = p0 ? s.token[p0 - 1] : 0xffffffffu, after = p1 < real ? s.token[p1] : 0xffffffffu;
        uint32_t token[2], position[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int64_t p = p0 + h * 32 + lane;
            token[h] = p < p1 ? s.token[p] : 0xffffffffu;
            position[h] = p < p1 ? s.position[p] : 0u;
        }
        const int live = (int)(p1 - p0);
        float sum[kVec] = {};
        uint32_t run = __shfl_sync(0xffffffffu, token[0], 0);
        bool carried = run == before;  // the run began in an earlier piece
        for (int g = 0; g < live; g += U) {
            float v[U][kVec];
            uint32_t t[U];
#pragma unroll
            for (int x = 0; x < U; ++x) {
                const int at = g + x;
                t[x] = __shfl_sync(0xffffffffu, at < 32 ? token[0] : token[1], at & 31);
                const uint32_t row = __shfl_sync(0xffffffffu, at < 32 ? position[0] : position[1], at & 31);
                if (at < live) Lane<T, ALIGNED>::load(dy + row * ldy, j0, s.n, lane, v[x]);
            }
#pragma unroll
            for (int x = 0; x < U; ++x) {
                if (g + x >= live) break;
                if (t[x] != run) {
                    if (carried)
                        Lane<float, ALIGNED>::store(s.partial + piece * 2 * s.width, j0, s.width, lane, sum);
                    else
                        emit<ALIGNED>(s, run, j0, lane, sum);
                    carried = false;
                    run = t[x];
#pragma unroll
                    for (int i = 0; i < kVec; ++i) sum[i] = 0.0f;
                }
#pragma unroll
                for (int i = 0; i < kVec; ++i) sum[i] += v[x][i];
            }
        }
        if (carried)
            Lane<float, ALIGNED>::store(s.partial + piece * 2 * s.width, j0, s.width, lane, sum);
        else if (run == after)
            Lane<float, ALIGNED>::store(s.partial + (piece * 2 + 1) * s.width, j0, s.width, lane, sum);
        else
            emit<ALIGNED>(s, run, j0, lane, sum);
    }
}

// Adds the partial sums of the runs that begin in piece blockIdx.x / spans and go on: its
// second row and the first rows of the pieces that follow, dealt out over the CTA's warps
// in order.
template <bool ALIGNED>
__global__ void __launch_bounds__(256) join_kernel(Sums s) {
    __shared__ float part[8][kSpan];
    pdl_wait();
    pdl_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t real = s.start[s.vocabulary];
    const int64_t piece = blockIdx.x / s.spans, j0 = blockIdx.x % s.spans * kSpan, end = (piece + 1) * kCut;
    if (end >= real) return;
    const uint32_t token = s.token[end - 1];
    if (s.token[end] != token || s.start[token] < piece * kCut) return;
    const int64_t last = (s.start[token + 1] - 1) / kCut, count = last - piece + 1, each = (count + 7) / 8;
    const int64_t b = min(count, warp * each), e = min(count, b + each);
    float sum[kVec] = {};
    for (int64_t c = b; c < e; ++c) {
        float v[kVec];
        const float* row = s.partial + ((piece + c) * 2 + (c == 0 ? 1 : 0)) * s.width;
        Lane<float, ALIGNED>::load(row, j0, s.width, lane, v);
#pragma unroll
        for (int i = 0; i < kVec; ++i) sum[i] += v[i];
    }
#pragma unroll
    for (int i = 0; i < kVec; ++i) part[warp][i * 32 + lane] = sum[i];
    __syncthreads();
    if (warp) return;
    const int64_t used = (count + each - 1) / each;
    for (int w = 1; w < used; ++w)
#pragma unroll
        for (int i = 0; i < kVec; ++i) sum[i] += part[w][i * 32 + lane];
    emit<ALIGNED>(s, token, j0, lane, sum);
}

int bits_of(int64_t v) {
    int b = 0;
    while (v >> b) ++b;
    return b;
}

// The workspace's layout from its sizes; the words it needs.
int64_t lay_out(int64_t count, int64_t vocabulary, int64_t n, Sort* s, Sums* m) {
    const int bits = std::max(1, bits_of(vocabulary));
    s->low = std::max(0, bits - 8);
    if (s->low > kMaxLow) s->low = kMaxLow;
    s->high = bits - s->low;
    s->count = count;
    s->vocabulary = vocabulary;
    // spans of at least 1024 positions: with more CTAs each would add up more counts
    s->ctas = (int)std::min<int64_t>(256, std::max<int64_t>(1, (count + 1023) / 1024));
    s->span = (count + s->ctas - 1) / s->ctas;
    m->pieces = (count + kCut - 1) / kCut;
    m->width = (n + kVec - 1) / kVec * kVec;
    auto words = [](int64_t v) { return (v + 31) / 32 * 32; };
    int64_t at = 0;
    uint32_t* base = s->counts;
    auto take = [&](int64_t v) {
        uint32_t* p = base + at;
        at += words(v);
        return p;
    };
    m->partial = reinterpret_cast<float*>(take(m->pieces * 2 * m->width));
    s->bucket = take((1 << s->high) + 1);
    s->key = take(count);
    s->place = take(count);
    s->token = take(count);
    s->position = take(count);
    s->start = take(vocabulary + 1);
    s->counts = take((int64_t)s->ctas << s->high);
    return at;
}

int check_backward(int64_t count, int64_t vocabulary, int64_t n) {
    RT_CHECK(count >= 0 && vocabulary >= 0 && n >= 0, "embedding: negative extent");
    RT_CHECK(count <= INT_MAX, "embedding: %lld positions are over 2^31 - 1", (long long)count);
    RT_CHECK(vocabulary <= kMaxVocabulary, "embedding: the gradient of %lld tokens is over 2^21 - 1", (long long)vocabulary);
    RT_CHECK(n <= (int64_t)1 << 31, "embedding: %lld columns are over 2^31", (long long)n);
    return RT_OK;
}

bool aligned(const rt_tensor* t) {
    return ((reinterpret_cast<uintptr_t>(t->ptr) | (uintptr_t)(t->ld * (int64_t)dtype_size(t->dtype))) & 15) == 0;
}

template <typename TE, typename TY>
int launch_lookup(rt_ctx* ctx, const rt_tensor* table, const rt_tensor* tokens, float scale, rt_tensor* y) {
    const int64_t spans = (y->cols + kSpan - 1) / kSpan, units = (y->rows + kRows - 1) / kRows * spans;
    const int64_t grid = std::min<int64_t>((units + 7) / 8, (int64_t)ctx->sm_count * 64);
    auto* kernel = aligned(table) && aligned(y) ? lookup_kernel<TE, TY, true> : lookup_kernel<TE, TY, false>;
    RT_CUDA(launch_k(ctx->pdl, kernel, (unsigned)grid, 256, 0, ctx->stream, static_cast<const TE*>(table->ptr), table->ld,
                     table->rows, static_cast<const uint32_t*>(tokens->ptr), y->rows, y->cols, spans, scale,
                     static_cast<TY*>(y->ptr), y->ld));
    count_launch(ctx);
    return RT_OK;
}

template <typename T>
int launch_sums(rt_ctx* ctx, const rt_tensor* dy, Sums m, bool all_aligned) {
    const int64_t piece_units = m.pieces * m.spans;
    const int64_t units = piece_units + (m.accumulate ? 0 : (m.vocabulary + kEmpty - 1) / kEmpty * m.spans);
    if (units == 0) return RT_OK;
    const int64_t grid = std::min<int64_t>((units + 7) / 8, (int64_t)ctx->sm_count * 64);
    auto* kernel = all_aligned ? sum_kernel<T, true> : sum_kernel<T, false>;
    RT_CUDA(launch_k(ctx->pdl, kernel, (unsigned)grid, 256, 0, ctx->stream, m, static_cast<const T*>(dy->ptr), dy->ld,
                     units, piece_units));
    count_launch(ctx);
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

int embedding_init() {
    const int deal = (1 << kMaxHigh) * 4 * (kSortWarps + 1);
    RT_CUDA(cudaFuncSetAttribute(bucket_deal_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, deal));
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
    m.n = dy->cols;
    m.spans = (m.n + kSpan - 1) / kSpan;
    RT_CHECK(m.pieces * m.spans <= INT_MAX, "rt_embedding_backward: dy is too large");
    if (dtable->rows == 0 || dtable->cols == 0) return RT_OK;
    RT_CUDA(cudaSetDevice(ctx->device));
    const uint32_t* t = static_cast<const uint32_t*>(tokens->ptr);
    const bool pdl = ctx->pdl;
    const int bins = 1 << s.high, low = 1 << s.low;
    RT_CUDA(launch_k(pdl, bucket_count_kernel, s.ctas, kSortThreads, bins * 4, ctx->stream, s, t));
    RT_CUDA(launch_k(pdl, bucket_deal_kernel, s.ctas, kSortThreads, bins * 4 * (kSortWarps + 1), ctx->stream, s, t));
    RT_CUDA(launch_k(pdl, bucket_sort_kernel, bins, kSortThreads, low * 4 * (kSortWarps + 1), ctx->stream, s));
    count_launch(ctx, 3);
    m.count = s.count;
    m.vocabulary = s.vocabulary;
    m.token = s.token;
    m.position = s.position;
    m.start = s.start;
    m.scale = scale;
    m.accumulate = accumulate != 0;
    m.out = static_cast<float*>(dtable->ptr);
    m.ldo = dtable->ld;
    const bool all = aligned(dy) && aligned(dtable);
    RT_TRY(dy->dtype == RT_BF16 ? launch_sums<__nv_bfloat16>(ctx, dy, m, all) : launch_sums<float>(ctx, dy, m, all));
    if (m.pieces > 1) {
        auto* kernel = all ? join_kernel<true> : join_kernel<false>;
        RT_CUDA(launch_k(pdl, kernel, (unsigned)(m.pieces * m.spans), 256, 0, ctx->stream, m));
        count_launch(ctx);
    }
    return RT_OK;
}

}  // extern "C"
