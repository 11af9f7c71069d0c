// Log probabilities of given tokens, entropies and the likeliest tokens of rows
// of logits (rqmv_logprobs).
//
// With m the largest logit of a row, s = sum e^(x - m) and t = sum (x - m) e^(x - m):
//     log p(i) = x_i - m - log s,      entropy = log s - t / s.
// Rows are read once, in slices of 1024 R logits, a workgroup each, kept in
// registers: (m, s, t) about the slice's own largest logit, and the slice's `top` largest
// logits. A second launch joins a row's slices: s and t move to another reference m' by
//     s' = e^(m - m') s,   t' = e^(m - m') (t + (m - m') s).
// A row of one slice is finished where it is read.
//
// The largest of a workgroup's logits: if `top` lanes of a wave have their own largest at or above T, what
// lies below T is out. A wave finds its largest such T by bisection over its upper bits
// (ballots), which may leave it a little low, and the workgroup takes the largest of its four. What
// remains goes into a list in LDS and is ranked by comparing each with all (the
// lowest index first among equals). Where many are equal a wave's share of the list overflows;
// then it bisects for the exact top-th largest of all its logits and takes the equal ones by their index.
//
// Bound: HBM, at few rows the two launches and their dependent loads.
#include "logprobs.h"

#include <limits.h>

#include "lanes.h"

namespace rq {

namespace {

constexpr int kWaves = 4, kThreads = 64 * kWaves;
constexpr int kList = 128;   // entries of a wave
constexpr int kSegment = 8;  // entries compared at once
constexpr float kLog2e = 1.44269504088896340736f;

struct Stats {
    float m, s, t;
};
struct Entry {
    float v;
    int i;
};

// e^(from - to) for to >= from, or to = -infinity (then 0).
__device__ __forceinline__ float moved(float from, float to) {
    return from == to ? (to == -INFINITY ? 0.f : 1.f) : __builtin_amdgcn_exp2f((from - to) * kLog2e);
}
// `a` about the reference `to`.
__device__ __forceinline__ Stats move(Stats a, float to) {
    const float f = moved(a.m, to);
    return Stats{to, f * a.s, f > 0.f && a.m != to ? f * fmaf(a.m - to, a.s, a.t) : f > 0.f ? a.t : 0.f};
}

// Floats to numbers in their order and back. (No NaNs and no -0.)
__device__ __forceinline__ uint32_t key_of(float v) {
    const uint32_t b = __builtin_bit_cast(uint32_t, v);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float of_key(uint32_t k) {
    return __builtin_bit_cast(float, k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
constexpr uint32_t kLowest = 0x00800000u;  // key_of(-FLT_MAX): what is below is no candidate

// What a wave's registers hold.
template <int N>
__device__ __forceinline__ Stats wave_stats(const float (&v)[N], float m) {
    Stats a{m, 0.f, 0.f};
    if (m == INFINITY) {  // these alone count, all alike
#pragma unroll
        for (int i = 0; i < N; ++i) a.s += v[i] == INFINITY ? 1.f : 0.f;
    } else if (m > -INFINITY) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float d = v[i] - m, e = __builtin_amdgcn_exp2f(d * kLog2e);
            a.s += e;
            a.t = fmaf(fmaxf(d, -1000.f), e, a.t);  // (-infinity times 0 would be NaN)
        }
    }
    a.s = all_sum(a.s);
    a.t = all_sum(a.t);
    return a;
}

struct Shared {
    Entry list[kWaves * kList + 2 * kSegment];
    int rank[kWaves * kList];
    Entry best[kLogprobMaxTop];
    Stats stats[kWaves];
    uint32_t least[kWaves];
    int count;
};

__device__ __forceinline__ int before(unsigned long long mask) {  // lanes of `mask` before this one
    return __builtin_amdgcn_mbcnt_hi((unsigned)(mask >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)mask, 0));
}

// A number that at least `top` of the wave's lanes reach with their largest value, close to the largest such.
__device__ __forceinline__ uint32_t wave_least(float lane_max, int top) {
    const uint32_t mine = key_of(lane_max);
    uint32_t T = 0;
#pragma unroll 1
    for (int b = 30; b >= 12; b -= 2) {  // (two bits a step: three ballots that do not wait for each other)
        const int c1 = __popcll(__ballot(mine >= (T | 1u << b))), c2 = __popcll(__ballot(mine >= (T | 2u << b))),
                  c3 = __popcll(__ballot(mine >= (T | 3u << b)));
        T |= (c3 >= top ? 3u : c2 >= top ? 2u : c1 >= top ? 1u : 0u) << b;
    }
    return T;
}

// The wave's values from `least` on into the workgroup's list; of more than kList the `top` first of the
// wave (value descending, index ascending). `index(i)`: of v[i], ascending by (i / G, lane, i % G).
template <int N, int G, typename F>
__device__ __forceinline__ void wave_top(Shared& sh, const float (&v)[N], uint32_t least_key, int top, F index) {
    const float least = of_key(max(least_key, kLowest));
    auto base_of = [&](int count) {  // a place for `count` entries
        int base = 0;
        if ((threadIdx.x & 63) == 0) base = atomicAdd(&sh.count, count);
        return __builtin_amdgcn_readfirstlane(base);
    };
    int count = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) count += __popcll(__ballot(v[i] >= least));
    if (count <= kList) {
        int at = base_of(count);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const unsigned long long hits = __ballot(v[i] >= least);
            if (hits) {
                if (v[i] >= least) sh.list[at + before(hits)] = Entry{v[i], index(i)};
                at += __popcll(hits);
            }
        }
        return;
    }
    // Too many: the exact border, then all above it and the first of those on it.
    uint32_t V = 0;
#pragma unroll 1
    for (int b = 31; b >= 0; --b) {
        const uint32_t up = V | 1u << b;
        int c = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) c += __popcll(__ballot(key_of(v[i]) >= up));
        if (c >= top) V = up;
    }
    const float border = of_key(max(V, kLowest));
    const int at = base_of(top);
    count = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const unsigned long long hits = __ballot(v[i] > border);
        if (v[i] > border) sh.list[at + count + before(hits)] = Entry{v[i], index(i)};  // (fewer than `top`)
        count += __popcll(hits);
    }
#pragma unroll
    for (int r = 0; r < N / G; ++r) {
        unsigned own = 0;
#pragma unroll
        for (int j = 0; j < G; ++j) own += v[G * r + j] == border ? 1 : 0;
        const unsigned upto = wave_scan(own);
        int k = count + (int)(upto - own);
#pragma unroll
        for (int j = 0; j < G; ++j)
            if (v[G * r + j] == border) {
                if (k < top) sh.list[at + k] = Entry{border, index(G * r + j)};
                ++k;
            }
        count = min(count + __builtin_amdgcn_readlane((int)upto, 63), top);
    }
}

// The `top` first of the workgroup's values in order, in sh.best ((-infinity, -1) past the last). The waves agree on the
// largest of their `least`s, each of which has `top` values above it; then every entry of the list is compared with
// all, its share of them by one of two threads while there are at most 128.
template <int N, int G, typename F>
__device__ __forceinline__ void group_top(Shared& sh, const float (&v)[N], float lane_max, int top, F index) {
    const uint32_t mine = wave_least(lane_max, top);
    if ((threadIdx.x & 63) == 0) sh.least[threadIdx.x >> 6] = mine;
    if (threadIdx.x == 0) sh.count = 0;
    for (int i = threadIdx.x; i < kWaves * kList; i += kThreads) sh.rank[i] = 0;
    __syncthreads();
    uint32_t least = sh.least[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) least = max(least, sh.least[w]);
    wave_top<N, G>(sh, v, least, top, index);
    __syncthreads();
    const int count = sh.count;
    // past the last: entries that are before none
    if (threadIdx.x < 2 * kSegment) sh.list[count + threadIdx.x] = Entry{-INFINITY, INT_MAX};
    __syncthreads();
    const bool halves = count <= kThreads / 2;
    const int each = halves ? (count / 2 + kSegment) & ~(kSegment - 1) : count;
    for (int p = halves ? threadIdx.x / 2 : threadIdx.x; p < count; p += kThreads) {
        const Entry own = sh.list[p];
        const int from = halves ? (threadIdx.x & 1) * each : 0;
        int rank = 0;
        for (int q = from; q < min(from + each, count); q += kSegment) {
#pragma unroll
            for (int k = 0; k < kSegment; ++k) {
                const Entry o = sh.list[q + k];
                rank += o.v > own.v || (o.v == own.v && o.i < own.i) ? 1 : 0;
            }
        }
        if (halves) atomicAdd(&sh.rank[p], rank);
        else sh.rank[p] = rank;
    }
    __syncthreads();
    for (int p = threadIdx.x; p < count; p += kThreads)
        if (sh.rank[p] < top) sh.best[sh.rank[p]] = sh.list[p];
    if ((int)threadIdx.x < top && (int)threadIdx.x >= count) sh.best[threadIdx.x] = Entry{-INFINITY, -1};
}

// The waves' stats as one. (Read behind a barrier.)
__device__ __forceinline__ Stats group_stats(const Shared& sh) {
    float m = sh.stats[0].m;
#pragma unroll
    for (int w = 1; w < kWaves; ++w) m = fmaxf(m, sh.stats[w].m);
    Stats a{m, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        const Stats b = move(sh.stats[w], m);
        a.s += b.s, a.t += b.t;
    }
    return a;
}

__device__ __forceinline__ float log_prob(float x, const Stats& a, float log_s) {
    if (!(x > -INFINITY) || a.m == -INFINITY) return -INFINITY;
    return x == a.m ? -log_s : (x - a.m) - log_s;
}

// A row's outputs from its stats, sh.best and the token's logit.
__device__ __forceinline__ void put_row(const LogprobArgs& a, int64_t row, const Stats& st, const Shared& sh) {
    const int t = threadIdx.x;
    const float log_s = st.m > -INFINITY ? logf(st.s) : 0.f;
    if (t < a.top) {
        const Entry e = sh.best[t];
        if (a.top_tokens) a.top_tokens[row * a.top + t] = e.i;
        if (a.top_logprobs) a.top_logprobs[row * a.top + t] = log_prob(e.v, st, log_s);
    } else if (t == 64) {
        if (a.entropy) a.entropy[row] = st.m > -INFINITY ? log_s - st.t / st.s : 0.f;
    } else if (t == 128 && a.logprob) {
        const int token = a.tokens[row];
        a.logprob[row] = log_prob((unsigned)token < (unsigned)a.n ? a.logits[row * a.ld + token] : -INFINITY, st, log_s);
    }
}

// A slice of 1024 R logits: to the outputs where the row has no other (parts null), or to the workspace.
template <int R, bool TOP>
__global__ void __launch_bounds__(kThreads) logprobs_slice_kernel(LogprobArgs a, float4* parts, Entry* tops) {
    __shared__ Shared sh;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c0 = (blockIdx.x * kWaves + wave) * 256 * R;
    for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
        const float* x = a.logits + row * a.ld + c0 + 4 * lane;
        float v[4 * R];
        if (c0 + 256 * R <= a.n) {
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int j = 0; j < 4; ++j) v[4 * r + j] = x[256 * r + j];  // (16 bytes a lane, aligned to 4 or more)
        } else {
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    v[4 * r + j] = c0 + 256 * r + 4 * lane + j < a.n ? x[256 * r + j] : -INFINITY;
        }
        float top1 = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4 * R; ++i) {
            v[i] = v[i] == v[i] ? v[i] + 0.f : -INFINITY;  // (NaNs are skipped; -0 is 0)
            top1 = fmaxf(top1, v[i]);
        }
        const Stats st = wave_stats(v, all_max(top1));
        if (lane == 0) sh.stats[wave] = st;
        if (TOP)
            group_top<4 * R, 4>(sh, v, top1, a.top, [&](int i) { return c0 + 256 * (i / 4) + 4 * lane + i % 4; });
        __syncthreads();
        const Stats all = group_stats(sh);
        if (!parts) {
            put_row(a, row, all, sh);
        } else {
            const int64_t at = row * gridDim.x + blockIdx.x;
            if (threadIdx.x == 0) parts[at] = make_float4(all.m, all.s, all.t, 0.f);
            if (TOP && (int)threadIdx.x < a.top) tops[at * a.top + threadIdx.x] = sh.best[threadIdx.x];
        }
        __syncthreads();
    }
}

// A row's slices (at most 256), and their lists of `top` entries: at most 64 N kWaves.
template <int N>
__global__ void __launch_bounds__(kThreads) logprobs_join_kernel(LogprobArgs a, const float4* parts, const Entry* tops,
                                                                 int slices) {
    __shared__ Shared sh;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        Stats st{-INFINITY, 0.f, 0.f};
        if ((int)threadIdx.x < slices) {
            const float4 p = parts[row * slices + threadIdx.x];
            st = Stats{p.x, p.y, p.z};
        }
        const float m = all_max(st.m);
        st = move(st, m);
        st.s = all_sum(st.s);
        st.t = all_sum(st.t);
        if (lane == 0) sh.stats[wave] = st;
        if (a.top) {
            // entry 256 i + thread is v[i]: a lane's are of unlike lists, and equal values stand in the order of their indices
            const int all = slices * a.top;
            float v[N], top1 = -INFINITY;
            int id[N];
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int e = kThreads * i + threadIdx.x;
                const Entry o = e < all ? tops[row * all + e] : Entry{-INFINITY, -1};
                v[i] = o.v, id[i] = o.i;
                top1 = fmaxf(top1, v[i]);
            }
            group_top<N, 1>(sh, v, top1, a.top, [&](int i) { return id[i]; });
        }
        __syncthreads();
        put_row(a, row, group_stats(sh), sh);
        __syncthreads();
    }
}

struct LogprobPlan {
    int r, slices;
};
LogprobPlan plan_logprobs(int rows, int n, int cus) {
    // Slices of 16,384 logits where that gives two workgroups a CU, else of 4,096.
    const int64_t large = (n + 16383) / 16384;
    const int r = large * rows >= 2 * cus ? 16 : 4;
    return LogprobPlan{r, (n + 1024 * r - 1) / (1024 * r)};
}

}  // namespace

size_t logprobs_workspace(int rows, int n, int top, int cus) {
    const LogprobPlan p = plan_logprobs(rows, n, cus);
    return p.slices > 1 ? (size_t)rows * p.slices * (sizeof(float4) + top * sizeof(Entry)) : 0;
}

hipError_t launch_logprobs(const LogprobArgs& a, void* workspace, int cus, hipStream_t stream) {
    const LogprobPlan p = plan_logprobs(a.rows, a.n, cus);
    float4* parts = p.slices > 1 ? static_cast<float4*>(workspace) : nullptr;
    Entry* tops = p.slices > 1 ? reinterpret_cast<Entry*>(parts + (int64_t)a.rows * p.slices) : nullptr;
    const dim3 grid(p.slices, a.rows < 65535 ? a.rows : 65535), threads(kThreads);
    if (p.r == 16 && a.top) hipLaunchKernelGGL((logprobs_slice_kernel<16, true>), grid, threads, 0, stream, a, parts, tops);
    else if (p.r == 16) hipLaunchKernelGGL((logprobs_slice_kernel<16, false>), grid, threads, 0, stream, a, parts, tops);
    else if (a.top) hipLaunchKernelGGL((logprobs_slice_kernel<4, true>), grid, threads, 0, stream, a, parts, tops);
    else hipLaunchKernelGGL((logprobs_slice_kernel<4, false>), grid, threads, 0, stream, a, parts, tops);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.slices == 1) return e;
    const dim3 rows(a.rows < (1 << 20) ? a.rows : 1 << 20);
    const int entries = p.slices * a.top;
    if (entries <= 1024) hipLaunchKernelGGL(logprobs_join_kernel<4>, rows, threads, 0, stream, a, parts, tops, p.slices);
    else hipLaunchKernelGGL(logprobs_join_kernel<32>, rows, threads, 0, stream, a, parts, tops, p.slices);
    return hipGetLastError();
}

}  // namespace rq
