// Log probabilities of given tokens, entropies and the likeliest tokens of rows
// of logits (rqmv_logprobs).
//
// With m the largest logit of a row, 1 + s = sum e^(x - m) and t = sum (x - m) e^(x - m):
//     log p(i) = x_i - m - log(1 + s),      entropy = log(1 + s) - t / (1 + s).
// The 1 is the term of one largest logit. It stays out of the sum: a token of probability 1 - 10^-8 has log probability
// -10^-8, which a sum of 1 + 10^-8 in fp32 does not hold. (With it in the sum 1500 rows of 128,256 take as long, with twenty
// alternatives 184 us instead of 186, of 32,000 58 instead of 61.)
// Rows are read once, 256 R logits a wave, kept in its registers: (m, s, t) about its own largest
// logit, and a list of at least its `top` largest ones. Of parts (m, s, t) the first with the largest m keeps its s, others
// with that m add 1 + s and t, and the rest move to the reference m' = that m:
//     e^(m - m') (1 + s),   e^(m - m') (t + (m - m') (1 + s)).
// A short row is finished by its workgroup; otherwise waves leave both in the workspace, on their
// own, and a second launch joins a row's.
//
// The largest of a wave's logits: if `top` of its lanes have their own largest at or above T, what lies below T is
// out. The wave finds its largest such T by bisection over its upper bits (ballots), which may leave it
// a little low, and lists what remains (some 1.2 to 1.4 times `top`). Where that is more than the list
// holds (many equal logits), it bisects for the exact top-th largest, and for the indices of the equal ones that belong
// to the first. At the end a workgroup takes the largest of its waves' T, and ranks
// what remains by comparing each with all (the lowest index first among equals).
//
// Bound: HBM, with the VALU as busy (1500 rows of 128,256 122 us, 6.3 TB/s read; with twenty alternatives 186); at few
// rows the two launches and the ranking's chain through LDS (17 rows, twenty alternatives: 16.7 us, 6.5 and 10.6 in a
// trace; 32 alternatives 26.5, 6.9 and 19.7).
#include "logprobs.h"

#include <limits.h>

#include "lanes.h"

namespace rq {

namespace {

constexpr int kWaves = 4, kThreads = 64 * kWaves;
constexpr int kList = 64;    // entries of a wave
constexpr int kSegment = 8;  // entries compared at once
constexpr float kLog2e = 1.44269504088896340736f;

struct Stats {
    float m, s, t;  // (no candidate: -infinity, 0, 0)
};
struct Entry {
    float v;
    int i;
};

// What `a` adds to the sums about `to` >= a.m; `first`: the 1 of these is its own.
__device__ __forceinline__ Stats move(Stats a, float to, bool first) {
    if (a.m == to) return Stats{to, first || to == -INFINITY ? a.s : 1.f + a.s, a.t};
    const float f = __builtin_amdgcn_exp2f((a.m - to) * kLog2e), s = 1.f + a.s;
    return f > 0.f ? Stats{to, f * s, f * fmaf(a.m - to, s, a.t)} : Stats{to, 0.f, 0.f};
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

// log(1 + s), s >= 0, to within two roundings: the logarithm of the rounded 1 + s and, to first order, of what its
// rounding left out.
__device__ __forceinline__ float log_of_one_and(float s) {
    const float u = 1.f + s;
    return logf(u) + (s - (u - 1.f)) * __builtin_amdgcn_rcpf(u);
}

// What a wave's registers hold.
template <int N>
__device__ __forceinline__ Stats wave_stats(const float (&v)[N], float m) {
    Stats a{m, 0.f, 0.f};
    float ones = 0.f;  // of the lane's terms
    if (m == INFINITY) {  // these alone count, all alike
#pragma unroll
        for (int i = 0; i < N; ++i) ones += v[i] == INFINITY ? 1.f : 0.f;
    } else if (m > -INFINITY) {
        // A lane adds up its terms below 1 by themselves; what all add up to says how many the others are.
        float all = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float d = v[i] - m, e = __builtin_amdgcn_exp2f(d * kLog2e);
            all += e;
            a.s += __builtin_amdgcn_fractf(e);
            a.t = fmaf(fmaxf(d, -1000.f), e, a.t);  // (-infinity times 0 would be NaN)
        }
        ones = rintf(all - a.s);
    }
    const unsigned long long has = __ballot(ones > 0.f);
    a.s += ones - ((int)(threadIdx.x & 63) == (has ? __builtin_ctzll(has) : 64) ? 1.f : 0.f);
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

// The wave's values from `least` on, or where these are more than kList the `top` first of the wave (value
// descending, index ascending): put(place, value, index), places from base(count) on. index.of(i): v[i]'s,
// index.below(i, x): whether it is below x.
template <int N, typename F, typename B, typename P>
__device__ __forceinline__ void wave_top(const float (&v)[N], uint32_t least_key, int top, const F& index, B base, P put) {
    float least = of_key(max(least_key, kLowest));
    int count = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) count += __popcll(__ballot(v[i] >= least));
    if (count <= kList) {
        int at = base(count);
        asm volatile("" : "+v"(least));  // (the comparisons again, not N kept masks)
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const unsigned long long hits = __ballot(v[i] >= least);
            if (hits) {
                if (v[i] >= least) put(at + before(hits), v[i], index.of(i));
                at += __popcll(hits);
            }
        }
        return;
    }
    // the largest key that `top` values reach
    uint32_t V = 0;
#pragma unroll 1
    for (int b = 31; b >= 0; --b) {
        const float up = of_key(V | 1u << b);  // (NaN beyond the infinities: no value reaches it)
        int c = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) c += __popcll(__ballot(v[i] >= up));
        if (c >= top) V |= 1u << b;
    }
    const float border = of_key(max(V, kLowest));
    int above = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) above += __popcll(__ballot(v[i] > border));
    // of those on the border as many as there is room for: the ones below index X
    int X = 0;
#pragma unroll 1
    for (int b = 20; b >= 0; --b) {
        const int up = X | 1 << b;
        int c = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) c += __popcll(__ballot(v[i] == border && index.below(i, up)));
        if (above + c <= top) X = up;
    }
    int at = base(top);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const bool take = v[i] > border || (v[i] == border && index.below(i, X));
        const unsigned long long hits = __ballot(take);
        if (take) put(at + before(hits), v[i], index.of(i));
        at += __popcll(hits);
    }
}

// The `top` first of the workgroup's values in order, in sh.best ((-infinity, -1) past the last). The waves agree on the
// largest of their `least`s, each of which has `top` values above it; then every entry of the list is compared with
// all, its share of them by one of two threads while there are at most 128.
template <int N, typename F>
__device__ __forceinline__ void group_top(Shared& sh, const float (&v)[N], float lane_max, int top, const F& index) {
    const uint32_t mine = wave_least(lane_max, top);
    if ((threadIdx.x & 63) == 0) sh.least[threadIdx.x >> 6] = mine;
    if (threadIdx.x == 0) sh.count = 0;
    for (int i = threadIdx.x; i < kWaves * kList; i += kThreads) sh.rank[i] = 0;
    __syncthreads();
    uint32_t least = sh.least[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) least = max(least, sh.least[w]);
    wave_top(
        v, least, top, index,
        [&](int count) {  // (a place in the workgroup's list)
            int base = 0;
            if ((threadIdx.x & 63) == 0) base = atomicAdd(&sh.count, count);
            return __builtin_amdgcn_readfirstlane(base);
        },
        [&](int at, float x, int i) { sh.list[at] = Entry{x, i}; });
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
    bool first = true;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        const Stats b = move(sh.stats[w], m, first);
        first = first && sh.stats[w].m != m;
        a.s += b.s, a.t += b.t;
    }
    return a;
}

__device__ __forceinline__ float log_prob(float x, const Stats& a, float log_s) {
    if (!(x > -INFINITY) || a.m == -INFINITY) return -INFINITY;
    return (x == a.m ? 0.f : x - a.m) - log_s;
}

// The logit of the row's token, asked for before it is needed (thread kGiven has it).
constexpr int kGiven = 128;
__device__ __forceinline__ float given_logit(const LogprobArgs& a, int64_t row) {
    if (threadIdx.x != kGiven || !a.logprob) return -INFINITY;
    const int token = a.tokens[row];
    return (unsigned)token < (unsigned)a.n ? a.logits[row * a.ld + token] : -INFINITY;
}

// A row's outputs from its stats, sh.best and the token's logit.
__device__ __forceinline__ void put_row(const LogprobArgs& a, int64_t row, const Stats& st, const Shared& sh, float given) {
    const int t = threadIdx.x;
    const float log_s = st.m > -INFINITY ? log_of_one_and(st.s) : 0.f;
    if (t < a.top) {
        const Entry e = sh.best[t];
        if (a.top_tokens) a.top_tokens[row * a.top + t] = e.i;
        if (a.top_logprobs) a.top_logprobs[row * a.top + t] = log_prob(e.v, st, log_s);
    } else if (t == 64) {
        if (a.entropy) a.entropy[row] = st.m > -INFINITY ? log_s - st.t / (1.f + st.s) : 0.f;
    } else if (t == kGiven) {
        if (a.logprob) a.logprob[row] = log_prob(given, st, log_s);
    }
}

// The indices of a wave's logits from c0 on, as load_logits puts them into its registers.
struct SliceIndex {
    int c0;
    __device__ __forceinline__ int of(int i) const { return c0 + 256 * (i / 4) + i % 4 + 4 * (int)(threadIdx.x & 63); }
    __device__ __forceinline__ bool below(int i, int x) const {
        return 4 * (int)(threadIdx.x & 63) < x - (c0 + 256 * (i / 4) + i % 4);
    }
};

// A wave's 256 R logits from c0 on, NaNs as -infinity and -0 as 0, and the lane's largest. (16 bytes a lane, aligned to 4
// or more; read once, so not kept in the caches: 1500 rows of 128,256 without alternatives 121 us, otherwise 134.)
template <int R>
__device__ __forceinline__ float load_logits(const LogprobArgs& a, int64_t row, int c0, float (&v)[4 * R]) {
    const int lane = threadIdx.x & 63;
    const float* x = a.logits + row * a.ld + c0 + 4 * lane;
    if (c0 + 256 * R <= a.n) {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int j = 0; j < 4; ++j) v[4 * r + j] = __builtin_nontemporal_load(x + 256 * r + j);
    } else {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int j = 0; j < 4; ++j) v[4 * r + j] = c0 + 256 * r + 4 * lane + j < a.n ? x[256 * r + j] : -INFINITY;
    }
    float most = -INFINITY;
#pragma unroll
    for (int i = 0; i < 4 * R; ++i) {
        v[i] = v[i] == v[i] ? v[i] + 0.f : -INFINITY;
        most = fmaxf(most, v[i]);
    }
    return most;
}

// Rows of at most 1024 R logits: one launch, no workspace. Bound: the chain of the load and the joins.
template <int R, bool TOP>
__global__ void __launch_bounds__(kThreads) logprobs_row_kernel(LogprobArgs a) {
    __shared__ Shared sh;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c0 = wave * 256 * R;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const float given = given_logit(a, row);
        float v[4 * R];
        const float most = load_logits<R>(a, row, c0, v);
        const Stats st = wave_stats(v, all_max(most));
        if (lane == 0) sh.stats[wave] = st;
        if (TOP) group_top(sh, v, most, a.top, SliceIndex{c0});
        __syncthreads();
        put_row(a, row, group_stats(sh), sh, given);
        __syncthreads();
    }
}

// What the waves leave of longer rows: of each (m, s, t, entries in its list), and the lists, [row][place][wave].
struct Parts {
    float4* stats;
    Entry* lists;
    int slices;  // waves of a row
};

template <int R, bool TOP>
__global__ void __launch_bounds__(kThreads) logprobs_slice_kernel(LogprobArgs a, Parts parts) {
    const int lane = threadIdx.x & 63;
    const int slice = blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c0 = slice * 256 * R;
    if (slice >= parts.slices) return;
    for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
        float v[4 * R];
        const float most = load_logits<R>(a, row, c0, v);
        const Stats st = wave_stats(v, all_max(most));
        int listed = 0;
        if (TOP) {
            Entry* list = parts.lists + row * kList * parts.slices + slice;
            wave_top(
                v, wave_least(most, a.top), a.top, SliceIndex{c0}, [&](int count) { return listed = count, 0; },
                [&](int at, float x, int i) { list[at * parts.slices] = Entry{x, i}; });
        }
        if (lane == 0) parts.stats[row * parts.slices + slice] = make_float4(st.m, st.s, st.t, __builtin_bit_cast(float, listed));
    }
}

// The waves of a row, more than SLOTS / 2 and at most SLOTS of them (8 to 256). A thread has every (256 / SLOTS)-th place
// of one wave's list; the first half of the places is asked for before it is known which are taken. So a workgroup's
// wave has at least 32 lanes with entries (where lists hold `top`), and its T leaves few. (With a lane for each of 16 slices
// T was 0, and all went through the exact bisection: 17 rows of 16,000 with twenty alternatives 27.7 us, so 12.7; 1500
// of 32,000 98, so 61.)
template <int SLOTS>
__global__ void __launch_bounds__(kThreads) logprobs_join_kernel(LogprobArgs a, Parts parts) {
    constexpr int SIDE = kThreads / SLOTS, N = kList / SIDE;
    __shared__ Shared sh;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), slices = parts.slices;
    const int slice = threadIdx.x % SLOTS, side = threadIdx.x / SLOTS;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const float given = given_logit(a, row);
        float4 p = make_float4(-INFINITY, 0.f, 0.f, 0.f);
        if (slice < slices) p = parts.stats[row * slices + slice];
        const Entry* list = parts.lists + row * kList * slices + min(slice, slices - 1);
        Entry e[N];
        if (a.top) {
#pragma unroll
            for (int i = 0; i < N / 2; ++i) e[i] = list[(i * SIDE + side) * slices];
        }
        const int listed = __builtin_bit_cast(int, p.w);
        Stats st = side == 0 ? Stats{p.x, p.y, p.z} : Stats{-INFINITY, 0.f, 0.f};
        const float m = all_max(st.m);
        st = move(st, m, lane == __builtin_ctzll(__ballot(st.m == m)));
        st.s = all_sum(st.s);
        st.t = all_sum(st.t);
        if (lane == 0) sh.stats[wave] = st;
        if (a.top) {
            struct Ids {
                int id[N];
                __device__ __forceinline__ int of(int i) const { return id[i]; }
                __device__ __forceinline__ bool below(int i, int x) const { return id[i] < x; }
            } ids;
            float v[N], most = -INFINITY;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const bool taken = i * SIDE + side < listed;
                if (i >= N / 2) {
                    e[i] = Entry{-INFINITY, -1};
                    if (taken) e[i] = list[(i * SIDE + side) * slices];
                }
                v[i] = taken ? e[i].v : -INFINITY;
                ids.id[i] = e[i].i;
                most = fmaxf(most, v[i]);
            }
            group_top(sh, v, most, a.top, ids);
        }
        __syncthreads();
        put_row(a, row, group_stats(sh), sh, given);
        __syncthreads();
    }
}

struct LogprobPlan {
    int r;
    bool whole;  // a row by its workgroup
    Parts parts;
};
LogprobPlan plan_logprobs(int rows, int n, int top, int cus) {
    // Without alternatives: rows of up to 8192 logits at once (17 rows of 8,000 4.8 us, by slices 8.0; 1500 12.5 and 14.5;
    // of 16,000 it would be 6.9 and 7.7, but 26.8 and 20.7), else 1024 logits a wave (100 rows of 128,256 13.8, of 4096
    // 16.3; 1500 122 and 122; 1500 of 32,000 34.6 and 39.7). With them: rows of up to 4096 at once (of 8,000, 17 rows, 32
    // alternatives, by slices 14.7, at once 21.0; 1500 rows, twenty 25.8 and 29.4); 1024 logits a wave, but 2048 where
    // these are enough for two workgroups a CU (twenty alternatives, 100 and 1500 rows of 128,256 25.7 and 186, of 1024
    // 27.2 and 204; 400 and 1500 of 32,000 26.7 and 60.6, 25.8 and 58.5). A row is 256 waves' at most.
    const bool many = (int64_t)((n + 16383) / 16384) * rows >= 2 * cus;
    LogprobPlan p;
    p.whole = n <= (top ? 4096 : 8192);
    p.r = p.whole ? (n <= 4096 ? 4 : 8) : top && many && n > 8192 ? 8 : 4;
    while (n > 256 * p.r * kThreads) p.r *= 2;
    p.parts.slices = (n + 256 * p.r - 1) / (256 * p.r);
    return p;
}

template <int R, bool TOP>
void launch_slices(const LogprobArgs& a, const LogprobPlan& p, hipStream_t stream) {
    const dim3 grid((p.parts.slices + kWaves - 1) / kWaves, a.rows < 65535 ? a.rows : 65535);
    hipLaunchKernelGGL((logprobs_slice_kernel<R, TOP>), grid, dim3(kThreads), 0, stream, a, p.parts);
}

}  // namespace

size_t logprobs_workspace(int rows, int n, int top, int cus) {
    const LogprobPlan p = plan_logprobs(rows, n, top, cus);
    return p.whole ? 0 : (size_t)rows * p.parts.slices * (sizeof(float4) + (top ? kList * sizeof(Entry) : 0));
}

hipError_t launch_logprobs(const LogprobArgs& a, void* workspace, int cus, hipStream_t stream) {
    LogprobPlan p = plan_logprobs(a.rows, a.n, a.top, cus);
    p.parts.stats = static_cast<float4*>(workspace);
    p.parts.lists = reinterpret_cast<Entry*>(p.parts.stats + (int64_t)a.rows * p.parts.slices);
    const dim3 rows(a.rows), threads(kThreads);
    if (p.whole) {
        const auto row = a.top      ? logprobs_row_kernel<4, true>
                         : p.r == 4 ? logprobs_row_kernel<4, false>
                                    : logprobs_row_kernel<8, false>;
        hipLaunchKernelGGL(row, rows, threads, 0, stream, a);
        return hipGetLastError();
    }
    if (a.top) {
        if (p.r == 4) launch_slices<4, true>(a, p, stream);
        else if (p.r == 8) launch_slices<8, true>(a, p, stream);
        else launch_slices<16, true>(a, p, stream);
    } else {
        if (p.r == 4) launch_slices<4, false>(a, p, stream);
        else if (p.r == 8) launch_slices<8, false>(a, p, stream);
        else launch_slices<16, false>(a, p, stream);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const auto join = p.parts.slices <= 8     ? logprobs_join_kernel<8>
                      : p.parts.slices <= 16  ? logprobs_join_kernel<16>
                      : p.parts.slices <= 32  ? logprobs_join_kernel<32>
                      : p.parts.slices <= 64  ? logprobs_join_kernel<64>
                      : p.parts.slices <= 128 ? logprobs_join_kernel<128>
                                              : logprobs_join_kernel<256>;
    hipLaunchKernelGGL(join, rows, threads, 0, stream, a, p.parts);
    return hipGetLastError();
}

}  // namespace rq
