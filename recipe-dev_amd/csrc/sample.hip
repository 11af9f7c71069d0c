// The next token of every row of logits (rqmv_sample).
//
// The candidates of a row, in the order of their logits (the lowest index first
// among equals), have e_i = exp((l_i - l_max) / temperature). The first top_k are
// kept; of these the shortest prefix with a sum of at least top_p times theirs;
// of these those with e_i >= min_p. Each step keeps a prefix of the order, so the
// set is the shortest of the three, and the draw is the candidate at which the
// running sum in that order first exceeds u times the kept sum.
//
// Exactness. e_i is held as a whole number of 2^-42 (mass_of: an f64 exponential,
// rounded once), and all sums are sums of whole numbers: they do not depend on
// their order, no partial sum is rounded, and the tokens are those of the
// definition in 64 bits but for draws within 2^-42 n of a border. The thresholds
// u and top_p are multiplied out in 128 bits. No sort: a prefix is found by
// its count or its mass in a radix select over the logits' bits.
#include "sample.h"

#include <math.h>

namespace rq {

namespace {

constexpr int kMassBits = 42;  // 2^20 candidates of mass 2^42: sums stay below 2^63

// Logits as whole numbers of the same order (-0 as +0); 0: no candidate (NaN, -infinity).
__device__ __forceinline__ uint32_t key_of(float l) {
    if (!(l > -INFINITY)) return 0;
    const uint32_t b = __float_as_uint(l + 0.f);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float logit_of(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

// exp((l - top) / temperature) in units of 2^-42, to the nearest: 2^t = 2^n e^x with
// t = n + f, x = f ln 2, |x| <= 0.3466, e^x by its series up to x^12 (the next term
// is below 2^-52).
__device__ __forceinline__ uint64_t mass_of(float l, float top, double inv_t) {
    const double d = (double)l - (double)top;
    if (l == top) return 1ull << kMassBits;
    const double t = d * inv_t * 1.4426950408889634;
    if (!(t > -64.0)) return 0;  // (an infinite top leaves only its equals)
    const double n = rint(t);
    const double x = (t - n) * 0.69314718055994531;
    double p = 1.0 / 479001600.0;
    p = fma(p, x, 1.0 / 39916800.0);
    p = fma(p, x, 1.0 / 3628800.0);
    p = fma(p, x, 1.0 / 362880.0);
    p = fma(p, x, 1.0 / 40320.0);
    p = fma(p, x, 1.0 / 5040.0);
    p = fma(p, x, 1.0 / 720.0);
    p = fma(p, x, 1.0 / 120.0);
    p = fma(p, x, 1.0 / 24.0);
    p = fma(p, x, 1.0 / 6.0);
    p = fma(p, x, 0.5);
    p = fma(p, x, 1.0);
    p = fma(p, x, 1.0);
    const double scale = __longlong_as_double((long long)(1023 + kMassBits + (int)n) << 52);
    // adding 2^52 leaves the rounded whole number in the low mantissa bits (p scale <= 2^42)
    return (uint64_t)__double_as_longlong(fma(p, scale, 4503599627370496.0)) & 0xFFFFFFFFFFFFFull;
}

// floor(v * mass) and ceil(v * mass) for 0 <= v <= 1.
__device__ __forceinline__ uint64_t part_of(float v, uint64_t mass, bool up) {
    if (!(v > 0.f)) return 0;
    int e = 0;
    const uint64_t m = (uint64_t)ldexpf(frexpf(v, &e), 24);  // v = m 2^(e - 24)
    const int shift = 24 - e;
    const unsigned __int128 x = (unsigned __int128)m * mass;
    if (shift >= 127) return up && x ? 1 : 0;
    const unsigned __int128 floor = x >> shift;
    return (uint64_t)floor + (up && (floor << shift) != x ? 1 : 0);
}

// A row's settings, with those that are off or out of range in their plain form.
struct Settings {
    double inv_t;
    bool greedy;
    int k;        // 0: all
    float p, m;   // 1: all, 0: all
    float u;
};
__device__ __forceinline__ Settings settings_of(const SampleArgs& a, int row) {
    Settings s;
    const float t = a.temperature ? a.temperature[row] : 1.f;
    s.greedy = !(t > 0.f);
    s.inv_t = s.greedy ? 1.0 : 1.0 / (double)t;
    const int k = a.top_k ? a.top_k[row] : 0;
    s.k = k > 0 && k < a.n ? k : 0;
    const float p = a.top_p ? a.top_p[row] : 1.f;
    s.p = p >= 0.f && p < 1.f ? p : 1.f;
    const float m = a.min_p ? a.min_p[row] : 0.f;
    s.m = m > 0.f ? fminf(m, 1.f) : 0.f;
    const float u = a.u[row];
    s.u = u > 0.f ? fminf(u, 1.f) : 0.f;
    return s;
}

// ------------------------------------------------- a row by one workgroup ----

// Radix selects over the whole row, eight bits of the keys at a time: as many passes
// over the logits as it takes, right for every row.
constexpr int kRowThreads = 1024;

struct RowShared {
    unsigned long long mass[256];
    unsigned count[256];
    unsigned long long red[kRowThreads / 64];
    unsigned redi[kRowThreads / 64];
    uint32_t digit;
    unsigned long long mass_above;
    unsigned count_above;
};

// Where a prefix ends: the key of its last candidate and what lies above that key.
struct Cut {
    uint32_t key;
    uint64_t above;    // mass of the larger keys
    unsigned count;    // their number
};

__device__ __forceinline__ uint64_t block_sum(RowShared& sh, uint64_t v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor((unsigned long long)v, d);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.red[threadIdx.x >> 6] = v;
    __syncthreads();
    uint64_t t = 0;
    for (int w = 0; w < kRowThreads / 64; ++w) t += sh.red[w];
    return t;
}

// The key at which the count (by_mass: the mass) of the candidates in order first reaches `target` (>= 1, reachable).
__device__ Cut select(RowShared& sh, const float* row, int n, float top, double inv_t, bool by_mass, uint64_t target) {
    uint32_t prefix = 0;
    uint64_t above = 0;
    unsigned count = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (int i = threadIdx.x; i < 256; i += kRowThreads) sh.mass[i] = 0, sh.count[i] = 0;
        __syncthreads();
        const uint32_t mask = shift == 24 ? 0u : ~0u << (shift + 8);
        for (int i = threadIdx.x; i < n; i += kRowThreads) {
            const uint32_t k = key_of(row[i]);
            if (!k || (k & mask) != prefix) continue;
            const uint32_t digit = (k >> shift) & 255;
            atomicAdd(&sh.count[digit], 1u);
            const uint64_t m = mass_of(logit_of(k), top, inv_t);
            if (m) atomicAdd(&sh.mass[digit], (unsigned long long)m);
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            uint64_t a = above;
            unsigned c = count;
            int d = 255;
            for (; d > 0; --d) {
                const uint64_t reach = by_mass ? a + sh.mass[d] : (uint64_t)c + sh.count[d];
                if (reach >= target) break;
                a += sh.mass[d];
                c += sh.count[d];
            }
            sh.digit = d;
            sh.mass_above = a;
            sh.count_above = c;
        }
        __syncthreads();
        prefix |= sh.digit << shift;
        above = sh.mass_above;
        count = sh.count_above;
        __syncthreads();
    }
    return Cut{prefix, above, count};
}

// The index of the `which`-th (from 0) candidate with this key, in the order of indices.
__device__ int index_of(RowShared& sh, const float* row, int n, uint32_t key, uint64_t which) {
    __shared__ int found;
    if (threadIdx.x == 0) found = -1;
    const int per = (n + kRowThreads - 1) / kRowThreads;  // a thread's run of indices
    const int lo = min((int)threadIdx.x * per, n), hi = min(lo + per, n);
    unsigned mine = 0;
    for (int i = lo; i < hi; ++i) mine += key_of(row[i]) == key;
    unsigned upto = mine;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const unsigned v = __shfl_up(upto, d);
        if (lane >= d) upto += v;
    }
    __syncthreads();
    if (lane == 63) sh.redi[wave] = upto;
    __syncthreads();
    for (int w = 0; w < wave; ++w) upto += sh.redi[w];
    if (which < upto && which >= upto - mine) {
        unsigned left = (unsigned)which - (upto - mine);
        for (int i = lo; i < hi; ++i)
            if (key_of(row[i]) == key && left-- == 0) {
                found = i;
                break;
            }
    }
    __syncthreads();
    return found;
}

__global__ void __launch_bounds__(kRowThreads) sample_row_kernel(SampleArgs a) {
    __shared__ RowShared sh;
    const int r = blockIdx.x;
    const float* row = a.logits + (int64_t)r * a.ld;
    const Settings s = settings_of(a, r);
    uint32_t best = 0;
    for (int i = threadIdx.x; i < a.n; i += kRowThreads) best = max(best, key_of(row[i]));
#pragma unroll
    for (int d = 32; d; d >>= 1) best = max(best, (uint32_t)__shfl_xor((int)best, d));
    if ((threadIdx.x & 63) == 0) sh.redi[threadIdx.x >> 6] = best;
    __syncthreads();
    for (int w = 0; w < kRowThreads / 64; ++w) best = max(best, sh.redi[w]);
    __syncthreads();
    int token = -1;
    float prob = 0.f;
    if (best && s.greedy) {
        token = index_of(sh, row, a.n, best, 0);
        prob = 1.f;
    } else if (best) {
        const float top = logit_of(best);
        uint64_t total = 0, large = 0;
        unsigned candidates = 0;
        const uint64_t least = (uint64_t)ceil((double)s.m * (double)(1ull << kMassBits));
        for (int i = threadIdx.x; i < a.n; i += kRowThreads) {
            const uint32_t k = key_of(row[i]);
            if (!k) continue;
            const uint64_t m = mass_of(logit_of(k), top, s.inv_t);
            total += m;
            ++candidates;
            if (m >= least) large += m;
        }
        total = block_sum(sh, total);
        large = block_sum(sh, large);
        candidates = (unsigned)block_sum(sh, candidates);
        uint64_t kept = total;
        if (s.k && (unsigned)s.k < candidates) {
            const Cut c = select(sh, row, a.n, top, s.inv_t, false, s.k);
            kept = c.above + (s.k - c.count) * mass_of(logit_of(c.key), top, s.inv_t);
        }
        if (s.p < 1.f) {
            const uint64_t target = max(part_of(s.p, kept, true), (uint64_t)1);
            const Cut c = select(sh, row, a.n, top, s.inv_t, true, target);
            const uint64_t m = mass_of(logit_of(c.key), top, s.inv_t);
            kept = c.above + (target - c.above + m - 1) / m * m;
        }
        kept = min(kept, large);
        const uint64_t at = min(part_of(s.u, kept, false), kept - 1);
        const Cut c = select(sh, row, a.n, top, s.inv_t, true, at + 1);
        const uint64_t m = mass_of(logit_of(c.key), top, s.inv_t);
        token = index_of(sh, row, a.n, c.key, (at - c.above) / m);
        prob = (float)((double)m / (double)kept);
    }
    if (threadIdx.x == 0) {
        a.tokens[r] = token;
        if (a.probs) a.probs[r] = prob;
    }
}

}  // namespace

size_t sample_workspace(int, int, int) { return 0; }

hipError_t launch_sample(const SampleArgs& a, void*, int, hipStream_t stream) {
    hipLaunchKernelGGL(sample_row_kernel, dim3(a.rows), dim3(kRowThreads), 0, stream, a);
    return hipGetLastError();
}

}  // namespace rq
