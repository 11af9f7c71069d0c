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
// u and top_p are multiplied out in 128 bits.
//
// A row is never sorted. Its logits are binned by their distance from the largest
// (kBins bins over the logits' range, or over the 30 temperatures below which a
// mass rounds to zero), and the bins' counts and masses tell in which bins the
// three prefixes and the draw can end; only their candidates are collected, sorted
// and summed one by one. Four launches over slices of the rows:
//   bounds   largest logit with its lowest index, smallest logit, per slice
//   bins     counts (rows with a top_k) or masses (without; both for a top_k above
//            kFewKept) per slice
//   collect  every slice adds up its row's bins, finds the wanted ones and appends its
//            candidates in them to the row's list; with a top_k up to kFewKept
//            these are all bins that hold any of the first top_k
//   finish   one workgroup per row
// Rows of at most kList logits need the last one only, on all of their candidates. A
// row whose wanted bins hold more than kList candidates (many equal logits, or an
// outlier far above a narrow rest) takes radix selects over its logits' bits instead,
// up to sixteen passes by one workgroup: 128,256 equal logits 1.1 ms, with top_k or top_p 2.0, with
// both 2.9 (64 such rows 1.2 to 3.0); an outlier above a narrow rest 0.4 to 0.8. Ordinary rows: 23 to 27 us,
// 64 of them 35 to 47. Up to kList logits: 18 us, 64 rows 19, 1,024 rows 74.
#include "sample.h"

#include <math.h>

#include "lanes.h"

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

// exp((l - top) / temperature) in units of 2^-42, to the nearest: e^z = 2^(m / 32) e^x with
// m = rint(32 z / ln 2) and x = z - m ln 2 / 32, |x| <= 0.0109, e^x by its series up to
// x^5 (the next term is below 2^-48). m needs no care, so it is taken in fp32; z and x are
// f64. `pow2` holds 2^(j / 32) in LDS. (The bins of 64 rows of 128,256 take 14.6 us, with a series
// to x^12 and no table 17.0.)
struct Masses {
    float top, up, c;  // up * c = 32 / (ln 2 temperature), which alone passes fp32's range below 10^-37
    double dtop, inv_t;
    const double* pow2;
    __device__ __forceinline__ Masses(float top_, double inv_t_, const double* pow2_)
        : top(top_), up(inv_t_ > 0x1p100 ? 0x1p40f : 1.f), c((float)(inv_t_ * (46.166241308446828 / up))), dtop(top_),
          inv_t(inv_t_), pow2(pow2_) {}
    __device__ __forceinline__ uint64_t operator()(float l) const {
        if (l == top) return 1ull << kMassBits;
        const float m = rintf((l - top) * up * c);
        if (!(m > -2000.f)) return 0;  // (an infinite top leaves only its equals)
        const double x = fma((double)m, -0.021660849392498290, ((double)l - dtop) * inv_t);
        double p = 1.0 / 120.0;
        p = fma(p, x, 1.0 / 24.0);
        p = fma(p, x, 1.0 / 6.0);
        p = fma(p, x, 0.5);
        p = fma(p, x, 1.0);
        p = fma(p, x, 1.0);
        const int i = (int)m;
        const double scale = __longlong_as_double(__double_as_longlong(pow2[i & 31]) +
                                                  ((long long)(kMassBits + (i >> 5)) << 52));
        // adding 2^52 leaves the rounded whole number in the low mantissa bits (p scale <= 2^42)
        return (uint64_t)__double_as_longlong(fma(p, scale, 4503599627370496.0)) & 0xFFFFFFFFFFFFFull;
    }
    // Whether min_p keeps l: (l - top) / temperature >= log(min_p). Unlike a comparison of masses, whose rounding
    // makes equals of neighbours, this is a border in the logits, as the bins are.
    __device__ __forceinline__ bool keeps(float l, double least_z) const {
        return l == top || ((double)l - dtop) * inv_t >= least_z;
    }
};
// (the workgroup's barrier before the first use is the caller's)
__device__ __forceinline__ void fill_pow2(double* pow2) {
    if (threadIdx.x < 32) pow2[threadIdx.x] = exp2((double)threadIdx.x / 32.0);
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

// What the steps compare running sums with: top_p's prefix ends at the first candidate
// that reaches this, the draw is the first that passes this, min_p keeps logits of at least this many
// temperatures above the largest (< 0).
__device__ __forceinline__ uint64_t p_target(const Settings& s, uint64_t mass) {
    return max(part_of(s.p, mass, true), (uint64_t)1);
}
__device__ __forceinline__ uint64_t u_target(const Settings& s, uint64_t kept) {
    return min(part_of(s.u, kept, false), kept - 1);
}
// (2^-54 less than the logarithm: an e this near to min_p is min_p in 64 bits)
__device__ __forceinline__ double least_z(const Settings& s) {
    return s.m > 0.f ? log((double)s.m) - 0x1p-54 : -INFINITY;
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
__device__ Cut select(RowShared& sh, const float* row, int n, const Masses& mass_of, bool by_mass, uint64_t target) {
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
            const uint64_t m = mass_of(logit_of(k));
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

// The whole row: (token, probability).
__device__ void sample_row(RowShared& sh, const float* row, int n, const Settings& s, const Masses& mass_of, int* token,
                           float* prob) {
    uint64_t total = 0, large = 0;
    unsigned candidates = 0;
    const double least = least_z(s);
    for (int i = threadIdx.x; i < n; i += kRowThreads) {
        const uint32_t k = key_of(row[i]);
        if (!k) continue;
        const uint64_t m = mass_of(logit_of(k));
        total += m;
        ++candidates;
        if (mass_of.keeps(logit_of(k), least)) large += m;
    }
    total = block_sum(sh, total);
    large = block_sum(sh, large);
    candidates = (unsigned)block_sum(sh, candidates);
    uint64_t kept = total;
    if (s.k && (unsigned)s.k < candidates) {
        const Cut c = select(sh, row, n, mass_of, false, s.k);
        kept = c.above + (s.k - c.count) * mass_of(logit_of(c.key));
    }
    if (s.p < 1.f) {
        const uint64_t target = p_target(s, kept);
        const Cut c = select(sh, row, n, mass_of, true, target);
        const uint64_t m = mass_of(logit_of(c.key));
        kept = c.above + (target - c.above + m - 1) / m * m;
    }
    kept = min(kept, large);
    const uint64_t at = u_target(s, kept);
    const Cut c = select(sh, row, n, mass_of, true, at + 1);
    const uint64_t m = mass_of(logit_of(c.key));
    *token = index_of(sh, row, n, c.key, (at - c.above) / m);
    *prob = (float)((double)m / (double)kept);
}

// ------------------------------------------------------ rows by their bins ----

constexpr int kBins = 1024;      // one per thread of a workgroup
constexpr int kThreads = kRowThreads;
constexpr int kList = 4096;      // candidates that finish sorts in LDS
constexpr int kFewKept = 1024;   // top_k up to which the whole kept set is collected
constexpr int kMaxSlices = 16;
constexpr int kRowsAtOnce = 1024;  // rows that one workspace holds

struct Bound {
    uint64_t best;  // key of the largest logit, then ~index (the lowest index among equals is the largest)
    uint32_t least, unused;
};

// A row's part of the workspace.
struct RowWork {
    Bound* bound;               // [slices]
    unsigned long long* mass;   // [slices][kBins]
    unsigned long long* list;   // [slices][kList]: key, ~index
    unsigned long long* above;  // [kBins]: mass of the bins before
    unsigned long long* total;  // [2]: mass of all bins, of the bins that min_p keeps for certain
    unsigned* listed;           // [kMaxSlices]
    unsigned* before;           // [kBins]: candidates in the bins before
    unsigned* count;            // [slices][kBins]
};
__host__ __device__ constexpr size_t row_work_bytes(int slices) {
    return (size_t)slices * (sizeof(Bound) + kBins * 12 + kList * 8) + kBins * 12 + 16 + kMaxSlices * 4;
}
__device__ __forceinline__ RowWork row_work(void* ws, int row, int slices) {
    char* p = static_cast<char*>(ws) + row * row_work_bytes(slices);
    auto take = [&](size_t bytes) {
        char* at = p;
        p += bytes;
        return at;
    };
    RowWork w;
    w.bound = reinterpret_cast<Bound*>(take(slices * sizeof(Bound)));
    w.mass = reinterpret_cast<unsigned long long*>(take((size_t)slices * kBins * 8));
    w.list = reinterpret_cast<unsigned long long*>(take((size_t)slices * kList * 8));
    w.above = reinterpret_cast<unsigned long long*>(take(kBins * 8));
    w.total = reinterpret_cast<unsigned long long*>(take(16));
    w.listed = reinterpret_cast<unsigned*>(take(kMaxSlices * 4));
    w.before = reinterpret_cast<unsigned*>(take(kBins * 4));
    w.count = reinterpret_cast<unsigned*>(take((size_t)slices * kBins * 4));
    return w;
}

// A workgroup's part of a row, eight logits per thread at a time. The first eight are
// requested when the kernel starts, before it has read what it needs to use them.
struct Slice {
    const float* row;
    int lo, hi;
    float v[8];
    __device__ __forceinline__ void load(int base) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = row[min(base + j * kThreads, hi - 1)];
    }
    __device__ __forceinline__ Slice(const SampleArgs& a, int r, int slice, int slices)
        : row(a.logits + r * a.ld), lo((int)((int64_t)a.n * slice / slices)),
          hi((int)((int64_t)a.n * (slice + 1) / slices)) {
        load(lo + threadIdx.x);
    }
    template <typename F>
    __device__ __forceinline__ void walk(F f) {  // f(index, logit)
        for (int base = lo + threadIdx.x;;) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (base + j * kThreads < hi) f(base + j * kThreads, v[j]);
            base += 8 * kThreads;
            if (base >= hi) break;
            load(base);
        }
    }
};

// All slices' bounds, the same in every thread (a slice per lane).
__device__ __forceinline__ Bound row_bound(const RowWork& w, int slices) {
    Bound b = w.bound[min((int)(threadIdx.x & (kMaxSlices - 1)), slices - 1)];
#pragma unroll
    for (int d = kMaxSlices / 2; d; d >>= 1) {
        b.best = max(b.best, (uint64_t)__shfl_xor((unsigned long long)b.best, d));
        b.least = min(b.least, (uint32_t)__shfl_xor((int)b.least, d));
    }
    return b;
}

// Logits to bins, in the order of the logits: every step rounds monotonically.
struct Bins {
    float top, per;
    bool clipped;  // the last bin holds what lies 30 temperatures and more below: masses of zero
    __device__ __forceinline__ float place(float l) const { return (top - l) * per; }
    __device__ __forceinline__ int at(float l) const { return (int)fminf(place(l), (float)(kBins - 1)); }
};
__device__ __forceinline__ Bins bins_of(const Bound& b, const Settings& s) {
    Bins r;
    r.top = logit_of((uint32_t)(b.best >> 32));
    const float all = r.top - logit_of(b.least);
    const double most = 30.0 / s.inv_t;  // (e^-30 (1 - 1/kBins) 2^42 = 0.43)
    r.clipped = (double)all > most;
    const float range = r.clipped ? (float)most : all;
    r.per = range > 1e-30f ? (float)kBins / range : 0.f;
    return r;
}
__device__ __forceinline__ bool by_bins(const Bound& b, const Settings& s) {
    // (an infinite range, from an infinite largest logit or the type's two ends, has no bins)
    return b.best && !s.greedy && logit_of((uint32_t)(b.best >> 32)) - logit_of(b.least) < INFINITY;
}

struct BoundShared {
    uint64_t best[kThreads / 64];
    uint32_t least[kThreads / 64];
};
// The workgroup's, the same in every thread.
__device__ __forceinline__ Bound block_bound(uint64_t best, uint32_t least, BoundShared& sh) {
#pragma unroll
    for (int d = 32; d; d >>= 1) {
        best = max(best, (uint64_t)__shfl_xor((unsigned long long)best, d));
        least = min(least, (uint32_t)__shfl_xor((int)least, d));
    }
    if ((threadIdx.x & 63) == 0) sh.best[threadIdx.x >> 6] = best, sh.least[threadIdx.x >> 6] = least;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kThreads / 64; ++i) best = max(best, sh.best[i]), least = min(least, sh.least[i]);
    __syncthreads();
    return Bound{best, least, 0};
}

__global__ void __launch_bounds__(kThreads) sample_bounds_kernel(SampleArgs a, void* ws, int slices) {
    __shared__ BoundShared sh;
    const int r = blockIdx.y, slice = blockIdx.x;
    const RowWork w = row_work(ws, r, slices);
    Slice logits(a, r, slice, slices);
    uint64_t best = 0;
    uint32_t least = ~0u;
    logits.walk([&](int i, float l) {
        const uint32_t k = key_of(l);
        if (!k) return;
        best = max(best, (uint64_t)k << 32 | (uint32_t)~i);
        least = min(least, k);
    });
    const Bound b = block_bound(best, least, sh);
    if (threadIdx.x == 0) w.bound[slice] = b;
}

__global__ void __launch_bounds__(kThreads) sample_bins_kernel(SampleArgs a, void* ws, int slices) {
    __shared__ unsigned long long mass[kBins];
    __shared__ unsigned count[kBins];
    __shared__ double pow2[32];
    const int r = blockIdx.y, slice = blockIdx.x;
    const RowWork w = row_work(ws, r, slices);
    Slice logits(a, r, slice, slices);
    const Settings s = settings_of(a, r);
    const Bound b = row_bound(w, slices);
    if (!by_bins(b, s)) return;
    const Bins bins = bins_of(b, s);
    const bool counts = s.k, masses = !s.k || s.k > kFewKept;
    mass[threadIdx.x] = 0;
    count[threadIdx.x] = 0;
    fill_pow2(pow2);
    const Masses mass_of(bins.top, s.inv_t, pow2);
    __syncthreads();
    logits.walk([&](int, float l) {
        if (!(l > -INFINITY)) return;
        const int bin = bins.at(l);
        if (counts) atomicAdd(&count[bin], 1u);
        if (masses) {
            const uint64_t m = mass_of(l);
            if (m) atomicAdd(&mass[bin], (unsigned long long)m);
        }
    });
    __syncthreads();
    if (counts) w.count[slice * kBins + threadIdx.x] = count[threadIdx.x];
    if (masses) w.mass[slice * kBins + threadIdx.x] = mass[threadIdx.x];
}

// Inclusive prefix sums over the workgroup.
template <typename T>
__device__ __forceinline__ T scan(T v, T* part) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    v = wave_scan(v);
    __syncthreads();
    if (lane == 63) part[wave] = v;
    __syncthreads();
    T before = 0;
#pragma unroll
    for (int i = 0; i < kThreads / 64; ++i) before += i < wave ? part[i] : 0;
    return v + before;
}

// Which of the row's bins are wanted (thread b: bin b). Every border lies between a
// lowest and a highest value that follow from the bins alone; a bin is wanted where it
// meets one of these ranges.
struct Wanted {
    bool mine;
    uint64_t above, total, sure;
    unsigned before;
};
__device__ Wanted wanted_bins(const RowWork& w, int slices, const Settings& s, const Bins& bins,
                              unsigned long long* part, unsigned long long* box) {
    const int b = threadIdx.x;
    uint64_t m = 0;
    unsigned c = 0;
    const bool counts = s.k, masses = !s.k || s.k > kFewKept;
    // (eight slices' values requested before the first is added)
    for (int i0 = 0; i0 < slices; i0 += 8) {
        unsigned vc[8];
        unsigned long long vm[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int at = min(i0 + i, slices - 1) * kBins + b;
            vc[i] = counts ? w.count[at] : 0;
            vm[i] = masses ? w.mass[at] : 0;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i0 + i < slices) c += vc[i], m += vm[i];
    }
    Wanted r{};
    unsigned long long candidates = 0;
    if (counts) {
        const unsigned long long upto = scan((unsigned long long)c, part);
        r.before = (unsigned)upto - c;
        if (b == kBins - 1) box[0] = upto;
        __syncthreads();
        candidates = box[0];
        __syncthreads();
    }
    const bool dead = bins.clipped && b == kBins - 1;  // masses of zero
    if (!masses) {
        r.mine = c && r.before < (unsigned)s.k && !dead;
        return r;
    }
    const unsigned long long upto = scan((unsigned long long)m, part);
    r.above = upto - m;
    // The borders are worked out by the first wave alone (64 rows: 2 us less than with every wave at it).
    // box: total; the first top_k's mass, at least and at most; top_p's target, at least and at
    // most; its prefix at most; min_p's bins' mass before and with; the draw's target, both; min_p's bin.
    const bool first_wave = threadIdx.x < 64;
    if (b == kBins - 1) box[0] = box[1] = box[2] = box[5] = box[6] = box[7] = upto;
    if (first_wave && s.m > 0.f) {  // the bin of the logit whose e is min_p
        // (rounded, as a bin's place is: the border lies in it or in a neighbour, for kBins in the last bin)
        const float cut = (float)(-least_z(s) / s.inv_t) * bins.per;
        if (b == 0) box[10] = cut < (float)(kBins + 1) ? (int)cut : 2 * kBins;
    }
    __syncthreads();
    r.total = box[0];
    if (s.k && (unsigned)s.k < candidates && r.before < (unsigned)s.k && (unsigned)s.k <= r.before + c && !dead) {
        r.mine = true;
        box[1] = max(r.above, (uint64_t)1);
        box[2] = upto;
    }
    if (s.m > 0.f) {
        const int cut = (int)box[10], first = max(cut - 1, 0), last = min(cut + 1, kBins - 1);
        if (cut <= kBins) {  // its bin and the neighbours
            if (m && b >= first && b <= last) r.mine = true;
            if (b == first) box[6] = r.above;
            if (b == last) box[7] = upto;
        }
    }
    __syncthreads();
    r.sure = box[6];
    if (s.p < 1.f) {
        if (first_wave) {
            const uint64_t lo = p_target(s, box[1]), hi = p_target(s, box[2]);
            if (b == 0) box[3] = lo, box[4] = hi;
        }
        __syncthreads();
        if (m && r.above < box[4] && upto >= box[3]) {
            r.mine = true;
            if (upto >= box[4]) box[5] = upto;  // (the one in which the highest target lies)
        }
        __syncthreads();
    }
    if (first_wave) {
        uint64_t lo = min((uint64_t)box[1], max((uint64_t)box[6], (uint64_t)1));
        if (s.p < 1.f) lo = min(lo, (uint64_t)box[3]);
        const uint64_t hi = min(min((uint64_t)box[2], (uint64_t)box[7]), (uint64_t)box[5]);
        const uint64_t u_lo = u_target(s, lo), u_hi = u_target(s, hi);
        if (b == 0) box[8] = u_lo, box[9] = u_hi;
    }
    __syncthreads();
    if (m && r.above <= box[9] && upto > box[8]) r.mine = true;
    return r;
}

__global__ void __launch_bounds__(kThreads) sample_collect_kernel(SampleArgs a, void* ws, int slices) {
    __shared__ unsigned long long part[kThreads / 64], box[11], list[kList];
    __shared__ unsigned long long want[kBins / 64];
    __shared__ unsigned count;
    const int r = blockIdx.y, slice = blockIdx.x;
    const RowWork w = row_work(ws, r, slices);
    Slice logits(a, r, slice, slices);
    const Settings s = settings_of(a, r);
    const Bound b = row_bound(w, slices);
    if (!by_bins(b, s)) return;
    const Bins bins = bins_of(b, s);
    const Wanted mine = wanted_bins(w, slices, s, bins, part, box);
    const unsigned long long bits = __ballot(mine.mine);
    if ((threadIdx.x & 63) == 0) want[threadIdx.x >> 6] = bits;
    if (threadIdx.x == 0) count = 0;
    if (slice == 0) {
        w.above[threadIdx.x] = mine.above;
        w.before[threadIdx.x] = mine.before;
        if (threadIdx.x == 0) w.total[0] = mine.total, w.total[1] = mine.sure;
    }
    __syncthreads();
    logits.walk([&](int i, float l) {
        if (!(l > -INFINITY)) return;
        const int bin = bins.at(l);
        if (!((want[bin >> 6] >> (bin & 63)) & 1)) return;
        const unsigned at = atomicAdd(&count, 1u);
        if (at < kList) list[at] = (unsigned long long)key_of(l) << 32 | (uint32_t)~i;
    });
    __syncthreads();
    if (threadIdx.x == 0) w.listed[slice] = count;
    for (unsigned i = threadIdx.x; i < min(count, (unsigned)kList); i += kThreads) w.list[slice * kList + i] = list[i];
}

// `n` values in descending order, by bitonic merges over the next power of two (zeros
// behind them). A thread holds values t and, PER > 1, t + 1024, ..: exchanges over fewer than 64
// places are lane exchanges, over 1024 and more register ones; only those between go
// through LDS and its barriers.
template <int PER>
__device__ void sort_list(unsigned long long* v, int n, int size) {
    const int t = threadIdx.x;
    unsigned long long x[PER];
#pragma unroll
    for (int r = 0; r < PER; ++r) x[r] = r * kThreads + t < n ? v[r * kThreads + t] : 0;
    for (int k = 2; k <= size; k <<= 1)
        for (int j = k >> 1; j; j >>= 1) {
            if (j >= kThreads) {
                if constexpr (PER == 4) {
                    // places r and r ^ (j / 1024)
#pragma unroll
                    for (int r = 0; r < PER; ++r) {
                        const int o = r ^ 1, o2 = r ^ 2;
                        const bool down = !((r * kThreads) & k);
                        if (j == kThreads && r < o && (x[r] < x[o]) == down) {
                            const unsigned long long y = x[r];
                            x[r] = x[o], x[o] = y;
                        }
                        if (j == 2 * kThreads && r < o2 && (x[r] < x[o2]) == down) {
                            const unsigned long long y = x[r];
                            x[r] = x[o2], x[o2] = y;
                        }
                    }
                }
                continue;
            }
            unsigned long long y[PER];
            if (j >= 64) {
                __syncthreads();
#pragma unroll
                for (int r = 0; r < PER; ++r) v[r * kThreads + t] = x[r];
                __syncthreads();
#pragma unroll
                for (int r = 0; r < PER; ++r) y[r] = v[r * kThreads + (t ^ j)];
            } else {
#pragma unroll
                for (int r = 0; r < PER; ++r) y[r] = __shfl_xor(x[r], j);
            }
#pragma unroll
            for (int r = 0; r < PER; ++r) {
                const bool larger = !((r * kThreads + t) & k) == !(t & j);  // this place keeps the larger one
                x[r] = (x[r] < y[r]) == larger ? y[r] : x[r];
            }
        }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < PER; ++r) v[r * kThreads + t] = x[r];
    __syncthreads();
}
// Short lists: a value's place is the number of larger ones (no two are equal), counted
// by 1024 / 256 threads each. 60 values: 0.6 us, by merges 3.4.
constexpr int kShort = 256;
__device__ void rank_list(unsigned long long* v, unsigned* rank, int n) {
    const int e = threadIdx.x % kShort, part = threadIdx.x / kShort;
    if (threadIdx.x < kShort) rank[threadIdx.x] = 0;
    const unsigned long long mine = e < n ? v[e] : 0;
    __syncthreads();
    constexpr int PARTS = kThreads / kShort;
    unsigned larger = 0;
    for (int i = part; i < n; i += PARTS) larger += v[i] > mine;
    if (e < n) atomicAdd(&rank[e], larger);
    __syncthreads();
    if (threadIdx.x < n) v[rank[threadIdx.x]] = mine;
    __syncthreads();
}
// Longer lists of a row with bins: the few bins that they come from, cut finer so that there are up to
// kBins again, in the order of the logits; then by counting within each of these. False, and nothing
// changed, where one has more than kPerBin values (many equal logits). 1,300 values from three bins:
// 3 us, by counting within the three 16, by merges 15.
constexpr unsigned kPerBin = 64;
struct BinSort {
    unsigned count[kBins], start[kBins], part[kThreads / 64], most, bins;
};
__device__ bool bin_list(unsigned long long* v, BinSort& sh, const Bins& bins, int n) {
    constexpr int PER = kList / kThreads;
    unsigned long long x[PER];
    int bin[PER];
    unsigned at[PER];
    sh.count[threadIdx.x] = 0;
    if (threadIdx.x == 0) sh.most = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int i = j * kThreads + threadIdx.x;
        if (i >= n) continue;
        x[j] = v[i];
        bin[j] = bins.at(logit_of((uint32_t)(x[j] >> 32)));
        sh.count[bin[j]] = 1;
    }
    __syncthreads();
    const unsigned used = sh.count[threadIdx.x], number = scan(used, sh.part);
    sh.start[threadIdx.x] = number - used;
    if (threadIdx.x == kThreads - 1) sh.bins = number;
    sh.count[threadIdx.x] = 0;
    __syncthreads();
    int fine = kBins;  // parts of a bin: kBins / (bins used, up to a power of two)
    while (fine > 1 && fine * sh.bins > kBins) fine >>= 1;
    unsigned own[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        if (j * kThreads + (int)threadIdx.x >= n) continue;
        own[j] = sh.start[bin[j]];
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        if (j * kThreads + (int)threadIdx.x >= n) continue;
        const float z = bins.place(logit_of((uint32_t)(x[j] >> 32))) - (float)bin[j];
        bin[j] = own[j] * fine + max(min((int)(z * (float)fine), fine - 1), 0);
        at[j] = atomicAdd(&sh.count[bin[j]], 1u);
    }
    __syncthreads();
    const unsigned c = sh.count[threadIdx.x];
    if (c > kPerBin) sh.most = c;
    sh.start[threadIdx.x] = scan(c, sh.part) - c;
    __syncthreads();
    if (sh.most) return false;
#pragma unroll
    for (int j = 0; j < PER; ++j)
        if (j * kThreads + (int)threadIdx.x < n) v[sh.start[bin[j]] + at[j]] = x[j];
    __syncthreads();
#pragma unroll
    for (int j = 0; j < PER; ++j)
        if (j * kThreads + (int)threadIdx.x < n) {
            const unsigned first = sh.start[bin[j]], end = first + sh.count[bin[j]];
            at[j] = first;
            for (unsigned i = first; i < end; ++i) at[j] += v[i] > x[j];
        }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < PER; ++j)
        if (j * kThreads + (int)threadIdx.x < n) v[at[j]] = x[j];
    __syncthreads();
    return true;
}
__device__ __forceinline__ void sort_list(unsigned long long* v, int n) {
    int size = 2;
    while (size < n) size <<= 1;
    if (size <= kThreads) sort_list<1>(v, n, size);
    else sort_list<kList / kThreads>(v, n, size);
}

struct DrawShared {
    unsigned long long first_sum[kBins];
    unsigned first_at[kBins];
    unsigned long long part[kThreads / 64], box[3];
    double least_z;
};

// The draw from the sorted list, PER candidates per thread: mass, running sum and rank of
// each. A list that starts with the row's first candidate needs no more; otherwise
// each bin's own run continues from what lies above the bin.
template <int PER>
__device__ void draw(const SampleArgs& a, void* ws, int slices, int r, const Settings& s, const Bins& bins,
                     const Masses& mass_of, const unsigned long long* list, unsigned n,
                     DrawShared& sh) {
    const bool prefix = !slices || (s.k && s.k <= kFewKept);
    const unsigned i0 = threadIdx.x * PER;
    uint64_t m[PER], end[PER], sum = 0;
    unsigned rank[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        m[j] = i0 + j < n ? mass_of(logit_of((uint32_t)(list[i0 + j] >> 32))) : 0;
        sum += m[j];
    }
    uint64_t run = scan((unsigned long long)sum, sh.part) - sum;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const unsigned i = i0 + j;
        run += m[j];
        end[j] = run;
        rank[j] = i;
        if (!prefix && i < n) {
            const int bin = bins.at(logit_of((uint32_t)(list[i] >> 32)));
            if (i == 0 || bins.at(logit_of((uint32_t)(list[i - 1] >> 32))) != bin) {
                sh.first_sum[bin] = run - m[j];
                sh.first_at[bin] = i;
            }
        }
    }
    const RowWork w = row_work(ws, r, max(slices, 1));
    // box: the mass of the first top_k, of top_p's prefix, of min_p's
    if (threadIdx.x == kThreads - 1) {
        const uint64_t all = prefix ? run : w.total[0];
        sh.box[0] = sh.box[1] = all;
        sh.box[2] = prefix ? 0 : w.total[1];
    }
    if (threadIdx.x < 64) {  // (a logarithm by one wave)
        const double z = least_z(s);
        if (threadIdx.x == 0) sh.least_z = z;
    }
    __syncthreads();
    const double least = sh.least_z;
    uint64_t large = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const unsigned i = i0 + j;
        if (i >= n) continue;
        if (!prefix) {
            const int bin = bins.at(logit_of((uint32_t)(list[i] >> 32)));
            end[j] += w.above[bin] - sh.first_sum[bin];
            rank[j] += w.before[bin] - sh.first_at[bin];
        }
        if (s.k && rank[j] == (unsigned)s.k - 1) sh.box[0] = end[j];
        if (mass_of.keeps(logit_of((uint32_t)(list[i] >> 32)), least)) large = end[j];
    }
    // (the last candidate that min_p keeps: of a wave, in the last lane that has one)
    const unsigned long long keeps = __ballot(large != 0);
    if (keeps && (int)(threadIdx.x & 63) == 63 - __clzll(keeps)) atomicMax(&sh.box[2], (unsigned long long)large);
    __syncthreads();
    uint64_t kept = sh.box[0];
    if (s.p < 1.f) {
        const uint64_t target = p_target(s, kept);
#pragma unroll
        for (int j = 0; j < PER; ++j)
            if (i0 + j < n && end[j] >= target && end[j] - m[j] < target) sh.box[1] = end[j];
        __syncthreads();
        kept = min(kept, (uint64_t)sh.box[1]);
    }
    kept = min(kept, (uint64_t)sh.box[2]);
    const uint64_t at = u_target(s, kept);
#pragma unroll
    for (int j = 0; j < PER; ++j)
        if (i0 + j < n && end[j] - m[j] <= at && at < end[j]) {  // (one candidate: the runs do not overlap)
            a.tokens[r] = (int)~(uint32_t)list[i0 + j];
            if (a.probs) a.probs[r] = (float)((double)m[j] / (double)kept);
        }
}

__global__ void __launch_bounds__(kThreads) sample_finish_kernel(SampleArgs a, void* ws, int slices) {
    __shared__ unsigned long long list[kList];
    __shared__ union {
        RowShared row;
        BoundShared bounds;
        unsigned rank[kShort];
        BinSort bins;
        DrawShared l;
    } sh;
    __shared__ unsigned listed;
    __shared__ double pow2[32];
    const int r = blockIdx.x;
    fill_pow2(pow2);  // (barriers follow before it is read)
    const float* row = a.logits + r * a.ld;
    const Settings s = settings_of(a, r);
    int token = -1;
    float prob = 0.f;
    Bound b{};
    Bins bins{};
    unsigned n = 0;
    const bool whole = !slices;  // all of the row's candidates
    if (whole) {
        constexpr int PER = kList / kThreads;
        float l[PER];
        uint64_t best = 0;
        uint32_t least = ~0u;
#pragma unroll
        for (int j = 0; j < PER; ++j) l[j] = row[min(j * kThreads + (int)threadIdx.x, a.n - 1)];
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int i = j * kThreads + threadIdx.x;
            const uint32_t k = key_of(l[j]);
            if (!k || i >= a.n) continue;
            best = max(best, (uint64_t)k << 32 | (uint32_t)~i);
            least = min(least, k);
        }
        b = block_bound(best, least, sh.bounds);
        if (b.best && !s.greedy) {
            // the candidates whose mass is not zero for certain
            bins = bins_of(b, s);
            const bool binned = by_bins(b, s), some = binned && bins.clipped;
            bool mine[PER];
            unsigned count = 0;
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                mine[j] = j * kThreads + (int)threadIdx.x < a.n && l[j] > -INFINITY &&
                          !(some && bins.at(l[j]) == kBins - 1);
                count += mine[j];
            }
            const unsigned upto = scan(count, sh.bins.part);
            if (threadIdx.x == kThreads - 1) listed = upto;
            unsigned at = upto - count;
#pragma unroll
            for (int j = 0; j < PER; ++j)
                if (mine[j])
                    list[at++] = (unsigned long long)key_of(l[j]) << 32 | (uint32_t)~(j * kThreads + threadIdx.x);
            __syncthreads();
            n = listed;
            if (n <= kShort) rank_list(list, sh.rank, n);
            else if (!binned || !bin_list(list, sh.bins, bins, n)) sort_list(list, n);
        }
    } else {
        // the slices' lists, 64 threads to a slice: the first 64 of each are requested before the counts are known
        const RowWork w = row_work(ws, r, slices);
        const int slice = threadIdx.x >> 6, lane = threadIdx.x & 63;
        const unsigned long long* mine = w.list + min(slice, slices - 1) * kList;
        const unsigned long long early = mine[lane];
        const unsigned count = lane < slices ? w.listed[lane] : 0;
        b = row_bound(w, slices);
        if (b.best && !s.greedy) {
            bins = bins_of(b, s);
            unsigned from = 0, own = 0;
            if (by_bins(b, s)) {
#pragma unroll
                for (int i = 0; i < kMaxSlices; ++i) {
                    const unsigned c = __shfl(count, i);
                    from += i < slice ? c : 0;
                    own = i == slice ? c : own;
                    n += c;
                }
            } else {
                n = kList + 1;
            }
            if (n > kList) {
                __syncthreads();
                sample_row(sh.row, row, a.n, s, Masses(logit_of((uint32_t)(b.best >> 32)), s.inv_t, pow2), &token, &prob);
                if (threadIdx.x == 0) {
                    a.tokens[r] = token;
                    if (a.probs) a.probs[r] = prob;
                }
                return;
            }
            if (lane < own) list[from + lane] = early;
            for (unsigned i = 64 + lane; i < own; i += 64) list[from + i] = mine[i];
            __syncthreads();
            if (n <= kShort) rank_list(list, sh.rank, n);
            else if (!bin_list(list, sh.bins, bins, n)) sort_list(list, n);
        }
    }
    if (b.best && s.greedy) {
        token = (int)~(uint32_t)b.best;
        prob = 1.f;
    } else if (b.best) {
        const Masses mass_of(logit_of((uint32_t)(b.best >> 32)), s.inv_t, pow2);
        if (n <= kThreads) draw<1>(a, ws, slices, r, s, bins, mass_of, list, n, sh.l);
        else draw<kList / kThreads>(a, ws, slices, r, s, bins, mass_of, list, n, sh.l);
        return;
    }
    if (threadIdx.x == 0) {
        a.tokens[r] = token;
        if (a.probs) a.probs[r] = prob;
    }
}

// Slices per row: a workgroup per CU (64 rows: 2.5 % less than with two), of 4096 logits at least.
int slices_of(int rows, int n, int cus) {
    int s = (cus + rows - 1) / rows;
    if (s > kMaxSlices) s = kMaxSlices;
    const int most = (n + kList - 1) / kList;
    return s < most ? s : most;
}

}  // namespace

size_t sample_workspace(int rows, int n, int cus) {
    if (n <= kList) return 0;
    const int at_once = rows < kRowsAtOnce ? rows : kRowsAtOnce;
    return at_once * row_work_bytes(slices_of(at_once, n, cus));
}

hipError_t launch_sample(const SampleArgs& all, void* workspace, int cus, hipStream_t stream) {
    const int at_once = all.n <= kList ? all.rows : all.rows < kRowsAtOnce ? all.rows : kRowsAtOnce;
    const int slices = all.n <= kList ? 0 : slices_of(at_once, all.n, cus);
    for (int row = 0; row < all.rows; row += at_once) {
        SampleArgs a = all;
        a.rows = all.rows - row < at_once ? all.rows - row : at_once;
        a.logits += row * all.ld;
        a.u += row;
        a.temperature += a.temperature ? row : 0;
        a.top_k += a.top_k ? row : 0;
        a.top_p += a.top_p ? row : 0;
        a.min_p += a.min_p ? row : 0;
        a.tokens += row;
        a.probs += a.probs ? row : 0;
        const dim3 grid(slices, a.rows);
        if (slices) {
            hipLaunchKernelGGL(sample_bounds_kernel, grid, dim3(kThreads), 0, stream, a, workspace, slices);
            hipLaunchKernelGGL(sample_bins_kernel, grid, dim3(kThreads), 0, stream, a, workspace, slices);
            hipLaunchKernelGGL(sample_collect_kernel, grid, dim3(kThreads), 0, stream, a, workspace, slices);
        }
        hipLaunchKernelGGL(sample_finish_kernel, dim3(a.rows), dim3(kThreads), 0, stream, a, workspace, slices);
    }
    return hipGetLastError();
}

}  // namespace rq
