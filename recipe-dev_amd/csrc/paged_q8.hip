// Queries and keys on their way to 8-bit pages, and the pages' values
// (rqmv_qk_norm_rope_q8, rqmv_paged_values_q8).
#include "lanes.h"
#include "paged_rows.h"
#include "q8.h"

namespace rq {

// Queries as in rqmv_qk_norm_rope. Keys and values are stored by runs: the rows of
// a call that fall into one group (16 slots) lie within 32 rows, and for the first
// of them a workgroup stores all, once for each kv head's keys and once for its values. With
//     e(a) = the smallest e in -24..9 with a < 127.5 * 2^e      (none: NaN)
// and a the run's largest magnitude, the group's exponent becomes e' = e(a) where
// the run holds the group's first row, which starts the group anew (its
// other rows become 0), and max(e, e(a)) otherwise; then the other rows' codes
// are c -> rint(c * 2^(e - e')) and the run's rint(y * 2^-e').
//
// A code is a whole number next to its borders, so keys are computed in 64 bits: a key's codes are those of the
// exact key, whatever the step it came in. (With keys in fp32 a prefill step of 3,480 rows took 4 us less of 48, before the
// rest was made faster.)
//
// A run's sixteen rows are shared by four waves, which join their exponents through LDS. Runs are looked for among the
// window of rows that a workgroup has; workgroups of runs come before those of queries (mixed, they
// wait for each other's loads: 85 us).
//
// Bound: at prefill HBM (3,480 rows of 32/8 heads of 128, fp32 to fp16: 27.3 us in a trace, the form over fp16 pages
// 25.5), at decode the chain of loads slots -> rows -> codes (24 requests: 4.3 us in a trace).
constexpr int kWaves = 4;

// Queries and the values of pages pass by the caches (3,480 rows, 32/8 heads of 128, with the values: 38.2 us, so 35.1;
// attention behind the append takes as long as after plain stores).
typedef uint32_t nt2_t __attribute__((ext_vector_type(2)));
typedef uint32_t nt4_t __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void stream4(float* p, const float* v) {
    __builtin_nontemporal_store(nt4_t{__builtin_bit_cast(uint32_t, v[0]), __builtin_bit_cast(uint32_t, v[1]),
                                      __builtin_bit_cast(uint32_t, v[2]), __builtin_bit_cast(uint32_t, v[3])},
                                reinterpret_cast<nt4_t*>(p));
}
__device__ __forceinline__ void stream4(__half* p, const float* v) {
    __builtin_nontemporal_store(nt2_t{__builtin_bit_cast(uint32_t, __floats2half2_rn(v[0], v[1])),
                                      __builtin_bit_cast(uint32_t, __floats2half2_rn(v[2], v[3]))},
                                reinterpret_cast<nt2_t*>(p));
}
__device__ __forceinline__ void stream4(uint4* p, uint4 v) {
    __builtin_nontemporal_store(nt4_t{v.x, v.y, v.z, v.w}, reinterpret_cast<nt4_t*>(p));
}

constexpr int kRunRows = 32;  // rows that a run's rows lie within
// Windows of 16 rows where a call has many (a prompt's 1000 rows of 32/8 heads of 128, with the values: 13.3 us, of 4 rows
// 15.0; 3,480 rows 38 and 45), of 4 for some, whose runs are short and would wait for each other (300 requests 18.7, of 16
// rows 34.2), of one for few (24 requests 8.7, of 4 rows 10.4; but a prompt of 128 takes 10.7 so, of 4 rows 8.6). The number of
// rows alone decides, so more than 512 requests of one token go by windows of 16 too: 1000 take 28.6 us by themselves, a
// prompt of 1000 rows 9.6, either over fp16 pages 9.3 and 8.3.
constexpr int kFewRows = 64, kSomeRows = 512;

// The slots around a window: of rows base - 31 .. base + 32 (`a`) and the sixteen after these (`b`); -1: none.
struct Slots {
    int a, b;
    int position;  // (lane i: of row base + i)
    // Of row base + at, from -31 to 48.
    __device__ __forceinline__ int of(int at) const {
        const int i = at + kRunRows - 1;
        return i < 64 ? __builtin_amdgcn_readlane(a, i) : __builtin_amdgcn_readlane(b, i - 64);
    }
    // The rows of row base + at's group among itself and the 31 behind it; 0: it has no slot, or one of the 31 before
    // it is of the group.
    __device__ __forceinline__ uint32_t run(int at) const {
        const int mine = of(at);
        if (mine < 0) return 0;
        const unsigned long long in_a = __ballot(a >= 0 && (a >> 4) == (mine >> 4));
        const unsigned long long in_b = __ballot(b >= 0 && (b >> 4) == (mine >> 4));
        if ((in_a >> at) & 0x7FFFFFFFull) return 0;
        return (uint32_t)(in_a >> (kRunRows - 1 + at) | in_b << (kRunRows + 1 - at));
    }
};

template <int HD, typename F>
__device__ __forceinline__ void store_run(const PagedBatch& b, const PagedCache& c, const PagedCodes& codes,
                                          const QkNormRope& p, int base, int at0, const Slots& slots, uint32_t run, int item,
                                          const HeadLane& norm, float* exponents, F load8) {
    constexpr int LPH = HD / 8, ROWS = 64 / LPH, PASSES = ROWS * kWaves < kGroup ? kGroup / (ROWS * kWaves) : 1;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), u = lane % LPH;
    const bool value = item >= c.kv_heads;
    const int kh = value ? item - c.kv_heads : item;
    const int mine = slots.of(at0);
    const int block = mine >> c.block_shift, first = mine & ((1 << c.block_shift) - 1) & ~(kGroup - 1);
    const int64_t row0 = (((int64_t)block * c.kv_heads + kh) << c.block_shift) + first;
    uint8_t* scale_at = (value ? codes.v_scale : codes.k_scale) + (row0 >> 4);
    int8_t* rows = (value ? codes.v : codes.k) + row0 * HD;
    const unsigned old_byte = *scale_at;
    // lane r < n: the run's row r as an offset from the first, and its row in the group (of the first sixteen)
    const int n = min((int)__popc(run), kGroup);
    int off = lane, in_group = (mine + lane) & (kGroup - 1);
    unsigned stored = ((1u << n) - 1) << (mine & (kGroup - 1));
    const int ahead = lane - (kRunRows - 1 + at0);
    if (run != (1u << n) - 1 || at0 + n > kRunRows || __any(ahead >= 0 && ahead < n && slots.a != mine + ahead)) {
        stored = 0;  // not rows next to each other with slots in their order
        for (int r = 0; r < n; ++r, run &= run - 1) {
            const int d = __builtin_ctz(run), g = slots.of(at0 + d) & (kGroup - 1);
            off = lane == r ? d : off;
            in_group = lane == r ? g : in_group;
            stored |= 1u << g;
        }
    }

    // the wave's rows and their largest magnitude (lanes past the last row repeat it)
    const HeadPlace place = head_place<HD>(p, value, u);
    double y[PASSES][8];
    float x[PASSES][8], exponent = kScaleLow;  // (of magnitudes without one: kScaleHigh + 1)
    HeadLane h[PASSES];
    auto row_of = [&](int i) { return (i * kWaves + wave) * ROWS + lane / LPH; };
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        const int at = at0 + __shfl(off, min(row_of(i), n - 1));
        load8(base + at, p.q_heads + item, place, x[i]);
        h[i] = norm;
        load_turn(p, __shfl(slots.position, at), place.turns ? u : 0, h[i]);
    }
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        if ((i * kWaves + wave) * ROWS >= n) break;
#pragma unroll
        for (int e = 0; e < 8; ++e) y[i][e] = x[i][e];
        if (!value) norm_and_turn<HD>(p.k_norm, place.turns, p.eps, h[i], y[i]);
        double top = 0;
        bool wild = false;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            top = fmax(top, fabs(y[i][e]));
            wild |= !(fabs(y[i][e]) < 127.5 * (1 << kScaleHigh));
        }
        const int ex = __builtin_amdgcn_frexp_exp(top) - 7;  // (of 0: 0, so compared)
        const int own = top > 0 ? ex + (__builtin_amdgcn_frexp_mant(top) * 128.0 >= 127.5 ? 1 : 0) : kScaleLow;
        exponent = fmaxf(exponent, wild ? (float)(kScaleHigh + 1) : (float)own);
    }
    exponent = all_max(exponent);
    const int old = __builtin_amdgcn_readfirstlane((int)old_byte);  // (here before any wave writes it)
    if (lane == 0) exponents[wave] = exponent;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) exponent = fmaxf(exponent, exponents[w]);
    int e = (int)exponent;
    const bool none = e > kScaleHigh;
    const bool anew = stored & 1;
    const int e_old = min(max(old - 127, kScaleLow), kScaleHigh);
    if (!anew) e = max(e, e_old);
    const bool nan = none || (!anew && old == kScaleNan);
    if (threadIdx.x == 0) *scale_at = (uint8_t)(nan ? kScaleNan : e + 127);

    // the group's other rows, 1024 bytes a wave
    if (anew || e > e_old) {
        const float f = ldexpf(1.f, e_old - e);
        const int o = wave * 1024 + lane * 16;
        if (o < kGroup * HD && !((stored >> (o / HD)) & 1)) {
            uint4* q = reinterpret_cast<uint4*>(rows + o);
            uint32_t w[4] = {0, 0, 0, 0};
            if (!anew) {
                const uint4 v = *q;
                w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    uint32_t r = 0;
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        r |= ((uint32_t)(int)rintf((float)(int8_t)(w[k] >> (8 * j)) * f) & 255u) << (8 * j);
                    w[k] = r;
                }
            }
            *q = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }

    // the run's rows
    const double f = ldexp(1.0, -e);
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        if ((i * kWaves + wave) * ROWS >= n) break;
        const int r = row_of(i), g = __shfl(in_group, min(r, n - 1));
        uint32_t w[2] = {0, 0};
#pragma unroll
        for (int e8 = 0; e8 < 8; ++e8) {
            const double z = rint(y[i][e8] * f);
            const int code = fabs(z) <= 127.0 ? (int)z : 0;  // (else the group is NaN)
            w[e8 / 4] |= ((uint32_t)code & 255u) << (8 * (e8 % 4));
        }
        if (r < n) {
            *reinterpret_cast<uint32_t*>(rows + g * HD + place.lo) = w[0];
            *reinterpret_cast<uint32_t*>(rows + g * HD + place.hi) = w[1];
        }
    }
}

// Workgroups y < kv_groups take runs (by number: item by item, for each the windows of `few` or 16 rows), the others queries.
template <int HD, bool MANY, typename X, typename Q>
__global__ void __launch_bounds__(64 * kWaves) qk_q8_kernel(PagedBatch b, PagedCache c, PagedCodes codes, QkNormRope p,
                                                            int kv_groups, int few) {
    const int window = MANY ? 16 : few;
    constexpr int LPH = HD / 8, HPB = 64 * kWaves / LPH;  // lanes per head, heads per workgroup
    auto load8 = [&](int t, int head, HeadPlace at, float (&x)[8]) {
        const X* src = static_cast<const X*>(p.qkv) + (int64_t)t * p.ld + head * HD;
        load4<X>(src + at.lo, x);
        load4<X>(src + at.hi, x + 4);
    };
    if ((int)blockIdx.y < kv_groups) {
        __shared__ float exponents[2][kWaves];
        const int64_t number = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
        const int windows = (b.tokens - 1) / window + 1, item = (int)(number / windows);
        const int base = (int)(number % windows) * window, lane = threadIdx.x & 63;
        if (item >= 2 * c.kv_heads) return;
        const int64_t size = (int64_t)c.blocks << c.block_shift;
        auto slot_of = [&](int row) {
            const int s = row >= 0 && row < b.tokens ? b.slots[row] : -1;
            return s < size ? s : -1;
        };
        Slots slots;
        slots.a = slot_of(base - (kRunRows - 1) + lane);
        slots.b = lane < 16 ? slot_of(base + kRunRows + 1 + lane) : -1;
        slots.position = b.positions[min(base + lane, b.tokens - 1)];
        HeadLane norm{};
        if (p.k_norm && item < c.kv_heads) load_norm(p.k_norm, head_place<HD>(p, false, lane % LPH), norm);
        // (a row of the group of the row before it starts no run)
        const int before = __shfl_up(slots.a, 1);
        unsigned long long starts = __ballot(slots.a >= 0 && (before < 0 || (before >> 4) != (slots.a >> 4))) >> (kRunRows - 1);
        starts &= (1ull << window) - 1;
        int turn = 0;
        for (; starts; starts &= starts - 1) {
            const int at = __builtin_ctzll(starts);
            const uint32_t run = slots.run(at);
            if (!run) continue;
            store_run<HD>(b, c, codes, p, base, at, slots, run, item, norm, exponents[turn], load8);
            turn ^= 1;  // (a wave may be a run ahead)
        }
        return;
    }
    const int token = blockIdx.x, head = (blockIdx.y - kv_groups) * HPB + threadIdx.x / LPH, u = threadIdx.x % LPH;
    if (head >= p.q_heads) return;  // (whole lane groups leave)
    const HeadPlace at = head_place<HD>(p, false, u);
    float x[8];
    load8(token, head, at, x);
    HeadLane h{};
    if (p.q_norm) load_norm(p.q_norm, at, h);
    if (at.turns) load_turn(p, b.positions[token], u, h);
    norm_and_turn<HD>(p.q_norm, at.turns, p.eps, h, x);
    Q* dst = static_cast<Q*>(p.q_out) + (int64_t)token * p.ldq + head * HD;
    stream4(dst + at.lo, x);
    stream4(dst + at.hi, x + 4);
}

template <int HD, typename X>
static void launch_x(const PagedBatch& b, const PagedCache& c, const PagedCodes& codes, const QkNormRope& p, bool q_f16,
                     hipStream_t stream) {
    constexpr int HPB = 64 * kWaves / (HD / 8);
    const bool many = b.tokens > kSomeRows;
    const int few = b.tokens <= kFewRows ? 1 : 4, window = many ? 16 : few;
    const int64_t runs = (int64_t)((b.tokens - 1) / window + 1) * 2 * c.kv_heads;
    const int kv_groups = (int)((runs - 1) / b.tokens + 1);
    const dim3 grid(b.tokens, kv_groups + (p.q_heads + HPB - 1) / HPB), threads(64 * kWaves);
    auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, threads, 0, stream, b, c, codes, p, kv_groups, few); };
    if (many) q_f16 ? launch(qk_q8_kernel<HD, true, X, __half>) : launch(qk_q8_kernel<HD, true, X, float>);
    else q_f16 ? launch(qk_q8_kernel<HD, false, X, __half>) : launch(qk_q8_kernel<HD, false, X, float>);
}

template <int HD>
static void launch_hd(const PagedBatch& b, const PagedCache& c, const PagedCodes& codes, const QkNormRope& p, bool x_f16,
                      bool q_f16, hipStream_t stream) {
    if (x_f16) launch_x<HD, __half>(b, c, codes, p, q_f16, stream);
    else launch_x<HD, float>(b, c, codes, p, q_f16, stream);
}

hipError_t launch_qk_norm_rope_q8(const PagedBatch& b, const PagedCache& c, const PagedCodes& codes, const QkNormRope& p,
                                  bool x_f16, bool q_f16, hipStream_t stream) {
    if (c.head_dim == 64) launch_hd<64>(b, c, codes, p, x_f16, q_f16, stream);
    else if (c.head_dim == 128) launch_hd<128>(b, c, codes, p, x_f16, q_f16, stream);
    else launch_hd<256>(b, c, codes, p, x_f16, q_f16, stream);
    return hipGetLastError();
}

// ------------------------------------------------------------- the values ----

// Sixteen codes a thread; keys and values by blockIdx.y. Bound: HBM (the pages behind the step of 3,480 rows: 8.6 us in a trace).
__global__ void __launch_bounds__(256) values_q8_kernel(PagedCodes codes, __half* k, __half* v, int64_t pieces,
                                                        int row_shift) {
    const int8_t* from = blockIdx.y ? codes.v : codes.k;
    const uint8_t* scale = blockIdx.y ? codes.v_scale : codes.k_scale;
    __half* to = blockIdx.y ? v : k;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < pieces; i += (int64_t)gridDim.x * 256) {
        const uint4 x = reinterpret_cast<const uint4*>(from)[i];
        const Scale s = scale_of(scale[i >> (row_shift + 4)]);
        uint4* out = reinterpret_cast<uint4*>(to) + 2 * i;
        stream4(out, codes_to_h(make_uint2(x.x, x.y), s));
        stream4(out + 1, codes_to_h(make_uint2(x.z, x.w), s));
    }
}

hipError_t launch_paged_values_q8(const PagedCache& c, const PagedCodes& codes, __half* k, __half* v, hipStream_t stream) {
    const int row_shift = c.head_dim == 64 ? 2 : c.head_dim == 128 ? 3 : 4;  // log2 of a row's pieces of 16
    const int64_t pieces = (((int64_t)c.blocks * c.kv_heads) << c.block_shift) << row_shift;
    const int64_t groups = (pieces + 255) / 256;
    hipLaunchKernelGGL(values_q8_kernel, dim3((unsigned)(groups < 8192 ? groups : 8192), 2), dim3(256), 0, stream, codes, k,
                       v, pieces, row_shift);
    return hipGetLastError();
}

}  // namespace rq
