// Queries and keys on their way to 8-bit pages, and the pages' values
// (rqmv_qk_norm_rope_q8, rqmv_paged_values_q8).
#include "paged_rows.h"
#include "q8.h"

namespace rq {

// Queries as in rqmv_qk_norm_rope. Keys and values are stored by runs: the rows of
// a call that fall into one group (16 slots) lie within 32 rows, and the first of
// them has a wave for each kv head's keys and one for its values, which looks for the others. With
//     e(a) = the smallest e in -24..9 with a < 127.5 * 2^e      (none: NaN)
// and a the run's largest magnitude, the group's exponent becomes e' = e(a) where
// the run holds the group's first row, which starts the group anew (its
// other rows become 0), and max(e, e(a)) otherwise; then the other rows' codes
// are c -> rint(c * 2^(e - e')) and the run's rint(y * 2^-e').
//
// A code is a whole number next to its borders, so keys are computed in 64 bits
// (some 60 instructions per eight values, hidden behind the rows' loads): a key's
// codes are those of the exact key, whatever the step it came in.
//
// Bound: HBM at prefill, one launch at decode. A row that starts no run costs the
// exit of its waves.
constexpr int kWaves = 4;
constexpr int kRunRows = 32;  // rows that a run's rows lie within

template <int HD, typename F>
__device__ __forceinline__ void store_run(const PagedBatch& b, const PagedCache& c, const PagedCodes& codes,
                                          const QkNormRope& p, int token, int item, F load8) {
    constexpr int LPH = HD / 8, ROWS = 64 / LPH, PASSES = 16 / ROWS;
    const int lane = threadIdx.x & 63, u = lane % LPH;
    const int64_t slots = (int64_t)c.blocks << c.block_shift;
    // slots of rows token - 31 .. token + 31 (lanes 0..62); -1: none
    constexpr int BACK = kRunRows - 1;
    int slot = -1;
    if (lane < 2 * kRunRows - 1 && token - BACK + lane >= 0 && token - BACK + lane < b.tokens)
        slot = b.slots[token - BACK + lane];
    if (slot >= slots) slot = -1;
    const int mine = __builtin_amdgcn_readlane(slot, BACK);
    if (mine < 0) return;
    const unsigned long long same = __ballot(slot >= 0 && (slot >> 4) == (mine >> 4));
    if (same & ((1ull << BACK) - 1)) return;  // (a row before this one starts the run)
    // lane r < n: the run's row r as an offset from `token`, and its row in the group
    const int n = min((int)__popcll(same >> BACK), kGroup);
    int off = 0;
    unsigned stored = 0;
    unsigned long long left = same >> BACK;
    for (int r = 0; r < n; ++r, left &= left - 1) {
        const int d = __builtin_ctzll(left);
        off = lane == r ? d : off;
        stored |= 1u << (__builtin_amdgcn_readlane(slot, BACK + d) & (kGroup - 1));
    }
    slot = __shfl(slot, BACK + off) & (kGroup - 1);
    const bool value = item >= c.kv_heads;
    const int kh = value ? item - c.kv_heads : item;
    const int block = mine >> c.block_shift, first = mine & ((1 << c.block_shift) - 1) & ~(kGroup - 1);
    const int64_t row0 = (((int64_t)block * c.kv_heads + kh) << c.block_shift) + first;
    uint8_t* scale_at = (value ? codes.v_scale : codes.k_scale) + (row0 >> 4);
    int8_t* rows = (value ? codes.v : codes.k) + row0 * HD;
    const unsigned old = *scale_at;

    // the run's rows, ROWS at a time, and their largest magnitude
    const HeadPlace at = head_place<HD>(p, value, u);
    double y[PASSES][8], top = 0;
    bool wild = false;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        if (i * ROWS >= n) break;
        // (lanes past the last row repeat it)
        const int row = token + __shfl(off, min(i * ROWS + lane / LPH, n - 1));
        float x[8];
        load8(row, p.q_heads + item, at, x);
#pragma unroll
        for (int e = 0; e < 8; ++e) y[i][e] = x[e];
        if (!value) norm_and_turn<HD>(b, p, p.k_norm, at, row, u, y[i]);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            top = fmax(top, fabs(y[i][e]));
            wild |= !(fabs(y[i][e]) < 127.5 * (1 << kScaleHigh));
        }
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) top = fmax(top, __shfl_xor(top, d));
    const bool none = __any(wild);
    int e = kScaleLow;
    if (top > 0) {
        const int x = __builtin_amdgcn_frexp_exp(top);
        e = x - 7 + (__builtin_amdgcn_frexp_mant(top) * 128.0 >= 127.5 ? 1 : 0);
        e = min(max(e, kScaleLow), kScaleHigh);
    }
    const bool anew = stored & 1;
    const int e_old = min(max((int)old - 127, kScaleLow), kScaleHigh);
    if (!anew) e = max(e, e_old);
    const bool nan = none || (!anew && old == kScaleNan);
    if (lane == 0) *scale_at = (uint8_t)(nan ? kScaleNan : e + 127);

    // the group's other rows
    if (anew || e > e_old) {
        const float f = ldexpf(1.f, e_old - e);
#pragma unroll
        for (int i = 0; i < HD / 64; ++i) {
            const int o = i * 1024 + lane * 16;
            if ((stored >> (o / HD)) & 1) continue;
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
        if (i * ROWS >= n) break;
        const int r = i * ROWS + lane / LPH;
        const int s = __shfl(slot, min(r, n - 1));
        uint32_t w[2] = {0, 0};
#pragma unroll
        for (int e8 = 0; e8 < 8; ++e8) {
            const double z = rint(y[i][e8] * f);
            const int code = fabs(z) <= 127.0 ? (int)z : 0;  // (else the group is NaN)
            w[e8 / 4] |= ((uint32_t)code & 255u) << (8 * (e8 % 4));
        }
        if (r < n) {
            *reinterpret_cast<uint32_t*>(rows + s * HD + at.lo) = w[0];
            *reinterpret_cast<uint32_t*>(rows + s * HD + at.hi) = w[1];
        }
    }
}

template <int HD, typename X, typename Q>
__global__ void __launch_bounds__(64 * kWaves) qk_q8_kernel(PagedBatch b, PagedCache c, PagedCodes codes, QkNormRope p,
                                                            int q_groups) {
    constexpr int LPH = HD / 8, HPB = 64 * kWaves / LPH;  // lanes per head, heads per workgroup
    const int token = blockIdx.x;
    auto load8 = [&](int t, int head, HeadPlace at, float (&x)[8]) {
        const X* src = static_cast<const X*>(p.qkv) + (int64_t)t * p.ld + head * HD;
        load4<X>(src + at.lo, x);
        load4<X>(src + at.hi, x + 4);
    };
    if ((int)blockIdx.y >= q_groups) {
        const int item = (blockIdx.y - q_groups) * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        if (item < 2 * c.kv_heads) store_run<HD>(b, c, codes, p, token, item, load8);
        return;
    }
    const int head = blockIdx.y * HPB + threadIdx.x / LPH, u = threadIdx.x % LPH;
    if (head >= p.q_heads) return;  // (whole lane groups leave)
    const HeadPlace at = head_place<HD>(p, false, u);
    float x[8];
    load8(token, head, at, x);
    norm_and_turn<HD>(b, p, p.q_norm, at, token, u, x);
    Q* dst = static_cast<Q*>(p.q_out) + (int64_t)token * p.ldq + head * HD;
    store4(dst + at.lo, x);
    store4(dst + at.hi, x + 4);
}

template <int HD, typename X>
static void launch_x(const PagedBatch& b, const PagedCache& c, const PagedCodes& codes, const QkNormRope& p, bool q_f16,
                     hipStream_t stream) {
    constexpr int HPB = 64 * kWaves / (HD / 8);
    const int q_groups = (p.q_heads + HPB - 1) / HPB;
    const dim3 grid(b.tokens, q_groups + (2 * c.kv_heads + kWaves - 1) / kWaves), threads(64 * kWaves);
    if (q_f16) hipLaunchKernelGGL((qk_q8_kernel<HD, X, __half>), grid, threads, 0, stream, b, c, codes, p, q_groups);
    else hipLaunchKernelGGL((qk_q8_kernel<HD, X, float>), grid, threads, 0, stream, b, c, codes, p, q_groups);
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

// Sixteen codes a thread; keys and values by blockIdx.y. Bound: HBM.
__global__ void __launch_bounds__(256) values_q8_kernel(PagedCodes codes, __half* k, __half* v, int64_t pieces,
                                                        int row_shift) {
    const int8_t* from = blockIdx.y ? codes.v : codes.k;
    const uint8_t* scale = blockIdx.y ? codes.v_scale : codes.k_scale;
    __half* to = blockIdx.y ? v : k;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < pieces; i += (int64_t)gridDim.x * 256) {
        const uint4 x = reinterpret_cast<const uint4*>(from)[i];
        const uint32_t s = scale_pair(scale[i >> (row_shift + 4)]);
        uint4* out = reinterpret_cast<uint4*>(to) + 2 * i;
        out[0] = codes_to_h(make_uint2(x.x, x.y), s);
        out[1] = codes_to_h(make_uint2(x.z, x.w), s);
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
