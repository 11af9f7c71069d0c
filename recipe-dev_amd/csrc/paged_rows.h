// A projected head on its way to the queries or the cache, by HD / 8 lanes of
// eight values each: what rqmv_qk_norm_rope (paged.hip) and its form for 8-bit
// pages (paged_q8.hip) share.
#pragma once

#include "paged.h"

namespace rq {

// y = x / sqrt(mean(x^2) + eps) * w per q and k head, then pair (i, i + rot / 2)
// turns by its position's (cos, sin). A head is taken by HD / 8 lanes of eight
// values: lane u < rot / 8 holds the pairs 4u..4u+3 (four values of each half, so
// both partners are at hand), a lane past them eight values that do not
// turn; a value head's lanes hold eight values in a row.
template <typename T>
__device__ __forceinline__ void load4(const T* p, float* v);
template <>
__device__ __forceinline__ void load4<float>(const float* p, float* v) {
    const float4 a = *reinterpret_cast<const float4*>(p);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
}
template <>
__device__ __forceinline__ void load4<__half>(const __half* p, float* v) {
    const uint2 a = *reinterpret_cast<const uint2*>(p);
    const __half2 lo = __builtin_bit_cast(__half2, a.x), hi = __builtin_bit_cast(__half2, a.y);
    v[0] = __low2float(lo), v[1] = __high2float(lo), v[2] = __low2float(hi), v[3] = __high2float(hi);
}

__device__ __forceinline__ void store4(float* p, const float* v) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void store4(__half* p, const float* v) {
    uint2 a;
    a.x = __builtin_bit_cast(uint32_t, __floats2half2_rn(v[0], v[1]));
    a.y = __builtin_bit_cast(uint32_t, __floats2half2_rn(v[2], v[3]));
    *reinterpret_cast<uint2*>(p) = a;
}

// Where lane u of a head has its values: lo..lo+3 and hi..hi+3.
struct HeadPlace {
    bool turns;
    int lo, hi;
};
template <int HD>
__device__ __forceinline__ HeadPlace head_place(const QkNormRope& p, bool value, int u) {
    const bool turns = !value && u < p.rot_dim / 8;
    const int lo = turns ? 4 * u : 8 * u;
    return HeadPlace{turns, lo, lo + (turns ? p.rot_dim / 2 : 4)};
}
// A q or k head's values through its norm (null: none) and the rotation, in T's arithmetic.
template <int HD, typename T>
__device__ __forceinline__ void norm_and_turn(const PagedBatch& b, const QkNormRope& p, const float* norm, HeadPlace at,
                                              int token, int u, T (&x)[8]) {
    constexpr int LPH = HD / 8;
    if (norm) {
        float w[8];
        T ss = 0;
        load4<float>(norm + at.lo, w);
        load4<float>(norm + at.hi, w + 4);
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fma(x[e], x[e], ss);
#pragma unroll
        for (int d = 1; d < LPH; d <<= 1) ss += __shfl_xor(ss, d);
        const T scale = T(1) / sqrt(ss / (T)HD + (T)p.eps);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = x[e] * scale * (T)w[e];
    }
    if (at.turns) {
        const int pos = min(max(b.positions[token], 0), p.rope_rows - 1);
        const float* cs = reinterpret_cast<const float*>(p.rope + (int64_t)pos * (p.rot_dim / 2) + 4 * u);
        float t[8];
        load4<float>(cs, t);
        load4<float>(cs + 4, t + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const T a = x[e], d = x[e + 4];
            x[e] = a * (T)t[2 * e] - d * (T)t[2 * e + 1];
            x[e + 4] = d * (T)t[2 * e] + a * (T)t[2 * e + 1];
        }
    }
}

}  // namespace rq
