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
// What a q or k head's lane needs besides its values: the norm's weights, and (cos, sin) of its pairs at a position.
struct HeadLane {
    float w[8], t[8];
};
__device__ __forceinline__ void load_norm(const float* norm, HeadPlace at, HeadLane& h) {
    load4<float>(norm + at.lo, h.w);
    load4<float>(norm + at.hi, h.w + 4);
}
__device__ __forceinline__ void load_turn(const QkNormRope& p, int position, int u, HeadLane& h) {
    const int pos = min(max(position, 0), p.rope_rows - 1);
    const float* cs = reinterpret_cast<const float*>(p.rope + (int64_t)pos * (p.rot_dim / 2) + 4 * u);
    load4<float>(cs, h.t);
    load4<float>(cs + 4, h.t + 4);
}
// The sum over a head's LPH lanes, the same in each. Partners by DPP up to 16 lanes: of quads by their lanes, of
// halves and rows mirrored (their lanes agree by then).
template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
    return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, false));
}
template <int CTRL>
__device__ __forceinline__ double dpp_add(double v) {
    const int2 w = __builtin_bit_cast(int2, v);
    return v + __builtin_bit_cast(double, make_int2(__builtin_amdgcn_update_dpp(0, w.x, CTRL, 0xf, 0xf, false),
                                                    __builtin_amdgcn_update_dpp(0, w.y, CTRL, 0xf, 0xf, false)));
}
template <int LPH, typename T>
__device__ __forceinline__ T head_sum(T v) {
    v = dpp_add<0xB1>(v);   // quad_perm 1, 0, 3, 2
    v = dpp_add<0x4E>(v);   // quad_perm 2, 3, 0, 1
    v = dpp_add<0x141>(v);  // row_half_mirror
    if constexpr (LPH > 8) v = dpp_add<0x140>(v);  // row_mirror
    if constexpr (LPH > 16) v += __shfl_xor(v, 16);
    return v;
}
// A head's values through its norm (if it has one) and the rotation (of lanes that turn), in T's arithmetic.
template <int HD, typename T>
__device__ __forceinline__ void norm_and_turn(bool norm, bool turns, float eps, const HeadLane& h, T (&x)[8]) {
    constexpr int LPH = HD / 8;
    if (norm) {
        T ss = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fma(x[e], x[e], ss);
        ss = head_sum<LPH>(ss);
        const T scale = T(1) / sqrt(ss / (T)HD + (T)eps);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = x[e] * scale * (T)h.w[e];
    }
    if (turns) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const T a = x[e], d = x[e + 4];
            x[e] = a * (T)h.t[2 * e] - d * (T)h.t[2 * e + 1];
            x[e + 4] = d * (T)h.t[2 * e] + a * (T)h.t[2 * e + 1];
        }
    }
}

}  // namespace rq
