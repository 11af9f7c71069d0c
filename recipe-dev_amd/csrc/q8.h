// The 8-bit pages' values: int8 codes, and per kv head one scale byte for each 16
// rows (a group): b stands for 2^(b - 127), with b in 103..136, and 255 for NaN. A
// code times its scale is an fp16 number, whatever they are (|code| <= 127: down to
// 2^-24, fp16's smallest, and up to 65,024), so kernels that multiply fp16
// operands take the values as they are, and a group whose largest value grows has
// its codes halved by whole powers of two instead of divided.
#pragma once

#include "halfcode.h"

namespace rq {

constexpr int kGroup = 16;                      // rows that share a scale
constexpr int kScaleLow = -24, kScaleHigh = 9;  // exponents of a scale
constexpr int kScaleNan = 255;

// A scale 2^e as a multiplier of codes in fp16 pairs. A code q comes as 1152 + q (q + 128 in the mantissa of 1024),
// so that q 2^e = fma(1152 + q, 2^e, -1152 * 2^e), exactly. Above 2^5 the last term leaves fp16's range: `more`
// is by how much (0 to 4), and the pair is (2^5, -1152 * 2^5) then.
struct Scale {
    uint32_t by, less;
    int more;
};
// Of a scale byte (those outside 103..136 as the nearest, 255 as NaN).
__device__ __forceinline__ Scale scale_of(unsigned byte) {
    const int e = min(max((int)byte, 127 + kScaleLow), 127 + kScaleHigh), low = min(e, 127 + 5);
    const float f = __builtin_bit_cast(float, low << 23);
    const _Float16 s = (_Float16)f, t = (_Float16)(-1152.f * f);
    const uint32_t hs = byte == kScaleNan ? 0x7E00u : (uint32_t)__builtin_bit_cast(uint16_t, s);
    const uint32_t ht = (uint32_t)__builtin_bit_cast(uint16_t, t);
    return Scale{hs << 16 | hs, ht << 16 | ht, e - low};
}

__device__ __forceinline__ uint32_t fma_h(uint32_t a, uint32_t b, uint32_t c) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(__builtin_bit_cast(hv2_t, a), __builtin_bit_cast(hv2_t, b),
                                                                  __builtin_bit_cast(hv2_t, c)));
}
__device__ __forceinline__ uint32_t mul_h(uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(hv2_t, a) * __builtin_bit_cast(hv2_t, b));
}

// Eight codes times their scale but for `more`, as fp16 pairs.
__device__ __forceinline__ uint4 codes_to_low(uint2 codes, const Scale& s) {
    uint32_t o[4];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const uint32_t u = (e ? codes.y : codes.x) ^ 0x80808080u;
        o[2 * e] = fma_h(__builtin_amdgcn_perm(0x64646464u, u, 0x04010400u), s.by, s.less);
        o[2 * e + 1] = fma_h(__builtin_amdgcn_perm(0x64646464u, u, 0x04030402u), s.by, s.less);
    }
    return make_uint4(o[0], o[1], o[2], o[3]);
}
// Eight codes times their scale.
__device__ __forceinline__ uint4 codes_to_h(uint2 codes, const Scale& s) {
    uint4 o = codes_to_low(codes, s);
    if (s.more) {
        const uint32_t by = (uint32_t)(15 + s.more) << 10, pair = by << 16 | by;
        o = make_uint4(mul_h(o.x, pair), mul_h(o.y, pair), mul_h(o.z, pair), mul_h(o.w, pair));
    }
    return o;
}

}  // namespace rq
