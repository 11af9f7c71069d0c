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

// A scale byte as a pair of fp16 (bytes outside 103..136 as the nearest).
__device__ __forceinline__ uint32_t scale_pair(unsigned byte) {
    const unsigned b = min(max(byte, 127u + kScaleLow), 127u + kScaleHigh);
    const _Float16 s = (_Float16)__builtin_bit_cast(float, b << 23);
    const uint32_t h = byte == kScaleNan ? 0x7E00u : (uint32_t)__builtin_bit_cast(uint16_t, s);
    return h << 16 | h;
}

// Eight codes times their scale, as fp16 pairs.
__device__ __forceinline__ uint4 codes_to_h(uint2 codes, uint32_t scale) {
    uint32_t o[4];
    bytes_to_h(codes.x, o[0], o[1]);
    bytes_to_h(codes.y, o[2], o[3]);
#pragma unroll
    for (int e = 0; e < 4; ++e)
        o[e] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(hv2_t, o[e]) * __builtin_bit_cast(hv2_t, scale));
    return make_uint4(o[0], o[1], o[2], o[3]);
}

}  // namespace rq
