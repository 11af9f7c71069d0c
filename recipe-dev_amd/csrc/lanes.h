// Exchanges between the lanes of a wave that need no LDS.
#pragma once

#include <hip/hip_runtime.h>

namespace rq {

// v combined with the value of lane ^ 16 and of lane ^ 32 through gfx950's
// VALU lane swaps (no LDS crossbar): v_permlane16_swap_b32 / 32 exchange odd
// 16-lane rows (upper 32 lanes) of the first register with even rows (lower
// 32 lanes) of the second; applied to two copies of v they leave, in every
// lane, the lower lane's value in the first and the upper lane's in the
// second. Written as inline assembly: this compiler's builtin loses the second
// result. The s_nop gives the wait states a VALU write needs before the swap
// reads it.
struct LanePair {
    float lo, hi;
};
__device__ __forceinline__ LanePair swap16(float v) {
    float a = v, b = v;
    asm volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(a), "+v"(b));
    return LanePair{a, b};
}
__device__ __forceinline__ LanePair swap32(float v) {
    float a = v, b = v;
    asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(a), "+v"(b));
    return LanePair{a, b};
}
__device__ __forceinline__ float swap16_sum(float v) {
    const LanePair p = swap16(v);
    return p.lo + p.hi;
}
__device__ __forceinline__ float swap32_sum(float v) {
    const LanePair p = swap32(v);
    return p.lo + p.hi;
}
__device__ __forceinline__ float swap16_max(float v) {
    const LanePair p = swap16(v);
    return fmaxf(p.lo, p.hi);
}
__device__ __forceinline__ float swap32_max(float v) {
    const LanePair p = swap32(v);
    return fmaxf(p.lo, p.hi);
}

// v of the lane that a DPP control selects, 0 where it selects none (rows outside `ROWS` too).
template <int CTRL, int ROWS>
__device__ __forceinline__ unsigned dpp(unsigned v) {
    return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ unsigned long long dpp(unsigned long long v) {
    return (unsigned long long)dpp<CTRL, ROWS>((unsigned)(v >> 32)) << 32 | dpp<CTRL, ROWS>((unsigned)v);
}
// Inclusive prefix sums over the wave: within rows of 16 by shifts, then each row's last
// sum to the row behind it and the lower half's to the upper (no LDS crossbar).
template <typename T>
__device__ __forceinline__ T wave_scan(T v) {
    v += dpp<0x111, 0xf>(v);  // row_shr:1, 2, 4, 8
    v += dpp<0x112, 0xf>(v);
    v += dpp<0x114, 0xf>(v);
    v += dpp<0x118, 0xf>(v);
    v += dpp<0x142, 0xa>(v);  // row_bcast:15 into rows 1 and 3
    v += dpp<0x143, 0xc>(v);  // row_bcast:31 into rows 2 and 3
    return v;
}

}  // namespace rq
