// The norms between two blocks (block_norm.hip).
#pragma once

#include <hip/hip_runtime.h>

namespace rq {

struct BlockNorm {
    const float* x;
    int64_t ldx;
    const float* delta;  // may be null, as what follows but scale and eps
    int64_t ldd;
    int rows, n;
    const float* post;
    const float* gate;
    int64_t ldg;
    float scale;
    const float* pre;
    float eps;
    float* x_out;
    int64_t ldxo;
    void* out;
    int64_t ldo;
};

constexpr int kBlockNormMaxN = 32768;

hipError_t launch_block_norm(const BlockNorm& p, bool out_f16, int cus, hipStream_t stream);

}  // namespace rq
