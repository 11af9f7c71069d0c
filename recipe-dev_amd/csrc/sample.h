// The choice of the next tokens (sample.hip).
#pragma once

#include <hip/hip_runtime.h>

namespace rq {

struct SampleArgs {
    const float* logits;
    int64_t ld;
    int rows, n;
    const float* u;
    const float* temperature;  // each may be null: 1, off, off, off
    const int* top_k;
    const float* top_p;
    const float* min_p;
    int* tokens;
    float* probs;  // may be null
};

constexpr int kSampleMaxN = 1 << 20;

size_t sample_workspace(int rows, int n, int cus);
hipError_t launch_sample(const SampleArgs& a, void* workspace, int cus, hipStream_t stream);

}  // namespace rq
