// Log probabilities, entropies and top alternatives of rows of logits (logprobs.hip).
#pragma once

#include <hip/hip_runtime.h>

namespace rq {

struct LogprobArgs {
    const float* logits;
    int64_t ld;
    int rows, n;
    const int* tokens;  // may be null, as each output
    int top;
    float* logprob;
    float* entropy;
    int* top_tokens;
    float* top_logprobs;
};

constexpr int kLogprobMaxN = 1 << 20;
constexpr int kLogprobMaxTop = 32;

size_t logprobs_workspace(int rows, int n, int top, int cus);
hipError_t launch_logprobs(const LogprobArgs& a, void* workspace, int cus, hipStream_t stream);

}  // namespace rq
