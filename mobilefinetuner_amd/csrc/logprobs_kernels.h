// Launchers of the token log probability kernels (logprobs.hip; called by
// logprobs_capi.cpp).
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace mft {

constexpr int kLogprobsMaxTop = 64;

struct LogprobsArgs {
    int64_t N, V, ld, ldg;
    int ignore, top;
    const void* z;
    const int32_t* tokens;
    float* logprob;
    float* entropy;      // may be null
    float2* stats;       // (max, log of the sum); may be null
    float* top_logprobs;
    int32_t* top_ids;
    int32_t* status;     // may be null
    // rows cut into parts: each part's (max, sum, sum of e d), then its alternatives' keys
    int parts;
    int64_t per_part;    // elements of a part
    float4* part;        // [N * parts]
    uint64_t* part_keys; // [N * parts][top]
    // backward
    const float2* stats_in;
    const float* entropy_in;
    const float* grad_logprob;
    const float* grad_entropy;
    void* grad;
};

size_t logprobs_workspace(int64_t N, int64_t V, int top);
hipError_t launch_logprobs_fwd(LogprobsArgs a, bool bf16, void* workspace, hipStream_t st);
hipError_t launch_logprobs_bwd(const LogprobsArgs& a, bool bf16, hipStream_t st);

}  // namespace mft
