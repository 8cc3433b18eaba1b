// Internal launch description of the mixture-of-experts layer (og_moe.cu).
#pragma once

#include <cuda_runtime.h>

#include <cstdint>
#include <functional>

namespace og {

constexpr int MOE_MAX_TOKENS = 128;
constexpr int MOE_MAX_EXPERTS = 512;
constexpr int MOE_MAX_TOP_K = 16;
constexpr int MOE_MAX_SIZE = 65536;

// What the CTAs of a launch count; all zero between launches.
struct MoeCounts {
    unsigned int arrivals;  // at the grid barriers
    unsigned int exits;     // CTAs that are through with the counts
    unsigned int tickets[MOE_MAX_TOKENS / 8];  // logits finished of each block of 8 tokens
};

// One validated layer, pointers resolved (offsets applied). Rows of the weights are contiguous over the summed axis:
// w_in [experts][up * expert_size][model_size] (up = 2 when gated: the gate's rows, then the other half's; else 1),
// w_out [experts][model_size][expert_size], each row with its scale.
struct MoeLaunch {
    int tokens, model, expert, experts, top_k;
    int activation, gated, normalize;
    int x_half, router_half;
    const void* x;
    const void* router;
    const int8_t* w_in;
    const float* in_scale;
    const int8_t* w_out;
    const float* out_scale;
    void* y;
    const void* residual;  // of y's type, possibly y itself, or null
    int32_t* ids_out;      // [tokens][top_k], or null
    float* weights_out;    // [tokens][top_k], or null
    // Workspace of the instance.
    int32_t* ids;                  // [tokens][top_k]
    float* weights;                // [tokens][top_k]
    float* hidden;                 // [tokens * top_k][expert], rows padded to 4
    double* logits;                // [tokens][experts]
    uint8_t* x_digits;             // [tokens][chunks of model][digits][128] of x
    uint8_t* h_digits;             // [tokens * top_k][chunks of expert][digits][128] of the hidden values
    uint32_t* x_most;              // [tokens] the bits of a token's largest magnitude
    uint32_t* h_most;              // [tokens * top_k] and of a pair's hidden values
    float* outputs;                // [tokens * top_k][model], rows padded to 4: weighted outputs of the chosen experts
    long long* segments;           // partial sums of units cut between warps
    MoeCounts* counts;
    int* error_flag;
    int num_sms;
    uint64_t wait_limit_ns;  // of the waits at the grid barriers
    int late_barrier;        // watchdog self-test: the barrier (1 .. 4) that one CTA comes late_ns late to, 0 for none
    uint64_t late_ns;
};

// The workspace sizes of the fused kernel, in bytes.
struct MoeFusedSizes {
    int64_t logits, hidden, x_digits, h_digits, x_most, h_most, outputs, segments;
};
MoeFusedSizes moe_fused_sizes(const MoeLaunch& L);
// Whether weight rows start on 16-byte boundaries, as TMA loads them.
bool moe_aligned(const MoeLaunch& L);
// Builds the tensor maps.
std::function<cudaError_t(cudaStream_t)> prepare_moe_fused(const MoeLaunch& L, cudaError_t* err);

}  // namespace og
