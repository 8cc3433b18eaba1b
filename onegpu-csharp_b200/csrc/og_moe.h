// Internal launch description of the mixture-of-experts layer (og_moe.cu).
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace og {

constexpr int MOE_MAX_TOKENS = 128;
constexpr int MOE_MAX_EXPERTS = 512;
constexpr int MOE_MAX_TOP_K = 16;
constexpr int MOE_MAX_SIZE = 65536;

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
    int32_t* ids;    // [tokens][top_k]
    float* weights;  // [tokens][top_k]
    float* hidden;   // [tokens * top_k][expert]
};

}  // namespace og
