// Shared definitions of the int8 product kernels: launch arguments and the per-element finishing step (zero-point
// correction, int/float bias, scale, requantization) that every product variant applies as it stores a sum.
#pragma once

#include <cstdint>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "og_act.cuh"

namespace og {

// OUT_ACT_F32 / OUT_ACT_F16: the float form with a scale per row of A, an activation and a residual
// (og_int8_gemm_encode_activated), stored as float32 or float16.
enum OutKind : int { OUT_I32 = 0, OUT_F32 = 1, OUT_U8 = 2, OUT_S8 = 3, OUT_ACT_F32 = 4, OUT_ACT_F16 = 5 };

__host__ __device__ constexpr bool out_activated(int out) { return out == OUT_ACT_F32 || out == OUT_ACT_F16; }
__host__ __device__ constexpr int out_bytes(int out) {
    return out == OUT_U8 || out == OUT_S8 ? 1 : out == OUT_ACT_F16 ? 2 : 4;
}

// What a product kernel needs to finish and store C[b, m, n]. Zero points: mode 0 absent, 1 one value, 2 one per row
// (A) or per column (B). The correction uses the byte sums of the other operand:
//   C = dot - zb[n] * rowsumA[b, m] - za[m] * colsumB[b, n] + K * za[m] * zb[n]   (all modulo 2^32)
// which equals sum_k (a - za)(b - zb) exactly in the integers, so also modulo 2^32.
struct Epilogue {
    int out_kind;
    void* c;              // output buffer (int32, float or bytes), already advanced by OffsetC
    int64_t ldc;          // N
    int64_t batch_stride_c;  // M * N
    int m, n, k;
    const uint8_t* za;    // zero point of A (already offset), or null
    int za_vector, za_signed;
    const uint8_t* zb;
    int zb_vector, zb_signed;
    const int32_t* row_sum_a;     // [batchA][M] byte sums of A, or null when no zero point of B is present
    int64_t row_sum_a_stride;     // M, or 0 when every batch shares A
    const int32_t* col_sum_b;     // [batchB][N] byte sums of B, or null when no zero point of A is present
    int64_t col_sum_b_stride;     // N, or 0 when every batch shares B
    int sum_splits;               // the sums are this many partial sums over K ranges, to be added up
    int64_t row_sum_split_stride; // batchA * M
    int64_t col_sum_split_stride; // batchB * N
    const int32_t* int_bias;      // per column, or null
    const float* scale;           // float form: scale; requantized form: multiplier
    int scale_vector;
    const float* scale_a;         // dequantize form: one scale of A multiplied into every column's scale, or null
    const float* float_bias;      // per column, or null
    int zero_point_y;
    int vec_ok;                   // every output row starts on a 16-byte boundary
    // Activated form: the scale of A (one, or one per row), the activation, and the residual (laid out like the output
    // and of its type, possibly the output itself) or null.
    const float* row_scale;
    int row_scale_vector;
    int activation;
    const void* residual;
};

__device__ __forceinline__ int32_t zp_value(const uint8_t* z, int vector, int is_signed, int idx) {
    if (z == nullptr) return 0;
    const uint8_t v = __ldg(z + (vector ? idx : 0));
    return is_signed ? static_cast<int32_t>(static_cast<int8_t>(v)) : static_cast<int32_t>(v);
}

// The byte sum of row m of A (batch b) and of column n of B: the partial sums of the K splits added up (wrapping).
// Four at a time: their loads are in flight together.
__device__ __forceinline__ uint32_t split_sum(const int32_t* p, int splits, int64_t stride) {
    uint32_t s = 0;
    for (int i = 0; i < splits; i += 4) {
        int32_t v[4];
#pragma unroll
        for (int u = 0; u < 4; u++) v[u] = i + u < splits ? __ldg(p + (i + u) * stride) : 0;
        s += static_cast<uint32_t>(v[0]) + static_cast<uint32_t>(v[1]) + static_cast<uint32_t>(v[2]) + static_cast<uint32_t>(v[3]);
    }
    return s;
}

__device__ __forceinline__ uint32_t row_sum_of(const Epilogue& e, int b, int m) {
    return split_sum(e.row_sum_a + b * e.row_sum_a_stride + m, e.sum_splits, e.row_sum_split_stride);
}

__device__ __forceinline__ uint32_t col_sum_of(const Epilogue& e, int b, int n) {
    return split_sum(e.col_sum_b + b * e.col_sum_b_stride + n, e.sum_splits, e.col_sum_split_stride);
}

// The scale of column n: scale[n] (or the single scale), times the scale of A when one is given - one float32
// product, the same rounding as forming scaleA * scaleB[n] in a pass of its own.
__device__ __forceinline__ float col_scale(const Epilogue& e, int n) {
    const float s = __ldg(e.scale + (e.scale_vector ? n : 0));
    return e.scale_a != nullptr ? __fmul_rn(__ldg(e.scale_a), s) : s;
}

// float(sum) * scale, then + float bias: two separate roundings, never fused (Int8GemmEpilogue.hlsli semantics).
__device__ __forceinline__ float finish_float(const Epilogue& e, int n, uint32_t s) {
    const float sc = col_scale(e, n);
    float f = __fmul_rn(__int2float_rn(static_cast<int32_t>(s)), sc);
    if (e.float_bias != nullptr) f = __fadd_rn(f, __ldg(e.float_bias + n));
    return f;
}

// The scale of row m of A in the activated form.
__device__ __forceinline__ float row_scale_of(const Epilogue& e, int m) {
    return __ldg(e.row_scale + (e.row_scale_vector ? m : 0));
}

// The activated form before its activation: float(sum) * (aScale * bScale[n]), then + float bias, each step rounded
// on its own as in the dequantize form.
__device__ __forceinline__ float scaled_sum(uint32_t s, float row_scale, float scale, bool biased, float bias) {
    const float f = __fmul_rn(__int2float_rn(static_cast<int32_t>(s)), __fmul_rn(row_scale, scale));
    return biased ? __fadd_rn(f, bias) : f;
}

// Element idx of the residual, as float32, past L1: the residual may be the output itself, which the launch before may
// have written.
template <int OUT>
__device__ __forceinline__ float residual_at(const Epilogue& e, int64_t idx) {
    if constexpr (OUT == OUT_ACT_F16)
        return __half2float(__ldcg(static_cast<const __half*>(e.residual) + idx));
    else
        return __ldcg(static_cast<const float*>(e.residual) + idx);
}

// One result of the activated form at element idx of the output (row m, column n), stored.
template <int OUT>
__device__ __forceinline__ void store_activated(const Epilogue& e, int64_t idx, int m, int n, uint32_t s) {
    float f[1] = {scaled_sum(s, row_scale_of(e, m), __ldg(e.scale + (e.scale_vector ? n : 0)), e.float_bias != nullptr,
                             e.float_bias != nullptr ? __ldg(e.float_bias + n) : 0.0f)};
    activate_all(f, e.activation);
    if (e.residual != nullptr) f[0] = __fadd_rn(f[0], residual_at<OUT>(e, idx));
    if constexpr (OUT == OUT_ACT_F16)
        static_cast<__half*>(e.c)[idx] = __float2half_rn(f[0]);
    else
        static_cast<float*>(e.c)[idx] = f[0];
}

// clamp(round_half_even(float(sum) * multiplier) + zeroPointY) to the output type, NaN to the smallest value
// (Int8Epilogue.hlsl Quantized semantics).
__device__ __forceinline__ uint8_t finish_byte(const Epilogue& e, int n, uint32_t s, bool out_unsigned) {
    const int lo = out_unsigned ? 0 : -128;
    const int hi = out_unsigned ? 255 : 127;
    const float mult = col_scale(e, n);
    const float v = __fmul_rn(__int2float_rn(static_cast<int32_t>(s)), mult);
    if (isnan(v)) return static_cast<uint8_t>(lo & 0xFF);
    float r = rintf(v);
    const float flo = static_cast<float>(lo - e.zero_point_y);
    const float fhi = static_cast<float>(hi - e.zero_point_y);
    r = r < flo ? flo : (r > fhi ? fhi : r);
    return static_cast<uint8_t>((static_cast<int>(r) + e.zero_point_y) & 0xFF);
}

// Error word shared by the kernels of one device: a kernel whose bounded wait gave up sets it.
struct DeviceStatus {
    int error;
};

}  // namespace og
