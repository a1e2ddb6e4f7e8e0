// Products of a matrix of E2M1 nibbles with group scales (MXFP4: E8M0 per 32, NVFP4: E4M3 per 16 and one fp32) with tokens.
//
//   W[n][k] = e2m1(values[n][k]) * scale[n][k / group] (* global)
//   y[m][n] = sum_k x[m][k] W[n][k]          dx[m][k] = sum_n dy[m][n] W[n][k]
// Sums are fp32, with one rounding at the end.
#pragma once
#include "number_types.cuh"

namespace ptwm {

struct ScaledMatrix {
    const uint8_t* values;       // [rows][value_pitch], two to a byte, the even one in the low nibble
    const uint8_t* scales;       // [rows][scale_pitch]
    const float* global_scale;   // or null
    uint64_t rows, cols;
    uint32_t value_pitch, scale_pitch;
    uint32_t group;              // 32: E8M0; 16: E4M3
};
struct TokenArgs {
    const void* x;
    const void* scales;
    uint64_t tokens;
    uint32_t scaled;
    void* y;
};

template <class T> __device__ __forceinline__ float token_value(const TokenArgs& t, uint64_t m, uint64_t k, uint64_t cols) {
    return to_f32(static_cast<const T*>(t.x)[m * cols + k]);
}
template <> __device__ __forceinline__ float token_value<uint8_t>(const TokenArgs& t, uint64_t m, uint64_t k, uint64_t cols) {
    const float v = e4m3_f32(static_cast<const uint8_t*>(t.x)[m * cols + k]);
    return t.scaled == SCALE_ROW ? v : v * e8m0_f32(static_cast<const uint8_t*>(t.scales)[m * (cols / 32) + k / 32]);
}

__device__ __forceinline__ void store_as(void* y, uint32_t dtype, uint64_t i, float v) {
    if (dtype == DT_BF16) static_cast<__nv_bfloat16*>(y)[i] = __float2bfloat16_rn(v);
    else if (dtype == DT_FP16) static_cast<__half*>(y)[i] = __float2half_rn(v);
    else static_cast<float*>(y)[i] = v;
}

}  // namespace ptwm
