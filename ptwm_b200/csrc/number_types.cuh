// The number types of the operators: fp32, fp16 and bf16 (public dtype codes 1, 4, 6), and E4M3 with scales.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace ptwm {

enum : uint32_t { DT_FP32 = 1, DT_FP16 = 4, DT_BF16 = 6, DT_E4M3 = 29 };
enum : uint32_t { SCALE_NONE = 0, SCALE_ROW = 1, SCALE_BLOCK = 2 };  // how 8-bit values are scaled: not, fp32 per row, E8M0 per 32

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return uint32_t(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Two 16-bit values of a word, the first in its lower half.
template <class T> __device__ __forceinline__ float2 two_f32(uint32_t w);
template <> __device__ __forceinline__ float2 two_f32<__half>(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
template <> __device__ __forceinline__ float2 two_f32<__nv_bfloat16>(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u)); }
template <class T> __device__ __forceinline__ uint32_t two_rounded(float2 v);
template <> __device__ __forceinline__ uint32_t two_rounded<__half>(float2 v) { const __half2 h = __float22half2_rn(v); return *reinterpret_cast<const uint32_t*>(&h); }
template <> __device__ __forceinline__ uint32_t two_rounded<__nv_bfloat16>(float2 v) { const __nv_bfloat162 h = __float22bfloat162_rn(v); return *reinterpret_cast<const uint32_t*>(&h); }

// Programmatic dependent launch.  A kernel of these operators may start while the one before it in the stream ends: it does nothing but
// find its place and make its barriers until after_those_before(), where all that was enqueued before it is done and can be seen.
// The one behind it may start from others_may_start() on.
__device__ __forceinline__ void others_may_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void after_those_before() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// 2^(e - 127) of an E8M0 code; 255 is NaN.  Code 0 is the subnormal 2^-127.
__device__ __forceinline__ float e8m0_f32(uint32_t e) { return e == 255 ? __uint_as_float(0x7FC00000u) : __uint_as_float(e ? e << 23 : 0x00400000u); }

__device__ __forceinline__ float e4m3_f32(uint8_t v) { return __half2float(__half(__nv_cvt_fp8_to_halfraw(v, __NV_E4M3))); }
// Nearest E4M3 value, ties to even; beyond 448 it is 448, NaN stays NaN.
__device__ __forceinline__ uint8_t f32_e4m3(float v) { return uint8_t(__nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3)); }

}  // namespace ptwm
