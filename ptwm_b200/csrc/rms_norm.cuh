// Root-mean-square norm with the residual's addition, into the input's type or into E4M3 with scales, and its gradient.
//
//   h = rn(x + residual)             the residual stream the next layer adds to, in x's type
//   r = (sum h^2 / K + eps)^(-1/2)
//   y = h r weight                   one rounding, from fp32
//   "row":   s = max|y| / 448, q = e4m3(y / s)
//   "block": e = ceil(log2(max|y| / 448)) over 32 values, q = e4m3(y 2^-e).  With max|y| = m 2^p, 1 <= m < 2, e is
//            p - 8 + (m > 1.75): the bits say it, no logarithm is taken.
// Sums are fp32; where a maximum is not finite its scale is NaN and so are its values.
#pragma once
#include "number_types.cuh"

namespace ptwm {

struct NormArgs {
    const void *x, *residual, *weight;
    void *h, *y, *scales;
    uint64_t rows, cols;
    float eps;
};

template <class Op> __device__ __forceinline__ float block_reduce(float v, float* shared, Op op, float none) {
    for (int o = 16; o; o >>= 1) v = op(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
    __syncthreads();
    v = threadIdx.x % 32 < (blockDim.x + 31) / 32 ? shared[threadIdx.x % 32] : none;
    for (int o = 16; o; o >>= 1) v = op(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
    return v;
}
struct Add { __device__ float operator()(float a, float b) const { return a + b; } };
// Of two magnitudes: NaN, whose bits are above infinity's, wins.
struct MaxMagnitude { __device__ float operator()(float a, float b) const { return __uint_as_float(max(__float_as_uint(a), __float_as_uint(b))); } };

__device__ __forceinline__ bool is_finite(float v) { return (__float_as_uint(v) & 0x7F800000u) != 0x7F800000u; }

// E8M0 code of a block whose largest magnitude is `most`; 255 where that is not finite.
__device__ __forceinline__ uint32_t block_scale(float most) {
    if (!is_finite(most)) return 255;
    uint32_t b = __float_as_uint(most);
    int p = int(b >> 23);          // biased exponent
    if (!p) {                       // subnormal or zero: the smallest scale
        return 0;
    }
    const int e = p - 8 + ((b & 0x7FFFFFu) > 0x600000u);
    return uint32_t(e < 0 ? 0 : e);  // at most 254 - 7: never 255
}
__device__ __forceinline__ float block_inverse(uint32_t e) {  // 2^(127 - e), exact; NaN for 255
    return e == 255 ? __uint_as_float(0x7FC00000u) : e == 254 ? __uint_as_float(0x00400000u) : __uint_as_float((254 - e) << 23);
}

// One block per row, three passes over it.
template <class T, class W>
__global__ void __launch_bounds__(256) rms_norm_kernel(NormArgs a, uint32_t quant) {
    __shared__ float shared[32];
    const uint64_t row = blockIdx.x, cols = a.cols;
    const T* x = static_cast<const T*>(a.x) + row * cols;
    const T* res = a.residual ? static_cast<const T*>(a.residual) + row * cols : nullptr;
    T* h = a.residual ? static_cast<T*>(a.h) + row * cols : nullptr;
    const W* w = static_cast<const W*>(a.weight);
    float sum = 0;
    for (uint64_t k = threadIdx.x; k < cols; k += blockDim.x) {
        float v = to_f32(x[k]);
        if (res) { const T s = from_f32<T>(v + to_f32(res[k])); h[k] = s; v = to_f32(s); }
        sum += v * v;
    }
    sum = block_reduce(sum, shared, Add(), 0.0f);
    const float r = rsqrtf(sum / float(cols) + a.eps);
    const T* in = res ? h : x;
    auto normed = [&](uint64_t k) { return to_f32(in[k]) * r * to_f32(w[k]); };
    if (quant == SCALE_NONE) {
        for (uint64_t k = threadIdx.x; k < cols; k += blockDim.x) static_cast<T*>(a.y)[row * cols + k] = from_f32<T>(normed(k));
        return;
    }
    uint8_t* q = static_cast<uint8_t*>(a.y) + row * cols;
    if (quant == SCALE_ROW) {
        float most = 0;
        for (uint64_t k = threadIdx.x; k < cols; k += blockDim.x) most = MaxMagnitude()(most, fabsf(normed(k)));
        most = block_reduce(most, shared, MaxMagnitude(), 0.0f);
        const float s = is_finite(most) ? most / 448.0f : __uint_as_float(0x7FC00000u);
        for (uint64_t k = threadIdx.x; k < cols; k += blockDim.x) q[k] = s == 0.0f ? 0 : f32_e4m3(normed(k) / s);
        if (threadIdx.x == 0) static_cast<float*>(a.scales)[row] = s;
        return;
    }
    for (uint64_t k = threadIdx.x; k < cols; k += blockDim.x) {  // cols is a multiple of 32: a warp has a block of values
        const float v = normed(k);
        float most = fabsf(v);
        for (int o = 16; o; o >>= 1) most = MaxMagnitude()(most, __shfl_xor_sync(0xFFFFFFFFu, most, o));
        const uint32_t e = block_scale(most);
        q[k] = f32_e4m3(v * block_inverse(e));
        if ((threadIdx.x & 31) == 0) static_cast<uint8_t*>(a.scales)[row * (cols / 32) + k / 32] = uint8_t(e);
    }
}

// Gradient.  With g = dy weight:  dx = dh + r g - h r^3 / K sum(g h)  (the residual's is the same),  dweight = sum over rows of dy h r.
struct NormGradArgs {
    const void *h, *weight, *dy, *dh;
    void* dx;
    float* partial;   // [blocks, cols]: each block's share of dweight
    void* dweight;
    uint64_t rows, cols;
    float eps;
    uint32_t blocks;
};

// A block takes rows blockIdx.x, + blocks, ...; its sums for dweight live in `partial`, where each column belongs to one thread.
template <class T, class W>
__global__ void __launch_bounds__(256) rms_norm_grad_kernel(NormGradArgs a) {
    __shared__ float shared[32];
    const uint64_t cols = a.cols;
    const W* w = static_cast<const W*>(a.weight);
    float* part = a.partial ? a.partial + blockIdx.x * cols : nullptr;
    if (part) for (uint64_t k = threadIdx.x; k < cols; k += blockDim.x) part[k] = 0;
    for (uint64_t row = blockIdx.x; row < a.rows; row += a.blocks) {
        const T* h = static_cast<const T*>(a.h) + row * cols;
        const T* dy = a.dy ? static_cast<const T*>(a.dy) + row * cols : nullptr;
        const T* dh = a.dh ? static_cast<const T*>(a.dh) + row * cols : nullptr;
        float sq = 0, dot = 0;
        for (uint64_t k = threadIdx.x; k < cols; k += blockDim.x) {
            const float v = to_f32(h[k]);
            sq += v * v;
            dot += to_f32(dy[k]) * to_f32(w[k]) * v;
        }
        sq = block_reduce(sq, shared, Add(), 0.0f);
        dot = block_reduce(dot, shared, Add(), 0.0f);
        const float r = rsqrtf(sq / float(cols) + a.eps);
        const float c = r * r * r * dot / float(cols);
        for (uint64_t k = threadIdx.x; k < cols; k += blockDim.x) {
            const float v = to_f32(h[k]), d = to_f32(dy[k]);
            float g = r * d * to_f32(w[k]) - v * c;
            if (dh) g += to_f32(dh[k]);
            if (a.dx) static_cast<T*>(a.dx)[row * cols + k] = from_f32<T>(g);
            if (part) part[k] += d * v * r;
        }
    }
}

// dweight from the blocks' shares, added in their order.
template <class W> __global__ void __launch_bounds__(256) rms_norm_grad_weight_kernel(NormGradArgs a) {
    const uint64_t k = uint64_t(blockIdx.x) * blockDim.x + threadIdx.x;
    if (k >= a.cols) return;
    float sum = 0;
    for (uint32_t b = 0; b < a.blocks; ++b) sum += a.partial[b * a.cols + k];
    static_cast<W*>(a.dweight)[k] = from_f32<W>(sum);
}

}  // namespace ptwm
