// Host side of the operators that apply decoded weights: rms_norm and matvec with 4-bit weights.  A translation unit of its
// own; every call enqueues its kernels on the caller's stream and returns.
#include <algorithm>

#include "errors.hpp"
#include "matvec.cuh"
#include "rms_norm.cuh"

using namespace ptwm;

namespace {

template <class T> T* at(uint64_t p) { return reinterpret_cast<T*>(uintptr_t(p)); }
cudaStream_t stream_of(uint64_t s) { return reinterpret_cast<cudaStream_t>(uintptr_t(s)); }
bool plain_type(uint32_t t) { return t == DT_FP32 || t == DT_FP16 || t == DT_BF16; }

// f(T()) with the C++ type of a plain dtype code.
template <class F> void with_type(uint32_t t, F f) {
    if (t == DT_FP32) f(float());
    else if (t == DT_FP16) f(__half());
    else f(__nv_bfloat16());
}

int64_t matrix_of(const ptwm_b200_scaled_weight* w, ScaledMatrix* out) {
    if (!w || !w->values || !w->scales) return fail(PTWM_RC_INVALID_INPUT, "scaled weight: null pointer");
    if (w->group != 16 && w->group != 32) return fail(PTWM_RC_INVALID_INPUT, "scaled weight: groups are 16 (E4M3 scales) or 32 (E8M0 scales) values");
    if (!w->rows || !w->cols || w->cols % w->group) return fail(PTWM_RC_INVALID_INPUT, "scaled weight: cols must be a positive multiple of the group");
    if (w->rows > (1u << 30) || w->cols > (1u << 30)) return fail(PTWM_RC_UNSUPPORTED, "scaled weight: more than 2^30 rows or columns");
    if (w->value_pitch % 16 || w->scale_pitch % 16 || w->values % 16 || w->scales % 16)
        return fail(PTWM_RC_INVALID_INPUT, "scaled weight: rows of values and scales start at multiples of 16 bytes");
    if (w->value_pitch < w->cols / 2 || w->scale_pitch < w->cols / w->group) return fail(PTWM_RC_INVALID_INPUT, "scaled weight: pitch shorter than a row");
    *out = ScaledMatrix{at<const uint8_t>(w->values), at<const uint8_t>(w->scales), at<const float>(w->global_scale), w->rows, w->cols, w->value_pitch, w->scale_pitch, w->group};
    return 0;
}

}  // namespace

extern "C" int64_t ptwm_b200_rms_norm(uint64_t x, uint64_t residual, uint64_t weight, uint64_t h, uint64_t y, uint64_t scales, uint64_t rows, uint64_t cols,
                                      uint32_t dtype, uint32_t weight_dtype, uint32_t scaled, float eps, uint32_t device, uint64_t stream) {
    if (!plain_type(dtype) || !plain_type(weight_dtype)) return fail(PTWM_RC_UNSUPPORTED, "rms_norm: x and weight are fp32, fp16 or bf16");
    if (scaled > SCALE_BLOCK) return fail(PTWM_RC_INVALID_INPUT, "rms_norm: unknown output scaling");
    if (!cols || (scaled == SCALE_BLOCK && cols % 32)) return fail(PTWM_RC_INVALID_INPUT, "rms_norm: rows must not be empty, and hold whole blocks of 32 for block scales");
    if (rows > 0x7FFFFFFFull || cols > 0x7FFFFFFFull) return fail(PTWM_RC_UNSUPPORTED, "rms_norm: more than 2^31 - 1 rows or columns");
    if (!rows) return 0;
    if (!x || !weight || !y || (residual && !h) || (scaled && !scales)) return fail(PTWM_RC_INVALID_INPUT, "rms_norm: null device pointer");
    DeviceGuard guard{int(device)};
    if (guard.err != cudaSuccess) return fail(PTWM_RC_CUDA, std::string("cudaSetDevice: ") + cudaGetErrorString(guard.err));
    const NormArgs a{at<void>(x), at<void>(residual), at<void>(weight), at<void>(h), at<void>(y), at<void>(scales), rows, cols, eps};
    with_type(dtype, [&](auto t) {
        with_type(weight_dtype, [&](auto w) { rms_norm_kernel<decltype(t), decltype(w)><<<uint32_t(rows), 256, 0, stream_of(stream)>>>(a, scaled); });
    });
    CUDA_TRY(cudaGetLastError());
    return 0;
}

extern "C" uint64_t ptwm_b200_rms_norm_grad_scratch_bytes(uint64_t rows, uint64_t cols) { return std::min<uint64_t>(rows, 296) * cols * 4; }

extern "C" int64_t ptwm_b200_rms_norm_grad(uint64_t h, uint64_t weight, uint64_t dy, uint64_t dh, uint64_t dx, uint64_t dweight, uint64_t scratch, uint64_t scratch_bytes,
                                           uint64_t rows, uint64_t cols, uint32_t dtype, uint32_t weight_dtype, float eps, uint32_t device, uint64_t stream) {
    if (!plain_type(dtype) || !plain_type(weight_dtype)) return fail(PTWM_RC_UNSUPPORTED, "rms_norm_grad: tensors are fp32, fp16 or bf16");
    if (!cols || rows > 0x7FFFFFFFull || cols > 0x7FFFFFFFull) return fail(PTWM_RC_UNSUPPORTED, "rms_norm_grad: rows of 1 to 2^31 - 1 values, at most as many of them");
    if (rows && (!h || !weight || !dy || (!dx && !dweight))) return fail(PTWM_RC_INVALID_INPUT, "rms_norm_grad: null device pointer");
    if (rows && dweight && (!scratch || scratch_bytes < ptwm_b200_rms_norm_grad_scratch_bytes(rows, cols))) return fail(PTWM_RC_BUFFER_TOO_SMALL, "rms_norm_grad: scratch too small");
    DeviceGuard guard{int(device)};
    if (guard.err != cudaSuccess) return fail(PTWM_RC_CUDA, std::string("cudaSetDevice: ") + cudaGetErrorString(guard.err));
    if (!rows) {
        if (dweight) CUDA_TRY(cudaMemsetAsync(at<void>(dweight), 0, cols * (weight_dtype == DT_FP32 ? 4 : 2), stream_of(stream)));
        return 0;
    }
    const uint32_t blocks = uint32_t(std::min<uint64_t>(rows, 296));
    const NormGradArgs a{at<void>(h), at<void>(weight), at<void>(dy), at<void>(dh), at<void>(dx), dweight ? at<float>(scratch) : nullptr, at<void>(dweight), rows, cols, eps, blocks};
    with_type(dtype, [&](auto t) {
        with_type(weight_dtype, [&](auto w) {
            rms_norm_grad_kernel<decltype(t), decltype(w)><<<blocks, 256, 0, stream_of(stream)>>>(a);
            if (dweight) rms_norm_grad_weight_kernel<decltype(w)><<<uint32_t((cols + 255) / 256), 256, 0, stream_of(stream)>>>(a);
        });
    });
    CUDA_TRY(cudaGetLastError());
    return 0;
}

extern "C" int64_t ptwm_b200_matvec(const ptwm_b200_scaled_weight* weight, uint64_t x, uint64_t x_scales, uint64_t y, uint64_t tokens, uint32_t x_dtype, uint32_t x_scaled,
                                    uint32_t y_dtype, uint32_t device, uint64_t stream) {
    ScaledMatrix w;
    if (const int64_t rc = matrix_of(weight, &w); rc < 0) return rc;
    if (!plain_type(y_dtype)) return fail(PTWM_RC_UNSUPPORTED, "matvec: the output is fp32, fp16 or bf16");
    if (x_dtype == DT_E4M3 ? (x_scaled != SCALE_ROW && x_scaled != SCALE_BLOCK) || !x_scales : !plain_type(x_dtype) || x_scaled)
        return fail(PTWM_RC_UNSUPPORTED, "matvec: tokens are fp32, fp16, bf16, or E4M3 with scales per row or block");
    if (x_scaled == SCALE_BLOCK && w.cols % 32) return fail(PTWM_RC_INVALID_INPUT, "matvec: block scales need whole blocks of 32 columns");
    if (tokens > (1u << 19)) return fail(PTWM_RC_UNSUPPORTED, "matvec: more than 2^19 tokens in a call");
    if (!tokens) return 0;
    if (!x || !y) return fail(PTWM_RC_INVALID_INPUT, "matvec: null device pointer");
    DeviceGuard guard{int(device)};
    if (guard.err != cudaSuccess) return fail(PTWM_RC_CUDA, std::string("cudaSetDevice: ") + cudaGetErrorString(guard.err));
    const TokenArgs t{at<void>(x), at<void>(x_scales), tokens, x_scaled, at<void>(y)};
    const dim3 grid(uint32_t((w.rows + 7) / 8), uint32_t((tokens + 7) / 8));
    with_type(y_dtype, [&](auto o) {
        if (x_dtype == DT_E4M3) matvec_kernel<uint8_t, decltype(o)><<<grid, 256, 0, stream_of(stream)>>>(w, t);
        else with_type(x_dtype, [&](auto v) { matvec_kernel<decltype(v), decltype(o)><<<grid, 256, 0, stream_of(stream)>>>(w, t); });
    });
    CUDA_TRY(cudaGetLastError());
    return 0;
}

extern "C" int64_t ptwm_b200_matvec_grad(const ptwm_b200_scaled_weight* weight, uint64_t dy, uint64_t dx, uint64_t tokens, uint32_t dtype, uint32_t device, uint64_t stream) {
    ScaledMatrix w;
    if (const int64_t rc = matrix_of(weight, &w); rc < 0) return rc;
    if (!plain_type(dtype)) return fail(PTWM_RC_UNSUPPORTED, "matvec_grad: gradients are fp32, fp16 or bf16");
    if (tokens > (1u << 19)) return fail(PTWM_RC_UNSUPPORTED, "matvec_grad: more than 2^19 tokens in a call");
    if (!tokens) return 0;
    if (!dy || !dx) return fail(PTWM_RC_INVALID_INPUT, "matvec_grad: null device pointer");
    DeviceGuard guard{int(device)};
    if (guard.err != cudaSuccess) return fail(PTWM_RC_CUDA, std::string("cudaSetDevice: ") + cudaGetErrorString(guard.err));
    const TokenArgs t{at<void>(dy), nullptr, tokens, SCALE_NONE, at<void>(dx)};
    const dim3 grid(uint32_t((w.cols / 2 + 127) / 128), uint32_t((tokens + 7) / 8));
    with_type(dtype, [&](auto v) { matvec_grad_kernel<decltype(v)><<<grid, 128, 0, stream_of(stream)>>>(w, t); });
    CUDA_TRY(cudaGetLastError());
    return 0;
}
