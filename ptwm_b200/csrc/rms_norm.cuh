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
#include <type_traits>

#include "number_types.cuh"

namespace ptwm {

struct NormArgs {
    const void *x, *residual, *weight;
    void *h, *y, *scales;
    uint64_t rows, cols;
    float eps;
};

// The larger magnitude; NaN wins.
__device__ __forceinline__ float max_magnitude(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(fabsf(a)), "f"(fabsf(b)));
    return r;
}

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

// 16 bytes of a row, as pairs of numbers: an instruction has a pair of sums or products.
template <class T> struct Piece {
    static constexpr int V = 16 / sizeof(T), P = V / 2;
    float2 v[P];
};
template <class T> __device__ __forceinline__ Piece<T> numbers(const uint4& w) {
    Piece<T> p;
    if constexpr (sizeof(T) == 4) {
        p.v[0] = make_float2(__uint_as_float(w.x), __uint_as_float(w.y));
        p.v[1] = make_float2(__uint_as_float(w.z), __uint_as_float(w.w));
    } else {
        p.v[0] = two_f32<T>(w.x); p.v[1] = two_f32<T>(w.y);
        p.v[2] = two_f32<T>(w.z); p.v[3] = two_f32<T>(w.w);
    }
    return p;
}
template <class T> __device__ __forceinline__ uint4 rounded(const Piece<T>& p) {
    if constexpr (sizeof(T) == 4) return make_uint4(__float_as_uint(p.v[0].x), __float_as_uint(p.v[0].y), __float_as_uint(p.v[1].x), __float_as_uint(p.v[1].y));
    else return make_uint4(two_rounded<T>(p.v[0]), two_rounded<T>(p.v[1]), two_rounded<T>(p.v[2]), two_rounded<T>(p.v[3]));
}
// The weights that belong to piece i of a row of T.
template <class T, class W> __device__ __forceinline__ Piece<T> weights(const void* weight, uint32_t i) {
    constexpr int PIECES = Piece<T>::V * sizeof(W) / 16;
    Piece<T> p;
    if constexpr (PIECES == 0) {  // fp32 rows, 16-bit weights: half a piece
        const uint2 w = __ldg(static_cast<const uint2*>(weight) + i);
        p.v[0] = two_f32<W>(w.x);
        p.v[1] = two_f32<W>(w.y);
    } else {
#pragma unroll
        for (int j = 0; j < PIECES; ++j) {
            const Piece<W> w = numbers<W>(__ldg(static_cast<const uint4*>(weight) + i * PIECES + j));  // (as an intrinsic: a plain load becomes eight of two bytes)
#pragma unroll
            for (int k = 0; k < Piece<W>::P; ++k) p.v[j * Piece<W>::P + k] = w.v[k];
        }
    }
    return p;
}
template <class T> __device__ __forceinline__ Piece<T> zeros() { Piece<T> p = {}; return p; }

// A sum and (TWO) a second one or (MOST) a largest magnitude, over the warp and, where a row has several, over the block: the warps'
// results are read back as they lie, four at a time, which is less work than another round of shuffles.
// LANES: 32, or 16 where a warp has two rows.
template <bool TWO, bool MOST, int LANES = 32> __device__ __forceinline__ void reduce(float& a, float& b, uint32_t warps, float (*shared)[32]) {
#pragma unroll
    for (int o = LANES / 2; o; o >>= 1) {
        a += __shfl_xor_sync(0xFFFFFFFFu, a, o);
        if (TWO) b += __shfl_xor_sync(0xFFFFFFFFu, b, o);
    }
    // magnitudes compare as whole numbers, and a NaN is above infinity
    if (MOST) b = __uint_as_float(__reduce_max_sync(LANES == 32 ? 0xFFFFFFFFu : 0xFFFFu << (threadIdx.x & 16), __float_as_uint(b)));
    if (warps == 1) return;
    const uint32_t warp = threadIdx.x / 32, up = (warps + 3) / 4 * 4;
    if ((threadIdx.x & 31) == 0) { shared[0][warp] = a; if (TWO || MOST) shared[1][warp] = b; }
    if (threadIdx.x >= warps && threadIdx.x < up) shared[0][threadIdx.x] = shared[1][threadIdx.x] = 0;  // (a warp has 32 threads: there are as many)
    __syncthreads();
    a = 0; b = 0;
    for (uint32_t i = 0; i < up; i += 4) {
        const float4 v = *reinterpret_cast<const float4*>(&shared[0][i]);
        a += (v.x + v.y) + (v.z + v.w);
        if (TWO || MOST) {
            const float4 u = *reinterpret_cast<const float4*>(&shared[1][i]);
            if (TWO) b += (u.x + u.y) + (u.z + u.w);
            else b = max_magnitude(max_magnitude(b, max_magnitude(u.x, u.y)), max_magnitude(u.z, u.w));
        }
    }
}

// A piece's numbers as E4M3, the first in the lowest byte.
template <class T> __device__ __forceinline__ typename std::conditional<Piece<T>::V == 8, uint2, uint32_t>::type pack_e4m3(const Piece<T>& p) {
    uint32_t out[Piece<T>::V / 4];
#pragma unroll
    for (int i = 0; i < Piece<T>::P; i += 2) {
        uint16_t lo, hi;  // the conversion puts its first operand in the upper byte
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(p.v[i].y), "f"(p.v[i].x));
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(p.v[i + 1].y), "f"(p.v[i + 1].x));
        out[i / 2] = uint32_t(lo) | uint32_t(hi) << 16;
    }
    if constexpr (Piece<T>::V == 8) return make_uint2(out[0], out[1]);
    else return out[0];
}
__device__ __forceinline__ float max_magnitude(float a, float2 b) { return max_magnitude(max_magnitude(a, b.x), b.y); }

template <class T> __device__ __forceinline__ void times(Piece<T>& p, float f) {
#pragma unroll
    for (int k = 0; k < Piece<T>::P; ++k) p.v[k] = __fmul2_rn(p.v[k], make_float2(f, f));
}

// A row's way into E4M3, from its largest |h weight| and r.
struct RowScale {
    float most, r, top, inverse;
    __device__ __forceinline__ RowScale(float most, float r) : most(most), r(r), top(most * r), inverse(0) {
        if (is_finite(top) && top > 0x1p-100f && most > 0x1p-100f) inverse = 448.0f / most;  // nearly always: a product for a division
    }
    __device__ __forceinline__ float scale() const { return is_finite(top) ? top / 448.0f : __uint_as_float(0x7FC00000u); }
    template <class T, int N> __device__ __forceinline__ void apply(Piece<T> (&t)[N]) const {
        if (inverse != 0.0f) {
#pragma unroll
            for (int j = 0; j < N; ++j) times(t[j], inverse);
            return;
        }
        // part is 0 only where s is, and not finite only where s is not
        const float s = scale(), part = most / 448.0f;
        auto divided = [&](float v) { return s == 0.0f ? 0.0f : s == s ? v / part : s; };
#pragma unroll
        for (int j = 0; j < N; ++j)
#pragma unroll
            for (int k = 0; k < Piece<T>::P; ++k) t[j].v[k] = make_float2(divided(t[j].v[k].x), divided(t[j].v[k].y));
    }
};

// Rows that start at multiples of 16 bytes.  Bound by memory, so everything is read once and a row stays in registers: N pieces of 16
// bytes to a thread, a row to 16 or 32 lanes (LANES) or to a block (0), which has the next row on its way while it reduces one.  One reduction is
// enough for any output: with t = h weight the largest |y| is r times the largest |t| (rounding keeps the order), and
// q = t / (max|t| / 448) needs no r at all.
//   8192 rows of 4096 bf16 with a residual: 39 us into E4M3 with row or block scales, 6.0 TB/s; 44.5 us into bf16; 60000 rows of 512:
// 36.2 us, 5.9 TB/s; 200,000 of 128: 33.6 us.  One row of 4096: 2.3 us.  A value took 29 instructions when each was taken out of its
// word and added, multiplied and rounded by itself, three quarters of what the SMs can issue: 38.2 us for the rows of 512.
template <class T, class W, int N, int LANES, uint32_t QUANT>
__global__ void __launch_bounds__(LANES ? 256 : 1024) rms_norm_rows_kernel(NormArgs a) {
    constexpr int V = Piece<T>::V, P = Piece<T>::P;
    constexpr bool WARP = LANES != 0;
    constexpr uint32_t PER = WARP ? LANES : 1;
    __shared__ __align__(16) float shared[2][2][32];
    const uint32_t lanes = WARP ? PER : blockDim.x, at = WARP ? threadIdx.x % PER : threadIdx.x, pieces = uint32_t(a.cols / V);
    const uint64_t step = WARP ? uint64_t(gridDim.x) * (blockDim.x / PER) : gridDim.x;
    uint64_t row = WARP ? uint64_t(blockIdx.x) * (blockDim.x / PER) + threadIdx.x / PER : blockIdx.x;
    const uint4 *xs = static_cast<const uint4*>(a.x), *rs = static_cast<const uint4*>(a.residual);
    uint4 in[N], more[N];
    auto ask = [&](uint64_t r) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const uint32_t i = at + j * lanes;
            in[j] = more[j] = make_uint4(0, 0, 0, 0);
            if (r < a.rows && i < pieces) {
                in[j] = __ldcs(xs + r * pieces + i);
                if (rs) more[j] = __ldcs(rs + r * pieces + i);
            }
        }
    };
    others_may_start();
    after_those_before();
    ask(row);
    // (two rows of a warp go on together: the shuffles want both)
    for (uint32_t turn = 0; LANES == 16 ? __any_sync(0xFFFFFFFFu, row < a.rows) : row < a.rows; row += step, turn ^= 1) {
        const bool there = LANES != 16 || row < a.rows;
        Piece<T> t[N];
        float2 sums = {};
        float most = 0;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const uint32_t i = at + j * lanes;
            const Piece<T> w = i < pieces ? weights<T, W>(a.weight, i) : zeros<T>();
            Piece<T> h = numbers<T>(in[j]);
            if (rs) {
                const Piece<T> r = numbers<T>(more[j]);
#pragma unroll
                for (int k = 0; k < P; ++k) h.v[k] = __fadd2_rn(h.v[k], r.v[k]);
                const uint4 stored = rounded<T>(h);
                if (there && i < pieces) static_cast<uint4*>(a.h)[row * pieces + i] = stored;
                h = numbers<T>(stored);
            }
#pragma unroll
            for (int k = 0; k < P; ++k) {
                sums = __ffma2_rn(h.v[k], h.v[k], sums);
                t[j].v[k] = __fmul2_rn(h.v[k], w.v[k]);
                if (QUANT == SCALE_ROW) most = max_magnitude(most, t[j].v[k]);
            }
        }
        float sum = sums.x + sums.y;
        ask(row + step);
        reduce<false, QUANT == SCALE_ROW, LANES == 16 ? 16 : 32>(sum, most, WARP ? 1 : lanes / 32, shared[turn]);
        const float r = __frsqrt_rn(sum / float(a.cols) + a.eps);
        if constexpr (QUANT == SCALE_NONE) {
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const uint32_t i = at + j * lanes;
                times(t[j], r);
                if (there && i < pieces) static_cast<uint4*>(a.y)[row * pieces + i] = rounded<T>(t[j]);
            }
        } else {
            auto* q = static_cast<decltype(pack_e4m3(t[0]))*>(a.y) + row * pieces;
            if constexpr (QUANT == SCALE_ROW) {
                const RowScale scale(most, r);
                if (there && at == 0) static_cast<float*>(a.scales)[row] = scale.scale();
                scale.apply(t);
            }
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const uint32_t i = at + j * lanes;
                if constexpr (QUANT == SCALE_BLOCK) {
                    float m = 0;
#pragma unroll
                    for (int k = 0; k < P; ++k) m = max_magnitude(m, t[j].v[k]);
#pragma unroll
                    for (int o = 1; o < 32 / V; o *= 2) m = max_magnitude(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));  // the threads of a block of 32
                    const uint32_t e = block_scale(m * r);
                    times(t[j], r);
                    times(t[j], block_inverse(e));
                    if (there && i < pieces && i % (32 / V) == 0) static_cast<uint8_t*>(a.scales)[row * (a.cols / 32) + i / (32 / V)] = uint8_t(e);
                }
                if (there && i < pieces) q[i] = pack_e4m3(t[j]);
            }
        }
    }
}

// The weights from number `o` on, which may begin before the first and end behind the last of them: zeros there.  Pieces that cover them are
// put in place by whole words and then by half of one; the block's threads have the same way to go.
template <class T, class W> __device__ __forceinline__ Piece<T> weights_from(const void* weight, int o, int cols) {
    constexpr int V = Piece<T>::V, G = sizeof(W) == 2 ? V : 4, WORDS = G * int(sizeof(W)) / 4, PIECES = V / G + 1, HALF = 4 / int(sizeof(W));
    Piece<T> p;
    const int first = (o >= 0 ? o : o - G + 1) / G, s = o - first * G;
    if (first >= 0 && (first + PIECES) * G <= cols) {
        uint32_t w[WORDS * PIECES];
#pragma unroll
        for (int j = 0; j < PIECES; ++j)
            if constexpr (WORDS == 4) {
                const uint4 v = __ldg(static_cast<const uint4*>(weight) + first + j);
                w[4 * j] = v.x; w[4 * j + 1] = v.y; w[4 * j + 2] = v.z; w[4 * j + 3] = v.w;
            } else {
                const uint2 v = __ldg(static_cast<const uint2*>(weight) + first + j);
                w[2 * j] = v.x; w[2 * j + 1] = v.y;
            }
#pragma unroll
        for (int b = WORDS / 2; b; b /= 2)
            if (s & (b * HALF)) {
#pragma unroll
                for (int j = 0; j + b < WORDS * PIECES; ++j) w[j] = w[j + b];
            }
        if constexpr (HALF == 2) {
            if (s & 1) {
#pragma unroll
                for (int j = 0; j + 1 < WORDS * PIECES; ++j) w[j] = __funnelshift_r(w[j], w[j + 1], 16);
            }
#pragma unroll
            for (int k = 0; k < V / 2; ++k) p.v[k] = two_f32<W>(w[k]);
        } else {
#pragma unroll
            for (int k = 0; k < V / 2; ++k) p.v[k] = make_float2(__uint_as_float(w[2 * k]), __uint_as_float(w[2 * k + 1]));
        }
    } else {
        auto one = [&](int k) { return k >= 0 && k < cols ? to_f32(static_cast<const W*>(weight)[k]) : 0.0f; };
#pragma unroll
        for (int k = 0; k < V / 2; ++k) p.v[k] = make_float2(one(o + 2 * k), one(o + 2 * k + 1));
    }
    return p;
}

// A piece of a tensor of so many values, whose last one may be cut short.
template <class T> __device__ __forceinline__ uint4 load_piece(const T* p, uint64_t piece, uint64_t values) {
    constexpr int V = Piece<T>::V;
    if ((piece + 1) * V <= values) return __ldcs(reinterpret_cast<const uint4*>(p) + piece);
    uint32_t w[4] = {};
#pragma unroll
    for (int k = 0; k < V; ++k)
        if (piece * V + k < values) {
            if constexpr (V == 4) w[k] = __float_as_uint(p[piece * V + k]);
            else w[k / 2] |= uint32_t(reinterpret_cast<const uint16_t*>(p)[piece * V + k]) << (k % 2 * 16);
        }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
// Of a piece whose first value has place `o` in a row (which may be before it): what is the row's, to memory, or with zeros for the rest.
template <class T> __device__ __forceinline__ void store_piece(T* to, int o, int cols, const uint4& w) {
    constexpr int V = Piece<T>::V;
    if (o >= 0 && o + V <= cols) {
        *reinterpret_cast<uint4*>(to) = w;
        return;
    }
    const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int k = 0; k < V; ++k)
        if (o + k >= 0 && o + k < cols) {
            if constexpr (V == 4) to[k] = __uint_as_float(words[k]);
            else reinterpret_cast<uint16_t*>(to)[k] = uint16_t(words[k / 2] >> (k % 2 * 16));
        }
}
template <bool BETWEEN, class T> __device__ __forceinline__ void store_e4m3(uint8_t* to, int o, int cols, const Piece<T>& p) {
    auto q = pack_e4m3(p);
    if constexpr (BETWEEN)
        if (o < 0 || o + Piece<T>::V > cols) {
#pragma unroll
            for (int k = 0; k < Piece<T>::V; ++k)
                if (o + k >= 0 && o + k < cols) {
                    if constexpr (Piece<T>::V == 4) to[k] = uint8_t(q >> (k * 8));
                    else to[k] = uint8_t((k < 4 ? q.x : q.y) >> (k % 4 * 8));
                }
            return;
        }
    *reinterpret_cast<decltype(q)*>(to) = q;
}
template <class T> __device__ __forceinline__ void keep_own(Piece<T>& p, int o, int cols) {
    if (o >= 0 && o + Piece<T>::V <= cols) return;
    auto own = [&](int k) { return o + k >= 0 && o + k < cols; };
#pragma unroll
    for (int k = 0; k < Piece<T>::P; ++k) p.v[k] = make_float2(own(2 * k) ? p.v[k].x : 0.0f, own(2 * k + 1) ? p.v[k].y : 0.0f);
}

// Rows of a length that no piece divides, in tensors that start at multiples of 16 bytes: the pieces are those of the whole tensor, so that
// everything but the weights still moves 16 bytes at a time; of the two at a row's ends, which belong to its neighbours as well, a
// block takes what is its own.  Two pieces to a thread, a row to a block, with the next one on its way.
//   8192 rows of 4097 bf16 with a residual into E4M3: 56.5 us, 4.2 TB/s (131.7 with a value to a load); 333 of 10501 fp16: 8.7 us (12.4), of
// which a row from memory to memory by itself takes 3.7.  Bound by instructions, two a value of them to put the weights in place.
template <class T, class W>
__global__ void __launch_bounds__(1024) rms_norm_between_kernel(NormArgs a, uint32_t quant) {
    constexpr int V = Piece<T>::V, P = Piece<T>::P, N = 2;
    __shared__ __align__(16) float shared[2][2][32];
    const uint32_t at = threadIdx.x, lanes = blockDim.x;
    const int cols = int(a.cols);
    const uint64_t values = a.rows * a.cols;
    const T *xs = static_cast<const T*>(a.x), *rs = static_cast<const T*>(a.residual);
    uint4 in[N], more[N];
    auto ask = [&](uint64_t row) {
        const uint64_t first = row * a.cols / V, end = (row + 1) * a.cols;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const uint64_t piece = first + at + j * lanes;
            in[j] = more[j] = make_uint4(0, 0, 0, 0);
            if (row < a.rows && piece * V < end) {
                in[j] = load_piece(xs, piece, values);
                if (rs) more[j] = load_piece(rs, piece, values);
            }
        }
    };
    others_may_start();
    after_those_before();
    ask(blockIdx.x);
    uint32_t turn = 0;
    for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
        const uint64_t first = row * a.cols / V;
        const int before = int(row * a.cols % V);   // values of the first piece that are the row's before
        Piece<T> t[N];
        float2 sums = {};
        float most = 0;
        auto place = [&](int j) { return int(at + j * lanes) * V - before; };  // of a piece in its row
        auto number = [&](int j) { return (first + at + j * lanes) * V; };            // of its first value in the tensor
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int o = place(j);
            Piece<T> h = numbers<T>(in[j]);
            if (rs) {
                const Piece<T> r = numbers<T>(more[j]);
#pragma unroll
                for (int k = 0; k < P; ++k) h.v[k] = __fadd2_rn(h.v[k], r.v[k]);
                const uint4 stored = rounded<T>(h);
                store_piece(static_cast<T*>(a.h) + number(j), o, cols, stored);
                h = numbers<T>(stored);
            }
            keep_own(h, o, cols);
            const Piece<T> w = weights_from<T, W>(a.weight, o, cols);
#pragma unroll
            for (int k = 0; k < P; ++k) {
                sums = __ffma2_rn(h.v[k], h.v[k], sums);
                t[j].v[k] = __fmul2_rn(h.v[k], w.v[k]);
                most = max_magnitude(most, t[j].v[k]);
            }
        }
        ask(row + gridDim.x);
        float sum = sums.x + sums.y;
        reduce<false, true>(sum, most, lanes / 32, shared[turn]);
        const RowScale scale(most, __frsqrt_rn(sum / float(a.cols) + a.eps));
        if (quant == SCALE_ROW) {
            if (at == 0) static_cast<float*>(a.scales)[row] = scale.scale();
            scale.apply(t);
        }
#pragma unroll
        for (int j = 0; j < N; ++j) {
            if (quant == SCALE_NONE) {
                times(t[j], scale.r);
                store_piece(static_cast<T*>(a.y) + number(j), place(j), cols, rounded<T>(t[j]));
                continue;
            }
            store_e4m3<true, T>(static_cast<uint8_t*>(a.y) + number(j), place(j), cols, t[j]);
        }
    }
}

// Rows that registers do not hold: twice over them, the second time from the caches, where what the rows of all blocks take has room.  BETWEEN:
// pieces of the whole tensor, as above.  2048 rows of 14336 fp32 with a residual: 92 us, 5.1 TB/s (a value to a load 122), into E4M3 with row or
// block scales 80 and 93 (124, 174); 1024 of 28672 bf16 62 (147).  Bound by memory and the second pass' trips to the L2.
template <class T, class W, bool BETWEEN>
__global__ void __launch_bounds__(512, 2) rms_norm_wide_kernel(NormArgs a, uint32_t quant) {
    constexpr int V = Piece<T>::V, P = Piece<T>::P;
    __shared__ __align__(16) float shared[2][32];
    const uint64_t row = blockIdx.x, begin = row * a.cols, first = begin / V, values = a.rows * a.cols;
    const int cols = int(a.cols), before = int(begin % V);
    const uint32_t pieces = (uint32_t(cols) + before + V - 1) / V, lanes = blockDim.x;
    const T *x = static_cast<const T*>(a.x), *res = static_cast<const T*>(a.residual);
    T* const h_out = static_cast<T*>(a.h);
    others_may_start();
    after_those_before();
    auto load = [&](const T* p, uint32_t i) {
        if constexpr (BETWEEN) return load_piece(p, first + i, values);
        else return __ldcg(reinterpret_cast<const uint4*>(p) + first + i);
    };
    auto store = [&](T* p, uint32_t i, const uint4& w) {
        if constexpr (BETWEEN) store_piece(p + (first + i) * V, int(i * V) - before, cols, w);
        else reinterpret_cast<uint4*>(p)[first + i] = w;
    };
    auto weight_of = [&](uint32_t i) {
        if constexpr (BETWEEN) return weights_from<T, W>(a.weight, int(i * V) - before, cols);
        else return weights<T, W>(a.weight, i);
    };
    float2 sums = {};
    float most = 0;
#pragma unroll 4
    for (uint32_t i = threadIdx.x; i < pieces; i += lanes) {
        Piece<T> h = numbers<T>(load(x, i));
        if (res) {
            const Piece<T> r = numbers<T>(load(res, i));
#pragma unroll
            for (int k = 0; k < P; ++k) h.v[k] = __fadd2_rn(h.v[k], r.v[k]);
            const uint4 stored = rounded<T>(h);
            store(h_out, i, stored);
            h = numbers<T>(stored);
        }
        if (BETWEEN) keep_own(h, int(i * V) - before, cols);
#pragma unroll
        for (int k = 0; k < P; ++k) sums = __ffma2_rn(h.v[k], h.v[k], sums);
        if (quant == SCALE_ROW) {
            const Piece<T> w = weight_of(i);
#pragma unroll
            for (int k = 0; k < P; ++k) most = max_magnitude(most, __fmul2_rn(h.v[k], w.v[k]));
        }
    }
    float sum = sums.x + sums.y;
    reduce<false, true>(sum, most, lanes / 32, shared);
    const float r = __frsqrt_rn(sum / float(a.cols) + a.eps);
    const RowScale scale(most, r);
    if (quant == SCALE_ROW && threadIdx.x == 0) static_cast<float*>(a.scales)[row] = scale.scale();
    for (uint32_t base = 0; base < pieces; base += lanes) {   // (a warp stays together: blocks of 32 values are several threads')
        const uint32_t i = base + threadIdx.x;
        Piece<T> t[1] = {};
        if (i < pieces) {
            // what this thread stored; of a piece that another row shares, what is not this row's does not matter
            t[0] = numbers<T>(load(res ? h_out : x, i));
            const Piece<T> w = weight_of(i);
#pragma unroll
            for (int k = 0; k < P; ++k) t[0].v[k] = __fmul2_rn(t[0].v[k], w.v[k]);
        }
        if (quant == SCALE_NONE) {
            times(t[0], r);
            if (i < pieces) store(static_cast<T*>(a.y), i, rounded<T>(t[0]));
            continue;
        }
        if (quant == SCALE_ROW) scale.apply(t);
        else {
            float m = 0;
#pragma unroll
            for (int k = 0; k < P; ++k) m = max_magnitude(m, t[0].v[k]);
#pragma unroll
            for (int o = 1; o < 32 / V; o *= 2) m = max_magnitude(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
            const uint32_t e = block_scale(m * r);
            times(t[0], r);
            times(t[0], block_inverse(e));
            if (i < pieces && i % (32 / V) == 0) static_cast<uint8_t*>(a.scales)[row * (a.cols / 32) + i / (32 / V)] = uint8_t(e);
        }
        if (i < pieces) store_e4m3<BETWEEN, T>(static_cast<uint8_t*>(a.y) + (first + i) * V, int(i * V) - before, cols, t[0]);
    }
}

// Rows that start anywhere (8192 of 4097 bf16 with a residual: 131.7 us), a value at a time: N values to a thread, a row to a block.
template <class T, class W, int N>
__global__ void __launch_bounds__(1024, 2) rms_norm_odd_rows_kernel(NormArgs a, uint32_t quant) {
    __shared__ __align__(16) float shared[2][32];
    const uint32_t cols = uint32_t(a.cols), lanes = blockDim.x;
    const uint64_t first = uint64_t(blockIdx.x) * cols;
    const T *x = static_cast<const T*>(a.x) + first, *res = static_cast<const T*>(a.residual) + first;
    const W* w = static_cast<const W*>(a.weight);
    others_may_start();
    after_those_before();
    float t[N], sum = 0, most = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const uint32_t k = threadIdx.x + j * lanes;
        t[j] = k < cols ? to_f32(x[k]) : 0.0f;
    }
    if (a.residual)
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const uint32_t k = threadIdx.x + j * lanes;
            if (k < cols) {
                const T h = from_f32<T>(t[j] + to_f32(res[k]));
                static_cast<T*>(a.h)[first + k] = h;
                t[j] = to_f32(h);
            }
        }
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const uint32_t k = threadIdx.x + j * lanes;
        sum += t[j] * t[j];
        t[j] = k < cols ? t[j] * to_f32(w[k]) : 0.0f;
        most = max_magnitude(most, fabsf(t[j]));
    }
    reduce<false, true>(sum, most, lanes / 32, shared);
    const float r = __frsqrt_rn(sum / float(cols) + a.eps), s = is_finite(most * r) ? most * r / 448.0f : __uint_as_float(0x7FC00000u), part = most / 448.0f, inverse = 448.0f / most;
    const bool plain = s > 0.0f && most > 0x1p-100f;
    if (quant == SCALE_ROW && threadIdx.x == 0) static_cast<float*>(a.scales)[blockIdx.x] = s;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const uint32_t k = threadIdx.x + j * lanes;
        if (k >= cols) continue;
        if (quant == SCALE_ROW) static_cast<uint8_t*>(a.y)[first + k] = f32_e4m3(plain ? t[j] * inverse : s == 0.0f ? 0.0f : s == s ? t[j] / part : s);
        else static_cast<T*>(a.y)[first + k] = from_f32<T>(t[j] * r);
    }
}

// Rows of any length and place: a block per row, twice over it, a value to a load (1024 of 28672 bf16 147 us; pieces of 16 bytes take 62).
template <class T, class W>
__global__ void __launch_bounds__(256) rms_norm_long_kernel(NormArgs a, uint32_t quant) {
    __shared__ __align__(16) float shared[2][32];
    const uint64_t row = blockIdx.x, cols = a.cols;
    const T* x = static_cast<const T*>(a.x) + row * cols;
    const T* res = a.residual ? static_cast<const T*>(a.residual) + row * cols : nullptr;
    T* h = a.residual ? static_cast<T*>(a.h) + row * cols : nullptr;
    const W* w = static_cast<const W*>(a.weight);
    others_may_start();
    after_those_before();
    float sum = 0, most = 0;
    for (uint64_t k = threadIdx.x; k < cols; k += blockDim.x) {
        float v = to_f32(x[k]);
        if (res) { const T s = from_f32<T>(v + to_f32(res[k])); h[k] = s; v = to_f32(s); }
        sum += v * v;
        most = max_magnitude(most, fabsf(v * to_f32(w[k])));
    }
    reduce<false, true>(sum, most, blockDim.x / 32, shared);
    const float r = __frsqrt_rn(sum / float(cols) + a.eps), s = is_finite(most * r) ? most * r / 448.0f : __uint_as_float(0x7FC00000u), part = most / 448.0f;
    const T* in = res ? h : x;
    uint8_t* q = static_cast<uint8_t*>(a.y) + row * cols;
    if (quant == SCALE_ROW && threadIdx.x == 0) static_cast<float*>(a.scales)[row] = s;
    for (uint64_t k = threadIdx.x; k < cols; k += blockDim.x) {  // a warp has a block of 32 values at a time, or less than one at the end
        const float t = to_f32(in[k]) * to_f32(w[k]);
        if (quant == SCALE_NONE) static_cast<T*>(a.y)[row * cols + k] = from_f32<T>(t * r);
        else if (quant == SCALE_ROW) q[k] = f32_e4m3(s == 0.0f ? 0.0f : s == s ? t / part : s);
        else {
            float m = fabsf(t);
            for (int o = 16; o; o >>= 1) m = max_magnitude(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
            const uint32_t e = block_scale(m * r);
            q[k] = f32_e4m3(t * r * block_inverse(e));
            if ((threadIdx.x & 31) == 0) static_cast<uint8_t*>(a.scales)[row * (cols / 32) + k / 32] = uint8_t(e);
        }
    }
}

// Gradient.  With g = dy weight:  dx = dh + r g - (h r) (sum(g h) r / K r)  (the residual's is the same),  dweight = sum over rows of dy (h r).
// In this order every number in between has the size of g, of r g or of a normed value.  r^3, with which the second term may also be written, leaves fp32's range from a
// root mean square of 10^13 on, and below 10^-13 without eps.
struct NormGradArgs {
    const void *h, *weight, *dy, *dh;
    void* dx;
    float* partial;   // [blocks, cols]: each block's share of dweight
    void* dweight;
    uint64_t rows, cols;
    float eps;
    uint32_t blocks;
};

// A block takes rows blockIdx.x, + blocks, ...  Its threads keep their columns, N pieces of 16 bytes, and with them their sums for
// dweight in registers; with 512 of them the next row is asked for before this one's reduction, which 64 registers of 1024 do not hold.
// Bound by memory and, at half its rate, by what a row waits for its reduction: 4096 rows of 4096 with the residual's gradient take 30.7 us
// in bf16 (4.4 TB/s; a value at a time took 6 % more), 49.9 in fp32 (5.4 TB/s), the weights' sum with it.
// BETWEEN: rows of a length that no piece divides, with the pieces of the whole tensor.  The blocks are as many as makes each one's rows
// begin at the same place of a piece, so a thread has the same columns in all of them (4096 rows of 4097: 66 us, 170 a value at a time).
template <class T, class W, int N, int MOST, bool BETWEEN>
__global__ void __launch_bounds__(MOST, N == 1 ? 2 : 1) rms_norm_grad_rows_kernel(NormGradArgs a) {
    constexpr int V = Piece<T>::V, P = Piece<T>::P;
    __shared__ __align__(16) float shared[2][2][32];
    const uint32_t lanes = blockDim.x, at = threadIdx.x;
    const int cols = int(a.cols), before = BETWEEN ? int(blockIdx.x * a.cols % V) : 0;
    const uint32_t pieces = uint32_t(cols + before + (BETWEEN ? V - 1 : 0)) / V;
    const uint64_t values = a.rows * a.cols;
    auto place = [&](int j) { return int(at + j * lanes) * V - before; };
    const uint4 *hs = static_cast<const uint4*>(a.h), *dys = static_cast<const uint4*>(a.dy), *dhs = static_cast<const uint4*>(a.dh);
    uint4 h[N], dy[N], dh[N];
    auto ask = [&](uint64_t row) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const uint32_t i = at + j * lanes;
            h[j] = dy[j] = dh[j] = make_uint4(0, 0, 0, 0);
            if (row < a.rows && i < pieces) {
                if constexpr (BETWEEN) {
                    const uint64_t piece = row * a.cols / V + i;
                    h[j] = load_piece(static_cast<const T*>(a.h), piece, values);
                    dy[j] = load_piece(static_cast<const T*>(a.dy), piece, values);
                    if (dhs) dh[j] = load_piece(static_cast<const T*>(a.dh), piece, values);
                } else {
                    h[j] = __ldcs(hs + row * pieces + i);
                    dy[j] = __ldcs(dys + row * pieces + i);
                    if (dhs) dh[j] = __ldcs(dhs + row * pieces + i);
                }
            }
        }
    };
    Piece<T> dw[N] = {}, kept;
    // the weights: in registers where a thread has one piece, else again for every use (they stay in the L1)
    auto weights_of = [&](int j) {
        if constexpr (BETWEEN) return weights_from<T, W>(a.weight, place(j), cols);
        else return at + j * lanes < pieces ? weights<T, W>(a.weight, at + j * lanes) : zeros<T>();
    };
    others_may_start();
    after_those_before();
    if (N == 1) kept = weights_of(0);
    if (MOST <= 512) ask(blockIdx.x);
    uint32_t turn = 0;
    for (uint64_t row = blockIdx.x; row < a.rows; row += a.blocks, turn ^= 1) {
        if (MOST > 512) ask(row);
        float2 sqs = {}, dots = {};
        Piece<T> v[N], d[N];
        uint4 r0[N];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            v[j] = numbers<T>(h[j]);
            d[j] = numbers<T>(dy[j]);
            if (BETWEEN) {
                keep_own(v[j], place(j), cols);
                keep_own(d[j], place(j), cols);
            }
            r0[j] = dh[j];
            const Piece<T> w = N > 1 ? weights_of(j) : kept;
#pragma unroll
            for (int k = 0; k < P; ++k) {
                sqs = __ffma2_rn(v[j].v[k], v[j].v[k], sqs);
                dots = __ffma2_rn(__fmul2_rn(d[j].v[k], w.v[k]), v[j].v[k], dots);
            }
        }
        float sq = sqs.x + sqs.y, dot = dots.x + dots.y;
        if (MOST <= 512) ask(row + a.blocks);
        reduce<true, false>(sq, dot, lanes / 32, shared[turn]);
        const float r = __frsqrt_rn(sq / float(a.cols) + a.eps), c = dot * r / float(a.cols) * r;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const uint32_t i = at + j * lanes;
            Piece<T> g;
            const Piece<T> w = N > 1 ? weights_of(j) : kept;
#pragma unroll
            for (int k = 0; k < P; ++k) {
                const float2 n = __fmul2_rn(v[j].v[k], make_float2(r, r));
                g.v[k] = __ffma2_rn(__fmul2_rn(d[j].v[k], make_float2(r, r)), w.v[k], __fmul2_rn(n, make_float2(-c, -c)));
                dw[j].v[k] = __ffma2_rn(d[j].v[k], n, dw[j].v[k]);
            }
            if (dhs) {
                const Piece<T> e = numbers<T>(r0[j]);
#pragma unroll
                for (int k = 0; k < P; ++k) g.v[k] = __fadd2_rn(g.v[k], e.v[k]);
            }
            if (a.dx && i < pieces) {
                if constexpr (BETWEEN) store_piece(static_cast<T*>(a.dx) + (row * a.cols / V + i) * V, place(j), cols, rounded<T>(g));
                else static_cast<uint4*>(a.dx)[row * pieces + i] = rounded<T>(g);
            }
        }
    }
    if (a.partial)
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const uint32_t i = at + j * lanes;
            if (BETWEEN) {
                float* to = a.partial + blockIdx.x * a.cols + place(j);
                auto own = [&](int k) { return place(j) + k >= 0 && place(j) + k < cols; };
#pragma unroll
                for (int k = 0; k < P; ++k) {
                    if (own(2 * k)) to[2 * k] = dw[j].v[k].x;
                    if (own(2 * k + 1)) to[2 * k + 1] = dw[j].v[k].y;
                }
            } else if (i < pieces)
#pragma unroll
                for (int k = 0; k < P; k += 2) *reinterpret_cast<float4*>(a.partial + blockIdx.x * a.cols + i * V + k * 2) = make_float4(dw[j].v[k].x, dw[j].v[k].y, dw[j].v[k + 1].x, dw[j].v[k + 1].y);
        }
}

// Rows that registers do not hold, up to 32 values for each of 512 threads: twice over them, the second time from the caches.  Columns and their
// sums stay with a thread, as above.  2048 rows of 14336 fp32 with the residual's gradient: 110 us, 4.3 TB/s (320 a value to a load, sums in memory); of
// 10001 137 (211).  Wider rows have the kernel below.
template <class T, class W, bool BETWEEN>
__global__ void __launch_bounds__(512, 2) rms_norm_grad_wide_kernel(NormGradArgs a) {
    constexpr int V = Piece<T>::V, P = Piece<T>::P, N = 32 / V;
    __shared__ __align__(16) float shared[2][2][32];
    const uint32_t lanes = blockDim.x;
    const int cols = int(a.cols), before = BETWEEN ? int(blockIdx.x * a.cols % V) : 0;
    const uint32_t pieces = (uint32_t(cols) + before + V - 1) / V;
    const uint64_t values = a.rows * a.cols;
    const T *hs = static_cast<const T*>(a.h), *dys = static_cast<const T*>(a.dy), *dhs = static_cast<const T*>(a.dh);
    auto place = [&](uint32_t i) { return int(i * V) - before; };
    auto load = [&](const T* p, uint64_t first, uint32_t i) {
        Piece<T> v;
        if constexpr (BETWEEN) {
            v = numbers<T>(load_piece(p, first + i, values));
            keep_own(v, place(i), cols);
        } else v = numbers<T>(__ldcg(reinterpret_cast<const uint4*>(p) + first + i));
        return v;
    };
    auto weight_of = [&](uint32_t i) {
        if constexpr (BETWEEN) return weights_from<T, W>(a.weight, place(i), cols);
        else return weights<T, W>(a.weight, i);
    };
    Piece<T> dw[N] = {};
    others_may_start();
    after_those_before();
    uint32_t turn = 0;
    for (uint64_t row = blockIdx.x; row < a.rows; row += a.blocks, turn ^= 1) {
        const uint64_t first = row * a.cols / V;
        float2 sqs = {}, dots = {};
#pragma unroll 2
        for (uint32_t i = threadIdx.x; i < pieces; i += lanes) {
            const Piece<T> v = load(hs, first, i), d = load(dys, first, i), w = weight_of(i);
#pragma unroll
            for (int k = 0; k < P; ++k) {
                sqs = __ffma2_rn(v.v[k], v.v[k], sqs);
                dots = __ffma2_rn(__fmul2_rn(d.v[k], w.v[k]), v.v[k], dots);
            }
        }
        float sq = sqs.x + sqs.y, dot = dots.x + dots.y;
        reduce<true, false>(sq, dot, lanes / 32, shared[turn]);
        const float r = __frsqrt_rn(sq / float(a.cols) + a.eps), c = dot * r / float(a.cols);
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const uint32_t i = threadIdx.x + j * lanes;
            if (i >= pieces) continue;
            const Piece<T> v = load(hs, first, i), d = load(dys, first, i), w = weight_of(i);
            Piece<T> g = dhs && a.dx ? load(dhs, first, i) : zeros<T>();
#pragma unroll
            for (int k = 0; k < P; ++k) {
                const float2 n = __fmul2_rn(v.v[k], make_float2(r, r));
                g.v[k] = __ffma2_rn(__ffma2_rn(n, make_float2(-c, -c), __fmul2_rn(d.v[k], w.v[k])), make_float2(r, r), g.v[k]);
                dw[j].v[k] = __ffma2_rn(d.v[k], n, dw[j].v[k]);
            }
            if (!a.dx) continue;
            if constexpr (BETWEEN) store_piece(static_cast<T*>(a.dx) + (first + i) * V, place(i), cols, rounded<T>(g));
            else static_cast<uint4*>(a.dx)[first + i] = rounded<T>(g);
        }
    }
    if (!a.partial) return;
    float* const to = a.partial + blockIdx.x * a.cols;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const int o = place(threadIdx.x + j * lanes);
#pragma unroll
        for (int k = 0; k < V; ++k)
            if (o + k >= 0 && o + k < cols) to[o + k] = k % 2 ? dw[j].v[k / 2].y : dw[j].v[k / 2].x;
    }
}

// Rows of any length and place; a block's sums for dweight live in `partial`, where each column belongs to one thread (1024 of 28672 bf16: 345 us).
template <class T, class W>
__global__ void __launch_bounds__(512) rms_norm_grad_long_kernel(NormGradArgs a) {
    __shared__ __align__(16) float shared[2][2][32];
    const uint64_t cols = a.cols;
    const W* w = static_cast<const W*>(a.weight);
    float* part = a.partial ? a.partial + blockIdx.x * cols : nullptr;
    others_may_start();
    after_those_before();
    if (part) for (uint64_t k = threadIdx.x; k < cols; k += blockDim.x) part[k] = 0;
    uint32_t turn = 0;
    for (uint64_t row = blockIdx.x; row < a.rows; row += a.blocks, turn ^= 1) {
        const T* h = static_cast<const T*>(a.h) + row * cols;
        const T* dy = static_cast<const T*>(a.dy) + row * cols;
        const T* dh = a.dh ? static_cast<const T*>(a.dh) + row * cols : nullptr;
        float sq = 0, dot = 0;
        for (uint64_t k = threadIdx.x; k < cols; k += blockDim.x) {
            const float v = to_f32(h[k]);
            sq += v * v;
            dot += to_f32(dy[k]) * to_f32(w[k]) * v;
        }
        reduce<true, false>(sq, dot, blockDim.x / 32, shared[turn]);
        const float r = __frsqrt_rn(sq / float(cols) + a.eps), c = dot * r / float(cols);
        for (uint64_t k = threadIdx.x; k < cols; k += blockDim.x) {
            const float n = to_f32(h[k]) * r, d = to_f32(dy[k]);
            const float g = (d * to_f32(w[k]) - n * c) * r + (dh ? to_f32(dh[k]) : 0.0f);
            if (a.dx) static_cast<T*>(a.dx)[row * cols + k] = from_f32<T>(g);
            if (part) part[k] += d * n;
        }
    }
}

// dweight from the blocks' shares: 32 columns to a block, 32 runs of shares to a column, added in their order (4096 columns of 296: 3.7 us,
// bound by the way to the L2 and back).
template <class W> __global__ void __launch_bounds__(1024) rms_norm_grad_weight_kernel(NormGradArgs a) {
    __shared__ float runs[32][33];
    const uint64_t k = uint64_t(blockIdx.x) * 32 + (threadIdx.x & 31);
    const uint32_t run = threadIdx.x / 32;
    others_may_start();
    after_those_before();
    float sum = 0;
    if (k < a.cols)
        for (uint32_t b = a.blocks * run / 32; b < a.blocks * (run + 1) / 32; ++b) sum += a.partial[b * a.cols + k];
    runs[run][threadIdx.x & 31] = sum;
    __syncthreads();
    if (run || k >= a.cols) return;
    sum = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) sum += runs[i][threadIdx.x];
    static_cast<W*>(a.dweight)[k] = from_f32<W>(sum);
}

}  // namespace ptwm
