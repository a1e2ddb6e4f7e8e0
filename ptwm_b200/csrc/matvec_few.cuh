// Products of a 4-bit matrix with up to 16 tokens.
//
// What bounds them is reading the matrix, so it goes through the SMs once, in boxes of 16 rows x 256 columns that every warp
// asks TMA for by itself, four ahead, without a barrier between warps.  A warp turns a box into the first operand of
// mma.m16n8k16 (16 rows of the matrix, 8 tokens): tcgen05 would want it written back to shared memory, or to tensor memory, in
// tiles of 128 rows first, for products that fill a sixteenth of its width.
//   Operands are fp16.  An E2M1 number fits it; so does its product with an E4M3 scale (six significant bits, 2^-10 to 2688), which
// NVFP4 takes before the MMA.  E8M0 scales range further: MXFP4 multiplies the sums of each group with them, in fp32.
//   Tokens become fp16 by a power of two that takes the largest of the block's share of them to [2^14, 2^15): bf16, fp16 and E4M3
// values down to 2^-29 of it or less are exact.  Where one is not, or tokens are fp32, what is left over goes through the same
// products again as another part, on a finer scale, until the parts are within 2^-23 of every value: one pass for nearly all
// bf16 tokens, two for fp32.
//   Columns are split over the warps of a block (`wk`) and the blocks of a cluster where rows alone do not fill the GPU; the shares are
// added in the order of the columns.
#pragma once
#include <cooperative_groups.h>

#include "matvec.cuh"
#include "tensor_core.cuh"

namespace ptwm {

constexpr uint32_t FEW_TOKENS = 16;
constexpr uint32_t BOX_COLS = 256, BOX_BYTES = 16 * BOX_COLS / 2, BOX_SCALES = 16 * 16, FEW_WARPS = 8;

struct FewArgs {
    const void* x;
    const void* x_scales;
    const float* global_scale;
    void* y;
    uint32_t* status;
    uint64_t rows, cols;
    uint32_t tokens, scaled, y_dtype, group;
    uint32_t boxes;      // of 256 columns
    uint32_t wk;         // warps of a block that share a row tile; 8 / wk row tiles to a block
    uint32_t depth;      // boxes under way per warp
    uint32_t pitch;      // bytes of a token's values in shared memory
    uint32_t wide;       // tokens can be read 8 values at a time
};

inline uint32_t few_pitch(uint32_t boxes) { return boxes * BOX_COLS * 2 + 64; }  // neighbours in different banks
inline uint32_t few_smem(uint32_t tokens, uint32_t boxes, uint32_t depth) {
    return 1024 + 1024 + FEW_WARPS * depth * (BOX_BYTES + BOX_SCALES) + tokens * few_pitch(boxes);
}

template <class T> __device__ __forceinline__ void load8(const FewArgs& a, uint64_t token, uint64_t k, float (&v)[8]) {
    const T* p = static_cast<const T*>(a.x) + token * a.cols + k;
    if (a.wide) {
        if constexpr (sizeof(T) == 4) {
            const float4 lo = reinterpret_cast<const float4*>(p)[0], hi = reinterpret_cast<const float4*>(p)[1];
            v[0] = lo.x; v[1] = lo.y; v[2] = lo.z; v[3] = lo.w; v[4] = hi.x; v[5] = hi.y; v[6] = hi.z; v[7] = hi.w;
        } else if constexpr (sizeof(T) == 2) {
            const uint4 w = *reinterpret_cast<const uint4*>(p);
            T e[8];
            memcpy(e, &w, 16);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = to_f32(e[i]);
        } else {
            const uint2 w = *reinterpret_cast<const uint2*>(p);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = e4m3_f32(uint8_t((i < 4 ? w.x : w.y) >> (8 * (i & 3))));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if constexpr (sizeof(T) == 1) v[i] = e4m3_f32(p[i]);
            else v[i] = to_f32(p[i]);
        }
    }
    if constexpr (sizeof(T) == 1)
        if (a.scaled == SCALE_BLOCK) {
            const float s = e8m0_f32(static_cast<const uint8_t*>(a.x_scales)[token * (a.cols / 32) + k / 32]);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] *= s;
        }
}

__device__ __forceinline__ float power_of_two(int e) {  // 2^e for -149 <= e <= 127
    return __uint_as_float(e >= -126 ? uint32_t(e + 127) << 23 : e >= -149 ? 1u << (e + 149) : 0u);
}
// v 2^e, exactly where the result is a number of fp32's; |e| up to 250.
__device__ __forceinline__ float times_power(float v, int e) { return v * power_of_two(e / 2) * power_of_two(e - e / 2); }

__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    uint32_t u;
    memcpy(&u, &h, 4);
    return u;
}

// Four bytes of nibbles -> four words of two fp16, the low nibble in the low half.
__device__ __forceinline__ void nibbles_to_half(uint32_t w, uint32_t (&h)[4]) {
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\tmov.b32 {b0, b1, b2, b3}, %4;\n\tcvt.rn.f16x2.e2m1x2 %0, b0;\n\tcvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, b2;\n\tcvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(w));
}
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t half2_mul(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

__device__ __forceinline__ void store_as(void* y, uint32_t dtype, uint64_t i, float v) {
    if (dtype == DT_BF16) static_cast<__nv_bfloat16*>(y)[i] = __float2bfloat16_rn(v);
    else if (dtype == DT_FP16) static_cast<__half*>(y)[i] = __float2half_rn(v);
    else static_cast<float*>(y)[i] = v;
}

// NT: groups of eight tokens.  MX: E8M0 scales per 32 columns, else E4M3 per 16.
template <class T, int NT, bool MX>
__global__ void __launch_bounds__(256) matvec_few_kernel(const __grid_constant__ CUtensorMap values, const __grid_constant__ CUtensorMap scales, const FewArgs a) {
    namespace cg = cooperative_groups;
    extern __shared__ uint8_t dynamic[];
    uint8_t* base = dynamic + (1024 - (smem_u32(dynamic) & 1023)) % 1024;
    // head: barriers of every warp and box, largest magnitude, flags
    uint32_t* const most = reinterpret_cast<uint32_t*>(base + 960);
    volatile uint32_t* const failed = reinterpret_cast<uint32_t*>(base + 964);
    uint8_t* const ring = base + 1024;
    uint8_t* const xs = ring + FEW_WARPS * a.depth * (BOX_BYTES + BOX_SCALES);
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x & 31, g = lane / 4, t = lane & 3;
    const cg::cluster_group cluster = cg::this_cluster();
    const uint32_t ranks = cluster.num_blocks(), rank = cluster.block_rank();

    // this block's boxes, and this warp's among them
    const uint32_t tiles = FEW_WARPS / a.wk, part = warp % a.wk;
    const uint32_t block_lo = uint32_t(uint64_t(a.boxes) * rank / ranks), block_hi = uint32_t(uint64_t(a.boxes) * (rank + 1) / ranks), block_n = block_hi - block_lo;
    const uint32_t lo = block_lo + block_n * part / a.wk, n = block_lo + block_n * (part + 1) / a.wk - lo;
    const uint32_t row0 = (blockIdx.x / ranks * tiles + warp / a.wk) * 16;
    const uint32_t mine = row0 < a.rows ? n : 0;

    const uint32_t bars = smem_u32(base) + warp * a.depth * 8;
    const uint32_t boxes_at = smem_u32(ring) + warp * a.depth * BOX_BYTES, scales_at = smem_u32(ring) + FEW_WARPS * a.depth * BOX_BYTES + warp * a.depth * BOX_SCALES;
    if (threadIdx.x == 0) { *most = 0; *failed = 0; }
    if (lane == 0) {
        for (uint32_t i = 0; i < a.depth; ++i) mbar_init(bars + 8 * i, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async_shared();
    }
    __syncwarp();
    // box i of this warp (counted through all passes)
    auto load = [&](uint32_t i) {
        const uint32_t slot = i % a.depth, box = lo + i % n;
        mbar_expect(bars + 8 * slot, BOX_BYTES + BOX_SCALES);
        tma_load(boxes_at + slot * BOX_BYTES, &values, bars + 8 * slot, int32_t(box * (BOX_COLS / 2)), int32_t(row0));
        // 16 bytes of scales: these 256 columns' (NVFP4), or theirs and a neighbour's (MXFP4, eight of them)
        tma_load(scales_at + slot * BOX_SCALES, &scales, bars + 8 * slot, int32_t(MX ? box / 2 * 16 : box * 16), int32_t(row0));
    };
    uint32_t issued = 0;
    if (lane == 0)
        for (; issued < mine && issued < a.depth; ++issued) load(issued);
    __syncthreads();

    // the largest finite magnitude of the block's share of the tokens
    const uint32_t pieces = a.tokens * block_n;  // of 256 values: one for a warp at a time
    {
        uint32_t m = 0;
        for (uint32_t i = warp; i < pieces; i += FEW_WARPS) {
            const uint64_t k = uint64_t(block_lo + i % block_n) * BOX_COLS + lane * 8;
            if (k < a.cols) {
                float v[8];
                load8<T>(a, i / block_n, k, v);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const uint32_t b = __float_as_uint(v[j]) & 0x7FFFFFFFu;
                    if (b < 0x7F800000u) m = max(m, b);
                }
            }
        }
        m = __reduce_max_sync(0xFFFFFFFFu, m);
        if (lane == 0 && m) atomicMax(most, m);
    }
    __syncthreads();
    const int shift = min(126, 141 - int(*most >> 23)), finer = sizeof(T) == 4 ? 12 : 39;

    float total[NT][4] = {};
    bool more = true;
    for (uint32_t pass = 0; more; ++pass) {
        // part `pass` of the tokens to shared memory
        const int up = shift + finer * int(pass);
        bool left = false;
        for (uint32_t i = warp; i < pieces; i += FEW_WARPS) {
            const uint32_t token = i / block_n, at = i % block_n * BOX_COLS + lane * 8;
            const uint64_t k = uint64_t(block_lo) * BOX_COLS + at;
            float v[8] = {};
            if (k < a.cols) load8<T>(a, token, k, v);
            uint32_t h[4];
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                float part_of[2];
#pragma unroll
                for (int i2 = 0; i2 < 2; ++i2) {
                    const float x = v[j + i2];
                    if ((__float_as_uint(x) & 0x7F800000u) == 0x7F800000u) { part_of[i2] = pass ? 0.0f : x; continue; }
                    float rest = x;
                    for (uint32_t p = 0; p < pass; ++p) {
                        const int e = shift + finer * int(p);
                        rest -= times_power(__half2float(__float2half_rn(times_power(rest, e))), -e);
                    }
                    part_of[i2] = times_power(rest, up);
                    rest -= times_power(__half2float(__float2half_rn(part_of[i2])), -up);
                    left |= fabsf(rest) > 0x1p-23f * fabsf(x);
                }
                h[j / 2] = pack_half(part_of[0], part_of[1]);
            }
            *reinterpret_cast<uint4*>(xs + token * a.pitch + at * 2) = make_uint4(h[0], h[1], h[2], h[3]);
        }
        more = __syncthreads_or(left) != 0 && pass < 9;
        const float down = power_of_two(-up);
        float sum[NT][4] = {};
        for (uint32_t i = 0; i < mine; ++i) {
            const uint32_t all = pass * n + i, slot = all % a.depth;
            mbar_wait(bars + 8 * slot, all / a.depth & 1, failed);
            const uint8_t* box = ring + (warp * a.depth + slot) * BOX_BYTES;
            const uint8_t* sc = ring + FEW_WARPS * a.depth * BOX_BYTES + (warp * a.depth + slot) * BOX_SCALES;
            uint32_t s0[4], s1[4];  // scales of rows g and g + 8
            if (MX) {
                const uint32_t half = ((lo + i) & 1) * 8;
                const uint2 p = *reinterpret_cast<const uint2*>(sc + g * 16 + half), q = *reinterpret_cast<const uint2*>(sc + (g + 8) * 16 + half);
                s0[0] = p.x; s0[1] = p.y; s1[0] = q.x; s1[1] = q.y;
            } else {
                const uint4 p = *reinterpret_cast<const uint4*>(sc + g * 16), q = *reinterpret_cast<const uint4*>(sc + (g + 8) * 16);
                s0[0] = p.x; s0[1] = p.y; s0[2] = p.z; s0[3] = p.w; s1[0] = q.x; s1[1] = q.y; s1[2] = q.z; s1[3] = q.w;
            }
            const uint8_t* xp = xs + g * a.pitch + (lo + i - block_lo) * (BOX_COLS * 2) + t * 16;
#pragma unroll
            for (int c = 0; c < 8; ++c) {  // 32 columns: 16 bytes of a row, four to a lane; TMA has swizzled the 16-byte pieces
                const uint32_t at = (uint32_t(c) ^ g) * 16 + t * 4;
                const uint32_t w0 = *reinterpret_cast<const uint32_t*>(box + g * 128 + at), w1 = *reinterpret_cast<const uint32_t*>(box + (g + 8) * 128 + at);
                uint32_t h0[4], h1[4];
                nibbles_to_half(w0, h0);
                nibbles_to_half(w1, h1);
                float f0 = 0, f1 = 0;
                if (MX) {
                    uint32_t pair;
                    asm("{\n\t.reg .b16 e;\n\tcvt.u16.u32 e, %1;\n\tcvt.rn.bf16x2.ue8m0x2 %0, e;\n\t}" : "=r"(pair) : "r"(__byte_perm(s0[c / 4], s1[c / 4], (c & 3) | (4 + (c & 3)) << 4)));
                    f0 = __uint_as_float(pair << 16) * down;
                    f1 = __uint_as_float(pair & 0xFFFF0000u) * down;
                    if (down > 1.0f) {  // an overflow is for the sums to have, not for a group of zeros
                        if (f0 > 3.4028235e38f) f0 = 3.4028235e38f;
                        if (f1 > 3.4028235e38f) f1 = 3.4028235e38f;
                    }
                } else {
                    const uint32_t b = (c & 1) * 2 + t / 2;  // lanes 0 and 1 hold the first group of 16 columns, 2 and 3 the second
                    uint32_t pair;
                    asm("{\n\t.reg .b16 e;\n\tcvt.u16.u32 e, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, e;\n\t}" : "=r"(pair) : "r"(__byte_perm(s0[c / 2], s1[c / 2], b | (4 + b) << 4)));
                    const uint32_t p0 = __byte_perm(pair, 0, 0x1010), p1 = __byte_perm(pair, 0, 0x3232);
#pragma unroll
                    for (int j = 0; j < 4; ++j) { h0[j] = half2_mul(h0[j], p0); h1[j] = half2_mul(h1[j], p1); }
                }
#pragma unroll
                for (int m = 0; m < NT; ++m) {
                    uint4 b = make_uint4(0, 0, 0, 0);
                    if (m * 8 + g < a.tokens) b = *reinterpret_cast<const uint4*>(xp + m * 8 * a.pitch + c * 64);
                    if (MX) {
                        float d[4] = {};
                        mma16816(d, h0[0], h1[0], h0[1], h1[1], b.x, b.y);
                        mma16816(d, h0[2], h1[2], h0[3], h1[3], b.z, b.w);
                        total[m][0] += d[0] * f0;
                        total[m][1] += d[1] * f0;
                        total[m][2] += d[2] * f1;
                        total[m][3] += d[3] * f1;
                    } else {
                        mma16816(sum[m], h0[0], h1[0], h0[1], h1[1], b.x, b.y);
                        mma16816(sum[m], h0[2], h1[2], h0[3], h1[3], b.z, b.w);
                    }
                }
            }
            __syncwarp();
            if (lane == 0 && !*failed)
                for (const uint32_t until = (pass + (more ? 2 : 1)) * n; issued < until && issued <= all + a.depth; ++issued) load(issued);
        }
        if (!MX)
#pragma unroll
            for (int m = 0; m < NT; ++m)
#pragma unroll
                for (int j = 0; j < 4; ++j) total[m][j] += sum[m][j] * down;
        if (more) __syncthreads();  // before the next part overwrites this one
    }
    if (*failed && lane == 0) let_copies_land();

    // shares of the warps, [row tile][share][token][row], then of the blocks
    __syncthreads();
    float* const shares = reinterpret_cast<float*>(ring);
    constexpr uint32_t PER = NT * 8 * 16;
#pragma unroll
    for (int m = 0; m < NT; ++m)
#pragma unroll
        for (int j = 0; j < 4; ++j) shares[warp * PER + (m * 8 + 2 * t + (j & 1)) * 16 + g + (j >> 1) * 8] = total[m][j];
    __syncthreads();
    float* const sums = shares + FEW_WARPS * PER;
    const uint32_t outs = tiles * PER;
    auto finish = [&](uint32_t e, float v) {
        const uint32_t tile = e / PER, token = e % PER / 16;
        const uint64_t row = uint64_t(blockIdx.x / ranks * tiles + tile) * 16 + e % 16;
        if (token >= a.tokens || row >= a.rows) return;
        if (a.global_scale) v *= *a.global_scale;
        if (a.scaled == SCALE_ROW) v *= static_cast<const float*>(a.x_scales)[token];
        store_as(a.y, a.y_dtype, token * a.rows + row, *failed ? __uint_as_float(0x7FC00000u) : v);
    };
    for (uint32_t e = threadIdx.x; e < outs; e += 256) {
        float v = 0;
        for (uint32_t p = 0; p < a.wk; ++p) v += shares[(e / PER * a.wk + p) * PER + e % PER];
        if (ranks == 1) finish(e, v);
        else sums[e] = v;
    }
    if (ranks > 1) {
        cluster.sync();
        for (uint32_t e = rank * 256 + threadIdx.x; e < outs; e += ranks * 256) {
            float v = 0;
            for (uint32_t r = 0; r < ranks; ++r) v += *cluster.map_shared_rank(sums + e, r);
            finish(e, v);
        }
        cluster.sync();  // nobody leaves while others read its sums
    }
    if (threadIdx.x == 0 && *failed) atomicExch(a.status, 1u);
}

}  // namespace ptwm
