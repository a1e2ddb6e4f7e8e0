// Products of a 4-bit matrix with up to 16 tokens.
//
// What bounds them is reading the matrix, so it goes through the SMs once, in boxes of 16 rows x 256 columns that every warp
// asks TMA for by itself, some ahead, without a barrier between warps; the scales of all of a block's rows come at once.  A warp turns a box into the first operand of
// mma.m16n8k16 (16 rows of the matrix, 8 tokens): tcgen05 would want it written back to shared memory, or to tensor memory, in
// tiles of 128 rows first, for products that fill a sixteenth of its width.
//   Operands are fp16.  An E2M1 number fits it; so does its product with an E4M3 scale (six significant bits, 2^-10 to 2688), which
// NVFP4 takes before the MMA.  E8M0 scales range further: MXFP4 multiplies the sums of each group with them, in fp32.
//   Tokens become fp16 by a power of two that takes the largest of the block's share of them to [2^14, 2^15).  That is exact for bf16
// values down to 2^-31 of it (fp16 2^-28, E4M3 2^-35).  Where the smallest is below, or tokens are fp32, what is left over goes through
// the same products again as another part on a finer scale: one pass for nearly all bf16 tokens, two for fp32, and always as many
// as bring the parts within 2^-23 of every value.  A pass goes over the matrix again: one token of 4096 x 14336 takes 12.5 us, 21.6 where one of its
// values is 2^-50.
//   MMAs cut what an fp32 sum does not hold.  Sums of fp32 tokens are therefore added up, rounded, after each group (MXFP4) or box (NVFP4): one token of
// 4096 x 14336 is within 2e-7 of its sum (in one piece 1.4e-6, and no faster).
//   A block per SM keeps its tokens in shared memory and has a run of row tiles.  Of up to 16 of them at a turn, its 16 warps take equal
// runs of boxes, so a warp works on one tile or two and ends each with its share of the sums; tokens that do not fit are split
// over the blocks of a cluster.  Shares are added in the order of the columns.
//   One token of 14336 x 4096 takes 10.2 us in MXFP4 and 10.5 in NVFP4 (the matrix alone 4.8 and 5.1), eight 12.3; one of 131072 x 4096 58 us,
// 4.9 to 5.2 TB/s.  A launch and its first trip to memory are some 4 us of it.
#pragma once
#include <cooperative_groups.h>

#include <type_traits>

#include "matvec.cuh"
#include "tensor_core.cuh"

namespace ptwm {

constexpr uint32_t FEW_TOKENS = 16;
constexpr uint32_t BOX_COLS = 256, BOX_BYTES = 16 * BOX_COLS / 2, FEW_WARPS = 16, FEW_DEPTH = 5, FEW_HEAD = 1024;  // FEW_DEPTH: boxes under way per warp, at most

// Up to so many matrices that read the same tokens, as one: their row tiles one after the other.
constexpr uint32_t FEW_MATRICES = 4;
struct FewMatrix {
    const float* global_scale;
    void* y;
    uint32_t rows, first;   // and the number of row tiles before its own
};
struct FewMaps { CUtensorMap values[FEW_MATRICES], scales[FEW_MATRICES]; };
struct FewArgs {
    const void* x;
    const void* x_scales;
    FewMatrix m[FEW_MATRICES];
    uint32_t* status;
    uint64_t cols;
    uint32_t count, tokens, scaled, y_dtype;
    uint32_t rank_boxes, rank_more;         // boxes of 256 columns to a block of a cluster, and how many blocks have one more
    uint32_t cluster_tiles, cluster_more;   // the same of row tiles to a cluster
    uint32_t turns;
    uint32_t depth;      // boxes under way per warp
    uint32_t pitch;      // bytes of a token's values in shared memory
    uint32_t most;       // row tiles of a turn
    uint32_t lines;      // 128-byte lines of scales to a row
    uint32_t wide;       // tokens can be read 8 values at a time
};

inline uint32_t few_pitch(uint32_t boxes) { return boxes * BOX_COLS * 2 + 64; }  // neighbours in different banks
// 128-byte lines of scales that a block with so many boxes has to a row, from the 16-byte piece on in which they begin.
inline uint32_t few_lines(uint32_t boxes, uint32_t group) { return (boxes * (BOX_COLS / group) + (group == 32 ? 8 : 0) + 127) / 128; }
// most: row tiles a block has at a turn.
inline uint64_t few_smem(uint32_t tokens, uint32_t boxes, uint32_t depth, uint32_t parts, uint32_t ranks, uint32_t most, uint32_t lines) {  // 64 bits: boxes are any matrix'
    const uint64_t shares = (2 * FEW_WARPS + (ranks > 1 ? most : 0)) * tokens * 64;
    return 1024 + FEW_HEAD + FEW_WARPS * depth * BOX_BYTES + uint64_t(most * 16) * lines * 128 + shares + uint64_t(parts * tokens) * few_pitch(boxes);
}

// Eight values of a token, as they lie.
template <class T> struct Eight { uint32_t w[sizeof(T) * 2]; };
template <class T> __device__ __forceinline__ Eight<T> load8(const FewArgs& a, uint64_t token, uint64_t k) {
    const T* p = static_cast<const T*>(a.x) + token * a.cols + k;
    Eight<T> e;
    if (a.wide) {
        if constexpr (sizeof(T) == 1) {
            const uint2 v = *reinterpret_cast<const uint2*>(p);
            e.w[0] = v.x; e.w[1] = v.y;
        } else {
#pragma unroll
            for (int i = 0; i < int(sizeof(T)) * 2; i += 4) {
                const uint4 v = reinterpret_cast<const uint4*>(p)[i / 4];
                e.w[i] = v.x; e.w[i + 1] = v.y; e.w[i + 2] = v.z; e.w[i + 3] = v.w;
            }
        }
    } else {
        T v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = p[i];
        memcpy(&e, v, sizeof e);
    }
    return e;
}
__device__ __forceinline__ uint32_t e4m3x2_half2(uint32_t two) {
    uint32_t h;
    asm("{\n\t.reg .b16 e;\n\tcvt.u16.u32 e, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, e;\n\t}" : "=r"(h) : "r"(two));
    return h;
}
__device__ __forceinline__ float2 half2_floats(uint32_t u) {
    __half2 h;
    memcpy(&h, &u, 4);
    return __half22float2(h);
}
// Scale of the block of 32 that holds value k of a token (E4M3 with block scales), else 1.
template <class T> __device__ __forceinline__ float block_of(const FewArgs& a, uint64_t token, uint64_t k) {
    if (sizeof(T) == 1 && a.scaled == SCALE_BLOCK) return e8m0_f32(static_cast<const uint8_t*>(a.x_scales)[token * (a.cols / 32) + k / 32]);
    return 1.0f;
}
template <class T> __device__ __forceinline__ void unpack8(const Eight<T>& e, float s, float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(e.w[i]);
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(e.w[i] << 16); v[2 * i + 1] = __uint_as_float(e.w[i] & 0xFFFF0000u); }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = half2_floats(sizeof(T) == 1 ? e4m3x2_half2(e.w[i / 2] >> (16 * (i & 1))) : e.w[i % (sizeof(T) * 2)]);
            v[2 * i] = f.x * s; v[2 * i + 1] = f.y * s;
        }
    }
}

__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) { uint32_t r; asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; }
__device__ __forceinline__ uint32_t min_u16x2(uint32_t a, uint32_t b) { uint32_t r; asm("min.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; }
__device__ __forceinline__ uint32_t less_one_u16x2(uint32_t a) { uint32_t r; asm("add.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(0xFFFFFFFFu)); return r; }

// Largest finite magnitude and smallest one that is not zero, as bits of fp32; 0 and 0xFFFFFFFF where there is none.
struct Extremes { uint32_t most = 0, least = 0xFFFFFFFFu; };
__device__ __forceinline__ void extremes_of(float v, Extremes& x) {
    const uint32_t b = __float_as_uint(v) & 0x7FFFFFFFu;
    if (b && b < 0x7F800000u) { x.most = max(x.most, b); x.least = min(x.least, b); }
}
template <class T> __device__ __forceinline__ void extremes8(const Eight<T>& e, float s, Extremes& x) {
    if constexpr (sizeof(T) == 2) {  // magnitudes compare as numbers: two at a time, and zero minus one is the largest
        uint32_t hi = 0, lo = 0xFFFFFFFFu;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t m = e.w[i] & 0x7FFF7FFFu;
            hi = max_u16x2(hi, m);
            lo = min_u16x2(lo, less_one_u16x2(m));
        }
        constexpr uint32_t INF = std::is_same<T, __half>::value ? 0x7C00 : 0x7F80;
        const uint32_t h = max(hi & 0xFFFF, hi >> 16), l = min(lo & 0xFFFF, lo >> 16) + 1;
        if (h < INF) {
            auto bits = [](uint32_t u) -> uint32_t {
                if (std::is_same<T, __nv_bfloat16>::value) return u << 16;
                return __float_as_uint(half2_floats(u).x);
            };
            x.most = max(x.most, bits(h));
            if (l <= 0xFFFF) x.least = min(x.least, bits(l));
            return;
        }
    }
    float v[8];
    unpack8<T>(e, s, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) extremes_of(v[i], x);
}

__device__ __forceinline__ float power_of_two(int e) {  // 2^e for -149 <= e <= 127, 0 below
    return __uint_as_float(e >= -126 ? uint32_t(e + 127) << 23 : e >= -149 ? 1u << (e + 149) : 0u);
}
// What a part leaves of a value that was scaled for it, scaled for the next part: eleven bits are taken.
__device__ __forceinline__ float after_part(float v, float finer) {
    return (__float_as_uint(v) & 0x7F800000u) == 0x7F800000u ? 0.0f : (v - __half2float(__float2half_rn(v))) * finer;
}

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

__device__ __forceinline__ void mma16816_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}

__device__ __forceinline__ uint32_t lds32(uint32_t at) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(at));
    return v;
}
__device__ __forceinline__ uint4 lds128(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
    return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t at) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at));
    return v;
}

__device__ __forceinline__ uint32_t lds16(uint32_t at) {
    uint16_t v;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(at));
    return v;
}
__device__ __forceinline__ uint32_t lds8(uint32_t at) {
    uint32_t v;
    asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(at));
    return v;
}
// Where a == b; v stays as it is elsewhere.
__device__ __forceinline__ void lds128_where(uint4& v, uint32_t at, uint32_t a, uint32_t b) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.eq.u32 p, %5, %6;\n\t@p ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];\n\t}" : "+r"(v.x), "+r"(v.y), "+r"(v.z), "+r"(v.w) : "r"(at), "r"(a), "r"(b));
}
// Two scales, the first in the lower byte.
template <bool MX> __device__ __forceinline__ float2 scale_pair(uint32_t two) {
    if (!MX) return half2_floats(e4m3x2_half2(two));
    uint32_t pair;
    asm("{\n\t.reg .b16 e;\n\tcvt.u16.u32 e, %1;\n\tcvt.rn.bf16x2.ue8m0x2 %0, e;\n\t}" : "=r"(pair) : "r"(two));
    return make_float2(__uint_as_float(pair << 16), __uint_as_float(pair & 0xFFFF0000u));
}

// TOKENS: at most so many, 1, 2, 8 or 16.  MX: E8M0 scales per 32 columns, else E4M3 per 16.
//   With one token or two the eight columns of an MMA are 8 / TOKENS groups of the matrix for each: a lane has the tokens' values only where
// the group is its column's, and zeros elsewhere (E2M1 has no infinities to multiply them with).  So one MMA after the other adds to the
// same sums, and their scales are wanted once for eight groups or four: 185 instructions to a box with one token, 280 with eight.
template <class T, int TOKENS, bool MX>
__global__ void __launch_bounds__(FEW_WARPS * 32, 1) matvec_few_kernel(const __grid_constant__ FewMaps maps, const __grid_constant__ FewArgs a) {
    namespace cg = cooperative_groups;
    constexpr int PARTS = sizeof(T) == 4 ? 2 : 1;       // kept side by side
    constexpr int NT = TOKENS > 8 ? 2 : 1, P = TOKENS < 8 ? TOKENS : 8;
    constexpr bool SPREAD = P < 8;
    static_assert(!SPREAD || PARTS == 1, "values in one part only are spread");
    constexpr int GROUPS = 8 / P, PERIOD = SPREAD ? (MX ? GROUPS : GROUPS / 2) : 1;  // groups side by side, and the chunks of 32 columns that have them
    constexpr int FINER = sizeof(T) == 4 ? 12 : 39;     // powers of two from one part to the next
    // from which power on, after scaling, values of the type are exact in the parts of a pass (fp32: to 2^-23)
    constexpr int FLOOR = sizeof(T) == 4 || std::is_same<T, __half>::value ? -14 : sizeof(T) == 1 ? -21 : -17;
    extern __shared__ uint8_t dynamic[];
    uint8_t* base = dynamic + (1024 - (smem_u32(dynamic) & 1023)) % 1024;
    // head: barriers of every warp and box and of the scales, extremes of every warp, flag
    static_assert(FEW_WARPS * FEW_DEPTH * 8 <= 768 && 776 + 2 * FEW_WARPS * 4 <= 960, "the head of shared memory does not overlap");
    const uint32_t scales_bar = smem_u32(base) + 768;
    uint32_t* const extremes = reinterpret_cast<uint32_t*>(base + 776);
    volatile uint32_t* const failed = reinterpret_cast<uint32_t*>(base + 960);
    uint8_t* const ring = base + FEW_HEAD;
    const uint32_t line_bytes = a.most * 16 * 128;      // a line of every row of a turn
    uint8_t* const scale_lines = ring + FEW_WARPS * a.depth * BOX_BYTES;
    float* const shares = reinterpret_cast<float*>(scale_lines + a.lines * line_bytes);
    const uint32_t per = a.tokens * 16;                 // results of a row tile
    float* const sums = shares + 2 * FEW_WARPS * per;
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x & 31, g = lane / 4, t = lane & 3;
    const cg::cluster_group cluster = cg::this_cluster();
    const uint32_t ranks = cluster.num_blocks(), rank = cluster.block_rank();
    uint8_t* const xs = reinterpret_cast<uint8_t*>(sums + (ranks > 1 ? a.most * per : 0));

    // this block's columns (boxes block_lo, + block_n) and row tiles (tile_lo, + tile_n), up to a.most of them at a turn
    const uint32_t block_lo = rank * a.rank_boxes + min(rank, a.rank_more), block_n = a.rank_boxes + (rank < a.rank_more);
    const uint32_t cluster_at = blockIdx.x >> (31 - __clz(ranks));
    const uint32_t tile_lo = cluster_at * a.cluster_tiles + min(cluster_at, a.cluster_more), tile_n = a.cluster_tiles + (cluster_at < a.cluster_more);
    const uint32_t turns = a.turns;
    // i / block_n of what fits shared memory (a few thousand boxes): exact, the half keeps it off the borders
    const float per_n = __frcp_rn(float(block_n));
    auto over_n = [&](uint32_t i) { return uint32_t((float(i) + 0.5f) * per_n); };
    // a turn's boxes in the order of tiles and columns; a warp has an equal run of them, at most as many as a tile has
    struct Run { uint32_t tile, lo, hi; };
    auto run_of = [&](uint32_t turn, uint32_t w) {
        const uint32_t first = turn * a.most, all = (first < tile_n ? min(tile_n - first, a.most) : 0) * block_n;
        return Run{tile_lo + first, all * w / FEW_WARPS, all * (w + 1) / FEW_WARPS};
    };

    const uint32_t bars = smem_u32(base) + warp * a.depth * 8;
    const uint32_t boxes_at = smem_u32(ring) + warp * a.depth * BOX_BYTES;
    // scales of a turn's rows, 16-byte pieces swizzled as those of the boxes
    const uint32_t scale_first = (MX ? block_lo / 2 : block_lo) * 16;
    auto matrix_at = [&](uint32_t tile) {
        uint32_t m = 0;
        while (m + 1 < a.count && tile >= a.m[m + 1].first) ++m;
        return m;
    };
    auto load_scales = [&](uint32_t turn) {
        // a box of all rows of the turn, or where they may be of several matrices one for each tile
        const uint32_t first = tile_lo + turn * a.most, n = a.count == 1 ? 1 : min(tile_n - turn * a.most, a.most);
        mbar_expect(scales_bar, a.lines * (a.count == 1 ? line_bytes : n * 2048));
        for (uint32_t q = 0; q < n; ++q) {
            const uint32_t m = matrix_at(first + q);
            for (uint32_t i = 0; i < a.lines; ++i)
                tma_load(smem_u32(scale_lines) + i * line_bytes + q * 2048, &maps.scales[m], scales_bar, int32_t(scale_first + i * 128), int32_t((first + q - a.m[m].first) * 16));
        }
    };
    // what lane 0 asks for next: ask_left boxes of the run, from column box ask_col of row tile ask_tile on, which is at ask_row of its matrix
    uint32_t ask_left, ask_col, ask_tile, ask_m, ask_row, ask_slot = 0, ask_pass = 0, ask_turn = 0;
    auto ask = [&](const Run& r) {
        const uint32_t q = over_n(r.lo);
        ask_left = r.hi - r.lo;
        ask_col = r.lo - q * block_n;
        ask_tile = r.tile + q;
        ask_m = matrix_at(ask_tile);
        ask_row = (ask_tile - a.m[ask_m].first) * 16;
    };
    ask(run_of(0, warp));
    auto load = [&] {
        const uint32_t bar = bars + 8 * ask_slot;
        mbar_expect(bar, BOX_BYTES);
        tma_load(boxes_at + ask_slot * BOX_BYTES, &maps.values[ask_m], bar, int32_t((block_lo + ask_col) * (BOX_COLS / 2)), int32_t(ask_row));
        if (++ask_slot == a.depth) ask_slot = 0;
        if (++ask_col == block_n) {
            ask_col = 0;
            ask_row += 16;
            if (ask_m + 1 < a.count && ++ask_tile == a.m[ask_m + 1].first) { ++ask_m; ask_row = 0; }
        }
        --ask_left;
    };
    // to the next pass or turn where a run has been asked for; false behind the last
    auto goes_on = [&](uint32_t passes) {
        while (!ask_left) {
            if (++ask_pass >= passes) {
                ask_pass = 0;
                if (++ask_turn >= turns) { ask_turn = turns; return false; }
            }
            ask(run_of(ask_turn, warp));
        }
        return true;
    };
    // HOLD pieces of 256 values of the tokens to a warp at a time; those of a block with few stay in registers.
    constexpr int HOLD = sizeof(T) == 4 ? 4 : 8;
    const uint32_t pieces = a.tokens * block_n;
    Eight<T> held[HOLD];
    auto fetch = [&](uint32_t from) {
#pragma unroll
        for (int j = 0; j < HOLD; ++j) {
            const uint32_t i = from + j * FEW_WARPS;
            held[j] = Eight<T>{};
            if (i >= pieces) continue;
            const uint32_t token = over_n(i);
            const uint64_t k = uint64_t(block_lo + i - token * block_n) * BOX_COLS + lane * 8;
            if (k < a.cols) held[j] = load8<T>(a, token, k);
        }
    };
    if (lane == 0) {
        for (uint32_t i = 0; i < a.depth; ++i) mbar_init(bars + 8 * i, 1);
        if (warp == 0) { *failed = 0; mbar_init(scales_bar, 1); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async_shared();
    }
    __syncwarp();
    others_may_start();
    after_those_before();
    fetch(warp);
    // Until the passes are known only the first one of the first turn is asked for, and before the tokens are staged two boxes of it: what a warp's
    // requests wait for one another (24 cycles each, sixteen warps) the tokens would wait for too.
    uint32_t under_way = 0;
    if (lane == 0) {
        if (warp == 0) load_scales(0);
        for (; under_way < 2 && ask_left; ++under_way) load();
    }
    __syncwarp();

    // the largest and the smallest magnitude of the block's share of the tokens
    uint32_t largest, smallest;
    {
        Extremes x;
        for (uint32_t from = warp; from < pieces; from += FEW_WARPS * HOLD) {
            if (from != warp) fetch(from);
#pragma unroll
            for (int j = 0; j < HOLD; ++j) {
                const uint32_t i = from + j * FEW_WARPS;
                if (i >= pieces) break;
                if (sizeof(T) == 1) {
                    const uint32_t token = over_n(i);
                    const uint64_t k = uint64_t(block_lo + i - token * block_n) * BOX_COLS + lane * 8;
                    if (k < a.cols) extremes8<T>(held[j], block_of<T>(a, token, k), x);
                } else {
                    extremes8<T>(held[j], 1.0f, x);  // what is behind the columns is zeros
                }
            }
        }
        x.most = __reduce_max_sync(0xFFFFFFFFu, x.most);
        x.least = __reduce_min_sync(0xFFFFFFFFu, x.least);
        if (lane == 0) { extremes[warp] = x.most; extremes[FEW_WARPS + warp] = x.least; }
        __syncthreads();
        const uint32_t v = extremes[lane];
        largest = __reduce_max_sync(0xFFFFFFFFu, lane < FEW_WARPS ? v : 0);
        smallest = __reduce_min_sync(0xFFFFFFFFu, lane < FEW_WARPS ? 0xFFFFFFFFu : v);
    }
    // 2^up takes the largest to [2^14, 2^15); a part has the bits down to 2^-24
    const int up0 = min(126, 141 - int(largest >> 23));
    const int bottom = largest ? max(int(smallest >> 23), 1) - 127 + up0 - (smallest >> 23 ? 0 : 23) : 0;
    const uint32_t passes = 1 + (bottom < FLOOR ? uint32_t(FLOOR - bottom + FINER * PARTS - 1) / (FINER * PARTS) : 0);

    const uint32_t part_bytes = a.tokens * a.pitch;
    auto stage = [&](uint32_t pass) {  // the parts of a pass of the tokens to shared memory
        const float first = power_of_two(up0);
        constexpr float FINE = float(1ull << FINER);
        for (uint32_t from = warp; from < pieces; from += FEW_WARPS * HOLD) {
            if (pieces > FEW_WARPS * HOLD || pass) fetch(from);
#pragma unroll
            for (int h = 0; h < HOLD; ++h) {
                const uint32_t i = from + h * FEW_WARPS, token = over_n(i), at = (i - token * block_n) * BOX_COLS + lane * 8;
                if (i >= pieces) break;
                const uint64_t k = uint64_t(block_lo) * BOX_COLS + at;
                float v[8];
                unpack8<T>(held[h], k < a.cols ? block_of<T>(a, token, k) : 1.0f, v);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] *= first;
                for (uint32_t p = 0; p < pass * PARTS; ++p)
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] = after_part(v[j], FINE);
#pragma unroll
                for (int p = 0; p < PARTS; ++p) {
                    uint32_t w[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) w[j] = pack_half(v[2 * j], v[2 * j + 1]);
                    *reinterpret_cast<uint4*>(xs + p * part_bytes + token * a.pitch + at * 2) = make_uint4(w[0], w[1], w[2], w[3]);
                    if (p + 1 < PARTS)
#pragma unroll
                        for (int j = 0; j < 8; ++j) v[j] = after_part(v[j], FINE);
                }
            }
        }
        __syncthreads();
    };
    if (passes == 1) stage(0);
    if (lane == 0)
        for (; under_way < a.depth && goes_on(passes); ++under_way) load();

    uint32_t tokens_at[NT];
#pragma unroll
    for (int m = 0; m < NT; ++m) tokens_at[m] = smem_u32(xs) + min(SPREAD ? g % P : m * 8 + g, a.tokens - 1) * a.pitch + t * 16;
    // spread: the chunk of a period whose values this lane has (NVFP4: lanes 0 and 1 of four hold a chunk's first group, 2 and 3 its second)
    const uint32_t mine = MX ? g / P : (g / P & 1) == t / 2 ? g / P / 2 : 99;
    uint4 spread[PERIOD];
#pragma unroll
    for (int c = 0; c < PERIOD; ++c) spread[c] = make_uint4(0, 0, 0, 0);
    uint32_t slot = 0, parity = 0;
    for (uint32_t turn = 0; turn < turns; ++turn) {
        const Run run = run_of(turn, warp);
        mbar_wait(scales_bar, turn & 1, failed);
        for (uint32_t pass = 0; pass < passes; ++pass) {
            if (passes > 1) {
                __syncthreads();  // before these parts take the place of the last
                stage(pass);
            }
            // What undoes the scaling: powers below one with the scales of a group, so that nothing overflows, the others at the end; so is what
            // of a power below one is no normal number, since a group's scale may bring the product back.
            const int up = up0 + FINER * PARTS * int(pass), with_scales = min(max(up, 0), 126);
            const float down = power_of_two(-with_scales), rest = power_of_two(with_scales - up);
            float sum[NT][4] = {};
            const uint32_t tile0 = over_n(run.lo);
            uint32_t col = run.lo - tile0 * block_n, scales_of = smem_u32(scale_lines) + (tile0 * 16 + g) * 128;
            // this warp's share of the tile that it has ended with: [token][row], in the first of its two places for its first tile
            float* my = shares + warp * 2 * per;
            auto hand_in = [&] {
                if constexpr (SPREAD) {  // a token's columns are those of its groups
                    if (P == 1) { sum[0][0] += sum[0][1]; sum[0][2] += sum[0][3]; }
#pragma unroll
                    for (int j = 0; j < 4; j += P == 1 ? 2 : 1)
#pragma unroll
                        for (int o = 1; o < 4; o *= 2) sum[0][j] += __shfl_xor_sync(0xFFFFFFFFu, sum[0][j], o);
                }
#pragma unroll
                for (int m = 0; m < NT; ++m)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        float v = sum[m][j];
                        v = (MX ? v : v * down) * rest;
                        const uint32_t token = m * 8 + 2 * t + (j & 1);
                        if (token < a.tokens && (!SPREAD || token < P)) {
                            float* const to = my + token * 16 + g + (j >> 1) * 8;
                            *to = pass ? *to + v : v;
                        }
                        sum[m][j] = 0;
                    }
                my += per;
            };
            for (uint32_t i = run.lo; i < run.hi; ++i) {
                mbar_wait(bars + 8 * slot, parity, failed);
                const uint32_t box = boxes_at + slot * BOX_BYTES + (g * 144 + t * 4);  // TMA has swizzled the 16-byte pieces of a line
                const uint32_t byte = MX ? (col + (block_lo & 1)) * 8 : col * 16;  // of a row's scales: 8 are the box's (MXFP4) or 16
                const uint32_t sc = scales_of + byte / 128 * line_bytes + ((byte / 16 ^ g) & 7) * 16 + byte % 16;
                if constexpr (SPREAD) {
                    const uint32_t xt = tokens_at[0] + col * (BOX_COLS * 2);
                    float d[4];
#pragma unroll
                    for (int c = 0; c < 8; ++c) {  // 32 columns: 16 bytes of a row, four to a lane
                        const uint32_t w = box ^ uint32_t(c << 4);
                        uint32_t h0[4], h1[4];
                        nibbles_to_half(lds32(w), h0);
                        nibbles_to_half(lds32(w + 1024), h1);
                        uint4& b = spread[c % PERIOD];
                        lds128_where(b, xt + c * 64, mine, uint32_t(c % PERIOD));
                        if (c % PERIOD == 0) mma16816_first(d, h0[0], h1[0], h0[1], h1[1], b.x, b.y);
                        else mma16816(d, h0[0], h1[0], h0[1], h1[1], b.x, b.y);
                        mma16816(d, h0[2], h1[2], h0[3], h1[3], b.z, b.w);  // (two chains of sums: no faster)
                        if (c % PERIOD == PERIOD - 1) {
                            // columns 2 t and 2 t + 1: two groups (P = 1), or one and both tokens
                            const uint32_t at = sc + c / PERIOD * GROUPS + (P == 1 ? 2 * t : t);
                            const uint32_t r0 = P == 1 ? lds16(at) : lds8(at), r1 = P == 1 ? lds16(at + 1024) : lds8(at + 1024);
                            const float2 f0 = scale_pair<MX>(r0), f1 = scale_pair<MX>(r1);
                            const float k = MX ? down : 1.0f;
                            sum[0][0] += d[0] * (f0.x * k);
                            sum[0][1] += d[1] * ((P == 1 ? f0.y : f0.x) * k);
                            sum[0][2] += d[2] * (f1.x * k);
                            sum[0][3] += d[3] * ((P == 1 ? f1.y : f1.x) * k);
                        }
                    }
                } else {
                uint32_t s0[4], s1[4];  // scales of rows g and g + 8
                if (MX) {
                    const uint2 p = lds64(sc), q = lds64(sc + 1024);
                    s0[0] = p.x; s0[1] = p.y; s1[0] = q.x; s1[1] = q.y;
                } else {
                    const uint4 p = lds128(sc), q = lds128(sc + 1024);
                    s0[0] = p.x; s0[1] = p.y; s0[2] = p.z; s0[3] = p.w; s1[0] = q.x; s1[1] = q.y; s1[2] = q.z; s1[3] = q.w;
                }
                uint32_t xt[NT];  // where there is no token, another's values make sums that nobody stores
#pragma unroll
                for (int m = 0; m < NT; ++m) xt[m] = tokens_at[m] + col * (BOX_COLS * 2);
                const uint32_t nib = t / 2;
                float of_box[PARTS][NT][4];  // of fp32 tokens against NVFP4: MMAs cut what a sum does not hold, so their sums are added up, rounded, after each box
#pragma unroll
                for (int c = 0; c < 8; ++c) {  // 32 columns: 16 bytes of a row, four to a lane
                    const uint32_t w = box ^ uint32_t(c << 4);
                    uint32_t h0[4], h1[4];
                    nibbles_to_half(lds32(w), h0);
                    nibbles_to_half(lds32(w + 1024), h1);
                    float f0 = 0, f1 = 0;
                    if (MX) {
                        const float2 f = scale_pair<MX>(__byte_perm(s0[c / 4], s1[c / 4], (c & 3) | (4 + (c & 3)) << 4));
                        f0 = f.x * down;
                        f1 = f.y * down;
                    } else {
                        const uint32_t b = (c & 1) * 2 + nib;  // lanes 0 and 1 hold the first group of 16 columns, 2 and 3 the second
                        const uint32_t pair = e4m3x2_half2(__byte_perm(s0[c / 2], s1[c / 2], b | (4 + b) << 4));
                        const uint32_t p0 = __byte_perm(pair, 0, 0x1010), p1 = __byte_perm(pair, 0, 0x3232);
#pragma unroll
                        for (int j = 0; j < 4; ++j) { h0[j] = half2_mul(h0[j], p0); h1[j] = half2_mul(h1[j], p1); }
                    }
#pragma unroll
                    for (int m = 0; m < NT; ++m) {
                        const uint4 b = lds128(xt[m] + c * 64);
                        uint4 b2;
                        if (PARTS == 2) b2 = lds128(xt[m] + part_bytes + c * 64);
                        if (MX) {
                            float d[4];
                            mma16816_first(d, h0[0], h1[0], h0[1], h1[1], b.x, b.y);
                            mma16816(d, h0[2], h1[2], h0[3], h1[3], b.z, b.w);
                            if (PARTS == 2) {
                                float e[4];
                                mma16816_first(e, h0[0], h1[0], h0[1], h1[1], b2.x, b2.y);
                                mma16816(e, h0[2], h1[2], h0[3], h1[3], b2.z, b2.w);
#pragma unroll
                                for (int j = 0; j < 4; ++j) d[j] += e[j] * (1.0f / float(1ull << FINER));
                            }
                            sum[m][0] += d[0] * f0;
                            sum[m][1] += d[1] * f0;
                            sum[m][2] += d[2] * f1;
                            sum[m][3] += d[3] * f1;
                        } else if constexpr (PARTS == 2) {
#pragma unroll
                            for (int p = 0; p < PARTS; ++p) {
                                const uint4& q = p ? b2 : b;
                                if (c == 0) mma16816_first(of_box[p][m], h0[0], h1[0], h0[1], h1[1], q.x, q.y);
                                else mma16816(of_box[p][m], h0[0], h1[0], h0[1], h1[1], q.x, q.y);
                                mma16816(of_box[p][m], h0[2], h1[2], h0[3], h1[3], q.z, q.w);
                            }
                        } else {
                            mma16816(sum[m], h0[0], h1[0], h0[1], h1[1], b.x, b.y);
                            mma16816(sum[m], h0[2], h1[2], h0[3], h1[3], b.z, b.w);
                        }
                    }
                }
                if constexpr (PARTS == 2 && !MX)
#pragma unroll
                    for (int m = 0; m < NT; ++m)
#pragma unroll
                        for (int j = 0; j < 4; ++j) sum[m][j] += of_box[0][m][j] + of_box[1][m][j] * (1.0f / float(1ull << FINER));
                }
                __syncwarp();
                if (lane == 0 && (ask_left || goes_on(passes)) && !*failed) load();
                if (++slot == a.depth) { slot = 0; parity ^= 1; }
                if (++col == block_n) { col = 0; scales_of += 16 * 128; hand_in(); }
            }
            if (col && run.hi > run.lo) hand_in();
        }
        __syncthreads();
        // A tile's boxes are [q block_n, (q + 1) block_n) of the turn's; the first warp that has one of them may have ended another tile before.
        const uint32_t first = turn * a.most, count = first < tile_n ? min(tile_n - first, a.most) : 0, all = count * block_n;
        auto finish = [&](uint32_t q, uint32_t token, float v) {
            const uint32_t m = matrix_at(tile_lo + first + q), row = (tile_lo + first + q - a.m[m].first) * 16 + (threadIdx.x & 15), rows = a.m[m].rows;
            if (row >= rows) return;
            if (a.m[m].global_scale) v *= *a.m[m].global_scale;
            if (a.scaled == SCALE_ROW) v *= static_cast<const float*>(a.x_scales)[token];
            store_as(a.m[m].y, a.y_dtype, uint64_t(token) * rows + row, *failed ? __uint_as_float(0x7FC00000u) : v);
        };
        // a thread has row threadIdx.x % 16 of every 32nd pair of tile and token
        const float per_token = __frcp_rn(float(a.tokens));
        for (uint32_t e = threadIdx.x; e < count * per; e += FEW_WARPS * 32) {
            const uint32_t q = uint32_t((float(e / 16) + 0.5f) * per_token), lo = q * block_n, hi = lo + block_n;
            uint32_t w = uint32_t((float(lo * FEW_WARPS) + 0.5f) * __frcp_rn(float(all)));
            float v = 0;
            for (uint32_t from = all * w / FEW_WARPS; from < hi && w < FEW_WARPS; ++w) {
                const uint32_t to = all * (w + 1) / FEW_WARPS;
                if (to > lo && to > from) v += shares[(w * 2 + (from < lo)) * per + e - q * per];
                from = to;
            }
            if (ranks == 1) finish(q, e / 16 - q * a.tokens, v);
            else sums[e] = v;
        }
        if (ranks > 1) {
            cluster.sync();
            for (uint32_t e = rank * FEW_WARPS * 32 + threadIdx.x; e < count * per; e += ranks * FEW_WARPS * 32) {
                float v = 0;
                for (uint32_t r = 0; r < ranks; ++r) v += *cluster.map_shared_rank(sums + e, r);
                const uint32_t q = uint32_t((float(e / 16) + 0.5f) * per_token);
                finish(q, e / 16 - q * a.tokens, v);
            }
            cluster.sync();  // before the sums are written again, and nobody leaves while others read its own
        } else if (turn + 1 < turns) {
            __syncthreads();
        }
        // the next turn's scales, where all have read this one's
        if (threadIdx.x == 0 && turn + 1 < turns) {
            fence_async_shared();
            load_scales(turn + 1);
        }
    }
    if (*failed && lane == 0) let_copies_land();
    if (threadIdx.x == 0 && *failed) atomicExch(a.status, 1u);
}

}  // namespace ptwm
