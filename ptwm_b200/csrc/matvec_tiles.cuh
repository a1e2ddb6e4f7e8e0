// Products of a 4-bit matrix with more than a few tokens, on tensor cores.
//
//   forward:   D[n][m] = sum_k W[n][k] x[m][k]       gradient: D[k][m] = sum_n W[n][k] dy[m][n]
// A block makes a tile of 128 rows of D (n, or k) and up to 256 tokens.  The matrix stays packed until it is in shared memory:
// TMA brings boxes of nibbles and scales, sixteen warps turn them into bf16 (exactly: a nibble times its scale has at most six
// significant bits) in the swizzled lines the tensor cores read, and one thread issues the MMAs.  Tokens come as bf16 by TMA.
// Tokens of other types are bf16 parts that add up to them: E4M3 is one, fp16 two, fp32 three (token_parts_kernel); each part is
// multiplied with the same converted tile, and all sums meet in the same fp32 accumulator.
//   Forward, a converted tile goes to tensor memory, whose lanes are the rows that the threads convert.  In shared memory it would be
// written and read beside the tokens, 128 bytes a cycle for all: with 256 tokens that is 830 cycles for a step whose MMAs take 512.
// In the gradient the contraction runs down the rows of the matrix, and the tile lies in shared memory as an MN-major operand.
//   The tensor cores cut what an fp32 sum cannot hold where others round: over 14336 values of fp32 tokens, three parts of them, that is
// 5e-6 of the result.  Where the results are fp32 (FLUSH), the sums of every 256 of the contraction are added up in registers: 8e-7
// (512: 1.5e-6, and 2 to 6 % less time; 128: 5e-7, 6 to 20 % more).  Results of 16 bits are rounded by a thousand times as much.
//   Where tiles are fewer than SMs, the blocks of a cluster share a tile's contraction and add their sums over distributed shared
// memory, in the order of their ranks.
//   512 tokens of 14336 x 4096 MXFP4 take 59.5 us, 1010 TFLOP/s (1.51 rounds of tiles cost two), 256 of them 31.7, their gradient 39.3, 32 of them 21.  Bound by shared memory
// (tokens in and out, 512 cycles a step, nibbles 80) beside the tensor cores (512); with up to 128 tokens by the instructions of conversion, which has
// a kernel for either kind of scales: one for both took 25.4 us for 32 tokens.
//   What a step costs: 512 cycles of MMA with 256 tokens; some 300 issue slots of conversion; and the issuing thread, to which a wait
// for a barrier is 170 cycles, a commit 100 and four MMAs 100, ready or not.  So a stage has one barrier for all that arrives in it and is
// two steps where tokens are few.
#pragma once
#include <cooperative_groups.h>

#include "matvec.cuh"
#include "tensor_core.cuh"

namespace ptwm {

constexpr uint32_t TILE_ROWS = 128;                 // rows of D to a block
constexpr uint32_t STEP = 64;                       // contraction to a converted tile: one 128-byte line of bf16
constexpr uint32_t RAW_STAGES = 6, RAW_BYTES = 8192, SCALES_BYTES = 8192, A_BYTES = TILE_ROWS * STEP * 2, MOST_STAGES = 6;
constexpr uint32_t TILES_THREADS = 640;             // warp 0: TMA of the matrix, 1: MMA, 2: TMA of the tokens, 4 to 19: conversion, then the results
constexpr uint32_t TILES_HEAD = 1024;               // barriers and the like, in front of the buffers

struct TilesArgs {
    uint64_t rows;             // of D: n, or k in the gradient
    uint64_t contraction;      // k, or n
    uint64_t tokens;
    uint64_t part_rows;        // rows from one part of the tokens to the next
    uint32_t parts;
    uint32_t tile_tokens;      // a multiple of 16, at most 256
    uint32_t stages;           // of `together` converted tiles and the tokens that belong to them
    uint32_t together;         // 1 or 2 steps
    uint32_t teams;            // of four warps that convert: 4, and no more than the steps of all stages
    uint32_t y_dtype;
    const float* global_scale;
    const float* token_scale;  // or null
    void* y;
    uint32_t* status;
};

__host__ __device__ constexpr uint32_t tiles_stage(uint32_t tile_tokens, uint32_t parts, uint32_t together, bool grad) {
    return together * ((grad ? A_BYTES : 0) + parts * tile_tokens * STEP * 2);
}
// Bytes of dynamic shared memory; 1024 more to align them.
inline uint32_t tiles_smem(uint32_t stage, uint32_t stages) { return 1024 + TILES_HEAD + RAW_STAGES * RAW_BYTES + SCALES_BYTES + stages * stage; }
// A block has an SM to itself: two that wait for tensor memory on each other's could wait for good.
constexpr uint32_t TILES_LEAST_SMEM = 120 * 1024;
constexpr uint32_t TMEM_COLS = 512, A_COLS = STEP / 2;   // columns of tensor memory; of a converted tile in it
constexpr uint32_t FLUSH_STEPS = 4, FLUSH_TOKENS = 128;  // tokens: what a thread has registers for
__host__ __device__ constexpr uint32_t tiles_sums(uint32_t tile_tokens, bool flush) { return (tile_tokens + 31) / 32 * 32 * (flush ? 2 : 1); }
inline uint32_t tiles_tmem_stages(uint32_t tile_tokens, uint32_t together, bool flush) { return (TMEM_COLS - tiles_sums(tile_tokens, flush)) / (together * A_COLS); }

// Eight nibbles -> eight bf16 in their order, times `scale`.  A word takes the even nibble of a byte to its low half and the odd one
// to its high half; a product puts their signs at bit 15 and the other three bits at 8..6, which reads as the number times 2^-126;
// `scale` is the group's times 2^126.  Every step is exact.
__device__ __forceinline__ void nibbles_to_bf16(uint32_t w, uint32_t scale, uint32_t (&out)[4]) {
    const uint32_t even = w & 0x0F0F0F0Fu, odd = w >> 4 & 0x0F0F0F0Fu;
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
        uint32_t v;   // (a byte's highest bit, in all of a byte, is 0: what __byte_perm does not offer)
        asm("prmt.b32 %0, %1, %2, %3;" : "=r"(v) : "r"(even), "r"(odd), "r"(i | (8 | i) << 4 | (4 + i) << 8 | (12 + i) << 12));
        const uint32_t bits = (v * 0x1040u) & 0x81C081C0u;
        asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(out[i]) : "r"(bits), "r"(scale));
    }
}

// Scale of a group as a pair of bf16.  MXFP4: 2^(e - 127) 2^126, and for e above 128 the rest in *more (else 1).  NVFP4: s 2^126 would
// pass bf16's range, so it is s 2^116, and the results are multiplied by 2^10.
__device__ __forceinline__ uint32_t mx_scale(uint32_t e, uint32_t* more) {
    const uint32_t hi = e > 128 ? 254 : e + 126, rest = e > 128 ? e - 1 : 127;
    *more = e == 255 ? 0x7FC07FC0u : rest * 0x00800080u;
    return hi * 0x00800080u;
}
__device__ __forceinline__ uint32_t nv_scale(uint32_t s) {
    const __nv_bfloat16 b = __float2bfloat16_rn(e4m3_f32(uint8_t(s)) * 0x1p116f);
    uint16_t u;
    memcpy(&u, &b, 2);
    return u * 0x00010001u;
}
constexpr float NV_REST = 1024.0f;

template <bool GRAD> struct TilesShared {
    static constexpr uint32_t raw = TILES_HEAD, scales = raw + RAW_STAGES * RAW_BYTES, stages = scales + SCALES_BYTES;
    static constexpr uint32_t raw_rows = GRAD ? STEP : TILE_ROWS, scale_bytes = raw_rows * 16, scale_slots = SCALES_BYTES / scale_bytes;
    // barriers: raw full / empty, scales full (a slot is free once all raw stages before raw - RAW_STAGES are), stage full / empty, two of sums done and
    // flushed
    static constexpr uint32_t raw_full = 0, raw_empty = 64, full = 128, empty = 192, scales_full = 256, done = 320, flushed = 336, tmem = 352, failed = 356;
    static_assert(RAW_STAGES <= 8 && MOST_STAGES <= 8 && scale_slots <= 8, "barriers do not overlap");
};

// 16 bytes of nibbles (32 values) -> four 16-byte pieces of bf16.  s: the scale of all (MXFP4), or of the first and the second half.
template <bool MX> __device__ __forceinline__ void convert32(const uint4& v, uint32_t s, uint4 (&out)[4]) {
    const uint32_t words[4] = {v.x, v.y, v.z, v.w};
    uint32_t more = 0x3F803F80u;
    const uint32_t s0 = MX ? mx_scale(s & 255, &more) : nv_scale(s & 255), s1 = MX ? s0 : nv_scale(s >> 8 & 255);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t o[4];
        nibbles_to_bf16(words[i], i < 2 ? s0 : s1, o);
        if (MX && more != 0x3F803F80u) {
#pragma unroll
            for (int j = 0; j < 4; ++j) asm("mul.rn.bf16x2 %0, %0, %1;" : "+r"(o[j]) : "r"(more));
        }
        out[i] = make_uint4(o[0], o[1], o[2], o[3]);
    }
}

template <bool GRAD, bool FLUSH, bool MX>
__global__ void __launch_bounds__(TILES_THREADS, 1) matvec_tiles_kernel(const __grid_constant__ CUtensorMap values, const __grid_constant__ CUtensorMap scales,
                                                                        const __grid_constant__ CUtensorMap tokens, const TilesArgs t) {
    namespace cg = cooperative_groups;
    using S = TilesShared<GRAD>;
    constexpr uint32_t GROUP = MX ? 32 : 16;
    extern __shared__ uint8_t dynamic[];
    uint8_t* base = dynamic + (1024 - (smem_u32(dynamic) & 1023)) % 1024;
    const uint32_t sb = smem_u32(base);
    volatile uint32_t* failed = reinterpret_cast<uint32_t*>(base + S::failed);
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x & 31;
    const cg::cluster_group cluster = cg::this_cluster();
    const uint32_t ranks = cluster.num_blocks(), rank = cluster.block_rank();
    const uint32_t row0 = blockIdx.x / ranks * TILE_ROWS, token0 = blockIdx.y * t.tile_tokens;
    // A raw stage is 128 k of 128 rows (two steps) forward, and 64 rows (one step) of the tile's 128 k in the gradient.  A box of scales is
    // 16 bytes of each row: 512 k (MXFP4) or 256 (NVFP4), so several raw stages forward, one in the gradient.
    const uint32_t scale_raws = GRAD ? 1 : MX ? 4 : 2, unit = GRAD ? t.together : 2 * scale_raws;
    // this block's steps: whole boxes of scales, and whole stages
    const uint32_t units = uint32_t((t.contraction + unit * STEP - 1) / (unit * STEP));
    const uint32_t step0 = units * rank / ranks * unit, all = uint32_t((t.contraction + STEP - 1) / STEP), end = min(units * (rank + 1) / ranks * unit, all);
    const uint32_t steps = (end > step0 ? end - step0 + t.together - 1 : 0) / t.together * t.together;  // what is behind the contraction is zeros
    const uint32_t raw0 = GRAD ? step0 : step0 / 2, raws = GRAD ? steps : (steps + 1) / 2;
    const uint32_t b_bytes = t.tile_tokens * STEP * 2, stage_bytes = tiles_stage(t.tile_tokens, t.parts, t.together, GRAD), b_first = GRAD ? t.together * A_BYTES : 0;

    if (threadIdx.x == 0) {
        *failed = 0;
        // four warps convert a step
        for (uint32_t i = 0; i < RAW_STAGES; ++i) { mbar_init(sb + S::raw_full + 8 * i, 1); mbar_init(sb + S::raw_empty + 8 * i, GRAD ? 4 : 8); }
        for (uint32_t i = 0; i < t.stages; ++i) { mbar_init(sb + S::full + 8 * i, 4 * t.together + 1); mbar_init(sb + S::empty + 8 * i, 1); }
        for (uint32_t i = 0; i < S::scale_slots; ++i) mbar_init(sb + S::scales_full + 8 * i, 1);
        for (uint32_t i = 0; i < 2; ++i) { mbar_init(sb + S::done + 8 * i, 1); mbar_init(sb + S::flushed + 8 * i, 16); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tmem_alloc(sb + S::tmem, TMEM_COLS);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(base + S::tmem);
    const uint32_t sums_cols = tiles_sums(t.tile_tokens, false), a_tmem = tmem + tiles_sums(t.tile_tokens, FLUSH);  // converted tiles behind the sums
    const uint32_t segments = FLUSH ? (steps + FLUSH_STEPS - 1) / FLUSH_STEPS : 1;
    others_may_start();
    after_those_before();

    // (counters instead of divisions in the warps of one thread: its latency is what they cost)
    if (warp == 0) {
        if (elect_one()) {
            uint32_t st = 0, parity = 1, slot = 0, piece = 0, scale_x = GRAD ? row0 / GROUP & ~15u : raw0 / scale_raws * 16;
            for (uint32_t raw = 0; raw < raws; ++raw) {
                const uint32_t full = sb + S::raw_full + 8 * st, dst = sb + S::raw + st * RAW_BYTES;
                if (raw >= RAW_STAGES && !mbar_wait(sb + S::raw_empty + 8 * st, parity, failed)) break;
                mbar_expect(full, S::raw_rows * 64);
                if (GRAD) tma_load(dst, &values, full, int32_t(row0 / 2), int32_t((raw0 + raw) * STEP));
                else tma_load(dst, &values, full, int32_t((raw0 + raw) * 64), int32_t(row0));
                if (piece == 0) {
                    // its slot was last read for raw stages before raw - RAW_STAGES: there are enough slots for those in between
                    const uint32_t bar = sb + S::scales_full + 8 * slot;
                    mbar_expect(bar, S::scale_bytes);
                    tma_load(sb + S::scales + slot * S::scale_bytes, &scales, bar, int32_t(scale_x), int32_t(GRAD ? (raw0 + raw) * STEP : row0));
                    if (!GRAD) scale_x += 16;
                    if (++slot == S::scale_slots) slot = 0;
                }
                if (++piece == scale_raws) piece = 0;
                if (++st == RAW_STAGES) { st = 0; parity ^= 1; }
            }
            // every load has been waited for by those who use it, unless something failed: then what is under way gets time to land
            if (*failed) let_copies_land();
        }
    } else if (warp == 2) {
        if (elect_one()) {
            uint32_t st = 0, parity = 1, round = 0;
            for (uint32_t step = 0; step < steps; step += t.together) {
                const uint32_t full = sb + S::full + 8 * st;
                uint32_t dst = sb + S::stages + st * stage_bytes + b_first;
                if (round && !mbar_wait(sb + S::empty + 8 * st, parity, failed)) break;
                mbar_expect(full, t.together * t.parts * b_bytes);
                for (uint32_t i = 0; i < t.together; ++i)
                    for (uint32_t p = 0; p < t.parts; ++p, dst += b_bytes) tma_load(dst, &tokens, full, int32_t((step0 + step + i) * STEP), int32_t(p * t.part_rows + token0));
                if (++st == t.stages) { st = 0; parity ^= 1; round = 1; }
            }
            if (*failed) let_copies_land();
        }
    } else if (warp == 1) {
        if (elect_one()) {
            const uint32_t idesc = instruction_desc(t.tile_tokens, GRAD);
            const uint64_t a_desc = operand_desc(sb + S::stages, 8192, 1024), b_desc = operand_desc(sb + S::stages + b_first, 16, 1024);
            uint32_t st = 0, parity = 0;
            bool more = false;
            uint32_t d = tmem, segment = 0;
            for (uint32_t step = 0; step < steps; step += t.together) {
                if (FLUSH && step && step % FLUSH_STEPS == 0) {  // the other sums, once what was in them has been taken
                    tc_commit(sb + S::done + 8 * (segment & 1));
                    ++segment;
                    if (segment > 1 && !mbar_wait(sb + S::flushed + 8 * (segment & 1), (segment / 2 - 1) & 1, failed)) break;
                    d = tmem + (segment & 1) * sums_cols;
                    more = false;
                }
                if (!mbar_wait(sb + S::full + 8 * st, parity, failed)) break;
                tc_fence_after();
                uint64_t ad = a_desc + st * (stage_bytes / 16), bd = b_desc + st * (stage_bytes / 16);
                uint32_t at = a_tmem + st * t.together * A_COLS;
                for (uint32_t i = 0; i < t.together; ++i, ad += A_BYTES / 16, at += A_COLS)
                    for (uint32_t p = 0; p < t.parts; ++p, bd += b_bytes / 16) {
#pragma unroll
                        for (uint32_t k = 0; k < STEP / 16; ++k) {
                            if (GRAD) mma_f16(d, ad + k * (2048 / 16), bd + k * 2, idesc, more);
                            else mma_f16_tmem(d, at + k * 8, bd + k * 2, idesc, more);
                            more = true;
                        }
                    }
                tc_commit(sb + S::empty + 8 * st);
                if (++st == t.stages) { st = 0; parity ^= 1; }
            }
            tc_commit(sb + S::done + 8 * (segment & 1));
        }
    } else if (warp >= 4) {
        // Teams of four warps take a step each in turn: a step is some 200 instructions of a thread in a row, and up to four of them are under way.
        // With no more teams than steps in all stages a team that waits for a stage to be free waits for its last use but one at most: two back, the
        // parity of its barrier would say that it is free.
        // A thread has 32 bytes of a row (64 values of it): forward the step's part of row c, in the gradient one half of row c % 64.  TMA has swizzled
        // the 16-byte pieces of a raw stage's 64-byte rows, so that neighbouring rows lie in different banks, and in shared memory they are stored swizzled.
        const uint32_t team = (warp - 4) / 4, c = threadIdx.x % 128, row = GRAD ? c % 64 : c, half = c / 64;
        const uint32_t first_group = GRAD ? row0 / GROUP & 15u : 0;
        const uint32_t out = half * 8192 + row / 8 * 1024 + row % 8 * 128;
        uint32_t st = team / t.together, round = 0;  // stage of the step, and how often the stages have been gone through
        while (st >= t.stages) { st -= t.stages; ++round; }
        const uint32_t lanes = warp % 4 * 32;
        float total[FLUSH ? FLUSH_TOKENS / 4 : 1];
        uint32_t next = 0;
        if (FLUSH)
#pragma unroll
            for (uint32_t i = 0; i < FLUSH_TOKENS / 4; ++i) total[i] = 0;
        auto flush = [&] {  // the sums of segment `next`: this team's columns of them
            const uint32_t which = next & 1;
            mbar_wait(sb + S::done + 8 * which, next / 2 & 1, failed);
            tc_fence_after();
#pragma unroll
            for (uint32_t i = 0; i < FLUSH_TOKENS / 64; ++i)
                if (team * 16 + i * 64 < t.tile_tokens) {
                    uint32_t v[16];
                    tmem_load16(tmem + which * sums_cols + (lanes << 16) + team * 16 + i * 64, v);
#pragma unroll
                    for (uint32_t j = 0; j < 16; ++j) total[i * 16 + j] += __uint_as_float(v[j]);
                }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(sb + S::flushed + 8 * which);
            ++next;
        };
        for (uint32_t step = team; step < steps && team < t.teams; step += t.teams) {
            if constexpr (FLUSH)
                while (next + 2 <= step / FLUSH_STEPS) flush();
            const uint32_t raw = GRAD ? step : step / 2, rs = raw % RAW_STAGES;
            const uint32_t pair = GRAD ? half : step % 2;  // which 64 of the 128 k
            if (!mbar_wait(sb + S::raw_full + 8 * rs, raw / RAW_STAGES & 1, failed)) break;
            const uint8_t* line = base + S::raw + rs * RAW_BYTES + row * 64;
            const uint4 v0 = *reinterpret_cast<const uint4*>(line + ((pair * 2 ^ row / 2) & 3) * 16), v1 = *reinterpret_cast<const uint4*>(line + ((pair * 2 + 1 ^ row / 2) & 3) * 16);
            const uint32_t scale_at = raw / scale_raws, slot = scale_at % S::scale_slots;
            if (!mbar_wait(sb + S::scales_full + 8 * slot, scale_at / S::scale_slots & 1, failed)) break;
            const uint8_t* sp = base + S::scales + slot * S::scale_bytes + row * 16;
            const uint32_t g = first_group + raw % scale_raws * (128 / GROUP) + pair * (64 / GROUP);
            const uint32_t s = MX ? *reinterpret_cast<const uint16_t*>(sp + g) : *reinterpret_cast<const uint32_t*>(sp + g);
            if (round && !mbar_wait(sb + S::empty + 8 * st, (round - 1) & 1, failed)) break;
            uint4 o[4];
            if constexpr (GRAD) {
                uint8_t* dst = base + S::stages + st * stage_bytes + step % t.together * A_BYTES + out;
                convert32<MX>(v0, s, o);
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j) *reinterpret_cast<uint4*>(dst + ((j ^ (row % 8)) * 16)) = o[j];
                convert32<MX>(v1, MX ? s >> 8 : s >> 16, o);
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j) *reinterpret_cast<uint4*>(dst + ((4 + j ^ (row % 8)) * 16)) = o[j];
                fence_async_shared();
            } else {
                tc_fence_after();  // the MMAs that read what was here before are done
                const uint32_t at = a_tmem + (warp % 4 * 32 << 16) + (st * t.together + step % t.together) * A_COLS;
                uint32_t v[16];
                convert32<MX>(v0, s, o);
                memcpy(v, o, 64);
                tmem_store16(at, v);
                convert32<MX>(v1, MX ? s >> 8 : s >> 16, o);
                memcpy(v, o, 64);
                tmem_store16(at + 16, v);
                tmem_wait_stores();
                tc_fence_before();
            }
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(sb + S::full + 8 * st);
                mbar_arrive(sb + S::raw_empty + 8 * rs);
            }
            st += t.teams / t.together;
            while (st >= t.stages) { st -= t.stages; ++round; }
        }
        // results: a warp reaches the 32 lanes (rows of D) that its number modulo 4 names; the four teams share the tokens
        if constexpr (FLUSH) {
            while (next < segments) flush();
        } else {
            mbar_wait(sb + S::done, 0, failed);
            tc_fence_after();
        }
        const uint64_t n = row0 + lanes + lane;
        float factor = MX ? 1.0f : NV_REST;
        if (t.global_scale) factor *= *t.global_scale;
        if (*failed) factor = __uint_as_float(0x7FC00000u);
        float* const sums = reinterpret_cast<float*>(base + TILES_HEAD);  // [token][row]: nothing reads or writes the buffers any more
#pragma unroll 1
        for (uint32_t i = 0; i < (FLUSH ? FLUSH_TOKENS / 64 : 4); ++i) {
            const uint32_t m = team * 16 + i * 64;
            if (m >= t.tile_tokens) break;
            uint32_t v[16];
            if constexpr (FLUSH) {
#pragma unroll
                for (uint32_t j = 0; j < 16; ++j) v[j] = __float_as_uint(i == 0 ? total[j] : total[16 + j]);
            } else {
                tmem_load16(tmem + (lanes << 16) + m, v);
            }
            if (ranks > 1) {
#pragma unroll
                for (uint32_t j = 0; j < 16; ++j) sums[(m + j) * TILE_ROWS + lanes + lane] = __uint_as_float(v[j]) * factor;
            } else if (n < t.rows) {
#pragma unroll
                for (uint32_t j = 0; j < 16; ++j) {
                    const uint64_t token = token0 + m + j;
                    if (token < t.tokens) {
                        const float f = __uint_as_float(v[j]) * factor;
                        store_as(t.y, t.y_dtype, token * t.rows + n, t.token_scale ? f * t.token_scale[token] : f);
                    }
                }
            }
        }
        tc_fence_before();
    }
    if (ranks > 1) {
        __syncwarp();
        cluster.sync();
        float* const sums = reinterpret_cast<float*>(base + TILES_HEAD);
        const uint32_t r = threadIdx.x % TILE_ROWS;
        const uint64_t n = row0 + r;
        for (uint32_t m = t.tile_tokens * rank / ranks + threadIdx.x / TILE_ROWS; m < t.tile_tokens * (rank + 1) / ranks; m += TILES_THREADS / TILE_ROWS) {
            float v = 0;
            for (uint32_t i = 0; i < ranks; ++i) v += *cluster.map_shared_rank(sums + m * TILE_ROWS + r, i);
            const uint64_t token = token0 + m;
            if (n < t.rows && token < t.tokens) store_as(t.y, t.y_dtype, token * t.rows + n, t.token_scale ? v * t.token_scale[token] : v);
        }
        cluster.sync();  // nobody leaves while others read its sums
    }
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_free(tmem, TMEM_COLS);
    }
    if (threadIdx.x == 0 && *failed) atomicExch(t.status, 1u);
}

// Eight values of a token from k on, where they lie at a multiple of their size.
__device__ __forceinline__ void eight_values(const float* p, float (&v)[8]) {
    const float4 a = __ldcs(reinterpret_cast<const float4*>(p)), b = __ldcs(reinterpret_cast<const float4*>(p) + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
template <class T> __device__ __forceinline__ void eight_values(const T* p, float (&v)[8]) {
    uint32_t w[4];
    if constexpr (sizeof(T) == 2) {
        const uint4 a = __ldcs(reinterpret_cast<const uint4*>(p));
        w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
    } else {
        const uint2 a = __ldcs(reinterpret_cast<const uint2*>(p));
        w[0] = a.x & 0xFFFF; w[1] = a.x >> 16; w[2] = a.y & 0xFFFF; w[3] = a.y >> 16;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float2 f;
        if constexpr (sizeof(T) == 2) f = two_f32<T>(w[i]);
        else f = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(__nv_fp8x2_storage_t(w[i]), __NV_E4M3)));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}

// Tokens as bf16 parts whose sum they are: part p of token m is row p * part_rows + m of `out`, `pitch` values long, with zeros behind
// `cols`.  E4M3 (times its block's scale) fits one bf16, fp16 two, fp32 three (each takes the next eight bits).  What is not finite is
// its first part alone.  Bound by memory: eight values to a thread, which are one load where the rows lie so (`wide`) and one
// store.  4096 tokens of 4096 E4M3 10 us, 5 TB/s (a value to a thread 70), 512 of them 1.9 (9.5).
template <class T>
__global__ void __launch_bounds__(256) token_parts_kernel(TokenArgs t, uint64_t cols, __nv_bfloat16* out, uint32_t pitch, uint64_t part_rows, bool wide) {
    constexpr int PARTS = sizeof(T) == 4 ? 3 : sizeof(T) == 1 ? 1 : std::is_same<T, __half>::value ? 2 : 1;
    const uint64_t m = blockIdx.x;
    others_may_start();
    after_those_before();
    for (uint64_t k = (uint64_t(blockIdx.y) * 256 + threadIdx.x) * 8; k < pitch; k += uint64_t(gridDim.y) * 2048) {
        float rest[8];
        if (wide) {
            eight_values(static_cast<const T*>(t.x) + m * cols + k, rest);
            if (sizeof(T) == 1 && t.scaled == SCALE_BLOCK) {
                const float s = e8m0_f32(static_cast<const uint8_t*>(t.scales)[m * (cols / 32) + k / 32]);
#pragma unroll
                for (int i = 0; i < 8; ++i) rest[i] *= s;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) rest[i] = k + i < cols ? token_value<T>(t, m, k + i, cols) : 0.0f;
        }
#pragma unroll
        for (int p = 0; p < PARTS; ++p) {
            uint32_t top[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                // cut, not rounded: a value near the largest stays finite
                const uint32_t bits = __float_as_uint(rest[i]);
                const bool finite = (bits & 0x7F800000u) != 0x7F800000u;
                top[i] = rest[i] == rest[i] ? bits & 0xFFFF0000u : 0x7FC00000u;
                rest[i] = finite ? rest[i] - __uint_as_float(top[i]) : 0.0f;
            }
            *reinterpret_cast<uint4*>(out + (p * part_rows + m) * pitch + k) =
                make_uint4(top[0] >> 16 | top[1], top[2] >> 16 | top[3], top[4] >> 16 | top[5], top[6] >> 16 | top[7]);
        }
    }
}

}  // namespace ptwm
