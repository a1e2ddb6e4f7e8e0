// Host side of the operators that apply decoded weights: rms_norm and matvec with 4-bit weights.  A translation unit of its
// own; every call enqueues its kernels on the caller's stream and returns.
#include <algorithm>
#include <exception>
#include <initializer_list>
#include <map>
#include <mutex>
#include <type_traits>

#include "errors.hpp"
#include "matvec.cuh"
#include "matvec_few.cuh"
#include "matvec_tiles.cuh"
#include "rms_norm.cuh"

using namespace ptwm;

namespace {

// The body of an entry point: no exception leaves it.
template <class F> int64_t guarded(F f) {
    try { return f(); } catch (const std::exception& e) { return fail(PTWM_RC_INTERNAL, e.what()); }
}

template <class T> T* at(uint64_t p) { return reinterpret_cast<T*>(uintptr_t(p)); }
cudaStream_t stream_of(uint64_t s) { return reinterpret_cast<cudaStream_t>(uintptr_t(s)); }
bool plain_type(uint32_t t) { return t == DT_FP32 || t == DT_FP16 || t == DT_BF16; }

// f(T()) with the C++ type of a plain dtype code.
template <class F> void with_type(uint32_t t, F f) {
    if (t == DT_FP32) f(float());
    else if (t == DT_FP16) f(__half());
    else f(__nv_bfloat16());
}

// Enqueues a kernel that may start while the one before it in the stream ends (see after_those_before).
template <class... P, class... A> cudaError_t enqueue(void (*kernel)(P...), dim3 grid, uint32_t threads, uint32_t smem, uint32_t ranks, cudaStream_t st, const A&... args) {
    cudaLaunchAttribute attrs[2];
    attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[0].val.programmaticStreamSerializationAllowed = 1;
    attrs[1].id = cudaLaunchAttributeClusterDimension;
    attrs[1].val.clusterDim = {ranks, 1, 1};
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = attrs;
    cfg.numAttrs = ranks > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

int64_t matrix_of(const ptwm_b200_scaled_weight* w, ScaledMatrix* out) {
    if (!w || !w->values || !w->scales) return fail(PTWM_RC_INVALID_INPUT, "scaled weight: null pointer");
    if (w->group != 16 && w->group != 32) return fail(PTWM_RC_INVALID_INPUT, "scaled weight: groups are 16 (E4M3 scales) or 32 (E8M0 scales) values");
    if (!w->rows || !w->cols || w->cols % w->group) return fail(PTWM_RC_INVALID_INPUT, "scaled weight: cols must be a positive multiple of the group");
    if (w->rows > (1u << 30) || w->cols > (1u << 30)) return fail(PTWM_RC_UNSUPPORTED, "scaled weight: more than 2^30 rows or columns");
    if (w->value_pitch % 16 || w->scale_pitch % 16 || w->values % 16 || w->scales % 16 || w->global_scale % 4)
        return fail(PTWM_RC_INVALID_INPUT, "scaled weight: rows of values and scales start at multiples of 16 bytes, the global scale at one of 4");
    if (w->value_pitch < w->cols / 2 || w->scale_pitch < w->cols / w->group) return fail(PTWM_RC_INVALID_INPUT, "scaled weight: pitch shorter than a row");
    *out = ScaledMatrix{at<const uint8_t>(w->values), at<const uint8_t>(w->scales), at<const float>(w->global_scale), w->rows, w->cols, w->value_pitch, w->scale_pitch, w->group};
    return 0;
}

constexpr uint32_t SMEM_MOST = 227 * 1024;

// How a product with few tokens is split: a block per SM, clusters of as few as let the tokens fit shared memory beside two boxes
// per warp (up to five where there is room).  depth 0: they do not.
struct FewSplit { uint32_t ranks, most, depth, smem, blocks, lines; };
FewSplit few_split(uint32_t tiles, uint32_t boxes, uint32_t tokens, uint32_t parts, uint32_t group) {
    constexpr uint32_t SMS = 148;
    // Where two blocks to a cluster, or for more than eight tokens one turn, are not enough, tiles are quicker: 8 tokens of 4096 x 14336 (NVFP4) take 22 us
    // in two blocks (21 in tiles), 9 of them 35 (21), 16 in four blocks 62 (21); 16 of 14336 x 4096 20 (21), one of 4096 x 14336 11.7.
    for (uint32_t ranks = 1; ranks <= 2 && ranks <= boxes; ranks *= 2) {
        const uint32_t share = (boxes + ranks - 1) / ranks, clusters = std::min(tiles, SMS / ranks), run = (tiles + clusters - 1) / clusters;
        const uint32_t lines = few_lines(share, group);
        // row tiles to a turn: as many as warps, fewer where the scales of all do not fit beside the rest
        for (uint32_t limit = FEW_WARPS; limit >= (tokens > 8 ? FEW_WARPS : 1); limit /= 2) {
            const uint32_t turns = (run + limit - 1) / limit, most = (run + turns - 1) / turns;
            for (uint32_t depth = FEW_DEPTH; depth >= 2; --depth)
                if (const uint64_t smem = few_smem(tokens, share, depth, parts, ranks, most, lines); smem <= SMEM_MOST) return {ranks, most, depth, uint32_t(smem), clusters * ranks, lines};
        }
    }
    return {};
}
uint32_t few_boxes(const ScaledMatrix& w) { return uint32_t((w.cols + BOX_COLS - 1) / BOX_COLS); }
uint32_t few_tiles(const ScaledMatrix& w) { return uint32_t((w.rows + 15) / 16); }
FewSplit few_split(const ScaledMatrix& w, uint32_t tiles, uint64_t tokens, uint32_t x_dtype) {
    return tokens > FEW_TOKENS ? FewSplit{} : few_split(tiles, few_boxes(w), uint32_t(tokens), x_dtype == DT_FP32 ? 2 : 1, w.group);
}

template <class F> void with_few(uint32_t x_dtype, uint32_t tokens, bool mx, F f) {
    auto pick = [&](auto v, auto m) {
        using T = decltype(v);
        constexpr bool MX = decltype(m)::value;
        if (tokens > 8) return f(matvec_few_kernel<T, 16, MX>);
        if constexpr (sizeof(T) < 4) {
            if (tokens == 1) return f(matvec_few_kernel<T, 1, MX>);
            if (tokens == 2) return f(matvec_few_kernel<T, 2, MX>);
        }
        f(matvec_few_kernel<T, 8, MX>);
    };
    auto either = [&](auto v) { mx ? pick(v, std::true_type()) : pick(v, std::false_type()); };
    if (x_dtype == DT_E4M3) either(uint8_t());
    else with_type(x_dtype, either);
}
cudaError_t allow_few() {
    cudaError_t e = cudaSuccess;
    for (uint32_t t : {DT_FP32, DT_FP16, DT_BF16, DT_E4M3})
        for (uint32_t tokens : {1u, 2u, 8u, 16u})
            for (bool mx : {false, true})
                if (e == cudaSuccess) with_few(t, tokens, mx, [&](auto f) { e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, int(SMEM_MOST)); });
    return e;
}

// Columns of a norm: the kernels have places in a row, and what is a few pieces behind its end, in signed 32 bits.
constexpr uint64_t NORM_COLS = 1ull << 30;
bool aligned(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
uint32_t warps_for(uint64_t threads) { return uint32_t((threads + 31) / 32 * 32); }

// One piece of 16 bytes to a thread where rows are few and a call takes as long as one of them (one row of 4096 bf16: 512 threads), two
// where there are many.  False: the rows are not made for it.
template <class T, class W, uint32_t QUANT> bool launch_norm_rows(const NormArgs& a, cudaStream_t st, cudaError_t& e) {
    constexpr uint64_t V = 16 / sizeof(T);
    if (a.cols % V || !aligned(a.x) || !aligned(a.residual) || !aligned(a.weight) || !aligned(a.h) || !aligned(a.y)) return false;
    const uint64_t pieces = a.cols / V;
    const uint32_t rows = uint32_t(a.rows);
    // A row to each of so many blocks that an SM has 1024 threads of them (2048: no faster; 1536 leaves some SMs with more than others), and the
    // next ones after it.  Rows of up to 128 pieces to half a warp or a warp, all at once (200,000 rows of 128 bf16: 46 us, 51 in turns).
    auto blocks = [&](uint32_t threads) { return std::min<uint32_t>(rows, 148 * std::max(1u, 1024 / threads)); };
    if (pieces <= 128 && a.rows > 148) {
        if (pieces <= 16) e = enqueue(rms_norm_rows_kernel<T, W, 1, 16, QUANT>, dim3((rows + 15) / 16), 256, 0, 1, st, a);
        else if (pieces <= 32) e = enqueue(rms_norm_rows_kernel<T, W, 1, 32, QUANT>, dim3((rows + 7) / 8), 256, 0, 1, st, a);
        else if (pieces <= 64) e = enqueue(rms_norm_rows_kernel<T, W, 2, 32, QUANT>, dim3((rows + 7) / 8), 256, 0, 1, st, a);
        else e = enqueue(rms_norm_rows_kernel<T, W, 4, 32, QUANT>, dim3((rows + 7) / 8), 256, 0, 1, st, a);
    } else if (pieces <= 1024 && a.rows <= 296) e = enqueue(rms_norm_rows_kernel<T, W, 1, 0, QUANT>, dim3(rows), warps_for(pieces), 0, 1, st, a);
    else if (pieces <= 2048) e = enqueue(rms_norm_rows_kernel<T, W, 2, 0, QUANT>, dim3(blocks(warps_for((pieces + 1) / 2))), warps_for((pieces + 1) / 2), 0, 1, st, a);
    else return false;
    return true;
}
template <class T, class W> cudaError_t launch_norm(const NormArgs& a, uint32_t scaled, cudaStream_t st) {
    const uint32_t rows = uint32_t(a.rows);
    cudaError_t e = cudaSuccess;
    if (scaled == SCALE_NONE ? launch_norm_rows<T, W, SCALE_NONE>(a, st, e) : scaled == SCALE_ROW ? launch_norm_rows<T, W, SCALE_ROW>(a, st, e) : launch_norm_rows<T, W, SCALE_BLOCK>(a, st, e)) return e;
    constexpr uint64_t V = 16 / sizeof(T);
    const uint64_t pieces = a.cols / V + 2;   // of the whole tensor that a row has a share of, at most
    const bool wide = aligned(a.x) && aligned(a.residual) && aligned(a.weight) && aligned(a.h) && aligned(a.y);
    if (wide && a.cols % V == 0) e = enqueue(rms_norm_wide_kernel<T, W, false>, dim3(rows), 512, 0, 1, st, a, scaled);
    else if (wide && pieces > 2048) e = enqueue(rms_norm_wide_kernel<T, W, true>, dim3(rows), 512, 0, 1, st, a, scaled);
    else if (wide) {
        const uint32_t threads = warps_for((pieces + 1) / 2);
        e = enqueue(rms_norm_between_kernel<T, W>, dim3(std::min<uint32_t>(rows, 148 * std::max(1u, 1024 / threads))), threads, 0, 1, st, a, scaled);
    } else if (scaled != SCALE_BLOCK && a.cols <= 16 * 1024) e = enqueue(rms_norm_odd_rows_kernel<T, W, 16>, dim3(rows), warps_for((a.cols + 15) / 16), 0, 1, st, a, scaled);
    else e = enqueue(rms_norm_long_kernel<T, W>, dim3(rows), 256, 0, 1, st, a, scaled);
    return e;
}

// Blocks of a gradient: each writes its share of dweight, so no more than fill the GPU.  296 rows on, a row begins at the same place of 16 bytes.
constexpr uint32_t GRAD_BLOCKS = 296;
static_assert(GRAD_BLOCKS % 8 == 0, "");
uint32_t grad_blocks(uint64_t rows) { return uint32_t(std::min<uint64_t>(rows, GRAD_BLOCKS)); }

template <class T, class W, bool BETWEEN> bool launch_norm_grad_rows(const NormGradArgs& a, uint64_t pieces, cudaStream_t st, cudaError_t& e) {
    if (pieces <= 512) e = enqueue(rms_norm_grad_rows_kernel<T, W, 1, 512, BETWEEN>, dim3(a.blocks), warps_for(pieces), 0, 1, st, a);
    else if (pieces <= 1024) e = enqueue(rms_norm_grad_rows_kernel<T, W, 2, 512, BETWEEN>, dim3(a.blocks), warps_for((pieces + 1) / 2), 0, 1, st, a);
    else if (pieces <= 2048) e = enqueue(rms_norm_grad_rows_kernel<T, W, 2, 1024, BETWEEN>, dim3(a.blocks), warps_for((pieces + 1) / 2), 0, 1, st, a);
    else return false;
    return true;
}
template <class T, class W> cudaError_t launch_norm_grad(const NormGradArgs& a, cudaStream_t st) {
    cudaError_t e;
    constexpr uint64_t V = 16 / sizeof(T);
    const bool wide = aligned(a.h) && aligned(a.weight) && aligned(a.dy) && aligned(a.dh) && aligned(a.dx) && aligned(a.partial);
    const bool between = a.cols % V != 0;
    const uint64_t pieces = a.cols / V + (between ? 2 : 0);
    if (wide && (between ? launch_norm_grad_rows<T, W, true>(a, pieces, st, e) : launch_norm_grad_rows<T, W, false>(a, pieces, st, e))) {}
    else if (wide && pieces <= 512 * 32 / V) e = enqueue(between ? rms_norm_grad_wide_kernel<T, W, true> : rms_norm_grad_wide_kernel<T, W, false>, dim3(a.blocks), 512, 0, 1, st, a);
    else e = enqueue(rms_norm_grad_long_kernel<T, W>, dim3(a.blocks), 512, 0, 1, st, a);
    if (a.dweight && e == cudaSuccess) e = enqueue(rms_norm_grad_weight_kernel<W>, dim3(uint32_t((a.cols + 31) / 32)), 1024, 0, 1, st, a);
    return e;
}

// Where a wait inside a kernel gave up, per device: read by ptwm_b200_operator_status.
__device__ uint32_t g_operator_status;

struct PerDevice { uint32_t* status = nullptr; bool attributes = false; };
std::mutex g_devices_mu;
std::map<int, PerDevice> g_devices;

// Once per device, with that device current.
int64_t device_of(int device, PerDevice* out) {
    std::lock_guard<std::mutex> g(g_devices_mu);
    PerDevice& d = g_devices[device];
    if (!d.attributes) {
        void* p = nullptr;
        CUDA_TRY(cudaGetSymbolAddress(&p, g_operator_status));
        d.status = static_cast<uint32_t*>(p);
        CUDA_TRY(allow_few());
        for (const auto f : {matvec_tiles_kernel<false, false, false>, matvec_tiles_kernel<false, false, true>, matvec_tiles_kernel<false, true, false>, matvec_tiles_kernel<false, true, true>,
                             matvec_tiles_kernel<true, false, false>, matvec_tiles_kernel<true, false, true>, matvec_tiles_kernel<true, true, false>, matvec_tiles_kernel<true, true, true>})
            CUDA_TRY(cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, int(SMEM_MOST)));
        d.attributes = true;
    }
    *out = d;
    return 0;
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_tiled() {
    static const EncodeTiled f = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess) p = nullptr;
        return reinterpret_cast<EncodeTiled>(p);
    }();
    return f;
}

// Map of a 2-D tensor: rows of `inner` values `pitch` bytes apart, loaded in boxes.
int64_t tensor_map(CUtensorMap* map, CUtensorMapDataType type, CUtensorMapSwizzle swizzle, const void* p, uint64_t inner, uint64_t rows, uint64_t pitch, uint32_t box_inner, uint32_t box_rows) {
    const EncodeTiled encode = encode_tiled();
    if (!encode) return fail(PTWM_RC_CUDA, "the driver has no cuTensorMapEncodeTiled");
    const cuuint64_t dims[2] = {inner, rows}, strides[1] = {pitch};
    const cuuint32_t box[2] = {box_inner, box_rows}, steps[2] = {1, 1};
    const CUresult e = encode(map, type, 2, const_cast<void*>(p), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (e != CUDA_SUCCESS) return fail(PTWM_RC_CUDA, "cuTensorMapEncodeTiled: error " + std::to_string(int(e)));
    return 0;
}

// Whether one of these addresses is none for values of the type.
bool beside(uint32_t dtype, std::initializer_list<uint64_t> pointers) {
    const uint64_t size = dtype == DT_FP32 ? 4 : dtype == DT_E4M3 ? 1 : 2;
    return std::any_of(pointers.begin(), pointers.end(), [&](uint64_t p) { return p % size != 0; });
}

// How the tokens of a product reach the tensor cores: as they are, or as parts in scratch.
struct Parts { uint32_t parts; uint64_t pitch; uint64_t bytes; };
Parts parts_of(uint64_t x, uint64_t tokens, uint64_t contraction, uint32_t dtype) {
    const uint32_t parts = dtype == DT_FP32 ? 3 : dtype == DT_FP16 ? 2 : 1;
    if (dtype == DT_BF16 && x % 16 == 0 && contraction % 8 == 0) return {1, contraction, 0};
    const uint64_t pitch = (contraction + 7) / 8 * 8;
    return {parts, pitch, parts * tokens * pitch * 2};
}

int64_t scratch_fits(const Parts& p, uint64_t scratch, uint64_t scratch_bytes) {
    if (p.bytes > scratch_bytes || (p.bytes && !scratch)) return fail(PTWM_RC_BUFFER_TOO_SMALL, "matvec: scratch too small");
    if (p.bytes && scratch % 16) return fail(PTWM_RC_INVALID_INPUT, "matvec: scratch starts at a multiple of 16 bytes");
    return 0;
}

// How a product is cut into tiles.
struct TilesSplit { uint32_t tile_tokens, ranks, stages, together; };
TilesSplit tiles_split(uint64_t rows, uint64_t contraction, uint64_t tokens, uint32_t parts, bool grad, bool flush, uint32_t group) {
    constexpr uint32_t SMS = 148;
    // as few tiles of tokens as 256 columns (128 where a stage holds parts, or results are flushed) allow, all of a size
    static_assert(FLUSH_TOKENS == 128, "");
    const uint64_t most = parts == 1 && !flush ? 256 : 128, across = (tokens + most - 1) / most;
    const uint32_t tile_tokens = uint32_t(((tokens + across - 1) / across + 15) / 16 * 16);
    // two steps to a stage where that leaves room for three
    const uint32_t room = SMEM_MOST - tiles_smem(0, 0), together = 3 * tiles_stage(tile_tokens, parts, 2, grad) <= room ? 2 : 1;
    uint32_t stages = std::min<uint32_t>(MOST_STAGES, room / tiles_stage(tile_tokens, parts, together, grad));
    if (!grad) stages = std::min(stages, tiles_tmem_stages(tile_tokens, together, flush));
    // blocks of a cluster for a tile's contraction: rounds of blocks x (steps of one, and what a block costs besides, in steps)
    const uint64_t tiles = (rows + TILE_ROWS - 1) / TILE_ROWS * across, steps = (contraction + STEP - 1) / STEP, unit = grad ? together : group == 32 ? 8 : 4;
    uint32_t ranks = 1;
    uint64_t least = ~0ull;
    for (uint32_t r = 1; r <= 8; r *= 2) {
        const uint64_t units = (steps + unit - 1) / unit, rounds = (tiles * r + SMS - 1) / SMS;
        if (r > units) break;
        const uint64_t cost = rounds * ((units + r - 1) / r * unit + (r == 1 ? 8 : 12));
        if (cost < least) { least = cost; ranks = r; }
    }
    return {tile_tokens, ranks, stages, together};
}

// there: a call before this one has left the parts of the same tokens in the scratch.
template <bool GRAD>
int64_t launch_tiles(const ScaledMatrix& w, const TokenArgs& x, uint32_t x_dtype, uint32_t y_dtype, uint64_t scratch, uint64_t scratch_bytes, bool there, int device, const PerDevice& dev, cudaStream_t st) {
    const uint64_t rows = GRAD ? w.cols : w.rows, contraction = GRAD ? w.rows : w.cols;
    const Parts p = parts_of(reinterpret_cast<uintptr_t>(x.x), x.tokens, contraction, x_dtype);
    if (const int64_t rc = scratch_fits(p, scratch, scratch_bytes); rc < 0) return rc;
    const void* tokens = x.x;
    if (p.bytes) {
        auto* out = at<__nv_bfloat16>(scratch);
        const dim3 grid(uint32_t(x.tokens), uint32_t(std::min<uint64_t>((p.pitch + 2047) / 2048, 64)));
        const bool wide = contraction % 8 == 0 && aligned(x.x);
        cudaError_t e = cudaSuccess;
        if (there) {}
        else if (x_dtype == DT_E4M3) e = enqueue(token_parts_kernel<uint8_t>, grid, 256, 0, 1, st, x, contraction, out, uint32_t(p.pitch), x.tokens, wide);
        else with_type(x_dtype, [&](auto v) { e = enqueue(token_parts_kernel<decltype(v)>, grid, 256, 0, 1, st, x, contraction, out, uint32_t(p.pitch), x.tokens, wide); });
        CUDA_TRY(e);
        tokens = out;
    }
    const bool flush = y_dtype == DT_FP32;
    const TilesSplit split = tiles_split(rows, contraction, x.tokens, p.parts, GRAD, flush, w.group);
    TilesArgs t{rows, contraction, x.tokens, x.tokens, p.parts, split.tile_tokens, split.stages, split.together, std::min<uint32_t>(4, split.stages * split.together), y_dtype, w.global_scale,
                x.scaled == SCALE_ROW ? static_cast<const float*>(x.scales) : nullptr, x.y, dev.status};
    CUDA_TRY(cudaSetDevice(device));  // a thread that has launched nothing yet (autograd's) has no context, which the tensor maps want
    CUtensorMap values, scales, tmap;
    int64_t rc = tensor_map(&values, CU_TENSOR_MAP_DATA_TYPE_UINT8, CU_TENSOR_MAP_SWIZZLE_64B, w.values, w.cols / 2, w.rows, w.value_pitch, 64, GRAD ? STEP : TILE_ROWS);
    if (rc == 0) rc = tensor_map(&scales, CU_TENSOR_MAP_DATA_TYPE_UINT8, CU_TENSOR_MAP_SWIZZLE_NONE, w.scales, w.cols / w.group, w.rows, w.scale_pitch, 16, GRAD ? STEP : TILE_ROWS);
    if (rc == 0) rc = tensor_map(&tmap, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, CU_TENSOR_MAP_SWIZZLE_128B, tokens, contraction, p.parts * x.tokens, p.pitch * 2, STEP, t.tile_tokens);
    if (rc < 0) return rc;
    const dim3 grid(uint32_t((rows + TILE_ROWS - 1) / TILE_ROWS) * split.ranks, uint32_t((x.tokens + t.tile_tokens - 1) / t.tile_tokens));
    const uint32_t smem = std::max(TILES_LEAST_SMEM, tiles_smem(tiles_stage(t.tile_tokens, t.parts, t.together, GRAD), t.stages));
    const auto kernel = w.group == 32 ? flush ? matvec_tiles_kernel<GRAD, true, true> : matvec_tiles_kernel<GRAD, false, true>
                                      : flush ? matvec_tiles_kernel<GRAD, true, false> : matvec_tiles_kernel<GRAD, false, false>;
    CUDA_TRY(enqueue(kernel, grid, TILES_THREADS, smem, split.ranks, st, values, scales, tmap, t));
    return 0;
}

// `count` matrices of the same columns and kind of scales; x.y is not looked at.
int64_t launch_few(const ScaledMatrix* w, const uint64_t* y, uint32_t count, uint32_t tiles, const TokenArgs& x, const FewSplit& s, uint32_t x_dtype, uint32_t y_dtype, int device,
                   const PerDevice& dev, cudaStream_t st) {
    const uint32_t boxes = few_boxes(*w), tokens = uint32_t(x.tokens), clusters = s.blocks / s.ranks;
    FewArgs a{x.x, x.scales, {}, dev.status, w->cols, count, tokens, x.scaled, y_dtype, boxes / s.ranks, boxes % s.ranks, tiles / clusters, tiles % clusters,
              ((tiles + clusters - 1) / clusters + s.most - 1) / s.most, s.depth, few_pitch((boxes + s.ranks - 1) / s.ranks), s.most, s.lines, reinterpret_cast<uintptr_t>(x.x) % 16 == 0};
    CUDA_TRY(cudaSetDevice(device));  // a thread that has launched nothing yet (autograd's) has no context, which the tensor maps want
    FewMaps maps;
    uint32_t first = 0;
    for (uint32_t i = 0; i < count; ++i) {
        int64_t rc = tensor_map(&maps.values[i], CU_TENSOR_MAP_DATA_TYPE_UINT8, CU_TENSOR_MAP_SWIZZLE_128B, w[i].values, w[i].cols / 2, w[i].rows, w[i].value_pitch, BOX_COLS / 2, 16);
        if (rc == 0) rc = tensor_map(&maps.scales[i], CU_TENSOR_MAP_DATA_TYPE_UINT8, CU_TENSOR_MAP_SWIZZLE_128B, w[i].scales, w[i].cols / w[i].group, w[i].rows, w[i].scale_pitch, 128, count == 1 ? s.most * 16 : 16);
        if (rc < 0) return rc;
        a.m[i] = FewMatrix{w[i].global_scale, at<void>(y[i]), uint32_t(w[i].rows), first};
        first += few_tiles(w[i]);
    }
    cudaError_t e = cudaSuccess;
    with_few(x_dtype, tokens, w->group == 32, [&](auto f) { e = enqueue(f, dim3(s.blocks), FEW_WARPS * 32, s.smem, s.ranks, st, maps, a); });
    CUDA_TRY(e);
    return 0;
}

}  // namespace

extern "C" int64_t ptwm_b200_operator_status(uint32_t device) {
    return guarded([&]() -> int64_t {
        DeviceGuard guard{int(device)};
        if (guard.err != cudaSuccess) return fail(PTWM_RC_CUDA, std::string("cudaSetDevice: ") + cudaGetErrorString(guard.err));
        uint32_t v = 0;
        CUDA_TRY(cudaMemcpyFromSymbol(&v, g_operator_status, 4));
        return v;
    });
}

extern "C" int64_t ptwm_b200_rms_norm(uint64_t x, uint64_t residual, uint64_t weight, uint64_t h, uint64_t y, uint64_t scales, uint64_t rows, uint64_t cols,
                                      uint32_t dtype, uint32_t weight_dtype, uint32_t scaled, float eps, uint32_t device, uint64_t stream) {
    return guarded([&]() -> int64_t {
        if (!plain_type(dtype) || !plain_type(weight_dtype)) return fail(PTWM_RC_UNSUPPORTED, "rms_norm: x and weight are fp32, fp16 or bf16");
        if (scaled > SCALE_BLOCK) return fail(PTWM_RC_INVALID_INPUT, "rms_norm: unknown output scaling");
        if (!cols || (scaled == SCALE_BLOCK && cols % 32)) return fail(PTWM_RC_INVALID_INPUT, "rms_norm: rows must not be empty, and hold whole blocks of 32 for block scales");
        if (rows > 0x7FFFFFFFull || cols > NORM_COLS) return fail(PTWM_RC_UNSUPPORTED, "rms_norm: more than 2^31 - 1 rows or 2^30 columns");
        if (!rows) return 0;
        if (!x || !weight || !y || (residual && !h) || (scaled && !scales)) return fail(PTWM_RC_INVALID_INPUT, "rms_norm: null device pointer");
        if (beside(dtype, {x, residual, h, scaled ? 0 : y}) || beside(weight_dtype, {weight}) || (scaled == SCALE_ROW && scales % 4)) return fail(PTWM_RC_INVALID_INPUT, "rms_norm: a tensor lies beside its type's alignment");
        DeviceGuard guard{int(device)};
        if (guard.err != cudaSuccess) return fail(PTWM_RC_CUDA, std::string("cudaSetDevice: ") + cudaGetErrorString(guard.err));
        const NormArgs a{at<void>(x), at<void>(residual), at<void>(weight), at<void>(h), at<void>(y), at<void>(scales), rows, cols, eps};
        cudaError_t e;
        with_type(dtype, [&](auto t) { with_type(weight_dtype, [&](auto w) { e = launch_norm<decltype(t), decltype(w)>(a, scaled, stream_of(stream)); }); });
        CUDA_TRY(e);
        return 0;
    });
}

extern "C" uint64_t ptwm_b200_rms_norm_grad_scratch_bytes(uint64_t rows, uint64_t cols) { return grad_blocks(rows) * cols * 4; }

extern "C" int64_t ptwm_b200_rms_norm_grad(uint64_t h, uint64_t weight, uint64_t dy, uint64_t dh, uint64_t dx, uint64_t dweight, uint64_t scratch, uint64_t scratch_bytes,
                                           uint64_t rows, uint64_t cols, uint32_t dtype, uint32_t weight_dtype, float eps, uint32_t device, uint64_t stream) {
    return guarded([&]() -> int64_t {
        if (!plain_type(dtype) || !plain_type(weight_dtype)) return fail(PTWM_RC_UNSUPPORTED, "rms_norm_grad: tensors are fp32, fp16 or bf16");
        if (!cols || rows > 0x7FFFFFFFull || cols > NORM_COLS) return fail(PTWM_RC_UNSUPPORTED, "rms_norm_grad: rows of 1 to 2^30 values, at most 2^31 - 1 of them");
        if (rows && (!h || !weight || !dy || (!dx && !dweight))) return fail(PTWM_RC_INVALID_INPUT, "rms_norm_grad: null device pointer");
        if (rows && dweight && (!scratch || scratch_bytes < ptwm_b200_rms_norm_grad_scratch_bytes(rows, cols))) return fail(PTWM_RC_BUFFER_TOO_SMALL, "rms_norm_grad: scratch too small");
        if (beside(dtype, {h, dy, dh, dx}) || beside(weight_dtype, {weight, dweight}) || beside(DT_FP32, {scratch})) return fail(PTWM_RC_INVALID_INPUT, "rms_norm_grad: a tensor lies beside its type's alignment");
        DeviceGuard guard{int(device)};
        if (guard.err != cudaSuccess) return fail(PTWM_RC_CUDA, std::string("cudaSetDevice: ") + cudaGetErrorString(guard.err));
        if (!rows) {
            if (dweight) CUDA_TRY(cudaMemsetAsync(at<void>(dweight), 0, cols * (weight_dtype == DT_FP32 ? 4 : 2), stream_of(stream)));
            return 0;
        }
        const uint32_t blocks = grad_blocks(rows);
        const NormGradArgs a{at<void>(h), at<void>(weight), at<void>(dy), at<void>(dh), at<void>(dx), dweight ? at<float>(scratch) : nullptr, at<void>(dweight), rows, cols, eps, blocks};
        cudaError_t e;
        with_type(dtype, [&](auto t) { with_type(weight_dtype, [&](auto w) { e = launch_norm_grad<decltype(t), decltype(w)>(a, stream_of(stream)); }); });
        CUDA_TRY(e);
        return 0;
    });
}

extern "C" uint64_t ptwm_b200_matvec_scratch_bytes(const ptwm_b200_scaled_weight* w, uint64_t x, uint64_t tokens, uint32_t x_dtype, uint32_t grad) {
    ScaledMatrix m;
    if (matrix_of(w, &m) < 0 || (!grad && few_split(m, few_tiles(m), tokens, x_dtype).depth)) return 0;
    return parts_of(x, tokens, grad ? m.rows : m.cols, x_dtype).bytes;
}

extern "C" int64_t ptwm_b200_matvec_group(const ptwm_b200_scaled_weight* const* weights, const uint64_t* y, uint32_t count, uint64_t x, uint64_t x_scales, uint64_t tokens,
                                          uint32_t x_dtype, uint32_t x_scaled, uint32_t y_dtype, uint64_t scratch, uint64_t scratch_bytes, uint32_t device, uint64_t stream) {
    return guarded([&]() -> int64_t {
        ScaledMatrix w[FEW_MATRICES];
        if (!weights || !y || !count) return fail(PTWM_RC_INVALID_INPUT, "matvec: no matrix");
        if (count > FEW_MATRICES) return fail(PTWM_RC_UNSUPPORTED, "matvec: more than 4 matrices in a call");
        uint64_t tiles = 0;
        for (uint32_t i = 0; i < count; ++i) {
            if (const int64_t rc = matrix_of(weights[i], &w[i]); rc < 0) return rc;
            if (w[i].cols != w[0].cols) return fail(PTWM_RC_INVALID_INPUT, "matvec: matrices of a call have the same columns");
            tiles += few_tiles(w[i]);
        }
        if (!plain_type(y_dtype)) return fail(PTWM_RC_UNSUPPORTED, "matvec: the output is fp32, fp16 or bf16");
        if (x_dtype == DT_E4M3 ? x_scaled != SCALE_ROW && x_scaled != SCALE_BLOCK : !plain_type(x_dtype) || x_scaled)
            return fail(PTWM_RC_UNSUPPORTED, "matvec: tokens are fp32, fp16, bf16, or E4M3 with scales per row or block");
        if (x_scaled == SCALE_BLOCK && w[0].cols % 32) return fail(PTWM_RC_INVALID_INPUT, "matvec: block scales need whole blocks of 32 columns");
        if (tokens > (1u << 19)) return fail(PTWM_RC_UNSUPPORTED, "matvec: more than 2^19 tokens in a call");
        if (!tokens) return 0;
        if (!x || (x_scaled && !x_scales)) return fail(PTWM_RC_INVALID_INPUT, "matvec: null device pointer");
        for (uint32_t i = 0; i < count; ++i)
            if (!y[i]) return fail(PTWM_RC_INVALID_INPUT, "matvec: null device pointer");
            else if (beside(y_dtype, {y[i]})) return fail(PTWM_RC_INVALID_INPUT, "matvec: a tensor lies beside its type's alignment");
        if (beside(x_dtype, {x}) || (x_scaled == SCALE_ROW && x_scales % 4)) return fail(PTWM_RC_INVALID_INPUT, "matvec: a tensor lies beside its type's alignment");
        // one split for all, or one for each; what scratch they want is looked at before anything is launched
        bool alike = true;
        for (uint32_t i = 1; i < count; ++i) alike &= w[i].group == w[0].group;
        const FewSplit all = alike ? few_split(w[0], uint32_t(tiles), tokens, x_dtype) : FewSplit{};
        FewSplit each[FEW_MATRICES] = {};
        if (!all.depth) {
            bool in_tiles = count == 1;
            if (count > 1)
                for (uint32_t i = 0; i < count; ++i) {
                    each[i] = few_split(w[i], few_tiles(w[i]), tokens, x_dtype);
                    in_tiles |= !each[i].depth;
                }
            if (in_tiles)
                if (const int64_t rc = scratch_fits(parts_of(x, tokens, w[0].cols, x_dtype), scratch, scratch_bytes); rc < 0) return rc;
        }
        DeviceGuard guard{int(device)};
        if (guard.err != cudaSuccess) return fail(PTWM_RC_CUDA, std::string("cudaSetDevice: ") + cudaGetErrorString(guard.err));
        TokenArgs t{at<void>(x), at<void>(x_scales), tokens, x_scaled, nullptr};
        PerDevice dev;
        if (const int64_t rc = device_of(int(device), &dev); rc < 0) return rc;
        if (all.depth) return launch_few(w, y, count, uint32_t(tiles), t, all, x_dtype, y_dtype, int(device), dev, stream_of(stream));
        bool there = false;
        for (uint32_t i = 0; i < count; ++i) {
            const FewSplit& s = each[i];
            t.y = at<void>(y[i]);
            const int64_t rc = s.depth ? launch_few(&w[i], y + i, 1, few_tiles(w[i]), t, s, x_dtype, y_dtype, int(device), dev, stream_of(stream))
                                       : launch_tiles<false>(w[i], t, x_dtype, y_dtype, scratch, scratch_bytes, there, int(device), dev, stream_of(stream));
            if (rc < 0) return rc;
            there |= !s.depth;
        }
        return 0;
    });
}

extern "C" int64_t ptwm_b200_matvec(const ptwm_b200_scaled_weight* weight, uint64_t x, uint64_t x_scales, uint64_t y, uint64_t tokens, uint32_t x_dtype, uint32_t x_scaled,
                                    uint32_t y_dtype, uint64_t scratch, uint64_t scratch_bytes, uint32_t device, uint64_t stream) {
    return ptwm_b200_matvec_group(&weight, &y, 1, x, x_scales, tokens, x_dtype, x_scaled, y_dtype, scratch, scratch_bytes, device, stream);
}

extern "C" int64_t ptwm_b200_matvec_grad_of(const ptwm_b200_scaled_weight* weight, uint64_t dy, uint64_t dx, uint64_t tokens, uint32_t dy_dtype, uint32_t dx_dtype, uint64_t scratch,
                                            uint64_t scratch_bytes, uint32_t device, uint64_t stream) {
    return guarded([&]() -> int64_t {
        ScaledMatrix w;
        if (const int64_t rc = matrix_of(weight, &w); rc < 0) return rc;
        if (!plain_type(dy_dtype) || !plain_type(dx_dtype)) return fail(PTWM_RC_UNSUPPORTED, "matvec_grad: gradients are fp32, fp16 or bf16");
        if (tokens > (1u << 19)) return fail(PTWM_RC_UNSUPPORTED, "matvec_grad: more than 2^19 tokens in a call");
        if (!tokens) return 0;
        if (!dy || !dx) return fail(PTWM_RC_INVALID_INPUT, "matvec_grad: null device pointer");
        if (beside(dy_dtype, {dy}) || beside(dx_dtype, {dx})) return fail(PTWM_RC_INVALID_INPUT, "matvec_grad: a tensor lies beside its type's alignment");
        DeviceGuard guard{int(device)};
        if (guard.err != cudaSuccess) return fail(PTWM_RC_CUDA, std::string("cudaSetDevice: ") + cudaGetErrorString(guard.err));
        const TokenArgs t{at<void>(dy), nullptr, tokens, SCALE_NONE, at<void>(dx)};
        PerDevice dev;
        if (const int64_t rc = device_of(int(device), &dev); rc < 0) return rc;
        return launch_tiles<true>(w, t, dy_dtype, dx_dtype, scratch, scratch_bytes, false, int(device), dev, stream_of(stream));
    });
}

extern "C" int64_t ptwm_b200_matvec_grad(const ptwm_b200_scaled_weight* weight, uint64_t dy, uint64_t dx, uint64_t tokens, uint32_t dtype, uint64_t scratch, uint64_t scratch_bytes,
                                         uint32_t device, uint64_t stream) {
    return ptwm_b200_matvec_grad_of(weight, dy, dx, tokens, dtype, dtype, scratch, scratch_bytes, device, stream);
}
