#pragma once
// Weight gradient of a linear layer from 8-bit operands:  dW[n, k] (+)= sum over tokens m of dy[m, n] * x[m, k], for one matrix or for
// every group of tokens (expert) its own.
//
//   1. block_cast_tokens_kernel: both bf16 operands -> e4m3 codes, in the order they have, with one power of two per feature and block
//      of 128 tokens, e the smallest integer with amax <= 448 * 2^e.  A block that ends a group is filled up with zeros.
//   2. fp8_wgrad_kernel: persistent, warp-specialised tcgen05 products of tiles of dW by pairs of CTAs, summed over the tokens in tensor
//      memory.  The tensor core transposes the token-major operands and multiplies the scales in, so that nothing has to be promoted.

#include <cstdint>
#include <type_traits>
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include "../gemm/fp8_gemm.cuh"
#include "block_scaled.cuh"
#include "token_groups.cuh"

namespace yan {

// ---------------------------------------------------------------------------------------------
// codes and scales
// ---------------------------------------------------------------------------------------------
struct CastTokensOperand {
    const __nv_bfloat16* z = nullptr;  // [rows][ld]
    uint64_t ld = 0;
    uint32_t cols = 0;
    uint32_t wide = 0;         // rows start on 32-byte boundaries and have whole groups of 16 columns
    uint8_t* codes = nullptr;  // [blocks * 128][codes_ld], codes_ld a multiple of 16
    uint32_t codes_ld = 0;
    uint8_t* scales = nullptr;  // [quads][ceil(cols / scale_cols)][ceil(scale_cols / 128)] scale tiles
    uint32_t scale_cols = 128;  // columns of one tile of products
};

struct CastTokensParams {
    TokenGroups groups;
    uint32_t max_blocks = 0;
    CastTokensOperand operand[2];
    uint32_t column_tiles[2] = {0, 0};
    uint32_t* counters = nullptr;  // cleared for the products' joined slices
    uint32_t num_counters = 0;
};

namespace detail {

// The scale byte e + 127 of a largest magnitude given as bf16 bits: the smallest e with amax <= 448 * 2^e = 1.75 * 2^(e + 8); 255 (NaN)
// for what is not finite.
__device__ __forceinline__ uint32_t scale_byte_of_amax(uint32_t bits) {
    const int e = static_cast<int>(bits >> 7) - 8 + ((bits & 0x7Fu) > 0x60u ? 1 : 0);
    return bits >= 0x7F80u ? 255u : static_cast<uint32_t>(max(e, 0));
}
__device__ __forceinline__ float inverse_of_scale(uint32_t byte) { return __uint_as_float((254u - min(byte, 253u)) << 23); }

__device__ __forceinline__ uint32_t quantize4(uint32_t lo, uint32_t hi, const float (&inv)[4]) {
    const float a = __uint_as_float(lo << 16) * inv[0], b = __uint_as_float(lo & 0xFFFF0000u) * inv[1];
    const float c = __uint_as_float(hi << 16) * inv[2], d = __uint_as_float(hi & 0xFFFF0000u) * inv[3];
    const uint32_t x = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t y = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return x | (y << 16);
}

}  // namespace detail

// One CTA of 256 threads: 128 tokens x 128 columns of one operand.  Eight threads share a row, 16 columns each; 32 rows at a time.  Bound by
// HBM (3 bytes per element): 8192 x (28672 + 8192) in 139 us, 6.5 TB/s.
template <bool kAllWide>
__global__ void __launch_bounds__(256) block_cast_tokens_kernel(const CastTokensParams p) {
    __shared__ TokenBlockTable table;
    __shared__ uint4 s_max[8][16];  // [warp][8 columns as packed bf16 magnitudes]
    __shared__ uint8_t s_scale[128];
    __shared__ __align__(16) uint16_t s_tile[kAllWide ? 1 : 128 * 128];
    ptx::grid_dependency_wait();
    // The products take the SMs as this kernel leaves them, and wait for its end before they read anything.
    ptx::grid_dependency_launch_dependents();
    const uint32_t block = blockIdx.y, second = blockIdx.x >= p.column_tiles[0] ? 1u : 0u;
    const uint32_t tile = blockIdx.x - (second != 0 ? p.column_tiles[0] : 0u);
    const CastTokensOperand& op = p.operand[second];
    const uint32_t thread = threadIdx.x, warp = thread / 32, lane = thread % 32;
    if (blockIdx.y == 0)
        for (uint32_t i = blockIdx.x * 256 + thread; i < p.num_counters; i += gridDim.x * 256) p.counters[i] = 0;

    uint32_t row0 = block * 128, rows = 0, quad = block / 4, byte = block % 4;
    if (p.groups.sizes == nullptr) {
        rows = min(p.groups.rows - row0, 128u);
    } else {
        if (warp == 0) build_token_blocks(p.groups, p.max_blocks, table);
        __syncthreads();
        if (block >= table.block[p.groups.num_groups]) return;
        const uint32_t g = group_of_block(table, p.groups.num_groups, block), in_group = block - table.block[g];
        row0 = group_start(p.groups, g) + in_group * 128;
        rows = min(group_size(p.groups, g) - in_group * 128, 128u);
        quad = table.quad[g] + in_group / 4;
        byte = in_group % 4;
    }

    const uint32_t octet = thread % 8, first_row = thread / 8, col = tile * 128 + octet * 16;
    uint4 v[4][2];
    if (kAllWide || op.wide != 0) {
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            const uint32_t r = first_row + 32 * i;
            v[i][0] = v[i][1] = make_uint4(0, 0, 0, 0);
            if (r < rows && col < op.cols) ptx::ld_global_32(v[i], op.z + static_cast<uint64_t>(row0 + r) * op.ld + col);
        }
    } else if constexpr (!kAllWide) {
        // Any alignment: an element per lane, through shared memory.
        const uint32_t c = thread % 128, column = tile * 128 + c, there = column < op.cols ? rows : 0u;
        const uint16_t* src = reinterpret_cast<const uint16_t*>(op.z) + static_cast<uint64_t>(row0 + thread / 128) * op.ld + column;
#pragma unroll 16
        for (uint32_t r = thread / 128; r < 128; r += 2, src += 2 * op.ld)
            s_tile[r * 128 + c] = r < there ? static_cast<uint16_t>(ptx::ld_global_u16(src)) : uint16_t(0);
        __syncthreads();
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            const uint4* from = reinterpret_cast<const uint4*>(s_tile + (first_row + 32 * i) * 128 + octet * 16);
            v[i][0] = from[0];
            v[i][1] = from[1];
        }
    }
    uint32_t m[8];
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) {
        m[j] = 0;
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) m[j] = __vmaxu2(m[j], reinterpret_cast<const uint32_t*>(v[i])[j] & 0x7FFF7FFFu);
        m[j] = __vmaxu2(m[j], __shfl_xor_sync(0xffffffffu, m[j], 8));
        m[j] = __vmaxu2(m[j], __shfl_xor_sync(0xffffffffu, m[j], 16));
    }
    if (lane < 8) {
        s_max[warp][lane * 2] = make_uint4(m[0], m[1], m[2], m[3]);
        s_max[warp][lane * 2 + 1] = make_uint4(m[4], m[5], m[6], m[7]);
    }
    __syncthreads();
    if (thread < 128) {
        uint32_t amax = 0;
#pragma unroll
        for (uint32_t w = 0; w < 8; ++w) amax = max(amax, static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(s_max[w])[thread]));
        const uint32_t scale = detail::scale_byte_of_amax(amax), c = tile * 128 + thread, in_tile = c % op.scale_cols;
        s_scale[thread] = static_cast<uint8_t>(scale);
        if (c < op.cols)
            op.scales[((static_cast<uint64_t>(quad) * ceil_div(op.cols, op.scale_cols) + c / op.scale_cols) * ceil_div(op.scale_cols, 128u) +
                       in_tile / 128) * kScaleTileBytes + scale_tile_offset(in_tile % 128, byte)] = static_cast<uint8_t>(scale);
    }
    __syncthreads();
    if (col >= op.codes_ld) return;
    float inv[4][4];
#pragma unroll
    for (uint32_t j = 0; j < 16; ++j) inv[j / 4][j % 4] = detail::inverse_of_scale(s_scale[octet * 16 + j]);
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
        uint4 q;
        q.x = detail::quantize4(v[i][0].x, v[i][0].y, inv[0]);
        q.y = detail::quantize4(v[i][0].z, v[i][0].w, inv[1]);
        q.z = detail::quantize4(v[i][1].x, v[i][1].y, inv[2]);
        q.w = detail::quantize4(v[i][1].z, v[i][1].w, inv[3]);
        *reinterpret_cast<uint4*>(op.codes + static_cast<uint64_t>(block * 128 + first_row + 32 * i) * op.codes_ld + col) = q;
    }
}

// ---------------------------------------------------------------------------------------------
// products
// ---------------------------------------------------------------------------------------------
struct WgradParams {
    TokenGroups groups;
    uint32_t max_blocks = 0;
    uint32_t n = 0, k = 0;                // sides of dW
    void* out = nullptr;                  // [groups][n][out_ld]
    uint64_t out_ld = 0, out_group = 0;   // elements
    uint32_t accumulate = 0;
    uint32_t tiles = 0, whole_tiles = 0;  // all of them; those that are dealt out one by one (see WgradSchedule)
    uint32_t store_cost = 0;              // k-blocks that take as long as storing a tile
    float4* partials = nullptr;           // [2 * pairs][2 CTAs][8 warps][columns of a warp / 4][32 lanes]
    uint32_t* counters = nullptr;         // [pairs][2 CTAs][8 warps], zero
    int* status = nullptr;
    unsigned long long timeout_ns = 0;
};

// Who computes what.  Tiles are numbered group by group, within a group in bands of eight tile rows, so that pairs at work at the same time
// share what they read.  The first whole_tiles of them, a multiple of the pairs, are dealt out in turn.  The rest, less than two waves,
// is shared evenly: laid end to end, a tile as long as its k-blocks or as its store takes, whichever is more, and cut into one
// stretch per pair.  A cut through the k-blocks of a tile goes to a multiple of four of them; tiles of fewer than kMinCut go whole to
// the pair in whose stretch they begin.
struct WgradSchedule {
    TokenBlockTable blocks;
    uint32_t length[kMaxTokenGroups + 1];  // of all tiles in front of a group
    uint32_t origin, rest;                 // where the shared tiles begin, and their length
    uint32_t stretches, shortest, longer;  // the first `longer` stretches are one longer than `shortest`
};

// A pair of CTAs computes 256 x kCols of dW at a time (64, 128, 192 or 256: choose_wgrad_cols), each CTA 128 rows of it: per 128 tokens it
// loads 128 rows of A and the box of B that holds its kCols / 2 columns, where a CTA by itself would need all kCols.  What bounds long
// sums is the power limit (1.28 GHz at N=28672 K=8192), so that bytes moved per product count more than cycles.  Quantization and
// products together take 1.66 ms there; when the tiles were chosen it was 1.74 with pairs and 256 columns, 1.81 with 192 (whose two
// accumulators lie side by side, so that nothing ever waits for sums to be read), 2.12 with 224, 1.95 with single CTAs of 128 x 256.
constexpr uint32_t kWgradRows = 256;
// Parts of a tile that meet in L2 cost about as much as twelve k-blocks (us with the shortest tile that is cut and the shortest stretch at
// 16 and 8, 24 and 12, 32 and 16 k-blocks: 2048 tokens N=1024 K=512 12.9, 11.3, 11.3; 3000 tokens N=2048 K=1024 22.4, 22.5, 16.8; 4096
// tokens N=K=1024 21.9, 18.7, 18.7; 3888 tokens N=K=128 12.8, 13.1, 13.6).
constexpr uint32_t kWgradMinCut = 32, kWgradMinStretch = 16, kWgradMaxStoreCost = 20;

// kOldItem: bytes of an element of dW whose old values are fetched ahead of the store that adds to them, or 0.  They wait in shared memory, and what
// counts is how many bytes are on their way; stages of products make room (us for fp32 in 16 experts N=4096 K=2048, 16384 tokens: added in L2
// 350; two boxes of a warp fetched ahead at five stages 345, four at four 300, six at three 287 but slower elsewhere; 8192 tokens
// N=7168 K=2048, where products count: 131, 131, 138, 156.  bf16, old values in registers a box ahead at six stages, four boxes at five
// and six at four: 326, 273 and 290; 126, 128 and 138).
template <uint32_t kCols, uint32_t kOldItem>
struct WgradTile {
    static constexpr uint32_t kStages = kOldItem == 0 ? 6 : kOldItem == 2 ? 5 : 4;
    // k-blocks that are summed in tensor memory before the sums move to registers.  An addition there rounds towards zero: 8192 tokens of
    // uneven size, relative error 1.3e-6 in one chain of 64 k-blocks, 5e-7 in chains of 32, 2.2e-7 in chains of 16.  Where the
    // accumulators share columns the products wait at the end of a chain: N=28672 K=8192, 8192 tokens, 1.72, 1.74 and 1.85 ms
    // (1.66 with 32 now).
    static constexpr uint32_t kChain = kCols <= 192 ? 16 : 32;
    static constexpr uint32_t kStageA = kMnBoxBytes, kStageB = kMnBoxBytes;
    static constexpr uint32_t kScaleTiles = 1 + ceil_div(kCols, 128u);
    static constexpr uint32_t kStageScales = kScaleTiles * kScaleTileBytes;
    static constexpr uint32_t kOffA = 0, kOffB = kOffA + kStages * kStageA, kOffScales = kOffB + kStages * kStageB;
    static constexpr uint32_t kBoxBytes = 16 * 128;  // output staging, one box per warp
    static constexpr uint32_t kOffStore = kOffScales + kStages * kStageScales;
    static constexpr uint32_t kOldBoxes = kOldItem == 0 ? 0 : 4, kOldBoxBytes = 16 * 32 * kOldItem;
    static constexpr uint32_t kOffOld = kOffStore + 8 * kBoxBytes;
    static constexpr uint32_t kOffSchedule = kOffOld + 8 * kOldBoxes * kOldBoxBytes;
    static constexpr uint32_t kOffBarriers = align_up(kOffSchedule + static_cast<uint32_t>(sizeof(WgradSchedule)), 8u);
    static constexpr uint32_t kNumBarriers = 2 * kStages + 6;
    static constexpr uint32_t kOffTmemSlot = kOffBarriers + kNumBarriers * 8, kOffAbort = kOffTmemSlot + 4;
    static constexpr uint32_t kSmemSize = kOffAbort + 4 + 1024;
    static constexpr uint32_t kWarpCols = kCols / 2;  // columns of a warp that reads sums
    // tensor memory: two accumulators, then three sets of scales.  Where they do not fit side by side the accumulators share kShared
    // columns, the last of the first and the first of the second, which are read before the others and handed on by themselves.
    static constexpr uint32_t kTmemCols = 512, kTmemScaleSet = kScaleTiles * 4;
    static constexpr uint32_t kShared = 2 * kCols + 3 * kTmemScaleSet <= kTmemCols ? 0 : align_up(2 * kCols + 3 * kTmemScaleSet - kTmemCols, 16u);
    static constexpr uint32_t kTmemSecond = kCols - kShared, kTmemScales = kTmemSecond + kCols;
    static_assert(kCols % 32 == 0 && kTmemScales + 3 * kTmemScaleSet <= kTmemCols && kShared <= kWarpCols);
    static_assert(kSmemSize <= 232448);
    static_assert(kStages <= 6 && kOldBoxes <= kWarpCols / 16);
    static_assert(kChain % 4 == 0 && kWgradMinCut % 4 == 0 && kWgradMinStretch >= 8);
};

namespace detail {

template <uint32_t kCols>
__device__ __forceinline__ uint32_t wgrad_tiles_per_group(const WgradParams& p) {
    return ceil_div(p.n, kWgradRows) * ceil_div(p.k, kCols);
}
// Length of a tile with so many k-blocks.  Nothing is left to do for an empty group that is added.
__device__ __forceinline__ uint32_t wgrad_length(const WgradParams& p, uint32_t blocks) {
    return blocks == 0 && p.accumulate != 0 ? 0u : max(blocks, p.store_cost);
}

// Called by one whole warp.
template <uint32_t kCols>
__device__ __forceinline__ void build_wgrad_schedule(const WgradParams& p, WgradSchedule& s) {
    build_token_blocks(p.groups, p.max_blocks, s.blocks);
    const uint32_t lane = ptx::lane_id(), per_group = wgrad_tiles_per_group<kCols>(p);
    uint32_t at = 0;
    for (uint32_t first = 0; first < p.groups.num_groups; first += 32) {
        const uint32_t g = first + lane;
        const uint32_t own = g < p.groups.num_groups ? per_group * wgrad_length(p, s.blocks.block[g + 1] - s.blocks.block[g]) : 0u;
        uint32_t until = own;
#pragma unroll
        for (uint32_t off = 1; off < 32; off *= 2) {
            const uint32_t v = __shfl_up_sync(0xffffffffu, until, off);
            if (lane >= off) until += v;
        }
        if (g < p.groups.num_groups) s.length[g] = at + until - own;
        at += __shfl_sync(0xffffffffu, until, 31);
    }
    __syncwarp();
    if (lane == 0) {
        s.length[p.groups.num_groups] = at;
        const uint32_t g = p.whole_tiles / per_group;
        s.origin = at;
        if (g < p.groups.num_groups)
            s.origin = s.length[g] + p.whole_tiles % per_group * wgrad_length(p, s.blocks.block[g + 1] - s.blocks.block[g]);
        s.rest = at - s.origin;
        // no more than pairs, or stretches of kWgradMinStretch, unless there are as many tiles; all of at least four k-blocks
        s.stretches = max(min(gridDim.x / 2, max(s.rest / kWgradMinStretch, min(p.tiles - p.whole_tiles, s.rest / 4))), 1u);
        s.shortest = s.rest / s.stretches;
        s.longer = s.rest % s.stretches;
    }
}

// What a pair computes at a time: k-blocks [begin, begin + count) of a group, of `blocks`, for one tile of its dW.
struct WgradUnit {
    uint32_t group, row0, col0;        // row0, col0: features of the tile's corner
    uint32_t block0, quad0;            // the group's first k-block and quad of scales
    uint32_t begin, count, blocks;
    uint32_t first_pair, last_pair;    // who shares the tile
};

// The pair's units one after the other; every role of both CTAs walks them.
template <uint32_t kCols>
struct WgradWalk {
    uint32_t pair, pairs;
    uint32_t tile, group, in_group;  // next of the dealt tiles: its number, its group and its number there
    uint32_t at, end;                // what is left of the pair's stretch

    __device__ __forceinline__ explicit WgradWalk(const WgradSchedule& s)
        : pair(blockIdx.x / 2), pairs(gridDim.x / 2), tile(blockIdx.x / 2), group(0), in_group(blockIdx.x / 2) {
        at = pair < s.stretches ? s.origin + pair * s.shortest + min(pair, s.longer) : 0u;
        end = pair < s.stretches ? at + s.shortest + (pair < s.longer ? 1u : 0u) : 0u;
    }

    __device__ __forceinline__ static void place(const WgradParams& p, const WgradSchedule& s, uint32_t group, uint32_t in_group, WgradUnit& u) {
        const uint32_t tiles_n = ceil_div(p.n, kWgradRows), tiles_k = ceil_div(p.k, kCols);
        const uint32_t band = in_group / (8 * tiles_k), in_band = in_group - band * (8 * tiles_k), rows = min(8u, tiles_n - band * 8);
        const uint32_t column = rows == 8 ? in_band / 8 : in_band / rows;
        u.group = group;
        u.row0 = (band * 8 + in_band - column * rows) * kWgradRows;
        u.col0 = column * kCols;
        u.block0 = s.blocks.block[group];
        u.quad0 = s.blocks.quad[group];
        u.blocks = s.blocks.block[group + 1] - u.block0;
    }
    // The pair in whose stretch a position lies.
    __device__ __forceinline__ static uint32_t owner(const WgradSchedule& s, uint32_t position) {
        const uint32_t x = position - s.origin, in_longer = s.longer * (s.shortest + 1);
        return x < in_longer ? x / (s.shortest + 1) : s.longer + (x - in_longer) / s.shortest;
    }

    __device__ __forceinline__ bool next(const WgradParams& p, const WgradSchedule& s, WgradUnit& u) {
        const uint32_t per_group = wgrad_tiles_per_group<kCols>(p);
        if (tile < p.whole_tiles) {
            while (in_group >= per_group) in_group -= per_group, ++group;
            place(p, s, group, in_group, u);
            u.begin = 0, u.count = u.blocks;
            u.first_pair = u.last_pair = pair;
            tile += pairs;
            in_group += pairs;
            return true;
        }
        while (at < end) {
            uint32_t low = 0, high = p.groups.num_groups;  // length[low] <= at < length[high]
            while (high - low > 1) {
                const uint32_t mid = (low + high) / 2;
                if (s.length[mid] <= at) low = mid;
                else high = mid;
            }
            const uint32_t blocks = s.blocks.block[low + 1] - s.blocks.block[low], length = wgrad_length(p, blocks);
            const uint32_t in_group = (at - s.length[low]) / length, start = s.length[low] + in_group * length;
            const uint32_t from = at - start;  // above zero only in the tile that the stretch begins in
            const uint32_t until = end - start;
            at = start + length;
            place(p, s, low, in_group, u);
            if (blocks < kWgradMinCut) {
                if (from != 0) continue;
                u.begin = 0, u.count = blocks;
                u.first_pair = u.last_pair = pair;
                return true;
            }
            u.begin = from >= blocks ? blocks : from & ~3u;
            u.count = (until >= blocks ? blocks : until & ~3u) - u.begin;
            if (u.count == 0) continue;
            u.first_pair = owner(s, start + 3);  // a stretch that ends in the first three k-blocks has none of them
            u.last_pair = owner(s, start + blocks - 1);
            return true;
        }
        return false;
    }
};

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    const __nv_bfloat162 t = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&t);
}

__device__ __forceinline__ void red_add(float* p, float v) { asm volatile("red.global.add.f32 [%0], %1;" ::"l"(p), "f"(v) : "memory"); }
__device__ __forceinline__ void red_add4(float* p, const float4& v) {
    asm volatile("red.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(p), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}

// The old values of dW on their way to a warp that adds them (fp32, vectors): boxes of 16 rows x 32 columns in the order in which they
// are stored are fetched into shared memory several boxes ahead, across the end of a tile, each lane the vectors that it adds itself.
template <typename out_t>
struct WgradOldRows {
    const out_t* from;  // this lane's vector in the first of its rows, which are four apart, and the leftmost 32 columns
    uint32_t rows;      // rows of the tile that dW has; zero where nothing is fetched
    uint32_t col;

    // Only what no other pair adds to, and if there is something to add.
    __device__ __forceinline__ static bool fetched(const WgradUnit& u) { return u.first_pair == u.last_pair && u.blocks != 0; }
    __device__ __forceinline__ WgradOldRows(const WgradParams& p, const WgradUnit& u, bool exists, uint32_t row_in_tile, uint32_t leftmost,
                                            uint32_t lane) {
        const uint32_t row0 = u.row0 + row_in_tile;
        rows = exists && fetched(u) && row0 < p.n ? min(p.n - row0, 32u) : 0u;
        col = u.col0 + leftmost + lane % 8 * 4;
        from = static_cast<const out_t*>(p.out) + u.group * p.out_group + static_cast<uint64_t>(row0 + lane / 8) * p.out_ld + col;
    }
    // One group of copies, whether there is something to fetch or not.
    __device__ __forceinline__ void fetch(const WgradParams& p, uint32_t number, uint32_t direction, uint32_t box, uint32_t lane) const {
        const uint32_t rows16 = number % 2;
        const int right = static_cast<int>(32 * direction * (number / 2));
        if (col + right < p.k) {
#pragma unroll
            for (uint32_t i = rows16 * 4; i < rows16 * 4 + 4; ++i)
                if (i * 4 + lane / 8 < rows) {
                    const out_t* src = from + i * 4 * p.out_ld + right;
                    if constexpr (sizeof(out_t) == 4) ptx::cp_async_16(box + (i % 4 * 32 + lane) * 16, src);
                    else ptx::cp_async_8(box + (i % 4 * 32 + lane) * 8, src);
                }
        }
        ptx::cp_async_commit();
    }
};

// The boxes of a warp in turn.
template <uint32_t kBoxes, uint32_t kBytes>
struct WgradOldRing {
    uint32_t first, now;
    __device__ __forceinline__ void advance() { now = now + kBytes == first + kBoxes * kBytes ? first : now + kBytes; }
    template <typename out_t>
    __device__ __forceinline__ void fill(const WgradParams& p, const WgradOldRows<out_t>& rows, uint32_t direction, uint32_t lane) {
#pragma unroll
        for (uint32_t i = 0; i < kBoxes; ++i, advance()) rows.fetch(p, i, direction, now, lane);
    }
};

// Stores a warp's 32 rows x kWarpCols columns; lane r holds row r, acc[c] column first_col + c / 16 * 16 * direction + c % 16.  They go
// through the warp's box in shared memory, 16 rows x 32 columns in fp32 at a time, so that a store instruction covers four pieces of 128
// contiguous bytes (kVector; otherwise one, an element per lane).  16-byte chunk j of box row r is at chunk j ^ r % 8.
// What bounds it is the number of pieces: an SM sends one in two cycles, whatever its size (pieces of 64 bytes: 6400 cycles for the 128 x 256
// of a CTA).
// What dW holds is fetched ahead (kOldBoxes), or fp32 is added to it where it lies, in L2: every element once, so that the order does not
// matter, and nothing waits for the old value.  The sum is the same.  (16 experts N=4096 K=2048, 16384 tokens: loads and stores at the end
// of a tile took twice as long as adding in L2, old values in registers a pass ahead 1.1 times: few of them are on their way at a time.)
// bf16 is added in 32 bits and rounded once.
template <typename out_t, uint32_t kWarpCols, bool kVector, uint32_t kOldBoxes = 0, typename Ring = int>
__device__ __forceinline__ void store_wgrad_rows(const WgradParams& p, const WgradUnit& u, uint32_t box, uint32_t row_in_tile, uint32_t first_col,
                                                 uint32_t direction, uint32_t lane, const float (&acc)[kWarpCols],
                                                 [[maybe_unused]] Ring* ring = nullptr, [[maybe_unused]] const WgradOldRows<out_t>* after = nullptr) {
    static_assert(kWarpCols % 32 == 0);
    const uint32_t row0 = u.row0 + row_in_tile;
    if (row0 >= p.n) return;
    const uint32_t rows = min(p.n - row0, 32u);
    // the leftmost of 32 columns, and where its pieces meet this lane: column lane_col of rows lane_row + kRowStep i
    constexpr uint32_t kRowStep = kVector ? 4 : 1;
    const uint32_t lane_row = kVector ? lane / 8 : 0u, lane_col = kVector ? lane % 8 * 4 : lane;
    uint32_t col = u.col0 + (direction == 1 ? first_col : first_col - 16) + lane_col;
    const uint32_t half = direction == 1 ? 0u : 4u;  // downwards the first 16 values are the right half
    const uint32_t write = box + lane % 16 * 128;
    out_t* dst = reinterpret_cast<out_t*>(p.out) + u.group * p.out_group + static_cast<uint64_t>(row0 + lane_row) * p.out_ld + col;
    const uint64_t step = kRowStep * p.out_ld;
    const bool accumulate = p.accumulate != 0;
    [[maybe_unused]] const WgradOldRows<out_t> here(p, u, kOldBoxes != 0, row_in_tile, direction == 1 ? first_col : first_col - 16, lane);
#pragma unroll
    for (uint32_t pass = 0; pass < kWarpCols / 32; ++pass) {
        out_t* to = dst;
#pragma unroll
        for (uint32_t rows16 = 0; rows16 < 2; ++rows16) {
            __syncwarp();  // the read-back in front is over
            if (lane / 16 == rows16) {
#pragma unroll
                for (uint32_t j = 0; j < 8; ++j) {
                    const float* a = acc + pass * 32 + j * 4;
                    ptx::st_shared_v4(write + (((j ^ half) ^ (lane % 8)) << 4),
                                      make_uint4(__float_as_uint(a[0]), __float_as_uint(a[1]), __float_as_uint(a[2]), __float_as_uint(a[3])));
                }
            }
            __syncwarp();
            const uint32_t there = col < p.k && rows > rows16 * 16 ? rows - rows16 * 16 : 0u;  // rows
            if constexpr (kOldBoxes != 0) {
                ptx::cp_async_wait_group<kOldBoxes - 1>();
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i, to += step) {
                    const uint32_t r = i * 4 + lane_row;
                    [[maybe_unused]] float4 v = ptx::ld_shared_v4_f32(box + r * 128 + ((lane % 8 ^ (r & 7u)) << 4));
                    if constexpr (sizeof(out_t) == 4) {
                        const float4 o = ptx::ld_shared_v4_f32(ring->now + (i * 32 + lane) * 16);
                        if (r < there) *reinterpret_cast<float4*>(to) = make_float4(v.x + o.x, v.y + o.y, v.z + o.z, v.w + o.w);
                    } else {
                        const uint2 o = ptx::ld_shared_v2(ring->now + (i * 32 + lane) * 8);
                        v.x += __uint_as_float(o.x << 16), v.y += __uint_as_float(o.x & 0xFFFF0000u);
                        v.z += __uint_as_float(o.y << 16), v.w += __uint_as_float(o.y & 0xFFFF0000u);
                        if (r < there) *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
                    }
                }
                __syncwarp();
                const uint32_t number = pass * 2 + rows16 + kOldBoxes;
                if (number < kWarpCols / 16) here.fetch(p, number, direction, ring->now, lane);
                else after->fetch(p, number - kWarpCols / 16, direction, ring->now, lane);
                ring->advance();
                continue;
            }
            if constexpr (kVector) {
                auto read = [&](uint32_t i) {
                    const uint32_t r = i * 4 + lane_row;
                    return ptx::ld_shared_v4_f32(box + r * 128 + ((lane % 8 ^ (r & 7u)) << 4));
                };
                // bf16: all of them before the first is rounded and stored (zeros for 36 experts N=3446 K=2944: 285 -> 250 us; fp32
                // gains nothing)
                float4 values[4];
                [[maybe_unused]] uint2 old_values[4];  // of a tile that others had a part in, too: not fetched ahead
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    if constexpr (sizeof(out_t) == 2) {
                        values[i] = read(i);
                        if (accumulate && i * 4 + lane_row < there) old_values[i] = *reinterpret_cast<const uint2*>(to + i * step);
                    }
                }
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i, to += step) {
                    float4 v = sizeof(out_t) == 2 ? values[i] : read(i);
                    if (i * 4 + lane_row >= there) continue;
                    if constexpr (sizeof(out_t) == 4) {
                        if (accumulate) red_add4(to, v);
                        else *reinterpret_cast<float4*>(to) = v;
                    } else {
                        if (accumulate) {
                            const uint2 o = old_values[i];
                            v.x += __uint_as_float(o.x << 16), v.y += __uint_as_float(o.x & 0xFFFF0000u);
                            v.z += __uint_as_float(o.y << 16), v.w += __uint_as_float(o.y & 0xFFFF0000u);
                        }
                        *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
                    }
                }
            } else {
                float values[16];
                [[maybe_unused]] float old_values[sizeof(out_t) == 2 ? 16 : 1];
#pragma unroll
                for (uint32_t r = 0; r < 16; ++r) {
                    values[r] = ptx::ld_shared_f32(box + r * 128 + (((lane / 4) ^ (r & 7u)) << 4) + lane % 4 * 4);
                    if constexpr (sizeof(out_t) == 2)
                        old_values[r] = accumulate && r < there ? __bfloat162float(to[r * p.out_ld]) : 0.0f;
                }
#pragma unroll
                for (uint32_t r = 0; r < 16; ++r, to += step) {
                    if (r >= there) continue;
                    if constexpr (sizeof(out_t) == 4) {
                        if (accumulate) red_add(to, values[r]);
                        else *to = values[r];
                    } else {
                        *to = __float2bfloat16_rn(values[r] + old_values[r]);
                    }
                }
            }
        }
        col += 32 * direction;
        dst += static_cast<int>(32 * direction);
    }
}

}  // namespace detail

struct WgradMaps {
    CUtensorMap n, k;                // codes of dy and x: boxes of 128 tokens x 128 features
    CUtensorMap scales_n, scales_k;  // their scale tiles: a box is what a tile of products needs
};

template <uint32_t kCols, typename out_t, bool kVector, bool kOldAhead>
__global__ void __launch_bounds__(384, 1) __cluster_dims__(2, 1, 1)
    fp8_wgrad_kernel(const WgradParams p, const __grid_constant__ WgradMaps maps) {
#if defined(__CUDA_ARCH__) && (__CUDA_ARCH__ >= 1000)
    using T = WgradTile<kCols, kOldAhead ? sizeof(out_t) : 0>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (ptx::smem_u32(smem_raw) & 1023u)) & 1023u);
    WgradSchedule& schedule = *reinterpret_cast<WgradSchedule*>(smem + T::kOffSchedule);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + T::kOffBarriers);  // of rank 0 alone, for the loads of both
    uint64_t* empty = full + T::kStages;
    uint64_t* sums_full = empty + T::kStages;
    uint64_t* sums_empty = sums_full + 2;    // of rank 0 alone: all columns have been read
    uint64_t* shared_empty = sums_empty + 2;  // of rank 0 alone: those that both accumulators use
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + T::kOffTmemSlot);
    volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(smem + T::kOffAbort);
    const uint32_t warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = ptx::lane_id(), rank = ptx::cluster_ctarank();

    if (warp == 0 && lane == 0 && p.max_blocks != 0) {
        ptx::tma_prefetch_desc(&maps.n);
        ptx::tma_prefetch_desc(&maps.k);
        ptx::tma_prefetch_desc(&maps.scales_n);
        ptx::tma_prefetch_desc(&maps.scales_k);
    }
    if (warp == 1 && lane == 0) {
#pragma unroll
        for (uint32_t i = 0; i < T::kStages; ++i) {
            ptx::mbar_init(full + i, 1);
            ptx::mbar_init(empty + i, 1);
        }
#pragma unroll
        for (uint32_t i = 0; i < 2; ++i) {
            ptx::mbar_init(sums_full + i, 1);
            ptx::mbar_init(sums_empty + i, 16);  // one arrival per warp that reads the sums, in both CTAs
            ptx::mbar_init(shared_empty + i, 8);  // half of them read the shared columns
        }
        *abort_flag = 0;
        ptx::fence_barrier_init();
        ptx::fence_proxy_async_smem();
    }
    // Up to here and for the tensor memory this kernel runs beside the cast in front of it, which lets it start when everything in front of
    // the cast has ended.  Group sizes are known only then, too, but one group of all rows is no secret.
    if (warp == 3 && p.groups.sizes == nullptr) detail::build_wgrad_schedule<kCols>(p, schedule);
    if (warp == 2) {
        ptx::tmem_alloc_pair(tmem_slot, T::kTmemCols);
        ptx::tmem_relinquish_alloc_permit_pair();
    }
    ptx::grid_dependency_wait();
    if (warp == 3 && p.groups.sizes != nullptr) detail::build_wgrad_schedule<kCols>(p, schedule);
    ptx::tcgen05_fence_before_thread_sync();
    __syncthreads();
    ptx::cluster_arrive(), ptx::cluster_wait();  // the other CTA's barriers and tensor memory are ready
    ptx::tcgen05_fence_after_thread_sync();
    const uint32_t tmem = *tmem_slot;
    detail::WgradWalk<kCols> walk(schedule);
    detail::WgradUnit u;

    if (warp < 4) {
        ptx::reg_dealloc<56>();
        if (warp == 0 && ptx::elect_one()) {
            // ---- loads: each CTA its rows of A and its half of B's columns per k-block, and with the first of four k-blocks its rows'
            // scales and all columns' ----
            const uint32_t tiles_n = ceil_div(p.n, 128u), tiles_k = ceil_div(p.k, kCols);
            const uint32_t full_of_pair = ptx::map_to_cta(ptx::smem_u32(full), 0);
            uint32_t stage = 0, phase = 0;
            bool alive = true;
            while (alive && walk.next(p, schedule, u)) {
                const uint32_t row = u.row0 + rank * 128, col = u.col0 + rank * (kCols / 2);
                for (uint32_t i = 0; i < u.count; ++i) {
                    const uint32_t kb = u.begin + i;
                    if (!detail::bounded_wait(empty + stage, phase ^ 1, abort_flag, p, 17)) {
                        alive = false;
                        break;
                    }
                    const bool scales = i == 0 || kb % 4 == 0;
                    if (rank == 0)
                        ptx::mbar_arrive_expect_tx(full + stage, 2 * (T::kStageA + T::kStageB + (scales ? T::kStageScales : 0u)));
                    const int32_t token = static_cast<int32_t>((u.block0 + kb) * 128);
                    const uint32_t bar = full_of_pair + stage * 8;
                    ptx::tma_load_2d_pair(smem + T::kOffA + stage * T::kStageA, &maps.n, bar, static_cast<int32_t>(row), token);
                    ptx::tma_load_2d_pair(smem + T::kOffB + stage * T::kStageB, &maps.k, bar, static_cast<int32_t>(col), token);
                    if (scales) {
                        const uint32_t quad = u.quad0 + kb / 4;
                        uint8_t* s = smem + T::kOffScales + stage * T::kStageScales;
                        // rows that dW does not have: any scales will do
                        ptx::tma_load_2d_pair(s, &maps.scales_n, bar, 0, static_cast<int32_t>(quad * tiles_n + min(row / 128, tiles_n - 1)));
                        ptx::tma_load_2d_pair(s + kScaleTileBytes, &maps.scales_k, bar, 0,
                                              static_cast<int32_t>((quad * tiles_k + u.col0 / kCols) * (T::kScaleTiles - 1)));
                    }
                    if (++stage == T::kStages) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
            }
            if (!alive) detail::drain_copies();
        } else if (warp == 1 && rank == 0 && ptx::elect_one()) {
            // ---- products of the pair ----
            constexpr uint32_t idesc = make_instr_desc_mx_mn_major(kWgradRows, kCols);
            const uint32_t a_low = make_smem_desc_mn_major_low(ptx::smem_u32(smem + T::kOffA));
            const uint32_t b_low = make_smem_desc_mn_major_low(ptx::smem_u32(smem + T::kOffB));
            const uint64_t scales_desc = make_smem_desc_scales(ptx::smem_u32(smem + T::kOffScales));
            uint32_t stage = 0, phase = 0, buf = 0, sums_phase = 0, set = 0;
            bool alive = true, loaded = false;  // loaded: the next stage was seen to be full already
            while (alive && walk.next(p, schedule, u)) {
                uint32_t left_in_chain = 0;
                for (uint32_t i = 0; i < u.count; ++i) {
                    const uint32_t kb = u.begin + i;
                    const bool begins = left_in_chain == 0;
                    if (begins) {
                        left_in_chain = min(T::kChain, u.count - i);
                        // this accumulator's sums of two chains ago, and the other's in the columns that both use
                        if (!detail::bounded_wait(sums_empty + buf, sums_phase ^ 1, abort_flag, p, 18) ||
                            (T::kShared != 0 && !detail::bounded_wait(shared_empty + (buf ^ 1), buf == 0 ? sums_phase ^ 1 : sums_phase, abort_flag, p, 21))) {
                            alive = false;
                            break;
                        }
                    }
                    if (!loaded && !detail::bounded_wait(full + stage, phase, abort_flag, p, 19)) {
                        alive = false;
                        break;
                    }
                    ptx::tcgen05_fence_after_thread_sync();
                    const uint32_t now = stage;
                    if (++stage == T::kStages) {
                        stage = 0;
                        phase ^= 1;
                    }
                    loaded = ptx::mbar_test_wait(full + stage, phase);
                    if (i == 0 || kb % 4 == 0) {
                        // Three sets in turn.  The set that is written now was last used three quads ago.  If that was in this chain or the
                        // one in front, at least five k-blocks lie in between, and the stage just filled was free: the products of kStages,
                        // at most six, k-blocks ago are complete.  If it was earlier, its accumulator has been read.
                        set = set == 2 ? 0 : set + 1;
#pragma unroll
                        for (uint32_t t = 0; t < T::kScaleTiles; ++t)
                            ptx::tmem_copy_scales_pair(tmem + T::kTmemScales + set * T::kTmemScaleSet + t * 4,
                                                       scales_desc + ((now * T::kStageScales + t * kScaleTileBytes) >> 4));
                    }
                    const uint32_t a = a_low + now * (T::kStageA >> 4), b = b_low + now * (T::kStageB >> 4);
                    const uint32_t scale_a = tmem + T::kTmemScales + set * T::kTmemScaleSet, sums = tmem + buf * T::kTmemSecond;
                    const uint32_t desc = with_scale_byte(idesc, kb % 4);
#pragma unroll
                    for (uint32_t s = 0; s < 4; ++s)
                        ptx::umma_mxf8f6f4_ss_pair(sums, a + s * kMnKStep, b + s * kMnKStep, desc, scale_a, scale_a + 4, !begins || s != 0);
                    ptx::umma_commit_pair(empty + now);
                    if (--left_in_chain == 0) {
                        ptx::umma_commit_pair(sums_full + buf);
                        buf ^= 1;
                        if (buf == 0) sums_phase ^= 1;
                    }
                }
            }
        }
        __syncwarp();
    } else {
        // ---- sums -> dW: this CTA's 128 rows ----
        ptx::reg_alloc<224>();  // 128 * 56 + 256 * 224 = 384 * 168, the launch's registers
        constexpr uint32_t kWarpCols = T::kWarpCols;
        const uint32_t quarter = warp % 4, part = warp - 4;
        // 16 columns at a time, the warps of the first half upwards and those of the second downwards: each begins with the columns that
        // both accumulators use.  acc[c] belongs to column first_col + c / 16 * 16 * direction + c % 16.
        const uint32_t first_col = part < 4 ? 0 : kCols - 16, direction = part < 4 ? 1 : ~0u;
        const uint32_t box = ptx::smem_u32(smem + T::kOffStore + part * T::kBoxBytes);
        const uint32_t empty_of_pair = ptx::map_to_cta(ptx::smem_u32(sums_empty), 0);
        [[maybe_unused]] const uint32_t shared_of_pair = ptx::map_to_cta(ptx::smem_u32(shared_empty), 0);
        const uint32_t row_in_tile = rank * 128 + quarter * 32;
        [[maybe_unused]] const uint32_t leftmost = direction == 1 ? first_col : first_col - 16;
        const uint32_t old_boxes = ptx::smem_u32(smem + T::kOffOld) + part * T::kOldBoxes * T::kOldBoxBytes;
        [[maybe_unused]] detail::WgradOldRing<T::kOldBoxes, T::kOldBoxBytes> ring{old_boxes, old_boxes};
        [[maybe_unused]] detail::WgradUnit after;  // the unit behind this one
        uint32_t buf = 0, sums_phase = 0;
        bool alive = true, more = walk.next(p, schedule, u);
        if constexpr (kOldAhead) {
            ring.fill(p, detail::WgradOldRows<out_t>(p, u, more, row_in_tile, leftmost, lane), direction, lane);
        }
        while (alive && more) {
            float acc[kWarpCols];
#pragma unroll
            for (uint32_t j = 0; j < kWarpCols; ++j) acc[j] = 0.0f;
#pragma unroll 1
            for (uint32_t i = 0; i < u.count; i += T::kChain) {
                const bool ok = detail::bounded_wait(sums_full + buf, sums_phase, abort_flag, p, 20);
                if (!__all_sync(0xffffffffu, ok)) {
                    alive = false;
                    break;
                }
                ptx::tcgen05_fence_after_thread_sync();
                const uint32_t from = tmem + ((quarter * 32u) << 16) + buf * T::kTmemSecond + first_col;
#pragma unroll
                for (uint32_t c = 0; c < kWarpCols; c += 16) {
                    uint32_t t[16];
                    ptx::tmem_ld_32x32b<16>(from + c * direction, t);
                    ptx::tmem_ld_wait<16>(t);
                    const bool last = c + 16 == kWarpCols;
                    if (last || (T::kShared != 0 && c + 16 == T::kShared)) {
                        ptx::tcgen05_fence_before_thread_sync();
                        __syncwarp();
                        if (lane == 0 && (last || (buf == 0) == (part >= 4))) ptx::mbar_arrive_cluster_relaxed((last ? empty_of_pair : shared_of_pair) + buf * 8);
                    }
#pragma unroll
                    for (uint32_t j = 0; j < 16; ++j) acc[c + j] += __uint_as_float(t[j]);
                }
                buf ^= 1;
                if (buf == 0) sums_phase ^= 1;
            }
            if (!alive || *abort_flag != 0) break;  // a wait ran out: the sums may be incomplete
            bool complete = true;  // here are all sums of the tile
            if (u.first_pair != u.last_pair) {
                // Partial tiles meet in L2; who counts itself last adds them in the order of the tokens.  A pair begins at most one tile
                // that others end, and ends at most one that another began: a slot for each.
                auto slot = [&](uint32_t pair) {
                    return p.partials + ((static_cast<uint64_t>(2 * pair + (pair == u.first_pair ? 1 : 0)) * 2 + rank) * 8 + part) * (kWarpCols / 4 * 32) + lane;
                };
                float4* mine = slot(walk.pair);
#pragma unroll
                for (uint32_t j = 0; j < kWarpCols / 4; ++j)
                    __stcg(mine + j * 32, make_float4(acc[4 * j], acc[4 * j + 1], acc[4 * j + 2], acc[4 * j + 3]));
                __threadfence();
                __syncwarp();
                uint32_t before = 0;
                if (lane == 0) before = atomicAdd(p.counters + (u.first_pair * 2 + rank) * 8 + part, 1u);
                complete = __shfl_sync(0xffffffffu, before, 0) == u.last_pair - u.first_pair;
                if (complete) {
                    __threadfence();
#pragma unroll
                    for (uint32_t j = 0; j < kWarpCols; ++j) acc[j] = 0.0f;
#pragma unroll 1
                    for (uint32_t pair = u.first_pair; pair <= u.last_pair; ++pair) {
                        const float4* from = slot(pair);
#pragma unroll
                        for (uint32_t j = 0; j < kWarpCols / 4; ++j) {
                            const float4 f = __ldcg(from + j * 32);
                            acc[4 * j] += f.x, acc[4 * j + 1] += f.y, acc[4 * j + 2] += f.z, acc[4 * j + 3] += f.w;
                        }
                    }
                }
            }
            if constexpr (kOldAhead) {
                more = walk.next(p, schedule, after);
                const detail::WgradOldRows<out_t> rows(p, after, more, row_in_tile, leftmost, lane);
                if (detail::WgradOldRows<out_t>::fetched(u) && u.row0 + row_in_tile < p.n) {
                    detail::store_wgrad_rows<out_t, kWarpCols, kVector, T::kOldBoxes>(p, u, box, row_in_tile, first_col, direction, lane, acc,
                                                                                      &ring, &rows);
                } else {
                    if (complete && u.blocks != 0)
                        detail::store_wgrad_rows<out_t, kWarpCols, kVector>(p, u, box, row_in_tile, first_col, direction, lane, acc);
                    ring.fill(p, rows, direction, lane);
                }
                u = after;
            } else {
                if (complete && (u.blocks != 0 || p.accumulate == 0))
                    detail::store_wgrad_rows<out_t, kWarpCols, kVector>(p, u, box, row_in_tile, first_col, direction, lane, acc);
                more = walk.next(p, schedule, u);
            }
        }
        if constexpr (kOldAhead) ptx::cp_async_wait_all();
        __syncwarp();
    }
    ptx::tcgen05_fence_before_thread_sync();
    __syncthreads();
    ptx::cluster_arrive(), ptx::cluster_wait();  // neither CTA's memory is needed by the other any more
    if (warp == 2) {
        ptx::tcgen05_fence_after_thread_sync();
        ptx::tmem_dealloc_pair(tmem, T::kTmemCols);
    }
#endif
}

// ---------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------
struct WgradArgs {
    const void* dy = nullptr;
    const void* x = nullptr;
    uint64_t dy_ld = 0, x_ld = 0;
    void* out = nullptr;
    uint64_t out_ld = 0, out_group = 0;
    TokenGroups groups;
    uint32_t n = 0, k = 0;
    bool out_bf16 = false, accumulate = false;
    void* workspace = nullptr;
    size_t workspace_bytes = 0;
    int num_sms = 0;
    int* status = nullptr;
    unsigned long long timeout_ns = 0;
};

// What lies in the workspace, in this order, each on a 256-byte boundary.
struct WgradWorkspace {
    size_t codes_n, codes_k, scales_n, scales_k, counters, partials, bytes;
    uint32_t codes_ld_n, codes_ld_k, blocks, quads, cols, tiles, whole_tiles, pairs, num_counters;
};

// How many tiles are dealt out whole (see WgradSchedule): full waves, one less where more than half of another wave is left, because that
// one would run nearly as long as a full one.
inline uint32_t choose_whole_wgrad_tiles(uint32_t tiles, uint32_t pairs) {
    const uint32_t waves = tiles / pairs, rest = tiles % pairs;
    return (2 * rest > pairs && waves > 0 ? waves - 1 : waves) * pairs;
}

// Columns of a tile.  Narrow ones where they still leave no more than a tile for each pair: its sums are read, joined and stored by more CTAs at
// a time, which is most of what few tiles take.  128 there; 64 where a pair's sum is short, or where many pairs share a tile either way (a
// k-block of a narrow tile takes longer than its part of the products: A's rows are loaded for fewer columns).  us for 256, 128 and 64:
//   tiles of 64 below a quarter of the pairs: 8192 tokens N=K=512 24.9, 22.2, 19.0; 20000 N=128 K=1024 39.6, 31.1, 28.5
//   up to 16 k-blocks, tiles of 64 below the pairs: 333 N=1030 K=517 14.3, 12.6, 10.9; 2048 N=1024 K=512 14.7, 12.0, 11.3
//   more k-blocks: 4096 N=K=1024 22.7, 18.5, 21.9; 4194 N=91 K=4352 33.0, 29.3, 34.2; 16384 N=K=1024 49.7, 44.2, 54.8
//   tiles of 128 above the pairs: 300 N=K=2048 11.6, 12.4, 12.6; 2048 N=4096 K=2048 27.3, 31.0, 40.5; 4096 N=4096 K=1024 40.6, 38.2, 44.9
// Otherwise 256, unless tiles of 192 overhang dW less.
inline uint32_t choose_wgrad_cols(uint32_t n, uint32_t k, uint32_t groups, uint32_t blocks, uint32_t pairs) {
    auto tiles = [&](uint32_t cols) { return static_cast<uint64_t>(ceil_div(n, kWgradRows)) * ceil_div(k, cols) * groups; };
    if (tiles(64) <= pairs && (blocks <= 16ull * groups || 4 * tiles(64) <= pairs)) return 64;
    if (tiles(128) <= pairs) return 128;
    return align_up(k, 192u) * 1.05 < align_up(k, 256u) ? 192 : 256;
}

inline bool plan_wgrad_workspace(uint32_t rows, uint32_t n, uint32_t k, uint32_t groups, bool grouped, uint32_t num_sms, WgradWorkspace& w) {
    w.blocks = max_token_blocks(rows, groups, grouped);
    w.codes_ld_n = align_up(n, 16u);
    w.codes_ld_k = align_up(k, 16u);
    const uint32_t all_pairs = num_sms > 1 ? num_sms / 2 : 1;
    w.cols = choose_wgrad_cols(n, k, groups, ceil_div(rows, 128u), all_pairs);
    const uint64_t tiles = static_cast<uint64_t>(ceil_div(n, kWgradRows)) * ceil_div(k, w.cols) * groups;
    if (tiles > 0x7fffffffull || static_cast<uint64_t>(w.blocks) * 128 > 0x7fffffffull || num_sms == 0) return false;
    w.tiles = static_cast<uint32_t>(tiles);
    // the length of all tiles (WgradSchedule) is counted in 32 bits
    if (tiles / groups * (w.blocks + static_cast<uint64_t>(groups) * kWgradMaxStoreCost) > 0xffffffffull) return false;
    // a pair per tile, or per kWgradMinCut k-blocks of one
    const uint64_t useful = tiles * (1 + w.blocks / kWgradMinCut);
    w.pairs = static_cast<uint32_t>(useful < all_pairs ? useful : all_pairs);
    w.whole_tiles = choose_whole_wgrad_tiles(w.tiles, w.pairs);
    const bool shared = w.whole_tiles != w.tiles && w.blocks >= kWgradMinCut;  // tiles may be cut
    const uint64_t quads = max_token_quads(w.blocks, groups), scale_rows = quads * (ceil_div(n, 128u) + 2ull * ceil_div(k, w.cols));
    if (scale_rows > 0x7fffffffull) return false;
    w.quads = static_cast<uint32_t>(quads);
    w.num_counters = shared ? w.pairs * 16 : 0;
    size_t at = 0;
    auto take = [&at](size_t bytes) {
        const size_t here = at;
        at = align_up(at + bytes, static_cast<size_t>(256));
        return here;
    };
    w.codes_n = take(static_cast<size_t>(w.blocks) * 128 * w.codes_ld_n);
    w.codes_k = take(static_cast<size_t>(w.blocks) * 128 * w.codes_ld_k);
    w.scales_n = take(quads * ceil_div(n, 128u) * kScaleTileBytes);
    w.scales_k = take(quads * ceil_div(k, w.cols) * 2 * kScaleTileBytes);  // two scale tiles for a tile of any width
    w.counters = take(w.num_counters * sizeof(uint32_t));
    w.partials = take(shared ? static_cast<size_t>(2) * w.pairs * kWgradRows * w.cols * sizeof(float) : 0);
    w.bytes = at;
    return true;
}

// Scale tiles as rows of 128 words; a box is `rows` of them.
inline CUtensorMap make_scale_tiles_desc(const void* base, uint64_t tiles, uint32_t rows, bool& ok) {
    CUtensorMap map{};
    EncodeTiledFn encode = get_encode_tiled();
    const cuuint64_t dims[2] = {kScaleTileBytes / 4, tiles}, strides[1] = {kScaleTileBytes};
    const cuuint32_t box[2] = {kScaleTileBytes / 4, rows}, elem_strides[2] = {1, 1};
    if (encode == nullptr || encode(&map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, const_cast<void*>(base), dims, strides, box, elem_strides,
                                    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        ok = false;
    return map;
}

template <uint32_t kCols, typename out_t, bool kVector, bool kOldAhead = false>
inline int launch_wgrad_products(const WgradParams& p, const WgradMaps& maps, uint32_t pairs, cudaStream_t stream) {
    constexpr uint32_t kSmem = WgradTile<kCols, kOldAhead ? sizeof(out_t) : 0>::kSmemSize;
    int device = 0, max_smem = 0;
    if (cudaGetDevice(&device) != cudaSuccess) return kLaunchFailed;
    cudaDeviceGetAttribute(&max_smem, cudaDevAttrMaxSharedMemoryPerBlockOptin, device);
    if (static_cast<int>(kSmem) > max_smem) return kSmemTooLarge;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2 * pairs);
    cfg.blockDim = dim3(384);
    cfg.dynamicSmemBytes = kSmem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    auto kernel = fp8_wgrad_kernel<kCols, out_t, kVector, kOldAhead>;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kSmem)) != cudaSuccess ||
        cudaLaunchKernelEx(&cfg, kernel, p, maps) != cudaSuccess) {
        cudaGetLastError();
        return kLaunchFailed;
    }
    return kOk;
}

inline int launch_fp8_wgrad(const WgradArgs& a, cudaStream_t stream) {
    const bool grouped = a.groups.sizes != nullptr;
    if (a.out == nullptr || a.n == 0 || a.k == 0 || a.num_sms <= 0 || a.groups.num_groups == 0 || a.groups.num_groups > kMaxTokenGroups)
        return kBadArgument;
    if ((a.groups.starts == nullptr) != !grouped || (!grouped && a.groups.num_groups != 1)) return kBadArgument;
    if (a.groups.rows != 0 && (a.dy == nullptr || a.x == nullptr || a.dy_ld < a.n || a.x_ld < a.k)) return kBadArgument;
    if (!is_aligned(a.dy, 2) || !is_aligned(a.x, 2) || !is_aligned(a.out, a.out_bf16 ? 2 : 4) || a.out_ld < a.k) return kBadArgument;
    WgradWorkspace w;
    if (!plan_wgrad_workspace(a.groups.rows, a.n, a.k, a.groups.num_groups, grouped, static_cast<uint32_t>(a.num_sms), w)) return kBadArgument;
    if (w.bytes != 0 && (a.workspace == nullptr || !is_aligned(a.workspace, 256))) return kBadArgument;
    if (a.workspace_bytes < w.bytes) return kWorkspaceTooSmall;
    if (w.blocks > 65535) return kBadArgument;  // the cast's grid
    int device = 0, sm_count = 0;
    if (cudaGetDevice(&device) != cudaSuccess) return kLaunchFailed;
    cudaDeviceGetAttribute(&sm_count, cudaDevAttrMultiProcessorCount, device);
    if (a.num_sms > sm_count) return kBadArgument;
    uint8_t* ws = static_cast<uint8_t*>(a.workspace);

    WgradMaps maps = {};
    if (w.blocks != 0) {
        bool ok = true;
        maps.n = make_2d_tma_desc_u8_sw128(ws + w.codes_n, static_cast<uint64_t>(w.blocks) * 128, a.n, w.codes_ld_n, 128, ok);
        maps.k = make_2d_tma_desc_u8_sw128(ws + w.codes_k, static_cast<uint64_t>(w.blocks) * 128, a.k, w.codes_ld_k, 128, ok);
        maps.scales_n = make_scale_tiles_desc(ws + w.scales_n, static_cast<uint64_t>(w.quads) * ceil_div(a.n, 128u), 1, ok);
        const uint32_t scale_tiles = ceil_div(w.cols, 128u);
        maps.scales_k = make_scale_tiles_desc(ws + w.scales_k, static_cast<uint64_t>(w.quads) * ceil_div(a.k, w.cols) * scale_tiles, scale_tiles, ok);
        if (!ok) return kTensorMapFailed;

        CastTokensParams c;
        c.groups = a.groups;
        c.max_blocks = w.blocks;
        auto operand = [](const void* z, uint64_t ld, uint32_t cols, uint8_t* codes, uint32_t codes_ld, uint8_t* scales, uint32_t scale_cols) {
            CastTokensOperand o;
            o.z = static_cast<const __nv_bfloat16*>(z);
            o.ld = ld, o.cols = cols;
            o.wide = is_aligned(z, 32) && ld % 16 == 0 && cols % 16 == 0;
            o.codes = codes, o.codes_ld = codes_ld, o.scales = scales, o.scale_cols = scale_cols;
            return o;
        };
        c.operand[0] = operand(a.dy, a.dy_ld, a.n, ws + w.codes_n, w.codes_ld_n, ws + w.scales_n, 128);
        c.operand[1] = operand(a.x, a.x_ld, a.k, ws + w.codes_k, w.codes_ld_k, ws + w.scales_k, w.cols);
        c.column_tiles[0] = ceil_div(a.n, 128u), c.column_tiles[1] = ceil_div(a.k, 128u);
        c.counters = reinterpret_cast<uint32_t*>(ws + w.counters);
        c.num_counters = w.num_counters;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(c.column_tiles[0] + c.column_tiles[1], w.blocks);
        cfg.blockDim = dim3(256);
        cfg.stream = stream;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        const bool wide = c.operand[0].wide != 0 && c.operand[1].wide != 0;
        if (cudaLaunchKernelEx(&cfg, wide ? block_cast_tokens_kernel<true> : block_cast_tokens_kernel<false>, c) != cudaSuccess) {
            cudaGetLastError();
            return kLaunchFailed;
        }
    }

    WgradParams p;
    p.groups = a.groups;
    p.max_blocks = w.blocks;
    p.n = a.n, p.k = a.k;
    p.out = a.out, p.out_ld = a.out_ld, p.out_group = a.out_group;
    p.accumulate = a.accumulate;
    const uint32_t vec = 4, item = a.out_bf16 ? 2 : 4;  // four columns at a time
    const bool vector = is_aligned(a.out, vec * item) && a.out_ld % vec == 0 && a.out_group % vec == 0 && a.k % vec == 0;
    p.tiles = w.tiles, p.whole_tiles = w.whole_tiles;
    // A CTA's 128 rows of a tile, about 100 KB in fp32, leave at 1/148 of the memory's rate in the time of about ten k-blocks.
    p.store_cost = (a.out_bf16 ? 5u : 10u) * (a.accumulate ? 2u : 1u);
    p.partials = reinterpret_cast<float4*>(ws + w.partials);
    p.counters = reinterpret_cast<uint32_t*>(ws + w.counters);
    p.status = a.status;
    p.timeout_ns = a.timeout_ns;
    // Old values are fetched ahead in bf16, and in fp32 where a tile has few k-blocks and its store is what takes long: us for 8, 16, 32 and 64
    // k-blocks per group (16 experts N=4096 K=2048; one N=7168 K=2048; 8 N=K=4096; one N=7168 K=2048) added in L2 350, 51.5, 585, 131, fetched
    // ahead 300, 50.1, 610, 138.  With a tile for each pair at most there is nothing to hide them behind (333 tokens N=1032 K=520 12.4, 12.8).
    const bool ahead = a.accumulate && w.cols >= 192 && (a.out_bf16 || (w.tiles > w.pairs && a.groups.rows <= 16u * 128 * a.groups.num_groups));
    auto launch = [&](auto out, auto vectors) {
        using out_t = decltype(out);
        constexpr bool kVector = decltype(vectors)::value;
        if constexpr (kVector) {
            if (ahead)
                return w.cols == 192 ? launch_wgrad_products<192, out_t, true, true>(p, maps, w.pairs, stream)
                                     : launch_wgrad_products<256, out_t, true, true>(p, maps, w.pairs, stream);
        }
        if (w.cols == 64) return launch_wgrad_products<64, out_t, kVector>(p, maps, w.pairs, stream);
        if (w.cols == 128) return launch_wgrad_products<128, out_t, kVector>(p, maps, w.pairs, stream);
        return w.cols == 192 ? launch_wgrad_products<192, out_t, kVector>(p, maps, w.pairs, stream)
                             : launch_wgrad_products<256, out_t, kVector>(p, maps, w.pairs, stream);
    };
    if (a.out_bf16) return vector ? launch(__nv_bfloat16(), std::true_type()) : launch(__nv_bfloat16(), std::false_type());
    return vector ? launch(float(), std::true_type()) : launch(float(), std::false_type());
}

}  // namespace yan
