#pragma once
// Weight gradient of a linear layer from 8-bit operands:  dW[n, k] (+)= sum over tokens m of dy[m, n] * x[m, k], for one matrix or for
// every group of tokens (expert) its own.
//
//   1. block_cast_tokens_kernel: both bf16 operands -> e4m3 codes, in the order they have, with one power of two per feature and block
//      of 128 tokens, e the smallest integer with amax <= 448 * 2^e.  A block that ends a group is filled up with zeros.
//   2. fp8_wgrad_kernel: persistent, warp-specialised tcgen05 products of 128 x 256 tiles of dW, summed over the tokens in tensor memory.
//      The tensor core transposes the token-major operands and multiplies the scales in, so that nothing has to be promoted.

#include <cstdint>
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
    uint8_t* scales = nullptr;  // [quads][ceil(cols / 128)] scale tiles
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

// One CTA of 256 threads: 128 tokens x 128 columns of one operand.  Eight threads share a row, 16 columns each; 32 rows at a time.
__global__ void __launch_bounds__(256) block_cast_tokens_kernel(const CastTokensParams p) {
    __shared__ TokenBlockTable table;
    __shared__ uint4 s_max[8][16];  // [warp][8 columns as packed bf16 magnitudes]
    __shared__ uint8_t s_scale[128];
    ptx::grid_dependency_wait();
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
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
        const uint32_t r = first_row + 32 * i;
        v[i][0] = v[i][1] = make_uint4(0, 0, 0, 0);
        if (r >= rows || col >= op.cols) continue;
        const __nv_bfloat16* src = op.z + static_cast<uint64_t>(row0 + r) * op.ld + col;
        if (op.wide != 0) {
            ptx::ld_global_32(v[i], src);
        } else {
            uint16_t h[16];
#pragma unroll
            for (uint32_t j = 0; j < 16; ++j) h[j] = col + j < op.cols ? *reinterpret_cast<const volatile uint16_t*>(src + j) : uint16_t(0);
            uint32_t w[8];
#pragma unroll
            for (uint32_t j = 0; j < 8; ++j) w[j] = h[2 * j] | (static_cast<uint32_t>(h[2 * j + 1]) << 16);
            v[i][0] = make_uint4(w[0], w[1], w[2], w[3]);
            v[i][1] = make_uint4(w[4], w[5], w[6], w[7]);
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
        const uint32_t scale = detail::scale_byte_of_amax(amax);
        s_scale[thread] = static_cast<uint8_t>(scale);
        op.scales[(static_cast<uint64_t>(quad) * p.column_tiles[second] + tile) * kScaleTileBytes + scale_tile_offset(thread, byte)] =
            static_cast<uint8_t>(scale);
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
    const uint8_t* scales_n = nullptr;    // of dy: [quads][ceil(n / 128)] scale tiles
    const uint8_t* scales_k = nullptr;    // of x
    void* out = nullptr;                  // [groups][n][out_ld]
    uint64_t out_ld = 0, out_group = 0;   // elements
    uint32_t accumulate = 0;
    uint32_t vector_store = 0;            // rows of dW allow four elements at a time
    uint32_t tiles = 0, whole_tiles = 0;  // all of them; those that are dealt out one by one (see WgradSchedule)
    uint32_t store_cost = 0;              // k-blocks that take as long as storing a tile
    float4* partials = nullptr;           // [2 * CTAs][8 warps][32][32 lanes]
    uint32_t* counters = nullptr;         // [CTAs][8 warps], zero
    int* status = nullptr;
    unsigned long long timeout_ns = 0;
};

// Who computes what.  Tiles are numbered group by group, within a group in bands of 16 tile rows, so that CTAs at work at the same time
// share what they read.  The first whole_tiles of them, a multiple of the CTAs, are dealt out in turn.  The rest, less than two waves,
// is shared evenly: laid end to end, a tile as long as its k-blocks or as its store takes, whichever is more, and cut into one
// stretch per CTA.  A cut through the k-blocks of a tile goes to a multiple of four of them; tiles of fewer than kMinCut go whole to
// the CTA in whose stretch they begin.
struct WgradSchedule {
    TokenBlockTable blocks;
    uint64_t length[kMaxTokenGroups + 1];  // of all tiles in front of a group
    uint64_t origin, rest;                 // where the shared tiles begin, and their length
    uint32_t stretches;
};

struct WgradTile {
    static constexpr uint32_t kBlockFeatures = 256;  // columns of a tile (features of x); its rows are 128 features of dy
    static constexpr uint32_t kStages = 4;
    // k-blocks that are summed in tensor memory before the sums move to registers.  An addition there rounds towards zero (8192 tokens of
    // uneven size, relative error: 1.3e-6 in one chain).
#ifndef YAN_WGRAD_CHAIN
#define YAN_WGRAD_CHAIN 32
#endif
    static constexpr uint32_t kChain = YAN_WGRAD_CHAIN;
    static constexpr uint32_t kMinCut = 8, kMinStretch = 8;
    static constexpr uint32_t kStageA = kMnBoxBytes, kStageB = 2 * kMnBoxBytes;
    static constexpr uint32_t kScaleTiles = 1 + kBlockFeatures / 128;
    static constexpr uint32_t kStageScales = kScaleTiles * kScaleTileBytes;
    static constexpr uint32_t kOffA = 0, kOffB = kOffA + kStages * kStageA, kOffScales = kOffB + kStages * kStageB;
    static constexpr uint32_t kBoxRowBytes = 64, kBoxBytes = 32 * kBoxRowBytes;  // output staging, one box per warp
    static constexpr uint32_t kOffStore = kOffScales + kStages * kStageScales;
    static constexpr uint32_t kOffSchedule = kOffStore + 8 * kBoxBytes;
    static constexpr uint32_t kOffBarriers = align_up(kOffSchedule + static_cast<uint32_t>(sizeof(WgradSchedule)), 8u);
    static constexpr uint32_t kNumBarriers = 2 * kStages + 2;
    static constexpr uint32_t kOffTmemSlot = kOffBarriers + kNumBarriers * 8, kOffAbort = kOffTmemSlot + 4;
    static constexpr uint32_t kSmemSize = kOffAbort + 4 + 1024;
    // tensor memory: the sums, then two sets of scales
    static constexpr uint32_t kTmemScales = kBlockFeatures, kTmemScaleSet = kScaleTiles * 4, kTmemCols = 512;
    static_assert(kTmemScales + 2 * kTmemScaleSet <= kTmemCols);
    static_assert(kSmemSize <= 232448);
    static_assert(kChain % 4 == 0 && kMinCut % 4 == 0 && kMinStretch >= 8);
};

namespace detail {

__device__ __forceinline__ uint32_t wgrad_tiles_per_group(const WgradParams& p) {
    return ceil_div(p.n, 128u) * ceil_div(p.k, WgradTile::kBlockFeatures);
}
// Length of a tile with so many k-blocks.  Nothing is left to do for an empty group that is added.
__device__ __forceinline__ uint32_t wgrad_length(const WgradParams& p, uint32_t blocks) {
    return blocks == 0 && p.accumulate != 0 ? 0u : max(blocks, p.store_cost);
}

// Called by one whole warp.
__device__ __forceinline__ void build_wgrad_schedule(const WgradParams& p, WgradSchedule& s) {
    build_token_blocks(p.groups, p.max_blocks, s.blocks);
    const uint32_t lane = ptx::lane_id(), per_group = wgrad_tiles_per_group(p);
    uint64_t at = 0;
    for (uint32_t first = 0; first < p.groups.num_groups; first += 32) {
        const uint32_t g = first + lane;
        const uint64_t own = g < p.groups.num_groups
                                 ? static_cast<uint64_t>(per_group) * wgrad_length(p, s.blocks.block[g + 1] - s.blocks.block[g]) : 0u;
        uint64_t until = own;
#pragma unroll
        for (uint32_t off = 1; off < 32; off *= 2) {
            const uint64_t v = __shfl_up_sync(0xffffffffu, until, off);
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
            s.origin = s.length[g] + static_cast<uint64_t>(p.whole_tiles % per_group) * wgrad_length(p, s.blocks.block[g + 1] - s.blocks.block[g]);
        s.rest = at - s.origin;
        s.stretches = static_cast<uint32_t>(max(min(static_cast<uint64_t>(gridDim.x), s.rest / WgradTile::kMinStretch), static_cast<uint64_t>(1)));
    }
}

// What one CTA computes at a time: k-blocks [begin, begin + count) of a group, of `blocks`, for one tile of its dW.
struct WgradUnit {
    uint32_t group, row0, col0;        // row0, col0: features of the tile's corner
    uint32_t block0, quad0;            // the group's first k-block and quad of scales
    uint32_t begin, count, blocks;
    uint32_t first_cta, last_cta;      // who shares the tile
};

// The CTA's units one after the other; every role of the CTA walks them.
struct WgradWalk {
    uint32_t tile;        // next of the dealt tiles
    uint64_t at, end;     // what is left of the CTA's stretch

    __device__ __forceinline__ explicit WgradWalk(const WgradSchedule& s)
        : tile(blockIdx.x),
          at(blockIdx.x < s.stretches ? s.origin + blockIdx.x * s.rest / s.stretches : 0u),
          end(blockIdx.x < s.stretches ? s.origin + (blockIdx.x + 1u) * s.rest / s.stretches : 0u) {}

    __device__ __forceinline__ static void place(const WgradParams& p, const WgradSchedule& s, uint32_t group, uint32_t in_group, WgradUnit& u) {
        const uint32_t tiles_n = ceil_div(p.n, 128u), tiles_k = ceil_div(p.k, WgradTile::kBlockFeatures);
        const uint32_t band = in_group / (16 * tiles_k), in_band = in_group % (16 * tiles_k), rows = min(16u, tiles_n - band * 16);
        u.group = group;
        u.row0 = (band * 16 + in_band % rows) * 128;
        u.col0 = in_band / rows * WgradTile::kBlockFeatures;
        u.block0 = s.blocks.block[group];
        u.quad0 = s.blocks.quad[group];
        u.blocks = s.blocks.block[group + 1] - u.block0;
    }
    // The CTA in whose stretch a position lies.
    __device__ __forceinline__ static uint32_t owner(const WgradSchedule& s, uint64_t position) {
        return static_cast<uint32_t>(((position - s.origin + 1) * s.stretches - 1) / s.rest);
    }

    __device__ __forceinline__ bool next(const WgradParams& p, const WgradSchedule& s, WgradUnit& u) {
        const uint32_t per_group = wgrad_tiles_per_group(p);
        if (tile < p.whole_tiles) {
            place(p, s, tile / per_group, tile % per_group, u);
            u.begin = 0, u.count = u.blocks;
            u.first_cta = u.last_cta = blockIdx.x;
            tile += gridDim.x;
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
            const uint32_t in_group = static_cast<uint32_t>((at - s.length[low]) / length);
            const uint64_t start = s.length[low] + static_cast<uint64_t>(in_group) * length;
            const uint32_t from = static_cast<uint32_t>(at - start);  // above zero only in the tile that the stretch begins in
            const uint64_t until = end - start;
            at = start + length;
            place(p, s, low, in_group, u);
            if (blocks < WgradTile::kMinCut) {
                if (from != 0) continue;
                u.begin = 0, u.count = blocks;
                u.first_cta = u.last_cta = blockIdx.x;
                return true;
            }
            u.begin = from >= blocks ? blocks : from & ~3u;
            u.count = (until >= blocks ? blocks : static_cast<uint32_t>(until) & ~3u) - u.begin;
            if (u.count == 0) continue;
            u.first_cta = owner(s, start + 3);  // a stretch that ends in the first three k-blocks has none of them
            u.last_cta = owner(s, start + blocks - 1);
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
__device__ __forceinline__ void red_add4(float* p, const uint4& v) {
    asm volatile("red.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(p), "f"(__uint_as_float(v.x)), "f"(__uint_as_float(v.y)),
                 "f"(__uint_as_float(v.z)), "f"(__uint_as_float(v.w))
                 : "memory");
}

// Stores a warp's 32 rows x 128 columns; lane r holds row r.  The rows go through the warp's box in shared memory, 16 columns at a time in
// fp32, so that a store instruction covers eight pieces of 64 contiguous bytes.  fp32 is added to what dW holds where dW lies, in L2:
// every element once, so that the order does not matter, and nothing waits for the old value (16 experts N=4096 K=2048, 16384 tokens:
// 535 us with loads and stores).  bf16 is loaded, added in 32 bits and rounded once.
template <typename out_t>
__device__ __forceinline__ void store_wgrad_rows(const WgradParams& p, const WgradUnit& u, uint32_t box, uint32_t row_in_tile, uint32_t col0,
                                                 uint32_t lane, const float (&acc)[128]) {
    out_t* out = reinterpret_cast<out_t*>(p.out) + u.group * p.out_group;
    const uint32_t row0 = u.row0 + row_in_tile;
    if (u.col0 + col0 >= p.k || row0 >= p.n) return;
#pragma unroll
    for (uint32_t pass = 0; pass < 8; ++pass) {
        const uint32_t chunk = lane % 4, col = u.col0 + col0 + pass * 16 + chunk * 4;
        [[maybe_unused]] uint2 old[4];
        if constexpr (sizeof(out_t) == 2) {
            if (p.vector_store != 0 && p.accumulate != 0) {
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    const uint32_t r = row0 + i * 8 + lane / 4;
                    old[i] = make_uint2(0, 0);
                    if (r < p.n && col < p.k) old[i] = *reinterpret_cast<const uint2*>(out + static_cast<uint64_t>(r) * p.out_ld + col);
                }
            }
        }
        __syncwarp();  // the read-back of the previous pass is over
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            const float* a = acc + pass * 16 + j * 4;
            ptx::st_shared_v4(box + lane * 64 + ((j ^ ((lane >> 1) & 3u)) << 4),
                              make_uint4(__float_as_uint(a[0]), __float_as_uint(a[1]), __float_as_uint(a[2]), __float_as_uint(a[3])));
        }
        __syncwarp();
        if (p.vector_store != 0) {
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                const uint32_t r = i * 8 + lane / 4;
                uint4 v = ptx::ld_shared_v4(box + r * 64 + ((chunk ^ ((r >> 1) & 3u)) << 4));
                if (row0 + r >= p.n || col >= p.k) continue;
                out_t* dst = out + static_cast<uint64_t>(row0 + r) * p.out_ld + col;
                if constexpr (sizeof(out_t) == 4) {
                    if (p.accumulate != 0) red_add4(dst, v);
                    else *reinterpret_cast<uint4*>(dst) = v;
                } else {
                    if (p.accumulate != 0) {
                        v.x = __float_as_uint(__uint_as_float(v.x) + __uint_as_float(old[i].x << 16));
                        v.y = __float_as_uint(__uint_as_float(v.y) + __uint_as_float(old[i].x & 0xFFFF0000u));
                        v.z = __float_as_uint(__uint_as_float(v.z) + __uint_as_float(old[i].y << 16));
                        v.w = __float_as_uint(__uint_as_float(v.w) + __uint_as_float(old[i].y & 0xFFFF0000u));
                    }
                    *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(__uint_as_float(v.x), __uint_as_float(v.y)),
                                                                pack_bf16(__uint_as_float(v.z), __uint_as_float(v.w)));
                }
            }
        } else {
            // one element per lane, two rows at a time
            const uint32_t c = lane % 16, column = u.col0 + col0 + pass * 16 + c;
#pragma unroll 4
            for (uint32_t r = lane / 16; r < 32; r += 2) {
                const float v = ptx::ld_shared_f32(box + r * 64 + (((c / 4) ^ ((r >> 1) & 3u)) << 4) + c % 4 * 4);
                if (row0 + r >= p.n || column >= p.k) continue;
                out_t* dst = out + static_cast<uint64_t>(row0 + r) * p.out_ld + column;
                if constexpr (sizeof(out_t) == 4) {
                    if (p.accumulate != 0) red_add(dst, v);
                    else *dst = v;
                } else {
                    *dst = __float2bfloat16_rn(p.accumulate != 0 ? v + __bfloat162float(*dst) : v);
                }
            }
        }
    }
}

}  // namespace detail

template <typename out_t>
__global__ void __launch_bounds__(384, 1)
    fp8_wgrad_kernel(const WgradParams p, const __grid_constant__ CUtensorMap map_n, const __grid_constant__ CUtensorMap map_k) {
#if defined(__CUDA_ARCH__) && (__CUDA_ARCH__ >= 1000)
    using T = WgradTile;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (ptx::smem_u32(smem_raw) & 1023u)) & 1023u);
    WgradSchedule& schedule = *reinterpret_cast<WgradSchedule*>(smem + T::kOffSchedule);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + T::kOffBarriers);
    uint64_t* empty = full + T::kStages;
    uint64_t* sums_full = empty + T::kStages;
    uint64_t* sums_empty = sums_full + 1;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + T::kOffTmemSlot);
    volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(smem + T::kOffAbort);
    const uint32_t warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = ptx::lane_id();

    if (warp == 0 && lane == 0 && p.max_blocks != 0) {
        ptx::tma_prefetch_desc(&map_n);
        ptx::tma_prefetch_desc(&map_k);
    }
    if (warp == 1 && lane == 0) {
#pragma unroll
        for (uint32_t i = 0; i < T::kStages; ++i) {
            ptx::mbar_init(full + i, 1);
            ptx::mbar_init(empty + i, 1);
        }
        ptx::mbar_init(sums_full, 1);
        ptx::mbar_init(sums_empty, 8);  // one arrival per warp that reads the sums
        *abort_flag = 0;
        ptx::fence_barrier_init();
        ptx::fence_proxy_async_smem();
    }
    ptx::grid_dependency_wait();
    if (warp == 3) detail::build_wgrad_schedule(p, schedule);
    if (warp == 2) {
        ptx::tmem_alloc(tmem_slot, T::kTmemCols);
        ptx::tmem_relinquish_alloc_permit();
    }
    ptx::tcgen05_fence_before_thread_sync();
    __syncthreads();
    ptx::tcgen05_fence_after_thread_sync();
    const uint32_t tmem = *tmem_slot;
    const uint32_t tiles_n = ceil_div(p.n, 128u), tiles_k128 = ceil_div(p.k, 128u);
    detail::WgradWalk walk(schedule);
    detail::WgradUnit u;

    if (warp < 4) {
        ptx::reg_dealloc<56>();
        if (warp == 0 && lane == 0) {
            // ---- loads: a k-block of both operands per stage, and the scales of four k-blocks with the first of them ----
            uint32_t stage = 0, phase = 0;
            bool alive = true;
            while (alive && walk.next(p, schedule, u)) {
                const bool second_box = u.col0 + 128 < p.k;
                const uint32_t boxes = second_box ? 2 : 1;
                for (uint32_t i = 0; i < u.count; ++i) {
                    const uint32_t kb = u.begin + i;
                    if (!detail::bounded_wait(empty + stage, phase ^ 1, abort_flag, p, 17)) {
                        alive = false;
                        break;
                    }
                    const bool scales = i == 0 || kb % 4 == 0;
                    ptx::mbar_arrive_expect_tx(full + stage, kMnBoxBytes * (1 + boxes) + (scales ? kScaleTileBytes * (1 + boxes) : 0u));
                    const int32_t token = static_cast<int32_t>((u.block0 + kb) * 128);
                    uint8_t* b = smem + T::kOffB + stage * T::kStageB;
                    ptx::tma_load_2d(smem + T::kOffA + stage * T::kStageA, &map_n, full + stage, static_cast<int32_t>(u.row0), token);
                    ptx::tma_load_2d(b, &map_k, full + stage, static_cast<int32_t>(u.col0), token);
                    if (second_box) ptx::tma_load_2d(b + kMnBoxBytes, &map_k, full + stage, static_cast<int32_t>(u.col0 + 128), token);
                    if (scales) {
                        const uint64_t quad = u.quad0 + kb / 4;
                        uint8_t* s = smem + T::kOffScales + stage * T::kStageScales;
                        ptx::bulk_load(s, p.scales_n + (quad * tiles_n + u.row0 / 128) * kScaleTileBytes, kScaleTileBytes, full + stage);
                        ptx::bulk_load(s + kScaleTileBytes, p.scales_k + (quad * tiles_k128 + u.col0 / 128) * kScaleTileBytes,
                                       kScaleTileBytes * boxes, full + stage);
                    }
                    if (++stage == T::kStages) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
            }
            if (!alive) detail::drain_copies();
        } else if (warp == 1 && lane == 0) {
            // ---- products ----
            constexpr uint32_t idesc = make_instr_desc_mx_mn_major(128, T::kBlockFeatures);
            uint32_t stage = 0, phase = 0, sums_phase = 0, set = 0;
            bool alive = true;
            while (alive && walk.next(p, schedule, u)) {
                for (uint32_t i = 0; i < u.count; ++i) {
                    const uint32_t kb = u.begin + i;
                    if (i % T::kChain == 0) {
                        if (!detail::bounded_wait(sums_empty, sums_phase ^ 1, abort_flag, p, 18)) {
                            alive = false;
                            break;
                        }
                        sums_phase ^= 1;
                    }
                    if (!detail::bounded_wait(full + stage, phase, abort_flag, p, 19)) {
                        alive = false;
                        break;
                    }
                    ptx::tcgen05_fence_after_thread_sync();
                    if (i == 0 || kb % 4 == 0) {
                        // Two sets in turn: the set that is written now was last used two quads ago, and a stage is loaded again only when
                        // its products are complete, four k-blocks ago; a tile begins when the one in front is complete.
                        set ^= 1;
                        const uint32_t s = ptx::smem_u32(smem + T::kOffScales + stage * T::kStageScales);
#pragma unroll
                        for (uint32_t t = 0; t < T::kScaleTiles; ++t)
                            ptx::tmem_copy_scales(tmem + T::kTmemScales + set * T::kTmemScaleSet + t * 4,
                                                  make_smem_desc_scales(s + t * kScaleTileBytes));
                    }
                    const uint64_t a = make_smem_desc_mn_major_sw128(ptx::smem_u32(smem + T::kOffA + stage * T::kStageA));
                    const uint64_t b = make_smem_desc_mn_major_sw128(ptx::smem_u32(smem + T::kOffB + stage * T::kStageB));
                    const uint32_t scale_a = tmem + T::kTmemScales + set * T::kTmemScaleSet;
#pragma unroll
                    for (uint32_t s = 0; s < 4; ++s)
                        ptx::umma_mxf8f6f4_ss(tmem, a + s * kMnKStep, b + s * kMnKStep, with_scale_byte(idesc, kb % 4), scale_a, scale_a + 4,
                                              i % T::kChain != 0 || s != 0);
                    ptx::umma_commit(empty + stage);
                    if (i % T::kChain == T::kChain - 1 || i + 1 == u.count) ptx::umma_commit(sums_full);
                    if (++stage == T::kStages) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
            }
        }
        __syncwarp();
    } else {
        // ---- sums -> dW ----
        ptx::reg_alloc<224>();  // 128 * 56 + 256 * 224 = 384 * 168, the launch's registers
        const uint32_t quarter = warp % 4, part = warp - 4, col0 = part / 4 * 128;
        const uint32_t box = ptx::smem_u32(smem + T::kOffStore + part * T::kBoxBytes);
        uint32_t sums_phase = 0;
        bool alive = true;
        while (alive && walk.next(p, schedule, u)) {
            float acc[128];
#pragma unroll
            for (uint32_t j = 0; j < 128; ++j) acc[j] = 0.0f;
#pragma unroll 1
            for (uint32_t i = 0; i < u.count; i += T::kChain) {
                const bool ok = detail::bounded_wait(sums_full, sums_phase, abort_flag, p, 20);
                if (!__all_sync(0xffffffffu, ok)) {
                    alive = false;
                    break;
                }
                sums_phase ^= 1;
                ptx::tcgen05_fence_after_thread_sync();
#pragma unroll
                for (uint32_t c = 0; c < 128; c += 32) {
                    uint32_t t[32];
                    ptx::tmem_ld_32x32b<32>(tmem + ((quarter * 32u) << 16) + col0 + c, t);
                    ptx::tmem_ld_wait<32>(t);
                    if (c == 96) {
                        ptx::tcgen05_fence_before_thread_sync();
                        __syncwarp();
                        if (lane == 0) ptx::mbar_arrive(sums_empty);
                    }
#pragma unroll
                    for (uint32_t j = 0; j < 32; ++j) acc[c + j] += __uint_as_float(t[j]);
                }
            }
            if (!alive || *abort_flag != 0) break;  // a wait ran out: the sums may be incomplete
            if (u.first_cta != u.last_cta) {
                // Partial tiles meet in L2; who counts itself last adds them in the order of the tokens.  A CTA begins at most one tile
                // that others end, and ends at most one that another began: a slot for each.
                auto slot = [&](uint32_t cta) {
                    return p.partials + (static_cast<uint64_t>(2 * cta + (cta == u.first_cta ? 1 : 0)) * 8 + part) * 1024 + lane;
                };
                float4* mine = slot(blockIdx.x);
#pragma unroll
                for (uint32_t j = 0; j < 32; ++j) __stcg(mine + j * 32, make_float4(acc[4 * j], acc[4 * j + 1], acc[4 * j + 2], acc[4 * j + 3]));
                __threadfence();
                __syncwarp();
                uint32_t before = 0;
                if (lane == 0) before = atomicAdd(p.counters + u.first_cta * 8 + part, 1u);
                if (__shfl_sync(0xffffffffu, before, 0) != u.last_cta - u.first_cta) continue;
                __threadfence();
#pragma unroll
                for (uint32_t j = 0; j < 128; ++j) acc[j] = 0.0f;
#pragma unroll 1
                for (uint32_t cta = u.first_cta; cta <= u.last_cta; ++cta) {
                    const float4* from = slot(cta);
#pragma unroll
                    for (uint32_t j = 0; j < 32; ++j) {
                        const float4 f = __ldcg(from + j * 32);
                        acc[4 * j] += f.x, acc[4 * j + 1] += f.y, acc[4 * j + 2] += f.z, acc[4 * j + 3] += f.w;
                    }
                }
            } else if (u.blocks == 0 && p.accumulate != 0) {
                continue;
            }
            detail::store_wgrad_rows<out_t>(p, u, box, quarter * 32, col0, lane, acc);
        }
        __syncwarp();
    }
    ptx::tcgen05_fence_before_thread_sync();
    __syncthreads();
    if (warp == 2) {
        ptx::tcgen05_fence_after_thread_sync();
        ptx::tmem_dealloc(tmem, T::kTmemCols);
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
    uint32_t codes_ld_n, codes_ld_k, blocks, tiles, whole_tiles, ctas, num_counters;
};

// How many tiles are dealt out whole (see WgradSchedule): full waves, one less where more than half of another wave is left, because that
// one would run nearly as long as a full one.
inline uint32_t choose_whole_wgrad_tiles(uint32_t tiles, uint32_t ctas) {
    const uint32_t waves = tiles / ctas, rest = tiles % ctas;
    return (2 * rest > ctas && waves > 0 ? waves - 1 : waves) * ctas;
}

inline bool plan_wgrad_workspace(uint32_t rows, uint32_t n, uint32_t k, uint32_t groups, bool grouped, uint32_t num_sms, WgradWorkspace& w) {
    w.blocks = max_token_blocks(rows, groups, grouped);
    w.codes_ld_n = align_up(n, 16u);
    w.codes_ld_k = align_up(k, 16u);
    const uint64_t tiles = static_cast<uint64_t>(ceil_div(n, 128u)) * ceil_div(k, WgradTile::kBlockFeatures) * groups;
    if (tiles > 0x7fffffffull || static_cast<uint64_t>(w.blocks) * 128 > 0x7fffffffull || num_sms == 0) return false;
    w.tiles = static_cast<uint32_t>(tiles);
    // a CTA per tile, or per kMinCut k-blocks of one
    const uint64_t useful = tiles * (1 + w.blocks / WgradTile::kMinCut);
    w.ctas = useful < num_sms ? static_cast<uint32_t>(useful) : num_sms;
    w.whole_tiles = choose_whole_wgrad_tiles(w.tiles, w.ctas);
    const bool shared = w.whole_tiles != w.tiles && w.blocks >= WgradTile::kMinCut;  // tiles may be cut
    const uint64_t quads = max_token_quads(w.blocks, groups);
    w.num_counters = shared ? w.ctas * 8 : 0;
    size_t at = 0;
    auto take = [&at](size_t bytes) {
        const size_t here = at;
        at = align_up(at + bytes, static_cast<size_t>(256));
        return here;
    };
    w.codes_n = take(static_cast<size_t>(w.blocks) * 128 * w.codes_ld_n);
    w.codes_k = take(static_cast<size_t>(w.blocks) * 128 * w.codes_ld_k);
    w.scales_n = take(quads * ceil_div(n, 128u) * kScaleTileBytes);
    w.scales_k = take(quads * ceil_div(k, 128u) * kScaleTileBytes);
    w.counters = take(w.num_counters * sizeof(uint32_t));
    w.partials = take(shared ? static_cast<size_t>(2) * w.ctas * 128 * WgradTile::kBlockFeatures * sizeof(float) : 0);
    w.bytes = at;
    return true;
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
    int device = 0, sm_count = 0, max_smem = 0;
    if (cudaGetDevice(&device) != cudaSuccess) return kLaunchFailed;
    cudaDeviceGetAttribute(&sm_count, cudaDevAttrMultiProcessorCount, device);
    cudaDeviceGetAttribute(&max_smem, cudaDevAttrMaxSharedMemoryPerBlockOptin, device);
    if (a.num_sms > sm_count) return kBadArgument;
    if (static_cast<int>(WgradTile::kSmemSize) > max_smem) return kSmemTooLarge;
    uint8_t* ws = static_cast<uint8_t*>(a.workspace);

    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;

    const uint32_t tiles_n = ceil_div(a.n, 128u), tiles_k128 = ceil_div(a.k, 128u);
    if (w.blocks != 0) {
        CastTokensParams c;
        c.groups = a.groups;
        c.max_blocks = w.blocks;
        auto operand = [](const void* z, uint64_t ld, uint32_t cols, uint8_t* codes, uint32_t codes_ld, uint8_t* scales) {
            CastTokensOperand o;
            o.z = static_cast<const __nv_bfloat16*>(z);
            o.ld = ld, o.cols = cols;
            o.wide = is_aligned(z, 32) && ld % 16 == 0 && cols % 16 == 0;
            o.codes = codes, o.codes_ld = codes_ld, o.scales = scales;
            return o;
        };
        c.operand[0] = operand(a.dy, a.dy_ld, a.n, ws + w.codes_n, w.codes_ld_n, ws + w.scales_n);
        c.operand[1] = operand(a.x, a.x_ld, a.k, ws + w.codes_k, w.codes_ld_k, ws + w.scales_k);
        c.column_tiles[0] = tiles_n, c.column_tiles[1] = tiles_k128;
        c.counters = reinterpret_cast<uint32_t*>(ws + w.counters);
        c.num_counters = w.num_counters;
        if (w.blocks > 65535) return kBadArgument;
        cfg.gridDim = dim3(tiles_n + tiles_k128, w.blocks);
        cfg.blockDim = dim3(256);
        if (cudaLaunchKernelEx(&cfg, block_cast_tokens_kernel, c) != cudaSuccess) {
            cudaGetLastError();
            return kLaunchFailed;
        }
    }

    bool ok = true;
    CUtensorMap map_n{}, map_k{};
    if (w.blocks != 0) {
        map_n = make_2d_tma_desc_u8_sw128(ws + w.codes_n, static_cast<uint64_t>(w.blocks) * 128, a.n, w.codes_ld_n, 128, ok);
        map_k = make_2d_tma_desc_u8_sw128(ws + w.codes_k, static_cast<uint64_t>(w.blocks) * 128, a.k, w.codes_ld_k, 128, ok);
    }
    if (!ok) return kTensorMapFailed;
    WgradParams p;
    p.groups = a.groups;
    p.max_blocks = w.blocks;
    p.n = a.n, p.k = a.k;
    p.scales_n = ws + w.scales_n, p.scales_k = ws + w.scales_k;
    p.out = a.out, p.out_ld = a.out_ld, p.out_group = a.out_group;
    p.accumulate = a.accumulate;
    const uint32_t vec = 4, item = a.out_bf16 ? 2 : 4;  // four columns at a time
    p.vector_store = is_aligned(a.out, vec * item) && a.out_ld % vec == 0 && a.out_group % vec == 0 && a.k % vec == 0;
    p.tiles = w.tiles, p.whole_tiles = w.whole_tiles;
    // A tile of 128 KB in fp32 leaves at 1/148 of the memory's rate in the time of about ten k-blocks.
    p.store_cost = (a.out_bf16 ? 5u : 10u) * (a.accumulate ? 2u : 1u);
    p.partials = reinterpret_cast<float4*>(ws + w.partials);
    p.counters = reinterpret_cast<uint32_t*>(ws + w.counters);
    p.status = a.status;
    p.timeout_ns = a.timeout_ns;
    cfg.gridDim = dim3(w.ctas);
    cfg.blockDim = dim3(384);
    cfg.dynamicSmemBytes = WgradTile::kSmemSize;
    auto kernel = a.out_bf16 ? fp8_wgrad_kernel<__nv_bfloat16> : fp8_wgrad_kernel<float>;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(WgradTile::kSmemSize)) != cudaSuccess ||
        cudaLaunchKernelEx(&cfg, kernel, p, map_n, map_k) != cudaSuccess) {
        cudaGetLastError();
        return kLaunchFailed;
    }
    return kOk;
}

}  // namespace yan
