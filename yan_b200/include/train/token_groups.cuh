#pragma once
// Groups of tokens (the rows that a router sent to one expert), given on the device, and their blocks of 128 rows.

#include <cstdint>

#include "../gemm/ptx.cuh"
#include "../gemm/utils.cuh"

namespace yan {

// Group g is rows [starts[g], starts[g] + sizes[g]) of a matrix of `rows` rows; sizes == nullptr: one group of all rows.
struct TokenGroups {
    const int* starts = nullptr;
    const int* sizes = nullptr;
    uint32_t num_groups = 1;
    uint32_t rows = 0;
};

constexpr uint32_t kMaxTokenGroups = 512;

// Blocks of 128 rows, and sets of four blocks, that disjoint groups can have in all.
__host__ __device__ constexpr uint32_t max_token_blocks(uint32_t rows, uint32_t groups, bool grouped) {
    return grouped ? rows / 128 + groups : ceil_div(rows, 128u);
}
__host__ __device__ constexpr uint32_t max_token_quads(uint32_t blocks, uint32_t groups) { return blocks / 4 + groups; }

// First block and first quad of every group, and the totals behind the last.
struct TokenBlockTable {
    uint32_t block[kMaxTokenGroups + 1];
    uint32_t quad[kMaxTokenGroups + 1];
};

__device__ __forceinline__ uint32_t group_start(const TokenGroups& g, uint32_t i) {
    return g.sizes == nullptr ? 0u : static_cast<uint32_t>(min(max(ptx::ld_global(g.starts + i), 0), static_cast<int>(g.rows)));
}
// Rows of the group that the matrix has: what lies outside of it is never touched, whatever the lists hold.
__device__ __forceinline__ uint32_t group_size(const TokenGroups& g, uint32_t i) {
    if (g.sizes == nullptr) return g.rows;
    return min(static_cast<uint32_t>(max(ptx::ld_global(g.sizes + i), 0)), g.rows - group_start(g, i));
}

// Called by one whole warp.  Groups that overlap could have more blocks than there is room for: those get none.
__device__ __forceinline__ void build_token_blocks(const TokenGroups& g, uint32_t max_blocks, TokenBlockTable& table) {
    const uint32_t lane = ptx::lane_id();
    uint32_t block = 0, quad = 0;
    for (uint32_t first = 0; first < g.num_groups; first += 32) {
        const uint32_t i = first + lane;
        uint32_t blocks = i < g.num_groups ? ceil_div(group_size(g, i), 128u) : 0u, until = blocks;
#pragma unroll
        for (uint32_t off = 1; off < 32; off *= 2) {
            const uint32_t v = __shfl_up_sync(0xffffffffu, until, off);
            if (lane >= off) until += v;
        }
        const uint32_t at = min(block + until - blocks, max_blocks);
        blocks = min(block + until, max_blocks) - at;
        uint32_t quads = ceil_div(blocks, 4u), quads_until = quads;
#pragma unroll
        for (uint32_t off = 1; off < 32; off *= 2) {
            const uint32_t v = __shfl_up_sync(0xffffffffu, quads_until, off);
            if (lane >= off) quads_until += v;
        }
        if (i < g.num_groups) {
            table.block[i] = at;
            table.quad[i] = quad + quads_until - quads;
        }
        block = min(block + __shfl_sync(0xffffffffu, until, 31), max_blocks);
        quad += __shfl_sync(0xffffffffu, quads_until, 31);
    }
    if (lane == 0) {
        table.block[g.num_groups] = block;
        table.quad[g.num_groups] = quad;
    }
    __syncwarp();
}

// The group that a block belongs to (block < table.block[num_groups]).
__device__ __forceinline__ uint32_t group_of_block(const TokenBlockTable& table, uint32_t num_groups, uint32_t block) {
    uint32_t low = 0, high = num_groups;  // table.block[low] <= block < table.block[high]
    while (high - low > 1) {
        const uint32_t mid = (low + high) / 2;
        if (table.block[mid] <= block) low = mid;
        else high = mid;
    }
    return low;
}

}  // namespace yan
