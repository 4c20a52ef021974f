#pragma once
// tcgen05 products of e4m3 operands whose scales the tensor core applies (kind::mxf8f6f4): one power of two (UE8M0, a byte that
// stands for 2^(byte - 127)) per row and 32 values of the summed dimension.  Here a scale holds for 128 values, so the four
// instructions of a 128-wide k-block name the same byte.
//
// Operands are M- (N-) major: a k-block of a [tokens, features] matrix is 128 rows (tokens, the summed dimension) of 128 bytes
// (features) in shared memory, as TMA writes them with the 128-byte swizzle, and the tensor core transposes on its way.
//
// Scales in tensor memory: the byte of row r is in lane r % 32 (and again in lanes 32.., 64.., 96..), column r / 32, and the four bytes of
// that 32-bit cell belong to four successive k-blocks.  `scale_tile` is that cell block of 128 rows and four k-blocks as 512 bytes in
// memory, [row % 32][row / 32][k-block % 4], which tcgen05.cp.32x128b.warpx4 copies as it stands.

#include <cstdint>

#include "../gemm/mma_utils.cuh"
#include "../gemm/ptx.cuh"

namespace yan {

constexpr uint32_t kScaleTileBytes = 512;  // 128 rows x 4 k-blocks

// Byte of (row, k-block) in its scale tile; row < 128, kb < 4.
__host__ __device__ constexpr uint32_t scale_tile_offset(uint32_t row, uint32_t kb) { return (row % 32) * 16 + (row / 32) * 4 + kb; }

// --- instruction descriptor for kind::mxf8f6f4 ---
//  [4,6)  which byte of a cell holds B's scale   [7,10), [10,13) formats: 0 = e4m3   [15], [16] A, B are M- / N-major
//  [17,23) N >> 3   [23] scale format: 1 = UE8M0   [24,29) M >> 4   [29,31) which byte holds A's scale
__host__ __device__ constexpr uint32_t make_instr_desc_mx_mn_major(uint32_t umma_m, uint32_t umma_n) {
    return (1u << 15) | (1u << 16) | ((umma_n >> 3) << 17) | (1u << 23) | ((umma_m >> 4) << 24);
}
__device__ __forceinline__ uint32_t with_scale_byte(uint32_t idesc, uint32_t byte) { return idesc | (byte << 4) | (byte << 29); }

// --- shared-memory descriptor of an M-major operand, 128-byte swizzle, in halves ---
// Stride offset: from 8 rows of the summed dimension to the next 8 (1024 bytes); leading offset: from 128 features to the next 128
// (a box of 128 x 128 bytes).  The high word is that of a K-major operand.
constexpr uint32_t kMnBoxBytes = 128 * 128;
__device__ __forceinline__ uint32_t make_smem_desc_mn_major_low(uint32_t smem_addr) {
    return ((smem_addr & 0x3FFFFu) >> 4) | ((kMnBoxBytes >> 4) << 16);
}
// 32 values of the summed dimension are 32 rows of 128 bytes.
constexpr uint32_t kMnKStep = (kUmmaK * 128) >> 4;

// --- shared-memory descriptor of a scale tile: 32 rows of 16 bytes, 8 of them (128 bytes) per core matrix, no swizzle ---
__device__ __forceinline__ uint64_t make_smem_desc_scales(uint32_t smem_addr) {
    return static_cast<uint64_t>((smem_addr & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(128 >> 4) << 32) | (static_cast<uint64_t>(1) << 46);
}

namespace ptx {

// ---- pairs of CTAs (cta_group::2): rank 0 issues the products of both; each CTA keeps its own 128 rows of A and of the sums, and half
// of B's columns in its shared memory ----

__device__ __forceinline__ void tmem_alloc_pair(uint32_t* smem_slot, uint32_t ncols) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(smem_slot)), "r"(ncols) : "memory");
}
__device__ __forceinline__ void tmem_relinquish_alloc_permit_pair() {
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc_pair(uint32_t taddr, uint32_t ncols) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}

// 512 bytes of scales, shared memory -> four columns of tensor memory, in all four lane quarters, in both CTAs (each from its own shared
// memory).  Issued by the thread that issues the products; a product issued behind it sees the scales.
__device__ __forceinline__ void tmem_copy_scales_pair(uint32_t taddr, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

// Descriptors by their low words.
__device__ __forceinline__ void umma_mxf8f6f4_ss_pair(uint32_t tmem_d, uint32_t desc_a_low, uint32_t desc_b_low, uint32_t idesc,
                                                      uint32_t tmem_scale_a, uint32_t tmem_scale_b, bool accumulate) {
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        ".reg .b64 a, b;\n\t"
        "mov.b64 a, {%1, %7};\n\t"
        "mov.b64 b, {%2, %7};\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], a, b, %3, [%4], [%5], p;\n\t"
        "}\n" ::"r"(tmem_d),
        "r"(desc_a_low), "r"(desc_b_low), "r"(idesc), "r"(tmem_scale_a), "r"(tmem_scale_b), "r"(static_cast<uint32_t>(accumulate)),
        "n"(kDescHigh)
        : "memory");
}

// Arrives on the barrier at this place in both CTAs once what this thread has issued so far is complete.
__device__ __forceinline__ void umma_commit_pair(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
                 "h"(static_cast<uint16_t>(3))
                 : "memory");
}

// A tile into this CTA's shared memory whose bytes complete a barrier of the pair (`bar`: an address in the cluster's shared memory).
__device__ __forceinline__ void tma_load_2d_pair(void* smem_dst, const CUtensorMap* desc, uint32_t bar, int32_t c_inner, int32_t c_outer) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(
            smem_u32(smem_dst)),
        "l"(reinterpret_cast<uint64_t>(desc)), "r"(bar), "r"(c_inner), "r"(c_outer)
        : "memory");
}

// Says that tensor memory has been read (tcgen05.wait::ld and tcgen05.fence::before_thread_sync lie in front of it), nothing about other
// memory: with release semantics it would wait for every store of the warp before it.
__device__ __forceinline__ void mbar_arrive_cluster_relaxed(uint32_t bar) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

}  // namespace ptx
}  // namespace yan
