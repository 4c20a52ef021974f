#pragma once
// One AdamW step over many tensors in one launch.  Per element, in fp32, each operation rounded by itself:
//     g = grad * grad_scale;  m = m b1 + g (1 - b1);  v = v b2 + (g g) (1 - b2);  r = sqrt(v)
//     p = p (1 - lr wd) - (m lr / (1 - b1^t)) / (r / sqrt(1 - b2^t) + eps)
// 8-bit states: blocks of 128 elements of a tensor, m and r as e4m3 codes times one power of two per block, the smallest 2^e with
// amax <= 448 * 2^e.  The root is kept instead of v because its range is half as many binades.  A root above zero never gets the code of
// zero (the next step would divide by the newest gradient alone): it rounds up to the smallest code.  This step uses m and r before
// they are rounded.  What is not finite gets the code of NaN and has no say in the block's scale; blocks below 2^-111 are zero.
//
// Bound by HBM: 28 bytes per element with fp32 states and gradients, 14 with 8-bit states and bf16 gradients, 2 more for a bf16 copy.

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include "../gemm/ptx.cuh"
#include "../gemm/utils.cuh"

namespace yan {

struct AdamwTensor {
    void* param;
    const void* grad;
    void* m;         // fp32, or e4m3 codes
    void* v;         // fp32, or e4m3 codes of the root
    float* m_scale;  // 8-bit states: one per 128 elements
    float* v_scale;
    __nv_bfloat16* copy;  // optional: the new parameters in bf16
    uint32_t numel_lo, numel_hi;
    float decay;     // 1 - lr * weight_decay
    uint32_t vector; // every pointer allows four elements at a time
};
static_assert(sizeof(AdamwTensor) == 72);

struct AdamwScalars {
    const float* grad_scale;  // optional, on the device
    float b1, one_minus_b1, b2, one_minus_b2, step_size, inv_root_correction, eps;
};

// The table of tensors travels with the launch (kernel parameters hold up to 32764 bytes), so that nothing about them has to be on the
// device beforehand.
template <uint32_t kCapacity>
struct AdamwParams {
    AdamwScalars s;
    uint32_t num_tensors;
    uint32_t first_chunk[kCapacity + 1];
    AdamwTensor tensor[kCapacity];
};
constexpr uint32_t kAdamwSmallCapacity = 48, kAdamwCapacity = 420;
static_assert(sizeof(AdamwParams<kAdamwSmallCapacity>) <= 4096 && sizeof(AdamwParams<kAdamwCapacity>) <= 32764);

constexpr uint32_t kAdamwThreads = 256, kAdamwBlocksPerWarp = 4;
constexpr uint32_t kAdamwChunk = kAdamwThreads / 32 * kAdamwBlocksPerWarp * 128;  // elements of one CTA

namespace detail {

// Four elements from index i on, fp32 or bf16.
template <typename T>
__device__ __forceinline__ void load4(const T* p, uint64_t i, uint32_t count, bool vector, float (&f)[4]) {
    if (vector && count == 4) {
        if constexpr (sizeof(T) == 4) {
            const float4 v = *reinterpret_cast<const float4*>(p + i);
            f[0] = v.x, f[1] = v.y, f[2] = v.z, f[3] = v.w;
        } else {
            const uint2 v = *reinterpret_cast<const uint2*>(p + i);
            f[0] = __uint_as_float(v.x << 16), f[1] = __uint_as_float(v.x & 0xFFFF0000u);
            f[2] = __uint_as_float(v.y << 16), f[3] = __uint_as_float(v.y & 0xFFFF0000u);
        }
    } else {
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) f[j] = j < count ? static_cast<float>(p[i + j]) : 0.0f;
    }
}

template <typename T>
__device__ __forceinline__ void store4(T* p, uint64_t i, uint32_t count, bool vector, const float (&f)[4]) {
    if (vector && count == 4) {
        if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<float4*>(p + i) = make_float4(f[0], f[1], f[2], f[3]);
        } else {
            const __nv_bfloat162 lo = __floats2bfloat162_rn(f[0], f[1]), hi = __floats2bfloat162_rn(f[2], f[3]);
            *reinterpret_cast<uint2*>(p + i) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
        }
    } else {
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j)
            if (j < count) p[i + j] = static_cast<T>(f[j]);
    }
}

__device__ __forceinline__ void decode4(uint32_t codes, float scale, float (&f)[4]) {
    const __half2 lo(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(codes & 0xFFFFu), __NV_E4M3));
    const __half2 hi(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(codes >> 16), __NV_E4M3));
    const float2 a = __half22float2(lo), b = __half22float2(hi);
    f[0] = a.x * scale, f[1] = a.y * scale, f[2] = b.x * scale, f[3] = b.y * scale;
}

// Codes of a warp's block of 128, four elements per lane, and its power of two.  Called by whole warps.
template <bool kRoot>
__device__ __forceinline__ uint32_t encode4(const float (&f)[4], float& scale) {
    uint32_t amax = 0;
    bool finite[4];
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) {
        const uint32_t magnitude = __float_as_uint(f[j]) & 0x7FFFFFFFu;
        finite[j] = magnitude < 0x7F800000u;
        amax = max(amax, finite[j] ? magnitude : 0u);
    }
    amax = __reduce_max_sync(0xffffffffu, amax);
    const bool known = amax >= (16u << 23);
    const uint32_t e = (amax >> 23) - 8u + ((amax & 0x7FFFFFu) > 0x600000u ? 1u : 0u);
    scale = known ? __uint_as_float(e << 23) : 0.0f;
    const float inverse = known ? __uint_as_float((254u - e) << 23) : 0.0f;
    const float smallest = known ? 0.001953125f : 0.0f;  // code 1
    float t[4];
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) {
        t[j] = f[j] * inverse;
        if constexpr (kRoot) t[j] = fmaxf(t[j], f[j] > 0.0f ? smallest : 0.0f);
        t[j] = finite[j] ? t[j] : __uint_as_float(0x7FFFFFFFu);
    }
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(t[0], t[1]), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(t[2], t[3]), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
}

__device__ __forceinline__ uint32_t load_codes(const uint8_t* p, uint64_t i, uint32_t count, bool vector) {
    if (vector && count == 4) return *reinterpret_cast<const uint32_t*>(p + i);
    uint32_t w = 0;
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) w |= j < count ? static_cast<uint32_t>(p[i + j]) << (8 * j) : 0u;
    return w;
}
__device__ __forceinline__ void store_codes(uint8_t* p, uint64_t i, uint32_t count, bool vector, uint32_t codes) {
    if (vector && count == 4) {
        *reinterpret_cast<uint32_t*>(p + i) = codes;
        return;
    }
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j)
        if (j < count) p[i + j] = static_cast<uint8_t>(codes >> (8 * j));
}

}  // namespace detail

// One CTA per chunk; a warp takes kAdamwBlocksPerWarp blocks of 128 elements, four elements per lane each, and has their loads in
// flight together.
template <typename param_t, typename grad_t, bool k8Bit, uint32_t kCapacity>
__global__ void __launch_bounds__(kAdamwThreads) adamw_kernel(const __grid_constant__ AdamwParams<kCapacity> p) {
    ptx::grid_dependency_wait();
    uint32_t low = 0, high = p.num_tensors;  // first_chunk[low] <= blockIdx.x < first_chunk[high]
    while (high - low > 1) {
        const uint32_t mid = (low + high) / 2;
        if (p.first_chunk[mid] <= blockIdx.x) low = mid;
        else high = mid;
    }
    const AdamwTensor& t = p.tensor[low];
    const uint64_t numel = t.numel_lo | (static_cast<uint64_t>(t.numel_hi) << 32);
    const bool vector = t.vector != 0;
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint64_t start = static_cast<uint64_t>(blockIdx.x - p.first_chunk[low]) * kAdamwChunk + warp * (kAdamwBlocksPerWarp * 128u) + lane * 4u;
    param_t* param = static_cast<param_t*>(t.param);
    const grad_t* grad = static_cast<const grad_t*>(t.grad);
    const float grad_scale = p.s.grad_scale != nullptr ? *p.s.grad_scale : 1.0f;

    float pv[kAdamwBlocksPerWarp][4], g[kAdamwBlocksPerWarp][4], m[kAdamwBlocksPerWarp][4], v[kAdamwBlocksPerWarp][4];
    uint32_t count[kAdamwBlocksPerWarp];
    [[maybe_unused]] uint32_t mc[kAdamwBlocksPerWarp], vc[kAdamwBlocksPerWarp];
    [[maybe_unused]] float ms[kAdamwBlocksPerWarp], vs[kAdamwBlocksPerWarp];
#pragma unroll
    for (uint32_t b = 0; b < kAdamwBlocksPerWarp; ++b) {
        const uint64_t i = start + b * 128u;
        count[b] = i < numel ? static_cast<uint32_t>(min(numel - i, static_cast<uint64_t>(4))) : 0u;
        detail::load4(param, i, count[b], vector, pv[b]);
        detail::load4(grad, i, count[b], vector, g[b]);
        if constexpr (k8Bit) {
            mc[b] = detail::load_codes(static_cast<const uint8_t*>(t.m), i, count[b], vector);
            vc[b] = detail::load_codes(static_cast<const uint8_t*>(t.v), i, count[b], vector);
            const bool any = i - lane * 4u < numel;
            ms[b] = any ? t.m_scale[i / 128u] : 0.0f;
            vs[b] = any ? t.v_scale[i / 128u] : 0.0f;
        } else {
            detail::load4(static_cast<const float*>(t.m), i, count[b], vector, m[b]);
            detail::load4(static_cast<const float*>(t.v), i, count[b], vector, v[b]);
        }
    }
#pragma unroll
    for (uint32_t b = 0; b < kAdamwBlocksPerWarp; ++b) {
        const uint64_t i = start + b * 128u;
        if constexpr (k8Bit) {
            detail::decode4(mc[b], ms[b], m[b]);
            detail::decode4(vc[b], vs[b], v[b]);
        }
        float root[4];
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            const float gj = __fmul_rn(g[b][j], grad_scale);
            if constexpr (k8Bit) v[b][j] = __fmul_rn(v[b][j], v[b][j]);
            m[b][j] = __fadd_rn(__fmul_rn(m[b][j], p.s.b1), __fmul_rn(gj, p.s.one_minus_b1));
            v[b][j] = __fadd_rn(__fmul_rn(v[b][j], p.s.b2), __fmul_rn(__fmul_rn(gj, gj), p.s.one_minus_b2));
            root[j] = __fsqrt_rn(v[b][j]);
            const float update = __fdividef(m[b][j] * p.s.step_size, fmaf(root[j], p.s.inv_root_correction, p.s.eps));
            pv[b][j] = fmaf(pv[b][j], t.decay, -update);
        }
        detail::store4(param, i, count[b], vector, pv[b]);
        if (t.copy != nullptr) detail::store4(t.copy, i, count[b], vector, pv[b]);
        if constexpr (k8Bit) {
            float m_scale, v_scale;
            const uint32_t m_codes = detail::encode4<false>(m[b], m_scale), v_codes = detail::encode4<true>(root, v_scale);
            detail::store_codes(static_cast<uint8_t*>(t.m), i, count[b], vector, m_codes);
            detail::store_codes(static_cast<uint8_t*>(t.v), i, count[b], vector, v_codes);
            if (lane == 0 && i < numel) {
                t.m_scale[i / 128u] = m_scale;
                t.v_scale[i / 128u] = v_scale;
            }
        } else {
            detail::store4(static_cast<float*>(t.m), i, count[b], vector, m[b]);
            detail::store4(static_cast<float*>(t.v), i, count[b], vector, v[b]);
        }
    }
}

// ---------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------
template <typename param_t, typename grad_t, bool k8Bit, uint32_t kCapacity>
inline int launch_adamw_as(const AdamwParams<kCapacity>& p, cudaStream_t stream) {
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.first_chunk[p.num_tensors]);
    cfg.blockDim = dim3(kAdamwThreads);
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, adamw_kernel<param_t, grad_t, k8Bit, kCapacity>, p) != cudaSuccess) {
        cudaGetLastError();
        return kLaunchFailed;
    }
    return kOk;
}

template <uint32_t kCapacity>
inline int launch_adamw(const AdamwParams<kCapacity>& p, bool param_bf16, bool grad_bf16, bool eight_bit, cudaStream_t stream) {
    using B = __nv_bfloat16;
    if (param_bf16) {
        if (grad_bf16) return eight_bit ? launch_adamw_as<B, B, true>(p, stream) : launch_adamw_as<B, B, false>(p, stream);
        return eight_bit ? launch_adamw_as<B, float, true>(p, stream) : launch_adamw_as<B, float, false>(p, stream);
    }
    if (grad_bf16) return eight_bit ? launch_adamw_as<float, B, true>(p, stream) : launch_adamw_as<float, B, false>(p, stream);
    return eight_bit ? launch_adamw_as<float, float, true>(p, stream) : launch_adamw_as<float, float, false>(p, stream);
}

}  // namespace yan
