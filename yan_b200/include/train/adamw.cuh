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
    float minus_zero = -0.0f;  // see rounded_product2
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

// A CTA is 256 threads whose warps take kBlocksPerWarp blocks of 128 elements each, all loads in flight together.  8-bit states bring
// fewer bytes per element and need more of them in flight: us for (200 M elements in 64 tensors, 12 M in 300) with one block 633, 39;
// two 591, 37; four at 64 registers per thread 532, 39 and at 80 648, 46; eight 526, 57.  32-bit states: (120 M elements in 12 tensors,
// 120 thousand in 48) with one block 523, 2.9; two 525, 3.4; four 523, 4.9.
template <bool k8Bit>
struct AdamwShape {
    static constexpr uint32_t kThreads = 256, kBlocksPerWarp = k8Bit ? 4 : 1, kMinCtas = k8Bit ? 4 : 1;
    static constexpr uint32_t kChunk = kThreads / 32 * kBlocksPerWarp * 128;  // elements of one CTA
};
constexpr uint32_t adamw_chunk(bool eight_bit) { return eight_bit ? AdamwShape<true>::kChunk : AdamwShape<false>::kChunk; }

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

// The power of two of a block and its reciprocal from the bits of its largest magnitude (finite): adding 0x1FFFFF carries into the exponent
// exactly where the significand is above 1.75.
__device__ __forceinline__ void block_scale(uint32_t amax, float& scale, float& inverse) {
    const uint32_t bits = ((amax + 0x1FFFFFu) & 0x7F800000u) - (8u << 23);
    const bool known = amax >= (16u << 23);
    scale = known ? __uint_as_float(bits) : 0.0f;
    inverse = known ? __uint_as_float((254u << 23) - bits) : 0.0f;
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
    float inverse;
    block_scale(amax, scale, inverse);
    const float smallest = scale != 0.0f ? 0.001953125f : 0.0f;  // code 1
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

// Two fp32 operations with one instruction, each rounded like the single one.
__device__ __forceinline__ uint64_t pack2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
// A product that is rounded by itself: a product of two feeds an addition of two as one fused operation, whatever rounding the
// instructions name (1.6 of 16.8 million sums came out differently); an fma onto a -0 that the compiler does not know is not fused again.
__device__ __forceinline__ uint64_t rounded_product2(uint64_t a, uint64_t b, float minus_zero) {
    return fma2(a, b, pack2(minus_zero, minus_zero));
}
__device__ __forceinline__ float approximate_rsqrt(float x) {
    float r;
    asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float approximate_reciprocal(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float max_or_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// One element; m and v become the new moments.
__device__ __forceinline__ void update_element(const AdamwScalars& c, float grad_scale, float decay, float& param, float grad, float& m, float& v,
                                               float& root) {
    const float g = __fmul_rn(grad, grad_scale);
    m = __fadd_rn(__fmul_rn(m, c.b1), __fmul_rn(g, c.one_minus_b1));
    v = __fadd_rn(__fmul_rn(v, c.b2), __fmul_rn(__fmul_rn(g, g), c.one_minus_b2));
    root = __fsqrt_rn(v);
    const float reciprocal = approximate_reciprocal(fmaf(root, c.inv_root_correction, c.eps));
    param = fmaf(__fmul_rn(m, -c.step_size), reciprocal, __fmul_rn(param, decay));
}

// One block of 128 elements, four per lane, 8-bit states: updates param, codes and scales in registers.  The same operations as
// update_element, two at a time; the root by one Newton step from the hardware's reciprocal root in the form of Markstein (s = v y,
// s + (v - s^2) y / 2), which rounds like sqrt for what is finite.  Returns false, with nothing changed, if an m or v is not finite.
__device__ __forceinline__ bool update_block_8bit(const AdamwScalars& c, float grad_scale, float decay, float (&param)[4], const float (&grad)[4],
                                                  uint32_t& m_codes, uint32_t& v_codes, float& m_scale, float& v_scale) {
    float md[4], rd[4];
    decode4(m_codes, m_scale, md);
    decode4(v_codes, v_scale, rd);
    uint64_t m[2], v[2], root[2];
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h) {
        const uint64_t g = mul2(pack2(grad[2 * h], grad[2 * h + 1]), pack2(grad_scale, grad_scale));
        const uint64_t old_root = pack2(rd[2 * h], rd[2 * h + 1]);
        m[h] = add2(rounded_product2(pack2(md[2 * h], md[2 * h + 1]), pack2(c.b1, c.b1), c.minus_zero),
                    rounded_product2(g, pack2(c.one_minus_b1, c.one_minus_b1), c.minus_zero));
        v[h] = add2(rounded_product2(mul2(old_root, old_root), pack2(c.b2, c.b2), c.minus_zero),
                    rounded_product2(mul2(g, g), pack2(c.one_minus_b2, c.one_minus_b2), c.minus_zero));
        float a, b;
        unpack2(v[h], a, b);
        // zero: s = 0 * y and its correction are zero, whatever the y
        const uint64_t y = pack2(approximate_rsqrt(fmaxf(a, 1.2e-38f)), approximate_rsqrt(fmaxf(b, 1.2e-38f)));
        const uint64_t s = mul2(v[h], y), minus_s = mul2(s, pack2(-1.0f, -1.0f));
        root[h] = fma2(fma2(minus_s, s, v[h]), mul2(y, pack2(0.5f, 0.5f)), s);
    }
    float ma[4], ra[4], va[4];
    unpack2(m[0], ma[0], ma[1]), unpack2(m[1], ma[2], ma[3]);
    unpack2(root[0], ra[0], ra[1]), unpack2(root[1], ra[2], ra[3]);
    unpack2(v[0], va[0], va[1]), unpack2(v[1], va[2], va[3]);
    const float m_top = max_or_nan(max_or_nan(fabsf(ma[0]), fabsf(ma[1])), max_or_nan(fabsf(ma[2]), fabsf(ma[3])));
    const float r_top = max_or_nan(max_or_nan(ra[0], ra[1]), max_or_nan(ra[2], ra[3]));  // NaN where v is not finite
    const uint32_t m_amax = __reduce_max_sync(0xffffffffu, __float_as_uint(m_top) & 0x7FFFFFFFu);
    const uint32_t r_amax = __reduce_max_sync(0xffffffffu, __float_as_uint(r_top) & 0x7FFFFFFFu);
    if (max(m_amax, r_amax) >= 0x7F800000u) return false;
    float m_inverse, r_inverse;
    block_scale(m_amax, m_scale, m_inverse);
    block_scale(r_amax, v_scale, r_inverse);
    const float smallest = v_scale != 0.0f ? 0.001953125f : 0.0f;  // code 1
    uint32_t mw[2], rw[2];
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h) {
        float a, b;
        unpack2(mul2(m[h], pack2(m_inverse, m_inverse)), a, b);
        mw[h] = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
        unpack2(mul2(root[h], pack2(r_inverse, r_inverse)), a, b);
        a = fmaxf(a, ra[2 * h] > 0.0f ? smallest : 0.0f), b = fmaxf(b, ra[2 * h + 1] > 0.0f ? smallest : 0.0f);
        rw[h] = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
        const uint64_t denominator = fma2(root[h], pack2(c.inv_root_correction, c.inv_root_correction), pack2(c.eps, c.eps));
        unpack2(denominator, a, b);
        const uint64_t step = mul2(m[h], pack2(-c.step_size, -c.step_size));
        const uint64_t kept = mul2(pack2(param[2 * h], param[2 * h + 1]), pack2(decay, decay));
        unpack2(fma2(step, pack2(approximate_reciprocal(a), approximate_reciprocal(b)), kept), param[2 * h], param[2 * h + 1]);
    }
    m_codes = mw[0] | (mw[1] << 16);
    v_codes = rw[0] | (rw[1] << 16);
    return true;
}

}  // namespace detail

// One CTA per chunk of a tensor, four elements of a block of 128 per lane.
template <typename param_t, typename grad_t, bool k8Bit, uint32_t kCapacity>
__global__ void __launch_bounds__(AdamwShape<k8Bit>::kThreads, AdamwShape<k8Bit>::kMinCtas)
    adamw_kernel(const __grid_constant__ AdamwParams<kCapacity> p) {
    constexpr uint32_t kBlocks = AdamwShape<k8Bit>::kBlocksPerWarp, kWarps = AdamwShape<k8Bit>::kThreads / 32;
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
    // the warp's blocks are kWarps apart, so that a short tensor occupies all warps
    const uint64_t start = static_cast<uint64_t>(blockIdx.x - p.first_chunk[low]) * AdamwShape<k8Bit>::kChunk + warp * 128u;
    if (start >= numel) return;
    const uint64_t mine = start + lane * 4u;
    param_t* param = static_cast<param_t*>(t.param) + mine;
    const grad_t* grad = static_cast<const grad_t*>(t.grad) + mine;
    __nv_bfloat16* copy = t.copy;
    const float grad_scale = p.s.grad_scale != nullptr ? *p.s.grad_scale : 1.0f;
    const uint64_t left = numel - start;  // elements from the warp's first block on

    float pv[kBlocks][4], g[kBlocks][4], m[kBlocks][4], v[kBlocks][4];
    if constexpr (k8Bit) {
        uint8_t *mp = static_cast<uint8_t*>(t.m) + mine, *vp = static_cast<uint8_t*>(t.v) + mine;
        float *msp = t.m_scale + start / 128u, *vsp = t.v_scale + start / 128u;
        uint32_t todo = (1u << kBlocks) - 1;  // blocks of the warp to be done
        auto store = [&](uint32_t b, const float (&pb)[4], uint32_t m_codes, uint32_t v_codes, float m_scale, float v_scale) {
            const uint32_t at = b * kWarps * 128u;
            detail::store4(param, at, 4, true, pb);
            if (copy != nullptr) detail::store4(copy + mine, at, 4, true, pb);
            detail::store_codes(mp, at, 4, true, m_codes);
            detail::store_codes(vp, at, 4, true, v_codes);
            if (lane == 0) {
                msp[b * kWarps] = m_scale;
                vsp[b * kWarps] = v_scale;
            }
            todo &= ~(1u << b);
        };
        // All blocks whole, in a tensor whose pointers allow four elements at a time: every load in flight before the first is used.  What
        // bounds it is the number of instructions: written like the general form below, 371 per 128 elements, 200 M elements took
        // 957 us; with a condition for each block's loads 610, without 532.
        if (vector && left >= ((kBlocks - 1) * kWarps + 1) * 128u) {
            float ms[kBlocks], vs[kBlocks];
            uint32_t mc[kBlocks], vc[kBlocks];
#pragma unroll
            for (uint32_t b = 0; b < kBlocks; ++b) {
                const uint32_t at = b * kWarps * 128u;
                detail::load4(param, at, 4, true, pv[b]);
                detail::load4(grad, at, 4, true, g[b]);
                mc[b] = detail::load_codes(mp, at, 4, true);
                vc[b] = detail::load_codes(vp, at, 4, true);
                ms[b] = msp[b * kWarps];
                vs[b] = vsp[b * kWarps];
            }
#pragma unroll
            for (uint32_t b = 0; b < kBlocks; ++b)
                if (detail::update_block_8bit(p.s, grad_scale, t.decay, pv[b], g[b], mc[b], vc[b], ms[b], vs[b]))
                    store(b, pv[b], mc[b], vc[b], ms[b], vs[b]);
        }
        // The end of a tensor, any alignment, something that is not finite: block by block.
#pragma unroll 1
        for (; todo != 0; todo &= todo - 1) {
            const uint32_t b = __ffs(static_cast<int>(todo)) - 1, at = b * kWarps * 128u;
            if (left <= at) break;
            const uint32_t count = left > at + lane * 4u ? static_cast<uint32_t>(min(left - at - lane * 4u, static_cast<uint64_t>(4))) : 0u;
            float pb[4], gb[4], mb[4], vb[4], root[4], m_scale = msp[b * kWarps], v_scale = vsp[b * kWarps];
            detail::load4(param, at, count, vector, pb);
            detail::load4(grad, at, count, vector, gb);
            uint32_t m_codes = detail::load_codes(mp, at, count, vector), v_codes = detail::load_codes(vp, at, count, vector);
            if (vector && left >= at + 128u && detail::update_block_8bit(p.s, grad_scale, t.decay, pb, gb, m_codes, v_codes, m_scale, v_scale)) {
                store(b, pb, m_codes, v_codes, m_scale, v_scale);
                todo |= 1u << b;  // for the step of the loop
                continue;
            }
            detail::decode4(m_codes, m_scale, mb);
            detail::decode4(v_codes, v_scale, vb);
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) {
                vb[j] = __fmul_rn(vb[j], vb[j]);
                detail::update_element(p.s, grad_scale, t.decay, pb[j], gb[j], mb[j], vb[j], root[j]);
            }
            m_codes = detail::encode4<false>(mb, m_scale), v_codes = detail::encode4<true>(root, v_scale);
            detail::store4(param, at, count, vector, pb);
            if (copy != nullptr) detail::store4(copy + mine, at, count, vector, pb);
            detail::store_codes(mp, at, count, vector, m_codes);
            detail::store_codes(vp, at, count, vector, v_codes);
            __syncwarp();  // every lane has read the scales
            if (lane == 0) {
                msp[b * kWarps] = m_scale;
                vsp[b * kWarps] = v_scale;
            }
        }
    } else {
        float *mp = static_cast<float*>(t.m) + mine, *vp = static_cast<float*>(t.v) + mine;
        uint32_t count[kBlocks];
#pragma unroll
        for (uint32_t b = 0; b < kBlocks; ++b) {
            const uint32_t at = b * kWarps * 128u;
            count[b] = left > at + lane * 4u ? static_cast<uint32_t>(min(left - at - lane * 4u, static_cast<uint64_t>(4))) : 0u;
            detail::load4(param, at, count[b], vector, pv[b]);
            detail::load4(grad, at, count[b], vector, g[b]);
            detail::load4(mp, at, count[b], vector, m[b]);
            detail::load4(vp, at, count[b], vector, v[b]);
        }
#pragma unroll
        for (uint32_t b = 0; b < kBlocks; ++b) {
            const uint32_t at = b * kWarps * 128u;
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) {
                float root;
                detail::update_element(p.s, grad_scale, t.decay, pv[b][j], g[b][j], m[b][j], v[b][j], root);
            }
            detail::store4(param, at, count[b], vector, pv[b]);
            if (copy != nullptr) detail::store4(copy + mine, at, count[b], vector, pv[b]);
            detail::store4(mp, at, count[b], vector, m[b]);
            detail::store4(vp, at, count[b], vector, v[b]);
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
    cfg.blockDim = dim3(AdamwShape<k8Bit>::kThreads);
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
