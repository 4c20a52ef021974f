#pragma once
// Balance loss of a router over experts, its gradient and the selections per expert.  For the tokens t of sequence s that count, n_s of
// them, with p[t] = softmax(z[t]) or sigmoid(z[t]) / sum sigmoid(z[t]) over E experts and k selections per token:
//     c[s, e] = selections of e,  P[s, e] = sum over t of p[t, e],  a[s, e] = coef / S * E / (k n_s^2) * c[s, e]
//     loss = sum over s, e of a[s, e] * P[s, e]
//     softmax: dz_j = p_j (a_j - sum over e of a_e p_e);  sigmoid: dz_j = s_j (1 - s_j) / sum(s) * (a_j - sum over e of a_e p_e)
// Few tokens: one launch of one cluster of CTAs, whose sums meet in distributed shared memory.  Many: three launches, sums over strips of
// tokens, the sums of the strips with a and the loss, the gradient.  No sum depends on the order in which anything runs.
//
// A strip is a fixed range of tokens; it may touch several sequences, and the sums of (strip, sequence) go to slot strip + sequence:
// both grow along the tokens, so that no two pairs share a slot and those of one sequence follow one another.

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "../gemm/ptx.cuh"
#include "../gemm/utils.cuh"

namespace yan {

constexpr uint32_t kMaxBalanceExperts = 1024;
constexpr uint32_t kMaxBalanceTop = 65535;  // the cluster kernel, for few tokens, counts selections in 32 bits
constexpr uint32_t kBalanceThreads = 256, kBalanceWarps = kBalanceThreads / 32;

struct BalanceParams {
    const void* logits = nullptr;
    uint64_t logits_ld = 0;
    const void* ids = nullptr;            // [tokens][top], int64 or int32; what is no expert selects nothing
    uint32_t ids_64 = 0;
    const uint8_t* mask = nullptr;        // optional, [tokens]: 0 = does not count
    const int* cu_seqlens = nullptr;      // optional, [sequences + 1]
    uint32_t tokens = 0, experts = 0, top = 0, sequences = 1;
    uint32_t sigmoid = 0;
    float coef = 0.0f;
    float* loss = nullptr;
    int* counts = nullptr;                // [sequences][experts]
    void* grad = nullptr;                 // [tokens][grad_ld], optional
    uint64_t grad_ld = 0;
    uint32_t strips = 0, strip_tokens = 0;
    // scratch
    float* slot_sums = nullptr;           // [strips + sequences][experts]
    int* slot_counts = nullptr;           // the same
    int* slot_tokens = nullptr;           // [strips + sequences]
    float* weights = nullptr;             // a, [sequences][experts]
    float* losses = nullptr;              // [sequences][ceil(experts / 32)]
    float2* rows = nullptr;               // [tokens]: what the gradient needs of a row's softmax (largest logit, 1 / sum)
};

namespace detail {

// The ends of the sequences in shared memory, as far as they fit: every kernel searches and walks them, and each look at global memory
// would be a round trip to L2.  Ends with a barrier of the CTA; null without sequences.
constexpr uint32_t kMaxSharedSequences = 1024;
__device__ __forceinline__ const int* stage_sequences(const BalanceParams& p, int (&s_cu)[kMaxSharedSequences + 1]) {
    if (p.cu_seqlens == nullptr || p.sequences > kMaxSharedSequences) return p.cu_seqlens;
    for (uint32_t i = threadIdx.x; i <= p.sequences; i += blockDim.x) s_cu[i] = ptx::ld_global(p.cu_seqlens + i);
    __syncthreads();
    return s_cu;
}

// Tokens of sequence s that exist.
__device__ __forceinline__ void sequence_range(const BalanceParams& p, const int* cu, uint32_t s, uint32_t& begin, uint32_t& end) {
    if (cu == nullptr) {
        begin = 0, end = p.tokens;
        return;
    }
    const int limit = static_cast<int>(p.tokens);
    begin = min(max(cu[s], 0), limit);
    end = max(min(cu[s + 1], limit), static_cast<int>(begin));
}

// First sequence that ends behind `token` (sequences if there is none); ends do not decrease.
__device__ __forceinline__ uint32_t first_sequence_behind(const BalanceParams& p, const int* cu, uint32_t token) {
    if (cu == nullptr) return 0;
    uint32_t low = 0, high = p.sequences;
    while (low < high) {
        const uint32_t mid = (low + high) / 2;
        if (cu[mid + 1] > static_cast<int>(token)) high = mid;
        else low = mid + 1;
    }
    return low;
}

// How the experts of a row lie over the lanes: kLanes lanes per row, kIter times kVec neighbouring experts each.  A warp works on
// kRows rows per group of lanes at a time, while as many are on their way.  What bounds it is the number of instructions beside the loads:
// 150 for a row of 256 experts in either pass (131072 x 256: 32 us for the sums, 4.4 TB/s, and 42 us for the gradient, 5.1 TB/s; one row
// at a time, not fetched ahead, 63 and 62).
template <typename T, uint32_t kVec, uint32_t kLanes, uint32_t kIter>
struct BalanceRow {
    static constexpr uint32_t kPerLane = kVec * kIter, kGroups = 32 / kLanes;
    static constexpr uint32_t kRows = kPerLane <= 2 ? 4 : kPerLane <= 8 ? 2 : 1, kRowsPerWarp = kGroups * kRows;

    __device__ __forceinline__ static uint32_t column(uint32_t lane, uint32_t c) {
        return (c / kVec * kLanes + lane % kLanes) * kVec + c % kVec;
    }
    // A row that does not count, and experts that do not exist, read as -inf: probability zero.
    __device__ __forceinline__ static void load(const T* row, bool there, uint32_t experts, uint32_t lane, float (&z)[kPerLane]) {
#pragma unroll
        for (uint32_t i = 0; i < kIter; ++i) {
            const uint32_t col = column(lane, i * kVec);
            if constexpr (kVec == 1) {
                z[i] = there && col < experts ? static_cast<float>(row[col]) : -INFINITY;
            } else {
                const uint32_t nothing = sizeof(T) == 4 ? 0xFF800000u : 0xFF80FF80u;
                uint4 v = make_uint4(nothing, nothing, nothing, nothing);
                if (there && col < experts) v = *reinterpret_cast<const uint4*>(row + col);
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j) {
                    if constexpr (sizeof(T) == 4) {
                        z[i * 4 + j] = __uint_as_float(w[j]);
                    } else {
                        z[i * 8 + 2 * j] = __uint_as_float(w[j] << 16);
                        z[i * 8 + 2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
                    }
                }
            }
        }
    }
    // The gradient is not read again here: it leaves L2 before the logits do.
    __device__ __forceinline__ static void store(T* row, uint32_t experts, uint32_t lane, const float (&z)[kPerLane]) {
#pragma unroll
        for (uint32_t i = 0; i < kIter; ++i) {
            const uint32_t col = column(lane, i * kVec);
            if (col >= experts) continue;
            if constexpr (kVec == 1) {
                row[col] = static_cast<T>(z[i]);
            } else if constexpr (sizeof(T) == 4) {
                __stcs(reinterpret_cast<float4*>(row + col), make_float4(z[i * 4], z[i * 4 + 1], z[i * 4 + 2], z[i * 4 + 3]));
            } else {
                uint32_t w[4];
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j) {
                    const __nv_bfloat162 t = __floats2bfloat162_rn(z[i * 8 + 2 * j], z[i * 8 + 2 * j + 1]);
                    w[j] = *reinterpret_cast<const uint32_t*>(&t);
                }
                __stcs(reinterpret_cast<uint4*>(row + col), make_uint4(w[0], w[1], w[2], w[3]));
            }
        }
    }
    __device__ __forceinline__ static float sum(float v) {
#pragma unroll
        for (uint32_t off = kLanes / 2; off >= 1; off /= 2) v += __shfl_xor_sync(0xffffffffu, v, off);
        return v;
    }
    __device__ __forceinline__ static float largest(float v) {
        if constexpr (kLanes == 32) {
            float r;
            asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
            return r;
        } else {
#pragma unroll
            for (uint32_t off = kLanes / 2; off >= 1; off /= 2) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, off));
            return v;
        }
    }
    // z -> scores before they are divided by their sum; `shift` is the largest logit (softmax).
    __device__ __forceinline__ static void scores(bool sigmoid, float (&z)[kPerLane], float shift) {
        if (sigmoid) {
#pragma unroll
            for (uint32_t c = 0; c < kPerLane; ++c) z[c] = __fdividef(1.0f, 1.0f + __expf(-z[c]));
        } else {
#pragma unroll
            for (uint32_t c = 0; c < kPerLane; ++c) z[c] = __expf(z[c] - shift);
        }
    }

    // Rows of one turn of a warp, on their way.
    struct Batch {
        float z[kRows][kPerLane];
        bool counts[kRows];

        // Tokens from `base` on, kGroups apart; those that count lie in [begin, end).
        __device__ __forceinline__ void load(const BalanceParams& p, uint32_t base, uint32_t begin, uint32_t end, uint32_t lane) {
#pragma unroll
            for (uint32_t r = 0; r < kRows; ++r) {
                const uint32_t token = base + r * kGroups + lane / kLanes;
                counts[r] = token >= begin && token < end && (p.mask == nullptr || p.mask[token] != 0);
                BalanceRow::load(static_cast<const T*>(p.logits) + static_cast<uint64_t>(token) * p.logits_ld, counts[r], p.experts, lane, z[r]);
            }
        }
    };

    // Takes the turns of a warp over tokens [from, end), the first to the last or backwards: the next turn's rows are fetched before this
    // one's are worked on.
    template <bool kBackwards, typename Work>
    __device__ __forceinline__ static void turns(const BalanceParams& p, uint32_t from, uint32_t begin, uint32_t end, uint32_t warp, uint32_t warps,
                                                 uint32_t lane, Work&& work) {
        const uint32_t first = from + warp * kRowsPerWarp, step = warps * kRowsPerWarp;
        if (first >= end) return;
        uint32_t left = ceil_div(end - first, step);  // turns
        uint32_t base = kBackwards ? first + (left - 1) * step : first;
        const uint32_t onward = kBackwards ? 0u - step : step;
        if constexpr (kPerLane > 16) {  // no registers for two
            Batch batch;
            for (; left != 0; --left, base += onward) {
                batch.load(p, base, begin, end, lane);
                work(batch, base);
            }
            return;
        }
        Batch batch[2];
        batch[0].load(p, base, begin, end, lane);
        for (;;) {
#pragma unroll
            for (uint32_t i = 0; i < 2; ++i) {
                if (left > 1) batch[i ^ 1].load(p, base + onward, begin, end, lane);
                work(batch[i], base);
                base += onward;
                if (--left == 0) return;
            }
        }
    }

    // Adds the probabilities of tokens [begin, end) that the warp has its turn for, and counts those that count.
    // rows[token - rows_from]: what their gradient needs, if there is to be one.
    __device__ __forceinline__ static void add(const BalanceParams& p, uint32_t begin, uint32_t end, uint32_t warp, uint32_t warps, uint32_t lane,
                                               float2* rows, uint32_t rows_from, float (&sums)[kPerLane], int& counted) {
        turns<false>(p, begin, begin, end, warp, warps, lane, [&](Batch& b, uint32_t base) {
            float shift[kRows], total[kRows];
#pragma unroll
            for (uint32_t r = 0; r < kRows; ++r) {
                shift[r] = 0.0f;
                if (p.sigmoid == 0) {
                    shift[r] = b.z[r][0];
#pragma unroll
                    for (uint32_t c = 1; c < kPerLane; ++c) shift[r] = fmaxf(shift[r], b.z[r][c]);
                    shift[r] = largest(shift[r]);
                    if (shift[r] == -INFINITY) shift[r] = 0.0f;
                }
            }
#pragma unroll
            for (uint32_t r = 0; r < kRows; ++r) {
                scores(p.sigmoid != 0, b.z[r], shift[r]);
                total[r] = 0.0f;
#pragma unroll
                for (uint32_t c = 0; c < kPerLane; ++c) total[r] += b.z[r][c];
                total[r] = sum(total[r]);
            }
#pragma unroll
            for (uint32_t r = 0; r < kRows; ++r) {
                const float inverse = total[r] == 0.0f ? 0.0f : __fdividef(1.0f, total[r]);  // a row of nothing but -inf has zeros
#pragma unroll
                for (uint32_t c = 0; c < kPerLane; ++c) sums[c] = fmaf(b.z[r][c], inverse, sums[c]);
                if (lane % kLanes == 0 && b.counts[r]) {
                    if (rows != nullptr) rows[base + r * kGroups + lane / kLanes - rows_from] = make_float2(shift[r], inverse);
                    ++counted;
                }
            }
        });
    }

    // The gradient of tokens [at, end) that the warp has its turn for; those in front of `begin` and those that do not count have zeros.
    __device__ __forceinline__ static void grad(const BalanceParams& p, uint32_t at, uint32_t begin, uint32_t end, uint32_t warp, uint32_t warps,
                                                uint32_t lane, const float2* rows, uint32_t rows_from, const float (&weights)[kPerLane]) {
        T* out = static_cast<T*>(p.grad);
        turns<true>(p, at, begin, end, warp, warps, lane, [&](Batch& b, uint32_t base) {
            float inner[kRows];
            float2 row[kRows];
#pragma unroll
            for (uint32_t r = 0; r < kRows; ++r)
                row[r] = b.counts[r] ? rows[base + r * kGroups + lane / kLanes - rows_from] : make_float2(0.0f, 0.0f);
#pragma unroll
            for (uint32_t r = 0; r < kRows; ++r) {
                scores(p.sigmoid != 0, b.z[r], row[r].x);
                inner[r] = 0.0f;
#pragma unroll
                for (uint32_t c = 0; c < kPerLane; ++c) inner[r] = fmaf(b.z[r][c], weights[c], inner[r]);
                inner[r] = sum(inner[r]);
            }
#pragma unroll
            for (uint32_t r = 0; r < kRows; ++r) {
                const uint32_t token = base + r * kGroups + lane / kLanes;
                inner[r] *= row[r].y;
#pragma unroll
                for (uint32_t c = 0; c < kPerLane; ++c) {
                    const float slope = p.sigmoid != 0 ? b.z[r][c] * (1.0f - b.z[r][c]) : b.z[r][c];
                    b.z[r][c] = b.counts[r] ? slope * row[r].y * (weights[c] - inner[r]) : 0.0f;
                }
                if (token < end) store(out + static_cast<uint64_t>(token) * p.grad_ld, p.experts, lane, b.z[r]);
            }
        });
    }
};

// Adds the selections of tokens [begin, end) that count to s_counts.
__device__ __forceinline__ void count_selections(const BalanceParams& p, uint32_t begin, uint32_t end, uint32_t thread, uint32_t threads,
                                                 int* s_counts) {
    const uint64_t first = static_cast<uint64_t>(begin) * p.top, last = static_cast<uint64_t>(end) * p.top;
    for (uint64_t at = first + thread; at < last; at += 4ull * threads) {
        int ids[4];  // in flight together
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            const uint64_t i = at + static_cast<uint64_t>(j) * threads;
            ids[j] = -1;
            if (i >= last) continue;
            const long long id = p.ids_64 != 0 ? static_cast<const long long*>(p.ids)[i] : static_cast<const int*>(p.ids)[i];
            if (id >= 0 && id < static_cast<long long>(p.experts)) ids[j] = static_cast<int>(id);
            if (p.mask != nullptr) {
                const uint32_t token = last <= 0xFFFFFFFFu ? static_cast<uint32_t>(i) / p.top : static_cast<uint32_t>(i / p.top);
                if (p.mask[token] == 0) ids[j] = -1;
            }
        }
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j)
            if (ids[j] >= 0) atomicAdd(&s_counts[ids[j]], 1);
    }
}

// a of an expert with `count` selections in a sequence of `tokens` that count.
__device__ __forceinline__ float balance_weight(const BalanceParams& p, int count, int tokens) {
    const float n = static_cast<float>(tokens);
    return tokens <= 0 ? 0.0f
                       : p.coef / static_cast<float>(p.sequences) * (static_cast<float>(p.experts) / (static_cast<float>(p.top) * n)) *
                             (static_cast<float>(count) / n);
}

}  // namespace detail

template <typename T, uint32_t kVec, uint32_t kLanes, uint32_t kIter>
__global__ void __launch_bounds__(kBalanceThreads, kVec * kIter <= 16 ? 3 : 1) balance_sums_kernel(const BalanceParams p) {
    using Row = detail::BalanceRow<T, kVec, kLanes, kIter>;
    constexpr uint32_t kPerLane = Row::kPerLane;
    extern __shared__ float s_sums[];  // [warps][experts]
    __shared__ int s_counts[kMaxBalanceExperts];
    __shared__ int s_tokens, s_cu[detail::kMaxSharedSequences + 1];
    ptx::grid_dependency_wait();
    ptx::grid_dependency_launch_dependents();  // the next launch waits for the end of this one before it reads anything
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t strip = blockIdx.x, first = strip * p.strip_tokens, last = min(first + p.strip_tokens, p.tokens);
    const int* cu = detail::stage_sequences(p, s_cu);
    for (uint32_t s = detail::first_sequence_behind(p, cu, first); s < p.sequences; ++s) {
        uint32_t begin, end;
        detail::sequence_range(p, cu, s, begin, end);
        if (begin >= last) break;
        begin = max(begin, first), end = min(end, last);
        if (begin >= end) continue;
        for (uint32_t e = threadIdx.x; e < p.experts; e += kBalanceThreads) s_counts[e] = 0;
        if (threadIdx.x == 0) s_tokens = 0;
        __syncthreads();
        detail::count_selections(p, begin, end, threadIdx.x, kBalanceThreads, s_counts);
        float sums[kPerLane];
#pragma unroll
        for (uint32_t c = 0; c < kPerLane; ++c) sums[c] = 0.0f;
        int counted = 0;
        Row::add(p, begin, end, warp, kBalanceWarps, lane, p.grad != nullptr ? p.rows : nullptr, 0, sums, counted);
        if (counted != 0) atomicAdd(&s_tokens, counted);
#pragma unroll
        for (uint32_t c = 0; c < kPerLane; ++c) {
#pragma unroll
            for (uint32_t off = kLanes; off < 32; off *= 2) sums[c] += __shfl_xor_sync(0xffffffffu, sums[c], off);
            const uint32_t col = Row::column(lane, c);
            if (lane < kLanes && col < p.experts) s_sums[warp * p.experts + col] = sums[c];
        }
        __syncthreads();
        const uint64_t slot = strip + s;
        for (uint32_t e = threadIdx.x; e < p.experts; e += kBalanceThreads) {
            float sum = 0.0f;
#pragma unroll
            for (uint32_t w = 0; w < kBalanceWarps; ++w) sum += s_sums[w * p.experts + e];
            p.slot_sums[slot * p.experts + e] = sum;
            p.slot_counts[slot * p.experts + e] = s_counts[e];
        }
        if (threadIdx.x == 0) p.slot_tokens[slot] = s_tokens;
        __syncthreads();
    }
}

// One CTA: 32 experts of one sequence; 32 warps share an expert's slots.
constexpr uint32_t kBalanceWeightWarps = 32;
__global__ void __launch_bounds__(kBalanceWeightWarps * 32) balance_weights_kernel(const BalanceParams p) {
    __shared__ float s_sum[kBalanceWeightWarps][32];
    __shared__ int s_count[kBalanceWeightWarps][32], s_tokens[kBalanceWeightWarps];
    ptx::grid_dependency_wait();
    ptx::grid_dependency_launch_dependents();
    const int* cu = p.cu_seqlens;
    const uint32_t s = blockIdx.y, lane = threadIdx.x % 32, e = blockIdx.x * 32 + lane, part = threadIdx.x / 32;
    uint32_t begin, end;
    detail::sequence_range(p, cu, s, begin, end);
    float sum = 0.0f;
    int count = 0, tokens = 0;
    if (begin < end) {
        const uint64_t from = begin / p.strip_tokens + s, to = (end - 1) / p.strip_tokens + s;
#pragma unroll 4
        for (uint64_t slot = from + part; slot <= to; slot += kBalanceWeightWarps) {
            if (e < p.experts) {
                sum += p.slot_sums[slot * p.experts + e];
                count += p.slot_counts[slot * p.experts + e];
            }
            tokens += p.slot_tokens[slot];
        }
    }
    s_sum[part][lane] = sum;
    s_count[part][lane] = count;
    if (lane == 0) s_tokens[part] = tokens;
    __syncthreads();
    if (part != 0) return;
    sum = 0.0f, count = 0, tokens = 0;
#pragma unroll
    for (uint32_t i = 0; i < kBalanceWeightWarps; ++i) sum += s_sum[i][lane], count += s_count[i][lane], tokens += s_tokens[i];
    float weight = 0.0f;
    if (e < p.experts) {
        weight = detail::balance_weight(p, count, tokens);
        p.weights[static_cast<uint64_t>(s) * p.experts + e] = weight;
        p.counts[static_cast<uint64_t>(s) * p.experts + e] = count;
    }
    float loss = weight * sum;
#pragma unroll
    for (uint32_t off = 16; off >= 1; off /= 2) loss += __shfl_xor_sync(0xffffffffu, loss, off);
    if (lane == 0) p.losses[s * gridDim.x + blockIdx.x] = loss;
}

// Strips run side by side, each from its last token to its first: what the first launch read last is what L2 still holds.
template <typename T, uint32_t kVec, uint32_t kLanes, uint32_t kIter>
__global__ void __launch_bounds__(kBalanceThreads, kVec * kIter <= 16 ? 3 : 1) balance_grad_kernel(const BalanceParams p, uint32_t num_losses) {
    using Row = detail::BalanceRow<T, kVec, kLanes, kIter>;
    constexpr uint32_t kPerLane = Row::kPerLane;
    __shared__ int s_cu[detail::kMaxSharedSequences + 1];
    ptx::grid_dependency_wait();
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    if (blockIdx.x == 0 && warp == 0) {
        float loss = 0.0f;
        for (uint32_t i = lane; i < num_losses; i += 32) loss += p.losses[i];
#pragma unroll
        for (uint32_t off = 16; off >= 1; off /= 2) loss += __shfl_xor_sync(0xffffffffu, loss, off);
        if (lane == 0) *p.loss = loss;
    }
    if (p.grad == nullptr) return;
    const uint32_t strip = blockIdx.x, first = strip * p.strip_tokens, last = min(first + p.strip_tokens, p.tokens);
    const int* cu = detail::stage_sequences(p, s_cu);
    float weights[kPerLane];
    uint32_t at = first;  // tokens below have their gradient
    for (uint32_t s = detail::first_sequence_behind(p, cu, first); at < last; ++s) {
        // the tokens up to the sequence belong to none: their gradient is zero
        uint32_t begin = last, end = last;
        if (s < p.sequences) detail::sequence_range(p, cu, s, begin, end);
        begin = min(max(begin, at), last), end = min(max(end, begin), last);
        if (begin < end) {
#pragma unroll
            for (uint32_t c = 0; c < kPerLane; ++c) {
                const uint32_t col = Row::column(lane, c);
                weights[c] = col < p.experts ? p.weights[static_cast<uint64_t>(s) * p.experts + col] : 0.0f;
            }
        }
        Row::grad(p, at, begin, end, warp, kBalanceWarps, lane, p.rows, 0, weights);
        at = end;
    }
}

// ---- few tokens: one cluster ----
// A cluster has 128 warps: it wins while each has few tokens and few experts per lane.  us for one cluster / for three launches, one behind
// the other in a graph, fp32: 64 x 64 4.9 / 6.5, 512 x 64 5.3 / 6.6, 128 x 512 7.6 / 11.8, 256 x 256 6.8 / 9.0, 1024 x 64 in 4 sequences
// 8.1 / 8.0, 512 x 256 8.8 / 8.9, 1024 x 256 14.6 / 9.2, 2048 x 64 10.5 / 7.2, 4096 x 32 10.6 / 7.0, 8192 x 8 15.9 / 8.1.
constexpr uint32_t kBalanceClusterMaxTokens = 1024, kBalanceClusterMaxLogits = 1u << 16;
constexpr uint32_t kBalanceClusterCtas = 8, kBalanceClusterThreads = 512, kBalanceClusterWarps = kBalanceClusterThreads / 32;

// Shared memory of a CTA, in words: per (sequence, expert) the sum, the selections and a; the slots of (warp, sequence) sums; per sequence its
// tokens; per row of the CTA what its gradient needs.
struct BalanceClusterLayout {
    uint32_t pairs, counts, weights, slots, tokens, rows, words;
    __host__ __device__ BalanceClusterLayout(uint32_t tokens_of_cta, uint32_t experts, uint32_t sequences) {
        pairs = experts * sequences;
        counts = pairs, weights = 2 * pairs, slots = 3 * pairs;
        tokens = slots + (kBalanceClusterWarps + sequences) * experts;
        rows = align_up(tokens + sequences, 2u);
        words = rows + 2 * tokens_of_cta;
    }
};

namespace detail {

__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ int ld_cluster_s32(uint32_t addr) {
    int v;
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
// The same word of every CTA of the cluster, added up in their order.
__device__ __forceinline__ float sum_of_cluster(const float* word) {
    float v[kBalanceClusterCtas], sum = 0.0f;
#pragma unroll
    for (uint32_t i = 0; i < kBalanceClusterCtas; ++i) v[i] = ld_cluster_f32(ptx::map_to_cta(ptx::smem_u32(word), i));
#pragma unroll
    for (uint32_t i = 0; i < kBalanceClusterCtas; ++i) sum += v[i];
    return sum;
}
__device__ __forceinline__ int sum_of_cluster(const int* word) {
    int sum = 0;
#pragma unroll
    for (uint32_t i = 0; i < kBalanceClusterCtas; ++i) sum += ld_cluster_s32(ptx::map_to_cta(ptx::smem_u32(word), i));
    return sum;
}

}  // namespace detail

template <typename T, uint32_t kVec, uint32_t kLanes, uint32_t kIter>
__global__ void __launch_bounds__(kBalanceClusterThreads) __cluster_dims__(kBalanceClusterCtas, 1, 1)
    balance_cluster_kernel(const BalanceParams p, uint32_t tokens_of_cta) {
    using Row = detail::BalanceRow<T, kVec, kLanes, kIter>;
    constexpr uint32_t kPerLane = Row::kPerLane;
    extern __shared__ float2 s_all[];
    __shared__ float s_losses[kBalanceClusterCtas], s_loss[kBalanceClusterWarps];
    __shared__ int s_cu[detail::kMaxSharedSequences + 1];
    const BalanceClusterLayout at(tokens_of_cta, p.experts, p.sequences);
    float* const s_sums = reinterpret_cast<float*>(s_all);
    int* const s_counts = reinterpret_cast<int*>(s_sums) + at.counts;
    float* const s_weights = s_sums + at.weights;
    float* const s_slots = s_sums + at.slots;
    int* const s_tokens = reinterpret_cast<int*>(s_sums) + at.tokens;
    float2* const s_rows = reinterpret_cast<float2*>(s_sums + at.rows);
    const uint32_t thread = threadIdx.x, warp = thread / 32, lane = thread % 32, rank = ptx::cluster_ctarank();
    const uint32_t first = min(rank * tokens_of_cta, p.tokens), last = min(first + tokens_of_cta, p.tokens);

    for (uint32_t i = thread; i < 2 * at.pairs; i += kBalanceClusterThreads) s_sums[i] = 0.0f;  // and the selections
    for (uint32_t i = thread; i < p.sequences; i += kBalanceClusterThreads) s_tokens[i] = 0;
    __syncthreads();
    ptx::grid_dependency_wait();

    const int* cu = detail::stage_sequences(p, s_cu);
    const uint32_t first_sequence = detail::first_sequence_behind(p, cu, first);

    // selections of the CTA's tokens
    for (uint32_t i = first * p.top + thread; i < last * p.top; i += kBalanceClusterThreads) {
        const uint32_t token = i / p.top;
        if (p.mask != nullptr && p.mask[token] == 0) continue;
        const long long id = p.ids_64 != 0 ? static_cast<const long long*>(p.ids)[i] : static_cast<const int*>(p.ids)[i];
        if (id < 0 || id >= static_cast<long long>(p.experts)) continue;
        const uint32_t s = detail::first_sequence_behind(p, cu, token);
        uint32_t begin = 0, end = 0;
        if (s < p.sequences) detail::sequence_range(p, cu, s, begin, end);
        if (token >= begin && token < end) atomicAdd(&s_counts[s * p.experts + static_cast<uint32_t>(id)], 1);
    }
    // Their probabilities: a strip of tokens for each warp.  A strip may touch several sequences; the sums of (warp, sequence) go to slot
    // warp + sequence, which no other pair has.
    const uint32_t strip = ceil_div(tokens_of_cta, kBalanceClusterWarps);
    const uint32_t from = min(first + warp * strip, last), to = min(from + strip, last);
    // not in front of the CTA's first, even where the ends of the sequences are out of order: the slots begin there
    const uint32_t from_sequence = from < to ? max(detail::first_sequence_behind(p, cu, from), first_sequence) : p.sequences;
    for (uint32_t s = from_sequence; s < p.sequences; ++s) {
        uint32_t begin, end;
        detail::sequence_range(p, cu, s, begin, end);
        if (begin >= to) break;
        begin = max(begin, from), end = min(end, to);
        if (begin >= end) continue;
        float sums[kPerLane];
#pragma unroll
        for (uint32_t c = 0; c < kPerLane; ++c) sums[c] = 0.0f;
        int counted = 0;
        Row::add(p, begin, end, 0, 1, lane, p.grad != nullptr ? s_rows : nullptr, first, sums, counted);
        if (counted != 0) atomicAdd(&s_tokens[s], counted);
        float* const into = s_slots + (warp + s - first_sequence) * p.experts;
#pragma unroll
        for (uint32_t c = 0; c < kPerLane; ++c) {
#pragma unroll
            for (uint32_t off = kLanes; off < 32; off *= 2) sums[c] += __shfl_xor_sync(0xffffffffu, sums[c], off);
            const uint32_t col = Row::column(lane, c);
            if (lane < kLanes && col < p.experts) into[col] = sums[c];
        }
    }
    __syncthreads();
    for (uint32_t i = first_sequence * p.experts + thread; i < at.pairs; i += kBalanceClusterThreads) {
        const uint32_t s = i / p.experts;
        uint32_t begin, end;
        detail::sequence_range(p, cu, s, begin, end);
        if (begin >= last) break;
        begin = max(begin, first), end = min(end, last);
        if (begin >= end) continue;
        const uint32_t until = (end - 1 - first) / strip;
        float sum = 0.0f;
        for (uint32_t w = (begin - first) / strip; w <= until; ++w) sum += s_slots[(w + s - first_sequence) * p.experts + i % p.experts];
        s_sums[i] = sum;
    }
    ptx::cluster_arrive(), ptx::cluster_wait();

    // The CTA's share of the pairs: counts, the loss, and a, which every CTA of the cluster gets.
    float loss = 0.0f;
    const uint32_t share = ceil_div(at.pairs, kBalanceClusterCtas), until = min((rank + 1) * share, at.pairs);
    for (uint32_t i = rank * share + thread; i < until; i += kBalanceClusterThreads) {
        const int count = detail::sum_of_cluster(s_counts + i);
        const float weight = detail::balance_weight(p, count, detail::sum_of_cluster(s_tokens + i / p.experts));
        p.counts[i] = count;
        loss = fmaf(weight, detail::sum_of_cluster(s_sums + i), loss);
#pragma unroll
        for (uint32_t cta = 0; cta < kBalanceClusterCtas; ++cta) ptx::st_cluster_f32(ptx::map_to_cta(ptx::smem_u32(s_weights + i), cta), weight);
    }
#pragma unroll
    for (uint32_t off = 16; off >= 1; off /= 2) loss += __shfl_xor_sync(0xffffffffu, loss, off);
    if (lane == 0) s_loss[warp] = loss;
    __syncthreads();
    if (thread == 0) {
        loss = 0.0f;
#pragma unroll
        for (uint32_t w = 0; w < kBalanceClusterWarps; ++w) loss += s_loss[w];
        ptx::st_cluster_f32(ptx::map_to_cta(ptx::smem_u32(s_losses + rank), 0), loss);
    }
    ptx::cluster_arrive(), ptx::cluster_wait();  // behind it nobody looks at another CTA's memory
    if (rank == 0 && thread == 0) {
        loss = 0.0f;
#pragma unroll
        for (uint32_t i = 0; i < kBalanceClusterCtas; ++i) loss += s_losses[i];
        *p.loss = loss;
    }

    if (p.grad == nullptr) return;
    float weights[kPerLane];
    uint32_t done = from;  // tokens below have their gradient
    for (uint32_t s = from_sequence; done < to; ++s) {
        uint32_t begin = to, end = to;
        if (s < p.sequences) detail::sequence_range(p, cu, s, begin, end);
        begin = min(max(begin, done), to), end = min(max(end, begin), to);
        if (begin < end) {
#pragma unroll
            for (uint32_t c = 0; c < kPerLane; ++c) {
                const uint32_t col = Row::column(lane, c);
                weights[c] = col < p.experts ? s_weights[s * p.experts + col] : 0.0f;
            }
        }
        Row::grad(p, done, begin, end, 0, 1, lane, s_rows, first, weights);
        done = end;
    }
}

// ---------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------
struct BalanceWorkspace {
    bool cluster;                  // one cluster does it, without scratch
    uint32_t strips, strip_tokens;  // tokens of a CTA in either case
    size_t sums, counts, tokens, weights, losses, rows, bytes;
};

inline BalanceWorkspace plan_balance_workspace(uint32_t tokens, uint32_t experts, uint32_t sequences, bool with_grad, uint32_t num_sms) {
    BalanceWorkspace w = {};
    w.cluster = num_sms >= kBalanceClusterCtas && tokens <= kBalanceClusterMaxTokens &&
                static_cast<uint64_t>(tokens) * experts <= kBalanceClusterMaxLogits;
    if (w.cluster) {
        w.strip_tokens = ceil_div(tokens, kBalanceClusterCtas);
        w.cluster = static_cast<uint64_t>(experts) * sequences <= 16384 &&
                    BalanceClusterLayout(w.strip_tokens, experts, sequences).words * 4 <= 200 * 1024;
        if (w.cluster) return w;
    }
    // three CTAs per SM, as many as run at a time, but at least four tokens per warp
    w.strip_tokens = ceil_div(tokens, 3 * num_sms);
    if (w.strip_tokens < 4 * kBalanceWarps) w.strip_tokens = 4 * kBalanceWarps;
    w.strips = ceil_div(tokens, w.strip_tokens);
    if (w.strips == 0) w.strips = 1;
    const size_t slots = static_cast<size_t>(w.strips) + sequences;
    size_t at = 0;
    auto take = [&at](size_t bytes) {
        const size_t here = at;
        at = align_up(at + bytes, static_cast<size_t>(256));
        return here;
    };
    w.sums = take(slots * experts * 4);
    w.counts = take(slots * experts * 4);
    w.tokens = take(slots * 4);
    w.weights = take(static_cast<size_t>(sequences) * experts * 4);
    w.losses = take(static_cast<size_t>(sequences) * ceil_div(experts, 32u) * 4);
    w.rows = take(with_grad ? static_cast<size_t>(tokens) * 8 : 0);
    w.bytes = at;
    return w;
}

template <typename T, uint32_t kVec, uint32_t kLanes, uint32_t kIter>
inline int launch_balance_as(const BalanceParams& p, bool cluster, cudaStream_t stream) {
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    if (cluster) {
        cfg.gridDim = dim3(kBalanceClusterCtas);
        cfg.blockDim = dim3(kBalanceClusterThreads);
        cfg.dynamicSmemBytes = BalanceClusterLayout(p.strip_tokens, p.experts, p.sequences).words * 4;
        cfg.stream = stream;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        auto kernel = balance_cluster_kernel<T, kVec, kLanes, kIter>;
        cudaError_t e = cudaSuccess;
        if (cfg.dynamicSmemBytes > 40 * 1024)
            e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(cfg.dynamicSmemBytes));
        if (e == cudaSuccess) e = cudaLaunchKernelEx(&cfg, kernel, p, p.strip_tokens);
        if (e == cudaSuccess) return kOk;
        cudaGetLastError();
        return kLaunchFailed;
    }
    cfg.gridDim = dim3(p.strips);
    cfg.blockDim = dim3(kBalanceThreads);
    cfg.dynamicSmemBytes = kBalanceWarps * p.experts * sizeof(float);
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaError_t e = cudaLaunchKernelEx(&cfg, balance_sums_kernel<T, kVec, kLanes, kIter>, p);
    cfg.dynamicSmemBytes = 0;
    const uint32_t parts = ceil_div(p.experts, 32u);
    cfg.gridDim = dim3(parts, p.sequences);
    cfg.blockDim = dim3(kBalanceWeightWarps * 32);
    if (e == cudaSuccess) e = cudaLaunchKernelEx(&cfg, balance_weights_kernel, p);
    cfg.gridDim = dim3(p.grad != nullptr ? p.strips : 1u);
    cfg.blockDim = dim3(kBalanceThreads);
    if (e == cudaSuccess) e = cudaLaunchKernelEx(&cfg, balance_grad_kernel<T, kVec, kLanes, kIter>, p, parts * p.sequences);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return kLaunchFailed;
    }
    return kOk;
}

template <typename T>
inline int launch_balance(const BalanceParams& p, bool cluster, cudaStream_t stream) {
    constexpr uint32_t kVec = 16 / sizeof(T);
    const bool vector = reinterpret_cast<uintptr_t>(p.logits) % 16 == 0 && reinterpret_cast<uintptr_t>(p.grad) % 16 == 0 &&
                        p.logits_ld % kVec == 0 && p.grad_ld % kVec == 0 && p.experts % kVec == 0;
    if (vector) {
        const uint32_t lanes = p.experts / kVec;
        if (lanes <= 8) return launch_balance_as<T, kVec, 8, 1>(p, cluster, stream);
        if (lanes <= 16) return launch_balance_as<T, kVec, 16, 1>(p, cluster, stream);
        if (lanes <= 32) return launch_balance_as<T, kVec, 32, 1>(p, cluster, stream);
        if (lanes <= 64) return launch_balance_as<T, kVec, 32, 2>(p, cluster, stream);
        if (lanes <= 128) return launch_balance_as<T, kVec, 32, 4>(p, cluster, stream);
        return launch_balance_as<T, kVec, 32, 1024 / kVec / 32>(p, cluster, stream);
    }
    // one expert per lane at a time: rows of few experts share a warp
    if (p.experts <= 8) return launch_balance_as<T, 1, 8, 1>(p, cluster, stream);
    if (p.experts <= 16) return launch_balance_as<T, 1, 8, 2>(p, cluster, stream);
    if (p.experts <= 32) return launch_balance_as<T, 1, 8, 4>(p, cluster, stream);
    if (p.experts <= 64) return launch_balance_as<T, 1, 16, 4>(p, cluster, stream);
    if (p.experts <= 128) return launch_balance_as<T, 1, 32, 4>(p, cluster, stream);
    if (p.experts <= 256) return launch_balance_as<T, 1, 32, 8>(p, cluster, stream);
    if (p.experts <= 384) return launch_balance_as<T, 1, 32, 12>(p, cluster, stream);
    if (p.experts <= 512) return launch_balance_as<T, 1, 32, 16>(p, cluster, stream);
    return launch_balance_as<T, 1, 32, 32>(p, cluster, stream);
}

}  // namespace yan
