// C ABI of the operators that train a layer: weight gradient, AdamW step, balance loss (declarations: include/yan_b200.h).

#include <cmath>
#include <cstdint>
#include <cuda_runtime.h>

#include "../../include/yan_b200.h"
#include "launch_state.h"
#include "train/adamw.cuh"
#include "train/fp8_wgrad.cuh"
#include "train/moe_balance.cuh"

namespace {

inline void set_rc(int* rc, int v) {
    if (rc != nullptr) *rc = v;
}

size_t wgrad_workspace_bytes(int m, int n, int k, int num_groups, int num_sms) {
    if (m < 0 || n <= 0 || k <= 0 || num_groups < 0 || num_sms <= 0) return 0;
    const bool grouped = num_groups != 0;
    yan::WgradWorkspace w;
    return yan::plan_wgrad_workspace(m, n, k, grouped ? num_groups : 1, grouped, num_sms, w) ? w.bytes : 0;
}

int wgrad(yan::WgradArgs& a, int m, int n, int k, long long dy_ld, long long x_ld, long long out_ld, long long out_group_stride,
          int out_dtype, int accumulate, void* workspace, size_t workspace_bytes, int num_sms, void* stream) {
    if (m < 0 || n <= 0 || k <= 0 || dy_ld < 0 || x_ld < 0 || out_ld <= 0 || out_group_stride < 0 || num_sms <= 0) return yan::kBadArgument;
    if (out_dtype != YAN_B200_F32 && out_dtype != YAN_B200_BF16) return yan::kBadArgument;
    a.groups.rows = m;
    a.n = n, a.k = k;
    a.dy_ld = dy_ld, a.x_ld = x_ld;
    a.out_ld = out_ld, a.out_group = out_group_stride;
    a.out_bf16 = out_dtype == YAN_B200_BF16;
    a.accumulate = accumulate != 0;
    a.workspace = workspace;
    a.workspace_bytes = workspace_bytes;
    a.num_sms = num_sms;
    a.status = yan::status_word_of_current_device();
    a.timeout_ns = yan::wait_timeout_ns();
    return yan::launch_fp8_wgrad(a, static_cast<cudaStream_t>(stream));
}

// Four elements at a time are 16 bytes in 32 bits, 8 in bf16 and 4 as codes.
bool adamw_vector(const yan_b200_adamw_tensor& t, bool param_bf16, bool grad_bf16, bool eight_bit) {
    return yan::is_aligned(t.param, param_bf16 ? 8 : 16) && yan::is_aligned(t.grad, grad_bf16 ? 8 : 16) &&
           yan::is_aligned(t.exp_avg, eight_bit ? 4 : 16) && yan::is_aligned(t.exp_avg_sq, eight_bit ? 4 : 16) &&
           yan::is_aligned(t.copy, 8);
}

bool adamw_tensor_ok(const yan_b200_adamw_tensor& t, bool param_bf16, bool grad_bf16, bool eight_bit) {
    if (t.numel < 0 || t.numel / yan::adamw_chunk(eight_bit) >= 0x7fffffff) return false;  // a grid reaches over a tensor
    if (t.numel == 0) return true;
    if (t.param == nullptr || t.grad == nullptr || t.exp_avg == nullptr || t.exp_avg_sq == nullptr) return false;
    if (eight_bit && (t.exp_avg_scale == nullptr || t.exp_avg_sq_scale == nullptr)) return false;
    return yan::is_aligned(t.param, param_bf16 ? 2 : 4) && yan::is_aligned(t.grad, grad_bf16 ? 2 : 4) && yan::is_aligned(t.copy, 2) &&
           (eight_bit ? yan::is_aligned(t.exp_avg_scale, 4) && yan::is_aligned(t.exp_avg_sq_scale, 4)
                      : yan::is_aligned(t.exp_avg, 4) && yan::is_aligned(t.exp_avg_sq, 4));
}

// Launches tensors [first, ...) as far as one table holds them and a grid reaches; returns the first tensor that is left.
template <uint32_t kCapacity>
int adamw_some(const yan_b200_adamw_tensor* tensors, int first, int count, const yan::AdamwScalars& scalars, double lr, bool param_bf16,
               bool grad_bf16, bool eight_bit, cudaStream_t stream, int* next) {
    yan::AdamwParams<kCapacity> p;
    p.s = scalars;
    const uint32_t chunk = yan::adamw_chunk(eight_bit);
    uint32_t used = 0;
    uint64_t chunks = 0;
    int i = first;
    for (; i < count && used < kCapacity; ++i) {
        const yan_b200_adamw_tensor& t = tensors[i];
        if (t.numel == 0) continue;
        const uint64_t more = (static_cast<uint64_t>(t.numel) + chunk - 1) / chunk;
        if (chunks + more > 0x7fffffffull) break;
        p.first_chunk[used] = static_cast<uint32_t>(chunks);
        yan::AdamwTensor& d = p.tensor[used];
        d.param = t.param, d.grad = t.grad, d.m = t.exp_avg, d.v = t.exp_avg_sq;
        d.m_scale = t.exp_avg_scale, d.v_scale = t.exp_avg_sq_scale;
        d.copy = static_cast<__nv_bfloat16*>(t.copy);
        d.numel_lo = static_cast<uint32_t>(t.numel);
        d.numel_hi = static_cast<uint32_t>(static_cast<uint64_t>(t.numel) >> 32);
        d.decay = static_cast<float>(1.0 - lr * static_cast<double>(t.weight_decay));
        d.vector = adamw_vector(t, param_bf16, grad_bf16, eight_bit);
        chunks += more;
        ++used;
    }
    *next = i;
    p.first_chunk[used] = static_cast<uint32_t>(chunks);
    p.num_tensors = used;
    return used == 0 ? yan::kOk : yan::launch_adamw(p, param_bf16, grad_bf16, eight_bit, stream);
}

}  // namespace

extern "C" {

#define YAN_EXPORT __attribute__((visibility("default")))

YAN_EXPORT size_t yan_b200_fp8_linear_wgrad_workspace_bytes(int m, int n, int k, int num_groups, int num_sms) {
    return wgrad_workspace_bytes(m, n, k, num_groups, num_sms);
}

YAN_EXPORT void yan_b200_fp8_linear_wgrad(const void* dy, const void* x, void* out, int m, int n, int k, long long dy_ld, long long x_ld,
                                          long long out_ld, int out_dtype, int accumulate, void* workspace, size_t workspace_bytes,
                                          void* stream, int num_sms, int* return_code) {
    yan::WgradArgs a;
    a.dy = dy, a.x = x, a.out = out;
    set_rc(return_code, wgrad(a, m, n, k, dy_ld, x_ld, out_ld, 0, out_dtype, accumulate, workspace, workspace_bytes, num_sms, stream));
}

YAN_EXPORT void yan_b200_k_grouped_fp8_linear_wgrad(const void* dy, const void* x, void* out, const int* group_starts,
                                                    const int* group_sizes, int num_groups, int m, int n, int k, long long dy_ld,
                                                    long long x_ld, long long out_ld, long long out_group_stride, int out_dtype,
                                                    int accumulate, void* workspace, size_t workspace_bytes, void* stream, int num_sms,
                                                    int* return_code) {
    if (group_starts == nullptr || group_sizes == nullptr || num_groups <= 0) return set_rc(return_code, yan::kBadArgument);
    yan::WgradArgs a;
    a.dy = dy, a.x = x, a.out = out;
    a.groups.starts = group_starts;
    a.groups.sizes = group_sizes;
    a.groups.num_groups = num_groups;
    set_rc(return_code, wgrad(a, m, n, k, dy_ld, x_ld, out_ld, out_group_stride, out_dtype, accumulate, workspace, workspace_bytes,
                              num_sms, stream));
}

YAN_EXPORT void yan_b200_adamw_step(const yan_b200_adamw_tensor* tensors, int num_tensors, int param_dtype, int grad_dtype, int state_bits,
                                    double lr, double beta1, double beta2, double eps, long long step, const float* grad_scale,
                                    void* stream, int* return_code) {
    if (num_tensors < 0 || (num_tensors > 0 && tensors == nullptr) || step < 1) return set_rc(return_code, yan::kBadArgument);
    if ((param_dtype != YAN_B200_F32 && param_dtype != YAN_B200_BF16) || (grad_dtype != YAN_B200_F32 && grad_dtype != YAN_B200_BF16) ||
        (state_bits != 32 && state_bits != 8))
        return set_rc(return_code, yan::kBadArgument);
    if (!(lr >= 0.0) || !(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0) || !(eps >= 0.0) || std::isinf(lr) || std::isinf(eps))
        return set_rc(return_code, yan::kBadArgument);
    const bool param_bf16 = param_dtype == YAN_B200_BF16, grad_bf16 = grad_dtype == YAN_B200_BF16, eight_bit = state_bits == 8;
    int filled = 0;
    for (int i = 0; i < num_tensors; ++i) {  // all of them before the first launch
        if (!adamw_tensor_ok(tensors[i], param_bf16, grad_bf16, eight_bit)) return set_rc(return_code, yan::kBadArgument);
        filled += tensors[i].numel != 0;
    }
    yan::AdamwScalars s;
    s.grad_scale = grad_scale;
    s.b1 = static_cast<float>(beta1), s.one_minus_b1 = static_cast<float>(1.0 - beta1);
    s.b2 = static_cast<float>(beta2), s.one_minus_b2 = static_cast<float>(1.0 - beta2);
    s.step_size = static_cast<float>(lr / (1.0 - std::pow(beta1, static_cast<double>(step))));
    s.inv_root_correction = static_cast<float>(1.0 / std::sqrt(1.0 - std::pow(beta2, static_cast<double>(step))));
    s.eps = static_cast<float>(eps);
    int rc = yan::kOk;
    for (int first = 0; first < num_tensors && rc == yan::kOk;)
        rc = filled <= static_cast<int>(yan::kAdamwSmallCapacity)
                 ? adamw_some<yan::kAdamwSmallCapacity>(tensors, first, num_tensors, s, lr, param_bf16, grad_bf16, eight_bit,
                                                        static_cast<cudaStream_t>(stream), &first)
                 : adamw_some<yan::kAdamwCapacity>(tensors, first, num_tensors, s, lr, param_bf16, grad_bf16, eight_bit,
                                                   static_cast<cudaStream_t>(stream), &first);
    set_rc(return_code, rc);
}

YAN_EXPORT size_t yan_b200_moe_balance_loss_workspace_bytes(int tokens, int experts, int sequences, int with_grad, int num_sms) {
    if (tokens < 0 || experts <= 0 || sequences <= 0 || num_sms <= 0) return 0;
    return yan::plan_balance_workspace(tokens, experts, sequences, with_grad != 0, num_sms).bytes;
}

YAN_EXPORT void yan_b200_moe_balance_loss(const void* logits, const void* expert_ids, const void* token_mask, const int* cu_seqlens,
                                          float* loss, int* counts, void* grad, int tokens, int experts, int top, int sequences,
                                          long long logits_ld, long long grad_ld, int logits_dtype, int ids_64, int score, float coef,
                                          void* workspace, size_t workspace_bytes, void* stream, int num_sms, int* return_code) {
    if (tokens < 0 || experts <= 0 || experts > static_cast<int>(yan::kMaxBalanceExperts) || top <= 0 ||
        top > static_cast<int>(yan::kMaxBalanceTop) || sequences <= 0 ||
        sequences > 65535 || num_sms <= 0 || loss == nullptr || counts == nullptr)
        return set_rc(return_code, yan::kBadArgument);
    if ((logits_dtype != YAN_B200_F32 && logits_dtype != YAN_B200_BF16) || (score != YAN_B200_SOFTMAX && score != YAN_B200_SIGMOID))
        return set_rc(return_code, yan::kBadArgument);
    if ((cu_seqlens == nullptr && sequences != 1) || logits_ld < experts || (grad != nullptr && grad_ld < experts))
        return set_rc(return_code, yan::kBadArgument);
    if (tokens > 0 && (logits == nullptr || expert_ids == nullptr)) return set_rc(return_code, yan::kBadArgument);
    const size_t item = logits_dtype == YAN_B200_F32 ? 4 : 2;
    if (!yan::is_aligned(logits, item) || !yan::is_aligned(grad, item) || !yan::is_aligned(expert_ids, ids_64 != 0 ? 8 : 4))
        return set_rc(return_code, yan::kBadArgument);
    const yan::BalanceWorkspace w = yan::plan_balance_workspace(tokens, experts, sequences, grad != nullptr, num_sms);
    if (w.bytes != 0 && (workspace == nullptr || !yan::is_aligned(workspace, 256))) return set_rc(return_code, yan::kBadArgument);
    if (workspace_bytes < w.bytes) return set_rc(return_code, yan::kWorkspaceTooSmall);
    char* ws = static_cast<char*>(workspace);
    yan::BalanceParams p;
    p.logits = logits, p.logits_ld = logits_ld;
    p.ids = expert_ids, p.ids_64 = ids_64 != 0;
    p.mask = static_cast<const uint8_t*>(token_mask);
    p.cu_seqlens = cu_seqlens;
    p.tokens = tokens, p.experts = experts, p.top = top, p.sequences = sequences;
    p.sigmoid = score == YAN_B200_SIGMOID;
    p.coef = coef;
    p.loss = loss, p.counts = counts;
    p.grad = grad, p.grad_ld = grad != nullptr ? grad_ld : 0;
    p.strips = w.strips, p.strip_tokens = w.strip_tokens;
    p.slot_sums = reinterpret_cast<float*>(ws + w.sums);
    p.slot_counts = reinterpret_cast<int*>(ws + w.counts);
    p.slot_tokens = reinterpret_cast<int*>(ws + w.tokens);
    p.weights = reinterpret_cast<float*>(ws + w.weights);
    p.losses = reinterpret_cast<float*>(ws + w.losses);
    p.rows = reinterpret_cast<float2*>(ws + w.rows);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    set_rc(return_code, logits_dtype == YAN_B200_F32 ? yan::launch_balance<float>(p, w.cluster, st)
                                                         : yan::launch_balance<__nv_bfloat16>(p, w.cluster, st));
}

}  // extern "C"
