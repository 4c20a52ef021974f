"""Balance loss of a mixture-of-experts router with its gradient and the selections per expert (CUDA only; kernels in
include/train/moe_balance.cuh).  No counterpart in the reference."""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from .. import _lib
from . import utils as _utils
from .utils import get_num_sms

MAX_EXPERTS = 1024
MAX_TOP = 65535
_DTYPES = {torch.float32: 0, torch.bfloat16: 1}
_SCORES = {"softmax": 0, "sigmoid": 1}


def moe_balance_loss_workspace_bytes(tokens: int, experts: int, sequences: int = 1, with_grad: bool = True) -> int:
    return int(_lib.lib().yan_b200_moe_balance_loss_workspace_bytes(tokens, experts, sequences, int(with_grad), get_num_sms()))


def moe_balance_loss(logits: torch.Tensor, expert_ids: torch.Tensor, *, coef: float = 1.0, score: str = "softmax",
                     token_mask: Optional[torch.Tensor] = None, cu_seqlens: Optional[torch.Tensor] = None, with_grad: bool = True,
                     grad: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None
                     ) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
    """(loss, counts, grad) of a router:

        p[t] = softmax(logits[t]), or sigmoid(logits[t]) over its sum;  n_s = tokens of sequence s that count
        counts[s, e] = selections of expert e,  P[s, e] = sum over t of p[t, e]
        loss = coef / S * sum over s of E / (top n_s^2) * sum over e of counts[s, e] * P[s, e]

    which is coef for perfectly balanced experts.  grad = d loss / d logits in the logits' type (the counts are constants), to be added to
    what the rest of the model sends back; None with with_grad=False.  counts, int32 [S, E], are the group sizes of
    k_grouped_fp8_linear_wgrad and masked_m of m_grouped_gemm_fp8_fp8_bf16_nt_masked (for S = 1).

    logits [T, E] fp32 or bf16, E <= 1024, rows may be strided; expert_ids [T, top <= 65535] int64 or int32, contiguous, an id outside of
    [0, E) selects nothing (a dropped token).  token_mask [T] bool: tokens that count; the logits of the others are not read and their
    gradient is zero.  cu_seqlens int32 [S + 1], S <= 65535, ascending, on the device: sequence s is tokens [cu_seqlens[s], cu_seqlens[s + 1]); without it
    all tokens are one sequence.  A sequence without tokens adds nothing.  loss is an fp32 tensor without dimensions."""
    if with_grad and grad is None and workspace is None and _utils._num_sms is not None and score in _SCORES:
        result = _lib.fast().balance(logits, expert_ids, token_mask, cu_seqlens, coef, _SCORES[score], _utils._num_sms)
        if type(result) is tuple:
            return result
        if result != -1:  # -1: not an ordinary call, left to the checks below
            _lib.check("yan_b200_moe_balance_loss", result)
    assert logits.is_cuda and logits.device.index == torch.cuda.current_device()
    assert logits.dim() == 2 and logits.dtype in _DTYPES, "logits are [T, E] in fp32 or bf16"
    t, e = logits.shape
    assert 0 < e <= MAX_EXPERTS and (e == 1 or logits.stride(1) == 1)
    assert expert_ids.device == logits.device and expert_ids.dim() == 2 and expert_ids.shape[0] == t and 0 < expert_ids.shape[1] <= MAX_TOP
    assert expert_ids.dtype in (torch.int64, torch.int32) and expert_ids.is_contiguous()
    assert score in _SCORES, "score is 'softmax' or 'sigmoid'"
    if token_mask is not None:
        assert token_mask.device == logits.device and token_mask.dtype == torch.bool and token_mask.shape == (t,) and token_mask.is_contiguous()
    sequences = 1
    if cu_seqlens is not None:
        assert cu_seqlens.device == logits.device and cu_seqlens.dtype == torch.int32 and cu_seqlens.dim() == 1 and cu_seqlens.is_contiguous()
        sequences = cu_seqlens.numel() - 1
        assert 0 < sequences <= 65535
    if grad is not None:
        assert with_grad and grad.device == logits.device and grad.dtype == logits.dtype and grad.shape == (t, e)
        assert e == 1 or grad.stride(1) == 1
    elif with_grad:
        grad = torch.empty((t, e), dtype=logits.dtype, device=logits.device)

    def row_stride(x):
        stride = x.stride(0) if t > 1 else max(x.stride(0), e)
        assert stride >= e, "rows overlap"
        return stride

    loss = torch.empty((), dtype=torch.float32, device=logits.device)
    counts = torch.empty((sequences, e), dtype=torch.int32, device=logits.device)
    need = moe_balance_loss_workspace_bytes(t, e, sequences, grad is not None)
    if workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=logits.device)
    assert workspace.is_cuda and workspace.dtype == torch.uint8 and workspace.is_contiguous() and workspace.numel() >= need
    _lib.call("yan_b200_moe_balance_loss", logits.data_ptr(), expert_ids.data_ptr(), token_mask.data_ptr() if token_mask is not None else None,
              cu_seqlens.data_ptr() if cu_seqlens is not None else None, loss.data_ptr(), counts.data_ptr(),
              grad.data_ptr() if grad is not None else None, t, e, expert_ids.shape[1], sequences, row_stride(logits),
              row_stride(grad) if grad is not None else 0, _DTYPES[logits.dtype], int(expert_ids.dtype == torch.int64), _SCORES[score], coef,
              workspace.data_ptr(), workspace.numel(), _lib.current_stream_ptr(), get_num_sms())
    return loss, counts, grad
