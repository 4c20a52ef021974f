"""AdamW over many tensors in one launch, with states in 32 or 8 bits (CUDA only; kernel in include/train/adamw.cuh).  No counterpart in
the reference."""
from __future__ import annotations

from typing import Optional, Sequence, Tuple, Union

import torch

from .. import _lib

State = Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]
STATE_BLOCK = 128  # elements that share a scale of an 8-bit state
_DTYPES = {torch.float32: 0, torch.bfloat16: 1}


def adamw_state(param: torch.Tensor, state_bits: int = 32) -> State:
    """A new first or second moment for `param`: zeros in fp32, or (e4m3 codes, one fp32 scale per 128 elements), both flat."""
    assert state_bits in (8, 32)
    if state_bits == 32:
        return torch.zeros(param.shape, dtype=torch.float32, device=param.device)
    blocks = (param.numel() + STATE_BLOCK - 1) // STATE_BLOCK
    return (torch.zeros(param.numel(), dtype=torch.uint8, device=param.device).view(torch.float8_e4m3fn),
            torch.zeros(blocks, dtype=torch.float32, device=param.device))


def _check_state(state: State, param: torch.Tensor, eight_bit: bool) -> Tuple[int, int]:
    """Addresses of the values (codes) and of the scales."""
    if not eight_bit:
        assert state.dtype == torch.float32 and state.numel() == param.numel() and state.is_contiguous() and state.device == param.device
        return state.data_ptr(), 0
    codes, scales = state
    assert codes.dtype == torch.float8_e4m3fn and codes.numel() == param.numel() and codes.is_contiguous() and codes.device == param.device
    assert scales.dtype == torch.float32 and scales.numel() == (param.numel() + STATE_BLOCK - 1) // STATE_BLOCK
    assert scales.is_contiguous() and scales.device == param.device
    return codes.data_ptr(), scales.data_ptr()


def adamw_step(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], exp_avgs: Sequence[State], exp_avg_sqs: Sequence[State], *,
               lr: float, beta1: float = 0.9, beta2: float = 0.999, eps: float = 1e-8,
               weight_decay: Union[float, Sequence[float]] = 0.0, step: int, grad_scale: Optional[torch.Tensor] = None,
               copies: Optional[Sequence[torch.Tensor]] = None) -> None:
    """One AdamW step, in place, over all tensors of the lists:

        g = grad * grad_scale;  m = beta1 m + (1 - beta1) g;  v = beta2 v + (1 - beta2) g^2
        p = p (1 - lr weight_decay) - lr / (1 - beta1^step) * m / (sqrt(v / (1 - beta2^step)) + eps)

    params and grads: contiguous tensors in fp32 or bf16, each list of one type, a grad as large as its param.  exp_avgs and exp_avg_sqs: m and
    v as `adamw_state` makes them, all in 32 or all in 8 bits; 8-bit states hold m and sqrt(v) as e4m3 codes times a power of two per
    128 elements, a quarter of the state's traffic.  weight_decay: one number, or one per tensor.  step counts from 1.
    grad_scale: fp32 tensor of one element on the device (a clipping factor, say), read when the kernel runs.
    copies: bf16 tensors that receive the new parameters, e.g. what per_block_cast_to_fp8 quantizes for the next forward pass.
    lr, step and the other numbers become part of a captured CUDA graph."""
    rc = _lib.fast().adamw(params, grads, exp_avgs, exp_avg_sqs, weight_decay, copies, grad_scale, lr, beta1, beta2, eps, step)
    if rc != -1:  # -1: not an ordinary call, left to the checks below
        return _lib.check("yan_b200_adamw_step", rc)
    count = len(params)
    assert len(grads) == count and len(exp_avgs) == count and len(exp_avg_sqs) == count and (copies is None or len(copies) == count)
    decays = [float(weight_decay)] * count if isinstance(weight_decay, (int, float)) else [float(w) for w in weight_decay]
    assert len(decays) == count and step >= 1 and 0.0 <= beta1 < 1.0 and 0.0 <= beta2 < 1.0 and eps >= 0.0 and lr >= 0.0
    if count == 0:
        return
    device, param_dtype, grad_dtype = params[0].device, params[0].dtype, grads[0].dtype
    assert params[0].is_cuda and device.index == torch.cuda.current_device()
    assert param_dtype in _DTYPES and grad_dtype in _DTYPES, "params and grads are fp32 or bf16 on the GPU"
    eight_bit = not isinstance(exp_avgs[0], torch.Tensor)
    if grad_scale is not None:
        assert grad_scale.device == device and grad_scale.dtype == torch.float32 and grad_scale.numel() == 1
    table = (_lib.AdamwTensor * count)()
    for i in range(count):
        p, g, row = params[i], grads[i], table[i]
        assert p.dtype == param_dtype and p.device == device and p.is_contiguous()
        assert g.dtype == grad_dtype and g.device == device and g.is_contiguous() and g.numel() == p.numel()
        row.param, row.grad, row.numel, row.weight_decay = p.data_ptr(), g.data_ptr(), p.numel(), decays[i]
        row.exp_avg, row.exp_avg_scale = _check_state(exp_avgs[i], p, eight_bit)
        row.exp_avg_sq, row.exp_avg_sq_scale = _check_state(exp_avg_sqs[i], p, eight_bit)
        if copies is not None:
            c = copies[i]
            assert c.dtype == torch.bfloat16 and c.device == device and c.is_contiguous() and c.numel() == p.numel()
            row.copy = c.data_ptr()
    torch.autograd.graph.increment_version([p for p in params if not p.is_inference()])  # autograd notices that they change
    _lib.call("yan_b200_adamw_step", table, count, _DTYPES[param_dtype], _DTYPES[grad_dtype], 8 if eight_bit else 32, lr, beta1, beta2, eps,
              step, grad_scale.data_ptr() if grad_scale is not None else None, _lib.current_stream_ptr())
