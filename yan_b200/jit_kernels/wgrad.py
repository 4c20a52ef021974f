"""Weight gradients of FP8 linear layers (CUDA only; kernels in include/train/fp8_wgrad.cuh).

The forward pass multiplies 1x128 groups along K (fp8_linear); the weight gradient sums over the tokens, so its operands are quantized in
blocks of 128 tokens per feature, with powers of two that the tensor core applies.  No counterpart in the reference.
"""
from __future__ import annotations

from typing import Optional

import torch

from .. import _lib
from . import utils as _utils
from .utils import get_num_sms

MAX_GROUPS = 512
_OUT_DTYPES = {torch.float32: 0, torch.bfloat16: 1}


def _check_operands(dy: torch.Tensor, x: torch.Tensor) -> None:
    assert dy.is_cuda and x.is_cuda and dy.device == x.device and dy.device.index == torch.cuda.current_device()
    assert dy.dtype == torch.bfloat16 and x.dtype == torch.bfloat16 and dy.dim() == 2 and x.dim() == 2
    assert dy.shape[0] == x.shape[0], "dy and x have a row per token"
    assert dy.shape[1] > 0 and x.shape[1] > 0
    assert (dy.shape[1] == 1 or dy.stride(1) == 1) and (x.shape[1] == 1 or x.stride(1) == 1), "the features of a token are contiguous"


def _row_stride(t: torch.Tensor) -> int:
    """Elements from one row to the next (a matrix of one row may claim any)."""
    stride = t.stride(-2) if t.shape[-2] > 1 else max(t.stride(-2), t.shape[-1])
    assert stride >= t.shape[-1], "rows overlap"
    return stride


def _check_out(out: torch.Tensor, shape, device) -> None:
    assert out.is_cuda and out.device == device and out.dtype in _OUT_DTYPES, "out is fp32 or bf16"
    assert tuple(out.shape) == tuple(shape) and (out.shape[-1] == 1 or out.stride(-1) == 1)


def _take_workspace(workspace: Optional[torch.Tensor], need: int, device) -> torch.Tensor:
    if workspace is None:
        return torch.empty(need, dtype=torch.uint8, device=device)
    assert workspace.is_cuda and workspace.dtype == torch.uint8 and workspace.is_contiguous() and workspace.numel() >= need
    assert workspace.data_ptr() % 256 == 0
    return workspace


def fp8_linear_wgrad_workspace_bytes(m: int, n: int, k: int, num_groups: int = 0) -> int:
    """Scratch of fp8_linear_wgrad (num_groups = 0) or k_grouped_fp8_linear_wgrad for dy [m, n] and x [m, k]."""
    return int(_lib.lib().yan_b200_fp8_linear_wgrad_workspace_bytes(m, n, k, num_groups, get_num_sms()))


def fp8_linear_wgrad(dy: torch.Tensor, x: torch.Tensor, out: Optional[torch.Tensor] = None, *, accumulate: bool = False,
                     workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Gradient of the weight of y = x @ W^T:  out [N, K] (+)= dy^T @ x for dy [M, N] and x [M, K] in bf16, from e4m3 operands.

    Each operand gets one power of two per feature and block of 128 tokens; the sums are held in fp32 and rounded once to `out`
    (fp32 by default, or bf16).  With accumulate=True the product is added to what `out` holds (gradients of several microbatches).
    Any number of tokens (none included) and of features and any row strides; rows on 32-byte boundaries with multiples of 16
    features are the fast case.  The scratch comes from torch's allocator unless a `workspace` of
    fp8_linear_wgrad_workspace_bytes(M, N, K) bytes is given."""
    if out is not None and _utils._num_sms is not None:
        rc = _lib.fast().wgrad(dy, x, out, accumulate, workspace, _utils._num_sms, None, None)
        if rc != -1:  # -1: not an ordinary call, left to the checks below
            _lib.check("yan_b200_fp8_linear_wgrad", rc)
            return out
    _check_operands(dy, x)
    m, n, k = dy.shape[0], dy.shape[1], x.shape[1]
    if out is None:
        assert not accumulate, "accumulate needs an out"
        out = torch.empty((n, k), dtype=torch.float32, device=dy.device)
    _check_out(out, (n, k), dy.device)
    workspace = _take_workspace(workspace, fp8_linear_wgrad_workspace_bytes(m, n, k), dy.device)
    _lib.call("yan_b200_fp8_linear_wgrad", dy.data_ptr(), x.data_ptr(), out.data_ptr(), m, n, k, _row_stride(dy), _row_stride(x),
              _row_stride(out), _OUT_DTYPES[out.dtype], int(accumulate), workspace.data_ptr(), workspace.numel(),
              _lib.current_stream_ptr(), get_num_sms())
    return out


def k_grouped_fp8_linear_wgrad(dy: torch.Tensor, x: torch.Tensor, group_starts: torch.Tensor, group_sizes: torch.Tensor,
                               out: Optional[torch.Tensor] = None, *, accumulate: bool = False,
                               workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The weight gradients of a layer of experts:  out[g] (+)= dy[rows of g]^T @ x[rows of g], out [G, N, K].

    The rows of group g are [group_starts[g], group_starts[g] + group_sizes[g]) (int32 on the device, G <= 512): the contiguous layout
    of m_grouped_gemm_fp8_fp8_bf16_nt_contiguous, whose starts are multiples of 128, or rows packed without gaps.  Groups do not
    overlap; rows outside of every group are not read.  A group without rows gives zeros, or leaves its part of `out` as it is
    with accumulate=True.  Otherwise like fp8_linear_wgrad."""
    if out is not None and _utils._num_sms is not None:
        rc = _lib.fast().wgrad(dy, x, out, accumulate, workspace, _utils._num_sms, group_starts, group_sizes)
        if rc != -1:
            _lib.check("yan_b200_k_grouped_fp8_linear_wgrad", rc)
            return out
    _check_operands(dy, x)
    m, n, k, g = dy.shape[0], dy.shape[1], x.shape[1], group_sizes.numel()
    assert 0 < g <= MAX_GROUPS
    for t in (group_starts, group_sizes):
        assert t.is_cuda and t.device == dy.device and t.dtype == torch.int32 and t.shape == (g,) and t.is_contiguous()
    if out is None:
        assert not accumulate, "accumulate needs an out"
        out = torch.empty((g, n, k), dtype=torch.float32, device=dy.device)
    _check_out(out, (g, n, k), dy.device)
    group_stride = out.stride(0) if g > 1 else n * _row_stride(out)
    assert group_stride >= (n - 1) * _row_stride(out) + k, "groups overlap in out"
    workspace = _take_workspace(workspace, fp8_linear_wgrad_workspace_bytes(m, n, k, g), dy.device)
    _lib.call("yan_b200_k_grouped_fp8_linear_wgrad", dy.data_ptr(), x.data_ptr(), out.data_ptr(), group_starts.data_ptr(),
              group_sizes.data_ptr(), g, m, n, k, _row_stride(dy), _row_stride(x), _row_stride(out), group_stride,
              _OUT_DTYPES[out.dtype], int(accumulate), workspace.data_ptr(), workspace.numel(), _lib.current_stream_ptr(), get_num_sms())
    return out
