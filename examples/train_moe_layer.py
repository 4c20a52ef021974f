"""Trains one mixture-of-experts layer with FP8 products, forward and backward, on one B200.

    python examples/train_moe_layer.py [--steps 60]

A step is: router logits, top-k and balance loss -> tokens gathered expert by expert -> grouped FP8 GEMM -> loss -> gradients of the weights
(k_grouped_fp8_linear_wgrad, with the router's counts as group sizes) and of the router -> AdamW (8-bit states for the experts, whose
bf16 copies are quantized for the next forward pass).  Nothing is copied to the host between two steps.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import yan_b200 as yan  # noqa: E402


class MoeLayer:
    """y[t] = sum over the chosen experts e of gate[t, e] * (x[t] @ W[e]^T), fp32 master weights, FP8 products."""

    def __init__(self, experts: int, inputs: int, outputs: int, top: int, seed: int = 0) -> None:
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.top, self.step = top, 0
        self.weight = torch.randn(experts, outputs, inputs, generator=gen, device="cuda") * inputs ** -0.5
        self.router = torch.randn(experts, inputs, generator=gen, device="cuda") * 0.02
        self.copy = self.weight.to(torch.bfloat16)
        self.weight_moments = [yan.adamw_state(self.weight, 8) for _ in range(2)]
        self.router_moments = [yan.adamw_state(self.router, 32) for _ in range(2)]
        self.weight_grad = torch.empty_like(self.weight)
        self.quantize()

    def quantize(self) -> None:
        e, n, k = self.weight.shape
        codes, scales = yan.per_block_cast_to_fp8(self.copy.view(e * n, k))
        self.rhs = codes.view(e, n, k), scales.view(e, n // 128, k // 128)

    def train_step(self, x: torch.Tensor, target: torch.Tensor, lr: float = 2e-3, balance: float = 1e-2):
        """(mean squared error, balance loss, selections per expert) of the step, as tensors on the device."""
        tokens, (experts, outputs, inputs) = x.shape[0], self.weight.shape
        # router
        logits = x.float() @ self.router.t()
        gates = torch.softmax(logits, dim=1)
        picked, ids = gates.topk(self.top, dim=1)
        balance_loss, counts, dlogits = yan.moe_balance_loss(logits, ids, coef=balance)
        sizes = counts[0]
        # rows of every expert together, each expert's from a multiple of 128 on
        align = yan.get_m_alignment_for_contiguous_layout()
        padded = (sizes + align - 1) // align * align
        starts = (padded.cumsum(0) - padded).to(torch.int32)
        flat = ids.reshape(-1)
        order = flat.argsort(stable=True)
        rank = torch.arange(tokens * self.top, device="cuda") - (sizes.cumsum(0) - sizes)[flat[order]]
        row = torch.empty_like(flat)
        row[order] = starts[flat[order]] + rank
        token = torch.arange(tokens, device="cuda").repeat_interleave(self.top)
        rows = (tokens * self.top + experts * (align - 1) + align - 1) // align * align
        m_indices = torch.full((rows,), -1, dtype=torch.int32, device="cuda")
        m_indices[row] = flat.to(torch.int32)
        gathered = torch.zeros(rows, inputs, dtype=torch.bfloat16, device="cuda")
        gathered[row] = x[token]
        # forward
        out = torch.zeros(rows, outputs, dtype=torch.bfloat16, device="cuda")
        yan.m_grouped_gemm_fp8_fp8_bf16_nt_contiguous(yan.per_token_cast_to_fp8(gathered), self.rhs, out, m_indices)
        chosen = out[row].float().view(tokens, self.top, outputs)
        error = (picked[..., None] * chosen).sum(1) - target
        # backward
        dy = error * (2.0 / error.numel())
        dout = torch.zeros(rows, outputs, dtype=torch.bfloat16, device="cuda")
        dout[row] = (picked[..., None] * dy[:, None]).view(-1, outputs).to(torch.bfloat16)
        yan.k_grouped_fp8_linear_wgrad(dout, gathered, starts, sizes, out=self.weight_grad)
        dgate = torch.zeros_like(gates).scatter_(1, ids, (chosen * dy[:, None]).sum(2))
        dlogits += gates * (dgate - (gates * dgate).sum(1, keepdim=True))
        # update
        self.step += 1
        (wm, wv), (rm, rv) = self.weight_moments, self.router_moments
        yan.adamw_step([self.weight], [self.weight_grad], [wm], [wv], lr=lr, step=self.step, copies=[self.copy])
        yan.adamw_step([self.router], [dlogits.t() @ x.float()], [rm], [rv], lr=lr, step=self.step)
        self.quantize()
        return error.square().mean(), balance_loss, sizes


def train(steps: int = 60, tokens: int = 2048, experts: int = 8, inputs: int = 512, outputs: int = 256, top: int = 2, seed: int = 0):
    """Fits targets that a hidden layer of the same kind makes; returns the errors of all steps."""
    gen = torch.Generator(device="cuda").manual_seed(seed + 1)
    layer = MoeLayer(experts, inputs, outputs, top, seed)
    hidden = torch.randn(outputs, inputs, generator=gen, device="cuda") * inputs ** -0.5
    errors = []
    for _ in range(steps):
        x = torch.randn(tokens, inputs, generator=gen, device="cuda").to(torch.bfloat16)
        error, balance, sizes = layer.train_step(x, x.float() @ hidden.t())
        errors.append(error)
    assert yan.read_device_status() == 0, "a device-side wait ran out"
    return torch.stack(errors).tolist(), balance.item(), sizes.tolist()


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=60)
    errors, balance, sizes = train(ap.parse_args().steps)
    print(f"mean squared error {errors[0]:.4f} -> {errors[-1]:.4f}, balance loss {balance:.5f}, selections per expert {sizes}")
