"""The training operators together, as the example runs them: the error falls, run after run to the same bits; and every operator gives the
same through its native front and without it."""
import importlib.util
import os

import pytest
import torch

from oracle import train as oracle

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _example():
    spec = importlib.util.spec_from_file_location("train_moe_layer", os.path.join(ROOT, "examples", "train_moe_layer.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def _plain_errors(layer, steps, tokens, inputs, outputs, seed):
    """The same training without quantization: torch's autograd and AdamW in 32 bits, on the example's data."""
    gen = torch.Generator(device="cuda").manual_seed(seed + 1)
    hidden = torch.randn(outputs, inputs, generator=gen, device="cuda") * inputs ** -0.5
    weight, router = (t.clone().requires_grad_(True) for t in (layer.weight, layer.router))
    optimizer = torch.optim.AdamW([weight, router], lr=2e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0)
    errors = []
    for _ in range(steps):
        x = torch.randn(tokens, inputs, generator=gen, device="cuda").to(torch.bfloat16).float()
        gates = torch.softmax(x @ router.t(), dim=1)
        picked, ids = gates.topk(layer.top, dim=1)
        all_out = torch.einsum("tk,enk->ten", x, weight)
        chosen = all_out.gather(1, ids[..., None].expand(-1, -1, outputs))
        error = ((picked[..., None] * chosen).sum(1) - x @ hidden.t()).square().mean()
        counts = torch.bincount(ids.reshape(-1), minlength=router.shape[0])
        balance = 1e-2 * router.shape[0] / (layer.top * tokens ** 2) * (counts * gates.sum(0)).sum()
        optimizer.zero_grad()
        (error + balance).backward()
        optimizer.step()
        errors.append(error.item())
    return errors


def test_the_layer_learns_as_without_quantization(cuda_lib):
    """The error of every step beside that of plain training from the same weights on the same data.  e4m3 rounds an operand by 2^-5 of its
    value at worst, 2^-5 / sqrt(3) in the mean square: both operands of a product by 2.6 %, an output (power 1.1) by 0.0007 in power, the
    gradients alike; 8-bit moments move a step by as much.  Steps that are off by 3 % at random leave an error that is a few percent off
    while it falls: 10 % and 0.01 are allowed."""
    example = _example()
    errors, balance, sizes = example.train(steps=40)
    plain = _plain_errors(example.MoeLayer(8, 512, 256, 2, 0), 40, 2048, 512, 256, 0)
    assert all(abs(e - p) <= 0.1 * p + 0.01 for e, p in zip(errors, plain)), (errors[-1], plain[-1])
    assert errors[-1] < 0.5 * errors[0]
    assert sum(sizes) == 2048 * 2 and balance > 0


def test_weight_gradient_of_the_layer(cuda_lib):
    """The gradient that a step leaves behind, against 64 bits from the same rows: experts' rows are where the router's counts say."""
    import yan_b200
    layer = _example().MoeLayer(4, 256, 128, 2)
    seen = {}
    wgrad = yan_b200.k_grouped_fp8_linear_wgrad

    def spy(dy, x, starts, sizes, out):
        seen.update(dy=dy.clone(), x=x.clone(), starts=starts.tolist(), sizes=sizes.tolist())
        return wgrad(dy, x, starts, sizes, out=out)

    yan_b200.k_grouped_fp8_linear_wgrad = spy
    try:
        x = torch.randn(700, 256, device="cuda").to(torch.bfloat16)
        layer.train_step(x, torch.randn(700, 128, device="cuda"))
    finally:
        yan_b200.k_grouped_fp8_linear_wgrad = wgrad
    assert sum(seen["sizes"]) == 1400 and all(s % 128 == 0 for s in seen["starts"])
    for g, (a, n) in enumerate(zip(seen["starts"], seen["sizes"])):
        want, size = oracle.weight_grad(seen["dy"][a:a + n], seen["x"][a:a + n])
        # the bound of the sums: 32 tokens at a time, 2^-22 of the magnitudes each
        assert ((layer.weight_grad[g].double() - want).abs() <= (n / 32 + 4) * 2.0 ** -22 * size + want.abs() * 2.0 ** -22).all()


def test_native_front_and_python_path_agree(cuda_lib, monkeypatch):
    import yan_b200
    from yan_b200 import _lib
    gen = torch.Generator(device="cuda").manual_seed(0)
    r = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    dy, x, old = r(300, 130).to(torch.bfloat16), r(300, 72).to(torch.bfloat16), r(130, 72)
    starts, sizes = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([0, 128], [100, 172]))
    params, grads = [r(777), r(40, 50)], [r(777).to(torch.bfloat16), r(40, 50).to(torch.bfloat16)]
    logits = r(333, 24)
    ids = logits.topk(3).indices
    mask, cu = torch.rand(333, device="cuda") < 0.5, torch.tensor([0, 100, 333], dtype=torch.int32, device="cuda")

    def run():
        yan_b200.get_num_sms()
        outs = [yan_b200.fp8_linear_wgrad(dy, x, out=old.clone(), accumulate=True),
                yan_b200.k_grouped_fp8_linear_wgrad(dy, x, starts, sizes, out=torch.empty(2, 130, 72, device="cuda", dtype=torch.bfloat16))]
        for bits in (8, 32):
            p, copies = [t.clone() for t in params], [torch.empty(t.shape, dtype=torch.bfloat16, device="cuda") for t in params]
            m, v = ([yan_b200.adamw_state(t, bits) for t in p] for _ in range(2))
            version = [t._version for t in p]
            yan_b200.adamw_step(p, grads, m, v, lr=1e-2, step=3, weight_decay=[0.1, 0.0], copies=copies, grad_scale=torch.full((1,), 0.5, device="cuda"))
            assert all(t._version > n for t, n in zip(p, version))
            outs += p + copies + [t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t for s in m + v for t in (s if bits == 8 else (s,))]
        return outs + list(yan_b200.moe_balance_loss(logits, ids, score="sigmoid", coef=0.3, token_mask=mask, cu_seqlens=cu))

    native = run()

    class NotTaken:
        def __getattr__(self, name):
            return lambda *args: -1

    monkeypatch.setattr(_lib, "_fast", NotTaken())
    assert all(torch.equal(a, b) for a, b in zip(native, run()))
