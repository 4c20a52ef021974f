"""moe_balance_loss against its definition in 64 bits.

Tolerances.  Scores are exponentials of differences rounded to fp32 (the difference and the product with log2 e: up to 2^-23 |z - max| each,
|z - max| <= 32 here where it matters) and the function's own 2^-22: relative 2^-17 at worst for a score, sums of at most 1024 of them
by partial sums 2^-20 more.  So P, the loss (all terms are positive) and p: relative 2^-16.  The gradient is p_j (a_j - sum a p):
|error| <= 2^-15 p_j (a_j + sum a p); for the sigmoid s_j (1 - s_j) / sum with 1 - s_j off by 2^-22.  bf16: half an ulp more, 2^-8."""
import pytest
import torch

from oracle import train

pytestmark = pytest.mark.gpu


def _inputs(t, e, top, seed=0, dtype=torch.float32, spread=1.5):
    g = torch.Generator().manual_seed(seed)
    z = (torch.randn(t, e, generator=g) * spread + torch.randn(e, generator=g) * 0.7).to(dtype)
    ids = torch.rand(t, e, generator=g).topk(top, dim=1).indices if t else torch.zeros(0, top, dtype=torch.int64)
    return z.cuda(), ids.cuda()


def _formula(z, ids, score, coef=1.0, mask=None, cu_seqlens=None):
    """(loss, counts, gradient by autograd in 64 bits, what bounds its rounding)."""
    x = z.double().clone()
    if mask is not None:
        x[~mask] = 0.0  # not read
    x.requires_grad_(True)
    loss, counts = train.balance_loss(x, ids, coef=coef, score=score, mask=mask, cu_seqlens=cu_seqlens)
    grad = torch.autograd.grad(loss, x)[0] if loss.requires_grad else torch.zeros_like(x)
    # size: the same with both parts of the difference positive
    t, e = z.shape
    p = torch.softmax(x.detach(), 1) if score == "softmax" else torch.sigmoid(x.detach()) / torch.sigmoid(x.detach()).sum(1, keepdim=True)
    size = torch.zeros_like(p)
    ends = [0, t] if cu_seqlens is None else cu_seqlens.tolist()
    for s, (b, end) in enumerate(zip(ends, ends[1:])):
        n = int((mask[b:end].sum() if mask is not None else end - b))
        if n:
            a = coef / (len(ends) - 1) * e / (ids.shape[1] * n * n) * counts[s].double()
            size[b:end] = p[b:end] * (a + (p[b:end] @ a)[:, None])
    return loss.detach(), counts, grad, size


def _check(got, want, dtype):
    loss, counts, grad = got
    wl, wc, wg, size = want
    assert loss.shape == () and loss.dtype == torch.float32 and counts.dtype == torch.int32 and grad.dtype == dtype
    assert torch.equal(counts, wc)
    assert (loss.double() - wl).abs() <= 2.0 ** -16 * wl.abs()
    bound = 2.0 ** -15 * size + 2.0 ** -120
    if dtype == torch.bfloat16:
        bound = bound + wg.abs() * 2.0 ** -8
    assert ((grad.double() - wg).abs() <= bound).all(), ((grad.double() - wg).abs() / bound).max().item()


@pytest.mark.parametrize("t", [1, 2, 33, 700, 5000])
@pytest.mark.parametrize("e,top", [(1, 1), (3, 2), (8, 2), (31, 4), (64, 6), (160, 6), (256, 8), (500, 1), (512, 10), (1000, 3), (1024, 8)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_one_sequence(cuda_lib, t, e, top, score):
    import yan_b200
    for dtype in (torch.float32, torch.bfloat16):
        z, ids = _inputs(t, e, top, seed=t + e, dtype=dtype)
        _check(yan_b200.moe_balance_loss(z, ids, score=score, coef=0.5), _formula(z, ids, score, coef=0.5), dtype)


@pytest.mark.parametrize("lengths", [[100], [1, 1, 1, 1], [0, 50, 0, 0, 3, 0], [300, 1, 700, 0, 64, 65], [7] * 90, [0, 0]])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("masked", [False, True])
def test_sequences_and_masks(cuda_lib, lengths, score, masked):
    """Ragged and empty sequences; masked tokens hold NaN and infinities and leave no trace; one sequence masked entirely."""
    import yan_b200
    t = sum(lengths)
    z, ids = _inputs(t, 72, 5, seed=t)
    cu = torch.tensor([0, *lengths], device="cuda").cumsum(0).to(torch.int32)
    mask = None
    if masked:
        mask = torch.rand(t, generator=torch.Generator().manual_seed(1)).cuda() < 0.7
        if len(lengths) > 2:
            mask[cu[2]:cu[3]] = False
        z[~mask] = torch.tensor([float("nan"), float("inf"), -float("inf")], device="cuda").repeat(24)
    got = yan_b200.moe_balance_loss(z, ids, score=score, token_mask=mask, cu_seqlens=cu)
    _check(got, _formula(z, ids, score, mask=mask, cu_seqlens=cu), torch.float32)
    if masked:
        assert (got[2][~mask] == 0).all()


def test_tokens_outside_of_the_sequences(cuda_lib):
    import yan_b200
    z, ids = _inputs(400, 16, 2)
    cu = torch.tensor([30, 100, 100, 350], dtype=torch.int32, device="cuda")
    loss, counts, grad = yan_b200.moe_balance_loss(z, ids, cu_seqlens=cu)
    _check((loss, counts, grad), _formula(z, ids, "softmax", cu_seqlens=cu), torch.float32)
    assert (grad[:30] == 0).all() and (grad[350:] == 0).all()


def test_dropped_selections_and_narrow_ids(cuda_lib):
    import yan_b200
    z, ids = _inputs(300, 24, 4)
    ids[::3, 1] = -1
    ids[::5, 2] = 24
    ids[7, 0] = 1 << 40
    _check(yan_b200.moe_balance_loss(z, ids), _formula(z, ids, "softmax"), torch.float32)
    ids[7, 0] = -1
    a, b = yan_b200.moe_balance_loss(z, ids), yan_b200.moe_balance_loss(z, ids.to(torch.int32))
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_masked_experts_and_lowest_values(cuda_lib, score):
    """Experts that a -inf or the type's lowest value takes out, for some tokens all of them."""
    import yan_b200
    low = torch.finfo(torch.float32).min
    z, ids = _inputs(200, 40, 3)
    z[:, 5] = -float("inf")
    z[::2, 6:20] = low
    z[11] = -float("inf")
    z[12] = low
    loss, counts, grad = yan_b200.moe_balance_loss(z, ids, score=score)
    x = z.clone()
    keep = torch.ones(200, dtype=torch.bool, device="cuda")
    keep[11] = False
    if score == "sigmoid":
        keep[12] = False
    wl, wc = train.balance_loss(x, ids, score=score)
    assert torch.equal(counts, wc) and (loss.double() - wl).abs() <= 2.0 ** -16 * wl
    assert torch.isfinite(grad).all() and (grad[~keep] == 0).all()
    # the gradient of the rows that have scores, without the rows that have none
    a = 40 / (3 * 200 * 200) * counts[0].double()
    s = torch.softmax(x.double(), 1) if score == "softmax" else torch.sigmoid(x.double())
    p = s[keep] / s[keep].sum(1, keepdim=True)
    slope = p if score == "softmax" else p * (1 - s[keep])
    want = slope * (a - (p @ a)[:, None])
    assert ((grad[keep].double() - want).abs() <= 2.0 ** -15 * slope * (a + (p @ a)[:, None]) + 2.0 ** -120).all()


def test_a_nan_logit_reaches_the_loss(cuda_lib):
    import yan_b200
    z, ids = _inputs(100, 16, 2)
    clean = yan_b200.moe_balance_loss(z, ids)
    z[40, 3] = float("nan")
    loss, counts, grad = yan_b200.moe_balance_loss(z, ids)
    assert torch.isnan(loss) and torch.isnan(grad[40]).all() and torch.equal(counts, clean[1])
    keep = torch.arange(100, device="cuda") != 40
    assert torch.equal(grad[keep], clean[2][keep])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offset,pad", [(0, 0), (1, 2), (8, 8), (4, 0)])
def test_strides(cuda_lib, dtype, offset, pad):
    """Columns of wider matrices for logits and gradient; what surrounds the gradient keeps its values."""
    import yan_b200
    z, ids = _inputs(222, 48, 4, dtype=dtype)
    wide = torch.full((222, 48 + offset + pad), float("nan"), dtype=dtype, device="cuda")
    wide[:, offset:offset + 48] = z
    out = torch.full_like(wide, 5.0)
    grad = out[:, offset:offset + 48]
    got = yan_b200.moe_balance_loss(wide[:, offset:offset + 48], ids, grad=grad)
    assert got[2] is grad
    _check(got, _formula(z, ids, "softmax"), dtype)
    grad.fill_(5.0)
    assert (out == 5.0).all()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_gradient_against_differences(cuda_lib, score):
    import yan_b200
    z, ids = _inputs(60, 20, 3, spread=1.0)
    cu = torch.tensor([0, 25, 60], dtype=torch.int32, device="cuda")
    loss, counts, grad = yan_b200.moe_balance_loss(z, ids, score=score, cu_seqlens=cu)
    h = 1e-4
    for seed in range(4):
        d = torch.randn(60, 20, dtype=torch.float64, generator=torch.Generator().manual_seed(seed)).cuda()
        up, down = (train.balance_loss(z.double() + s * h * d, ids, score=score, cu_seqlens=cu, counts=counts)[0] for s in (1, -1))
        slope = (up - down) / (2 * h)
        # h^2 times a third derivative of order |grad| |d|^3, and 2^-15 of the gradient's size
        assert (slope - (grad.double() * d).sum()).abs() <= (1e-6 + 2.0 ** -14) * (grad.double().abs() * d.abs()).sum() + 1e-9 * loss


def test_without_gradient_empty_and_repeated(cuda_lib):
    import yan_b200
    z, ids = _inputs(3000, 96, 4)
    a = yan_b200.moe_balance_loss(z, ids)
    b = yan_b200.moe_balance_loss(z, ids, with_grad=False)
    assert b[2] is None and torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    c = yan_b200.moe_balance_loss(z, ids)
    assert all(torch.equal(x, y) for x, y in zip(a, c))  # the same bits
    loss, counts, grad = yan_b200.moe_balance_loss(z[:0], ids[:0])
    assert loss.item() == 0 and (counts == 0).all() and grad.shape == (0, 96)


def test_balanced_experts_give_the_coefficient(cuda_lib):
    import yan_b200
    ids = (torch.arange(640, device="cuda")[:, None] * 2 + torch.arange(2, device="cuda")) % 64
    loss, counts, grad = yan_b200.moe_balance_loss(torch.zeros(640, 64, device="cuda"), ids, coef=0.25)
    assert (counts == 20).all() and abs(loss.item() - 0.25) <= 0.25 * 2.0 ** -16 and grad.abs().max() <= 2.0 ** -15 * 0.25 / 640


def test_dirty_workspace_other_stream_and_graph(cuda_lib):
    import yan_b200
    z0, ids = _inputs(2500, 128, 8)
    want = yan_b200.moe_balance_loss(z0, ids)
    ws = torch.full((yan_b200.moe_balance_loss_workspace_bytes(2500, 128),), 255, dtype=torch.uint8, device="cuda")
    assert all(torch.equal(x, y) for x, y in zip(want, yan_b200.moe_balance_loss(z0, ids, workspace=ws)))
    z = torch.zeros_like(z0)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(2_000_000)
        z.copy_(z0)
        got = yan_b200.moe_balance_loss(z, ids)
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = yan_b200.moe_balance_loss(z, ids)
    z.copy_(z0 * 0.5)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(captured, yan_b200.moe_balance_loss(z0 * 0.5, ids)))
