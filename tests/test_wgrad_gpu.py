"""fp8_linear_wgrad and k_grouped_fp8_linear_wgrad against their definition in 64 bits.

Tolerances.  Codes and scales are exact (the definition has one answer), products of two e4m3 values and powers of two are exact, so
that only the sums round.  A chain of additions in the accumulator takes 32 tokens at a time and rounds each to at worst 2^-22 of what
has been summed in magnitude: |error| <= (tokens / 32 + 4) * 2^-22 * sum of |a b|.  As a matrix, with errors of either sign or at worst
one ulp (2^-23) of the running sum each: relative Frobenius error <= (tokens / 32 + 4) * 2^-23.  bf16 output adds half an ulp, 2^-8
relative with margin; accumulation one rounding of the sum, 2^-23."""
import pytest
import torch

from oracle import train

pytestmark = pytest.mark.gpu


def _inputs(m, n, k, seed=0, dy_scale=1e-3):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k, generator=g)
    x *= torch.where(torch.rand(k, generator=g) < 0.02, 20.0, 1.0)
    dy = torch.randn(m, n, generator=g) * torch.exp(torch.randn(m, 1, generator=g)) * dy_scale
    return dy.to(torch.bfloat16).cuda(), x.to(torch.bfloat16).cuda()


def _check(out, want, size, tokens, old=None):
    want, got = want + (0 if old is None else old.double()), out.double()
    steps = tokens / 32 + 4
    bound = steps * 2.0 ** -22 * size + want.abs() * 2.0 ** -22
    if out.dtype == torch.bfloat16:
        bound = bound + want.abs() * 2.0 ** -8
    assert torch.isfinite(got).all()
    assert ((got - want).abs() <= bound).all(), ((got - want).abs() / bound.clamp(min=1e-300)).max().item()
    if want.norm() > 0:
        far = ((got - want).norm() / want.norm()).item()
        assert far <= (2.0 ** -8 if out.dtype == torch.bfloat16 else steps * 2.0 ** -23), far


@pytest.mark.parametrize("m", [1, 31, 128, 129, 640, 2085])
@pytest.mark.parametrize("n,k", [(1, 1), (7, 300), (130, 16), (128, 256), (257, 129), (272, 528)])
def test_dense(cuda_lib, m, n, k):
    import yan_b200
    dy, x = _inputs(m, n, k, seed=m + n + k)
    out = yan_b200.fp8_linear_wgrad(dy, x)
    assert out.dtype == torch.float32 and out.shape == (n, k)
    _check(out, *train.weight_grad(dy, x), m)
    assert yan_b200.read_device_status() == 0


@pytest.mark.parametrize("m,n,k", [(4096, 640, 512), (9000, 200, 72), (20000, 128, 256), (1024, 2304, 2560)])
def test_larger_and_shared_tokens(cuda_lib, m, n, k):
    """Whole waves of tiles, and few tiles with many tokens (several CTAs share a tile); twice with the same bits."""
    import yan_b200
    dy, x = _inputs(m, n, k, seed=1)
    out = yan_b200.fp8_linear_wgrad(dy, x)
    _check(out, *train.weight_grad(dy, x), m)
    assert torch.equal(out, yan_b200.fp8_linear_wgrad(dy, x))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", [(300, 200, 264), (300, 131, 77), (0, 64, 64), (6000, 100, 60)])
def test_accumulate_and_output_types(cuda_lib, dtype, m, n, k):
    import yan_b200
    dy, x = _inputs(m, n, k, seed=2)
    old = (torch.randn(n, k, device="cuda") * 0.05).to(dtype)
    want = train.weight_grad(dy, x)
    out = old.clone()
    assert yan_b200.fp8_linear_wgrad(dy, x, out=out, accumulate=True) is out
    _check(out, *want, m, old)
    fresh = torch.full((n, k), float("nan"), device="cuda", dtype=dtype)
    yan_b200.fp8_linear_wgrad(dy, x, out=fresh)
    _check(fresh, *want, m)


@pytest.mark.parametrize("offset,pad", [(0, 8), (1, 3), (8, 24), (16, 16)])
def test_strides_and_alignment(cuda_lib, offset, pad):
    """Column slices of wider matrices for both operands and the output; what surrounds the output keeps its values."""
    import yan_b200
    m, n, k = 333, 144, 208
    dy, x = _inputs(m, n, k, seed=3)
    wide_dy = torch.full((m, n + offset + pad), float("nan"), dtype=torch.bfloat16, device="cuda")
    wide_x = torch.full((m, k + offset + pad), float("nan"), dtype=torch.bfloat16, device="cuda")
    wide_dy[:, offset:offset + n], wide_x[:, offset:offset + k] = dy, x
    out = torch.full((n + 2, k + offset + pad), 7.0, device="cuda")
    yan_b200.fp8_linear_wgrad(wide_dy[:, offset:offset + n], wide_x[:, offset:offset + k], out=out[1:n + 1, offset:offset + k])
    _check(out[1:n + 1, offset:offset + k], *train.weight_grad(dy, x), m)
    out[1:n + 1, offset:offset + k] = 7.0
    assert (out == 7.0).all()


def test_values_at_the_edges_of_the_formats(cuda_lib):
    """Columns of zeros, of bf16's smallest and largest magnitudes, amax on and beside 448 * 2^e, ties of the codes."""
    import yan_b200
    m = 200
    dy = torch.zeros(m, 128, dtype=torch.bfloat16)
    x = torch.zeros(m, 64, dtype=torch.bfloat16)
    g = torch.Generator().manual_seed(4)
    base = torch.randn(m, generator=g)
    for c, s in enumerate((2.0 ** -133, 2.0 ** -127, 2.0 ** -119, 1e-30, 1e-8, 1.0, 448.0, 2.0 ** 100)):
        dy[:, c] = (base.sign() * s).to(torch.bfloat16)
        dy[:, 8 + c] = (base * s).to(torch.bfloat16)
    for c, top in enumerate((448.0, 450.0, 446.0, 1.75, 1.7578125, 0.875, 224.0, 256.0)):
        dy[:, 16 + c] = (base.clamp(-1, 1) * top).to(torch.bfloat16)
        dy[0, 16 + c] = top
        x[:, c] = (torch.randint(-17, 18, (m,), generator=g).float() * 0.5 * top).to(torch.bfloat16)
    x[:, 8:] = torch.randn(m, 56, generator=g).to(torch.bfloat16)
    dy, x = dy.cuda(), x.cuda()
    out = yan_b200.fp8_linear_wgrad(dy, x)
    want, size = train.weight_grad(dy, x)
    bound = (m / 32 + 4) * 2.0 ** -22 * size + 2.0 ** -126  # what fp32 flushes or rounds below its normal range
    assert ((out.double() - want).abs() <= bound).all()
    assert (out[24:] == 0).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_not_finite_values_stay_in_their_row_and_column(cuda_lib, bad):
    import yan_b200
    m, n, k = 300, 140, 200
    dy, x = _inputs(m, n, k, seed=5)
    clean = yan_b200.fp8_linear_wgrad(dy, x)
    dy[177, 33] = bad
    x[5, 120] = bad
    out = yan_b200.fp8_linear_wgrad(dy, x)
    assert torch.isnan(out[33]).all() and torch.isnan(out[:, 120]).all()
    out[33], out[:, 120] = clean[33], clean[:, 120]
    assert torch.equal(out, clean)


GROUPS = {
    "one": [300],
    "ragged": [0, 1, 127, 128, 129, 500, 0, 3],
    "empty at the ends": [0, 700, 0],
    "all empty": [0, 0, 0, 0],
    "many": [(i * 37) % 150 for i in range(70)],
}


@pytest.mark.parametrize("name", GROUPS)
@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("accumulate", [True, False])
def test_groups(cuda_lib, name, aligned, accumulate):
    """Starts on multiples of 128 or rows packed; rows outside of every group hold NaN."""
    import yan_b200
    sizes, n, k = GROUPS[name], 136, 264
    starts, at = [], 5 if not aligned else 0
    for s in sizes:
        starts.append(at)
        at += -(-s // 128) * 128 if aligned else s
    rows = at + 3
    dy, x = _inputs(rows, n, k, seed=6)
    inside = torch.zeros(rows, dtype=torch.bool, device="cuda")
    for a, s in zip(starts, sizes):
        inside[a:a + s] = True
    dy[~inside], x[~inside] = float("nan"), float("nan")
    old = torch.randn(len(sizes), n, k, device="cuda") * 0.01
    out = old.clone()
    to = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    yan_b200.k_grouped_fp8_linear_wgrad(dy, x, to(starts), to(sizes), out=out, accumulate=accumulate)
    for g, (a, s) in enumerate(zip(starts, sizes)):
        if s == 0:
            assert torch.equal(out[g], old[g] if accumulate else torch.zeros_like(old[g]))
        else:
            _check(out[g], *train.weight_grad(dy[a:a + s], x[a:a + s]), s, old[g] if accumulate else None)
    assert yan_b200.read_device_status() == 0


def test_groups_in_any_order_and_shared_tokens(cuda_lib):
    """Starts that do not ascend; few tiles, so that several CTAs share the tokens of a group, more than a small one has."""
    import yan_b200
    sizes, starts, n, k = [3000, 4, 0, 1100], [1200, 0, 9, 90], 100, 250
    dy, x = _inputs(4300, n, k, seed=7)
    to = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    out = yan_b200.k_grouped_fp8_linear_wgrad(dy, x, to(starts), to(sizes))
    for g, (a, s) in enumerate(zip(starts, sizes)):
        if s:
            _check(out[g], *train.weight_grad(dy[a:a + s], x[a:a + s]), s)
        else:
            assert (out[g] == 0).all()


def test_group_lists_that_leave_the_matrix_are_cut(cuda_lib):
    import yan_b200
    dy, x = _inputs(500, 64, 80, seed=8)
    to = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    out = yan_b200.k_grouped_fp8_linear_wgrad(dy, x, to([400, 600, -20, 130]), to([1000, 50, 120, -5]))
    _check(out[0], *train.weight_grad(dy[400:], x[400:]), 100)
    assert (out[1] == 0).all() and (out[3] == 0).all()
    _check(out[2], *train.weight_grad(dy[:120], x[:120]), 120)


def test_dirty_workspace_other_stream_and_graph(cuda_lib):
    """The scratch's content does not matter; the work runs on the current stream; a captured call replays on new inputs."""
    import yan_b200
    m, n, k = 5000, 120, 96
    dy, x = _inputs(m, n, k, seed=9)
    want = yan_b200.fp8_linear_wgrad(dy, x)
    ws = torch.full((yan_b200.fp8_linear_wgrad_workspace_bytes(m, n, k),), 255, dtype=torch.uint8, device="cuda")
    assert torch.equal(want, yan_b200.fp8_linear_wgrad(dy, x, workspace=ws))
    side = torch.cuda.Stream()
    later = torch.zeros_like(dy)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(2_000_000)
        later.copy_(dy)
        out = yan_b200.fp8_linear_wgrad(later, x)
    side.synchronize()
    assert torch.equal(out, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = yan_b200.fp8_linear_wgrad(later, x)
    other = _inputs(m, n, k, seed=10)[0]
    later.copy_(other)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(captured, yan_b200.fp8_linear_wgrad(other, x))


def test_is_the_gradient(cuda_lib):
    """Against differences: loss(W) = sum of dy * (x W^T) over the quantized operands, along random directions."""
    import yan_b200
    dy, x = _inputs(260, 96, 112, seed=11, dy_scale=1.0)
    out = yan_b200.fp8_linear_wgrad(dy, x).double()
    a, b = train.cast_tokens(dy), train.cast_tokens(x)
    w = torch.randn(96, 112, dtype=torch.float64, device="cuda")
    for seed in range(3):
        d = torch.randn(96, 112, dtype=torch.float64, device="cuda", generator=torch.Generator("cuda").manual_seed(seed))
        slope = ((a * (b @ (w + d).t())).sum() - (a * (b @ (w - d).t())).sum()) / 2
        # (tokens / 32 + 4) 2^-22 of the magnitudes in fp32, 2^-40 in the differences
        bound = (260 / 32 + 4) * 2.0 ** -22 * ((a.abs().t() @ b.abs()) * d.abs()).sum() + 2.0 ** -40 * (a.abs() * (b.abs() @ w.abs().t())).sum()
        assert (slope - (out * d).sum()).abs() <= bound


@pytest.mark.parametrize("sms", [2, 6, 14])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", [(300, 700, 392), (300, 300, 188), (1, 1000, 768), (2048, 520, 960), (5000, 530, 380), (8200, 260, 572)])
def test_accumulate_with_several_tiles_per_pair(cuda_lib, monkeypatch, sms, dtype, m, n, k):
    """What the matrix holds is fetched while the tile in front is stored: tiles whose rows or columns end early, tiles that pairs share
    between whole ones, both widths of tiles; a slice of a wider matrix, whose surroundings keep their values."""
    import yan_b200
    from yan_b200.jit_kernels import utils
    monkeypatch.setattr(utils, "_num_sms", sms)
    dy, x = _inputs(m, n, k, seed=sms)
    wide = (torch.randn(n, k + 24, device="cuda") * 0.05).to(dtype)
    before = wide.clone()
    yan_b200.fp8_linear_wgrad(dy, x, out=wide[:, 8:8 + k], accumulate=True)
    _check(wide[:, 8:8 + k], *train.weight_grad(dy, x), m, before[:, 8:8 + k])
    assert torch.equal(wide[:, :8], before[:, :8]) and torch.equal(wide[:, 8 + k:], before[:, 8 + k:])
    assert yan_b200.read_device_status() == 0


@pytest.mark.parametrize("sms", [2, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("sizes", [[0, 130, 1, 0, 700, 257], [64] * 20, [0, 0, 0], [4200, 0, 90]])
def test_accumulate_over_groups_with_several_tiles_per_pair(cuda_lib, monkeypatch, sms, dtype, sizes):
    import yan_b200
    from yan_b200.jit_kernels import utils
    monkeypatch.setattr(utils, "_num_sms", sms)
    n, k = 300, 264
    dy, x = _inputs(max(sum(sizes), 1), n, k, seed=sms)
    lengths = torch.tensor(sizes, dtype=torch.int32, device="cuda")
    starts = lengths.cumsum(0).to(torch.int32) - lengths
    old = (torch.randn(len(sizes), n, k, device="cuda") * 0.05).to(dtype)
    out = old.clone()
    yan_b200.k_grouped_fp8_linear_wgrad(dy, x, starts, lengths, out=out, accumulate=True)
    for g, (start, size) in enumerate(zip(starts.tolist(), sizes)):
        if size == 0:
            assert torch.equal(out[g], old[g])
        else:
            _check(out[g], *train.weight_grad(dy[start:start + size], x[start:start + size]), size, old[g])
