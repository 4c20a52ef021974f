"""adamw_step against its definition in 64 bits, and its 8-bit states against the definition's own sequence of fp32 operations.

Tolerances.  m and v are two products and a sum in fp32: 3 roundings, |error| <= 2^-22 (|b m| + |(1 - b) g|) with the constants' own
rounding.  The parameter adds the decay product (2^-24), its rounding (2^-24 |p|) and the update, whose factors are off by 2^-20
relative in all (roots, quotient, constants): |error| <= 2^-22 |p| + 2^-18 |update|.  bf16 results: half an ulp, 2^-8 relative with margin.
8-bit states: the operator defines each fp32 operation in front of the rounding to a code, so codes and scales are compared bit for
bit (gradients and codes are coarse numbers, whose sums lie on the codes' rounding points more often than by chance: one element in a
hundred falls to the other side when the sum is done in 64 bits).  Against 64 bits a value is one code off at most, a step of 2^-3 of
the value or 2^-9 of the scale.  The parameter is compared with 64 bits from the fp32 m and v: where the two terms of m cancel, its own
rounding is no longer small beside it."""
import pytest
import torch

from oracle import train

pytestmark = pytest.mark.gpu

HYPER = dict(lr=2e-3, beta1=0.9, beta2=0.95, eps=1e-8)


def _tensors(sizes, dtype, seed, scale):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=g) * scale).to(dtype).cuda() for s in sizes]


def _decode(state):
    codes, scales = state
    return codes.double() * scales.double().repeat_interleave(128)[:codes.numel()]


def _check_param(got, want, before, update):
    bound = 2.0 ** -22 * before.double().abs() + 2.0 ** -18 * update.abs() + 2.0 ** -140
    if got.dtype == torch.bfloat16:
        bound = bound + want.abs() * 2.0 ** -8
    assert ((got.double() - want).abs() <= bound).all(), ((got.double() - want).abs() / bound).max().item()


SIZES = {"one element": [1], "odd": [1, 2, 3, 5, 127, 128, 129, 4095, 4096, 4097, 10001], "large": [1 << 20, 300_007],
         "many": [(i * 613) % 700 + 1 for i in range(500)]}


@pytest.mark.parametrize("name", SIZES)
@pytest.mark.parametrize("param", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("grad", [torch.float32, torch.bfloat16])
def test_32_bit_states(cuda_lib, name, param, grad):
    import yan_b200
    sizes = SIZES[name]
    p, g = _tensors(sizes, param, 0, 0.02), _tensors(sizes, grad, 1, 1e-3)
    m, v = _tensors(sizes, torch.float32, 2, 1e-3), [t.square() for t in _tensors(sizes, torch.float32, 3, 1e-3)]
    decays = [0.1 * (i % 2) for i in range(len(sizes))]
    scale = torch.tensor([0.37], device="cuda")
    before = [[t.clone() for t in l] for l in (p, m, v)]
    copies = [torch.zeros(s, dtype=torch.bfloat16, device="cuda") for s in sizes]
    yan_b200.adamw_step(p, g, m, v, **HYPER, weight_decay=decays, step=7, grad_scale=scale, copies=copies)
    for i in range(len(sizes)):
        p0, m0, v0 = (l[i] for l in before)
        wp, wm, wv, root = train.adamw(p0, g[i], m0, v0, **HYPER, weight_decay=decays[i], step=7, grad_scale=scale.double().item())
        gs = g[i].double().abs() * 0.37
        assert ((m[i].double() - wm).abs() <= 2.0 ** -22 * (0.9 * m0.double().abs() + 0.1 * gs) + 2.0 ** -149).all()
        assert ((v[i].double() - wv).abs() <= 2.0 ** -21 * wv + 2.0 ** -149).all()
        _check_param(p[i], wp, p0, wp - p0.double())
        _check_param(copies[i], wp, p0, wp - p0.double())


@pytest.mark.parametrize("name", SIZES)
@pytest.mark.parametrize("param,grad", [(torch.float32, torch.float32), (torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16),
                                        (torch.bfloat16, torch.float32)])
def test_8_bit_states(cuda_lib, name, param, grad):
    """From new states, three steps: each against the definition applied to the state that the step found."""
    import yan_b200
    sizes = SIZES[name]
    betas = dict(beta1=HYPER["beta1"], beta2=HYPER["beta2"])
    p = _tensors(sizes, param, 0, 0.02)
    m, v = ([yan_b200.adamw_state(t, 8) for t in p] for _ in range(2))
    for step in (1, 2, 3):
        g = _tensors(sizes, grad, 10 + step, 1e-3)
        before = [(p[i].clone(), _decode(m[i]), _decode(v[i])) for i in range(len(sizes))]
        yan_b200.adamw_step(p, g, m, v, **HYPER, weight_decay=0.1, step=step)
        for i in range(len(sizes)):
            p0, m0, r0 = before[i]
            _, wm, wv, root = train.adamw(p0, g[i], m0, r0.square(), **HYPER, weight_decay=0.1, step=step)
            fm, fv, froot = train.adamw_states_fp32(g[i], m0, r0.square(), **betas)
            wp, update = train.adamw_param(p0, fm, fv, **HYPER, weight_decay=0.1, step=step)
            _check_param(p[i], wp, p0, update)
            for state, exact, own, positive in ((m[i], wm, fm, False), (v[i], root, froot, True)):
                got = _decode(state)
                value, scale = train.encode_state(own, positive)
                assert torch.equal(state[1].double(), scale) and torch.equal(got, value)
                value, scale = train.encode_state(exact, positive)
                same_scale = (state[1].double() == scale).repeat_interleave(128)[:got.numel()]
                step_size = torch.maximum(value.abs() * 2.0 ** -3, scale.repeat_interleave(128)[:got.numel()] * 2.0 ** -9) * 1.001
                assert ((got - value).abs() <= torch.where(same_scale, step_size, step_size * 2)).all()
                if positive:
                    assert ((got > 0) == (exact > 0)).all()


@pytest.mark.parametrize("bits", [8, 32])
def test_alignment(cuda_lib, bits):
    """Pieces of flat buffers that start anywhere give what aligned tensors give, and their neighbours keep their values."""
    import yan_b200
    sizes = [1000, 257, 4100]
    p, g = _tensors(sizes, torch.float32, 0, 0.02), _tensors(sizes, torch.bfloat16, 1, 1e-3)

    def states():
        return [yan_b200.adamw_state(t, bits) for t in p]

    def shifted(tensors):
        flat = [torch.full((t.numel() + 9,), 3.0, device="cuda").to(t.dtype) if t.dtype != torch.float8_e4m3fn else
                torch.full((t.numel() + 9,), 3, dtype=torch.uint8, device="cuda").view(t.dtype) for t in tensors]
        out = [f[1 + i % 3:1 + i % 3 + t.numel()] for i, (f, t) in enumerate(zip(flat, tensors))]
        for o, t in zip(out, tensors):
            o.view(torch.uint8 if t.dtype == torch.float8_e4m3fn else t.dtype).copy_(t.view(torch.uint8 if t.dtype == torch.float8_e4m3fn else t.dtype))
        return flat, out

    m, v, m2, v2 = states(), states(), states(), states()
    flat_p, p2 = shifted(p)
    _, g2 = shifted(g)
    if bits == 8:
        m2 = list(zip(shifted([s[0] for s in m2])[1], [s[1] for s in m2]))
        v2 = list(zip(shifted([s[0] for s in v2])[1], [s[1] for s in v2]))
    else:
        m2, v2 = shifted(m2)[1], shifted(v2)[1]
    for step in (1, 2):
        yan_b200.adamw_step(p, g, m, v, **HYPER, step=step)
        yan_b200.adamw_step(p2, g2, m2, v2, **HYPER, step=step)
    for i in range(len(sizes)):
        assert torch.equal(p[i], p2[i])
        for a, b in ((m[i], m2[i]), (v[i], v2[i])):
            if bits == 8:
                assert torch.equal(a[0].view(torch.uint8), b[0].view(torch.uint8)) and torch.equal(a[1], b[1])
            else:
                assert torch.equal(a, b)
        flat_p[i][1 + i % 3:1 + i % 3 + sizes[i]] = 3.0
        assert (flat_p[i] == 3.0).all()


def test_not_finite_values_stay_in_their_element(cuda_lib):
    import yan_b200
    for bits in (8, 32):
        runs = []
        for poison in (False, True):
            p = _tensors([600], torch.float32, 0, 0.02)
            g = _tensors([600], torch.float32, 1, 1e-3)
            g[0][17] = 0.0
            g[0][400] = 0.0
            if poison:
                g[0][17], g[0][400] = float("nan"), float("inf")
            m, v = [yan_b200.adamw_state(p[0], bits)], [yan_b200.adamw_state(p[0], bits)]
            yan_b200.adamw_step(p, g, m, v, **HYPER, step=1)
            runs.append((p[0], *((_decode(m[0]), _decode(v[0])) if bits == 8 else (m[0], v[0]))))
        for clean, hit in zip(*runs):
            assert not torch.isfinite(hit[[17, 400]]).any() or hit is runs[1][0]
            assert torch.isnan(hit[17])
            keep = torch.ones(600, dtype=torch.bool, device="cuda")
            keep[[17, 400]] = False
            assert torch.equal(clean[keep], hit[keep])


def test_extreme_magnitudes(cuda_lib):
    """Gradients whose squares vanish in fp32, blocks below 2^-111, and large ones: no code of zero for a root above zero, nothing turns
    infinite or NaN."""
    import yan_b200
    g = torch.cat([torch.full((128,), 1e-30), torch.full((128,), 1e-36), torch.linspace(1e-19, 1e-3, 128), torch.full((128,), 1e15)]).cuda()
    p = [torch.ones(512, device="cuda")]
    m, v = [yan_b200.adamw_state(p[0], 8)], [yan_b200.adamw_state(p[0], 8)]
    yan_b200.adamw_step(p, [g], m, v, **HYPER, step=1)
    assert torch.isfinite(p[0]).all()
    values, roots = _decode(m[0]), _decode(v[0])
    assert (values[128:256] == 0).all() and (roots[:256] == 0).all()  # 1e-36 / 10 is below 2^-111; the squares vanish
    assert (roots[256:] > 0).all() and torch.isfinite(roots).all()


def test_empty_lists_and_tensors(cuda_lib):
    import yan_b200
    yan_b200.adamw_step([], [], [], [], lr=1e-3, step=1)
    p, g = _tensors([0, 10, 0], torch.float32, 0, 1.0), _tensors([0, 10, 0], torch.float32, 1, 1.0)
    m, v = ([torch.zeros_like(t) for t in p] for _ in range(2))
    before = p[1].clone()
    yan_b200.adamw_step(p, g, m, v, lr=1e-3, step=1)
    assert not torch.equal(before, p[1])
    yan_b200.adamw_step(p[:1], g[:1], m[:1], v[:1], lr=1e-3, step=1)


def test_shapes_other_stream_and_graph(cuda_lib):
    """Tensors of several dimensions; on another stream, behind what writes the gradient there; as a replayed graph."""
    import yan_b200
    shape = (64, 3, 50)
    g0 = torch.randn(shape, device="cuda")

    def fresh():
        p = [torch.ones(shape, device="cuda")]
        return p, [torch.zeros(shape, device="cuda")], [torch.zeros(shape, device="cuda")]

    p, m, v = fresh()
    yan_b200.adamw_step(p, [g0], m, v, **HYPER, step=1)
    q, m2, v2 = fresh()
    g = torch.zeros(shape, device="cuda")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(2_000_000)
        g.copy_(g0)
        yan_b200.adamw_step(q, [g], m2, v2, **HYPER, step=1)
    side.synchronize()
    assert torch.equal(p[0], q[0]) and torch.equal(m[0], m2[0]) and torch.equal(v[0], v2[0])
    q, m2, v2 = fresh()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        yan_b200.adamw_step(q, [g], m2, v2, **HYPER, step=1)
    for t, start in zip((q, m2, v2), fresh()):
        t[0].copy_(start[0])
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(p[0], q[0])
