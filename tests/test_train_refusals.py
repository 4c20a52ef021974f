"""What the training operators refuse: the C entry points by their return code, before any CUDA call (no GPU needed), the Python
operators by an assertion."""
import ctypes

import pytest
import torch

BAD, SMALL = 1, 7
P = 0x10000  # an address that is never read: every call here is refused on the host


def _rc(name, *args):
    from yan_b200 import _lib
    return _lib.call_rc(name, *args)


def _wgrad(dy=P, x=P, out=P, m=64, n=32, k=48, dy_ld=32, x_ld=48, out_ld=48, dtype=0, accumulate=0, ws=P, ws_bytes=1 << 40, sms=148):
    return _rc("yan_b200_fp8_linear_wgrad", dy, x, out, m, n, k, dy_ld, x_ld, out_ld, dtype, accumulate, ws, ws_bytes, None, sms)


@pytest.mark.parametrize("change", [dict(m=-1), dict(n=0), dict(k=-4), dict(dy=None), dict(x=None), dict(out=None), dict(dy_ld=31), dict(x_ld=47),
                                    dict(out_ld=47), dict(dtype=2), dict(dy=P + 1), dict(out=P + 2), dict(ws=None), dict(ws=P + 128),
                                    dict(sms=0)])
def test_wgrad_arguments(change):
    assert _wgrad(**change) == BAD


def test_wgrad_workspace():
    from yan_b200 import _lib
    size = _lib.lib().yan_b200_fp8_linear_wgrad_workspace_bytes
    assert _wgrad(ws_bytes=size(64, 32, 48, 0, 148) - 1) == SMALL
    assert size(-1, 32, 48, 0, 148) == 0 and size(64, 0, 48, 0, 148) == 0 and size(64, 32, 48, 0, 0) == 0
    # codes of 128 tokens, scale tiles (128 features of dy; up to 256 of x), and nothing shared between CTAs
    assert size(64, 32, 48, 0, 148) == 128 * 32 + 128 * 48 + 512 + 1024
    # groups can begin anywhere: a block of tokens more for each
    assert size(64, 32, 48, 4, 148) == 4 * 128 * (32 + 48) + 5 * (512 + 1024)


@pytest.mark.parametrize("change", [dict(starts=None), dict(sizes=None), dict(groups=0), dict(groups=513)])
def test_grouped_wgrad_arguments(change):
    a = dict(starts=P, sizes=P, groups=4) | change
    assert _rc("yan_b200_k_grouped_fp8_linear_wgrad", P, P, P, a["starts"], a["sizes"], a["groups"], 64, 32, 48, 32, 48, 48, 32 * 48, 0, 0, P,
               1 << 40, None, 148) == BAD


def _adamw(numel=256, count=1, param=P, grad=P, m=P, v=P, ms=P, vs=P, copy=0, param_dtype=0, grad_dtype=0, bits=32, lr=1e-3, beta1=0.9, beta2=0.99,
           eps=1e-8, step=1, table=True):
    from yan_b200 import _lib
    t = (_lib.AdamwTensor * 2)()
    # a good tensor without elements in front of the one in question
    t[1].param, t[1].grad, t[1].exp_avg, t[1].exp_avg_sq = param, grad, m, v
    t[1].exp_avg_scale, t[1].exp_avg_sq_scale, t[1].copy, t[1].numel = ms, vs, copy, numel
    return _rc("yan_b200_adamw_step", t if table else None, 2 if count == 1 else count, param_dtype, grad_dtype, bits, lr, beta1, beta2, eps,
               step, None, None)


@pytest.mark.parametrize("change", [dict(numel=-1), dict(numel=1 << 62), dict(numel=1 << 62, bits=8), dict(count=-1), dict(param=0), dict(grad=0), dict(m=0), dict(v=0), dict(param=P + 2),
                                    dict(grad=P + 2), dict(m=P + 2), dict(v=P + 1), dict(copy=P + 1), dict(param_dtype=2), dict(grad_dtype=-1),
                                    dict(bits=16), dict(lr=-1.0), dict(lr=float("nan")), dict(lr=float("inf")), dict(beta1=1.0),
                                    dict(beta2=-0.1), dict(beta2=float("nan")), dict(eps=-1e-8), dict(step=0), dict(table=False),
                                    dict(bits=8, ms=0), dict(bits=8, vs=0), dict(bits=8, vs=P + 2)])
def test_adamw_arguments(change):
    assert _adamw(**change) == BAD


def test_adamw_of_nothing():
    assert _rc("yan_b200_adamw_step", None, 0, 0, 0, 32, 1e-3, 0.9, 0.99, 1e-8, 1, None, None) == 0
    assert _adamw(numel=0) == 0


def _balance(logits=P, ids=P, mask=None, cu=None, loss=P, counts=P, grad=P, t=200000, e=32, top=2, s=1, ld=32, grad_ld=32, dtype=0, ids_64=1, score=0,
             ws=P, ws_bytes=1 << 40, sms=148):
    return _rc("yan_b200_moe_balance_loss", logits, ids, mask, cu, loss, counts, grad, t, e, top, s, ld, grad_ld, dtype, ids_64, score, 1.0, ws,
               ws_bytes, None, sms)


@pytest.mark.parametrize("change", [dict(t=-1), dict(e=0), dict(e=1025, ld=2048, grad_ld=2048), dict(top=0), dict(top=65536), dict(s=0), dict(s=2), dict(s=70000, cu=P),
                                    dict(ld=31), dict(grad_ld=31), dict(dtype=2), dict(score=2), dict(logits=None), dict(ids=None),
                                    dict(loss=None), dict(counts=None), dict(logits=P + 2), dict(grad=P + 1), dict(ids=P + 4), dict(ws=None),
                                    dict(ws=P + 16), dict(sms=0)])
def test_balance_arguments(change):
    assert _balance(**change) == BAD


def test_balance_workspace():
    from yan_b200 import _lib
    size = _lib.lib().yan_b200_moe_balance_loss_workspace_bytes
    assert size(200000, 32, 1, 1, 148) > 0 and _balance(ws_bytes=size(200000, 32, 1, 1, 148) - 1) == SMALL
    assert size(64, 32, 1, 1, 148) == 0  # few tokens need none
    assert size(64, 0, 1, 1, 148) == 0


def test_python_operators_refuse_tensors_of_the_host():
    import yan_b200
    b = torch.zeros(4, 8, dtype=torch.bfloat16)
    with pytest.raises(AssertionError):
        yan_b200.fp8_linear_wgrad(b, b)
    with pytest.raises(AssertionError):
        yan_b200.k_grouped_fp8_linear_wgrad(b, b, torch.zeros(1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
    p = [torch.zeros(4)]
    with pytest.raises(AssertionError):
        yan_b200.adamw_step(p, p, p, p, lr=1e-3, step=1)
    with pytest.raises(AssertionError):
        yan_b200.moe_balance_loss(torch.zeros(4, 8), torch.zeros(4, 2, dtype=torch.int64))
    assert yan_b200.adamw_state(torch.zeros(130), 8)[1].shape == (2,) and ctypes.sizeof(__import__("yan_b200")._lib.AdamwTensor) == 72


@pytest.mark.gpu
def test_python_operators_refuse(cuda_lib):
    """Wrong types, shapes and layouts, and a matrix whose groups share memory: an AssertionError, and nothing is launched."""
    import yan_b200
    z = lambda *s, d=torch.bfloat16: torch.zeros(*s, dtype=d, device="cuda")  # noqa: E731
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    dy, x = z(64, 16), z(64, 32)
    for args, kw in [((dy.float(), x), {}), ((dy[:32], x), {}), ((dy.t(), x), {}), ((dy, x), dict(accumulate=True)),
                     ((dy, x), dict(out=z(16, 33, d=torch.float32))), ((dy, x), dict(out=z(16, 32, d=torch.float16))),
                     ((dy, x), dict(out=z(32, 16, d=torch.float32).t())), ((dy, x), dict(workspace=z(16, d=torch.uint8))),
                     ((dy.expand(64, 16), x[:1].expand(64, 32)), {})]:
        with pytest.raises(AssertionError):
            yan_b200.fp8_linear_wgrad(*args, **kw)
    for starts, sizes, kw in [(i32(0), i32(1, 2), {}), (i32(0, 1).long(), i32(1, 2), {}), (i32(0, 32), i32(32, 32), dict(out=z(1, 16, 32, d=torch.float32))),
                              (i32(0, 32), i32(32, 32), dict(out=z(1, 16, 32, d=torch.float32).expand(2, 16, 32))),
                              (i32(*range(513)), i32(*range(513)), {})]:
        with pytest.raises(AssertionError):
            yan_b200.k_grouped_fp8_linear_wgrad(dy, x, starts, sizes, **kw)
    f = lambda n=8, d=torch.float32: z(n, d=d)  # noqa: E731
    s8 = yan_b200.adamw_state(f(), 8)
    for p, g, m, v, kw in [([f()], [f(9)], [f()], [f()], {}), ([f()], [f(), f()], [f()], [f()], {}), ([f(d=torch.float16)], [f()], [f()], [f()], {}),
                           ([f(), f(d=torch.bfloat16)], [f(), f()], [f(), f()], [f(), f()], {}), ([f()], [f()], [s8], [f()], {}),
                           ([f()], [f()], [f()], [f(9)], {}), ([f(256)], [f(256)], [s8], [s8], {}), ([z(4, 8, d=torch.float32).t()], [f(32)], [f(32)], [f(32)], {}),
                           ([f()], [f()], [f()], [f()], dict(copies=[f()])), ([f()], [f()], [f()], [f()], dict(grad_scale=torch.ones(1))),
                           ([f()], [f()], [f()], [f()], dict(weight_decay=[0.1, 0.2])), ([f()], [f()], [f()], [f()], dict(step=0))]:
        with pytest.raises((AssertionError, AttributeError, TypeError, ValueError)):
            yan_b200.adamw_step(p, g, m, v, **(dict(lr=1e-3, step=1) | kw))
    logits, ids = z(64, 16, d=torch.float32), z(64, 2, d=torch.int64)
    for args, kw in [((logits.half(), ids), {}), ((logits, ids[:32]), {}), ((logits, ids.float()), {}), ((logits, ids.t().contiguous().t()), {}),
                     ((logits, ids), dict(score="relu")), ((logits, ids), dict(token_mask=z(64, d=torch.uint8))),
                     ((logits, ids), dict(token_mask=z(63, d=torch.bool))), ((logits, ids), dict(cu_seqlens=i32(0, 64).long())),
                     ((logits, ids), dict(cu_seqlens=i32(0))), ((logits, ids), dict(grad=z(64, 16))), ((logits.t(), ids), {}),
                     ((z(64, 1025, d=torch.float32), ids), {}), ((z(200000, 16, d=torch.float32), z(200000, 2, d=torch.int64)), dict(workspace=z(8, d=torch.uint8)))]:
        with pytest.raises(AssertionError):
            yan_b200.moe_balance_loss(*args, **kw)


def test_the_native_front_leaves_unusual_arguments_to_python():
    from yan_b200 import _lib
    f = _lib.fast()
    t = torch.zeros(4, 8, dtype=torch.bfloat16)
    assert f.wgrad(t, t, t, False, None, 148, None, None) == -1 and f.wgrad(t) == -1 and f.wgrad(1, 2, 3, 4, 5, 6, 7, 8) == -1
    args = (0.1, None, None, 1e-3, 0.9, 0.99, 1e-8, 1)
    assert f.adamw([t], [t], [t], [t], *args) == -1 and f.adamw([], [], [], [], *args) == -1 and f.adamw() == -1
    assert f.adamw(t, t, t, t, *args) == -1 and f.adamw([t], [t, t], [t], [t], *args) == -1 and f.adamw([1], [None], ["x"], [t], *args) == -1
    assert f.balance(t, t, None, None, 1.0, 0, 148) == -1 and f.balance() == -1 and f.balance("x", 1, 2, 3, 4, 5, 6) == -1
    with pytest.raises(TypeError):
        f.bind_train(1)
