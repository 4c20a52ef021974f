"""The training operators restated from their definitions in 64 bits (test infrastructure only; runs on any device)."""
import torch


def e4m3(x):
    """Nearest e4m3 value of doubles within +-448, ties to even."""
    _, e = torch.frexp(x)
    unit = torch.ldexp(torch.ones_like(x), (e - 4).clamp(min=-9))
    return torch.round(x / unit) * unit


def block_power(amax):
    """Smallest power of two s, at least 2^-127, with amax <= 448 s."""
    fraction, e = torch.frexp(amax / 448.0)
    e = torch.where(fraction == 0.5, e - 1, e)
    return torch.ldexp(torch.ones_like(amax), torch.where(amax > 0, e, -127).clamp(min=-127))


def cast_tokens(z):
    """[M, C] -> the values that its codes stand for; one power of two per column and 128 rows.  A block of a column with a value that
    is not finite is NaN."""
    out = torch.empty(z.shape, dtype=torch.float64, device=z.device)
    for b in range(0, z.shape[0], 128):
        block = z[b:b + 128].double()
        amax = block.abs().amax(0)
        bad = ~torch.isfinite(block).all(0)
        s = block_power(torch.where(bad, 0.0, amax))
        out[b:b + 128] = torch.where(bad, float("nan"), e4m3(torch.where(bad, 0.0, block) / s) * s)
    return out


def weight_grad(dy, x):
    """(dW, the same with every product made positive) of the quantized operands."""
    a, b = cast_tokens(dy), cast_tokens(x)
    return a.t() @ b, a.abs().t() @ b.abs()


def encode_state(x, positive):
    """Flat [L] -> (values that the codes stand for, scales): blocks of 128, blocks below 2^-111 are zero.  positive: the codes of what
    is above zero are above zero."""
    blocks = torch.nn.functional.pad(x.double(), (0, -x.numel() % 128)).view(-1, 128)
    finite = torch.isfinite(blocks)
    kept = torch.where(finite, blocks, 0.0)
    amax = kept.abs().amax(1, keepdim=True)
    known = amax >= 2.0 ** -111
    s = block_power(torch.where(known, amax, 0.0))
    code = e4m3(kept / s)
    if positive:
        code = torch.where((code == 0) & (kept > 0), 2.0 ** -9, code)
    value = torch.where(finite, torch.where(known, code * s, 0.0), float("nan"))
    return value.reshape(-1)[:x.numel()], torch.where(known, s, 0.0).view(-1)


def adamw(p, g, m, v, *, lr, beta1, beta2, eps, weight_decay, step, grad_scale=1.0):
    """(p, m, v, sqrt(v)) after one step; v is the second moment itself."""
    p, g, m, v = (t.double() for t in (p, g, m, v))
    g = g * grad_scale
    m = beta1 * m + (1 - beta1) * g
    v = beta2 * v + (1 - beta2) * g * g
    p = p - lr * weight_decay * p - lr * (m / (1 - beta1 ** step)) / ((v / (1 - beta2 ** step)).sqrt() + eps)
    return p, m, v, v.sqrt()


def adamw_states_fp32(g, m, v, *, beta1, beta2, grad_scale=1.0):
    """(m, v, sqrt(v)) by the operator's own sequence of fp32 operations, each rounded by itself (torch does one operation at a time)."""
    g = g.float() * torch.tensor(grad_scale, dtype=torch.float32, device=g.device)
    m = m.float() * beta1 + g * (1 - beta1)
    v = v.float() * beta2 + (g * g) * (1 - beta2)
    return m, v, torch.sqrt(v)


def adamw_param(p, m, v, *, lr, beta1, beta2, eps, weight_decay, step):
    """(new parameter, size of the update) in 64 bits from the new m and v."""
    update = lr * (m.double() / (1 - beta1 ** step)) / ((v.double() / (1 - beta2 ** step)).sqrt() + eps)
    return p.double() * (1 - lr * weight_decay) - update, update.abs()


def balance_loss(z, ids, *, coef=1.0, score="softmax", mask=None, cu_seqlens=None, counts=None):
    """(loss, counts) from logits; `counts` given: those are used (differences of the loss keep them constant)."""
    z = z.double()
    t, e = z.shape
    ends = [0, t] if cu_seqlens is None else cu_seqlens.tolist()
    loss, found = torch.zeros((), dtype=torch.float64, device=z.device), []
    for s, (begin, end) in enumerate(zip(ends, ends[1:])):
        rows = torch.arange(begin, end, device=z.device)
        if mask is not None:
            rows = rows[mask[begin:end]]
        picked = ids[rows].reshape(-1).long()
        picked = picked[(picked >= 0) & (picked < e)]
        c = torch.bincount(picked, minlength=e) if counts is None else counts[s]
        found.append(c)
        if rows.numel() == 0:
            continue
        zr = z[rows]
        if score == "softmax":
            top = zr.amax(1, keepdim=True)
            u = torch.exp(zr - torch.where(top == -float("inf"), 0.0, top))
        else:
            u = torch.sigmoid(zr)
        total = u.sum(1, keepdim=True)
        p = torch.where(total == 0, 0.0, u / total)
        loss = loss + coef / (len(ends) - 1) * e / (ids.shape[1] * rows.numel() ** 2) * (c * p.sum(0)).sum()
    return loss, torch.stack(found).to(torch.int32)
