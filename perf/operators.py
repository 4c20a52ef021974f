"""The operators that train an FP8 layer, as a training program calls them: the weight gradient of a linear layer (and of a layer of
experts) from 8-bit operands, the AdamW step over many tensors, and the router's balance loss with its gradient.

`run` does one pass: with `own` through this package's entry points, otherwise in elementary torch operations in 32 bits.  `exact`
restates an operator from its definition in 64 bits.

Weight gradient   dW[n, k] (+)= sum over blocks b of 128 tokens of 2^(e_dy[b, n] + e_x[b, k]) * sum over m in b of q_dy[m, n] * q_x[m, k]
                  with e the smallest integer for which amax <= 448 * 2^e over the block of a column, q = e4m3(z / 2^e)
AdamW             m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2;  p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v / (1 - b2^t)) + eps)
                  8-bit states: blocks of 128 elements, m and sqrt(v) as e4m3 codes times a power of two chosen like e above
Balance loss      coef / S * sum over sequences s of E / (k n_s^2) * sum over e of c[s, e] * P[s, e], with n_s the valid tokens of a
                  sequence, c the selections and P the sums of the normalized scores of an expert
"""
import random

import torch

own = False

BETA1, BETA2, EPS, LR, DECAY = 0.9, 0.95, 1e-8, 3e-4, 0.1
COEF = 1e-2


# ---------------------------------------------------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------------------------------------------------

def listed():
    return [
        # a small adapter's gradient, added to what earlier microbatches left: odd sizes, latency counts
        {"name": "wgrad small odd", "op": "wgrad", "tokens": 333, "n": 1030, "k": 517, "groups": 0, "accumulate": True, "out": "fp32"},
        # the projection N=7168 K=2048 of the decode benchmark, as it is trained
        {"name": "wgrad projection", "op": "wgrad", "tokens": 8192, "n": 7168, "k": 2048, "groups": 0, "accumulate": False, "out": "fp32"},
        # the large prefill layer, N=28672 K=8192, as it is trained; the gradient goes to a bf16 buffer
        {"name": "wgrad large layer", "op": "wgrad", "tokens": 8192, "n": 28672, "k": 8192, "groups": 0, "accumulate": False, "out": "bf16"},
        # a layer of 16 experts: rows as the router left them, some experts with none, added to the gradients of earlier microbatches
        {"name": "wgrad experts", "op": "wgrad", "tokens": 16384, "n": 4096, "k": 2048, "groups": 16, "accumulate": True, "out": "fp32",
         "aligned": True, "layout": 3},
        # norms, biases and the router's weights: many small tensors, latency counts
        {"name": "adamw small tensors", "op": "adamw", "bits": 32, "tensors": 48, "total": 120_000, "layout": 1, "param": "fp32",
         "grad": "fp32", "copy": False},
        # the large weights of a dense layer, 32-bit states, master weights with bf16 copies for the next forward pass
        {"name": "adamw layer", "op": "adamw", "bits": 32, "tensors": 12, "total": 120_000_000, "layout": 2, "param": "fp32",
         "grad": "fp32", "copy": True},
        # a layer of experts with 8-bit states: master weights in 32 bits, gradients in bf16
        {"name": "adamw experts 8 bit", "op": "adamw", "bits": 8, "tensors": 64, "total": 200_000_000, "layout": 3, "param": "fp32",
         "grad": "bf16", "copy": True},
        # bf16 weights without a master copy, 8-bit states, hundreds of tensors of odd sizes
        {"name": "adamw bf16 ragged", "op": "adamw", "bits": 8, "tensors": 300, "total": 12_000_000, "layout": 4, "param": "bf16",
         "grad": "bf16", "copy": False},
        # the router of a short microbatch, latency counts
        {"name": "balance short", "op": "balance", "tokens": 64, "experts": 64, "top": 6, "sequences": 1, "score": "softmax",
         "logits": "fp32", "masked": False, "layout": 1},
        # the sequence-wise loss of sigmoid scores over ragged sequences, padding tokens masked
        {"name": "balance sequences", "op": "balance", "tokens": 16384, "experts": 256, "top": 8, "sequences": 5, "score": "sigmoid",
         "logits": "fp32", "masked": True, "layout": 2},
        # bf16 logits, odd numbers of tokens and experts
        {"name": "balance odd", "op": "balance", "tokens": 4093, "experts": 61, "top": 4, "sequences": 1, "score": "softmax",
         "logits": "bf16", "masked": True, "layout": 3},
        # a whole batch at once
        {"name": "balance large", "op": "balance", "tokens": 131072, "experts": 256, "top": 8, "sequences": 1, "score": "softmax",
         "logits": "fp32", "masked": False, "layout": 4},
    ]


def _spread(rng, low, high):
    """A whole number between low and high, spread over the logarithm."""
    return min(high, int(low * (high / low) ** rng.random() + 0.5))


def draw(rng):
    op = rng.choice(("wgrad", "adamw", "balance"))
    if op == "wgrad":
        def side():
            v = _spread(rng, 64, 16384)
            return v if rng.random() < 0.3 else max(128, v // 128 * 128)
        grouped = rng.random() < 0.4
        while True:
            case = {"op": op, "tokens": _spread(rng, 1, 32768), "n": side(), "k": side(), "groups": rng.randint(2, 64) if grouped else 0,
                    "accumulate": rng.random() < 0.5, "out": rng.choice(("fp32", "fp32", "bf16"))}
            if grouped:
                case |= {"aligned": rng.random() < 0.5, "layout": rng.randrange(1 << 20)}
            # what the largest listed case costs, and room for the plain form's padded groups
            area = case["n"] * case["k"] * max(1, case["groups"])
            if case["tokens"] * case["n"] * case["k"] <= 8192 * 28672 * 8192 and area <= 400_000_000 and \
                    (not grouped or case["tokens"] * (case["n"] + case["k"]) * case["groups"] <= 3_000_000_000):
                return case
    if op == "adamw":
        total = _spread(rng, 1000, 200_000_000)
        return {"op": op, "bits": rng.choice((8, 32)), "tensors": _spread(rng, 1, min(600, total // 100)), "total": total,
                "layout": rng.randrange(1 << 20), "param": rng.choice(("fp32", "fp32", "bf16")), "grad": rng.choice(("fp32", "bf16")),
                "copy": False} | ({"copy": True} if rng.random() < 0.4 else {})
    experts = _spread(rng, 4, 512)
    return {"op": op, "tokens": _spread(rng, 1, 65536), "experts": experts, "top": rng.randint(1, min(12, experts)),
            "sequences": _spread(rng, 1, 48), "score": rng.choice(("softmax", "sigmoid")), "logits": rng.choice(("fp32", "bf16")),
            "masked": rng.random() < 0.5, "layout": rng.randrange(1 << 20)}


def _shares(rng, total, parts, skew):
    """`parts` non-negative numbers that add up to `total`, unequal by `skew`."""
    w = [rng.random() ** skew for _ in range(parts)]
    s = [int(total * x / sum(w)) for x in w]
    s[s.index(max(s))] += total - sum(s)
    return s


def _group_rows(case):
    """Sizes and first rows of the groups, and the rows in all."""
    rng = random.Random(case["layout"])
    sizes = _shares(rng, case["tokens"], case["groups"], 1.5)
    if case["groups"] >= 8:  # an expert that no token chose
        i = rng.randrange(case["groups"])
        j = (i + 1) % case["groups"]
        sizes[j], sizes[i] = sizes[j] + sizes[i], 0
    starts, at = [], 0
    for s in sizes:
        starts.append(at)
        at += -(-s // 128) * 128 if case["aligned"] else s
    return sizes, starts, max(at, 1)


def _tensor_sizes(case):
    """Elements of each tensor: most of them in a few, all above zero."""
    rng = random.Random(case["layout"])
    sizes = [s + 1 for s in _shares(rng, case["total"], case["tensors"], 3.0)]
    return [s - s % 256 if s > 1_000_000 else s for s in sizes]  # large weights have even sides


def _sequence_ends(case):
    rng = random.Random(case["layout"])
    ends, at = [0], 0
    for s in _shares(rng, case["tokens"], case["sequences"], 1.0):
        at += s
        ends.append(at)
    return ends


def work(case):
    if case["op"] == "wgrad":
        m, n, k, item = case["tokens"], case["n"], case["k"], 4 if case["out"] == "fp32" else 2
        out = n * k * max(1, case["groups"]) * item
        return {"bytes": 2.0 * m * (n + k) + out * (2 if case["accumulate"] else 1), "flops": 2.0 * m * n * k}
    if case["op"] == "adamw":
        count = sum(_tensor_sizes(case))
        param, grad = 4 if case["param"] == "fp32" else 2, 4 if case["grad"] == "fp32" else 2
        states = 16 if case["bits"] == 32 else 4 + 16 / 128
        return {"bytes": count * (2.0 * param + grad + states + (2 if case["copy"] else 0)), "flops": 16.0 * count}
    t, e, k = case["tokens"], case["experts"], case["top"]
    return {"bytes": 2.0 * t * e * (4 if case["logits"] == "fp32" else 2) + 8.0 * t * k + (t if case["masked"] else 0),
            "flops": 12.0 * t * e}


# ---------------------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    if case["op"] == "wgrad":
        rows = case["tokens"]
        state = {"case": case, "op": "wgrad", "accumulate": case["accumulate"]}
        lead = ()
        if case["groups"]:
            sizes, starts, rows = _group_rows(case)
            state |= {"sizes": torch.tensor(sizes, dtype=torch.int32, device="cuda"),
                      "starts": torch.tensor(starts, dtype=torch.int32, device="cuda"), "longest": max(1, max(sizes))}
            lead = (case["groups"],)
        # activations with 1 % of their channels 20 times as large; gradients of a mean over tokens, uneven from token to token
        x = normal(rows, case["k"])
        x *= torch.where(torch.rand(case["k"], generator=gen, device="cuda") < 0.01, 20.0, 1.0)
        dy = normal(rows, case["n"]) * (1e-3 * torch.exp(normal(rows, 1)))
        state["dy"], state["x"] = dy.to(torch.bfloat16), x.to(torch.bfloat16)
        dtype = torch.float32 if case["out"] == "fp32" else torch.bfloat16
        state["out"] = (normal(*lead, case["n"], case["k"]) * 1e-2).to(dtype) if case["accumulate"] else \
            torch.empty(*lead, case["n"], case["k"], dtype=dtype, device="cuda")
        return state

    if case["op"] == "adamw":
        # every tensor is a piece of one buffer and starts on a multiple of 128 elements, as flattened parameters do; what lies
        # between two of them is zero
        sizes = _tensor_sizes(case)
        first, at = [], 0
        for s in sizes:
            first.append(at)
            at += -(-s // 128) * 128
        sizes_d, first_d = torch.tensor(sizes, device="cuda"), torch.tensor(first, device="cuda")
        place = torch.arange(at, device="cuda")
        owner = torch.searchsorted(first_d, place, right=True) - 1
        inside = place - first_d[owner] < sizes_d[owner]
        del place
        decays = [DECAY if s > 4096 else 0.0 for s in sizes]
        dtype = {"fp32": torch.float32, "bf16": torch.bfloat16}
        spread = torch.exp(normal(len(sizes)))[owner]  # gradients differ in size from tensor to tensor
        m, v = normal(at) * 1e-4 * spread * inside, (normal(at) * 3e-4 * spread * inside).square()
        state = {"case": case, "op": "adamw", "bits": case["bits"], "step": 100, "p": (normal(at) * 0.02 * inside).to(dtype[case["param"]]),
                 "g": (normal(at) * 1e-3 * spread * inside).to(dtype[case["grad"]]), "decays": decays,
                 "decay": torch.tensor(decays, device="cuda")[owner], "grad_scale": torch.full((1,), 0.7, device="cuda"),
                 "copy": torch.zeros(at, dtype=torch.bfloat16, device="cuda") if case["copy"] else None}
        if case["bits"] == 8:
            (state["m"], state["m_scale"]), (state["v"], state["v_scale"]) = _encode(m, False), _encode(torch.sqrt(v), True)
        else:
            state["m"], state["v"] = m, v

        def pieces(flat):
            return [flat[f:f + s] for f, s in zip(first, sizes)]

        def blocks(flat):
            return [flat[f // 128:f // 128 + -(-s // 128)] for f, s in zip(first, sizes)]

        state["lists"] = {"p": pieces(state["p"]), "g": pieces(state["g"]),
                          "m": list(zip(pieces(state["m"]), blocks(state["m_scale"]))) if case["bits"] == 8 else pieces(state["m"]),
                          "v": list(zip(pieces(state["v"]), blocks(state["v_scale"]))) if case["bits"] == 8 else pieces(state["v"]),
                          "copy": pieces(state["copy"]) if case["copy"] else None}
        return state

    t, e = case["tokens"], case["experts"]
    # a router that prefers some experts
    logits = (normal(t, e) * 1.5 + normal(e) * 0.7).to(torch.float32 if case["logits"] == "fp32" else torch.bfloat16)
    ids = torch.topk(logits.float(), case["top"], dim=1).indices
    ends = torch.tensor(_sequence_ends(case), dtype=torch.int32, device="cuda")
    return {"case": case, "op": "balance", "logits": logits, "ids": ids, "score": case["score"], "ends": ends if case["sequences"] > 1 else None,
            "sequences": case["sequences"], "mask": torch.rand(t, generator=gen, device="cuda") < 0.9 if case["masked"] else None}


# ---------------------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------------------

def run(state):
    return {"wgrad": _run_wgrad, "adamw": _run_adamw, "balance": _run_balance}[state["op"]](state)


def _run_wgrad(state):
    if own:
        import yan_b200
        if "sizes" in state:
            return yan_b200.k_grouped_fp8_linear_wgrad(state["dy"], state["x"], state["starts"], state["sizes"], out=state["out"],
                                                       accumulate=state["accumulate"])
        return yan_b200.fp8_linear_wgrad(state["dy"], state["x"], out=state["out"], accumulate=state["accumulate"])
    if "sizes" in state:
        # every group as a batch of its own, filled up with zeros to the longest
        step = torch.arange(-(-state["longest"] // 128) * 128, device="cuda")
        valid = step < state["sizes"][:, None]
        at = torch.where(valid, state["starts"][:, None] + step, 0)
        dy, x = (torch.where(valid[..., None], state[z][at].float(), 0.0) for z in ("dy", "x"))
    else:
        fill = -state["dy"].shape[0] % 128
        dy, x = (torch.nn.functional.pad(state[z].float(), (0, 0, 0, fill))[None] for z in ("dy", "x"))
    grad = torch.matmul(_rounded(dy).transpose(1, 2), _rounded(x)).view(state["out"].shape)
    if state["accumulate"]:
        state["out"].copy_(state["out"].float() + grad)
        return state["out"]
    return grad.to(state["out"].dtype)


def _rounded(z):
    """[G, L, C] fp32 -> the values that its codes and scales stand for; blocks of 128 along L."""
    g, length, c = z.shape
    blocks = z.view(g, length // 128, 128, c)
    bits = blocks.abs().amax(2, keepdim=True).view(torch.int32).to(torch.int64)
    e = ((bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000)).clamp(0, 254) - 127
    power = ((e + 1023) << 52).view(torch.float64)
    codes = (blocks * (1.0 / power).float()).to(torch.float8_e4m3fn)
    return (codes.float() * power.float()).view(g, length, c)


def _encode(x, positive):
    """fp32 [L] -> e4m3 codes and the power of two of each block of 128; `positive`: what is above zero stays above zero."""
    blocks = x.view(-1, 128)
    bits = blocks.abs().amax(1, keepdim=True).view(torch.int32)
    known = bits >= (16 << 23)
    e = (bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000)
    scale = torch.where(known, e << 23, 0).view(torch.float32)
    inverse = torch.where(known, (254 - e) << 23, 0).view(torch.float32)
    codes = (blocks * inverse).to(torch.float8_e4m3fn)
    if positive:
        byte = codes.view(torch.uint8)
        codes = torch.where((byte == 0) & (blocks > 0) & known, 1, byte).view(torch.float8_e4m3fn)
    return codes.view(-1), scale.view(-1)


def _run_adamw(s):
    s["step"] += 1
    b1, b2 = 1.0 - BETA1 ** s["step"], 1.0 - BETA2 ** s["step"]
    if own:
        import yan_b200
        lists = s["lists"]
        yan_b200.adamw_step(lists["p"], lists["g"], lists["m"], lists["v"], lr=LR, beta1=BETA1, beta2=BETA2, eps=EPS,
                            weight_decay=s["decays"], step=s["step"], grad_scale=s["grad_scale"], copies=lists["copy"])
    else:
        g = s["g"].float() * s["grad_scale"]
        if s["bits"] == 8:
            m = (s["m"].float().view(-1, 128) * s["m_scale"][:, None]).view(-1)
            root = (s["v"].float().view(-1, 128) * s["v_scale"][:, None]).view(-1)
            v = root * root
        else:
            m, v = s["m"], s["v"]
        m = m * BETA1 + g * (1.0 - BETA1)
        v = v * BETA2 + (g * g) * (1.0 - BETA2)
        root = torch.sqrt(v)
        p = s["p"].float()
        p = p * (1.0 - s["decay"] * LR) - (m * (LR / b1)) / (root * (1.0 / b2 ** 0.5) + EPS)
        s["p"].copy_(p)
        if s["copy"] is not None:
            s["copy"].copy_(p)
        if s["bits"] == 8:
            for name, value in (("m", _encode(m, False)), ("v", _encode(root, True))):
                s[name].copy_(value[0])
                s[name + "_scale"].copy_(value[1])
        else:
            s["m"].copy_(m)
            s["v"].copy_(v)
    return {n: s[n] for n in ("p", "m", "v", "m_scale", "v_scale", "copy") if s.get(n) is not None}


def _run_balance(s):
    if own:
        import yan_b200
        loss, counts, grad = yan_b200.moe_balance_loss(s["logits"], s["ids"], coef=COEF, score=s["score"], token_mask=s["mask"],
                                                       cu_seqlens=s["ends"])
        return {"loss": loss, "counts": counts, "grad": grad}
    z, ids, count = s["logits"].float(), s["ids"], s["sequences"]
    t, e = z.shape
    place = torch.arange(t, device="cuda", dtype=torch.int32)
    owner = torch.searchsorted(s["ends"][1:], place, right=True) if count > 1 else torch.zeros_like(place, dtype=torch.int64)
    valid = s["mask"] if s["mask"] is not None else torch.ones(t, dtype=torch.bool, device="cuda")
    member = ((owner == torch.arange(count, device="cuda")[:, None]) & valid).float()  # [S, T]
    if s["score"] == "softmax":
        score = torch.exp(z - z.amax(1, keepdim=True))
    else:
        score = 1.0 / (1.0 + torch.exp(-z))
    total = score.sum(1, keepdim=True)
    p = score / total
    picked = (owner[:, None] * e + ids)[valid].view(-1)
    counts = torch.zeros(count * e, dtype=torch.int32, device="cuda").index_add_(0, picked, torch.ones_like(picked, dtype=torch.int32))
    counts = counts.view(count, e)
    n = member.sum(1, keepdim=True)
    weight = torch.where(n > 0, COEF / count * e / (ids.shape[1] * n * n).clamp(min=1.0), 0.0)
    a = weight * counts.float()
    loss = (a * (member @ p)).sum()
    mine = a[owner]
    inner = mine - (mine * p).sum(1, keepdim=True)
    grad = p * inner if s["score"] == "softmax" else score * (1.0 - score) / total * inner
    grad = torch.where(valid[:, None], grad, 0.0).to(s["logits"].dtype)
    return {"loss": loss, "counts": counts, "grad": grad}


# ---------------------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    return {"wgrad": _exact_wgrad, "adamw": _exact_adamw, "balance": _exact_balance}[case["op"]](state)


def _e4m3(x):
    """The nearest e4m3 value, ties to even, of doubles within its range."""
    _, e = torch.frexp(x)
    unit = torch.ldexp(torch.ones_like(x), (e - 4).clamp(min=-9))  # four significant bits; multiples of 2^-9 below 2^-6
    return torch.round(x / unit) * unit


def _block_power(amax):
    """The smallest power of two s with amax <= 448 s, and 1 for an empty block."""
    fraction, e = torch.frexp(amax / 448.0)  # amax / 448 = fraction * 2^e, fraction in [1/2, 1)
    return torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), torch.where(fraction == 0.5, e - 1, e)), 1.0)


def _exact_wgrad(state):
    case = state["case"]
    spans = list(zip(*_group_rows(case)[:2])) if case["groups"] else [(case["tokens"], 0)]
    out = state["out"].double().view(len(spans), case["n"], case["k"]) if state["accumulate"] else \
        torch.zeros(len(spans), case["n"], case["k"], dtype=torch.float64, device="cuda")
    for i, (size, start) in enumerate(spans):
        sides = []
        for z in (state["dy"], state["x"]):
            z = z[start:start + size].double()
            for b in range(0, size, 128):
                s = _block_power(z[b:b + 128].abs().amax(0))
                z[b:b + 128] = _e4m3(z[b:b + 128] / s) * s
            sides.append(z)
        if size:
            out[i].addmm_(sides[0].t(), sides[1])
    return out.view(state["out"].shape)


def _exact_adamw(s):
    t, sizes = s["step"] + 1, s["p"].numel()
    g = s["g"].double() * s["grad_scale"].double()
    m, v = s["m"].double(), s["v"].double()
    if s["bits"] == 8:
        m, v = m * s["m_scale"].double().repeat_interleave(128), (v * s["v_scale"].double().repeat_interleave(128)).square()
    m.mul_(BETA1).add_(g, alpha=1 - BETA1)
    v.mul_(BETA2).addcmul_(g, g, value=1 - BETA2)
    root = v.sqrt()
    p = s["p"].double()
    p = p - LR * s["decay"].double() * p - LR * (m / (1 - BETA1 ** t)) / (root / (1 - BETA2 ** t) ** 0.5 + EPS)
    out = {"p": p} | ({"copy": p} if s["copy"] is not None else {})
    if s["bits"] == 32:
        return out | {"m": m, "v": v}
    for name, x in (("m", m), ("v", root)):
        x = x.view(sizes // 128, 128)
        scale = _block_power(x.abs().amax(1, keepdim=True))
        code = _e4m3(x / scale)
        if name == "v":
            code = torch.where((code == 0) & (x > 0), 2.0 ** -9, code)
        out |= {name: code.view(-1), name + "_scale": torch.where(x.abs().amax(1, keepdim=True) > 0, scale, 0.0).view(-1)}
    return out


def _exact_balance(s):
    z, ids, case = s["logits"].double(), s["ids"], s["case"]
    ends = _sequence_ends(case)
    p = torch.softmax(z, 1)
    score = torch.sigmoid(z)
    if s["score"] == "sigmoid":
        p = score / score.sum(1, keepdim=True)
    loss, grad = torch.zeros((), dtype=torch.float64, device="cuda"), torch.zeros_like(z)
    for start, end in zip(ends, ends[1:]):
        rows = torch.arange(start, end, device="cuda")
        if s["mask"] is not None:
            rows = rows[s["mask"][start:end]]
        n = rows.numel()
        if n == 0:
            continue
        chosen = torch.bincount(ids[rows].view(-1), minlength=case["experts"]).double()
        a = COEF / case["sequences"] * case["experts"] / (case["top"] * n * n) * chosen
        loss = loss + (a * p[rows].sum(0)).sum()
        inner = a - (p[rows] @ a)[:, None]
        if s["score"] == "softmax":
            grad[rows] = p[rows] * inner
        else:
            grad[rows] = score[rows] * (1 - score[rows]) / score[rows].sum(1, keepdim=True) * inner
    return {"loss": loss, "counts": None, "grad": grad}
