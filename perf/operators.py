"""Cases of the dropout and group-norm operators: inputs, plain forms and 64-bit results.

Dropout draws its mask from a counter-based generator and never stores it: Philox-4x32
with 7 rounds, key = (seed low, seed high), counter = (block low, block high, step, half).
Draw m takes halfword m % 8 (low half of a word first) of block m // 8: its high 16 bits
come from half 0, its low 16 bits from half 1. Element i uses draw i // share, is kept
when the 32-bit draw is >= rint(p 2^32), and is then scaled by 1 / (1 - p).

Group norm works on channels-last tensors [N, ..., C]: mean and biased variance over the
pixels and the C / groups channels of a group, scale, shift, activation, then dropout.
"""
import functools
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ROUNDS = 7
LOW = 0xFFFFFFFF


def listed():
    return [
        # the opacities of a small splat model: latency alone
        {"name": "dropout_opacities_f32", "op": "dropout", "dir": "fwd", "rows": 4096, "cols": 1, "share": 1,
         "type": "f32", "residual": False, "p": 0.1},
        # whole splats dropped from a training step: one draw for the 48 SH coefficients of each of a million splats
        {"name": "dropout_splat_rows_f32", "op": "dropout", "dir": "fwd", "rows": 1_000_000, "cols": 48, "share": 48,
         "type": "f32", "residual": False, "p": 0.2},
        # a residual block's output over a half-resolution frame of 64 features
        {"name": "dropout_residual_bf16", "op": "dropout", "dir": "fwd", "rows": 540 * 960, "cols": 64, "share": 1,
         "type": "bf16", "residual": True, "p": 0.1},
        # the gradient through dropout on an odd crop
        {"name": "dropout_backward_odd_f16", "op": "dropout", "dir": "bwd", "rows": 3 * 271 * 479, "cols": 37,
         "share": 1, "type": "f16", "residual": False, "p": 0.35},
        # one small feature tile while editing: latency alone
        {"name": "norm_tile_f32", "op": "norm", "dir": "fwd", "n": 1, "h": 16, "w": 16, "c": 32, "groups": 8,
         "type": "f32", "params": "f32", "act": "silu", "p": 0.0},
        # a training batch of feature maps
        {"name": "norm_batch_bf16", "op": "norm", "dir": "fwd", "n": 8, "h": 64, "w": 64, "c": 256, "groups": 32,
         "type": "bf16", "params": "f32", "act": "silu", "p": 0.0},
        # a full frame of 64 features, one sample: larger than the L2 cache
        {"name": "norm_frame_bf16", "op": "norm", "dir": "fwd", "n": 1, "h": 1080, "w": 1920, "c": 64, "groups": 16,
         "type": "bf16", "params": "f32", "act": "silu", "p": 0.0},
        # one pooled feature vector for each of many views: a group is one short run of channels
        {"name": "norm_vectors_f16", "op": "norm", "dir": "fwd", "n": 2048, "h": 1, "w": 1, "c": 512, "groups": 32,
         "type": "f16", "params": "same", "act": "silu", "p": 0.0},
        # the gradient for the training batch
        {"name": "norm_backward_batch_bf16", "op": "norm", "dir": "bwd", "n": 8, "h": 64, "w": 64, "c": 256,
         "groups": 32, "type": "bf16", "params": "f32", "act": "silu", "p": 0.0},
        # the gradient of odd crops, channels that fill no vector
        {"name": "norm_backward_odd_f32", "op": "norm", "dir": "bwd", "n": 2, "h": 101, "w": 77, "c": 90, "groups": 6,
         "type": "f32", "params": "f32", "act": "gelu_tanh", "p": 0.0},
        # the gradient of a half-resolution frame of 128 features
        {"name": "norm_backward_frame_bf16", "op": "norm", "dir": "bwd", "n": 1, "h": 540, "w": 960, "c": 128,
         "groups": 32, "type": "bf16", "params": "same", "act": "silu", "p": 0.0},
        # normalise, activate and drop, forward and backward of one training step
        {"name": "norm_dropout_step_bf16", "op": "norm", "dir": "both", "n": 4, "h": 128, "w": 128, "c": 128,
         "groups": 32, "type": "bf16", "params": "f32", "act": "silu", "p": 0.1},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["f32", "bf16", "f16"])
    p = round(rng.uniform(0.02, 0.6), 3)
    if rng.random() < 0.4:
        cols = _log(rng, 1, 700)
        rows = max(1, _log(rng, 2000, 30_000_000) // cols)
        return {"op": "dropout", "dir": rng.choice(["fwd", "bwd"]), "rows": rows, "cols": cols,
                "share": rng.choice([1, 1, cols]), "type": kind, "residual": rng.random() < 0.5, "p": p}
    groups = rng.choice([1, 2, 4, 5, 8, 16, 32])
    c = groups * _log(rng, 1, max(2, 1024 // groups))
    n = _log(rng, 1, 64)
    pixels = max(1, _log(rng, 4000, 30_000_000) // (n * c))
    h = max(1, int(math.sqrt(pixels) * rng.uniform(0.5, 1.5)))
    w = max(1, pixels // h)
    return {"op": "norm", "dir": rng.choice(["fwd", "bwd", "both"]), "n": n, "h": h, "w": w, "c": c, "groups": groups,
            "type": kind, "params": rng.choice(["f32", "same"]), "act": rng.choice(["none", "silu", "gelu_tanh"]),
            "p": rng.choice([0.0, p])}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[case["type"]]
    normal = lambda *shape: torch.randn(shape, generator=gen, device="cuda")  # noqa: E731
    s = {"case": case, "seed": 1234567 + 7919 * seed, "step": 3 + seed % 1000}
    if case["op"] == "dropout":
        s["x"] = normal(case["rows"], case["cols"]).to(t)
        s["residual"] = normal(case["rows"], case["cols"]).to(t) if case["residual"] else None
        return s
    n, c, g = case["n"], case["c"], case["groups"]
    shape = (n, case["h"], case["w"], c)
    pt = t if case["params"] == "same" else torch.float32
    # features have a mean and a spread of their own for each channel and sample
    x = normal(*shape) * (0.5 + torch.rand((n, 1, 1, c), generator=gen, device="cuda")) + 0.7 * normal(n, 1, 1, c)
    s["x"] = x.to(t)
    s["weight"] = (1.0 + 0.2 * normal(c)).to(pt)
    s["bias"] = (0.3 * normal(c)).to(pt)
    s["v"] = normal(*shape).to(t) if case["dir"] != "fwd" else None
    if case["dir"] == "bwd":  # the forward pass left these
        xg = s["x"].double().reshape(n, -1, g, c // g)
        mean = xg.mean((1, 3))
        var = (xg - mean[:, None, :, None]).square().mean((1, 3))
        s["mean"], s["rstd"] = mean.float(), (var + 1e-5).rsqrt().float()
    return s


# ---- the plain forms -------------------------------------------------------------------


def _mul(a, m):
    prod = a * m  # the low 64 bits, as two's complement
    return (prod >> 32) & LOW, prod & LOW


def _round(ck, _):
    (c0, c1, c2, c3), (k0, k1) = ck
    h0, l0 = _mul(c0, 0xD2511F53)
    h1, l1 = _mul(c2, 0xCD9E8D57)
    return (h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0), ((k0 + 0x9E3779B9) & LOW, (k1 + 0xBB67AE85) & LOW)


def _halves(blocks, seed, step, half):
    """[blocks, 8] halfwords of the generator."""
    q = torch.arange(blocks, device="cuda", dtype=torch.int64)
    zero = torch.zeros_like(q)
    start = ((q & LOW, q >> 32, zero + (step & LOW), zero + half), (seed & LOW, (seed >> 32) & LOW))
    (w0, w1, w2, w3), _ = functools.reduce(_round, range(ROUNDS), start)
    words = torch.stack((w0, w1, w2, w3), 1)
    return torch.stack((words & 0xFFFF, words >> 16), 2).reshape(blocks, 8)


def _kept(count, share, p, seed, step):
    """Which of `count` elements stay."""
    draws = -(-count // share)
    blocks = -(-draws // 8)
    u = (_halves(blocks, seed, step, 0) << 16) | _halves(blocks, seed, step, 1)
    keep = u.reshape(-1)[:draws] >= round(p * 2.0**32)
    if share > 1:
        keep = keep[:, None].expand(draws, share).reshape(-1)[:count]
    return keep


def _drop(x, case, s):
    keep = _kept(x.numel(), case.get("share", 1), case["p"], s["seed"], s["step"]).reshape(x.shape)
    return torch.where(keep, x * (1.0 / (1.0 - case["p"])), torch.zeros_like(x))


def _gate(z, act):
    """act(z) = z * gate(z); the gate and its derivative."""
    if act == "none":
        return torch.ones_like(z), torch.zeros_like(z)
    if act == "silu":
        w, dw = z, 1.0
    else:
        a, b = 2.0 * math.sqrt(2.0 / math.pi), 0.044715
        w, dw = a * (z + b * z * z * z), a * (1.0 + 3.0 * b * z * z)
    g = 1.0 / (1.0 + (-w).exp())
    return g, g * (1.0 - g) * dw


def _plain_dropout(s):
    case = s["case"]
    y = _drop(s["x"].float(), case, s)
    if case["dir"] == "bwd" and s["residual"] is not None:
        return {"v_x": y.to(s["x"].dtype), "v_residual": s["x"]}
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return {"out": y.to(s["x"].dtype)}


def _plain_forward(s):
    case, x = s["case"], s["x"]
    n, c, g = case["n"], case["c"], case["groups"]
    xg = x.float().reshape(n, -1, g, c // g)
    mean = xg.mean((1, 3))
    off = xg - mean[:, None, :, None]
    rstd = 1.0 / (off.square().mean((1, 3)) + 1e-5).sqrt()
    z = (off * rstd[:, None, :, None]).reshape(x.shape) * s["weight"].float() + s["bias"].float()
    y = z * _gate(z, case["act"])[0]
    if case["p"] > 0:
        y = _drop(y, case, s)
    return y.to(x.dtype), mean, rstd


def _plain_backward(s, mean, rstd):
    case, x = s["case"], s["x"]
    n, c, g = case["n"], case["c"], case["groups"]
    xh = ((x.float().reshape(n, -1, g, c // g) - mean[:, None, :, None]) * rstd[:, None, :, None]).reshape(n, -1, c)
    weight, bias = s["weight"].float(), s["bias"].float()
    z = xh * weight + bias
    gate, slope = _gate(z, case["act"])
    v = s["v"].float()
    if case["p"] > 0:
        v = _drop(v, case, s)
    dz = v.reshape(n, -1, c) * (gate + z * slope)
    a, b = dz.sum(1), (dz * xh).sum(1)  # [n, c]
    count = xh.shape[1] * (c // g)
    s1 = (a * weight).reshape(n, g, -1).sum(2) / count
    s2 = (b * weight).reshape(n, g, -1).sum(2) / count
    of = lambda q: q.repeat_interleave(c // g, 1)[:, None, :]  # noqa: E731
    v_x = of(rstd) * (dz * weight - of(s1) - xh * of(s2))
    return (v_x.reshape(x.shape).to(x.dtype), b.sum(0).to(s["weight"].dtype), a.sum(0).to(s["bias"].dtype))


def _named(case, forward, backward):
    out = {}
    if forward is not None:
        out |= {"out": forward[0], "mean": forward[1], "rstd": forward[2]}
    if backward is not None:
        out |= {"v_x": backward[0], "v_weight": backward[1], "v_bias": backward[2]}
    return out


# ---- the framework's operators ---------------------------------------------------------


def _own_dropout(s):
    import brush_b200 as bsx

    case = s["case"]
    cfg = bsx.DropoutConfig(p=case["p"], seed=s["seed"], step=s["step"], share=case["share"])
    if case["dir"] == "fwd":
        return {"out": bsx.dropout_forward(s["x"], cfg, residual=s["residual"])}
    v_x = bsx.dropout_backward(s["x"], cfg)
    if s["residual"] is not None:  # the residual's gradient is the incoming one
        return {"v_x": v_x, "v_residual": s["x"]}
    return {"out": v_x}


def _own_norm(s):
    import brush_b200 as bsx

    case = s["case"]
    drop = bsx.DropoutConfig(p=case["p"], seed=s["seed"], step=s["step"]) if case["p"] > 0 else None
    cfg = bsx.GroupNormConfig(groups=case["groups"], eps=1e-5, activation=case["act"], dropout=drop)
    forward = backward = None
    mean, rstd = s.get("mean"), s.get("rstd")
    if case["dir"] != "bwd":
        forward = bsx.group_norm_forward(s["x"], s["weight"], s["bias"], cfg)
        mean, rstd = forward[1], forward[2]
    if case["dir"] != "fwd":
        backward = bsx.group_norm_backward(s["v"], s["x"], s["weight"], s["bias"], mean, rstd, cfg)
    return _named(case, forward, backward)


def run(state):
    case = state["case"]
    if own:
        return _own_dropout(state) if case["op"] == "dropout" else _own_norm(state)
    if case["op"] == "dropout":
        return _plain_dropout(state)
    forward = backward = None
    mean, rstd = state.get("mean"), state.get("rstd")
    if case["dir"] != "bwd":
        forward = _plain_forward(state)
        mean, rstd = forward[1], forward[2]
    if case["dir"] != "fwd":
        backward = _plain_backward(state, mean, rstd)
    return _named(case, forward, backward)


def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2}[case["type"]]
    if case["op"] == "dropout":
        n = case["rows"] * case["cols"]
        adds = bool(case["residual"]) and case["dir"] == "fwd"
        return {"bytes": n * size * (3 if adds else 2), "flops": n * (2 if adds else 1)}
    n = case["n"] * case["h"] * case["w"] * case["c"]
    psize = size if case["params"] == "same" else 4
    stats = 8 * case["n"] * case["groups"]
    cost = {"none": 0, "silu": 4, "gelu_tanh": 9}[case["act"]] + (1 if case["p"] > 0 else 0)
    forward = (2 * n * size + 2 * case["c"] * psize + stats, n * (8 + cost))
    backward = (3 * n * size + 4 * case["c"] * psize + stats, n * (16 + 2 * cost))
    parts = {"fwd": [forward], "bwd": [backward], "both": [forward, backward]}[case["dir"]]
    return {"bytes": sum(b for b, _ in parts), "flops": sum(f for _, f in parts)}


# ---- the definitions in 64 bits --------------------------------------------------------


def _wide(a, m):
    """High and low 32 bits of a 32 x 32 bit product, from 16-bit limbs."""
    a0, a1, m0, m1 = a % 65536, a // 65536, m % 65536, m // 65536
    mid = a1 * m0 + (a0 * m0) // 65536
    mid2 = a0 * m1 + mid % 65536
    return a1 * m1 + mid // 65536 + mid2 // 65536, (mid2 % 65536) * 65536 + (a0 * m0) % 65536


def _exact_mask(count, share, p, seed, step):
    index = torch.arange(-(-count // share), device="cuda")
    block, lane = torch.arange((index.numel() + 7) // 8, device="cuda"), index % 8
    value = torch.zeros_like(index)
    for half in (0, 1):
        x = [block % 2**32, block // 2**32, torch.full_like(block, step % 2**32), torch.full_like(block, half)]
        for r in range(ROUNDS):
            key0 = (seed % 2**32 + r * 0x9E3779B9) % 2**32
            key1 = (seed // 2**32 % 2**32 + r * 0xBB67AE85) % 2**32
            (ha, la), (hb, lb) = _wide(x[0], 0xD2511F53), _wide(x[2], 0xCD9E8D57)
            x = [hb ^ x[1] ^ key0, lb, ha ^ x[3] ^ key1, la]
        word = torch.stack(x)[lane // 2, index // 8]
        value = value * 65536 + torch.where(lane % 2 == 0, word % 65536, word // 65536)
    return (value >= round(p * 2**32)).repeat_interleave(share)[:count]


def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].double()

    def dropped(v):
        if case["p"] == 0:
            return v
        keep = _exact_mask(v.numel(), case.get("share", 1), case["p"], s["seed"], s["step"]).reshape(v.shape)
        return v.masked_fill(~keep, 0.0) / (1.0 - case["p"])

    if case["op"] == "dropout":
        y = dropped(x)
        if case["dir"] == "bwd" and s["residual"] is not None:
            return {"v_x": y, "v_residual": x}
        return {"out": y if s["residual"] is None else y + s["residual"].double()}
    n, c, g = case["n"], case["c"], case["groups"]
    per = c // g
    x = x.reshape(n, -1, c)
    groups = x.reshape(n, -1, g, per).transpose(1, 2).reshape(n, g, -1)
    mean, rstd = groups.mean(2), (groups.var(2, correction=0) + 1e-5) ** -0.5
    if case["dir"] == "bwd":
        mean, rstd = s["mean"].double(), s["rstd"].double()
    of = lambda q: q.repeat_interleave(per, 1).unsqueeze(1)  # noqa: E731
    gamma, beta = s["weight"].double(), s["bias"].double()
    xh = (x - of(mean)) * of(rstd)
    z = gamma * xh + beta
    if case["act"] == "none":
        y, dact = z, torch.ones_like(z)
    elif case["act"] == "silu":
        y = z * torch.sigmoid(z)
        dact = torch.sigmoid(z) * (1.0 + z * torch.sigmoid(-z))
    else:
        k = math.sqrt(2.0 / math.pi)
        t = torch.tanh(k * (z + 0.044715 * z**3))
        y = 0.5 * z * (1.0 + t)
        dact = 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * k * (1.0 + 3 * 0.044715 * z * z)
    forward = backward = None
    if case["dir"] != "bwd":
        forward = (dropped(y).reshape(s["x"].shape), mean, rstd)
    if case["dir"] != "fwd":
        dz = dropped(s["v"].double()).reshape(x.shape) * dact
        to_bias, to_weight = dz.sum(1), (dz * xh).sum(1)
        dxh = dz * gamma
        size = groups.shape[2]
        sums = lambda q: q.reshape(n, -1, g, per).sum((1, 3)) / size  # noqa: E731
        v_x = of(rstd) * (dxh - of(sums(dxh)) - xh * of(sums(dxh * xh)))
        backward = (v_x.reshape(s["x"].shape), to_weight.sum(0), to_bias.sum(0))
    return _named(case, forward, backward)
