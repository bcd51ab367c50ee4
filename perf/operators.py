"""The gated delta rule (over sequences and for single tokens), layer norm and counter-based
dropout as cases to time: each kind of case makes the calls that a training loop or a
generation loop makes.

Where `own` is false, `run` computes the same results from elementary torch operations in
32 bits. `exact` restates the definitions at 64 bits, token by token.
"""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
CHUNK = 64


def listed():
    return [
        # Generation, one sequence: a single token through one mixer of 8 heads. Latency counts.
        {"name": "delta step b1 h8 d128", "kind": "step", "type": "bf16", "batch": 1, "qk_heads": 8, "heads": 8,
         "key": 128, "value": 128},
        # Serving, a full batch: the states no longer fit any cache.
        {"name": "delta step b128 h16 d128", "kind": "step", "type": "bf16", "batch": 128, "qk_heads": 8, "heads": 16,
         "key": 128, "value": 128},
        # A prompt of ragged length before generation: outputs and the state that generation goes on from.
        {"name": "delta prompt b1 t777 h8 d128", "kind": "prompt", "type": "bf16", "batch": 1, "length": 777,
         "qk_heads": 8, "heads": 8, "key": 128, "value": 128, "carried": False},
        # Long prompts, two at a time.
        {"name": "delta prompt b2 t16381 h16 d128", "kind": "prompt", "type": "bf16", "batch": 2, "length": 16381,
         "qk_heads": 16, "heads": 16, "key": 128, "value": 128, "carried": False},
        # One mixer of the 8-layer benchmark model's width (1024), batch and length, forward and backward.
        {"name": "delta train b8 t2047 h8 d128", "kind": "train", "type": "bf16", "batch": 8, "length": 2047,
         "qk_heads": 8, "heads": 8, "key": 128, "value": 128, "carried": False},
        # A truncated-backpropagation chunk at batch 1: state carried in, two value heads to a key head.
        {"name": "delta train b1 t2048 h16 d128", "kind": "train", "type": "bf16", "batch": 1, "length": 2048,
         "qk_heads": 8, "heads": 16, "key": 128, "value": 128, "carried": True},
        # The single layer of the fp32 configuration (width 512), heads of 64.
        {"name": "delta train fp32 b4 t1024 d64", "kind": "train", "type": "f32", "batch": 4, "length": 1024,
         "qk_heads": 8, "heads": 8, "key": 64, "value": 64, "carried": False},
        # Norm of the residual stream after a bf16 branch, forward and backward, 8-layer benchmark model.
        {"name": "layer norm b8 t2047 d1024", "kind": "norm", "type": "bf16", "batch": 8, "length": 2047, "width": 1024,
         "branch": True, "drop": 0.0},
        # A few rows of an odd width in fp32: launches and the ragged path.
        {"name": "layer norm fp32 b2 t65 d1001", "kind": "norm", "type": "f32", "batch": 2, "length": 65, "width": 1001,
         "branch": False, "drop": 0.0},
        # The 1 B parameter configuration's rows (batch 4, 4096 bytes, width 2048), branch dropped on its way in.
        {"name": "layer norm drop b4 t4095 d2048", "kind": "norm", "type": "bf16", "batch": 4, "length": 4095,
         "width": 2048, "branch": True, "drop": 0.1},
        # Dropout of a branch and its residual add, forward and backward, 8-layer benchmark model.
        {"name": "dropout b8 t2047 d1024", "kind": "drop", "type": "bf16", "batch": 8, "length": 2047, "width": 1024,
         "branch": True, "drop": 0.1},
        # Dropout by itself over an odd number of values.
        {"name": "dropout fp32 b1 t777 d1001", "kind": "drop", "type": "f32", "batch": 1, "length": 777, "width": 1001,
         "branch": False, "drop": 0.25},
    ]


def _between(rng, low, high, of=1):
    """A multiple of `of` in [low, high], spread over the logarithm."""
    v = math.exp(rng.uniform(math.log(low), math.log(high)))
    return int(min(high, max(low, round(v / of) * of)))


def draw(rng):
    kind = rng.choice(["train", "train", "prompt", "prompt", "step", "step", "norm", "norm", "drop"])
    case = {"kind": kind, "type": rng.choice(["bf16", "bf16", "f32"])}
    if kind in ("norm", "drop"):
        width = _between(rng, 64, 2048, rng.choice([1, 4, 8, 64]))
        rows = _between(rng, 16, min(16380, 16380 * 2048 // width))
        batch = rng.choice([b for b in (1, 2, 3, 4, 8) if b <= rows])
        branch = rng.random() < 0.7
        return {**case, "batch": batch, "length": rows // batch, "width": width, "branch": branch,
                "drop": rng.choice([0.05, 0.1, 0.5]) if kind == "drop" else rng.choice([0.0, 0.1]) if branch else 0.0}
    qk_heads, group = rng.randint(1, 16), rng.choice([1, 1, 1, 2, 4])
    heads = qk_heads * group if qk_heads * group <= 32 else qk_heads
    key = rng.choice([32, 64, 64, 128, 128, _between(rng, 16, 128, 8)])
    value = rng.choice([key, key, _between(rng, 16, 128, 8), 2 * key])
    case.update(qk_heads=qk_heads, heads=heads, key=key, value=value)
    if kind == "step":
        return {**case, "batch": min(_between(rng, 1, 256), max(1, 2 ** 25 // (heads * key * value)))}
    # tokens x heads x state up to what the largest listed case has
    most = (2 ** 31 if kind == "train" else 2 ** 33) // (4 if case["type"] == "f32" else 1)
    length = min(_between(rng, 1, 2300) if kind == "train" else _between(rng, 1, 16400), most // (heads * key * value))
    batch = max(1, min(rng.choice([1, 1, 2, 4, 8]), most // (length * heads * key * value)))
    return {**case, "batch": batch, "length": length, "carried": rng.random() < 0.5}


# ---------------------------------------------------------------- inputs

def _delta_inputs(case, gen, steps):
    """Queries and keys as a mixer has them (activated, so not centred, then normalised), decays
    from slow to fast over the heads, write strengths in (0, 1)."""
    b, h, hk, dk, dv = case["batch"], case["heads"], case["qk_heads"], case["key"], case["value"]
    t = TYPES[case["type"]]

    def normal(*size):
        return torch.randn(*size, generator=gen, device=DEV)

    def unit(x):
        return x / x.square().sum(-1, keepdim=True).add(1e-6).sqrt()

    q, k = (unit(torch.nn.functional.silu(normal(b, *steps, hk, dk))) for _ in range(2))
    rate = torch.logspace(-2.0, 0.5, h, device=DEV)
    g = -rate * torch.nn.functional.softplus(normal(b, *steps, h) - 1.0)
    return {"q": q.to(t), "k": k.to(t), "v": normal(b, *steps, h, dv).to(t), "g": g.to(t),
            "beta": torch.sigmoid(normal(b, *steps, h)).to(t)}


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    kind, t = case["kind"], TYPES[case["type"]]
    s = {"case": dict(case), "seed": seed * 7919 + 13}
    if kind in ("norm", "drop"):
        size = (case["batch"], case["length"], case["width"])
        s["x"] = torch.randn(size, generator=gen, device=DEV).to(t)
        # the stream that the branch x joins, and the gradient that reaches it from later layers
        s["residual"] = torch.randn(size, generator=gen, device=DEV) if case["branch"] else None
        s["dy"] = torch.randn(size, generator=gen, device=DEV).to(t if kind == "norm" or not case["branch"] else torch.float32)
        if kind == "norm":
            s["dres"] = torch.randn(size, generator=gen, device=DEV) if case["branch"] else None
            s["w"] = 1.0 + 0.1 * torch.randn(size[-1], generator=gen, device=DEV)
            s["b"] = 0.1 * torch.randn(size[-1], generator=gen, device=DEV)
        for name in ("x", "residual", "w", "b"):
            if s.get(name) is not None:
                s[name].requires_grad_(True)
        return s
    s.update(_delta_inputs(case, gen, () if kind == "step" else (case["length"],)))
    b, h, dk, dv = case["batch"], case["heads"], case["key"], case["value"]
    s["state"] = None
    if kind == "step" or case["carried"]:
        s["state"] = 0.3 * torch.randn(b, h, dk, dv, generator=gen, device=DEV)
    if kind == "train":
        s["do"] = torch.randn(b, case["length"], h, dv, generator=gen, device=DEV).to(t)
        for name in ("q", "k", "v", "g", "beta", "state"):
            if s[name] is not None:
                s[name].requires_grad_(True)
    return s


# ---------------------------------------------------------------- plain forms

def _unit_lower_inverse(a):
    """(I + a)^-1 for strictly lower triangular a [..., C, C]: the inverses of diagonal blocks of
    1, 2, 4, ... rows, each from the two halves' before it."""
    c = a.shape[-1]
    x = torch.ones(*a.shape[:-2], c, 1, 1, device=a.device, dtype=a.dtype)
    size = 1
    while size < c:
        n = c // (2 * size)
        blocks = a.unflatten(-1, (n, 2 * size)).unflatten(-3, (n, 2 * size))  # [..., n, 2s, n, 2s]
        low = blocks.diagonal(dim1=-4, dim2=-2).movedim(-1, -3)[..., size:, :size]
        first, second = x[..., 0::2, :, :], x[..., 1::2, :, :]
        left = -(second @ low @ first)
        x = torch.cat([torch.cat([first, torch.zeros_like(first)], -1), torch.cat([left, second], -1)], -2)
        size *= 2
    return x[..., 0, :, :]


def _plain_delta(q, k, v, g, beta, state):
    """Chunks of CHUNK tokens: within a chunk matrix products over all chunks at once, and one
    pass over the chunks for the state, which each chunk hands to the next."""
    b, t, hk, dk = q.shape
    h, dv = v.shape[2:]
    scale, n = dk ** -0.5, -(-t // CHUNK)

    def chunks(x):  # [B, T, H, ...] -> [B, H, n, C, ...], in 32 bits
        x = x.float()
        x = torch.cat([x, x.new_zeros(b, n * CHUNK - t, *x.shape[2:])], 1) if n * CHUNK > t else x
        x = x.transpose(1, 2).unflatten(2, (n, CHUNK))
        return x.repeat_interleave(h // x.shape[1], 1) if x.shape[1] != h else x

    q, k, v, g, beta = (chunks(x) for x in (q, k, v, g, beta))
    total = g.double().cumsum(-1)  # a difference of two sums is what counts: taken in 64 bits
    lower = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=q.device).tril()
    decay = (total.unsqueeze(-1) - total.unsqueeze(-2)).masked_fill(~lower, -math.inf).exp().float()
    solve = _unit_lower_inverse((beta.unsqueeze(-1) * (k @ k.transpose(-1, -2)) * decay).tril(-1))
    near = scale * (q @ k.transpose(-1, -2)) * decay
    since = total.exp().float().unsqueeze(-1)
    until = (total[..., -1:] - total).exp().float().unsqueeze(-1)
    beta = beta.unsqueeze(-1)
    s = q.new_zeros(b, h, dk, dv) if state is None else state
    out = []
    for i in range(n):
        e = since[:, :, i]
        d = solve[:, :, i] @ (beta[:, :, i] * (v[:, :, i] - e * (k[:, :, i] @ s)))
        out.append(scale * e * (q[:, :, i] @ s) + near[:, :, i] @ d)
        s = e[:, :, -1:] * s + (until[:, :, i] * k[:, :, i]).transpose(-1, -2) @ d
    o = torch.stack(out, 2).flatten(2, 3)[:, :, :t].transpose(1, 2)
    return o, s


def _plain_step(q, k, v, g, beta, state):
    h = v.shape[1]
    q, k, v, g, beta = (x.float() for x in (q, k, v, g, beta))
    q, k = (x.repeat_interleave(h // x.shape[1], 1) for x in (q, k))
    s = g.exp()[..., None, None] * state
    d = beta[..., None] * (v - (k.unsqueeze(-2) @ s).squeeze(-2))
    s = s + k.unsqueeze(-1) * d.unsqueeze(-2)
    return q.shape[-1] ** -0.5 * (q.unsqueeze(-2) @ s).squeeze(-2), s


def _plain_words(n, seed, offset):
    """The n first 32-bit words of Philox4x32-10 (Salmon et al. 2011) for a 64-bit key `seed` and
    the counters (i, offset), i = 0, 1, ..., four words each."""
    mask = 0xFFFFFFFF
    i = torch.arange((n + 3) // 4, device=DEV)
    c = [i & mask, i >> 32, torch.full_like(i, offset & mask), torch.full_like(i, offset >> 32)]
    k0, k1 = seed & mask, seed >> 32
    for _ in range(10):
        p0, p1 = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [((p1 >> 32) & mask) ^ c[1] ^ k0, p1 & mask, ((p0 >> 32) & mask) ^ c[3] ^ k1, p0 & mask]
        k0, k1 = (k0 + 0x9E3779B9) & mask, (k1 + 0xBB67AE85) & mask
    return torch.stack(c, -1).flatten()[:n]


def _plain_scales(x, p, seed, offset):
    """What dropout multiplies each value by: 0, or 1 / (1 - p)."""
    keep = _plain_words(x.numel(), seed, offset) >= int(p * 2 ** 32)
    return keep.float().view(x.shape) / (1.0 - p)


def _plain_norm(s, case):
    t = TYPES[case["type"]]
    x = s["x"].detach().float()
    w, bias, dy = s["w"].detach(), s["b"].detach(), s["dy"].float()
    scales = _plain_scales(x, case["drop"], s["seed"], 3) if case["drop"] else None
    if scales is not None:
        x = x * scales
    if case["branch"]:
        x = s["residual"].detach() + x
    mean = x.mean(-1, keepdim=True)
    rstd = ((x - mean).square().mean(-1, keepdim=True) + 1e-5).rsqrt()
    hat = (x - mean) * rstd
    y = (hat * w + bias).to(t)
    gw = dy * w
    dx = rstd * (gw - gw.mean(-1, keepdim=True) - hat * (gw * hat).mean(-1, keepdim=True))
    dw, db = (dy * hat).flatten(0, 1).sum(0), dy.flatten(0, 1).sum(0)
    if not case["branch"]:
        return {"y": y, "dx": dx.to(t), "dw": dw, "db": db}
    dx = dx + s["dres"]
    dbranch = dx if scales is None else dx * scales
    return {"x": x, "y": y, "dresidual": dx, "dx": dbranch.to(t), "dw": dw, "db": db}


def _plain_drop(s, case):
    t = TYPES[case["type"]]
    scales = _plain_scales(s["x"], case["drop"], s["seed"], 5)
    y, dx = s["x"].detach().float() * scales, s["dy"].float() * scales
    if case["branch"]:
        return {"y": s["residual"].detach() + y, "dx": dx.to(t)}
    return {"y": y.to(t), "dx": dx.to(t)}


# ---------------------------------------------------------------- one pass

def run(s):
    case = s["case"]
    kind = case["kind"]
    if kind == "norm":
        if not own:
            return _plain_norm(s, case)
        from gruboros_amd.norm import add_layer_norm, layer_norm

        if not case["branch"]:
            y = layer_norm(s["x"], s["w"], s["b"])
            dx, dw, db = torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["dy"])
            return {"y": y, "dx": dx, "dw": dw, "db": db}
        x, y = add_layer_norm(s["residual"], s["x"], s["w"], s["b"], out_dtype=TYPES[case["type"]],
                              dropout_p=case["drop"], seed=s["seed"], offset=3)
        dr, dx, dw, db = torch.autograd.grad((x, y), (s["residual"], s["x"], s["w"], s["b"]), (s["dres"], s["dy"]))
        return {"x": x, "y": y, "dresidual": dr, "dx": dx, "dw": dw, "db": db}
    if kind == "drop":
        if not own:
            return _plain_drop(s, case)
        from gruboros_amd.dropout import dropout

        y = dropout(s["x"], case["drop"], s["seed"], offset=5, residual=s["residual"])
        return {"y": y, "dx": torch.autograd.grad(y, s["x"], s["dy"])[0]}
    args = [s[name] for name in ("q", "k", "v", "g", "beta")]
    if kind == "step":
        if own:
            from gruboros_amd.delta import gated_delta_step

            return {"o": gated_delta_step(*args, s["state"]), "state": s["state"]}
        o, state = _plain_step(*args, s["state"])
        s["state"].copy_(state)
        return {"o": o.to(args[0].dtype), "state": s["state"]}
    if own:
        from gruboros_amd.delta import gated_delta_rule as rule
    else:
        rule = None
    if kind == "prompt":
        with torch.no_grad():
            if own:
                o, state = rule(*args, initial_state=s["state"], return_state=True)
            else:
                o, state = _plain_delta(*args, s["state"])
        return {"o": o.to(args[0].dtype), "state": state}
    if own:
        o = rule(*args, initial_state=s["state"])
    else:
        o = _plain_delta(*args, s["state"])[0].to(args[0].dtype)
    leaves = args if s["state"] is None else [*args, s["state"]]
    grads = torch.autograd.grad(o, leaves, s["do"])
    return {"o": o, **{"d" + name: x for name, x in zip(("q", "k", "v", "g", "beta", "state"), grads)}}


# ---------------------------------------------------------------- work

def work(case):
    e = 2 if case["type"] == "bf16" else 4
    if case["kind"] in ("norm", "drop"):
        n, r = case["batch"] * case["length"] * case["width"], case["branch"]
        if case["kind"] == "drop":  # x, dy in, y, dx out; the residual in
            return {"bytes": n * ((e + 4 + 4 + 4 + e) if r else 4 * e), "flops": 4 * n}
        # x, dy in, y, dx out, and of a joined branch: the stream, its gradient, their new values
        return {"bytes": n * (4 * e + (16 if r else 0)) + 16 * case["width"], "flops": 20 * n}
    b, h, hk, dk, dv = case["batch"], case["heads"], case["qk_heads"], case["key"], case["value"]
    t = 1 if case["kind"] == "step" else case["length"]
    rows = b * t * (2 * hk * dk + h * dv + 2 * h)  # q, k, v, g, beta
    state = 4 * b * h * dk * dv
    flops = 7 * b * t * h * dk * dv  # decay, k S, the rank-one update, q S
    if case["kind"] == "step":
        return {"bytes": e * (rows + b * h * dv) + 2 * state, "flops": flops}
    if case["kind"] == "prompt":
        return {"bytes": e * (rows + b * t * h * dv) + state * (2 if case["carried"] else 1), "flops": flops}
    return {"bytes": e * (2 * rows + 2 * b * t * h * dv) + state * (2 if case["carried"] else 0), "flops": flops + 14 * b * t * h * dk * dv}


# ---------------------------------------------------------------- the definitions in 64 bits

def _exact_delta(s, case, backward):
    """The rule token by token; with `backward` its gradients, by the adjoint of each step."""
    q, k, v, g, beta = (s[name].detach().double() for name in ("q", "k", "v", "g", "beta"))
    if case["kind"] == "step":
        q, k, v, g, beta = (x.unsqueeze(1) for x in (q, k, v, g, beta))
    b, t, h, dv = v.shape
    hk, dk = q.shape[2:]
    q, k = (x.repeat_interleave(h // hk, 2) for x in (q, k))
    scale = 1.0 / math.sqrt(dk)
    state = s["state"].detach().double().clone() if s["state"] is not None else torch.zeros(b, h, dk, dv, device=DEV, dtype=torch.float64)
    first, kept = state, []
    o = torch.empty_like(v)
    for i in range(t):
        state = state * g[:, i].exp()[..., None, None]
        err = v[:, i] - torch.matmul(k[:, i].unsqueeze(2), state).squeeze(2)
        state = state + torch.matmul((beta[:, i].unsqueeze(-1) * k[:, i]).unsqueeze(-1), err.unsqueeze(2))
        o[:, i] = scale * torch.matmul(q[:, i].unsqueeze(2), state).squeeze(2)
        if backward:
            kept.append(state)
    if not backward:
        return o, state
    do = s["do"].double()
    dq, dk_, dv_, dg, db = (torch.empty_like(x) for x in (q, k, v, g, beta))
    ds = torch.zeros_like(state)
    for i in reversed(range(t)):
        after, before = kept[i], kept[i - 1] if i else first
        ki, a, bi = k[:, i], g[:, i].exp()[..., None, None], beta[:, i].unsqueeze(-1)
        doi = do[:, i]
        ds = ds + scale * q[:, i].unsqueeze(-1) * doi.unsqueeze(2)
        dq[:, i] = scale * torch.matmul(after, doi.unsqueeze(-1)).squeeze(-1)
        decayed = a * before
        err = v[:, i] - torch.matmul(ki.unsqueeze(2), decayed).squeeze(2)
        kds = torch.matmul(ki.unsqueeze(2), ds).squeeze(2)
        db[:, i] = (kds * err).sum(-1)
        derr = bi * kds
        dv_[:, i] = derr
        dk_[:, i] = bi * torch.matmul(ds, err.unsqueeze(-1)).squeeze(-1) - torch.matmul(decayed, derr.unsqueeze(-1)).squeeze(-1)
        ds = ds - ki.unsqueeze(-1) * derr.unsqueeze(2)
        dg[:, i] = (ds * decayed).sum((-1, -2))
        ds = ds * a
    dq, dk_ = (x.unflatten(2, (hk, h // hk)).sum(3) for x in (dq, dk_))
    out = {"o": o, "dq": dq, "dk": dk_, "dv": dv_, "dg": dg, "dbeta": db}
    return {**out, "dstate": ds} if s["state"] is not None else out


def _exact_words(n, seed, offset):
    """Philox4x32-10 on numpy's unsigned 64-bit integers."""
    import numpy as np

    m = np.uint64(0xFFFFFFFF)
    up = np.uint64(32)
    i = np.arange((n + 3) // 4, dtype=np.uint64)
    a, b = i & m, i >> up
    c, d = np.full_like(i, offset & 0xFFFFFFFF), np.full_like(i, offset >> 32)
    key = [seed & 0xFFFFFFFF, seed >> 32]
    for r in range(10):
        x, y = np.uint64(0xD2511F53) * a, np.uint64(0xCD9E8D57) * c
        a, b, c, d = (y >> up) ^ b ^ np.uint64(key[0]), y & m, (x >> up) ^ d ^ np.uint64(key[1]), x & m
        key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
    return torch.from_numpy(np.stack([a, b, c, d], 1).reshape(-1)[:n].astype(np.int64)).to(DEV)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] in ("step", "prompt"):
        o, state = _exact_delta(s, case, False)
        return {"o": o.squeeze(1) if case["kind"] == "step" else o, "state": state}
    if case["kind"] == "train":
        return _exact_delta(s, case, True)
    x, dy = s["x"].detach().double(), s["dy"].double()
    factor = None
    if case["drop"]:
        words = _exact_words(x.numel(), s["seed"], 5 if case["kind"] == "drop" else 3)
        factor = torch.where(words < int(case["drop"] * 2 ** 32), 0.0, 1.0 / (1.0 - case["drop"])).double().view(x.shape)
        x = x * factor
    if case["branch"]:
        x = x + s["residual"].detach().double()
    if case["kind"] == "drop":
        return {"y": x, "dx": dy * factor}
    w, d = s["w"].detach().double(), x.shape[-1]
    centred = x - x.sum(-1, keepdim=True) / d
    sigma = (centred.square().sum(-1, keepdim=True) / d + 1e-5).sqrt()
    hat = centred / sigma
    y = hat * w + s["b"].detach().double()
    up = dy * w
    dx = (up - up.sum(-1, keepdim=True) / d - hat * ((up * hat).sum(-1, keepdim=True) / d)) / sigma
    grads = {"dw": (dy * hat).sum((0, 1)), "db": dy.sum((0, 1))}
    if not case["branch"]:
        return {"y": y, "dx": dx, **grads}
    dx = dx + s["dres"].double()
    return {"x": x, "y": y, "dresidual": dx, "dx": dx if factor is None else dx * factor, **grads}
