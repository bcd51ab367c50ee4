"""The parts of a recurrent token model that learns from a teacher, as cases to time: the gated linear
recurrence (over sequences and for single tokens), the norms around a block with its gate and residual
scale, the scaled embedding of a large vocabulary, and distillation from a teacher's top logits. Each
kind of case makes the calls that a training loop or a generation loop makes.

Where `own` is false, `run` computes the same results from elementary torch operations in 32 bits.
`exact` restates the definitions at 64 bits.
"""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
RATE = 8.0  # the recurrence's constant c
EPS = 1e-6
FIRST = 2.7  # the most frequent token's weight is 1 / FIRST
ALPHA, TEMPERATURE, SCALE = 0.7, 2.0, 11.3


def listed():
    return [
        # Generation, one sequence: a single token through one recurrence of width 1024. Latency counts.
        {"name": "recurrence step b1 d1024", "kind": "step", "type": "bf16", "batch": 1, "width": 1024},
        # One mixer of the 8-layer benchmark model's width (1024), batch and length, forward and backward.
        {"name": "recurrence train b8 t2047 d1024", "kind": "train", "type": "bf16", "batch": 8, "length": 2047,
         "width": 1024, "carried": False, "packed": False},
        # Long rows of packed documents before generation goes on from their last state.
        {"name": "recurrence prompt b2 t16381 d2048", "kind": "prompt", "type": "bf16", "batch": 2, "length": 16381,
         "width": 2048, "carried": True, "packed": True},
        # The single layer of the fp32 configuration (batch 4, 1024 steps, width 512), packed.
        {"name": "recurrence train fp32 b4 t1024 d512", "kind": "train", "type": "f32", "batch": 4, "length": 1024,
         "width": 512, "carried": True, "packed": True},
        # The norms between two blocks of the 8-layer benchmark model, forward and backward.
        {"name": "block norms b8 t2047 d1024", "kind": "norm", "type": "bf16", "batch": 8, "length": 2047, "width": 1024,
         "gate": "silu", "scaled": True, "grad": True},
        # A few rows of an odd width in fp32, no gate: launches and the ragged path.
        {"name": "block norms fp32 b2 t65 d1001", "kind": "norm", "type": "f32", "batch": 2, "length": 65, "width": 1001,
         "gate": "none", "scaled": True, "grad": True},
        # One token each of eight sequences in generation.
        {"name": "block norms serve b8 t1 d2048", "kind": "norm", "type": "bf16", "batch": 8, "length": 1, "width": 2048,
         "gate": "silu", "scaled": True, "grad": False},
        # The token embedding of a student with a vocabulary of 32000, batch and length of the benchmark model.
        {"name": "embedding b8 t2047 v32000 d1024", "kind": "embed", "type": "bf16", "table": "f32", "batch": 8,
         "length": 2047, "vocab": 32000, "width": 1024},
        # Long rows over a large vocabulary kept in bf16.
        {"name": "embedding b8 t8191 v131071 d1024", "kind": "embed", "type": "bf16", "table": "bf16", "batch": 8,
         "length": 8191, "vocab": 131071, "width": 1024},
        # A teacher's eight best of a small vocabulary, fp32.
        {"name": "distill fp32 b1 t65 v1001 k8", "kind": "distill", "type": "f32", "batch": 1, "length": 65,
         "vocab": 1001, "top": 8, "labels": False},
        # A student's training step: 64 logits of the teacher to a token, and the labels.
        {"name": "distill b8 t2047 v32000 k64", "kind": "distill", "type": "bf16", "batch": 8, "length": 2047,
         "vocab": 32000, "top": 64, "labels": True},
        # Rows of a large, odd vocabulary, from the teacher alone.
        {"name": "distill b4 t511 v131071 k32", "kind": "distill", "type": "bf16", "batch": 4, "length": 511,
         "vocab": 131071, "top": 32, "labels": False},
    ]


def _between(rng, low, high, of=1):
    """A multiple of `of` in [low, high], spread over the logarithm."""
    v = math.exp(rng.uniform(math.log(low), math.log(high)))
    return int(min(high, max(low, round(v / of) * of)))


def _rows(rng, most):
    """(batch, length) of up to `most` rows."""
    n = _between(rng, 1, max(1, most))
    batch = rng.choice([b for b in (1, 1, 2, 3, 4, 8) if b <= n])
    return batch, n // batch


def draw(rng):
    kind = rng.choice(["train", "train", "prompt", "step", "norm", "norm", "embed", "embed", "distill", "distill"])
    case = {"kind": kind, "type": rng.choice(["bf16", "bf16", "f32"])}
    e = 2 if case["type"] == "bf16" else 4
    of = rng.choice([1, 4, 8, 64])
    if kind == "step":
        return {**case, "batch": _between(rng, 1, 256), "width": _between(rng, 64, 8192, of)}
    if kind in ("train", "prompt"):
        width = _between(rng, 64, 2560, of)
        # values up to what the largest listed case has
        most = (2 ** 24 if kind == "train" else 2 ** 26) * 2 // e // width
        length = min(_between(rng, 1, 2300) if kind == "train" else _between(rng, 1, 16400), most)
        batch = max(1, min(rng.choice([1, 1, 2, 3, 4, 8]), most // length))
        return {**case, "batch": batch, "length": length, "width": width, "carried": rng.random() < 0.5, "packed": rng.random() < 0.5}
    if kind == "norm":
        width = _between(rng, 64, 8192, of)
        batch, length = _rows(rng, 16380 * 1024 * 2 // e // width)
        return {**case, "batch": batch, "length": length, "width": width, "gate": rng.choice(["silu", "sigmoid", "none"]),
                "scaled": rng.random() < 0.7, "grad": rng.random() < 0.7}
    if kind == "embed":
        width, vocab = _between(rng, 64, 2048, of), _between(rng, 600, 200000)
        vocab = min(vocab, 2 ** 27 // width)
        batch, length = _rows(rng, min(65536, 2 ** 26 // width))
        return {**case, "table": rng.choice(["f32", "f32", "bf16"]), "batch": batch, "length": length, "vocab": vocab, "width": width}
    vocab = _between(rng, 64, 140000, rng.choice([1, 1, 8, 64]))
    batch, length = _rows(rng, min(16384, 2 ** 29 * 2 // e // vocab))
    return {**case, "batch": batch, "length": length, "vocab": vocab, "top": min(vocab, _between(rng, 1, 128)),
            "labels": rng.random() < 0.6}


# ---------------------------------------------------------------- inputs

def _shares(vocab):
    """How often each token comes, from the most frequent on: about as 1 / (rank + 3)."""
    rank = torch.arange(vocab, dtype=torch.float64)
    return torch.log1p(1.0 / (rank + FIRST)) / math.log1p(vocab / FIRST)


def _ranks(u, vocab):
    """The same distribution from uniform numbers."""
    return (FIRST * torch.expm1(u * math.log1p(vocab / FIRST))).long().clamp_max(vocab - 1)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    kind, t = case["kind"], TYPES[case["type"]]

    def normal(*size):
        return torch.randn(*size, generator=gen, device=DEV)

    s = {"case": dict(case)}
    b, n, d = case["batch"], case.get("length", 1), case.get("width")
    if kind in ("step", "train", "prompt"):
        size = (b, d) if kind == "step" else (b, n, d)
        s["x"] = normal(*size).to(t)
        s["input_gate"], s["decay_gate"] = normal(*size).to(t), normal(*size).to(t)
        # a wide open gate forgets at rates from 1 - 0.999 to 1 - 0.9 over the channels
        rate = -torch.log(0.9 + 0.099 * torch.rand(d, generator=gen, device=DEV)) / RATE
        s["decay"] = torch.log(torch.expm1(rate))
        s["state"] = normal(b, d) if kind == "step" or case["carried"] else None
        s["reset"] = torch.rand(b, n, generator=gen, device=DEV) < 1.0 / 500 if case.get("packed") else None
        if kind == "train":
            s["dh"] = normal(*size).to(t)
            leaves = ("x", "input_gate", "decay_gate", "decay", "state")
    elif kind == "norm":
        s["x"], s["branch"] = normal(b, n, d), normal(b, n, d).to(t)
        s["gate"] = normal(b, n, d).to(t) if case["gate"] != "none" else None
        s["w_branch"], s["w"] = 1.0 + 0.1 * normal(d), 1.0 + 0.1 * normal(d)
        s["scale"] = 0.3 + 0.1 * normal(d) if case["scaled"] else None
        if case["grad"]:
            s["dx"], s["dy"] = normal(b, n, d), normal(b, n, d).to(t)
            leaves = ("x", "branch", "w_branch", "w", "gate", "scale")
    elif kind == "embed":
        ranks = _ranks(torch.rand(b * n, generator=gen, device=DEV, dtype=torch.float64), case["vocab"])
        s["ids"] = torch.randperm(case["vocab"], generator=gen, device=DEV)[ranks].view(b, n)
        s["weight"] = normal(case["vocab"], d).mul_(0.02).to(TYPES[case["table"]])
        s["dy"] = normal(b, n, d).to(t)
        leaves = ("weight",)
    else:
        v = case["vocab"]
        s["logits"] = torch.empty(b, n, v, device=DEV, dtype=t)
        s["ids"] = torch.empty(b, n, case["top"], device=DEV, dtype=torch.int64)
        s["top"] = torch.empty(b, n, case["top"], device=DEV)
        rows = s["logits"].view(-1, v)
        step = max(1, 2 ** 26 // v)
        for i in range(0, b * n, step):  # (a teacher that the student follows, by parts)
            z = 2.0 * normal(min(step, b * n - i), v)
            rows[i:i + step] = z.to(t)
            top = (z + normal(*z.shape)).topk(case["top"])
            s["ids"].view(-1, case["top"])[i:i + step] = top.indices
            s["top"].view(-1, case["top"])[i:i + step] = top.values
        # padding at the end of some rows: no teacher and no label
        padded = torch.arange(n, device=DEV) >= n - (torch.rand(b, 1, generator=gen, device=DEV) * 0.1 * n).floor()
        s["ids"].masked_fill_(padded.unsqueeze(-1), -1)
        s["labels"] = None
        if case["labels"]:
            s["labels"] = torch.randint(v, (b, n), generator=gen, device=DEV).masked_fill_(padded, -100)
        leaves = ("logits",)
    if kind in ("train", "embed", "distill") or case.get("grad"):
        s["leaves"] = [name for name in leaves if s[name] is not None]
        for name in s["leaves"]:
            s[name].requires_grad_(True)
    return s



# ---------------------------------------------------------------- plain forms

def _scan(a, v):
    """h_t = a_t h_{t-1} + v_t along dim 1 from h_{-1} = 0, by doubling."""
    step, n = 1, a.shape[1]
    while step < n:
        v = torch.cat([v[:, :step], v[:, step:] + a[:, step:] * v[:, :-step]], 1)
        a = torch.cat([a[:, :step], a[:, step:] * a[:, :-step]], 1)
        step *= 2
    return v


def _plain_terms(s):
    """What a token's step is made of: x, i, r, log a, a, sqrt(1 - a^2), all in 32 bits."""
    x, gi, gr = (s[name].detach().float() for name in ("x", "input_gate", "decay_gate"))
    decay = s["decay"].detach()
    i, r = torch.sigmoid(gi), torch.sigmoid(gr)
    rate = torch.log1p(torch.exp(-decay.abs())) + decay.clamp_min(0.0)  # softplus
    log_a = -RATE * rate * r
    a, m = torch.exp(log_a), torch.sqrt(-torch.expm1(2.0 * log_a))
    return x, i, r, rate, log_a, a, m


def _plain_recurrence(s, case):
    t = TYPES[case["type"]]
    x, i, r, rate, log_a, a, m = _plain_terms(s)
    if case["kind"] == "step":
        h = a * s["state"] + m * i * x
        s["state"].copy_(h)
        return {"h": h.to(t), "state": s["state"]}
    if s["reset"] is not None:
        start = s["reset"].unsqueeze(-1)
        a, m = a.masked_fill(start, 0.0), m.masked_fill(start, 1.0)
    v = m * i * x
    first = None if s["state"] is None else s["state"].detach()
    if first is not None:
        v = torch.cat([v[:, :1] + (a[:, 0] * first).unsqueeze(1), v[:, 1:]], 1)
    h = _scan(a, v)
    if case["kind"] == "prompt":
        return {"h": h.to(t), "state": h[:, -1].clone()}
    dh = s["dh"].float()
    after = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)  # a_{t+1}
    lam = _scan(after.flip(1), dh.flip(1)).flip(1)
    before = torch.cat([torch.zeros_like(h[:, :1]) if first is None else first.unsqueeze(1), h[:, :-1]], 1)
    u = i * x
    w = lam * log_a * (a * before - u * a * a / m)
    ratio = torch.sigmoid(s["decay"].detach()) / rate
    out = {"h": h.to(t), "dx": (lam * m * i).to(t), "dinput_gate": (lam * m * u * (1.0 - i)).to(t),
           "ddecay_gate": (w * (1.0 - r)).to(t), "ddecay": ratio * w.flatten(0, 1).sum(0)}
    if first is not None:
        out["dstate"] = a[:, 0] * lam[:, 0]
    return out


def _plain_norm(s, case):
    t = TYPES[case["type"]]
    x, f = s["x"].detach(), s["branch"].detach().float()
    wf, w = s["w_branch"].detach(), s["w"].detach()
    rf = (f.square().mean(-1, keepdim=True) + EPS).rsqrt()
    hat = f * rf
    if s["gate"] is not None:
        g = s["gate"].detach().float()
        sig = torch.sigmoid(g)
        act = g * sig if case["gate"] == "silu" else sig
    else:
        act = 1.0
    scale = 1.0 if s["scale"] is None else s["scale"].detach()
    xn = x + scale * (act * (hat * wf))
    rx = (xn.square().mean(-1, keepdim=True) + EPS).rsqrt()
    hx = xn * rx
    out = {"x": xn, "y": (hx * w).to(t)}
    if not case["grad"]:
        return out
    dy = s["dy"].float()
    up = dy * w
    dxn = s["dx"] + rx * (up - hx * (up * hx).mean(-1, keepdim=True))
    db = dxn * scale
    dhat = db * act * wf
    out.update(dx=dxn, dbranch=(rf * (dhat - hat * (dhat * hat).mean(-1, keepdim=True))).to(t),
               dw_branch=(db * act * hat).flatten(0, 1).sum(0), dw=(dy * hx).flatten(0, 1).sum(0))
    if s["gate"] is not None:
        slope = sig * (1.0 + g * (1.0 - sig)) if case["gate"] == "silu" else sig * (1.0 - sig)
        out["dgate"] = (db * hat * wf * slope).to(t)
    if s["scale"] is not None:
        out["dscale"] = (dxn * act * hat * wf).flatten(0, 1).sum(0)
    return out


def _plain_embed(s, case):
    w, ids = s["weight"].detach(), s["ids"].flatten()
    y = (SCALE * w[ids].float()).to(TYPES[case["type"]]).view(*s["ids"].shape, -1)
    dw = torch.zeros(w.shape, device=DEV).index_add_(0, ids, SCALE * s["dy"].float().flatten(0, 1))
    return {"y": y, "dweight": dw.to(w.dtype)}


def _plain_distill(s, case):
    z = s["logits"].detach().float().flatten(0, 1)
    ids, top = s["ids"].flatten(0, 1), s["top"].flatten(0, 1) / TEMPERATURE
    live = ids >= 0
    count = live.any(-1).sum()
    e = torch.exp(top - top.max(-1, keepdim=True).values) * live
    p = e / e.sum(-1, keepdim=True).clamp_min(1e-30)
    high = z.max(-1, keepdim=True).values
    soft = torch.exp((z - high) / TEMPERATURE)
    total = soft.sum(-1, keepdim=True)
    at = ids.clamp_min(0)
    log_q = (z.gather(-1, at) - high) / TEMPERATURE - torch.log(total)
    each = (p * (torch.log(p.clamp_min(1e-30)) - log_q)).sum(-1)
    part = TEMPERATURE ** 2 * each.sum() / count
    # without labels the teacher's part is the whole loss
    share = 1.0 if s["labels"] is None else ALPHA
    loss = share * part
    dz = (soft / total * live.any(-1, keepdim=True)).scatter_add_(-1, at, -p)
    dz = dz * (share * TEMPERATURE / count)
    if s["labels"] is not None:
        labels = s["labels"].flatten()
        kept = labels >= 0
        at, counted = labels.clamp_min(0).unsqueeze(-1), kept.sum()
        hard = torch.exp(z - high)
        total = hard.sum(-1, keepdim=True)
        ce = torch.log(total) + high - z.gather(-1, at)
        loss = loss + (1.0 - ALPHA) * (ce.squeeze(-1) * kept).sum() / counted
        dz = dz + (hard / total).scatter_add_(-1, at, -torch.ones_like(total)) * (kept.unsqueeze(-1) * ((1.0 - ALPHA) / counted))
    return {"loss": loss, "dlogits": dz.to(TYPES[case["type"]]).view(s["logits"].shape)}


# ---------------------------------------------------------------- one pass

def run(s):
    case = s["case"]
    kind = case["kind"]
    if not own:
        return {"norm": _plain_norm, "embed": _plain_embed, "distill": _plain_distill}.get(kind, _plain_recurrence)(s, case)
    if kind == "norm":
        from gruboros_amd.norm import add_gated_rms_norm

        activation = case["gate"] if s["gate"] is not None else "silu"
        x, y = add_gated_rms_norm(s["x"], s["branch"], s["w_branch"], s["w"], gate=s["gate"], activation=activation,
                                  scale=s["scale"], out_dtype=TYPES[case["type"]], eps=EPS)
        if not case["grad"]:
            return {"x": x, "y": y}
        grads = torch.autograd.grad((x, y), [s[name] for name in s["leaves"]], (s["dx"], s["dy"]))
        return {"x": x, "y": y, **{"d" + name: g for name, g in zip(s["leaves"], grads)}}
    if kind == "embed":
        from gruboros_amd.embed import scaled_embedding

        y = scaled_embedding(s["ids"], s["weight"], SCALE, out_dtype=TYPES[case["type"]])
        return {"y": y, "dweight": torch.autograd.grad(y, s["weight"], s["dy"])[0]}
    if kind == "distill":
        from gruboros_amd.loss import distillation_loss

        loss = distillation_loss(s["logits"], s["ids"], s["top"], s["labels"], temperature=TEMPERATURE,
                                 alpha=1.0 if s["labels"] is None else ALPHA)
        return {"loss": loss, "dlogits": torch.autograd.grad(loss, s["logits"])[0]}
    from gruboros_amd.recurrence import gated_recurrence, gated_recurrence_step

    args = [s[name] for name in ("x", "input_gate", "decay_gate", "decay")]
    if kind == "step":
        return {"h": gated_recurrence_step(*args, s["state"]), "state": s["state"]}
    if kind == "prompt":
        h, state = gated_recurrence(*args, initial_state=s["state"], reset=s["reset"], return_state=True)
        return {"h": h, "state": state}
    h = gated_recurrence(*args, initial_state=s["state"], reset=s["reset"])
    grads = torch.autograd.grad(h, [s[name] for name in s["leaves"]], s["dh"])
    return {"h": h, **{"d" + name: g for name, g in zip(s["leaves"], grads)}}


# ---------------------------------------------------------------- work

def work(case):
    e = 2 if case["type"] == "bf16" else 4
    kind, rows, d = case["kind"], case["batch"] * case.get("length", 1), case.get("width")
    if kind == "distill":
        n = rows * case["vocab"]
        return {"bytes": 2 * n * e + rows * (12 * case["top"] + 8 * case["labels"]), "flops": 12 * n}
    n = rows * d
    if kind == "embed":
        # the rows of the table that come at all
        seen = float(-torch.expm1(rows * torch.log1p(-_shares(case["vocab"]))).sum())
        table = 2 if case["table"] == "bf16" else 4
        return {"bytes": int(8 * rows + seen * d * table + 2 * n * e + case["vocab"] * d * table), "flops": 3 * n}
    if kind == "norm":
        gated = case["gate"] != "none"
        once = 8 + e * (2 + gated)  # x, the branch, the gate in; x', y out
        back = 4 + e + 4 + e * (1 + gated)  # their gradients in; those of the inputs out
        return {"bytes": n * (once + (back if case["grad"] else 0)) + 12 * d, "flops": n * (40 if case["grad"] else 15)}
    marks = rows if case.get("packed") else 0
    state = 4 * case["batch"] * d
    if kind == "step":
        return {"bytes": 4 * n * e + 2 * state + 4 * d, "flops": 20 * n}
    if kind == "prompt":
        return {"bytes": 4 * n * e + state * (1 + case["carried"]) + 4 * d + marks, "flops": 20 * n}
    return {"bytes": 8 * n * e + 2 * state * case["carried"] + 8 * d + marks, "flops": 60 * n}


# ---------------------------------------------------------------- the definitions in 64 bits

def _exact_recurrence(s, case):
    """Token by token, and the adjoint of each step."""
    one = case["kind"] == "step"
    x, gi, gr = ((s[name].detach().double().unsqueeze(1) if one else s[name].detach().double())
                 for name in ("x", "input_gate", "decay_gate"))
    decay = s["decay"].detach().double()
    b, n, d = x.shape
    c = RATE * torch.log1p(decay.exp())
    i, r = 1.0 / (1.0 + (-gi).exp()), 1.0 / (1.0 + (-gr).exp())
    la = -c * r
    a, m = la.exp(), (-torch.expm1(2.0 * la)).sqrt()
    start = torch.zeros(b, n, 1, dtype=torch.bool, device=DEV)
    if s["reset"] is not None:
        start = s["reset"].unsqueeze(-1)
        a, m = torch.where(start, 0.0, a), torch.where(start, 1.0, m)
    h0 = torch.zeros(b, d, dtype=torch.float64, device=DEV) if s["state"] is None else s["state"].detach().double()
    h = torch.empty_like(x)
    v, cur = m * i * x, h0
    for t in range(n):
        cur = torch.addcmul(v[:, t], a[:, t], cur)
        h[:, t] = cur
    if one:
        return {"h": h[:, 0], "state": cur}
    if case["kind"] == "prompt":
        return {"h": h, "state": cur}
    lam, cur = torch.empty_like(x), torch.zeros_like(h0)
    dh = s["dh"].double()
    for t in reversed(range(n)):
        cur = dh[:, t] + cur
        lam[:, t] = cur
        cur = a[:, t] * cur
    before = torch.cat([h0.unsqueeze(1), h[:, :-1]], 1)
    # through a, and through sqrt(1 - a^2) by a; no path at the start of a sequence, where a is 0 whatever the gate
    dla = torch.where(start, 0.0, lam * (before - i * x * a / m) * a)
    out = {"h": h, "dx": lam * m * i, "dinput_gate": lam * m * x * i * (1.0 - i), "ddecay_gate": -c * dla * r * (1.0 - r),
           "ddecay": (dla * -RATE * r).sum((0, 1)) / (1.0 + (-decay).exp())}
    return {**out, "dstate": cur} if s["state"] is not None else out


def _exact_norm(s, case):
    def at64(name):
        return None if s[name] is None else s[name].detach().double().requires_grad_(True)

    x, f, wf, w, g, scale = (at64(name) for name in ("x", "branch", "w_branch", "w", "gate", "scale"))
    d = x.shape[-1]
    b = f / ((f * f).sum(-1, keepdim=True) / d + EPS).sqrt() * wf
    if g is not None:
        b = b * (g if case["gate"] == "silu" else 1.0) / (1.0 + (-g).exp())
    xn = x + (b if scale is None else scale * b)
    y = xn / ((xn * xn).sum(-1, keepdim=True) / d + EPS).sqrt() * w
    out = {"x": xn.detach(), "y": y.detach()}
    if case["grad"]:
        leaves = {"x": x, "branch": f, "w_branch": wf, "w": w, "gate": g, "scale": scale}
        leaves = {k: t for k, t in leaves.items() if t is not None}
        grads = torch.autograd.grad((xn, y), list(leaves.values()), (s["dx"].double(), s["dy"].double()))
        out.update({"d" + k: t for k, t in zip(leaves, grads)})
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] in ("step", "train", "prompt"):
        return _exact_recurrence(s, case)
    if case["kind"] == "norm":
        return _exact_norm(s, case)
    if case["kind"] == "embed":
        ids = s["ids"].flatten()
        order = ids.argsort(stable=True)
        seen, counts = ids[order].unique_consecutive(return_counts=True)
        dw = torch.zeros(case["vocab"], case["width"], dtype=torch.float64, device=DEV)
        for at in range(0, case["width"], 256):  # a token's rows are one run of the sorted ones
            rows = s["dy"].flatten(0, 1)[:, at:at + 256].double()[order]
            dw[seen, at:at + 256] = torch.segment_reduce(rows, "sum", lengths=counts, axis=0) * SCALE
        return {"y": torch.nn.functional.embedding(s["ids"], s["weight"].detach().double()) * SCALE, "dweight": dw}
    t, share = TEMPERATURE, 1.0 if s["labels"] is None else ALPHA
    ids, tops = s["ids"].flatten(0, 1), s["top"].flatten(0, 1).double()
    labels = None if s["labels"] is None else s["labels"].flatten()
    taught = int((ids[:, 0] >= 0).sum())
    told = 0 if labels is None else int((labels >= 0).sum())
    rows = s["logits"].detach().flatten(0, 1)
    loss = torch.zeros((), dtype=torch.float64, device=DEV)
    grad = torch.zeros(rows.shape, dtype=torch.float64, device=DEV)
    step = max(1, 2 ** 26 // case["vocab"])
    for i in range(0, rows.shape[0], step):
        z = rows[i:i + step].double()
        part = slice(i, i + z.shape[0])
        on = torch.nonzero(ids[part, 0] >= 0).flatten()
        z_on, id_on = z[on], ids[part][on]
        p = torch.softmax(tops[part][on] / t, -1)
        q = torch.log_softmax(z_on / t, -1)
        loss += share * t * t / taught * (torch.special.xlogy(p, p) - p * q.gather(-1, id_on)).sum()
        grad[i + on] = share * t / taught * (q.exp() - torch.zeros_like(q).scatter_(-1, id_on, p))
        if labels is not None:
            on = torch.nonzero(labels[part] >= 0).flatten()
            at = labels[part][on]
            q = torch.log_softmax(z[on], -1)
            loss -= (1.0 - share) / told * q.gather(-1, at.unsqueeze(-1)).sum()
            q = q.exp()
            q[torch.arange(len(on), device=DEV), at] -= 1.0
            grad[i + on] += (1.0 - share) / told * q
    return {"loss": loss, "dlogits": grad.view(s["logits"].shape)}
