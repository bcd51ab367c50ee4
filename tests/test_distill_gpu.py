"""Distillation from a teacher's top logits against float64.

Tolerances before any run. A row's sum of V exponentials of one sign: 2^-21 of itself (exp's 2^-23, the
fused argument's half step at |z k + b| <= 64, a thread's 128 terms that add like a root), so each
probability is off by 2e-6 of itself, and a gradient by 2e-6 of the sum of the sizes of its terms
(softmax and teacher); the loss by 2e-6 of a log's size, |log2| <= 64: 1e-5 absolute and 1e-5 of it.
bfloat16: half a step, 2^-8 of the gradient, on top; inputs are exact.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
f32, bf16 = torch.float32, torch.bfloat16


def _reference(z, ids, top, labels, temperature, alpha):
    """(loss, dz, size of dz's terms) in float64; rows that do not count are left out by hand."""
    V = z.shape[-1]
    z, ids, top = z.double().reshape(-1, V), ids.long().reshape(-1, ids.shape[-1]), top.double().reshape(-1, ids.shape[-1])
    dz, size = torch.zeros_like(z), torch.zeros_like(z)
    live = (ids >= 0) & (ids < V) & (top != -float("inf"))
    loss = 0.0
    if alpha > 0 and bool(live.any()):
        rows = live.any(-1).nonzero().flatten()
        w = alpha * temperature / len(rows)
        for r in rows.tolist():
            i, t = ids[r][live[r]], top[r][live[r]]
            p = torch.softmax(t / temperature, 0)
            logq = torch.log_softmax(z[r] / temperature, 0)
            at = logq[i]
            loss += w * temperature * float(torch.where(p > 0, p * (p.log() - at), torch.zeros_like(p)).sum())
            q = logq.exp()
            pr = torch.zeros_like(q).index_add_(0, i, p)
            dz[r] += w * (q - pr)
            size[r] += w * (q + pr)
    if labels is not None and alpha < 1:
        lab = labels.long().reshape(-1)
        rows = ((lab >= 0) & (lab < V)).nonzero().flatten()
        for r in rows.tolist():
            w = (1 - alpha) / len(rows)
            logq = torch.log_softmax(z[r], 0)
            loss -= w * float(logq[lab[r]])
            q = logq.exp()
            dz[r] += w * q
            dz[r, lab[r]] -= w
            size[r] += w * q
            size[r, lab[r]] += w
    return loss, dz, size


def _operands(rows, V, K, dtype, seed=0, masked=True):
    gen = torch.Generator().manual_seed(seed + V + K)
    z = (3.0 * torch.randn(*rows, V, generator=gen)).to(dtype)
    ids = torch.stack([torch.randperm(V, generator=gen)[:K] for _ in range(torch.Size(rows).numel())]).view(*rows, K)
    top = 3.0 * torch.randn(*rows, K, generator=gen)
    labels = torch.randint(0, V, rows, generator=gen)
    if masked:
        drop = torch.rand(*rows, generator=gen)
        ids[drop < 0.3] = -1
        labels[(drop > 0.2) & (drop < 0.5)] = -100
        top[torch.rand(top.shape, generator=gen) < 0.1] = -float("inf")
        ids[torch.rand(ids.shape, generator=gen) < 0.1] = V + 3
    return z, ids, top, labels


def _check(z, ids, top, labels, temperature, alpha, upstream=None):
    from gruboros_amd.loss import distillation_loss

    zg = z.to(DEV).requires_grad_(True)
    loss = distillation_loss(zg, ids.to(DEV), top.to(DEV), None if labels is None else labels.to(DEV), temperature, alpha)
    assert loss.shape == () and loss.dtype == f32
    want, dz, size = _reference(z, ids, top, labels, temperature, alpha)
    big = max(temperature ** 2, 1.0)
    assert abs(float(loss.detach()) - want) <= 1e-5 * (abs(want) + big), (float(loss), want)
    with torch.no_grad():
        assert torch.equal(loss.detach(), distillation_loss(zg, ids.to(DEV), top.to(DEV), None if labels is None else labels.to(DEV), temperature, alpha))
    up = 1.0 if upstream is None else upstream
    (g,) = torch.autograd.grad(loss, zg, None if upstream is None else torch.tensor(up, device=DEV))
    assert g.dtype == z.dtype and g.shape == z.shape
    half = 2.0 ** -8 * (1 if upstream is None else 2) if z.dtype == bf16 else 0.0
    err = (g.double().cpu().reshape(dz.shape) - up * dz).abs()
    lim = abs(up) * (4e-6 * size + half * dz.abs() + 1e-12 + (1e-38 if half else 0))
    assert bool((err <= lim).all()), float((err / lim).max())
    return g


@pytest.mark.parametrize("dtype", [f32, bf16], ids=["f32", "bf16"])
@pytest.mark.parametrize("V,K", [(1, 1), (3, 2), (64, 5), (1001, 8), (2048, 64), (2049, 33), (4100, 300), (8200, 512), (16391, 20), (32768, 64),
                                 (33001, 7), (65537, 9), (131071, 32), (131073, 5), (200003, 16)])
def test_parity(V, K, dtype):
    rows = (2, 6) if V < 9000 else (1, 5)
    ops = _operands(rows, V, K, dtype)
    _check(*ops, 2.0, 0.7)
    _check(*ops[:3], None, 1.0, 1.0)


@pytest.mark.parametrize("dtype", [f32, bf16], ids=["f32", "bf16"])
@pytest.mark.parametrize("V", [2, 6, 7, 8, 9, 13, 14, 15, 16, 17, 23, 31, 513, 514])
def test_rows_begin_anywhere_in_a_vector(V, dtype):
    """Nine rows, each at another distance from a multiple of 16 bytes; few values, of which no vector may be full; strides."""
    ops = _operands((9,), V, 2, dtype)
    _check(*ops, 2.0, 0.7)
    _check(*_operands((3, 4), V, 2, dtype, seed=5), 1.0, 0.4)
    z, ids, top, labels = _operands((3, 4), V, 2, dtype, seed=6)
    _check(torch.cat([z, z[:, :1] * float("nan")], 1)[:, :-1], ids, top, labels, 4.0, 0.5)


@pytest.mark.parametrize("dtype", [f32, bf16], ids=["f32", "bf16"])
@pytest.mark.parametrize("V,K", [(515, 64), (1030, 64), (1030, 65), (2056, 7), (2060, 64), (3070, 64), (4100, 64), (4101, 65), (6143, 1), (6150, 64),
                                 (8191, 64), (8199, 63)])
def test_up_to_64_entries_and_more(V, K, dtype):
    """Rows that one wave, two or more have, at the ends of each."""
    ops = _operands((1, 7), V, K, dtype)
    _check(*ops, 2.0, 0.7)
    _check(*ops, 3.0, 0.3)
    _check(*ops[:3], None, 1.0, 1.0)


@pytest.mark.parametrize("temperature,alpha", [(1.0, 0.5), (0.25, 1.0), (7.0, 0.0), (4.0, 0.9), (1000.0, 0.5)])
def test_shares_and_temperatures(temperature, alpha):
    for dtype in (f32, bf16):
        _check(*_operands((3, 7), 777, 12, dtype), temperature, alpha)
        _check(*_operands((21,), 777, 12, dtype, masked=False), temperature, alpha, upstream=0.3)


def test_many_rows():
    """More rows than workgroups, and than one pass of the count."""
    from gruboros_amd.loss import distillation_loss

    z, ids, top, labels = _operands((5, 4001), 40, 3, f32)
    _check(z, ids, top, labels, 2.0, 0.6)
    a = [t.to(DEV) for t in (z, ids, top, labels)]
    assert torch.equal(distillation_loss(*a, 2.0, 0.6), distillation_loss(a[0], a[1].int(), a[2], a[3].int(), 2.0, 0.6))


@pytest.mark.parametrize("N,V,K,dtype", [(6500, 261, 4, f32), (3300, 71, 70, bf16), (1600, 12001, 9, bf16), (1100, 17003, 5, bf16), (600, 33001, 5, bf16),
                                         (300, 66001, 5, bf16), (300, 131077, 3, bf16)])
def test_several_rows_of_one_workgroup(N, V, K, dtype):
    """Rows that are loaded while the one before is written, with entries, heads and ends of their own."""
    _check(*_operands((N,), V, K, dtype), 2.0, 0.6)


def test_listed_twice_and_labels_among_the_listed():
    z, ids, top, labels = _operands((4, 5), 100, 30, f32, masked=False)
    ids[..., 10:20] = ids[..., :10]
    ids[..., 25] = ids[..., 3]
    labels[0] = ids[0, :, 3]
    labels[1] = ids[1, :, 29]
    _check(z, ids, top, labels, 2.0, 0.5)
    _check(z.to(bf16), torch.zeros_like(ids), top, torch.zeros_like(labels), 3.0, 0.5)


@pytest.mark.parametrize("dtype", [f32, bf16], ids=["f32", "bf16"])
def test_rows_that_do_not_count(dtype):
    """Padding is not read: NaN in it, and in entries that are none, changes nothing; no row at all gives 0."""
    from gruboros_amd.loss import distillation_loss

    z, ids, top, labels = _operands((4, 6), 300, 9, dtype)
    ids[1], labels[1] = -1, -100
    g = _check(z, ids, top, labels, 2.0, 0.5)
    assert bool((g[1] == 0).all())
    spoilt, far = z.clone(), top.clone()
    spoilt[1] = float("nan")
    far[ids < 0] = float("nan")
    far[ids >= 300] = float("inf")
    zs = spoilt.to(DEV).requires_grad_(True)
    rest = (ids.to(DEV), far.to(DEV), labels.to(DEV), 2.0, 0.5)
    loss = distillation_loss(zs, *rest)
    assert torch.equal(loss, distillation_loss(z.to(DEV), ids.to(DEV), top.to(DEV), labels.to(DEV), 2.0, 0.5))
    assert torch.equal(torch.autograd.grad(loss, zs)[0], g)
    for i, lab, alpha in ((torch.full_like(ids, -1), torch.full_like(labels, -100), 0.5), (torch.full_like(ids, 300), None, 1.0)):
        zs = spoilt.to(DEV).requires_grad_(True)
        loss = distillation_loss(zs, i.to(DEV), top.to(DEV), None if lab is None else lab.to(DEV), 2.0, alpha)
        assert float(loss.detach()) == 0.0 and bool((torch.autograd.grad(loss, zs)[0] == 0).all())
    # each part counts its own rows
    _check(z, torch.full_like(ids, -1), top, labels, 2.0, 0.5)
    _check(z, ids, top, torch.full_like(labels, 300), 2.0, 0.5)


def test_logits_of_minus_infinity_and_large_ones():
    from gruboros_amd.loss import distillation_loss

    z, ids, top, labels = _operands((2, 8), 500, 6, f32, masked=False)
    z[:, :, 100:200] = -float("inf")  # (as a mask leaves them)
    z[0, 1] = torch.finfo(f32).min
    z[0, 2] = 3e4 * torch.randn(500, generator=torch.Generator().manual_seed(1))
    z[0, 3] += 1e5
    ids = torch.where((ids >= 100) & (ids < 200), ids + 150, ids)
    labels = torch.where((labels >= 100) & (labels < 200), labels + 150, labels)
    keep = torch.ones(2, 8, dtype=torch.bool)
    keep[0, 1:4] = False
    zz, ii, ll = z.clone(), ids.clone(), labels.clone()
    ii[~keep], ll[~keep] = -1, -100
    g = _check(zz, ii, top, ll, 2.0, 0.5)
    assert bool((g[..., 100:200] == 0).all())
    # rows of large logits: the gradient alone (the loss's size is theirs)
    zg = z.to(DEV).requires_grad_(True)
    loss = distillation_loss(zg, ids.to(DEV), top.to(DEV), labels.to(DEV), 2.0, 0.5)
    want, dz, size = _reference(z, ids, top, labels, 2.0, 0.5)
    err = (torch.autograd.grad(loss, zg)[0].double().cpu().reshape(dz.shape) - dz).abs()
    # (the argument of exp is rounded at |z| k <= 3e5: 2^-24 of it, 2e-2)
    assert bool((err <= 2e-2 * size + 1e-12).all()) and abs(float(loss.detach()) - want) <= 1e-5 * abs(want)
    # a listed or labelled token of probability 0 costs infinity, with a finite gradient
    ids[1, 0, 0] = 150
    zg = z.to(DEV).requires_grad_(True)
    loss = distillation_loss(zg, ids.to(DEV), top.to(DEV), temperature=2.0)
    assert float(loss.detach()) == float("inf") and bool(torch.isfinite(torch.autograd.grad(loss, zg)[0]).all())
    # NaN where it counts is seen
    z[1, 1, 7] = float("nan")
    assert bool(torch.isnan(distillation_loss(z.to(DEV), ids.to(DEV), top.to(DEV))))


def test_strided_logits_and_other_types():
    """logits[:, :-1] against labels[:, 1:], transposed batches, bf16 teachers."""
    from gruboros_amd.loss import distillation_loss

    z, ids, top, labels = _operands((3, 9), 401, 11, bf16)
    top = top.to(bf16)
    zg = z.to(DEV).requires_grad_(True)
    loss = distillation_loss(zg[:, :-1], ids.to(DEV)[:, :-1], top.to(DEV)[:, :-1], labels.to(DEV)[:, 1:], 2.0, 0.5)
    want, dz, size = _reference(z[:, :-1], ids[:, :-1], top[:, :-1], labels[:, 1:], 2.0, 0.5)
    assert abs(float(loss.detach()) - want) <= 1e-5 * (abs(want) + 4)
    (g,) = torch.autograd.grad(loss, zg)
    assert bool((g[:, -1] == 0).all())
    err = (g[:, :-1].double().cpu().reshape(dz.shape) - dz).abs()
    assert bool((err <= 4e-6 * size + 2.0 ** -8 * dz.abs() + 1e-12).all())
    args = (ids.to(DEV), top.to(DEV), labels.to(DEV), 2.0, 0.5)
    same = distillation_loss(z.to(DEV), *args)
    assert torch.equal(same, distillation_loss(z.to(DEV).transpose(0, 1).contiguous().transpose(0, 1), *args))
    wide = torch.stack([z.to(DEV), z.to(DEV)], -1)
    assert torch.equal(same, distillation_loss(wide[..., 0], *args))


def test_against_differences():
    from gruboros_amd.loss import distillation_loss

    z, ids, top, labels = _operands((2, 5), 60, 7, f32)
    zg = z.to(DEV).requires_grad_(True)
    (g,) = torch.autograd.grad(distillation_loss(zg, ids.to(DEV), top.to(DEV), labels.to(DEV), 1.5, 0.6), zg)
    gen, h = torch.Generator().manual_seed(3), 1e-5
    for _ in range(4):
        d = torch.randn(z.shape, generator=gen, dtype=torch.float64)
        diff = (_reference(z.double() + h * d, ids, top, labels, 1.5, 0.6)[0] - _reference(z.double() - h * d, ids, top, labels, 1.5, 0.6)[0]) / (2 * h)
        assert abs(float((g.double().cpu() * d).sum()) - diff) <= 2e-5


def test_backward_twice_and_upstream():
    """A retained graph's second backward, other gradients of the loss, a leaf that accumulates."""
    from gruboros_amd.loss import distillation_loss

    ops = [t.to(DEV) for t in _operands((3, 5), 700, 8, f32)]
    z = ops[0].clone().requires_grad_(True)
    call = lambda: distillation_loss(z, *ops[1:], 2.0, 0.5)  # noqa: E731
    loss = call()
    one = torch.autograd.grad(loss, z, retain_graph=True)[0].clone()
    half = torch.autograd.grad(loss, z, torch.tensor(0.5, device=DEV), retain_graph=True)[0]
    again = torch.autograd.grad(loss, z, retain_graph=True)[0]
    assert torch.equal(again, one) and torch.equal(half, one * 0.5)
    (call() / 4).backward()
    (call() / 4).backward()
    assert torch.equal(z.grad, one / 2)
    z.grad = None
    (3.0 * call() + call()).backward()
    assert float((z.grad - 4 * one).abs().max()) <= 2.0 ** -22 * float(one.abs().max()) * 4
    assert torch.equal(torch.autograd.grad(call(), z, torch.zeros((), device=DEV))[0], torch.zeros_like(z))
    with pytest.raises(RuntimeError):
        torch.autograd.grad(call(), z, create_graph=True)[0].sum().backward()


def test_streams_and_graphs():
    from gruboros_amd.loss import distillation_loss

    made = []
    for seed in (0, 1):
        ops = [t.to(DEV) for t in _operands((2, 40), 3001, 16, bf16, seed=seed)]
        ops[0].requires_grad_(True)

        def call(ops=ops):
            loss = distillation_loss(*ops, 2.0, 0.5)
            return [loss.detach(), torch.autograd.grad(loss, ops[0])[0]]

        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        made.append((graph, out, ops, call))
    gen = torch.Generator(device=DEV).manual_seed(3)
    for _ in range(4):
        for graph, out, ops, call in made:
            with torch.no_grad():
                ops[0].copy_(torch.randn(ops[0].shape, generator=gen, device=DEV))
                ops[1][:, ::3] = -1
            graph.replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in out]
            assert all(torch.equal(a, b) for a, b in zip(got, call()))
    want = [m[3]() for m in made]
    torch.cuda.synchronize()
    for _ in range(3):
        for m in made:
            with torch.cuda.stream(torch.cuda.Stream()):
                m[0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for v, m in zip(want, made) for a, b in zip(m[1], v))


def test_backward_captured_without_its_forward():
    """Each replay gives the gradient once, not multiplied again, and an eager backward leaves a captured forward's alone."""
    from gruboros_amd.loss import distillation_loss

    ops = [t.to(DEV) for t in _operands((2, 40), 3001, 16, bf16)]
    z = ops[0].requires_grad_(True)
    call = lambda: distillation_loss(*ops, 2.0, 0.5)  # noqa: E731
    up = torch.tensor(0.5, device=DEV)
    (want,) = torch.autograd.grad(call(), z, up)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        loss = call()
        torch.autograd.grad(loss, z, up, retain_graph=True)
        eager = call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        (first,) = torch.autograd.grad(loss, z, up, retain_graph=True)  # (handed over before)
        (g,) = torch.autograd.grad(eager, z, up, retain_graph=True)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(first, want) and torch.equal(g, want)
    (again,) = torch.autograd.grad(eager, z, up, retain_graph=True)
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(again, want) and torch.equal(g, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        inside = call()
    graph.replay()
    grads = [torch.autograd.grad(inside, z, up, retain_graph=True)[0] for _ in range(2)]
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(t, want) for t in grads)


def test_values_beyond_32_bit_offsets():
    from gruboros_amd.loss import distillation_loss

    V, K = 65537, 4
    N = 2 ** 31 // V + 30
    gen = torch.Generator(device=DEV).manual_seed(0)
    z = torch.randn(N, V, generator=gen, device=DEV, dtype=bf16).requires_grad_(True)
    ids = torch.randint(0, V, (N, K), generator=gen, device=DEV)
    top = torch.randn(N, K, generator=gen, device=DEV)
    ids[: N - 16] = -1  # the last rows alone count
    (g,) = torch.autograd.grad(distillation_loss(z, ids, top, temperature=2.0), z)
    few = z.detach()[N - 16:].clone().requires_grad_(True)
    (h,) = torch.autograd.grad(distillation_loss(few, ids[N - 16:], top[N - 16:], temperature=2.0), few)
    assert torch.equal(g[N - 16:], h) and int(g[: N - 16].count_nonzero()) == 0


@pytest.mark.parametrize("grad", [True, False], ids=["grad", "no grad"])
def test_dual_tensors_are_refused(grad):
    import torch.autograd.forward_ad as fwd

    from gruboros_amd.loss import distillation_loss

    z, ids, top, labels = (t.to(DEV) for t in _operands((2, 3), 50, 4, f32))
    with torch.set_grad_enabled(grad), fwd.dual_level():
        for a in ((fwd.make_dual(z, torch.ones_like(z)), ids, top), (z, ids, fwd.make_dual(top, torch.ones_like(top)))):
            with pytest.raises((RuntimeError, NotImplementedError)):
                distillation_loss(*a, labels, 2.0, 0.5)
        distillation_loss(z, ids, top, labels, 2.0, 0.5)


def test_no_rows():
    from gruboros_amd.loss import distillation_loss

    z = torch.zeros(2, 0, 7, device=DEV).requires_grad_(True)
    loss = distillation_loss(z, torch.zeros(2, 0, 3, device=DEV, dtype=torch.int64), torch.zeros(2, 0, 3, device=DEV))
    assert float(loss.detach()) == 0.0 and torch.autograd.grad(loss, z)[0].shape == z.shape


def test_refusals():
    from gruboros_amd._lib import MingruHipError
    from gruboros_amd.loss import distillation_loss

    z, ids, top, labels = (t.to(DEV) for t in _operands((2, 3), 50, 4, f32))
    good = dict(logits=z, top_ids=ids, top_logits=top, labels=labels, temperature=2.0, alpha=0.5)
    for bad in (dict(logits=z[0, 0]), dict(logits=z[..., :0]), dict(top_ids=ids.float()), dict(top_ids=ids[:1]), dict(top_ids=ids[..., :0]),
                dict(top_logits=top[..., :3]), dict(labels=labels[:, :2]), dict(labels=labels.float()), dict(labels=None), dict(temperature=0.0),
                dict(temperature=float("nan")), dict(alpha=1.5), dict(alpha=-0.1), dict(top_logits=top.clone().requires_grad_(True)),
                dict(top_ids=ids.repeat(1, 1, 200), top_logits=top.repeat(1, 1, 200))):
        with pytest.raises(ValueError):
            distillation_loss(**{**good, **bad})
    for bad in (dict(logits=z.half()), dict(top_logits=top.half()), dict(labels=labels.cpu()), dict(top_ids=ids.cpu())):
        with pytest.raises(MingruHipError):
            distillation_loss(**{**good, **bad})
