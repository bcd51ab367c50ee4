"""The scaled embedding and its gradient by sorted tokens against float64.

Tolerances before any run. The lookup: one product, half a step of the output's type (2^-24, 2^-8),
and another half step in fp32 before a bf16 rounding (2^-24). The gradient of a row: n values summed
in fp32, pieces of 32 and then the pieces, so at most 32 + n / 32 + 64 terms in a row, each sum off
by half a step of its size: (96 + n / 32) 2^-24 of the sum of the values' sizes, and half a step of
the table's type.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
f32, bf16 = torch.float32, torch.bfloat16
HALF = {f32: 2.0 ** -24, bf16: 2.0 ** -8}


def _want(ids, dy, V, scale, skip=()):
    """(dw, sum of sizes) in float64"""
    flat, rows = ids.flatten().long().cpu(), dy.double().cpu().reshape(ids.numel(), -1)
    ok = (flat >= 0) & (flat < V)
    for s in skip:
        ok &= flat != s
    dw = torch.zeros(V, rows.shape[1], dtype=torch.float64).index_add_(0, flat[ok], rows[ok] * scale)
    return dw, torch.zeros_like(dw).index_add_(0, flat[ok], (rows[ok] * scale).abs())


def _check(ids, V, D, wt, yt, scale=1.7, skip=None, seed=0):
    from gruboros_amd.embed import scaled_embedding

    gen = torch.Generator().manual_seed(seed + V + D)
    w = torch.randn(V, D, generator=gen).to(wt)
    dy = torch.randn(*ids.shape, D, generator=gen).to(yt)
    wg = w.to(DEV).requires_grad_(True)
    y = scaled_embedding(ids.to(DEV), wg, scale, yt, skip)
    assert y.dtype == yt and y.shape == (*ids.shape, D)
    inside = (ids >= 0) & (ids < V)
    ref = w.double()[ids.long().clamp(0, V - 1)] * scale
    lim = (HALF[yt] + 2.0 ** -23) * ref.abs() + 1e-37
    assert bool(((y.detach().double().cpu() - ref).abs() <= lim)[inside].all())
    assert bool(torch.isnan(y.cpu()[~inside]).all())
    (g,) = torch.autograd.grad(y, wg, dy.to(DEV))
    assert g.dtype == wt and g.shape == w.shape
    want, size = _want(ids, dy, V, scale, () if skip is None else (skip % V,))
    most = int(torch.bincount(ids[inside].flatten().long(), minlength=1).max()) if bool(inside.any()) else 0
    lim = (96 + most / 32) * 2.0 ** -24 * size + HALF[wt] * want.abs() + 1e-37
    err = (g.double().cpu() - want).abs()
    assert bool((err <= lim).all()), float((err - lim).max())
    return g


TYPES = pytest.mark.parametrize("types", [(f32, f32), (f32, bf16), (bf16, bf16), (bf16, f32)], ids=lambda t: "-".join(str(x)[6:] for x in t))


@TYPES
@pytest.mark.parametrize("size", [(1, 1, 1), (3, 2, 7), (65, 1001, 250), (31, 600, 64), (33, 1, 40), (1000, 1023, 17), (1000, 1024, 8), (4096, 5000, 24),
                                  (4097, 5000, 24), (9000, 70000, 12), (5000, 1 << 20, 3), (300, 40, 1030)], ids=lambda s: "x".join(map(str, s)))
def test_parity(size, types):
    N, V, D = size
    gen = torch.Generator().manual_seed(N)
    _check(torch.randint(0, V, (N,), generator=gen), V, D, *types)


@pytest.mark.parametrize("N", [40, 3000, 20000])
@pytest.mark.parametrize("form", ["one", "two", "common", "sorted", "backwards", "ends"])
def test_distributions(N, form):
    """Ids of many tokens: runs that start and end within pieces, one id only, the table's first and last rows."""
    gen = torch.Generator().manual_seed(N)
    V = 50000
    ids = {"one": torch.full((N,), 17), "two": torch.randint(0, 2, (N,), generator=gen) * 777,
           "common": torch.where(torch.rand(N, generator=gen) < 0.6, torch.tensor(31999), torch.randint(0, V, (N,), generator=gen)),
           "sorted": torch.arange(N) % V, "backwards": (V - 1) - torch.arange(N) // 100, "ends": torch.randint(0, 2, (N,), generator=gen) * (V - 1)}[form]
    _check(ids, V, 72, f32, f32)
    _check(ids, V, 513, f32, bf16)


def test_ids_outside_the_table_and_padding():
    gen = torch.Generator().manual_seed(1)
    for N in (50, 7000):
        ids = torch.randint(-3, 1005, (N,), generator=gen)
        ids[::7] = torch.tensor([-2 ** 40, 2 ** 40, 2 ** 32 + 5, -1, 1000, 2 ** 31])[torch.arange(len(ids[::7])) % 6]
        _check(ids, 1000, 33, f32, f32)
        _check(ids, 1000, 33, bf16, bf16, skip=5)
        g = _check(ids, 1000, 33, f32, bf16, skip=-1)
        assert bool((g[999] == 0).all())
    _check(torch.full((100,), -1), 10, 8, f32, f32)  # nothing is looked up


def test_int32_ids_views_and_shapes():
    from gruboros_amd.embed import scaled_embedding

    gen = torch.Generator().manual_seed(2)
    ids = torch.randint(0, 900, (6, 50), generator=gen)
    a = _check(ids, 900, 20, f32, f32)
    assert torch.equal(a, _check(ids.int(), 900, 20, f32, f32))
    w = torch.randn(900, 41, generator=gen).to(DEV)
    view = w[:, 1:].detach().requires_grad_(True)  # (rows at odd distances)
    cols = ids.to(DEV).t()
    y = scaled_embedding(cols, view, 2.0)
    assert torch.equal(y, (2.0 * view)[cols])
    g = torch.autograd.grad(y.sum(), view)[0]  # (a gradient that is broadcast)
    count = torch.bincount(ids.flatten(), minlength=900).to(DEV)
    assert torch.equal(g, (2.0 * count).unsqueeze(-1).expand_as(g).float())
    assert scaled_embedding(torch.tensor(3, device=DEV), w).shape == (41,)


def test_not_finite_rows_stay_apart():
    from gruboros_amd.embed import scaled_embedding

    gen = torch.Generator().manual_seed(3)
    ids = torch.randint(0, 50, (3000,), generator=gen).to(DEV)
    w = torch.randn(60, 24, generator=gen).to(DEV).requires_grad_(True)
    dy = torch.randn(3000, 24, generator=gen).to(DEV)
    clean = torch.autograd.grad(scaled_embedding(ids, w), w, dy)[0]
    dy[ids == 7] = float("nan")
    g = torch.autograd.grad(scaled_embedding(ids, w), w, dy)[0]
    rest = torch.arange(60, device=DEV) != 7
    assert torch.equal(g[rest], clean[rest]) and bool(torch.isnan(g[7]).all())
    # (without the tokens of row 7 the other runs lie elsewhere among the pieces: the same values in another grouping)
    g = torch.autograd.grad(scaled_embedding(ids, w, padding_idx=7), w, dy)[0].double().cpu()
    want, size = _want(ids, torch.nan_to_num(dy), 60, 1.0, (7,))
    assert bool(((g - want).abs() <= 200 * 2.0 ** -24 * size).all()) and bool((g[7] == 0).all())


def test_the_byte_vocabulary_agrees():
    """Tables of up to 512 rows have mg_embedding_bwd too."""
    from gruboros_amd.embed import embedding, scaled_embedding

    gen = torch.Generator().manual_seed(4)
    ids = torch.randint(0, 256, (4, 777), generator=gen).to(DEV)
    w = torch.randn(256, 64, generator=gen).to(DEV).requires_grad_(True)
    dy = torch.randn(4, 777, 64, generator=gen).to(DEV)
    assert torch.equal(embedding(ids, w), scaled_embedding(ids, w))
    a, b = (torch.autograd.grad(f(ids, w), w, dy)[0] for f in (embedding, scaled_embedding))
    assert float((a - b).abs().max()) <= 100 * 2.0 ** -24 * float(dy.abs().sum((0, 1)).max())


def test_bits_repeat_and_no_values():
    from gruboros_amd.embed import scaled_embedding

    gen = torch.Generator().manual_seed(5)
    ids = torch.randint(0, 300, (20000,), generator=gen).to(DEV)
    w = torch.randn(30000, 32, generator=gen).to(DEV).requires_grad_(True)
    dy = torch.randn(20000, 32, generator=gen).to(DEV)
    y = scaled_embedding(ids, w, 0.5)
    first = torch.autograd.grad(y, w, dy, retain_graph=True)[0]
    for _ in range(5):
        assert torch.equal(first, torch.autograd.grad(y, w, dy, retain_graph=True)[0])
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y, w, dy.clone().requires_grad_(True), create_graph=True)[0].sum().backward()
    for shape in ((0,), (3, 0)):
        y = scaled_embedding(torch.zeros(shape, dtype=torch.int64, device=DEV), w, out_dtype=bf16)
        assert y.shape == (*shape, 32) and y.dtype == bf16
        assert bool((torch.autograd.grad(y.sum(), w)[0] == 0).all())


def test_streams_and_graphs():
    from gruboros_amd.embed import scaled_embedding

    made = []
    for seed, N in ((0, 3000), (1, 9000)):
        gen = torch.Generator().manual_seed(seed)
        ids = torch.randint(0, 2000, (N,), generator=gen).to(DEV)
        w = torch.randn(20000, 48, generator=gen).to(DEV).requires_grad_(True)
        dy = torch.randn(N, 48, generator=gen).to(DEV)

        def call(ids=ids, w=w, dy=dy):
            y = scaled_embedding(ids, w, 3.0)
            return [y.detach(), torch.autograd.grad(y, w, dy)[0]]

        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        made.append((graph, out, ids, call))
    for rep in range(4):
        for graph, out, ids, call in made:
            ids.copy_(torch.randint(0, 20000, ids.shape, generator=torch.Generator().manual_seed(rep)))
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


def test_values_beyond_32_bit_offsets():
    """A table and a gradient of more than 2^31 values, and outputs of more."""
    from gruboros_amd.embed import scaled_embedding

    V, D = 2 ** 21 + 5, 1030
    w = torch.zeros(V, D, dtype=bf16, device=DEV)
    rows = torch.tensor([0, 1, V // 2, V - 2, V - 1], device=DEV)
    w[rows] = torch.randn(5, D, generator=torch.Generator().manual_seed(6)).to(DEV).to(bf16)
    w.requires_grad_(True)
    ids = rows[torch.randint(0, 5, (6000,), generator=torch.Generator().manual_seed(7)).to(DEV)]
    y = scaled_embedding(ids, w, 1.0)
    assert torch.equal(y, w.detach()[ids])
    (g,) = torch.autograd.grad(y, w, torch.ones_like(y))
    counts = torch.bincount(torch.searchsorted(rows, ids), minlength=5)
    assert torch.equal(g[rows], counts.to(bf16).unsqueeze(-1).expand(5, D).contiguous())
    assert int(g.count_nonzero(-1).count_nonzero()) == 5
    del w, y, g
    N = 2 ** 21 + 100  # (outputs beyond 2^31 values)
    w = torch.randn(40, 1030, generator=torch.Generator().manual_seed(8)).to(DEV).to(bf16).requires_grad_(True)
    ids = torch.arange(N, device=DEV) % 40
    y = scaled_embedding(ids, w, 1.0)
    assert torch.equal(y[-80:], w.detach()[ids[-80:]])
    (g,) = torch.autograd.grad(y, w, torch.ones_like(y))
    count = torch.bincount(ids, minlength=40).to(bf16)
    assert torch.equal(g, count.unsqueeze(-1).expand(40, 1030).contiguous())


def test_the_largest_table():
    """2^28 - 1 rows: three passes of digits, more rows than one dimension of a launch has threads for."""
    from gruboros_amd.embed import scaled_embedding

    V = 2 ** 28 - 1
    ids = torch.randint(0, V, (5000,), generator=torch.Generator().manual_seed(9)).to(DEV)
    ids[:900] = V - 1
    ids[900:907] = torch.tensor([0, 2 ** 20 - 1, 2 ** 20, 2 ** 24, 2 ** 27, V, -1], device=DEV)
    w = torch.ones(V, 1, dtype=bf16, device=DEV).requires_grad_(True)
    y = scaled_embedding(ids, w, 2.0)
    outside = (ids < 0) | (ids >= V)
    assert torch.equal(y.isnan().flatten(), outside) and bool((y[~outside] == 2.0).all())
    (g,) = torch.autograd.grad(y, w, torch.ones_like(y))
    at, count = torch.unique(ids[~outside], return_counts=True)
    assert torch.equal(g[at, 0], (2 * count).to(bf16)) and int(torch.count_nonzero(g)) == len(at)


@pytest.mark.parametrize("grad", [True, False], ids=["grad", "no grad"])
def test_dual_tensors_are_refused(grad):
    import torch.autograd.forward_ad as fwd

    from gruboros_amd.embed import scaled_embedding

    w, ids = torch.randn(9, 4, device=DEV), torch.arange(3, device=DEV)
    with torch.set_grad_enabled(grad), fwd.dual_level():
        with pytest.raises((RuntimeError, NotImplementedError)):
            scaled_embedding(ids, fwd.make_dual(w, torch.ones_like(w)))
        scaled_embedding(ids, w)


def test_refusals():
    from gruboros_amd._lib import MingruHipError
    from gruboros_amd.embed import scaled_embedding

    w, ids = torch.randn(9, 4, device=DEV), torch.arange(3, device=DEV)
    for a, k in (((ids.float(), w), {}), ((ids.bool(), w), {}), ((ids, w[0]), {}), ((ids, w[:0]), {}), ((ids, w), {"padding_idx": 9}),
                 ((ids, w), {"padding_idx": -10})):
        with pytest.raises(ValueError):
            scaled_embedding(*a, **k)
    for a, k in (((ids, w.half()), {}), ((ids, w), {"out_dtype": torch.float16}), ((ids.cpu(), w), {}), ((ids, w.cpu()), {})):
        with pytest.raises(MingruHipError):
            scaled_embedding(*a, **k)
