"""A student in training and in generation: the scaled embedding, blocks of the gated recurrence between their norms, and
the distillation loss, run together as a program would, against the same model in float64.

Tolerances before any run, of a gradient's size. float32: a recurrence is within 2e-5 (its own tests), products of at
most 288 terms and norms within 2e-6; two blocks and the head, forward and backward, add to 1e-4, and a block's
gates, norms and residual add hand an error on with a gain of at most 2: 4e-4. bfloat16: some 14 tensors of
activations and as many of gradients are rounded by at most 2^-8 each, and five weights by as much; errors of either
sign add like a root, sqrt(33) 2^-8 = 0.022, with the same gain of 2 for each of two blocks: 0.09. The loss, a mean over
rows of values that are bounded by the logits: 1e-4 and 0.02.
"""
import pytest
import torch
import torch.nn.functional as F

from oracle.recurrence_oracle import gated_recurrence as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"
f32, bf16 = torch.float32, torch.bfloat16
V, D, E, LAYERS, EPS = 1000, 96, 64, 2, 1e-6
SCALE = D ** 0.5


class Student(torch.nn.Module):
    def __init__(self, dtype):
        super().__init__()
        gen = torch.Generator().manual_seed(11)
        n = lambda *s, std=1.0: torch.nn.Parameter(torch.randn(*s, generator=gen) * std)  # noqa: E731
        self.dtype = dtype
        self.table = n(V, D, std=0.1)
        self.first = torch.nn.Parameter(1 + 0.1 * n(D).data)
        self.blocks = torch.nn.ModuleList()
        for _ in range(LAYERS):
            b = torch.nn.Module()
            b.inp = torch.nn.Linear(D, 3 * E + D, bias=False)
            b.out = torch.nn.Linear(E, D, bias=False)
            b.inp.weight, b.out.weight = n(3 * E + D, D, std=D ** -0.5), n(D, E, std=E ** -0.5)
            b.decay, b.scale = n(E), n(D, std=0.5)
            b.w_branch, b.w = (torch.nn.Parameter(1 + 0.1 * n(D).data) for _ in range(2))
            self.blocks.append(b)
        self.head = torch.nn.Linear(D, V, bias=False)
        self.head.weight = n(V, D, std=D ** -0.5)

    def forward(self, ids, reset=None, states=None, step=False):
        """logits and the blocks' last states; with `step` of one token, on states that are updated in place"""
        from gruboros_amd.embed import scaled_embedding
        from gruboros_amd.linear import linear
        from gruboros_amd.norm import add_gated_rms_norm, rms_norm
        from gruboros_amd.recurrence import gated_recurrence, gated_recurrence_step

        x = scaled_embedding(ids, self.table, SCALE, out_dtype=f32)
        n = rms_norm(x, self.first, out_dtype=self.dtype)
        last = []
        for i, b in enumerate(self.blocks):
            u, gi, gr, gate = linear(n, b.inp).split([E, E, E, D], -1)
            if step:
                h = gated_recurrence_step(u, gi, gr, b.decay, states[i])
                last.append(states[i])
            else:
                h, state = gated_recurrence(u, gi, gr, b.decay, None if states is None else states[i], reset, return_state=True)
                last.append(state)
            x, n = add_gated_rms_norm(x, linear(h, b.out), b.w_branch, b.w, gate=gate, scale=b.scale, out_dtype=self.dtype, eps=EPS)
        return linear(n, self.head), last


def _plain(p, ids, reset):
    """The same in p's type from the definitions."""
    norm = lambda t, w, eps: t * torch.rsqrt(t.square().mean(-1, keepdim=True) + eps) * w  # noqa: E731
    x = SCALE * p["table"][ids]
    n = norm(x, p["first"], torch.finfo(f32).eps)
    for i in range(LAYERS):
        b = {k.split(".", 2)[2]: v for k, v in p.items() if k.startswith(f"blocks.{i}.")}
        u, gi, gr, gate = (n @ b["inp.weight"].T).split([E, E, E, D], -1)
        h, _ = oracle(u, gi, gr, b["decay"], reset=reset)
        x = x + b["scale"] * F.silu(gate) * norm(h @ b["out.weight"].T, b["w_branch"], EPS)
        n = norm(x, b["w"], EPS)
    return n @ p["head.weight"].T


def _batch(B, T, K=8, seed=0):
    gen = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, V, (B, T), generator=gen)
    reset = torch.rand(B, T, generator=gen) < 0.1
    top_ids = torch.stack([torch.randperm(V, generator=gen)[:K] for _ in range(B * T)]).view(B, T, K)
    top = torch.randn(B, T, K, generator=gen)
    labels = torch.randint(0, V, (B, T), generator=gen)
    top_ids[:, -2:], labels[:, -1] = -1, -100  # (a padded end)
    return ids, reset, top_ids, top, labels


def _train(model, ids, reset, top_ids, top, labels):
    from gruboros_amd.loss import distillation_loss

    logits, _ = model(ids, reset)
    loss = distillation_loss(logits, top_ids, top, labels, temperature=2.0, alpha=0.7)
    return loss.detach(), torch.autograd.grad(loss, list(model.parameters()))


@pytest.mark.parametrize("dtype", [f32, bf16], ids=["f32", "bf16"])
@pytest.mark.parametrize("B,T", [(1, 3), (2, 37), (3, 130)])
def test_training_step(B, T, dtype):
    model = Student(dtype).to(DEV)
    ids, reset, top_ids, top, labels = _batch(B, T)
    loss, grads = _train(model, *(t.to(DEV) for t in (ids, reset, top_ids, top, labels)))
    p = {k: v.detach().double().cpu().requires_grad_(True) for k, v in model.named_parameters()}
    z = _plain(p, ids, reset)
    rows, told = (top_ids[..., 0] >= 0), labels >= 0
    t = torch.softmax(top[rows].double() / 2.0, -1)
    q = torch.log_softmax(z[rows] / 2.0, -1).gather(-1, top_ids[rows])
    loss_ref = 0.7 * 4.0 * (t * (t.log() - q)).sum(-1).mean() + 0.3 * F.cross_entropy(z[told], labels[told])
    want = float(loss_ref.detach())
    assert abs(float(loss) - want) <= (1e-4 if dtype == f32 else 0.02) * want
    for (name, leaf), g, w in zip(p.items(), grads, torch.autograd.grad(loss_ref, list(p.values()))):
        assert g.dtype == f32 and g.shape == leaf.shape
        rel = float((g.double().cpu() - w).norm() / w.norm())
        assert rel <= (4e-4 if dtype == f32 else 0.09), f"{name}: {rel:.2e}"


@pytest.mark.parametrize("dtype", [f32, bf16], ids=["f32", "bf16"])
def test_generation_goes_on_from_a_prompt(dtype):
    """A prompt's last states and single tokens give the logits of the whole sequence: in float32 within 4e-4; in
    bfloat16 products over few rows sum in another order, so that each of the 14 roundings may fall to the other side."""
    model = Student(dtype).to(DEV)
    ids = _batch(3, 29)[0].to(DEV)
    with torch.no_grad():
        whole, last = model(ids)
        _, states = model(ids[:, :17])
        for t in range(17, 29):
            z, states = model(ids[:, t], states=states, step=True)
            err = float((z.double() - whole[:, t].double()).norm() / whole[:, t].double().norm())
            assert err <= (4e-4 if dtype == f32 else 0.09), f"token {t}: {err:.2e}"
        for a, b in zip(states, last):
            assert float((a - b).norm() / b.norm()) <= (4e-4 if dtype == f32 else 0.09)


def test_captured_training_step():
    """The whole step in a graph, replayed on other batches with eager steps between."""
    model = Student(bf16).to(DEV)
    batch = [t.to(DEV) for t in _batch(2, 65)]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        _train(model, *batch)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        loss, grads = _train(model, *batch)
    for seed in range(4):
        for t, new in zip(batch, _batch(2, 65, seed=seed)):
            t.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        got = [loss.clone()] + [g.clone() for g in grads]
        eager, eager_grads = _train(model, *batch)
        for a, b in zip(got, [eager, *eager_grads]):
            assert float((a - b).norm()) <= 1e-5 * float(b.norm())
