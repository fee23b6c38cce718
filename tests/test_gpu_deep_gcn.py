"""The deep GCN with layer norms and residual blocks, trained from a teacher's
top logits: the operators together, against a dense 64-bit evaluation, their
autograd nodes, and the command that trains it.

The forward SpMM rounds its input to TF32; the dense evaluation does the same.
A value that fp32 arithmetic leaves off by about 16 u = 2^-20 rounds to the other
side with a probability of 2^-20 / 2^-10 and then differs by 2^-10: rel-L2 3e-5
for each of the four products, in the gradients again: 3e-4."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
REL = 3e-4


def rel_l2(a, b):
    a = a.detach().double().cpu()
    return float((a - b).norm() / b.norm().clamp(min=1e-30))


class TF32(torch.autograd.Function):
    """Rounding to TF32 in the forward pass, the identity backwards."""

    @staticmethod
    def forward(ctx, x):
        b = x.float().numpy().view(np.uint32).astype(np.uint64)
        return torch.from_numpy(((b + 0x1000) & 0xFFFFE000).astype(np.uint32).view(np.float32)).double()

    @staticmethod
    def backward(ctx, d):
        return d


def normed(h, w, b):
    d = h - h.mean(1, keepdim=True)
    return torch.nn.functional.silu(d / torch.sqrt(d.pow(2).mean(1, keepdim=True) + 1e-5) * w + b)


def dense_loss(model, A, ids, entries, T):
    """The student's loss and the gradients of all its parameters."""
    p = {k: v.detach().double().cpu().requires_grad_(True) for k, v in model.named_parameters()}
    h = (A @ TF32.apply(p["embedding.weight"][ids] * model.embedding.scale)) @ p["conv1.weights"]
    y = normed(h, p["norm.weight"], p["norm.bias"])
    for k in range(len(model.convs)):
        h = h + (A @ TF32.apply(y)) @ p[f"convs.{k}.weights"]
        y = normed(h, p[f"norms.{k}.weight"], p[f"norms.{k}.bias"])
    z = A @ TF32.apply(y @ p["conv_final.weights"])
    values, at, rest = (t.cpu() for t in entries)
    log_q = torch.log_softmax(z / T, 1)
    others = torch.ones_like(z, dtype=torch.bool).scatter(1, at.long(), False)
    mine = torch.cat([log_q.gather(1, at.long()), torch.logsumexp(log_q.masked_fill(~others, -np.inf), 1, keepdim=True)], 1)
    log_p = torch.log_softmax(torch.cat([values.double(), rest.double()[:, None]], 1) / T, 1)
    loss = T * T * (log_p.exp() * (log_p - mine)).sum(1).mean()
    return z.detach(), loss.detach(), dict(zip(p, torch.autograd.grad(loss, list(p.values()))))


def small_batch(norm="layer", blocks=2):
    from tcc_amd import gcn
    from tcc_amd.train_embeddings import batch_of_graphs

    torch.manual_seed(1)
    rows, cols, ids, offsets, longest = batch_of_graphs(700, 25, 40, 3)
    n = ids.numel()
    graph = gcn.LayerGraph(rows, cols, n, n)
    A = torch.zeros((n, n), dtype=torch.float64)
    A[rows, cols] = 1.0
    model = gcn.EmbeddingGCN(700, 24, 48, 9, activation="silu", norm=norm, blocks=blocks)
    with torch.no_grad():
        for name, p in model.named_parameters():
            if "norm" in name:
                p.add_(torch.randn_like(p) * 0.2)
    return model, graph, A, ids, offsets, longest


def test_step_matches_dense_reference(gpu):
    from tcc_amd import gcn, training

    model, graph, A, ids, _, _ = small_batch()
    T = 2.0
    entries = training.top_logits(torch.randn((ids.numel(), 9), device="cuda") * 3, 4, temperature=T)
    loss_fcn = gcn.DistillationLoss(T)
    out = model(graph, ids.cuda())
    loss = loss_fcn(out, entries)
    loss.backward()
    assert model.embedding.error() == 0 and loss_fcn.error() == 0
    want, want_loss, grads = dense_loss(model, A, ids, entries, T)
    assert rel_l2(out, want) < REL and abs(float(loss.detach()) - float(want_loss)) < REL * float(want_loss)
    for name, p in model.named_parameters():
        assert rel_l2(p.grad, grads[name]) < REL, name


def test_models_that_were_there_stay(gpu):
    """The same parameters under the same names, from the same random numbers."""
    from tcc_amd import gcn

    torch.manual_seed(3)
    model = gcn.EmbeddingGCN(50, 16, 32, 4)
    assert list(model.state_dict()) == ["embedding.weight", "conv1.weights", "norm.weight", "norm.bias", "conv_final.weights"]
    assert isinstance(model.norm, gcn.NodeGroupNorm)
    torch.manual_seed(3)
    table = torch.randn((50, 16), device="cuda").div_(4.0)
    assert torch.equal(model.embedding.weight, table)
    for bad in (dict(norm="batch"), dict(blocks=1), dict(norm="layer", blocks=-1)):
        with pytest.raises(ValueError):
            gcn.EmbeddingGCN(50, 16, 32, 4, **bad)


def test_layer_norm_node(gpu):
    """One output used, the other, both; a residual that is x itself; parameters
    and inputs of 16 bits; no weight."""
    from tcc_amd import gcn

    gen = torch.Generator(device="cuda").manual_seed(5)
    leaf = lambda *s: torch.randn(s, generator=gen, device="cuda").requires_grad_(True)  # noqa: E731
    x, r, w, b = leaf(40, 30), leaf(40, 30), leaf(30), leaf(30)
    d, e = torch.randn((2, 40, 30), generator=gen, device="cuda")

    def plain(x, r, w, b, d, e):
        h = x if r is None else x + r
        y = torch.nn.functional.layer_norm(h, (30,), w, b)
        return sum((a * t).sum() for a, t in ((d, torch.nn.functional.gelu(y)), (e, h)) if a is not None)

    def own(x, r, w, b, d, e):
        y, h = gcn.LayerNormFunction.apply(x, r, w, b, 1e-5, "gelu")
        return sum((a * t).sum() for a, t in ((d, y), (e, h)) if a is not None)

    for residual in (r, x):
        for de in ((d, e), (d, None), (None, e)):
            leaves = [t for t in ((x, r) if residual is r else (x,))] + ([w, b] if de[0] is not None else [])
            got = torch.autograd.grad(own(x, residual, w, b, *de), leaves)
            doubles = [t.detach().double().requires_grad_(True) for t in leaves]
            by = dict(zip(map(id, leaves), doubles))
            args = [by.get(id(t), t.detach().double()) for t in (x, residual, w, b)]
            want = torch.autograd.grad(plain(*args, *(None if t is None else t.double() for t in de)), doubles)
            for p, q in zip(got, want):  # sums of 30 and of 40 terms
                assert rel_l2(p, q.cpu()) < 64 * 2.0**-24
    h = x.detach().bfloat16().requires_grad_(True)
    w16 = w.detach().bfloat16().requires_grad_(True)
    y = gcn.LayerNormFunction.apply(h, None, w16, None, 1e-5, "none")
    y.backward(d.bfloat16())
    assert y.dtype == h.grad.dtype == w16.grad.dtype == torch.bfloat16


def test_second_derivatives_are_refused(gpu):
    from tcc_amd import gcn, training

    gen = torch.Generator(device="cuda").manual_seed(4)
    leaf = lambda *s: torch.randn(s, generator=gen, device="cuda").requires_grad_(True)  # noqa: E731
    x, r, w, b, z = leaf(30, 16), leaf(30, 16), leaf(16), leaf(16), leaf(30, 16)
    entries = training.top_logits(torch.randn((30, 16), device="cuda"), 3)
    loss_fcn = gcn.DistillationLoss()
    nodes = [
        (lambda: gcn.LayerNormFunction.apply(x, None, w, b, 1e-5, "none").sum(), (x, w)),
        (lambda: sum(t.square().sum() for t in gcn.LayerNormFunction.apply(x, r, w, b, 1e-5, "silu")), (x, r, w, b)),
        (lambda: loss_fcn(z, entries), (z,)),
    ]
    for f, leaves in nodes:
        plain = torch.autograd.grad(f(), leaves)
        grads = torch.autograd.grad(f(), leaves, create_graph=True)
        for g, p in zip(grads, plain):
            assert torch.equal(g, p)
        for g, t in zip(grads, leaves):
            with pytest.raises(RuntimeError, match="second derivative"):
                torch.autograd.grad((g * t).sum(), t, retain_graph=True)


def test_entries_are_constants_and_reported(gpu):
    from tcc_amd import gcn, training

    z = torch.randn((20, 12), device="cuda", requires_grad=True)
    values, ids, rest = training.top_logits(z, 3)
    assert not values.requires_grad and not rest.requires_grad
    loss_fcn = gcn.DistillationLoss(weight=torch.ones(20, device="cuda"))
    with pytest.raises(ValueError, match="constants"):
        loss_fcn(z, (z[:, :3], ids, rest))
    ids[3, 1] = 12
    loss_fcn(z, (values, ids, None)).backward()
    assert loss_fcn.error() == 7 and loss_fcn.error() == 0
    assert bool(torch.isfinite(z.grad).all())
    moved = loss_fcn.to("cpu")
    assert moved.device_error.device.type == moved.weight.device.type == "cpu" and list(moved.state_dict()) == []


def test_captured_step(gpu):
    """A whole step, forward and backward, replayed from a graph with other
    inputs: every replay has the eager bits."""
    from tcc_amd import gcn, training

    gen = torch.Generator(device="cuda").manual_seed(6)
    new = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    x, r, entries_of = new(2000, 96), new(2000, 96), new(2000, 96)
    norm, loss_fcn = gcn.NodeLayerNorm(96, "gelu"), gcn.DistillationLoss(2.0)
    teacher = [t.clone() for t in training.top_logits(entries_of, 8, temperature=2.0)]

    def step():
        y, h = norm(x, r)
        loss = loss_fcn(y + h, teacher)
        return (loss.detach(), *torch.autograd.grad(loss, list(norm.parameters())))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(3):
        for t in (x, r):
            t.copy_(new(2000, 96))
        for p, q in zip(teacher, training.top_logits(new(2000, 96), 8, temperature=2.0)):
            p.copy_(q)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(out, step()):
            assert torch.equal(p, q)


def test_capture_beside_a_living_eager_graph_is_refused(gpu):
    """Its gradients belong to the default stream, which a capture may not wait
    for; refused before anything of the backward pass runs."""
    from tcc_amd import gcn, training

    gen = torch.Generator(device="cuda").manual_seed(8)
    x = torch.randn((300, 40), generator=gen, device="cuda")
    teacher = training.top_logits(x * 2, 3)
    norm, loss_fcn = gcn.NodeLayerNorm(40, "silu"), gcn.DistillationLoss()
    logits = x.clone().requires_grad_()
    alive = norm(x), loss_fcn(logits, teacher)
    assert training.held_by_default_stream([None, norm.weight]) and training.held_by_default_stream([logits])
    assert not training.held_by_default_stream([None, x])
    for call in (lambda: norm(x), lambda: loss_fcn(logits, teacher)):
        with pytest.raises(RuntimeError, match="is alive"), torch.cuda.graph(torch.cuda.CUDAGraph()):
            x + 1
            call()
    with torch.no_grad(), torch.cuda.graph(torch.cuda.CUDAGraph()):
        norm(x)  # nothing to differentiate
    del alive
    assert not training.held_by_default_stream([norm.weight, norm.bias, logits])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = torch.autograd.grad(norm(x), list(norm.parameters()), torch.ones_like(x))
    graph.replay()
    torch.cuda.synchronize()
    for p, q in zip(out, torch.autograd.grad(norm(x), list(norm.parameters()), torch.ones_like(x))):
        assert torch.equal(p, q)


def test_two_streams_at_once(gpu):
    """Calls on two streams share no workspace."""
    from tcc_amd import training

    gen = torch.Generator(device="cuda").manual_seed(7)
    z = torch.randn((2, 4000, 300), generator=gen, device="cuda")
    entries = [training.top_logits(z[k] * 2, 9) for k in range(2)]
    w, d = torch.rand(300, generator=gen, device="cuda"), torch.randn((2, 4000, 300), generator=gen, device="cuda")
    stats = [training.layer_norm(z[k], w) for k in range(2)]

    def work(k, stream=None):
        loss = training.distill_loss(z[k], *entries[k], stream=stream)[0]
        return (loss, *training.layer_norm_grad(d[k], z[k], stats[k][2], stats[k][3], w, stream=stream)[:2])

    want = [work(k) for k in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[work(k, s) for k, s in enumerate(streams)] for _ in range(20)]
    torch.cuda.synchronize()
    for pair in got:
        for a, b in zip(pair, want):
            for p, q in zip(a, b):
                assert torch.equal(p, q)


@pytest.mark.parametrize("norm,blocks", [("layer", 2), ("group", 0)])
def test_command_runs(gpu, norm, blocks):
    from tcc_amd import train_embeddings

    lines = []
    losses, norms, student = train_embeddings.train(nodes=500, graphs=12, mean_rows=30, dim=32, hidden=64, steps=3,
                                                    log=lines.append, norm=norm, blocks=blocks, classes=12, distill=4)
    assert len(losses) == 3 and len(lines) == 6 and lines[3].startswith("student: step 0")
    assert np.isfinite(losses).all() and np.isfinite(norms).all()
    assert all(bool(torch.isfinite(p.grad).all()) and bool((p.grad != 0).any()) for p in student.parameters())
    assert student.conv1.weights.shape == (8, 16)
