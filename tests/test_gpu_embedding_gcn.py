"""The GCN with learned node rows (tcc_amd.gcn.EmbeddingGCN) against a dense
64-bit evaluation, its optimizer, and the example that trains it.

The forward SpMM rounds its input to TF32 (2^-11 of each value); the dense
evaluation does the same where the model does, so that what is left is fp32
arithmetic: rel-L2 1e-4, as for the GCN with given features."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
REL = 1e-4


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


def dense_step(A, table, ids, W1, w, b, W2, labels, at, groups, scale):
    t = [v.detach().double().cpu().requires_grad_(True) for v in (table, W1, w, b, W2)]
    x = t[0][ids] * scale
    h = (A @ TF32.apply(x)) @ t[1] if W1.shape[1] >= W1.shape[0] else A @ TF32.apply(x @ t[1])
    parts = []
    for lo, hi in zip(at[:-1], at[1:]):
        v = h[lo:hi].view(hi - lo, groups, -1)
        d = v - v.mean((0, 2), keepdim=True)
        parts.append((d / torch.sqrt(d.pow(2).mean((0, 2), keepdim=True) + 1e-5)).reshape(hi - lo, -1))
    r = torch.relu(torch.cat(parts) * t[2] + t[3])
    out = A @ TF32.apply(r @ t[4])
    loss = torch.nn.functional.cross_entropy(out, labels)
    return out.detach(), loss.detach(), torch.autograd.grad(loss, t)


@pytest.mark.parametrize("batch", [True, False])
def test_step_matches_dense_reference(gpu, batch):
    from tcc_amd import gcn
    from tcc_amd.train_embeddings import batch_of_graphs

    torch.manual_seed(1)
    nodes, dim, hidden, classes, groups = 700, 24, 48, 3, 6
    rows, cols, ids, offsets, longest = batch_of_graphs(nodes, 25, 40, 3)
    n = ids.numel()
    graph = gcn.LayerGraph(rows, cols, n, n)
    model = gcn.EmbeddingGCN(nodes, dim, hidden, classes, num_groups=groups)
    labels = gcn.synthetic_labels(n, classes, 5)
    with torch.no_grad():
        model.norm.weight.uniform_(0.5, 1.5)
        model.norm.bias.normal_()
    off = offsets.cuda() if batch else None
    out = model(graph, ids.cuda(), off, longest if batch else None)
    loss = gcn.cross_entropy(out, labels)
    loss.backward()
    assert model.embedding.error() == 0
    A = torch.zeros((n, n), dtype=torch.float64)
    A[rows, cols] = 1.0
    at = offsets.tolist() if batch else [0, n]
    params = (model.embedding.weight, model.conv1.weights, model.norm.weight, model.norm.bias, model.conv_final.weights)
    want, want_loss, grads = dense_step(A, params[0], ids, params[1], params[2], params[3], params[4], labels.cpu(), at,
                                        groups, model.embedding.scale)
    assert rel_l2(out, want) < REL and abs(float(loss) - float(want_loss)) < REL
    for p, g in zip(params, grads):
        assert rel_l2(p.grad, g) < REL
    untouched = torch.ones(nodes, dtype=torch.bool)
    untouched[ids] = False
    assert int(torch.count_nonzero(model.embedding.weight.grad.cpu()[untouched])) == 0


def test_second_derivatives_are_refused(gpu):
    """A gradient that is taken with create_graph=True has its value, and a
    second differentiation raises: nothing counts as a constant silently."""
    from tcc_amd import gcn

    gen = torch.Generator(device="cuda").manual_seed(4)
    leaf = lambda *s: torch.randn(s, generator=gen, device="cuda").requires_grad_(True)  # noqa: E731
    table, x, w, b, w1, wide = leaf(9, 16), leaf(30, 16), leaf(16), leaf(16), leaf(16, 24), leaf(24, 2)
    ids = torch.randint(0, 9, (30,), generator=gen, device="cuda")
    graph, small = (gcn.LayerGraph(torch.arange(n), (torch.arange(n) * 7) % n, n, n) for n in (30, 16))
    norm = lambda act: gcn.GroupNormFunction.apply(x, w, b, 4, None, 1e-5, act, None)  # noqa: E731
    nodes = [
        (lambda: gcn.EmbeddingFunction.apply(table, ids, 1.0, None, None).square().sum(), (table,)),
        (lambda: norm("silu").square().sum(), (x, w, b)),
        (lambda: norm("none").sum(), (x, w, b)),  # the slope depends on x and w alone
        (lambda: gcn.CNICSPMMFunction.apply(graph, None, x, w1).square().sum(), (x, w1)),
        (lambda: gcn.TransformFirstFunction.apply(small, w1, wide).square().sum(), (w1, wide)),
    ]
    for f, leaves in nodes:
        plain = torch.autograd.grad(f(), leaves)
        grads = torch.autograd.grad(f(), leaves, create_graph=True)
        for g, p in zip(grads, plain):
            assert torch.equal(g, p)
        for g, t in zip(grads, leaves):
            with pytest.raises(RuntimeError, match="second derivative"):
                torch.autograd.grad((g * t).sum(), t, retain_graph=True)
    # a gradient that is a constant stays one: the lookup is linear
    (g,) = torch.autograd.grad(gcn.EmbeddingFunction.apply(table, ids, 1.0, None, None).sum(), table, create_graph=True)
    (again,) = torch.autograd.grad((g * table).sum(), table)
    assert torch.equal(again, g)


def test_padding_row_stays_and_bad_ids_are_reported(gpu):
    from tcc_amd import gcn, swtcf

    e = gcn.NodeEmbedding(20, 8, padding_idx=3)
    ids = torch.tensor([3, 5, 3, 7], device="cuda")
    y = e(ids)
    assert torch.equal(y[0], torch.zeros(8, device="cuda"))
    y.sum().backward()
    assert int(torch.count_nonzero(e.weight.grad[3])) == 0 and int(torch.count_nonzero(e.weight.grad[5])) == 8
    assert e.error() == 0
    e(torch.tensor([25], device="cuda"))
    assert e.error() == swtcf.DEVERR_FEATURE_INDEX and e.error() == 0


def test_optimizer_follows_torch(gpu):
    """ClippedAdam against clip_grad_norm_ and torch.optim.AdamW over steps with
    gradients above and below the largest norm."""
    from tcc_amd import gcn

    gen = torch.Generator(device="cuda").manual_seed(2)
    new = lambda: [torch.nn.Parameter(torch.randn(s, generator=gen, device="cuda")) for s in ((30, 7), (11,))]  # noqa: E731
    mine = new()
    twin = [torch.nn.Parameter(p.detach().clone()) for p in mine]
    unused = torch.nn.Parameter(torch.ones(4, device="cuda"))
    a = gcn.ClippedAdam(mine + [unused], lr=0.02, weight_decay=0.1, max_norm=1.0)
    b = torch.optim.AdamW(twin, lr=0.02, weight_decay=0.1)
    for k in range(6):
        for p, q in zip(mine, twin):
            p.grad = torch.randn(p.shape, generator=gen, device="cuda") * (0.01 if k % 2 else 1.0)
            q.grad = p.grad.clone()
        norm = a.step()
        want = torch.nn.utils.clip_grad_norm_(twin, 1.0)
        b.step()
        assert abs(float(norm) - float(want)) <= 1e-6 * float(want)
        for p, q in zip(mine, twin):
            assert float((p - q).abs().max()) <= 1e-6 * (k + 1) * 4
    assert torch.equal(unused, torch.ones(4, device="cuda"))
    with pytest.raises(ValueError):
        gcn.ClippedAdam([{"params": mine}, {"params": [unused]}])


@pytest.mark.parametrize("max_norm", [None, 1.0])
def test_optimizer_counts_steps_for_each_parameter(gpu, max_norm):
    """Parameters whose gradients begin late or miss a step, against
    torch.optim.AdamW: fp32 rounding of the update is below 1e-6 a step at
    this rate, as in test_optimizer_follows_torch."""
    from tcc_amd import gcn

    gen = torch.Generator(device="cuda").manual_seed(3)
    sizes = ((30, 7), (11,), (64,), (5, 5))
    mine = [torch.nn.Parameter(torch.randn(s, generator=gen, device="cuda")) for s in sizes]
    twin = [torch.nn.Parameter(p.detach().clone()) for p in mine]
    a = gcn.ClippedAdam(mine, lr=0.02, weight_decay=0.1, max_norm=max_norm)
    b = torch.optim.AdamW(twin, lr=0.02, weight_decay=0.1)
    assert not a.state[mine[3]]  # a look at a state that is not there yet changes nothing
    for k in range(9):
        for i, (p, q) in enumerate(zip(mine, twin)):
            p.grad = q.grad = None
            if (i == 1 and k < 3) or (i == 2 and k % 3 == 1) or (i == 3 and k in (0, 5)):
                continue
            p.grad = torch.randn(p.shape, generator=gen, device="cuda")
            q.grad = p.grad.clone()
        norm = a.step()
        if max_norm is None:
            assert norm is None
        else:
            want = torch.nn.utils.clip_grad_norm_(twin, max_norm)
            assert abs(float(norm) - float(want)) <= 1e-6 * float(want)
        b.step()
        for p, q in zip(mine, twin):
            assert float((p - q).abs().max()) <= 1e-6 * (k + 1) * 4


@pytest.mark.parametrize("where", ["memory", "cpu"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_optimizer_resumes(gpu, dtype, where):
    """A run that goes on from a checkpoint has the bits of one that was not
    interrupted: moments in fp32, counts, parameters without a gradient so far."""
    import io

    from tcc_amd import gcn

    gen = torch.Generator(device="cuda").manual_seed(6)
    grads = [[(torch.randn(s, generator=gen, device="cuda") * 0.1).to(dtype) for s in ((40, 8), (9,), (3,))]
             for _ in range(6)]
    start = [torch.randn(g.shape, generator=gen, device="cuda").to(dtype) for g in grads[0]]

    def make(values):
        params = [torch.nn.Parameter(v.detach().clone()) for v in values]
        return params, gcn.ClippedAdam(params, lr=0.02, weight_decay=0.1, max_norm=0.5)

    def run(params, optimizer, steps):
        for k in steps:
            for i, p in enumerate(params):
                p.grad = None if i == 2 or (i == 1 and k == 0) else grads[k][i]  # the last one never, the second later
            optimizer.step()

    whole, one = make(start)
    run(whole, one, range(6))
    half, two = make(start)
    run(half, two, range(3))
    state = two.state_dict()
    if where == "cpu":
        buffer = io.BytesIO()
        torch.save(state, buffer)
        buffer.seek(0)
        state = torch.load(buffer, map_location="cpu", weights_only=True)
    rest, three = make(half)
    three.load_state_dict(state)
    run(half, two, range(3, 6))  # the checkpoint's own run goes on: nothing is shared with it
    run(rest, three, range(3, 6))
    for p, q, r in zip(whole, half, rest):
        assert torch.equal(p, q) and torch.equal(p, r)
        a, b = one.state[p], three.state[r]
        assert set(a) == set(b)
        for name in a:
            assert a[name].dtype == b[name].dtype and b[name].device == r.device and torch.equal(a[name], b[name])


def test_optimizer_takes_checkpoints_with_one_count(gpu):
    """The count of all parameters in their group, as it once was kept."""
    from tcc_amd import gcn

    p = torch.nn.Parameter(torch.ones(5, device="cuda"))
    q = torch.nn.Parameter(torch.ones(5, device="cuda"))
    a, b = gcn.ClippedAdam([p], lr=0.1), gcn.ClippedAdam([q], lr=0.1)
    p.grad = q.grad = torch.linspace(-1, 1, 5, device="cuda")
    for _ in range(3):
        a.step()
    state = a.state_dict()
    state["param_groups"][0]["step"] = state["state"][0].pop("step")
    b.load_state_dict(state)
    with torch.no_grad():
        q.copy_(p)
    assert int(b.state[q]["step"]) == 3 and "step" not in b.param_groups[0]
    state["state"][0]["step"] = state["param_groups"][0].pop("step")
    a.step()
    b.step()
    assert torch.equal(p, q)


def test_optimizer_returns_the_closures_loss(gpu):
    from tcc_amd import gcn

    p = torch.nn.Parameter(torch.full((4,), 3.0, device="cuda"))
    optimizer = gcn.ClippedAdam([p], max_norm=1.0)

    def closure():
        optimizer.zero_grad()
        loss = p.square().sum()
        loss.backward()
        return loss

    assert float(optimizer.step(closure)) == 36.0
    assert float(optimizer.norm) == 12.0  # sqrt(4 * 6^2)
    optimizer.zero_grad()
    p.sum().backward()
    norm = optimizer.step()
    assert float(norm) == 2.0 and norm is optimizer.norm


def test_autograd_sees_what_is_written_in_place(gpu):
    """A graph that saved a parameter refuses its backward pass once a step
    has changed it, as with torch's optimizers, and every tensor that a call
    writes has a new version (one that it only reads has not)."""
    from tcc_amd import gcn, training

    p = torch.nn.Parameter(torch.randn(6, device="cuda"))
    optimizer = gcn.ClippedAdam([p], max_norm=1.0)
    loss = (p * p).sum()
    loss.backward(retain_graph=True)
    optimizer.step()
    with pytest.raises(RuntimeError, match="inplace operation"):
        loss.backward()
    new = lambda *s: torch.rand(s, device="cuda")  # noqa: E731
    table, ids, room, grads, out = new(9, 4), torch.arange(3, device="cuda"), new(3, 4), [new(5), new(2, 2)], [new(5), new(2, 2)]
    moments = [new(5), new(2, 2)], [new(5), new(2, 2)]
    step = torch.zeros((), dtype=torch.int64, device="cuda")
    calls = [
        (lambda: training.embedding_lookup(table, ids, out=room), [room], [table, ids]),
        (lambda: training.embedding_grad(room, ids, 9, grad=table, accumulate=True), [table], [room, ids]),
        (lambda: training.clip_grad_norm(grads, 0.1, out=out), out, grads),
        (lambda: training.clip_grad_norm(grads, 0.1), grads, out),
        (lambda: training.adam_step(out, grads, *moments, step, max_norm=1.0), out + moments[0] + moments[1] + [step], grads),
    ]
    for call, written, read in calls:
        before = [t._version for t in written], [t._version for t in read]
        call()
        assert all(t._version > v for t, v in zip(written, before[0]))
        assert [t._version for t in read] == before[1]
    with torch.inference_mode():  # tensors without versions
        training.clip_grad_norm([new(5)], 0.1)


def test_example_trains(gpu):
    from tcc_amd import train_embeddings

    losses, norms, _ = train_embeddings.train(nodes=2000, graphs=60, mean_rows=30, dim=16, hidden=32, steps=30,
                                              log=lambda s: None)
    assert all(np.isfinite(losses)) and all(np.isfinite(norms))
    assert losses[-1] < 0.8 * losses[0]
