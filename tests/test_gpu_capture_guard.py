"""A backward pass that is captured beside a living eager graph of the same
leaves is refused by the modules, however far behind their inputs these lie.
Only forward passes are captured here; the refusal comes before any backward."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def refused(call):
    with pytest.raises(RuntimeError, match="is alive"), torch.cuda.graph(torch.cuda.CUDAGraph()):
        call()


def small_model(norm, blocks=0):
    from tcc_amd import gcn
    from tcc_amd.train_embeddings import batch_of_graphs

    torch.manual_seed(2)
    rows, cols, ids, offsets, longest = batch_of_graphs(200, 5, 20, 1)
    n = ids.numel()
    return gcn.EmbeddingGCN(200, 16, 32, 6, norm=norm, blocks=blocks), gcn.LayerGraph(rows, cols, n, n), ids.cuda(), offsets.cuda(), longest


def test_leaves_behind_the_logits_are_seen(gpu):
    from tcc_amd import training

    leaf = torch.randn((8, 5), device="cuda", requires_grad=True)
    x = torch.randn((20, 8), device="cuda")
    held = training.held_by_default_stream
    y = torch.relu(x @ leaf) * 2
    assert held([y]) and held([None, x, y.view(10, 10)])
    assert not held([y.detach(), x, None])
    del y
    assert not held([leaf])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = torch.relu(x @ leaf) * 2
    torch.cuda.current_stream().wait_stream(side)
    assert not held([y]) and not held([leaf])


def test_logits_of_a_deep_graph(gpu):
    """As many nodes as a recursion could not hold, each an input of two others."""
    from tcc_amd import training

    leaf = torch.zeros(3, device="cuda", requires_grad=True)
    y = leaf
    for _ in range(30_000):
        y = y + y
    assert training.held_by_default_stream([y])


@pytest.mark.parametrize("norm", ["group", "layer"])
def test_a_models_step_beside_a_living_eager_one(gpu, norm):
    """Where the norms are frozen too: what the eager graph holds are the
    embedding's and the convolutions' leaves."""
    from tcc_amd import gcn, training

    model, graph, ids, offsets, longest = small_model(norm)
    model.norm.requires_grad_(False)
    teacher = training.top_logits(torch.randn((ids.numel(), 6), device="cuda"), 2)
    loss_fcn = gcn.DistillationLoss()
    logits = torch.randn((ids.numel(), 6), device="cuda")
    w = torch.randn((6, 6), device="cuda", requires_grad=True)
    loss = loss_fcn(logits @ w, teacher)  # eager
    refused(lambda: loss_fcn(logits @ w, teacher))
    del loss
    alive = model(graph, ids, offsets, longest)
    assert training.held_by_default_stream([alive])
    refused(lambda: loss_fcn(alive * 1.0, teacher))
    with torch.no_grad(), torch.cuda.graph(torch.cuda.CUDAGraph()):
        loss_fcn(alive * 1.0, teacher)  # nothing to differentiate


def test_a_norm_of_what_a_leaf_gave(gpu):
    """Of x and of the residual."""
    from tcc_amd import gcn

    norm = gcn.NodeLayerNorm(12)
    norm.requires_grad_(False)
    x = torch.randn((30, 12), device="cuda")
    w = torch.randn((12, 12), device="cuda", requires_grad=True)
    alive = x @ w
    refused(lambda: norm(x @ w))
    refused(lambda: norm(x, x @ w))
    del alive
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        norm(x @ w, x)
