"""Layer norms whose parameters take no gradient: nothing is summed for them."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def inputs(N=500, C=70):
    gen = torch.Generator(device="cuda").manual_seed(1)
    x, r, d = torch.randn((3, N, C), generator=gen, device="cuda")
    w, b = torch.rand((2, C), generator=gen, device="cuda") + 0.5
    return x, r, d, w, b


@pytest.mark.parametrize("C", [3, 70, 4000])
def test_the_input_s_gradient_alone(gpu, C):
    from tcc_amd import training

    x, r, d, w, b = inputs(300, C)
    _, h, mean, rstd = training.layer_norm(x, w, b, residual=r, activation="gelu")
    args = d, h, mean, rstd, w, b
    dx, dw, db = training.layer_norm_grad(*args, d_sum=r, activation="gelu", parameters=False)
    assert dw is None and db is None
    want = training.layer_norm_grad(*args, d_sum=r, activation="gelu")
    assert torch.equal(dx, want[0]) and want[1] is not None and want[2] is not None


@pytest.mark.parametrize("weight,bias", [(False, False), (True, False), (False, True), (True, True)])
def test_frozen_parameters_are_not_summed(gpu, monkeypatch, weight, bias):
    from tcc_amd import gcn, training

    x, r, d, w, b = inputs()
    x.requires_grad_()
    norm = gcn.NodeLayerNorm(70, "silu")
    with torch.no_grad():
        norm.weight.copy_(w)
        norm.bias.copy_(b)
    y, h = norm(x, r)
    want = torch.autograd.grad((y * d).sum() + h.sum(), (x, norm.weight, norm.bias))
    norm.weight.requires_grad_(weight)
    norm.bias.requires_grad_(bias)
    asked, plain = [], training.layer_norm_grad

    def grad(*args, **kwargs):
        out = plain(*args, **kwargs)
        asked.append((out[1] is not None, out[2] is not None))
        return out

    monkeypatch.setattr(training, "layer_norm_grad", grad)
    y, h = norm(x, r)
    ((y * d).sum() + h.sum()).backward()
    assert asked == [(weight or bias,) * 2]
    assert torch.equal(x.grad, want[0])
    for p, g, there in ((norm.weight, want[1], weight), (norm.bias, want[2], bias)):
        assert torch.equal(p.grad, g) if there else p.grad is None
