"""Arguments of clip_grad_norm_ that could do harm or have no factor: the parameters in place
of their gradients; a bound of infinity or of zero."""
import pytest
import torch

import mxfp8gg
from mxfp8gg import _lib

pytestmark = pytest.mark.gpu


@pytest.fixture(params=[True, False], ids=["native", "python"])
def host(request, monkeypatch):
    _lib.load()
    if not request.param:
        monkeypatch.setattr(_lib, "_native", None)


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_parameters_are_refused(gpu, host, dtype, grad):
    """torch's function of the name takes parameters; here they would be scaled themselves."""
    model = torch.nn.Sequential(torch.nn.Linear(64, 32), torch.nn.Linear(32, 8)).to(gpu, dtype)
    model(torch.ones((4, 64), device=gpu, dtype=dtype)).float().square().sum().backward()
    before = [p.detach().clone() for p in model.parameters()]
    versions = [p._version for p in model.parameters()]
    grads = [p.grad for p in model.parameters()]
    with torch.set_grad_enabled(grad):
        for args in (model.parameters(), list(model.parameters()), [*grads, model[0].weight],
                     model[0].weight):
            with pytest.raises(ValueError, match="gradients"):
                mxfp8gg.clip_grad_norm_(args, 1e-3)
        for p, b, v in zip(model.parameters(), before, versions):
            assert torch.equal(p, b) and p._version == v
        norm = mxfp8gg.clip_grad_norm_(grads, 1e-3)
    assert float(norm) > 1e-3 and abs(float(mxfp8gg.grad_norm(grads)) - 1e-3) < 1e-5


def test_gradients_with_a_graph_are_clipped(gpu, host):
    """Under create_graph gradients require grad themselves, but are no leaves."""
    p = torch.nn.Parameter(torch.linspace(-2, 2, 500, device=gpu))
    p.square().sum().backward(create_graph=True)
    assert p.grad.requires_grad
    want = p.grad.detach().clone()
    norm = mxfp8gg.AdamW([p]).clip_grad_norm_(0.5)
    assert abs(float(norm) - float(want.norm())) < 1e-4
    assert torch.allclose(p.grad, want * (0.5 / float(want.norm())), rtol=1e-5, atol=0)
    p.grad = None


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("max_norm,eps,worst", [
    (float("inf"), 1e-6, 2.0), (float("inf"), 1e-6, float("inf")), (float("inf"), 0.0, 0.0),
    (float("inf"), 0.0, float("inf")), (float("inf"), float("inf"), 2.0), (0.0, 0.0, 0.0),
    (1.0, 0.0, 0.0), (0.0, 1e-6, 0.0)])
def test_nothing_to_clip(gpu, host, dtype, max_norm, eps, worst):
    """An infinite bound, whatever the norm, and gradients of zero, whatever the bound:
    the factors inf / inf and 0 / 0 do not exist, and nothing is written."""
    grads = [torch.zeros(5000, device=gpu, dtype=dtype), torch.zeros(3, device=gpu, dtype=dtype)]
    grads[1][1], grads[0][7] = worst, -0.0
    if worst:
        grads[0][100:200] = torch.linspace(-1, 1, 100)
    before = [g.clone() for g in grads]
    norm = mxfp8gg.clip_grad_norm_(grads, max_norm, eps)
    assert torch.equal(norm, mxfp8gg.grad_norm(before))
    for g, b in zip(grads, before):
        assert torch.equal(g.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("max_norm,eps,factor", [(0.0, 0.0, 0.0), (0.0, 1e-6, 0.0),
                                                 (2.0, float("inf"), 0.0), (2.5, 0.0, 0.5)])
def test_extreme_bounds_of_a_finite_norm(gpu, host, max_norm, eps, factor):
    g = torch.tensor([3.0, -4.0], device=gpu)
    assert float(mxfp8gg.clip_grad_norm_([g], max_norm, eps)) == 5.0
    assert g.tolist() == [3.0 * factor, -4.0 * factor]


def test_a_nan_stays_under_an_infinite_bound(gpu, host):
    g = [torch.ones(9, device=gpu), torch.ones(9, device=gpu, dtype=torch.bfloat16)]
    g[0][3] = float("nan")
    assert torch.isnan(mxfp8gg.clip_grad_norm_(g, float("inf")))
    assert all(torch.isnan(t).all() for t in g)
