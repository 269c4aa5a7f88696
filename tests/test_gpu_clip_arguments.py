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
