"""Tangents that reach a backward pass (forward-mode differentiation of a gradient) are
refused by the operators that are differentiable once: their gradients would come without
one."""
import pytest
import torch
from torch.autograd import forward_ad as fw

import mxfp8gg
from mxfp8gg import _lib

pytestmark = pytest.mark.gpu

CALLS = {
    "fp8_block_linear": lambda x, w, t: mxfp8gg.fp8_block_linear(x, w),
    "add_rms_norm": lambda x, w, t: mxfp8gg.add_rms_norm(x, x.detach(), w[0])[0],
    "add_rms_norm, both": lambda x, w, t: torch.cat(mxfp8gg.add_rms_norm(x, x.detach(), w[0])),
    "token_log_probs": lambda x, w, t: mxfp8gg.token_log_probs(x, t).log_probs,
    "token_log_probs, entropy": lambda x, w, t: mxfp8gg.token_log_probs(x, t).entropy,
    "token_log_probs, top": lambda x, w, t: mxfp8gg.token_log_probs(x, t, topk=3).top_log_probs,
    "route_topk": lambda x, w, t: mxfp8gg.route_topk(x, 4)[1],
    "layer_norm": lambda x, w, t: mxfp8gg.layer_norm(x, w[0], w[1]),
    "rms_norm": lambda x, w, t: mxfp8gg.rms_norm(x, w[0]),
    "linear_cross_entropy": lambda x, w, t: mxfp8gg.linear_cross_entropy(x, w, t),
}


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("op", CALLS)
def test_tangents_of_incoming_gradients_are_refused(gpu, monkeypatch, op, native):
    _lib.load()
    if not native:
        monkeypatch.setattr(_lib, "_native", None)
    g = torch.Generator().manual_seed(9)
    x = torch.randn((12, 64), generator=g).bfloat16().to(gpu).requires_grad_(True)
    w = torch.randn((48, 64), generator=g).bfloat16().to(gpu)
    t = torch.arange(12, device=gpu)
    y = CALLS[op](x, w, t)
    d = torch.randn(y.shape, generator=g).to(gpu, y.dtype)
    want, = torch.autograd.grad(y, x, d, retain_graph=True)
    with fw.dual_level():
        got, = torch.autograd.grad(y, x, d, retain_graph=True)
        assert torch.equal(got, want) and fw.unpack_dual(got).tangent is None
        dual = fw.make_dual(d, torch.ones_like(d))
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(y, x, dual, retain_graph=True)
    assert torch.equal(torch.autograd.grad(y, x, d)[0], want)


@pytest.mark.parametrize("native", [True, False])
def test_the_sum_alone_passes_its_gradient_on(gpu, monkeypatch, native):
    """Where only h = x + residual was used, dx is dh itself, with its tangent."""
    _lib.load()
    if not native:
        monkeypatch.setattr(_lib, "_native", None)
    x = torch.linspace(-1, 1, 64, device=gpu).view(4, 16).requires_grad_(True)
    h = mxfp8gg.add_rms_norm(x, x.detach())[1]
    with fw.dual_level():
        dual = fw.make_dual(torch.ones_like(h), torch.full_like(h, 3.0))
        dx, = torch.autograd.grad(h, x, dual)
        assert torch.equal(fw.unpack_dual(dx).primal, torch.ones_like(x))
        assert torch.equal(fw.unpack_dual(dx).tangent, torch.full_like(x, 3.0))
