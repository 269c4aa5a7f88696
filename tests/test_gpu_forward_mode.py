"""Forward-mode differentiation of route_topk, the norms and the loss is refused: a
result without its tangent would be a derivative of zero."""
import pytest
import torch
from torch.autograd import forward_ad as fw

import mxfp8gg
from mxfp8gg import _lib

pytestmark = pytest.mark.gpu


def _call(op, x, w, t):
    if op == "route_topk":
        return mxfp8gg.route_topk(x, 4)[1]
    if op == "layer_norm":
        return mxfp8gg.layer_norm(x, w[0], w[1])
    if op == "rms_norm":
        return mxfp8gg.rms_norm(x, w[0])
    return mxfp8gg.linear_cross_entropy(x, w, t)


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("op", ["route_topk", "layer_norm", "rms_norm", "linear_cross_entropy"])
def test_tangents_are_refused(gpu, monkeypatch, op, native):
    if not native:
        _lib.load()
        monkeypatch.setattr(_lib, "_native", None)
    g = torch.Generator().manual_seed(3)
    x = torch.randn((12, 64), generator=g).bfloat16().to(gpu)
    w = torch.randn((40, 64), generator=g).bfloat16().to(gpu)
    t = torch.randint(0, 40, (12,), generator=g).to(gpu)
    want = _call(op, x, w, t)
    with fw.dual_level():
        assert torch.equal(_call(op, x, w, t), want)
        dx, dw = fw.make_dual(x, torch.ones_like(x)), fw.make_dual(w, torch.ones_like(w))
        for grad in (False, True):
            with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward-mode"):
                _call(op, dx, w, t)
        if op != "route_topk":
            with pytest.raises(RuntimeError, match="forward-mode"):
                _call(op, x, dw, t)

        class Own(torch.autograd.Function):
            """Brings its own tangent: inside it forward mode is off."""

            @staticmethod
            def forward(ctx, x):
                return _call(op, x, w, t)

            @staticmethod
            def jvp(ctx, dx):
                return torch.ones_like(want)

        assert torch.equal(fw.unpack_dual(Own.apply(dx)).primal, want)
