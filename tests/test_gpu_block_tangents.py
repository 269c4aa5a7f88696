"""Tangents of forward-mode differentiation are refused by the block-scaled casts and
products and by the gradients' norm and clipping: their results would come without one,
which reads as a derivative of zero."""
import pytest
import torch
from torch.autograd import forward_ad as fw

import mxfp8gg
from mxfp8gg import _lib

pytestmark = pytest.mark.gpu


def _inputs(gpu):
    g = torch.Generator().manual_seed(5)
    x = torch.randn((24, 144), generator=g).bfloat16().to(gpu)
    w = torch.randn((48, 144), generator=g).bfloat16().to(gpu)
    q, s = mxfp8gg.to_fp8_block_dim0(x)
    wq, ws = mxfp8gg.to_fp8_block_weight(w)
    xt, xs, _ = mxfp8gg.to_fp8_block_dim1(x)
    wt, wts, _ = mxfp8gg.to_fp8_block_dim1(w[:24].contiguous())
    return dict(x=x, w=w, q=q, s=s, wq=wq, ws=ws, xt=xt, xs=xs, wt=wt, wts=wts,
                g=x.float().contiguous())


CALLS = {  # the call, and the inputs that can carry a tangent
    "to_fp8_block_dim0": (lambda t: mxfp8gg.to_fp8_block_dim0(t["x"]), ["x"]),
    "to_fp8_block_dim1": (lambda t: mxfp8gg.to_fp8_block_dim1(t["x"])[:2], ["x"]),
    "to_fp8_block_weight": (lambda t: mxfp8gg.to_fp8_block_weight(t["w"], dual=True), ["w"]),
    "fp8_block_mm": (lambda t: [mxfp8gg.fp8_block_mm(t["q"], t["s"], t["wq"], t["ws"])], ["s", "ws"]),
    "fp8_block_wgrad": (lambda t: [mxfp8gg.fp8_block_wgrad(t["xt"], t["xs"], t["wt"], t["wts"])],
                        ["xs", "wts"]),
    "grad_norm": (lambda t: [mxfp8gg.grad_norm([t["w"], t["g"]])], ["g", "w"]),
    "clip_grad_norm_": (lambda t: [mxfp8gg.clip_grad_norm_([t["w"].clone(), t["g"]], 1e9)], ["g"]),
}


def _bytes(x):
    return x.detach().clone(memory_format=torch.contiguous_format).reshape(-1).view(torch.uint8)


def _same(a, b):
    return all(torch.equal(_bytes(x), _bytes(y)) for x, y in zip(a, b))


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("op", CALLS)
def test_tangents_are_refused(gpu, monkeypatch, op, native):
    _lib.load()
    if not native:
        monkeypatch.setattr(_lib, "_native", None)
    call, names = CALLS[op]
    t = _inputs(gpu)
    want = call(t)
    with fw.dual_level():
        assert _same(call(t), want)
        for name in names:
            dual = fw.make_dual(t[name], torch.ones_like(t[name]))
            for grad in (False, True):
                with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward-mode"):
                    call(dict(t, **{name: dual}))
    assert _same(call(t), want)
