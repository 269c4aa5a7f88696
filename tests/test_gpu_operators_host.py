"""The native host path of route_topk, the norms, the loss and adamw_step
(csrc/host.cpp) and their Python form call the same kernels with the same
arguments: equal bits, types, shapes and gradients, also on another stream and
through autograd's own accumulation."""
import pytest
import torch

import mxfp8gg
from mxfp8gg import _lib

pytestmark = pytest.mark.gpu


def _both(monkeypatch, f):
    """f() on the native path and on the Python form."""
    _lib.load()
    if _lib.native() is None:
        pytest.skip("the host module is not built")
    a = f()
    with monkeypatch.context() as m:
        m.setattr(_lib, "_native", None)
        assert _lib.native() is None
        b = f()
    return a, b


def _same(a, b):
    assert len(a) == len(b)
    for x, y in zip(a, b):
        assert x.dtype == y.dtype and x.shape == y.shape and x.device == y.device
        assert torch.equal(x.reshape(-1).view(torch.uint8), y.reshape(-1).view(torch.uint8))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("score,renorm", [("softmax", True), ("softmax", False),
                                          ("sigmoid", True)])
def test_route_topk(gpu, monkeypatch, dtype, score, renorm):
    g = torch.Generator().manual_seed(0)
    x0 = torch.randn((200, 64), generator=g).to(dtype).to(gpu)
    bias = (torch.randn(64, generator=g) * 0.1).to(gpu) if score == "sigmoid" else None
    d = torch.randn((200, 6), generator=g).to(gpu)

    def f():
        x = x0.clone().requires_grad_(True)
        idx, w = mxfp8gg.route_topk(x, 6, score=score, bias=bias, num_groups=4, top_groups=2,
                                    renormalize=renorm, scale=1.5)
        assert not idx.requires_grad and w.requires_grad
        (w * d).sum().backward()
        with torch.no_grad():
            i2, w2 = mxfp8gg.route_topk(x, 6, score=score, bias=bias, num_groups=4, top_groups=2,
                                        renormalize=renorm, scale=1.5)
        assert not w2.requires_grad
        return idx, w.detach(), x.grad, i2, w2
    _same(*_both(monkeypatch, f))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("wtype", [None, torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(3, 50, 77), (150, 4096), (9,)])
def test_norms(gpu, monkeypatch, dtype, wtype, shape):
    g = torch.Generator().manual_seed(1)
    x0 = torch.randn(shape, generator=g).to(dtype).to(gpu)
    d = torch.randn(shape, generator=g).to(dtype).to(gpu)
    p0 = [None if wtype is None else torch.randn(shape[-1], generator=g).to(wtype).to(gpu)
          for _ in range(2)]

    def f():
        x = x0.clone().requires_grad_(True)
        w, b = (None if p is None else p.clone().requires_grad_(True) for p in p0)
        y, z = mxfp8gg.layer_norm(x, w, b), mxfp8gg.rms_norm(x, w)
        torch.autograd.backward([y, z], [d, d])
        return [y.detach(), z.detach()] + [t.grad for t in (x, w, b) if t is not None]
    _same(*_both(monkeypatch, f))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("master", [True, False])
def test_adamw(gpu, monkeypatch, bits, master):
    g = torch.Generator().manual_seed(2)
    sizes = [(33,), (64, 100), (5000,), (1,)]
    p0 = [torch.randn(s, generator=g).to(torch.bfloat16).to(gpu) for s in sizes]
    g0 = [torch.randn(s, generator=g).to(gpu) for s in sizes]

    def f():
        params, masters = [p.clone() for p in p0], [p.float() for p in p0] if master else None
        states = [[mxfp8gg.adamw_state(p, bits) for p in p0] for _ in range(2)]
        flat = [t for s in states for e in s for t in (e if bits == 8 else (e,))]
        for step in (1, 2):
            old = [t._version for t in params + flat + (masters or [])]
            mxfp8gg.adamw_step(params, g0, *states, step=step, masters=masters)
            assert all(t._version > v for t, v in zip(params + flat + (masters or []), old))
        return params + flat + (masters or [])
    _same(*_both(monkeypatch, f))


@pytest.mark.parametrize("shape,itype", [((70,), torch.int64), ((2, 35), torch.int32)])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_linear_cross_entropy(gpu, monkeypatch, shape, itype, reduction):
    g = torch.Generator().manual_seed(3)
    x0 = torch.randn((*shape, 64), generator=g).to(torch.bfloat16).to(gpu)
    w0 = (torch.randn((300, 64), generator=g) / 8).to(torch.bfloat16).to(gpu)
    t = torch.randint(0, 300, shape, generator=g).to(itype).to(gpu)
    t.view(-1)[::5] = -100
    d = torch.randn(shape if reduction == "none" else (), generator=g).to(gpu)

    def f():
        x, w = (p.clone().requires_grad_(True) for p in (x0, w0))
        loss = mxfp8gg.linear_cross_entropy(x, w, t, reduction=reduction)
        loss.backward(d)
        only = w0.clone().requires_grad_(True)
        mxfp8gg.linear_cross_entropy(x0, only, t, reduction=reduction).backward(d)
        with torch.no_grad():
            again = mxfp8gg.linear_cross_entropy(x, w, t, reduction=reduction)
        return loss.detach(), x.grad, w.grad, only.grad, again
    _same(*_both(monkeypatch, f))


def test_backward_on_the_forward_stream(gpu, monkeypatch):
    """Forward on a side stream, backward called under another: autograd runs it
    where the forward ran, and the gradients are those of one stream."""
    x0 = torch.randn((4000, 512), device=gpu)
    w = torch.randn(512, device=gpu)

    def f(stream):
        x = x0.clone().requires_grad_(True)
        with torch.cuda.stream(stream):
            stream.wait_stream(torch.cuda.default_stream())
            s = mxfp8gg.route_topk(mxfp8gg.layer_norm(x, w), 4)[1]
            loss = (s * s).sum()
        torch.cuda.default_stream().wait_stream(stream)
        loss.backward()
        torch.cuda.synchronize()
        return x.grad
    want = f(torch.cuda.default_stream())
    a, b = _both(monkeypatch, lambda: [f(torch.cuda.Stream())])
    _same(a, [want])
    _same(b, [want])


@pytest.mark.parametrize("op", ["route_topk", "norm", "linear_cross_entropy"])
def test_second_derivatives_are_refused(gpu, monkeypatch, op):
    """create_graph would leave these operators' part of a second derivative out: it is
    refused, and the same graph still gives its first derivative."""
    g = torch.Generator().manual_seed(3)
    x0 = torch.randn((12, 64), generator=g).bfloat16().to(gpu)
    w0 = torch.randn((40, 64), generator=g).bfloat16().to(gpu)
    t = torch.randint(0, 40, (12,), generator=g).to(gpu)

    def f():
        x = x0.clone().requires_grad_(True)
        if op == "route_topk":
            y = mxfp8gg.route_topk(x, 4)[1]
        elif op == "norm":
            y = mxfp8gg.rms_norm(x)
        else:
            y = mxfp8gg.linear_cross_entropy(x, w0, t)
        total = y.float().sum() + x.float().pow(2).sum()
        with pytest.raises(RuntimeError, match=f"{op} cannot be differentiated twice"):
            torch.autograd.grad(total, x, create_graph=True, retain_graph=True)
        return torch.autograd.grad(total, x)
    _same(*_both(monkeypatch, f))
