"""The native host path (csrc/host.cpp) of the block-scaled products, the norms with
residual, the log probabilities and the gradient clipping, and their Python form: equal
bits, types, shapes and gradients, on another stream too; what has no derivative is
refused in both."""
import pytest
import torch
from torch.autograd import forward_ad as fw

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
        assert (x is None) == (y is None)
        if x is None:
            continue
        assert x.dtype == y.dtype and x.shape == y.shape and x.device == y.device
        assert x.requires_grad == y.requires_grad
        x, y = (v.detach().clone(memory_format=torch.contiguous_format) for v in (x, y))
        assert torch.equal(x.reshape(-1).view(torch.uint8), y.reshape(-1).view(torch.uint8))


def _rand(shape, seed, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(dtype).cuda()


@pytest.mark.parametrize("need", [(1, 1), (1, 0), (0, 1), (0, 0)])
@pytest.mark.parametrize("shape,groups", [((150, 256), 0), ((2, 3, 48), 0), ((48,), 0), ((0, 64), 0),
                                          ((300, 144), 3)])
def test_block_linear(gpu, monkeypatch, shape, groups, need):
    K, N = shape[-1], 80
    x0 = _rand(shape, 0)
    w0 = _rand((groups, N, K) if groups else (N, K), 1)
    offs = torch.tensor([100, 100, 250], dtype=torch.int32, device=gpu) if groups else None
    d = _rand((*shape[:-1], N), 2)

    def f():
        x, w = (t.clone().requires_grad_(bool(r)) for t, r in zip((x0, w0), need))
        y = mxfp8gg.fp8_block_linear(x, w, offs)
        if any(need):
            y.backward(d)
        with torch.no_grad():
            again = mxfp8gg.fp8_block_linear(x, w, offs)
        q, s = mxfp8gg.to_fp8_block_dim0(x0.view(-1, K))
        return y, x.grad, w.grad, again, q, s
    _same(*_both(monkeypatch, f))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("wtype", [None, torch.float32, torch.bfloat16])
@pytest.mark.parametrize("used", ["both", "y", "h"])
@pytest.mark.parametrize("shape", [(3, 50, 96), (64,), (0, 96)])
def test_add_rms_norm(gpu, monkeypatch, dtype, wtype, used, shape):
    x0, r0, dy, dh = (_rand(shape, i, dtype) for i in range(4))
    w0 = None if wtype is None else _rand(shape[-1:], 4, wtype)

    def f():
        x, r = x0.clone().requires_grad_(True), r0.clone().requires_grad_(True)
        w = None if w0 is None else w0.clone().requires_grad_(True)
        y, h = mxfp8gg.add_rms_norm(x, r, w)
        outs, grads = [y, h], [dy, dh]
        if used != "both":
            i = used == "h"
            outs, grads = outs[i:i + 1], grads[i:i + 1]
        torch.autograd.backward(outs, grads)
        with torch.no_grad():
            q = mxfp8gg.rms_norm_quant(x, w, r)
        return [y, h, x.grad, r.grad, None if w is None else w.grad, *q]
    _same(*_both(monkeypatch, f))


def test_add_rms_norm_of_one_tensor(gpu, monkeypatch):
    """x as its own residual, the one gradient in two places, and grads of a part."""
    x0, d = _rand((40, 128), 0), _rand((40, 128), 1)

    def f():
        x = x0.clone().requires_grad_(True)
        y, h = mxfp8gg.add_rms_norm(x, x)
        torch.autograd.backward([y, h], [d, d])
        a, b = x0.clone().requires_grad_(True), x0.clone().requires_grad_(True)
        mxfp8gg.add_rms_norm(a, b)[0].backward(d)
        a.grad += 1  # the two leaves own their gradients
        c = x0.clone().requires_grad_(True)
        mxfp8gg.add_rms_norm(c, x0)[0].backward(d)
        assert torch.equal(b.grad, c.grad) and torch.equal(a.grad, c.grad + 1)
        return x.grad, a.grad, b.grad, c.grad
    a, b = _both(monkeypatch, f)
    _same(a, b)


@pytest.mark.parametrize("itype", [torch.int32, torch.int64, None])
@pytest.mark.parametrize("topk", [0, 3])
@pytest.mark.parametrize("shape", [(20, 300), (2, 3, 70), (50,), (0, 50), (2, 40000)])
def test_token_log_probs(gpu, monkeypatch, itype, topk, shape):
    z0 = _rand(shape, 0, torch.float32)
    t = None
    if itype is not None:
        t = torch.randint(0, shape[-1], shape[:-1], device=gpu).to(itype)
        if t.dim():
            t.view(-1)[::3] = -100
    d = [_rand(shape[:-1], 1, torch.float32), _rand(shape[:-1], 2, torch.float32), None,
         _rand((*shape[:-1], topk), 3, torch.float32)]

    def f():
        out = []
        for use in ((0, 1, 3), (1,), (3,), (0,)):
            z = z0.clone().requires_grad_(True)
            r = mxfp8gg.token_log_probs(z, t, temperature=0.7, topk=topk)
            pairs = [(r[i], d[i]) for i in use if r[i] is not None]
            if not pairs:
                continue
            torch.autograd.backward(*map(list, zip(*pairs)))
            out += [*r, z.grad]
        with torch.no_grad():
            out += mxfp8gg.token_log_probs(z0, t, temperature=0.7, topk=topk)
        return out
    _same(*_both(monkeypatch, f))


def test_clip(gpu, monkeypatch):
    g0 = [_rand((33,), 0), _rand((64, 100), 1, torch.float32), _rand((5000,), 2)]

    def f():
        g = [t.clone() for t in g0]
        n = mxfp8gg.clip_grad_norm_(g, 1.5)
        return [n, mxfp8gg.grad_norm(g), *g]
    _same(*_both(monkeypatch, f))


def _step(x, r, w, wl, t):
    y, h = mxfp8gg.add_rms_norm(x, r, w)
    z = mxfp8gg.fp8_block_linear(y, wl) + h[:, :wl.shape[0]]
    p = mxfp8gg.token_log_probs(z, t, topk=2)
    return p.log_probs.sum() + 0.1 * p.entropy.sum() + 0.01 * p.top_log_probs.sum()


def test_backward_on_the_forward_stream(gpu, monkeypatch):
    """Forward on a side stream, backward called under another: autograd runs it where the
    forward ran, and the gradients are those of one stream."""
    x0, r, w, wl = _rand((2000, 512), 0), _rand((2000, 512), 1), _rand((512,), 2), _rand((256, 512), 3)
    t = torch.randint(0, 256, (2000,), device=gpu)

    def f(stream):
        x, l = x0.clone().requires_grad_(True), wl.clone().requires_grad_(True)
        with torch.cuda.stream(stream):
            stream.wait_stream(torch.cuda.default_stream())
            loss = _step(x, r, w, l, t)
        torch.cuda.default_stream().wait_stream(stream)
        loss.backward()
        torch.cuda.synchronize()
        return x.grad, l.grad
    want = f(torch.cuda.default_stream())
    a, b = _both(monkeypatch, lambda: f(torch.cuda.Stream()))
    _same(a, want)
    _same(b, want)


CALLS = {
    "fp8_block_linear": lambda x, w, t: mxfp8gg.fp8_block_linear(x, w),
    "add_rms_norm": lambda x, w, t: mxfp8gg.add_rms_norm(x, x.detach(), w[0])[0],
    "token_log_probs": lambda x, w, t: mxfp8gg.token_log_probs(x, t).log_probs,
}


def _inputs():
    return _rand((12, 64), 0), _rand((48, 64), 1), torch.arange(12, device="cuda")


@pytest.mark.parametrize("op", CALLS)
def test_second_derivatives_are_refused(gpu, monkeypatch, op):
    x0, w, t = _inputs()

    def f():
        x = x0.clone().requires_grad_(True)
        total = CALLS[op](x, w, t).float().sum() + x.float().pow(2).sum()
        with pytest.raises(RuntimeError, match=f"{op} cannot be differentiated twice"):
            torch.autograd.grad(total, x, create_graph=True, retain_graph=True)
        first = torch.autograd.grad(total, x, retain_graph=True)
        _same(first, torch.autograd.grad(total, x))
        return first
    _same(*_both(monkeypatch, f))


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("op", CALLS)
def test_tangents_are_refused(gpu, monkeypatch, op, native):
    if not native:
        _lib.load()
        monkeypatch.setattr(_lib, "_native", None)
    x, w, t = _inputs()
    want = CALLS[op](x, w, t)
    with fw.dual_level():
        assert torch.equal(CALLS[op](x, w, t), want)
        dx, dw = fw.make_dual(x, torch.ones_like(x)), fw.make_dual(w, torch.ones_like(w))
        for grad in (False, True):
            with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward-mode"):
                CALLS[op](dx, w, t)
        if op != "token_log_probs":
            with pytest.raises(RuntimeError, match="forward-mode"):
                CALLS[op](x, dw, t)


@pytest.mark.parametrize("native", [True, False])
def test_training_step_in_a_graph(gpu, monkeypatch, native):
    """Forward, backward and clipping captured: every replay, with eager work between,
    gives the eager results for the inputs of then."""
    if not native:
        _lib.load()
        monkeypatch.setattr(_lib, "_native", None)
    x0, r, w, wl = _rand((64, 256), 0), _rand((64, 256), 1), _rand((256,), 2), _rand((128, 256), 3)
    t = torch.randint(0, 128, (64,), device=gpu)
    x, wp, lp = (a.clone().requires_grad_(True) for a in (x0, w, wl))

    def step():
        grads = torch.autograd.grad(_step(x, r, wp, lp, t), (x, wp, lp))
        grads = [g.clone() for g in grads]
        return [mxfp8gg.clip_grad_norm_(grads, 0.5), *grads]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        with torch.no_grad():
            x.copy_(_rand((64, 256), 10 + i))
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        _same(out, want)
