"""Inputs, weights and incoming gradients of any layout (expanded, transposed, overlapping,
sliced, of one row or none): the results and gradients of contiguous copies, in both host
forms."""
import pytest
import torch

import mxfp8gg
from mxfp8gg import _lib

pytestmark = pytest.mark.gpu


def _rand(shape, seed, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(dtype).cuda()


LAYOUTS = {
    "contiguous": lambda r, c, d: _rand((r, c), 1, d),
    "expanded": lambda r, c, d: _rand((1, c), 2, d).expand(r, c),
    "scalar": lambda r, c, d: _rand((1, 1), 3, d).expand(r, c),
    "transposed": lambda r, c, d: _rand((c, r), 4, d).t(),
    "sliced": lambda r, c, d: _rand((r, c + 24), 5, d)[:, 8:8 + c],
    "odd": lambda r, c, d: _rand((r, c + 3), 6, d)[:, 1:1 + c],
    "every other": lambda r, c, d: _rand((2 * r, c), 7, d)[::2],
    "overlapping": lambda r, c, d: _rand((r * 16 + c,), 8, d).as_strided((r, c), (16, 1)),
    "reversed": lambda r, c, d: _rand((r, c), 9, d).flip(0),
    "columns": lambda r, c, d: _rand((r, 2 * c), 10, d)[:, ::2],
}


def _run(f, tensors, grads):
    leaves = [t.detach().requires_grad_(True) for t in tensors]
    out = [o for o in f(*leaves) if o is not None]
    d = [o for o in out if o.requires_grad]
    got = torch.autograd.grad(d, leaves, grads[:len(d)])
    with torch.no_grad():
        plain = [o for o in f(*leaves) if o is not None]
    return [o.detach() for o in out] + list(got) + plain


def _same(a, b):
    assert len(a) == len(b)
    for x, y in zip(a, b):
        assert x.shape == y.shape and x.dtype == y.dtype
        assert torch.equal(x, y)


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("rows", [1, 33])
@pytest.mark.parametrize("layout", LAYOUTS)
def test_layouts(gpu, monkeypatch, native, rows, layout):
    if not native:
        _lib.load()
        monkeypatch.setattr(_lib, "_native", None)
    make, c = LAYOUTS[layout], 144
    copy = lambda t: t.clone(memory_format=torch.contiguous_format)  # noqa: E731
    x, r, dy = (make(rows, c, torch.bfloat16) for _ in range(3))
    w = _rand((2 * c,), 11, torch.float32)[::2]

    def norm(x, r, w):
        return mxfp8gg.add_rms_norm(x, r, w)
    _same(_run(norm, (x, r, w), [dy, dy]), _run(norm, (copy(x), copy(r), copy(w)), [copy(dy)] * 2))
    for fmt in ("fp8_block",):
        with torch.no_grad():
            a = mxfp8gg.rms_norm_quant(x, w, r, out_format=fmt)
            b = mxfp8gg.rms_norm_quant(copy(x), copy(w), copy(r), out_format=fmt)
        for p, q in zip(a, b):
            assert torch.equal(p.float(), q.float())

    wl, dl = make(80, c, torch.bfloat16), make(rows, 80, torch.bfloat16)

    def linear(x, w):
        return [mxfp8gg.fp8_block_linear(x, w)]
    _same(_run(linear, (x, wl), [dl]), _run(linear, (copy(x), copy(wl)), [copy(dl)]))
    q, s = mxfp8gg.to_fp8_block_dim0(x)
    p, t = mxfp8gg.to_fp8_block_dim0(copy(x))
    assert torch.equal(q.float(), p.float()) and torch.equal(s, t)

    target = torch.arange(2 * rows, device=gpu)[::2] % c
    up = [make(rows, 1, torch.float32)[:, 0], make(rows, 1, torch.float32)[:, 0],
          make(rows, 3, torch.float32)]

    def logp(z):
        o = mxfp8gg.token_log_probs(z, target, topk=3)
        return [o.log_probs, o.entropy, o.top_log_probs, o.top_ids]

    def plain(z):
        o = mxfp8gg.token_log_probs(z, copy(target), topk=3)
        return [o.log_probs, o.entropy, o.top_log_probs, o.top_ids]
    _same(_run(logp, (x,), up), _run(plain, (copy(x),), [copy(u) for u in up]))


@pytest.mark.parametrize("native", [True, False])
def test_sums_backward(gpu, monkeypatch, native):
    """Gradients that torch makes by expanding one number, through inputs that are used twice."""
    if not native:
        _lib.load()
        monkeypatch.setattr(_lib, "_native", None)
    x0, w0 = _rand((20, 64), 1), _rand((48, 64), 2)
    x, w = x0.clone().requires_grad_(True), w0.clone().requires_grad_(True)
    y, h = mxfp8gg.add_rms_norm(x, x)
    z = mxfp8gg.fp8_block_linear(y, w) + mxfp8gg.fp8_block_linear(h, w)
    mxfp8gg.token_log_probs(z, topk=2).top_log_probs.sum().backward()
    assert torch.isfinite(x.grad).all() and torch.isfinite(w.grad).all()
    y2, h2 = mxfp8gg.add_rms_norm(x0.clone().requires_grad_(True), x0)
    (y2.sum() + h2.sum()).backward()
    u = x0.clone().requires_grad_(True)
    mxfp8gg.fp8_block_linear(u, w0).sum().backward()
    one = torch.ones((20, 48), device=gpu, dtype=torch.bfloat16)
    v = x0.clone().requires_grad_(True)
    mxfp8gg.fp8_block_linear(v, w0).backward(one)
    assert torch.equal(u.grad, v.grad)
