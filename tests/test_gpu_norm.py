"""GPU parity of layer_norm and rms_norm with the 64-bit oracle.

Bounds, from the operations: statistics are fp32 sums of cols terms over 64 to
512 lanes of at most 64 terms each, so their relative error is below 80 units
of 2^-24 (5e-6); xhat, y and dx are a few products of them.  fp32 outputs: 2e-5
of the row's largest magnitude plus, where the mean is far above the deviation,
2^-22 of mean / deviation (the input's own cancellation).  bf16 outputs: half a
unit more, 2^-8 relative.  dweight and dbias add `rows` such terms: 2e-5 of the
sum of their magnitudes.
"""
import numpy as np
import pytest
import torch

import mxfp8gg
from tests import _operators_oracle as R

pytestmark = pytest.mark.gpu

SHAPES = [(1, 1), (1, 7168), (3, 2), (5, 7), (64, 64), (17, 65), (130, 257), (7, 1001), (33, 1024),
          (3, 4100), (600, 96), (9, 8192), (4, 8200), (3, 16384), (2, 16391), (2, 32768),
          (2, 32767), (1500, 33)]


def _wide(t):
    return None if t is None else t.detach().cpu().double().numpy()


def _inputs(gpu, rows, cols, dtype, affine, center, seed, pdtype=torch.float32, mean=0.3):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn((rows, cols), generator=g) * 1.7 + mean).to(dtype).to(gpu)
    dy = torch.randn((rows, cols), generator=g).to(dtype).to(gpu)
    w = b = None
    if affine:
        w = (1 + 0.2 * torch.randn(cols, generator=g)).to(pdtype).to(gpu)
        b = torch.randn(cols, generator=g).to(pdtype).to(gpu) if center else None
    return x, dy, w, b


def _near(got, want, bound, dtype):
    got = _wide(got)
    assert got.shape == want.shape
    if dtype is torch.bfloat16:
        bound = bound + 2.0 ** -8 * np.abs(want)
    bad = np.abs(got - want) > bound
    assert not bad.any(), (np.argwhere(bad)[0], got[bad][0], want[bad][0])


def _check(x, dy, w, b, center, eps):
    leaves = [t.detach().requires_grad_(True) if t is not None else None for t in (x, w, b)]
    call = (lambda: mxfp8gg.layer_norm(*leaves, eps=eps)) if center else \
        (lambda: mxfp8gg.rms_norm(leaves[0], leaves[1], eps=eps))
    y = call()
    with torch.no_grad():
        assert torch.equal(call(), y)                     # without autograd: the same bits
    assert y.dtype == x.dtype
    X, DY, W, B = map(_wide, (x, dy, w, b))
    ry, xhat, r = R.norm(X, W, B, eps, center)
    mu = np.abs(X.mean(axis=-1, keepdims=True)) if center else 0.0
    ill = 1 + 2.0 ** -22 / 2e-5 * mu * r
    top = lambda a: np.abs(a).max(axis=-1, keepdims=True)  # noqa: E731
    wide_w = 1.0 if W is None else np.abs(W).max()
    _near(y, ry, 2e-5 * ill * (top(xhat) * wide_w + (0 if B is None else np.abs(B))), x.dtype)
    names = [t for t in leaves if t is not None]
    grads = torch.autograd.grad(y, names, dy)
    dx, dw, db = R.norm_grad(DY, X, W, eps, center)
    _near(grads[0], dx, 2e-5 * ill * r * wide_w * top(DY) * (2 + top(xhat)), x.dtype)
    if w is not None:
        assert grads[1].dtype == w.dtype
        _near(grads[1], dw, 2e-5 * (np.abs(DY) * ill * (np.abs(xhat) + 1)).sum(axis=0), w.dtype)
    if b is not None:
        _near(grads[2], db, 2e-5 * np.abs(DY).sum(axis=0), b.dtype)
    again = torch.autograd.grad(call(), names, dy)
    assert all(torch.equal(p, q) for p, q in zip(grads, again))   # no order that changes


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("center", [True, False])
def test_matches_oracle(gpu, rows, cols, dtype, center):
    for affine in (True, False):
        _check(*_inputs(gpu, rows, cols, dtype, affine, center, rows + cols), center, 1e-5)


@pytest.mark.parametrize("pdtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_parameter_types(gpu, pdtype, dtype):
    _check(*_inputs(gpu, 40, 130, dtype, True, True, 1, pdtype), True, 1e-3)


def test_mean_far_above_deviation(gpu):
    _check(*_inputs(gpu, 20, 3000, torch.float32, True, True, 2, mean=500.0), True, 1e-5)


def test_constant_zero_and_non_finite_rows(gpu):
    x = torch.zeros((5, 96), device=gpu)
    x[1] = 3.0
    x[2, 5] = float("inf")
    x[3, 7] = float("nan")
    x[4] = torch.arange(96.0)
    y = mxfp8gg.layer_norm(x)
    assert (y[:2] == 0).all() and torch.isnan(y[2:4]).all() and torch.isfinite(y[4]).all()
    y = mxfp8gg.rms_norm(x)
    assert (y[0] == 0).all() and torch.isfinite(y[1]).all() and torch.isnan(y[2, 5])
    assert (y[2, :5] == 0).all() and torch.isnan(y[3]).all()


def test_many_rows_reduce_the_weight_gradient(gpu):
    # more rows than workgroups, fewer, and none
    for rows in (70001, 3, 0):
        x, dy, w, b = _inputs(gpu, rows, 40, torch.float32, True, True, 5)
        leaves = [t.requires_grad_(True) for t in (x, w, b)]
        dx, dw, db = torch.autograd.grad(mxfp8gg.layer_norm(*leaves), leaves, dy)
        if rows == 0:
            assert dx.shape == x.shape and (dw == 0).all() and (db == 0).all()
            continue
        _, xhat, _ = R.norm(_wide(x))
        np.testing.assert_allclose(_wide(dw), (_wide(dy) * xhat).sum(0), rtol=0,
                                   atol=2e-5 * np.abs(_wide(dy) * xhat).sum(0).max())
        np.testing.assert_allclose(_wide(db), _wide(dy).sum(0), rtol=0,
                                   atol=2e-5 * np.abs(_wide(dy)).sum(0).max())


def test_only_some_gradients(gpu):
    x, dy, w, b = _inputs(gpu, 50, 300, torch.bfloat16, True, True, 6)
    full = torch.autograd.grad(
        mxfp8gg.layer_norm(*(t.requires_grad_(True) for t in (x, w, b))), (x, w, b), dy)
    for keep in range(3):
        t = [p.detach().requires_grad_(i == keep) for i, p in enumerate((x, w, b))]
        g, = torch.autograd.grad(mxfp8gg.layer_norm(*t), t[keep], dy)
        assert torch.equal(g, full[keep])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layouts(gpu, dtype):
    big = torch.randn((2, 30, 200), generator=torch.Generator().manual_seed(0)).to(dtype).to(gpu)
    w = torch.randn(77, device=gpu)
    for v in (big[:, :, 13:90], big[:, ::2, 1:78], big.transpose(0, 1)[:, :, 100:177],
              big.transpose(1, 2)[:, :77].transpose(1, 2)):
        assert torch.equal(mxfp8gg.rms_norm(v, w), mxfp8gg.rms_norm(v.contiguous(), w))
    # gradients that arrive broadcast, transposed and in another type
    x = big[:, :, :77].reshape(60, 77).requires_grad_(True)
    y = mxfp8gg.layer_norm(x, w)
    one, = torch.autograd.grad(y.sum(), x, retain_graph=True)
    two, = torch.autograd.grad(y, x, torch.ones_like(y), retain_graph=True)
    row = torch.randn(77, device=gpu).to(dtype)
    three, = torch.autograd.grad(y, x, row.expand(60, 77), retain_graph=True)
    four, = torch.autograd.grad(y, x, row.expand(60, 77).contiguous().t().contiguous().t())
    assert torch.equal(one, two) and torch.equal(three, four)


def test_gradient_matches_differences(gpu):
    """Central differences of the kernel's fp32 forward, step 2^-6: truncation
    2^-12 / 6 of a third derivative below 8, rounding 2^-22 / 2^-6 per output:
    1e-3 of |dy| |direction| covers both."""
    x, dy, w, b = _inputs(gpu, 25, 48, torch.float32, True, True, 7)
    d = torch.randn(x.shape, generator=torch.Generator().manual_seed(1)).to(gpu) / 48 ** 0.5
    step = 2.0 ** -6
    for f in (lambda z: mxfp8gg.layer_norm(z, w, b), lambda z: mxfp8gg.rms_norm(z, w)):
        want = ((f(x + step * d).double() - f(x - step * d).double()) / (2 * step) * dy).sum(1)
        z = x.clone().requires_grad_(True)
        dx, = torch.autograd.grad(f(z), z, dy)
        got = (dx.double() * d).sum(1)
        assert (got - want).abs().max() <= 1e-3 * float(dy.norm(dim=1).max() * d.norm(dim=1).max())


def test_refusals(gpu):
    x = torch.zeros((4, 16), device=gpu)
    with pytest.raises(TypeError):
        mxfp8gg.layer_norm(x.half())
    with pytest.raises(TypeError):
        mxfp8gg.layer_norm(x, torch.zeros(16, device=gpu, dtype=torch.float16))
    for bad in (dict(weight=torch.zeros(15, device=gpu)), dict(bias=torch.zeros((1, 16), device=gpu)),
                dict(weight=torch.zeros(16))):
        with pytest.raises(ValueError):
            mxfp8gg.layer_norm(x, **bad)
    with pytest.raises(ValueError):
        mxfp8gg.layer_norm(torch.zeros((1, 32769), device=gpu))
    with pytest.raises(ValueError):
        mxfp8gg.rms_norm(torch.zeros((3, 0), device=gpu))
    with pytest.raises(ValueError):
        mxfp8gg.rms_norm(x.cpu())
