"""linear_cross_entropy where targets are ignored: no token that counts leaves a mean
of NaN (0 / 0, as torch's) and gradients of exactly zero, whatever the gradient that
comes in.  The values are exact, so nothing here has a tolerance."""
import pytest
import torch

import mxfp8gg
from mxfp8gg import _lib

pytestmark = pytest.mark.gpu

# few tokens, a split product, small tiles, large tiles
SHAPES = [(1, 500, 64), (5, 20011, 256), (40, 300, 2048), (300, 700, 96), (300, 20000, 128)]


def _inputs(gpu, T, V, H):
    g = torch.Generator(device=gpu).manual_seed(T + V)
    x = torch.randn((T, H), generator=g, device=gpu).to(torch.bfloat16).requires_grad_(True)
    w = torch.randn((V, H), generator=g, device=gpu).to(torch.bfloat16).requires_grad_(True)
    return x, w, torch.randint(0, V, (T,), generator=g, device=gpu)


def _path(monkeypatch, native):
    if not native:
        _lib.load()
        monkeypatch.setattr(_lib, "_native", None)


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("T,V,H", SHAPES)
def test_every_token_ignored(gpu, monkeypatch, T, V, H, native):
    _path(monkeypatch, native)
    x, w, t = _inputs(gpu, T, V, H)
    t = torch.full_like(t, -100)
    for reduction in ("mean", "sum", "none"):
        for scale in (1.75, float("inf"), float("nan")):
            loss = mxfp8gg.linear_cross_entropy(x, w, t, reduction=reduction)
            up = torch.full_like(loss, scale)
            dx, dw = torch.autograd.grad(loss, (x, w), up)
            assert torch.isnan(loss) if reduction == "mean" else (loss == 0).all()
            assert (dx == 0).all() and (dw == 0).all(), (reduction, scale)
            only, = torch.autograd.grad(mxfp8gg.linear_cross_entropy(x.detach(), w, t,
                                                                     reduction=reduction), w, up)
            assert (only == 0).all()


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("T,V,H", SHAPES[1:] + [(16400, 70001, 72)])
def test_ignored_rows_of_a_gradient_that_is_not_finite(gpu, monkeypatch, T, V, H, native):
    """Also in vocabularies of several pieces; the rows that count are not finite."""
    _path(monkeypatch, native)
    x, w, t = _inputs(gpu, T, V, H)
    out = torch.rand(T, device=gpu) < 0.5
    out[0], out[-1] = True, False
    t[out] = -100
    for reduction in ("mean", "sum", "none"):
        for scale in (float("inf"), float("nan")):
            loss = mxfp8gg.linear_cross_entropy(x, w, t, reduction=reduction)
            dx, = torch.autograd.grad(loss, x, torch.full_like(loss, scale))
            assert (dx[out] == 0).all(), (reduction, scale)
            assert not torch.isfinite(dx[~out]).any(dim=1).all()
