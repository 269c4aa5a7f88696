"""GPU parity of linear_cross_entropy with the 64-bit oracle.

Bounds: a logit is an fp32 sum of hidden products of bf16 values, off by at most
hidden * 2^-24 of the sum of their magnitudes (the matrix cores add in blocks, so
this is generous); a token's loss by that at two words and a few units of 2^-22
of its value.  A gradient is a sum over words (or tokens) of d times a bf16
value: d is rounded to bf16 (2^-9 on average, 2^-8 at most, of |d|) and moved
by the logits' error, both bounded by 2^-8 + 4 * the logit error of the sum of
the terms' magnitudes; the result is rounded to bf16, 2^-8 of it.
"""
import numpy as np
import pytest
import torch

import mxfp8gg
from tests import _operators_oracle as R

pytestmark = pytest.mark.gpu

SHAPES = [  # tokens, vocab, hidden
    (1, 1, 8), (1, 1000, 64), (5, 255, 72), (37, 257, 128), (256, 256, 64), (257, 513, 200),
    (130, 4099, 1032), (600, 700, 96), (3, 20011, 256), (1025, 300, 64), (64, 2048, 2048)]


def _inputs(gpu, T, V, H, seed, ignored=True, itype=torch.int64, scale=1.5):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((T, H), generator=g).to(torch.bfloat16).to(gpu)
    w = (torch.randn((V, H), generator=g) * scale / H ** 0.5).to(torch.bfloat16).to(gpu)
    t = torch.randint(0, V, (T,), generator=g).to(itype)
    if ignored and T > 2:
        t[torch.rand(T, generator=g) < 0.3] = -100
        t[0], t[-1] = V - 1, 0
    return x, w, t.to(gpu)


def _wide(t):
    return t.detach().cpu().double().numpy()


def _logit_error(x, w):
    return x.shape[1] * 2.0 ** -24 * (np.abs(x) @ np.abs(w).T).max()


def _near_bf16(got, want, bound):
    got = _wide(got)
    bad = np.abs(got - want) > bound + 2.0 ** -8 * np.abs(want)
    assert not bad.any(), (np.argwhere(bad)[0], got[bad][0], want[bad][0])


def _check(x, w, t, reduction, dloss=None):
    X, W, T = _wide(x), _wide(w), t.cpu().numpy().astype(np.int64)
    ref, d = R.linear_cross_entropy(X, W, T)
    n = max(1, int((T != -100).sum()))
    err = 2 * _logit_error(X, W)
    leaves = [x.detach().requires_grad_(True), w.detach().requires_grad_(True)]
    loss = mxfp8gg.linear_cross_entropy(*leaves, t, reduction=reduction)
    assert loss.dtype == torch.float32
    with torch.no_grad():
        assert torch.equal(mxfp8gg.linear_cross_entropy(x, w, t, reduction=reduction), loss)
    if reduction == "none":
        assert loss.shape == t.shape
        assert (np.abs(_wide(loss) - ref) <= err + 2.0 ** -20 * (1 + np.abs(ref))).all()
        assert (_wide(loss)[T == -100] == 0).all()
        g = _wide(dloss)
        d = d * g[:, None]
    else:
        assert loss.dim() == 0
        want = ref.sum() / (n if reduction == "mean" else 1)
        slack = (err + 2.0 ** -20 * (1 + np.abs(ref).max())) * (1 if reduction == "mean" else n)
        assert abs(float(loss.detach()) - want) <= slack + 2.0 ** -20 * abs(want)
        d = d * (1.75 / (n if reduction == "mean" else 1))
        dloss = torch.tensor(1.75, device=x.device)
    dx, dw = torch.autograd.grad(loss, leaves, dloss, retain_graph=True)
    assert dx.dtype == dw.dtype == torch.bfloat16
    rel = 2.0 ** -8 + 4 * _logit_error(X, W)
    _near_bf16(dx, d @ W, rel * (np.abs(d) @ np.abs(W)))
    _near_bf16(dw, d.T @ X, rel * (np.abs(d).T @ np.abs(X)))
    again = torch.autograd.grad(loss, leaves, dloss)
    assert torch.equal(again[0], dx) and torch.equal(again[1], dw)
    return dx, dw


@pytest.mark.parametrize("T,V,H", SHAPES)
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_matches_oracle(gpu, T, V, H, reduction):
    x, w, t = _inputs(gpu, T, V, H, T + V, itype=torch.int32 if T % 2 else torch.int64)
    dl = torch.randn(T, generator=torch.Generator().manual_seed(1)).to(gpu)
    _check(x, w, t, reduction, dl)


@pytest.mark.parametrize("T,V,H", [
    (1, 64, 8), (2, 70100, 40), (16, 8191, 520), (17, 30000, 72), (32, 65, 1000), (33, 129, 2056),
    (48, 5000, 136), (64, 16384, 24), (64, 4097, 264)])
def test_few_tokens(gpu, T, V, H):
    """Workgroups with one tile of words and with several, vocabularies that end
    inside one, contractions that end inside a stage and that some waves have no part
    of, one to four blocks of tokens; strided rows give the same bits."""
    x, w, t = _inputs(gpu, T, V, H, 7 * T + V)
    _check(x, w, t, "none", torch.randn(T, generator=torch.Generator().manual_seed(2)).to(gpu))
    ref = mxfp8gg.linear_cross_entropy(x, w, t)
    xs, ws = (torch.full((len(m), H + 24), float("nan"), dtype=m.dtype, device=gpu) for m in (x, w))
    xs[:, :H], ws[:, :H] = x, w
    assert torch.equal(mxfp8gg.linear_cross_entropy(xs[:, :H], ws[:, :H], t), ref)


def test_many_pieces(gpu):
    """Long rows, and a vocabulary of several pieces (of 1 GiB of 2 T bytes a
    word: three), the last one shorter; tokens and words past a tile."""
    for T, V, H in ((1000, 33000, 32768), (4100, 70001, 72), (16400, 70001, 72)):
        _large(gpu, T, V, H)


def _large(gpu, T, V, H):
    g = torch.Generator(device=gpu).manual_seed(2)
    x = torch.randn((T, H), generator=g, device=gpu).to(torch.bfloat16)
    w = (torch.randn((V, H), generator=g, device=gpu) / H ** 0.5).to(torch.bfloat16)
    t = torch.randint(0, V, (T,), generator=g, device=gpu)
    x.requires_grad_(True), w.requires_grad_(True)
    loss = mxfp8gg.linear_cross_entropy(x, w, t)
    dx, dw = torch.autograd.grad(loss, (x, w))
    z = x.detach().double() @ w.detach().double().t()
    lse = torch.logsumexp(z, dim=1)
    want = (lse - z.gather(1, t[:, None])[:, 0]).mean()
    assert abs(float(loss.detach()) - float(want)) <= 1e-4
    d = (z - lse[:, None]).exp_()
    d.scatter_add_(1, t[:, None], -torch.ones((T, 1), device=gpu, dtype=torch.float64))
    d /= T
    rel = 2.0 ** -8 + 1e-4
    for got, a, b in ((dx, d, w), (dw, d.t(), x)):
        b = b.detach().double()
        ref, size = a @ b, a.abs() @ b.abs()
        assert ((got.double() - ref).abs() <= rel * size + 2.0 ** -8 * ref.abs()).all()


def test_large_logits_do_not_overflow(gpu):
    x, w, t = _inputs(gpu, 50, 300, 64, 3, scale=400.0)
    loss = mxfp8gg.linear_cross_entropy(x, w, t, reduction="none")
    ref, _ = R.linear_cross_entropy(_wide(x), _wide(w), t.cpu().numpy())
    assert ref.max() > 1000
    np.testing.assert_allclose(_wide(loss), ref, rtol=1e-5, atol=2 * _logit_error(_wide(x), _wide(w)))


def test_ignored_and_invalid_targets(gpu):
    x, w, t = _inputs(gpu, 20, 100, 64, 4, ignored=False)
    leaves = (x.requires_grad_(True), w.requires_grad_(True))
    none = torch.full_like(t, -100)
    loss = mxfp8gg.linear_cross_entropy(x, w, none)
    assert torch.isnan(loss)                               # as torch's mean of nothing
    assert mxfp8gg.linear_cross_entropy(x, w, none, reduction="sum") == 0
    dx, dw = torch.autograd.grad(mxfp8gg.linear_cross_entropy(x, w, none, reduction="sum"), leaves)
    assert (dx == 0).all() and (dw == 0).all()
    # an ignored word of the vocabulary, and an ignored token that is not finite
    y = x.detach().clone()
    y[3] = float("nan")
    s = t.clone()
    s[3] = 7
    s[5] = 7
    y.requires_grad_(True)
    loss = mxfp8gg.linear_cross_entropy(y, w, s, ignore_index=7)
    dy, dw = torch.autograd.grad(loss, (y, w))
    assert torch.isfinite(loss) and (dy[[3, 5]] == 0).all() and torch.isfinite(dy).all()
    for bad in (100, 10 ** 6, -1):
        u = t.clone()
        u[2] = bad
        loss = mxfp8gg.linear_cross_entropy(x, w, u, reduction="none")
        assert torch.isnan(loss[2]) and torch.isfinite(loss[torch.arange(20) != 2]).all()


def test_only_one_gradient(gpu):
    x, w, t = _inputs(gpu, 300, 600, 128, 5)
    dx, dw = _check(x, w, t, "mean")
    for keep in range(2):
        a, b = x.detach().requires_grad_(keep == 0), w.detach().requires_grad_(keep == 1)
        g, = torch.autograd.grad(mxfp8gg.linear_cross_entropy(a, b, t), (a, b)[keep],
                                 torch.tensor(1.75, device=gpu))
        assert torch.equal(g, (dx, dw)[keep])


def test_layouts_and_leading_dimensions(gpu):
    x, w, t = _inputs(gpu, 60, 300, 64, 6)
    want = mxfp8gg.linear_cross_entropy(x, w, t, reduction="none")
    wide = torch.zeros((60, 200), dtype=torch.bfloat16, device=gpu)
    for off in (64, 8, 3):                                 # 3: rows off the 16-byte grid
        wide[:, off:off + 64] = x
        assert torch.equal(mxfp8gg.linear_cross_entropy(wide[:, off:off + 64], w, t,
                                                        reduction="none"), want)
    got = mxfp8gg.linear_cross_entropy(x.view(6, 10, 64), w.t().contiguous().t(), t.view(6, 10),
                                       reduction="none")
    assert torch.equal(got, want.view(6, 10))
    one = mxfp8gg.linear_cross_entropy(x[0].expand(4, 64), w, t[:1].expand(4), reduction="none")
    assert torch.equal(one, want[:1].expand(4))
    assert torch.equal(mxfp8gg.linear_cross_entropy(x[0], w, t[0], reduction="none"), want[0])


def test_no_tokens(gpu):
    w = torch.randn((50, 64), device=gpu).to(torch.bfloat16).requires_grad_(True)
    x = torch.empty((0, 64), device=gpu, dtype=torch.bfloat16, requires_grad=True)
    t = torch.empty(0, device=gpu, dtype=torch.int64)
    assert mxfp8gg.linear_cross_entropy(x, w, t, reduction="none").shape == (0,)
    assert torch.isnan(mxfp8gg.linear_cross_entropy(x, w, t))
    dx, dw = torch.autograd.grad(mxfp8gg.linear_cross_entropy(x, w, t, reduction="sum"), (x, w))
    assert dx.shape == (0, 64) and (dw == 0).all()


def test_gradient_matches_differences(gpu):
    """Central differences of the 64-bit loss in directions of x (bf16 inputs leave
    no room for small steps of their own): 1e-2 of |dx| |direction|, the bf16
    rounding of d and dx."""
    x, w, t = _inputs(gpu, 30, 90, 64, 8, ignored=False)
    x.requires_grad_(True)
    dx, = torch.autograd.grad(mxfp8gg.linear_cross_entropy(x, w, t, reduction="sum"), x)
    d = torch.randn((30, 64), generator=torch.Generator().manual_seed(1)).double().numpy()
    f = lambda s: R.linear_cross_entropy(_wide(x) + s * d, _wide(w), t.cpu().numpy())[0]  # noqa: E731
    want = (f(1e-5) - f(-1e-5)) / 2e-5
    got = (_wide(dx) * d).sum(axis=1)
    size = np.linalg.norm(_wide(dx), axis=1) * np.linalg.norm(d, axis=1)
    assert (np.abs(got - want) <= 1e-2 * size).all()


def test_other_stream(gpu):
    x, w, t = _inputs(gpu, 300, 1000, 256, 9)
    want = mxfp8gg.linear_cross_entropy(x, w, t)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = mxfp8gg.linear_cross_entropy(x, w, t)
    side.synchronize()
    assert torch.equal(got, want)


def test_refusals(gpu):
    x, w, t = _inputs(gpu, 8, 30, 64, 1)
    for bad in (dict(x=x.float()), dict(weight=w.float()), dict(target=t.float())):
        with pytest.raises(TypeError):
            mxfp8gg.linear_cross_entropy(**{**dict(x=x, weight=w, target=t), **bad})
    for bad in (dict(x=x[:, :32]), dict(target=t[:4]), dict(weight=w[0]), dict(reduction="max"),
                dict(target=t.cpu()), dict(x=x.cpu()),
                dict(x=x[:, :12].contiguous(), weight=w[:, :12].contiguous()),
                dict(x=x[:, :0], weight=w[:, :0]), dict(weight=w[:0])):
        with pytest.raises(ValueError):
            mxfp8gg.linear_cross_entropy(**{**dict(x=x, weight=w, target=t), **bad})
