"""route_topk where scores are close, saturated or taken on different paths."""
import numpy as np
import pytest
import torch

import mxfp8gg

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("E,G,K", [(256, 8, 8), (32, 1, 8), (320, 8, 6), (1000, 1, 3), (24, 4, 4),
                                   (120, 3, 5)])
def test_softmax_scores_do_not_depend_on_the_batch(gpu, E, G, K, biased):
    """Scores that hold the row's whole sum, and choices that go by them: the same bits
    in a call that shares a token out over more lanes."""
    g = torch.Generator(device=gpu).manual_seed(E)
    T = 2_500_000 // E
    x = 1.5 * torch.randn((T, E), generator=g, device=gpu)
    bias = 0.01 * torch.randn(E, generator=g, device=gpu) if biased else None
    f = lambda z: mxfp8gg.route_topk(z, K, score="softmax", num_groups=G,  # noqa: E731
                                     top_groups=(G + 1) // 2, bias=bias, renormalize=False)
    idx, w = f(x)
    for a in (0, 777, T - 300):
        i, v = f(x[a:a + 300])
        assert torch.equal(i, idx[a:a + 300]) and torch.equal(v, w[a:a + 300])


@pytest.mark.parametrize("renorm", [False, True])
def test_gradient_of_saturated_sigmoids(gpu, renorm):
    """sigma(x) sigma(-x) keeps its digits where sigma(x) is 1 to the last bit.  A slot's
    terms are a few fp32 operations each, 2^-20 relative; where scores are divided by
    their sum the difference of two such terms, of their magnitudes."""
    g = torch.Generator().manual_seed(1)
    T, E, K = 500, 16, 5
    x = ((torch.rand((T, E), generator=g) * 2 - 1) * 80).to(gpu).requires_grad_(True)
    dw = torch.randn((T, K), generator=g).to(gpu)
    idx, w = mxfp8gg.route_topk(x, K, score="sigmoid", renormalize=renorm)
    dx, = torch.autograd.grad(w, x, dw)
    at = idx.cpu().numpy().astype(np.int64)
    z = np.take_along_axis(x.detach().cpu().double().numpy(), at, 1)
    got = np.take_along_axis(dx.cpu().double().numpy(), at, 1)
    d = dw.cpu().double().numpy()
    s, slope = 1 / (1 + np.exp(-z)), 1 / (1 + np.exp(-z)) / (1 + np.exp(z))
    if renorm:
        total = s.sum(axis=1, keepdims=True)
        want = (d - (d * s).sum(axis=1, keepdims=True) / total) / total * slope
        size = (np.abs(d) + (np.abs(d) * s).sum(axis=1, keepdims=True) / total) / total * slope
    else:
        want, size = d * slope, np.abs(d) * slope
    assert (z > 30).mean() > 0.3
    bad = np.abs(got - want) > 2.0 ** -20 * size + 1e-37
    assert not bad.any(), (z[bad][:5], got[bad][:5], want[bad][:5])


def test_gradient_where_every_sigmoid_underflows(gpu):
    """Weights that are 0 because the sum of the scores is have no gradient; slots beside
    a score that is not 0 have that of their tiny slope."""
    x = torch.tensor([[-90.0, -95.0, -100.0, -200.0], [-90.0, 0.0, -200.0, -300.0]], device=gpu)
    x.requires_grad_(True)
    idx, w = mxfp8gg.route_topk(x, 2, score="sigmoid")
    assert idx.tolist() == [[0, 1], [1, 0]] and w.tolist() == [[0.0, 0.0], [1.0, 0.0]]
    dx, = torch.autograd.grad(w, x, torch.tensor([[1.0, 2.0], [1.0, 3.0]], device=gpu))
    assert (dx[0] == 0).all() and (dx[1, 1:] == 0).all() and 0 <= float(dx[1, 0]) < 1e-37


def test_sigmoids_of_both_paths_are_the_same_bits(gpu):
    """Waves whose logits and biases are moderate take sigmoids by a shorter sequence.
    Runs of 32 neighbouring fp32 logits rank the same whether the expert that always
    comes first has a large finite bias or an infinite one, which takes the general
    sequence: a rounding apart would make a tie of two ranks or two ranks of a tie."""
    g = torch.Generator(device=gpu).manual_seed(2)
    T, E = 1 << 17, 33
    base = torch.rand((T, 1), generator=g, device=gpu) * 37 - 20
    base[: T // 8] *= 1e-3
    step = torch.rand((T, 32), generator=g, device=gpu).argsort(dim=1).to(torch.int32)
    near = (base.view(torch.int32) + step).view(torch.float32)
    x = torch.cat([near, torch.zeros((T, 1), device=gpu)], dim=1)
    assert torch.isfinite(x).all() and x.abs().max() < 87
    out = []
    for first in (1e30, float("inf")):
        bias = torch.zeros(E, device=gpu)
        bias[-1] = first
        out.append(mxfp8gg.route_topk(x, 32, score="sigmoid", bias=bias)[0])
    assert (out[0][:, 0] == E - 1).all()
    assert torch.equal(*out)
