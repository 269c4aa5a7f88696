"""GPU parity of the routing decision (route_topk) and its gradient against the
64-bit oracle.

Ids are compared exactly: the inputs have distinct ranks or exact ties, which
go to the lowest index.  Scores are a quotient of at most 32 exponentials
(each within a few units of 2^-24, arguments within 24 of zero, so 2^-19.4
relative at most): relative tolerance 1e-5.  Gradients are sums of at most 33
such terms of size scale * |dw|: 2e-5 of that, and half a unit of bf16 (2^-8
relative) where the logits are bf16.
"""
import numpy as np
import pytest
import torch

import mxfp8gg
from tests import _operators_oracle as R

pytestmark = pytest.mark.gpu


def _logits(gpu, T, E, dtype, seed, masked=False):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((T, E), generator=g) * 1.5
    if dtype is torch.float32:
        x[:, ::3] = torch.round(x[:, ::3] * 4) / 4     # exact ties between experts
    x = x.to(dtype)
    if masked:
        x[torch.rand((T, E), generator=g) < 0.4] = -float("inf")
        x[::3] = -float("inf")                          # tokens that nothing is left of
        x[1:2] = torch.finfo(dtype).min                   # the type's lowest value is no mask
    return x.to(gpu)


def _wide(x):
    return x.detach().cpu().double().numpy()


def _check(x, K, opt, bias=None):
    idx, w = mxfp8gg.route_topk(x, K, bias=bias, **opt)
    assert idx.dtype == torch.int32 and w.dtype == torch.float32
    assert idx.shape == w.shape == (x.shape[0], K)
    ridx, rw = R.route_topk(_wide(x), K, bias=None if bias is None else _wide(bias), **opt)
    assert np.array_equal(idx.cpu().numpy(), ridx)
    np.testing.assert_allclose(_wide(w), rw, rtol=1e-5, atol=1e-30)
    return idx, w


CASES = [
    # T, E, K, groups, top_groups
    (1, 1, 1, 1, 1), (1, 256, 8, 8, 4), (3, 5, 5, 1, 1), (64, 32, 8, 1, 1), (65, 33, 7, 3, 2),
    (37, 256, 8, 1, 1), (130, 257, 9, 1, 1), (40, 512, 16, 16, 5), (33, 1024, 32, 1, 1),
    (50, 1023, 20, 33, 7), (29, 40, 6, 8, 8), (31, 64, 17, 64, 33), (257, 8, 2, 2, 1),
    (20, 96, 32, 3, 2), (12, 480, 8, 5, 3)]


@pytest.mark.parametrize("T,E,K,G,keep", CASES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("score,biased,best,renorm", [
    ("softmax", False, 1, True), ("softmax", False, 1, False), ("sigmoid", True, 2, True),
    ("sigmoid", False, 1, False), ("softmax", True, 1, True)])
def test_decision_matches_oracle(gpu, T, E, K, G, keep, dtype, score, biased, best, renorm):
    for masked in (False, True):
        x = _logits(gpu, T, E, dtype, 3 * T + E, masked)
        bias = None
        if biased:
            bias = (torch.randn(E, generator=torch.Generator().manual_seed(E)) * 0.1).to(gpu)
        _check(x, K, dict(score=score, num_groups=G, top_groups=keep, group_best=best,
                          renormalize=renorm, scale=2.5), bias)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_groups_by_two_best_scores(gpu, score):
    x = _logits(gpu, 77, 60, torch.bfloat16, 5).float()
    x += torch.rand(x.shape, generator=torch.Generator().manual_seed(1)).to(gpu)  # no ties
    _check(x, 6, dict(score=score, num_groups=6, top_groups=2, group_best=2, renormalize=True))


@pytest.mark.parametrize("score,biased,best", [("softmax", False, 1), ("sigmoid", True, 2)])
@pytest.mark.parametrize("E,G,K", [(256, 8, 8), (32, 1, 8), (320, 8, 6), (1024, 1, 3)])
def test_large_and_small_calls_agree(gpu, E, G, K, score, biased, best):
    """The same bits whether a token comes in a call of millions of logits or in
    one of few (other shares of a token to a lane)."""
    T = 2_500_000 // E
    x = _logits(gpu, T, E, torch.float32, E)
    bias = (torch.randn(E, generator=torch.Generator().manual_seed(E)) * 0.1).to(gpu)
    f = lambda z: mxfp8gg.route_topk(z, K, score=score, num_groups=G, top_groups=(G + 1) // 2,  # noqa: E731
                                     group_best=best, bias=bias if biased else None)
    idx, w = f(x)
    for a in (0, 777, T - 100):
        i, v = f(x[a:a + 100])
        assert torch.equal(i, idx[a:a + 100]) and torch.equal(v, w[a:a + 100])


def test_all_experts_equal_take_the_lowest_ids(gpu):
    for E, K, G in ((64, 8, 1), (256, 8, 8), (1024, 32, 4)):
        idx, w = mxfp8gg.route_topk(torch.zeros((5, E), device=gpu), K, num_groups=G, top_groups=1)
        assert torch.equal(idx.cpu(), torch.arange(K, dtype=torch.int32).expand(5, K))
        assert torch.equal(w.cpu(), torch.full((5, K), 1.0 / K))
    idx, _ = mxfp8gg.route_topk(torch.tensor([[-0.0, 0.0, -0.0, 0.0]], device=gpu), 4)
    assert idx.tolist() == [[0, 1, 2, 3]]


def test_masked_rows_and_slots(gpu):
    x = torch.full((4, 16), -float("inf"), device=gpu)
    x[1, 5] = 2.0
    x[2, [3, 9]] = torch.finfo(torch.float32).min
    x[3] = 200.0                                        # large, equal
    for score in ("softmax", "sigmoid"):
        idx, w = mxfp8gg.route_topk(x, 3, score=score)
        assert idx.tolist() == [[-1, -1, -1], [5, -1, -1], [3, 9, -1], [0, 1, 2]]
        assert w[0].tolist() == [0.0] * 3 and w[1].tolist() == [1.0, 0.0, 0.0]
        if score == "softmax":
            assert w[2].tolist() == [0.5, 0.5, 0.0]
        else:                                           # both scores underflow to zero
            assert w[2].tolist() == [0.0] * 3
        assert torch.equal(w[3].cpu(), torch.full((3,), 1 / 3))
    # a bias of -inf takes an expert out for every token
    b = torch.zeros(16, device=gpu)
    b[0] = -float("inf")
    idx, _ = mxfp8gg.route_topk(x, 3, score="sigmoid", bias=b)
    assert idx.tolist()[3] == [1, 2, 3]


def test_nan_and_infinities(gpu):
    nan, inf = float("nan"), float("inf")
    x = torch.tensor([[0.0, nan, 1.0, 2.0], [0.0, inf, 1.0, -inf]], device=gpu)
    idx, w = mxfp8gg.route_topk(x, 2)
    assert idx.tolist() == [[1, 3], [1, 2]]
    assert torch.isnan(w).all()                         # inf - inf in the softmax
    idx, w = mxfp8gg.route_topk(x, 2, score="sigmoid", renormalize=False)
    assert idx.tolist() == [[1, 3], [1, 2]]
    assert torch.isnan(w[0, 0]) and w[1, 0] == 1.0 and torch.isfinite(w[:, 1]).all()


def test_plan_drops_what_the_decision_leaves_out(gpu):
    x = _logits(gpu, 50, 12, torch.float32, 9, masked=True)
    idx, _ = mxfp8gg.route_topk(x, 4)
    plan = mxfp8gg.route_plan(idx, 12, 1)
    assert int(plan.counts.sum()) == int((idx >= 0).sum()) < idx.numel()


@pytest.mark.parametrize("T,E,K,G,keep", CASES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("score,renorm", [("softmax", True), ("softmax", False),
                                          ("sigmoid", True), ("sigmoid", False)])
def test_gradient_matches_formula(gpu, T, E, K, G, keep, dtype, score, renorm):
    x = _logits(gpu, T, E, dtype, T + E).requires_grad_(True)
    g = torch.Generator().manual_seed(T)
    dw = torch.randn((T, K), generator=g).to(gpu)
    bias = (torch.randn(E, generator=g) * 0.1).to(gpu) if score == "sigmoid" else None
    idx, w = mxfp8gg.route_topk(x, K, score=score, bias=bias, num_groups=G, top_groups=keep,
                                renormalize=renorm, scale=2.5)
    dx, = torch.autograd.grad(w, x, dw)
    assert dx.dtype == dtype and dx.shape == x.shape
    ref = R.route_grad(_wide(x), idx.cpu().numpy(), _wide(dw), score, renorm, 2.5)
    # with a renormalised sum S of small scores the terms are dw * s / S, below dw
    bound = 2e-5 * 2.5 * _wide(dw.abs().amax(dim=1, keepdim=True))
    if dtype is torch.bfloat16:
        bound = bound + 2.0 ** -8 * np.abs(ref)
    assert (np.abs(_wide(dx) - ref) <= bound).all()


@pytest.mark.parametrize("score,renorm", [("softmax", True), ("softmax", False),
                                          ("sigmoid", True), ("sigmoid", False)])
def test_gradient_matches_differences(gpu, score, renorm):
    """Central differences of the kernel's own forward along random directions.
    Step 2^-7: truncation below 2^-14 of the third derivative (scores have
    derivatives below 1), rounding 2^-22 / 2^-7: 1e-3 of |dw| |dir| covers both."""
    T, E, K = 40, 24, 5
    g = torch.Generator().manual_seed(3)
    # ranks two steps apart, so no direction changes the choice
    x = torch.stack([torch.randperm(E, generator=g) for _ in range(T)]).float().mul_(0.1).to(gpu)
    d = (torch.rand((T, E), generator=g) * 2 - 1).to(gpu)
    dw = torch.randn((T, K), generator=g).to(gpu)
    f = lambda z: mxfp8gg.route_topk(z, K, score=score, renormalize=renorm)  # noqa: E731
    step = 2.0 ** -7
    (ia, a), (ib, b) = f(x + step * d), f(x - step * d)
    assert torch.equal(ia, ib)
    want = (((a.double() - b.double()) / (2 * step)) * dw).sum(dim=1)
    z = x.clone().requires_grad_(True)
    dx, = torch.autograd.grad(f(z)[1], z, dw)
    got = (dx.double() * d).sum(dim=1)
    assert (got - want).abs().max() <= 1e-3 * float(dw.norm(dim=1).max() * d.norm(dim=1).max())


def test_gradient_of_empty_and_masked_rows(gpu):
    x = _logits(gpu, 60, 20, torch.float32, 4, masked=True).requires_grad_(True)
    for score, renorm in (("softmax", True), ("softmax", False), ("sigmoid", True)):
        idx, w = mxfp8gg.route_topk(x, 4, score=score, renormalize=renorm)
        dx, = torch.autograd.grad(w.sum(), x)
        assert torch.isfinite(dx).all()
        assert (dx[x == -float("inf")] == 0).all()
        assert (dx[(idx < 0).all(dim=1)] == 0).all()
    x = torch.empty((0, 16), device=gpu, requires_grad=True)
    idx, w = mxfp8gg.route_topk(x, 4)
    assert idx.shape == (0, 4)
    assert torch.autograd.grad(w.sum(), x)[0].shape == (0, 16)


def test_strided_logits_and_other_stream(gpu):
    big = _logits(gpu, 70, 100, torch.float32, 8)
    x = big[:, 10:74]
    want = mxfp8gg.route_topk(x.clone(), 6)
    for v in (x, x.t().contiguous().t()):
        got = mxfp8gg.route_topk(v, 6)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # a slice that starts two bytes past a 16-byte boundary
    flat = _logits(gpu, 1, 1 + 33 * 9, torch.bfloat16, 2)[0]
    y = flat[1:].view(33, 9)
    a, b = mxfp8gg.route_topk(y, 3), mxfp8gg.route_topk(y.clone(), 3)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = mxfp8gg.route_topk(x, 6)
    side.synchronize()
    assert torch.equal(got[0], want[0])


def test_refusals(gpu):
    x = torch.zeros((4, 16), device=gpu)
    for bad in (dict(topk=0), dict(topk=17), dict(topk=2, num_groups=3),
                dict(topk=2, num_groups=4, top_groups=5), dict(topk=2, top_groups=0),
                dict(topk=2, score="relu"), dict(topk=2, group_best=3),
                dict(topk=2, bias=torch.zeros(15, device=gpu))):
        with pytest.raises(ValueError):
            mxfp8gg.route_topk(x, **bad)
    with pytest.raises(TypeError):
        mxfp8gg.route_topk(x.half(), 2)
    with pytest.raises(TypeError):
        mxfp8gg.route_topk(x[0], 2)
    with pytest.raises(ValueError):
        mxfp8gg.route_topk(torch.zeros((2, 1025), device=gpu), 2)
    with pytest.raises(ValueError):
        mxfp8gg.route_topk(torch.zeros((2, 64), device=gpu), 33)
    with pytest.raises(ValueError):
        mxfp8gg.route_topk(x.cpu(), 2)
