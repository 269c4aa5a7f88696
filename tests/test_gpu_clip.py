"""GPU parity of grad_norm and clip_grad_norm_ with 64 bits.

Squares of fp32 and bf16 values are exact in fp64 and so are, to 2^-50, their sums: the
norm is the fp32 rounding of its 64-bit value, 2^-24.  A clipped gradient is the product
with an fp32 factor, 2 * 2^-24 of the value, and half a step of bf16, 2^-8.
"""
import math

import pytest
import torch

import mxfp8gg

pytestmark = pytest.mark.gpu


def _grads(gpu, sizes, dtypes=(torch.float32, torch.bfloat16), scale=1.0, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(n, generator=g) * scale).to(dtypes[i % len(dtypes)]).to(gpu)
            for i, n in enumerate(sizes)]


def _norm(grads):
    return math.sqrt(math.fsum(float(g.double().square().sum()) for g in grads))


def _check(grads, max_norm):
    before = [g.clone() for g in grads]
    want = _norm(grads)
    n = mxfp8gg.grad_norm(grads)
    assert all(torch.equal(a, b) for a, b in zip(grads, before))
    got = mxfp8gg.clip_grad_norm_(grads, max_norm)
    assert got.shape == () and got.dtype is torch.float32 and torch.equal(n, got)
    assert abs(float(got) - want) <= 2.0 ** -24 * want * 1.01
    f = max_norm / (want + 1e-6)
    for a, b in zip(grads, before):
        if f >= 1 + 1e-6:
            assert torch.equal(a, b)
            continue
        ref = b.double() * f
        bound = 3 * 2.0 ** -24 * ref.abs() + 2.0 ** -149
        if a.dtype is torch.bfloat16:
            bound = bound + 2.0 ** -8 * ref.abs()
        assert not bool(((a.double() - ref).abs() > bound).any())


@pytest.mark.parametrize("sizes", [[1], [7, 0, 1], [8191, 8192, 8193], [3] * 500, [1 << 22, 5, 100003],
                                   [0, 0], [2048 * 8192 + 17]])
@pytest.mark.parametrize("dtypes", [(torch.float32,), (torch.bfloat16,), (torch.bfloat16, torch.float32)])
def test_matches_64_bits(gpu, sizes, dtypes):
    for factor in (0.25, 2.0):
        grads = _grads(gpu, sizes, dtypes)
        _check(grads, factor * max(_norm(grads), 1e-3))


@pytest.mark.parametrize("scale", [1e25, 1e-25])
def test_no_overflow_of_squares(gpu, scale):
    grads = _grads(gpu, [1000, 333], scale=scale)
    want = _norm(grads)
    assert abs(float(mxfp8gg.grad_norm(grads)) / want - 1) < 1e-6


def test_unaligned_and_permuted(gpu):
    base = torch.randn(5000, device=gpu)
    half = torch.randn(5000, device=gpu).to(torch.bfloat16)
    grads = [base[1:4000], half[3:4998], torch.randn((30, 50), device=gpu).t(),
             torch.randn((4, 3, 8, 6), device=gpu).to(memory_format=torch.channels_last)]
    rest = base[4000:].clone(), half[:3].clone(), half[4998:].clone(), base[:1].clone()
    _check(grads, 1.0)
    assert torch.equal(base[4000:], rest[0]) and torch.equal(half[:3], rest[1])
    assert torch.equal(half[4998:], rest[2]) and torch.equal(base[:1], rest[3])


def test_non_finite(gpu):
    grads = _grads(gpu, [100, 200])
    grads[1][3] = float("inf")
    assert math.isinf(float(mxfp8gg.clip_grad_norm_(grads, 1.0)))
    assert (grads[0] == 0).all() and torch.isnan(grads[1][3]) and (grads[1][4:] == 0).all()
    grads = _grads(gpu, [100, 200])
    grads[0][3] = float("nan")
    assert math.isnan(float(mxfp8gg.clip_grad_norm_(grads, 1.0)))
    assert all(torch.isnan(g).all() for g in grads)


def test_same_bits_on_every_run_and_in_a_graph(gpu):
    grads = _grads(gpu, [100000, 70001, 9])
    first = mxfp8gg.grad_norm(grads)
    keep = [g.clone() for g in grads]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        mxfp8gg.grad_norm(grads)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = mxfp8gg.clip_grad_norm_(grads, 1.0)
    for i in range(3):
        for g, k in zip(grads, keep):
            g.copy_(k * (i + 1))
        eager = [g.clone() for g in grads]
        want = mxfp8gg.clip_grad_norm_(eager, 1.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(norm, want) and all(torch.equal(a, b) for a, b in zip(grads, eager))
    assert torch.equal(mxfp8gg.grad_norm(keep), first)


def test_optimizer_clips_what_it_steps(gpu):
    p = [torch.nn.Parameter(torch.randn(50, device=gpu)), torch.nn.Parameter(torch.randn(9, device=gpu))]
    opt = mxfp8gg.AdamW([dict(params=[p[0]]), dict(params=[p[1]], lr=1e-4)])
    assert opt.clip_grad_norm_(1.0) is None
    (p[0].sum() * 3 + p[1].square().sum()).backward()
    version = p[0].grad._version
    want = _norm([p[0].grad, p[1].grad])
    got = opt.clip_grad_norm_(0.5)
    assert abs(float(got) - want) < 1e-5 and p[0].grad._version > version
    assert abs(_norm([p[0].grad, p[1].grad]) - 0.5) < 1e-5
    opt.step()


def test_refusals(gpu):
    m, g = mxfp8gg, torch.zeros(8, device=gpu)
    for call in (lambda: m.grad_norm([]), lambda: m.clip_grad_norm_([g, g], 1.0),
                 lambda: m.clip_grad_norm_([g], -1.0), lambda: m.clip_grad_norm_([g], float("nan")),
                 lambda: m.grad_norm([torch.zeros((4, 8), device=gpu)[:, ::2]]),
                 lambda: m.grad_norm([torch.zeros(1, device=gpu).expand(5)]),
                 lambda: m.grad_norm([g, g.cpu()])):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        m.grad_norm([g.half()])
    with pytest.raises(TypeError):
        m.grad_norm([torch.zeros((4, 4), device=gpu).to_sparse()])
    with pytest.raises(TypeError):
        m.grad_norm([None])
