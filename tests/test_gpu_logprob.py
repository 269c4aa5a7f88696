"""GPU parity of token_log_probs with 64 bits.

The logits are exact.  An exponent (z - m) log2(e) / T is off by three roundings of its
magnitude, at most 2^-22 |z - m| / T; only exponents above -40 carry weight, so a term's
relative error is below 40 * 2^-22 + 2^-22 (the hardware's power of two) < 1e-5, and so
is that of their sum S (added fp32 sums of up to V / 512 terms a thread: V / 512 * 2^-24
more, below 2e-5 at 2^17).  log S is off by that and 2^-23 of itself; a log probability by
3e-5 + 2^-22 (|z - m| / T + log S).  The entropy is a mean of exponents up to log V with
such weights: 1e-4 * (1 + log V) covers both its parts.  Gradients: p is off by 4e-5 of
itself (and by the log probability's error), times the sum of the incoming gradients'
magnitudes, entropy's with |log p + H|; half a step, 2^-8 of the value, for bf16.
"""
import math

import pytest
import torch

import mxfp8gg

pytestmark = pytest.mark.gpu

NEG = float("-inf")


def _logits(gpu, T, V, dtype, seed=0, scale=2.0, shift=0.0):
    g = torch.Generator().manual_seed(seed + T + V)
    z = (torch.randn((T, V), generator=g) * scale + shift).to(dtype).to(gpu)
    t = torch.randint(0, V, (T,), generator=g).to(gpu)
    return z, t


def _reference(z, temperature):
    """(log p, entropy) in 64 bits; rows of -inf: -inf and 0."""
    x = z.double() / temperature
    dead = (x == NEG).all(dim=-1, keepdim=True)
    lp = torch.log_softmax(torch.where(dead, 0.0, x), dim=-1)
    lp = torch.where(dead | (x == NEG), NEG, lp)
    fin = torch.where(lp == NEG, 0.0, lp)
    return lp, -(lp.exp() * fin).sum(dim=-1)


def _check(z, target, temperature=1.0, topk=0, grads=True, ignore=-100):
    V = z.shape[-1]
    leaf = z.detach().requires_grad_(grads)
    r = mxfp8gg.token_log_probs(leaf, target, temperature=temperature, topk=topk, ignore_index=ignore)
    with torch.no_grad():
        again = mxfp8gg.token_log_probs(z, target, temperature=temperature, topk=topk, ignore_index=ignore)
    for a, b in zip(r, again):
        assert (a is None) == (b is None) and (a is None or torch.equal(a.detach(), b))
    lp, ent = _reference(z, temperature)
    live = torch.ones(z.shape[0], dtype=torch.bool, device=z.device) if target is None else target != ignore
    span = torch.where(lp == NEG, 0.0, lp.amax(dim=-1, keepdim=True) - lp)  # |z - m| / T
    loose = 3e-5 + 2.0 ** -22 * (span + math.log(V))

    def same(got, want, bound):
        want = torch.where(want.float().isinf(), want.float().double(), want)  # past fp32's range
        fin = torch.isfinite(want)
        assert torch.equal(got.double()[~fin], want[~fin])
        assert not bool(((got.double() - want).abs() > bound)[fin].any())

    at = torch.where(live, target, 0)[:, None] if target is not None else None
    if target is not None:
        same(r.log_probs.detach(), torch.where(live, lp.gather(1, at)[:, 0], 0.0), loose.gather(1, at)[:, 0])
    same(r.entropy.detach(), torch.where(live, ent, 0.0), torch.full_like(ent, 1e-4 * (1 + math.log(V))))
    if topk:
        order = z.double().sort(dim=-1, descending=True, stable=True).indices[:, :topk]
        best = lp.gather(1, order)
        kept = live[:, None] & (best > NEG)
        assert torch.equal(r.top_ids, torch.where(kept, order, -1).int())
        same(r.top_log_probs.detach(), torch.where(kept, best, NEG), loose.gather(1, order))
    if not grads:
        return
    g = torch.Generator().manual_seed(7)
    up = [torch.randn(o.shape, generator=g).to(z.device) if o is not None and o.is_floating_point() else None
          for o in r]
    p = torch.where(lp == NEG, 0.0, lp.exp())
    dead = (lp == NEG).all(dim=-1)
    on = (live & ~dead).double()[:, None]
    for used in ((0, 1, 3), (0,), (1,), (3,)):
        pairs = [(r[i], up[i]) for i in used if r[i] is not None]
        if not pairs:
            continue
        got, = torch.autograd.grad([o for o, _ in pairs], leaf, [u for _, u in pairs], retain_graph=True)
        assert got.dtype is z.dtype
        chosen = torch.zeros_like(lp)
        total = torch.zeros_like(ent)
        size = torch.zeros_like(ent)
        if 0 in used and target is not None:
            chosen.scatter_add_(1, at, up[0].double()[:, None])
            total, size = total + up[0].double(), size + up[0].double().abs()
        if 3 in used and topk:
            u = up[3].double() * (r.top_ids >= 0)
            chosen.scatter_add_(1, r.top_ids.long().clamp_min(0), u)
            total, size = total + u.sum(dim=1), size + u.abs().sum(dim=1)
        gh = up[1].double() if 1 in used else torch.zeros_like(ent)
        inner = torch.where(lp == NEG, 0.0, lp + ent[:, None])
        want = on * (chosen - p * (total[:, None] + gh[:, None] * inner)) / temperature
        err = (4e-5 + loose) * p * (size[:, None] + gh.abs()[:, None] * (1 + inner.abs())) \
            + p * gh.abs()[:, None] * (loose + 1e-4 * (1 + math.log(V))) + 2.0 ** -23 * chosen.abs()
        bound = err / temperature + 1e-30
        if z.dtype is torch.bfloat16:
            bound = bound + 2.0 ** -8 * want.abs()
        bad = (got.double() - want).abs() > bound
        assert not bool(bad.any()), (used, torch.nonzero(bad)[0].tolist(), float(got[bad][0]),
                                     float(want[bad][0]), float(bound[bad][0]))


SIZES = [(1, 1), (1, 7), (3, 64), (5, 100), (2, 4097), (17, 8192), (600, 1003), (1, 131072),
         (4, 50021), (1, 300007), (3, 20000)]


@pytest.mark.parametrize("T,V", SIZES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_matches_64_bits(gpu, T, V, dtype):
    z, t = _logits(gpu, T, V, dtype)
    _check(z, t, topk=min(V, 8))
    _check(z, t.int(), temperature=0.6)
    _check(z, None, temperature=1.7, topk=min(V, 3))


@pytest.mark.parametrize("topk", [1, 2, 20, 33, 64])
@pytest.mark.parametrize("T,V", [(2, 64), (3, 129), (5, 3000), (2, 40000), (530, 5001)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_alternatives(gpu, topk, T, V, dtype):
    z, t = _logits(gpu, T, V, dtype, seed=1)
    _check(z, t, topk=topk, grads=False)


@pytest.mark.parametrize("V", [500, 3000, 70000, 270000])
def test_ties_go_to_the_lowest_index(gpu, V):
    z = torch.zeros((4, V), device=gpu)          # all equal
    z[1] = torch.arange(V, device=gpu) % 3       # a third of them
    z[2, V - 5:] = 1.0                           # few, at the end
    z[3] = torch.arange(V, device=gpu) / V       # rising
    _check(z, None, topk=20, grads=False)
    _check(z.to(torch.bfloat16), None, topk=20, grads=False)


def test_masks(gpu):
    z, t = _logits(gpu, 12, 5000, torch.float32)
    z[0] = NEG
    z[1, 1:] = NEG
    z[2, :] = NEG
    z[2, 4990:] = 0.5
    z[3] = torch.finfo(torch.float32).min
    z[4, ::2] = torch.finfo(torch.float32).min
    z[5, 10:] = -1e30
    z[6, t[6]] = NEG
    z[7, :4096] = NEG
    _check(z, t, topk=16)
    _check(z, t, topk=16, temperature=0.01)
    low = z.to(torch.bfloat16)
    low[3] = torch.finfo(torch.bfloat16).min
    _check(low, t, topk=16)


def test_ignored_targets(gpu):
    z, t = _logits(gpu, 9, 5000, torch.bfloat16)
    z[2] = float("nan")                           # not read
    t[2] = t[5] = -100
    _check(z, t, topk=4)
    t[2] = t[5] = 7
    z[2] = 0.0
    _check(z, t, topk=4, ignore=7)


def test_large_offset_and_spread(gpu):
    z, t = _logits(gpu, 5, 3001, torch.float32, shift=1e6)
    _check(z, t, topk=5)
    z, t = _logits(gpu, 5, 3001, torch.float32, scale=300.0)
    _check(z, t, topk=5)


def test_non_finite(gpu):
    z, t = _logits(gpu, 4, 9000, torch.float32)
    z[0, 8000] = float("nan")
    z[1, 5] = float("inf")
    leaf = z.clone().requires_grad_(True)
    r = mxfp8gg.token_log_probs(leaf, t, topk=3)
    for o in (r.log_probs, r.entropy, r.top_log_probs):
        assert torch.isnan(o[:2]).all() and torch.isfinite(o[2:]).all()
    assert (r.top_ids[:2] == -1).all() and (r.top_ids[2:] >= 0).all()
    dz, = torch.autograd.grad(r.log_probs.sum(), leaf)
    assert torch.isnan(dz[:2]).all() and torch.isfinite(dz[2:]).all()


def test_target_out_of_range(gpu):
    z, t = _logits(gpu, 4, 500, torch.float32)
    t[1], t[2] = 500, -1
    leaf = z.clone().requires_grad_(True)
    r = mxfp8gg.token_log_probs(leaf, t)
    assert torch.isnan(r.log_probs[1:3]).all() and torch.isfinite(r.entropy).all()
    dz, = torch.autograd.grad(r.log_probs.sum(), leaf)
    assert torch.isnan(dz[1:3]).all() and torch.isfinite(dz[0]).all() and torch.isfinite(dz[3]).all()


def test_gradient_by_differences(gpu):
    z, t = _logits(gpu, 3, 50, torch.float32)
    g = torch.Generator().manual_seed(2)
    u = [torch.randn(s, generator=g).to(gpu) for s in ((3,), (3,), (3, 4))]
    leaf = z.clone().requires_grad_(True)
    r = mxfp8gg.token_log_probs(leaf, t, temperature=0.8, topk=4)
    got, = torch.autograd.grad([r.log_probs, r.entropy, r.top_log_probs], leaf, u)

    def f(x):
        lp, ent = _reference(x, 0.8)
        return ((lp.gather(1, t[:, None])[:, 0] * u[0]).sum() + (ent * u[1]).sum()
                + (lp.gather(1, r.top_ids.long()) * u[2]).sum())

    step = torch.randn(z.shape, generator=g).double().to(gpu)
    slope = float((f(z.double() + 1e-6 * step) - f(z.double() - 1e-6 * step)) / 2e-6)
    assert abs(slope - float((got.double() * step).sum())) < 1e-3 * max(1.0, abs(slope))


def test_layouts(gpu):
    z, t = _logits(gpu, 6, 1001, torch.bfloat16)
    want = mxfp8gg.token_log_probs(z, t, topk=4)
    wide = torch.zeros((6, 1100), dtype=torch.bfloat16, device=gpu)
    wide[:, 3:1004] = z
    for v, tt, lead in ((wide[:, 3:1004], t, (6,)), (z.t().contiguous().t(), t, (6,)),
                        (z.view(2, 3, 1001), t.view(2, 3), (2, 3)), (z.view(2, 3, 1001), t.int().view(2, 3), (2, 3))):
        leaf = v.detach().requires_grad_(True)
        r = mxfp8gg.token_log_probs(leaf, tt, topk=4)
        assert r.log_probs.shape == lead and r.top_ids.shape == (*lead, 4)
        for a, b in zip(r, want):
            assert torch.equal(a.detach().reshape(b.shape), b)
        assert torch.autograd.grad(r.entropy.sum(), leaf)[0].shape == v.shape
    e = mxfp8gg.token_log_probs(z[:0], t[:0], topk=4)
    assert e.log_probs.shape == (0,) and e.top_ids.shape == (0, 4)
    one = mxfp8gg.token_log_probs(z[0], t[0])
    assert one.log_probs.shape == () and torch.equal(one.log_probs, want.log_probs[0])


def test_graph_replays(gpu):
    z, t = _logits(gpu, 2, 50000, torch.bfloat16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        mxfp8gg.token_log_probs(z, t, topk=8)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = mxfp8gg.token_log_probs(z, t, topk=8)
    for i in range(3):
        z.copy_(_logits(gpu, 2, 50000, torch.bfloat16, seed=i + 5)[0])
        want = mxfp8gg.token_log_probs(z, t, topk=8)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(r, want))


def test_refusals(gpu):
    m = mxfp8gg.token_log_probs
    z, t = _logits(gpu, 4, 100, torch.float32)
    for call in (lambda: m(z, t[:3]), lambda: m(z, t, topk=65), lambda: m(z, t, topk=-1),
                 lambda: m(z[:, :5], t, topk=6), lambda: m(z, t, temperature=0.0),
                 lambda: m(z, t, temperature=-1.0), lambda: m(z, t, temperature=float("nan")),
                 lambda: m(z, t.cpu()), lambda: m(z[:, :0], t), lambda: m(z, t, topk=1.5)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: m(z.half(), t), lambda: m(z, t.float()), lambda: m(None)):
        with pytest.raises(TypeError):
            call()
    leaf = z.clone().requires_grad_(True)
    with pytest.raises(RuntimeError, match="differentiated twice"):
        torch.autograd.grad(m(leaf, t).log_probs.sum(), leaf, create_graph=True)
