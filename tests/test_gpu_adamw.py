"""GPU parity of adamw_step and AdamW with the 64-bit oracle.

Bounds: every product, sum, root and quotient is one fp32 rounding, 2^-24
relative (the scalars another).  m and v: 2^-21 of the sum of their terms'
magnitudes.  The weight: 2^-21 of |p| + 8 |update|; half a unit of bf16 (2^-8
relative) more where it is bf16.  8-bit states round what fp32 holds to e4m3:
2^-4 of the value or 2^-10 of the block's scale (half a unit above and below
e4m3's normal range), and 2^-20 of the value for the fp32 steps before.
"""
import copy

import numpy as np
import pytest
import torch

import mxfp8gg
from tests import _operators_oracle as R

pytestmark = pytest.mark.gpu

HYPER = dict(step=7, lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
SIZES = [1, 31, 32, 33, 4096, 4097, 7, 12345, 65, 100003, 0, 8]


def _wide(t):
    return t.detach().cpu().double().numpy().reshape(-1)


def _bytes(t):
    return t.detach().cpu().view(torch.uint8).numpy().reshape(-1)


def _tensors(gpu, sizes, ptype, gtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    make = lambda n, s: torch.randn(n, generator=g) * s  # noqa: E731
    params = [make(n, 0.5).to(ptype).to(gpu) for n in sizes]
    grads = [make(n, 1e-2).to(gtype).to(gpu) for n in sizes]
    m = [make(n, 1e-2).to(gpu) for n in sizes]
    v = [(make(n, 1e-2) ** 2).to(gpu) for n in sizes]
    return params, grads, m, v


def _check_param(got, want, old, bf16):
    bound = 2.0 ** -21 * (np.abs(want) + 8 * np.abs(want - old))
    if bf16:
        bound = bound + 2.0 ** -8 * np.abs(want)
    assert (np.abs(_wide(got) - want) <= bound).all()


@pytest.mark.parametrize("ptype,gtype,master", [
    (torch.float32, torch.float32, False), (torch.bfloat16, torch.bfloat16, False),
    (torch.bfloat16, torch.float32, True), (torch.float32, torch.bfloat16, False),
    (torch.bfloat16, torch.bfloat16, True)])
@pytest.mark.parametrize("sizes", [SIZES, [50] * 100, [200001]])
def test_32_bit_states(gpu, ptype, gtype, master, sizes):
    params, grads, m, v = _tensors(gpu, sizes, ptype, gtype)
    masters = [p.float() + 1e-4 for p in params] if master else None
    source = masters if master else params
    before = [tuple(map(_wide, t)) for t in zip(source, grads, m, v)]
    mxfp8gg.adamw_step(params, grads, m, v, masters=masters, **HYPER)
    for i, (p0, g0, m0, v0) in enumerate(before):
        rp, rm, rv = R.adamw(p0, g0, m0, v0, **HYPER)
        b1, b2 = HYPER["betas"]
        assert (np.abs(_wide(m[i]) - rm) <= 2.0 ** -21 * (np.abs(m0) + np.abs(g0))).all()
        assert (np.abs(_wide(v[i]) - rv) <= 2.0 ** -21 * (v0 + g0 * g0)).all()
        if master:
            _check_param(masters[i], rp, p0, False)
            assert torch.equal(params[i], masters[i].to(ptype))
        else:
            _check_param(params[i], rp, p0, ptype is torch.bfloat16)


def _pack(x):
    """fp32 values -> an 8-bit state, by torch's own conversion."""
    b = torch.nn.functional.pad(x.reshape(-1), (0, -x.numel() % 32)).view(-1, 32)
    amax = b.abs().amax(dim=1, keepdim=True)
    mant, exp = torch.frexp(amax)
    j = torch.where(amax > 0, exp - 9 + (mant > 0.875), -126).clamp(-126, 127)
    q = torch.ldexp(b, -j).to(torch.float8_e4m3fn).view(-1)[:x.numel()].view(x.shape)
    return q.contiguous(), (j + 127).to(torch.uint8).view(-1)


def _check_state(state, want):
    q, s = _bytes(state[0]), _bytes(state[1])
    if want.size == 0:
        return
    pad = np.pad(want, (0, -want.size % 32)).reshape(-1, 32)
    amax = np.abs(pad).max(axis=1)
    with np.errstate(divide="ignore", invalid="ignore"):
        j = np.ceil(np.log2(amax / 448))
        edge = np.abs(np.log2(amax / 448) - np.rint(np.log2(amax / 448))) < 1e-6
    b = np.clip(j, -126, 127) + 127
    assert ((s == b) | edge).all()
    unit = 2.0 ** -10 * np.repeat(2.0 ** (s.astype(int) - 127), 32)[:want.size]
    err = np.abs(R.mx8_values(q, s) - want)
    assert (err <= np.maximum(2.0 ** -4 * np.abs(want), unit) + 2.0 ** -20 * np.abs(want)).all()


@pytest.mark.parametrize("ptype,gtype,master", [
    (torch.float32, torch.float32, False), (torch.bfloat16, torch.bfloat16, False),
    (torch.bfloat16, torch.float32, True)])
@pytest.mark.parametrize("sizes", [SIZES, [50] * 100, [200001]])
def test_8_bit_states(gpu, ptype, gtype, master, sizes):
    params, grads, m, v = _tensors(gpu, sizes, ptype, gtype, 1)
    for g in grads:
        g[10:90] = 0                                     # blocks without a gradient
    for t in m + v:
        t[20:70] = 0
        t[100:164] *= 1e-30                              # and blocks of tiny values
    m, v = [_pack(t) for t in m], [_pack(t.sqrt()) for t in v]
    masters = [p.float() for p in params] if master else None
    before = []
    for p, g, a, r in zip(masters or params, grads, m, v):
        before.append((_wide(p), _wide(g), R.mx8_values(_bytes(a[0]), _bytes(a[1])),
                       R.mx8_values(_bytes(r[0]), _bytes(r[1]))))
    mxfp8gg.adamw_step(params, grads, m, v, masters=masters, **HYPER)
    for i, (p0, g0, m0, r0) in enumerate(before):
        rp, rm, rv = R.adamw(p0, g0, m0, r0 * r0, **HYPER)
        _check_param((masters or params)[i], rp, p0, not master and ptype is torch.bfloat16)
        _check_state(m[i], rm)
        _check_state(v[i], np.sqrt(rv))


def test_8_bit_blocks_with_non_finite_values(gpu):
    n = 32 * 6 + 5
    p, g = torch.ones(n, device=gpu), torch.full((n,), 0.5, device=gpu)
    g[40] = float("nan")
    g[70] = float("inf")
    m, v = [mxfp8gg.adamw_state(p, 8)], [mxfp8gg.adamw_state(p, 8)]
    mxfp8gg.adamw_step([p], [g], m, v, step=1)
    for s in (m, v):
        x = R.mx8_values(_bytes(s[0][0]), _bytes(s[0][1]))
        assert np.isnan(x[32:96]).all() and np.isfinite(np.delete(x, slice(32, 96))).all()
    assert torch.isnan(p[40]) and torch.isfinite(p[:40]).all() and torch.isfinite(p[96:]).all()


def test_unaligned_views(gpu):
    """Views that start one element into their storage: the same bits."""
    params, grads, m, v = _tensors(gpu, [1001, 5000], torch.bfloat16, torch.bfloat16, 3)
    shift = lambda t: torch.cat([t[:1], t])[1:]  # noqa: E731
    for small in (False, True):
        st = [[_pack(t) if small else t.clone() for t in x] for x in (m, v)]
        st2 = [[tuple(map(shift, t)) if small else shift(t) for t in x] for x in st]
        a, b = [p.clone() for p in params], [shift(p) for p in params]
        mxfp8gg.adamw_step(a, grads, *st, **HYPER)
        mxfp8gg.adamw_step(b, [shift(g) for g in grads], *st2, **HYPER)
        for x, y in zip(a, b):
            assert torch.equal(x, y)
        flat = lambda s: [t for x in s for e in x for t in (e if small else (e,))]  # noqa: E731
        for x, y in zip(flat(st), flat(st2)):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


def test_first_step_from_zero_state(gpu):
    p = torch.full((100,), 2.0, device=gpu)
    g = torch.cat([torch.full((50,), 3e-3, device=gpu), torch.zeros(50, device=gpu)])
    for bits in (32, 8):
        q = p.clone()
        mxfp8gg.adamw_step([q], [g], [mxfp8gg.adamw_state(p, bits)], [mxfp8gg.adamw_state(p, bits)],
                           step=1, lr=0.1, weight_decay=0.0)
        assert torch.allclose(q[:50], torch.full((50,), 1.9, device=gpu), atol=1e-5)
        assert (q[50:] == 2.0).all()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("master", [True, False])
def test_optimizer(gpu, bits, master):
    """Groups, skipped parameters, schedulers, the version counter that weight
    caches watch, and a state that survives saving."""
    g = torch.Generator().manual_seed(4)
    make = lambda *s: torch.nn.Parameter(torch.randn(s, generator=g).to(torch.bfloat16).to(gpu))  # noqa: E731
    a, b, c, d = make(40, 33), make(129), make(7), make(64, 2)
    opt = mxfp8gg.AdamW([dict(params=[a, b]), dict(params=[c, d], lr=1e-2, weight_decay=0.0)],
                        lr=1e-3, state_bits=bits, master_weights=master)
    sched = torch.optim.lr_scheduler.LambdaLR(opt, lambda n: 0.5 ** n)
    for k in range(3):
        opt.zero_grad()
        for p in (a, b, d) if k else (a, b):
            p.grad = torch.randn(p.shape, generator=g).to(torch.bfloat16).to(gpu)
        d_t = d.grad
        if d_t is not None:
            d.grad = d_t.t().contiguous().t()            # another layout
        versions = [p._version for p in (a, b, c, d)]
        old = [p.detach().clone() for p in (a, b, c, d)]
        opt.step()
        sched.step()
        moved = [p._version > n for p, n in zip((a, b, c, d), versions)]
        assert moved == [True, True, False, k > 0]
        assert torch.equal(c, old[2]) and not torch.equal(a, old[0])
    assert opt.state[a]["step"] == 3 and opt.state[d]["step"] == 2 and not opt.state.get(c)
    # the step of a saved and loaded optimizer is the step of the original
    saved = copy.deepcopy(opt.state_dict())
    twins = [torch.nn.Parameter(p.detach().clone()) for p in (a, b, c, d)]
    other = mxfp8gg.AdamW([dict(params=twins[:2]), dict(params=twins[2:], lr=1e-2)], lr=1e-3)
    other.load_state_dict(saved)
    for p, q in zip((a, b, c, d), twins):
        p.grad = q.grad = torch.randn(p.shape, generator=g).to(torch.bfloat16).to(gpu)
    opt.step()
    other.step()
    for p, q in zip((a, b, c, d), twins):
        assert torch.equal(p, q)
        for k, v in opt.state[p].items():
            w = other.state[q][k]
            assert v == w if not isinstance(v, torch.Tensor) else (
                v.dtype == w.dtype and torch.equal(v.view(torch.uint8), w.view(torch.uint8)))


def test_weight_cache_sees_the_step(gpu):
    w = torch.nn.Parameter(torch.randn((2, 64, 64), device=gpu).to(torch.bfloat16))
    cache = mxfp8gg.WeightCastCache()
    cache.get(w)
    opt = mxfp8gg.AdamW([w], lr=0.1)
    w.grad = torch.ones_like(w)
    opt.step()
    (q, _), _ = cache.get(w)
    assert cache.misses == 2
    want, _ = mxfp8gg.to_mxfp8_dim0(w.detach())
    assert torch.equal(q.view(torch.uint8), want.view(torch.uint8))


def test_other_stream(gpu):
    params, grads, m, v = _tensors(gpu, [70000], torch.float32, torch.float32, 5)
    twin = [[t.clone() for t in x] for x in (params, m, v)]
    mxfp8gg.adamw_step(params, grads, m, v, **HYPER)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        mxfp8gg.adamw_step(twin[0], grads, twin[1], twin[2], **HYPER)
    side.synchronize()
    assert torch.equal(params[0], twin[0][0]) and torch.equal(v[0], twin[2][0])


def test_refusals(gpu):
    p, g = torch.zeros(64, device=gpu), torch.zeros(64, device=gpu)
    s = lambda: torch.zeros(64, device=gpu)  # noqa: E731
    ok = dict(params=[p], grads=[g], exp_avg=[s()], exp_avg_sq=[s()], step=1)
    mxfp8gg.adamw_step(**ok)
    mxfp8gg.adamw_step([], [], [], [], step=1)
    pair = mxfp8gg.adamw_state(p, 8)
    for bad in (dict(grads=[]), dict(masters=[s(), s()]), dict(step=0), dict(lr=-1.0),
                dict(betas=(1.0, 0.9)), dict(eps=float("nan")), dict(grads=[g[:32]]),
                dict(grads=[g.cpu()]), dict(exp_avg=[pair]), dict(params=[p.cpu()]),
                dict(exp_avg=[pair], exp_avg_sq=[(pair[0], pair[1][:1])]),
                dict(grads=[torch.zeros(128, device=gpu)[::2]])):
        with pytest.raises(ValueError):
            mxfp8gg.adamw_step(**{**ok, **bad})
    for bad in (dict(params=[p.half()]), dict(grads=[g.half()]), dict(exp_avg=[s().bfloat16()]),
                dict(masters=[s().bfloat16()])):
        with pytest.raises(TypeError):
            mxfp8gg.adamw_step(**{**ok, **bad})
    with pytest.raises(ValueError):
        mxfp8gg.AdamW([torch.nn.Parameter(p)], state_bits=16)
    with pytest.raises(ValueError):
        mxfp8gg.AdamW([torch.nn.Parameter(p)], lr=-1.0)
