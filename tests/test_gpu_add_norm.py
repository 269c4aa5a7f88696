"""GPU parity of add_rms_norm and rms_norm_quant with the 64-bit definition.

h is the fp32 sum rounded to its type: the same bits as torch's addition.  y, dx and
dweight as in the norms' own tests: statistics are fp32 sums of cols terms with a
relative error below 5e-6; 2e-5 of a row's largest magnitude, and half a step, 2^-8 of
the value, for bf16 outputs.  8-bit outputs: the value before rounding is within 2e-5
of its row's largest magnitude (relative, xhat's error is proportional to xhat: 1e-5 of the
value); the stored one is off by half a step more, 2^-4 of the value, or half the
format's smallest step under the scale.
"""
import pytest
import torch

import mxfp8gg

pytestmark = pytest.mark.gpu

SHAPES = [(1, 32), (1, 7168), (3, 64), (17, 1024), (600, 96), (33, 1056), (130, 4128), (5, 8192),
          (3, 16416), (2, 32768), (1100, 2080)]


def _inputs(gpu, rows, cols, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + rows + cols)
    make = lambda s, m=0.0: (torch.randn((rows, cols), generator=g) * s + m).to(dtype).to(gpu)  # noqa: E731
    w = (1 + 0.2 * torch.randn(cols, generator=g)).to(gpu)
    return make(0.7), make(1.7, 0.2), w, make(1.0), make(0.5)


def _norm(h, w, eps=1e-6):
    h = h.double()
    r = (h.square().mean(dim=-1, keepdim=True) + eps).rsqrt()
    return h * r * (1.0 if w is None else w.double()), r


def _close(got, want, bound):
    if got.dtype is torch.bfloat16:
        bound = bound + 2.0 ** -8 * want.abs()
    bad = (got.double() - want).abs() > bound
    assert not bool(bad.any()), (torch.nonzero(bad)[0].tolist(), float(got[bad][0]), float(want[bad][0]))


def _top(x):
    return x.abs().amax(dim=-1, keepdim=True)


@pytest.mark.parametrize("rows,cols", SHAPES + [(1, 1), (4, 7), (70, 1001), (9, 4100)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_forward_and_gradients(gpu, rows, cols, dtype):
    x, res, w, dy, dh = _inputs(gpu, rows, cols, dtype)
    for weight in (w, w.to(torch.bfloat16), None):
        leaves = [t.detach().requires_grad_(True) for t in (x, res) + (() if weight is None else (weight,))]
        y, h = mxfp8gg.add_rms_norm(*leaves[:2], leaves[2] if weight is not None else None)
        with torch.no_grad():
            y2, h2 = mxfp8gg.add_rms_norm(x, res, weight)
        assert torch.equal(y, y2) and torch.equal(h, h2)
        assert torch.equal(h, x + res)
        want, r = _norm(h.detach(), weight)
        ww = 1.0 if weight is None else weight.double()
        _close(y, want, 2e-5 * _top(want))
        for up in ((dy, dh), (dy, None), (None, dh)):
            used = [(o, u) for o, u in zip((y, h), up) if u is not None]
            got = torch.autograd.grad([o for o, _ in used], leaves, [u for _, u in used],
                                      retain_graph=True, allow_unused=True)
            dyd = torch.zeros_like(want) if up[0] is None else dy.double()
            u = dyd * ww
            xhat = h.detach().double() * r
            d = r * (u - xhat * (u * xhat).mean(dim=-1, keepdim=True))
            d = d + (0 if up[1] is None else dh.double())
            bound = 2e-5 * r * _top(u) * (2 + _top(xhat)) + 2.0 ** -24 * _top(dh.double())
            assert torch.equal(got[0], got[1]) and got[0].dtype is dtype
            _close(got[0], d, bound)
            if weight is not None:
                _close(got[2], (dyd * xhat).sum(dim=0), 2e-5 * (dyd * xhat).abs().sum(dim=0))


def test_gradient_by_differences(gpu):
    g = torch.Generator().manual_seed(3)
    x, res, dy, dh = (torch.randn((3, 40), generator=g).to(gpu) for _ in range(4))
    w = torch.rand(40, generator=g).to(gpu) + 0.5
    leaves = [t.clone().requires_grad_(True) for t in (x, res, w)]
    grads = torch.autograd.grad(mxfp8gg.add_rms_norm(*leaves), leaves, (dy, dh))

    def f(a, b, c):
        h = a + b
        return (_norm(h, c)[0] * dy).sum() + (h * dh).sum()

    for i, got in enumerate(grads):
        args = [t.double() for t in (x, res, w)]
        step = torch.randn(args[i].shape, generator=g).double().to(gpu)
        e = 1e-6
        hi, lo = list(args), list(args)
        hi[i], lo[i] = args[i] + e * step, args[i] - e * step
        slope = float((f(*hi) - f(*lo)) / (2 * e))
        assert abs(slope - float((got.double() * step).sum())) < 1e-3 * max(1.0, abs(slope))


def _mx_values(q, s):
    up = torch.exp2(s.double() - 127)
    return q.double() * up.repeat_interleave(32, 1), up.repeat_interleave(32, 1)


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("mode", ["rceil", "floor"])
def test_mxfp8(gpu, rows, cols, dtype, mode):
    x, res, w, _, _ = _inputs(gpu, rows, cols, dtype)
    x[:, :32] = 0
    res[:, :32] = 0
    q, s, h = mxfp8gg.rms_norm_quant(x, w, res, scaling_mode=mode)
    assert q.shape == (rows, cols) and s.shape == (rows, cols // 32) and torch.equal(h, x + res)
    want, _ = _norm(h, w)
    got, up = _mx_values(q, s)
    size = want.abs().clamp_max(448 * up) if mode == "floor" else want.abs()
    target = torch.sign(want) * size
    bound = 1e-5 * want.abs() + 2.0 ** -4 * size + 2.0 ** -10 * up
    assert not bool(((got - target).abs() > bound).any())
    # scales: exact wherever the block's largest value is not at the edge of two
    amax = want.view(rows, -1, 32).abs().amax(dim=2)
    j = torch.ceil(torch.log2(amax / 448)) if mode == "rceil" else torch.floor(torch.log2(amax)) - 8
    edge = torch.log2(amax / 448 if mode == "rceil" else amax)
    sure = (edge - edge.round()).abs() > 1e-4
    expect = torch.where(amax > 0, (j + 127).clamp(0, 254), torch.zeros_like(j))
    ok = (s.double() == expect) | ~(sure | (amax == 0))
    assert bool(ok.all())
    # without the residual: of h itself
    q2, s2, none = mxfp8gg.rms_norm_quant(h, w, scaling_mode=mode)
    assert none is None and torch.equal(s2, s)
    assert torch.equal(q2.view(torch.uint8), q.view(torch.uint8))


@pytest.mark.parametrize("rows,cols", SHAPES + [(4, 16), (70, 1008), (9, 144), (5, 4112)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_fp8_block(gpu, rows, cols, dtype):
    x, res, w, _, _ = _inputs(gpu, rows, cols, dtype)
    q, s, h = mxfp8gg.rms_norm_quant(x, w, res, out_format="fp8_block")
    blocks = (cols + 127) // 128
    assert q.shape == (rows, cols) and s.shape == (rows, blocks) and s.dtype is torch.float32
    want, _ = _norm(h, w)
    up = s.double().repeat_interleave(128, 1)[:, :cols]
    assert not bool(((q.double() * up - want).abs()
                     > 1e-5 * want.abs() + 2.0 ** -4 * want.abs() + 2.0 ** -10 * up).any())
    pad = torch.zeros((rows, blocks * 128), dtype=torch.float64, device=gpu)
    pad[:, :cols] = want
    amax = pad.view(rows, -1, 128).abs().amax(dim=2)
    torch.testing.assert_close(s.double(), amax / 448, rtol=1e-5, atol=0)
    q2, s2, _ = mxfp8gg.rms_norm_quant(h, w, out_format="fp8_block")
    assert torch.equal(s2, s) and torch.equal(q2.view(torch.uint8), q.view(torch.uint8))


def test_feeds_the_products(gpu):
    x, res, w, _, _ = _inputs(gpu, 70, 512, torch.bfloat16)
    g = torch.Generator().manual_seed(5)
    weight = (torch.randn((256, 512), generator=g) / 22).to(torch.bfloat16).to(gpu)
    want = _norm(x + res, w)[0]
    q, s, _ = mxfp8gg.rms_norm_quant(x, w, res, out_format="fp8_block")
    y = mxfp8gg.fp8_block_mm(q, s, *mxfp8gg.to_fp8_block_weight(weight))
    q, s, _ = mxfp8gg.rms_norm_quant(x, w, res)
    wq, ws = mxfp8gg.to_mxfp8_dim0(weight[None])
    offs = torch.tensor([70], dtype=torch.int32, device=gpu)
    z = mxfp8gg.grouped_mm(q, wq, offs, s, ws)
    ref = want @ weight.double().t()
    # both operands rounded to 2^-4 of each value: at most 2 * 2^-4 + 2^-8 of the magnitudes' sum
    size = want.abs() @ weight.double().abs().t()
    for got in (y, z):
        assert float(((got.double() - ref).abs() / size).max()) < 2 * 2.0 ** -4 + 2.0 ** -7


def test_strides_and_shapes(gpu):
    x, res, w, dy, _ = _inputs(gpu, 24, 96, torch.bfloat16)
    wide = torch.zeros((24, 200), dtype=torch.bfloat16, device=gpu)
    wide[:, 3:99] = x
    y, h = mxfp8gg.add_rms_norm(wide[:, 3:99], res.t().contiguous().t(), w)
    y2, h2 = mxfp8gg.add_rms_norm(x, res, w)
    assert torch.equal(y, y2) and torch.equal(h, h2)
    y3, h3 = mxfp8gg.add_rms_norm(x.view(2, 3, 4, 96), res.view(2, 3, 4, 96), w)
    assert y3.shape == h3.shape == (2, 3, 4, 96) and torch.equal(y3.view(24, 96), y)
    q, s, h4 = mxfp8gg.rms_norm_quant(wide[:, 3:99], w, res)
    q5, s5, h5 = mxfp8gg.rms_norm_quant(x.view(4, 6, 96), w, res.view(4, 6, 96))
    assert torch.equal(q.view(torch.uint8), q5.view(torch.uint8)) and torch.equal(s, s5)
    assert torch.equal(h4, h5.view(24, 96))
    e = x.new_zeros((0, 96))
    y, h = mxfp8gg.add_rms_norm(e, e, w)
    assert y.shape == h.shape == (0, 96)
    q, s, h = mxfp8gg.rms_norm_quant(e, w, e)
    assert q.shape == (0, 96) and s.shape == (0, 3)


def test_non_finite_rows(gpu):
    x = torch.ones((3, 256), device=gpu)
    x[1, 5] = float("inf")
    x[2, 7] = float("nan")
    for fmt in ("mxfp8", "fp8_block"):
        q, s, _ = mxfp8gg.rms_norm_quant(x, out_format=fmt)
        v = q.float()
        assert torch.isfinite(v[0]).all() and (v[0] != 0).all()
        assert torch.isnan(v[1, 5]) and torch.isnan(v[2]).all()


def test_refusals(gpu):
    x = torch.zeros((4, 96), device=gpu)
    m = mxfp8gg
    for call in (lambda: m.add_rms_norm(x, x[:2]), lambda: m.add_rms_norm(x, x.bfloat16()),
                 lambda: m.add_rms_norm(x, x, x[0, :5]), lambda: m.add_rms_norm(x, x.cpu()),
                 lambda: m.rms_norm_quant(x[:, :40].contiguous()),
                 lambda: m.rms_norm_quant(x[:, :40].contiguous(), out_format="fp8_block"),
                 lambda: m.rms_norm_quant(x, out_format="int8"),
                 lambda: m.rms_norm_quant(x, scaling_mode="even"),
                 lambda: m.add_rms_norm(torch.zeros((2, 32769), device=gpu), torch.zeros((2, 32769), device=gpu))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        m.add_rms_norm(x.half(), x.half())
    with pytest.raises(TypeError):
        m.add_rms_norm(x, None)
    with pytest.raises(RuntimeError, match="no gradient"):
        m.rms_norm_quant(x.requires_grad_(True))
    y, _ = m.add_rms_norm(x, x.detach())
    with pytest.raises(RuntimeError, match="differentiated twice"):
        torch.autograd.grad(y.sum(), x, create_graph=True)
