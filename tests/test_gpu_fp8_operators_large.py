"""Tensors of more than 2^31 elements: the last rows, found from the end of the memory,
are those of a call on these rows alone."""
import pytest
import torch

import mxfp8gg

pytestmark = pytest.mark.gpu


def _big(rows, cols, seed, dtype=torch.bfloat16):
    """Zeros but for the last 256 rows."""
    x = torch.zeros((rows, cols), dtype=dtype, device="cuda")
    g = torch.Generator().manual_seed(seed)
    x[-256:] = torch.randn((256, cols), generator=g).to(dtype).cuda()
    return x


def _equal(a, b):
    assert torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def test_block_casts_and_product(gpu):
    """Payloads of more than 2^31 bytes, a result of more than 2^31 elements."""
    M, K, N = 262144 + 256, 8256, 8320
    x = _big(M, K, 0)
    q, s = mxfp8gg.to_fp8_block_dim0(x)
    ql, sl = mxfp8gg.to_fp8_block_dim0(x[-256:])
    _equal(q[-256:], ql)
    _equal(s[-256:], sl)
    qt, st = mxfp8gg.to_fp8_block_dim1(x)[:2]
    qtl, stl = mxfp8gg.to_fp8_block_dim1(x[-256:])[:2]
    _equal(qt[:, -256:], qtl)
    _equal(st[:, -2:], stl)
    del x, qt, st
    w, ws = mxfp8gg.to_fp8_block_weight(
        torch.randn((N, K), generator=torch.Generator().manual_seed(1)).bfloat16().cuda())
    y = mxfp8gg.fp8_block_mm(q, s, w, ws)
    assert y.numel() > 1 << 31
    exact = (ql.double().view(256, -1) * sl.double().repeat_interleave(128, 1)[:, :K]) @ (
        w.double() * ws.double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]).t()
    # bf16's rounding and the products' (far smaller): half a step, and 2^-9 of a row's size
    err = (y[-256:].double() - exact).abs()
    assert (err <= exact.abs() * 2.0 ** -8 + exact.abs().amax() * 2.0 ** -9).all()
    assert not y[:-256].any()


@pytest.mark.parametrize("need", ["norm", "quant"])
def test_add_norm(gpu, need):
    M, K = 262144 + 256, 8256
    x, r = _big(M, K, 0), _big(M, K, 1)
    w = torch.linspace(0.5, 1.5, K, device=gpu)
    if need == "quant":
        got, want = (mxfp8gg.rms_norm_quant(a, w, b) for a, b in ((x, r), (x[-256:], r[-256:])))
        for a, b in zip(got, want):
            _equal(a[-256:], b)
        return
    xg = x.requires_grad_(True)
    y, h = mxfp8gg.add_rms_norm(xg, r, w)
    xl = x.detach()[-256:].requires_grad_(True)
    yl, hl = mxfp8gg.add_rms_norm(xl, r[-256:], w)
    _equal(y.detach()[-256:], yl.detach())
    _equal(h.detach()[-256:], hl.detach())
    torch.autograd.backward([y, h], [r, r])
    torch.autograd.backward([yl, hl], [r[-256:], r[-256:]])
    _equal(xg.grad[-256:], xl.grad)


def test_log_probs(gpu):
    T, V = 16640, 131088
    z = _big(T, V, 0).requires_grad_(True)
    t = torch.arange(T, device=gpu) * 7 % V
    r = mxfp8gg.token_log_probs(z, t, topk=4)
    tail = z.detach()[-256:].double()
    lp = tail.log_softmax(1)
    assert z.numel() > 1 << 31
    # sums of V terms of one sign in fp32, in parts: far below 2^-12 of log probabilities near 11
    assert (r.log_probs[-256:] - lp.gather(1, t[-256:, None])[:, 0]).abs().max() < 2.0 ** -12
    assert (r.entropy[-256:] + (lp.exp() * lp).sum(1)).abs().max() < 2.0 ** -12
    assert (r.top_log_probs[-256:] - lp.topk(4).values).abs().max() < 2.0 ** -12
    assert torch.equal(tail.gather(1, r.top_ids[-256:].long()), tail.topk(4).values)
    r.log_probs.sum().backward()
    want = -lp.exp()
    want[torch.arange(256), t[-256:]] += 1
    got = z.grad[-256:].double()
    assert ((got - want).abs() <= want.abs() * 2.0 ** -8 * 1.01 + 1e-12).all()


def test_clip(gpu):
    n = (1 << 31) + 12345
    g = torch.zeros(n, dtype=torch.bfloat16, device=gpu)
    g[-5:] = 3.0
    g[0] = 6.0
    small = torch.full((7,), 1.0, device=gpu)
    norm = mxfp8gg.clip_grad_norm_([g, small], 1.0)
    want = (45 + 36 + 7) ** 0.5
    assert abs(float(norm) - want) < want * 2.0 ** -22
    scale = 1 / (want + 1e-6)
    assert abs(float(g[-1]) - 3 * scale) <= 3 * scale * 2.0 ** -8 * 1.01
    assert abs(float(g[0]) - 6 * scale) <= 6 * scale * 2.0 ** -8 * 1.01
    assert abs(float(small[3]) - scale) <= scale * 2.0 ** -22
    assert int(torch.count_nonzero(g)) == 6
