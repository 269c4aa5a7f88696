"""GPU parity of the block-scaled e4m3 casts and products.

Casts are compared bit for bit with the definition: scale max(amax / 448, 2^-126) in
fp32, payload the format's rounding of x * (1 / scale).

Products against 64 bits, S the sum of the products' magnitudes.  The matrix instruction
aligns each eight consecutive products of e4m3 values to the largest of them and cuts what
lies 13 bits below its exponent (seen from its results: beside a product of 2^16 one of 2^3
is kept and one of 2^2 is not; from the ninth position on down to 2^-7): the other seven
lose less than 2^-13 of the largest each, at most 7 * 2^-13 S in all.  The sixteen sums of
eight are added in fp32, with the block under its scale, itself the product of two: at most
(16 + blocks + 4) roundings of one unit, 2^-23 S.  bf16 outputs: half a step, 2^-8 of the
value, more.
"""
import pytest
import torch

import mxfp8gg

pytestmark = pytest.mark.gpu

FP8 = torch.float8_e4m3fn


def _x(gpu, *shape, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * scale
    x = x * torch.exp2(torch.randint(-6, 7, (*shape[:-1], 1), generator=g).float())
    return x.to(torch.bfloat16).to(gpu)


def _pad(x, *dims):
    size = list(x.shape)
    for d in dims:
        size[d] = (size[d] + 127) // 128 * 128
    out = x.new_zeros(size)
    out[tuple(slice(0, n) for n in x.shape)] = x
    return out


def _cast(b, dims):
    """(payload, scale) of fp32 blocks spanning `dims` of b."""
    a = b.abs().amax(dim=dims, keepdim=True)
    # a quotient of tensors: by a number torch multiplies with its reciprocal
    s = torch.clamp(a / torch.full_like(a, 448.0), min=2.0 ** -126)
    return (b * (1 / s)).to(FP8), s


def _ref_rows(x):
    b = _pad(x.float(), 1).view(x.shape[0], -1, 128)
    q, s = _cast(b, 2)
    return q.view(x.shape[0], -1)[:, :x.shape[1]], s[:, :, 0]


def _ref_tiles(w):
    b = _pad(w.float(), 0, 1)
    v = b.view(b.shape[0] // 128, 128, -1, 128)
    q, s = _cast(v, (1, 3))
    return q.view(b.shape)[:w.shape[0], :w.shape[1]], s[:, 0, :, 0]


def _same(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def _wide(q, s, tile=False):
    """Values of a payload under its scales, in 64 bits."""
    s = s.double().repeat_interleave(128, 1)[:, :q.shape[1]]
    if tile:
        s = s.repeat_interleave(128, 0)[:q.shape[0]]
    return q.double() * s


def _near(got, want, size, blocks):
    err = (got.double() - want).abs()
    bound = (7 * 2.0 ** -13 + (16 + blocks + 4) * 2.0 ** -23) * size
    if got.dtype is torch.bfloat16:
        bound = bound + 2.0 ** -8 * (want.abs() + bound)
    bad = err > bound
    assert not bool(bad.any()), (torch.nonzero(bad)[0].tolist(), float(err[bad][0]),
                                 float(bound[bad][0]), int(bad.sum()))


@pytest.mark.parametrize("M,K", [(1, 16), (1, 7168), (3, 128), (33, 144), (130, 2048), (257, 1008)])
def test_cast_rows(gpu, M, K):
    x = _x(gpu, M, K, seed=M + K)
    x[0, :16] = 0
    if M > 2:
        x[2] = 0
    q, s = mxfp8gg.to_fp8_block_dim0(x)
    rq, rs = _ref_rows(x)
    assert q.shape == (M, K) and s.shape == rs.shape
    assert _same(q, rq) and torch.equal(s, rs)
    wide = torch.zeros((M, K + 24), dtype=torch.bfloat16, device=gpu)
    wide[:, 8:8 + K] = x                          # a view with a row stride
    q2, s2 = mxfp8gg.to_fp8_block_dim0(wide[:, 8:8 + K])
    assert _same(q2, q) and torch.equal(s2, s)


def test_cast_extremes(gpu):
    x = torch.zeros((6, 256), dtype=torch.bfloat16, device=gpu)
    x[1, 3] = 1e-38
    x[2, 5] = 3e38
    x[3, 7] = float("inf")
    x[4, 130] = float("nan")
    x[5] = 448.0
    q, s = mxfp8gg.to_fp8_block_dim0(x)
    assert float(s[0, 0]) == 2.0 ** -126 and not q[0].float().any()
    assert float(q[2, 5]) == 448.0
    assert torch.isinf(s[3, 0]) and torch.isnan(q[3, 7].float()) and float(s[3, 1]) == 2.0 ** -126
    assert torch.isnan(s[4, 1]) and torch.isnan(q[4, 128:].float()).all()
    assert not q[4, :128].float().any()
    assert (s[5] == 1).all() and (q[5].float() == 448).all()
    # the tile cast of the same values
    q, s = mxfp8gg.to_fp8_block_weight(x)
    assert torch.isinf(s[0, 0]) and torch.isnan(s[0, 1])


@pytest.mark.parametrize("shape", [(16, 16), (128, 128), (130, 144), (2, 160, 272), (3, 256, 128)])
def test_cast_weight(gpu, shape):
    w = _x(gpu, *shape, seed=sum(shape))
    q, s = mxfp8gg.to_fp8_block_weight(w)
    three = w if w.dim() == 3 else w[None]
    for e in range(three.shape[0]):
        rq, rs = _ref_tiles(three[e])
        assert _same(q.view(three.shape)[e], rq)
        assert torch.equal(s.view(three.shape[0], *rs.shape)[e], rs)
    if shape[-2] % 16 == 0:
        q2, s2, qt, st = mxfp8gg.to_fp8_block_weight(w, dual=True)
        assert _same(q2, q) and torch.equal(s2, s)
        assert _same(qt, q.transpose(-1, -2)) and torch.equal(st, s.transpose(-1, -2))


@pytest.mark.parametrize("sizes,C", [(None, 144), ([5, 0, 300, 128], 128), ([0, 1, 129], 1040),
                                     ([0, 0], 16), ([256, 64], 272)])
def test_cast_tokens(gpu, sizes, C):
    M = 391 if sizes is None else sum(sizes) + 3
    x = _x(gpu, M, C, seed=C)
    offs = None if sizes is None else torch.tensor(sizes, device=gpu).cumsum(0).int()
    qt, st, pad = mxfp8gg.to_fp8_block_dim1(x, offs)
    q, s, qt2, st2, _ = mxfp8gg.block._dim1(x, offs, True)
    assert _same(qt2, qt) and torch.equal(st2, st)
    rq, rs = _ref_rows(x)
    last = M if sizes is None else sum(sizes)
    assert _same(q[:last], rq[:last]) and torch.equal(s[:last], rs[:last])
    at = row = 0
    for i, n in enumerate([M] if sizes is None else sizes):
        full = (n + 127) // 128 * 128
        if n:
            b = _pad(x[row:row + n].float(), 0).t()
            eq, es = _ref_rows(b)
            assert _same(qt[:, at:at + full], eq) and torch.equal(st[:, at // 128:(at + full) // 128], es)
        row += n
        at += full
        assert pad is None or int(pad[i]) == at
    assert not qt[:, at:].float().any()


def _weights(gpu, E, N, K, seed):
    w = _x(gpu, E, N, K, seed=seed, scale=K ** -0.5)
    return mxfp8gg.to_fp8_block_weight(w)


MM = [(1, 16, 16), (1, 4096, 7168), (5, 130, 144), (16, 256, 1024), (17, 48, 2064), (33, 100, 400),
      (64, 272, 512), (65, 128, 128), (100, 130, 1040), (128, 384, 256), (200, 2112, 784),
      (257, 300, 272), (700, 1000, 144), (2049, 4000, 400), (4096, 4096, 256)]


@pytest.mark.parametrize("M,N,K", MM)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_mm(gpu, M, N, K, dtype):
    x = _x(gpu, M, K, seed=M + N)
    q, s = mxfp8gg.to_fp8_block_dim0(x)
    wq, ws = _weights(gpu, 1, N, K, seed=N)
    wq, ws = wq[0], ws[0]
    y = mxfp8gg.fp8_block_mm(q, s, wq, ws, out_dtype=dtype)
    a, b = _wide(q, s), _wide(wq, ws, True)
    _near(y, a @ b.t(), a.abs() @ b.abs().t(), (K + 127) // 128)
    assert torch.equal(y, mxfp8gg.fp8_block_mm(q, s.contiguous(), wq, ws, out_dtype=dtype))


@pytest.mark.parametrize("sizes,N,K", [([3, 0, 9, 1], 144, 272), ([0, 0, 0, 1], 256, 128),
                                       ([70, 0, 300, 129, 1], 272, 400), ([1000, 0, 24, 300], 520, 144),
                                       ([513, 2000, 0, 255, 1300], 2000, 256), ([0, 0], 16, 16),
                                       ([5] * 100, 64, 128)])
def test_grouped_mm(gpu, sizes, N, K):
    M = sum(sizes) + 5
    x = _x(gpu, M, K, seed=M)
    q, s = mxfp8gg.to_fp8_block_dim0(x)
    wq, ws = _weights(gpu, len(sizes), N, K, seed=N)
    offs = torch.tensor(sizes, device=gpu).cumsum(0).int()
    y = mxfp8gg.fp8_block_mm(q, s, wq, ws, offs)
    at = 0
    for e, n in enumerate(sizes):
        a, b = _wide(q[at:at + n], s[at:at + n]), _wide(wq[e], ws[e], True)
        _near(y[at:at + n], a @ b.t(), a.abs() @ b.abs().t(), (K + 127) // 128)
        at += n


@pytest.mark.parametrize("M,N,K", [(1, 16, 16), (130, 144, 272), (1000, 256, 512), (300, 4096, 4112)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_wgrad(gpu, M, N, K, dtype):
    gt, gs, _ = mxfp8gg.to_fp8_block_dim1(_x(gpu, M, N, seed=M))
    xt, xs, _ = mxfp8gg.to_fp8_block_dim1(_x(gpu, M, K, seed=K))
    dw = mxfp8gg.fp8_block_wgrad(gt, gs, xt, xs, out_dtype=dtype)
    a, b = _wide(gt, gs), _wide(xt, xs)
    _near(dw, a @ b.t(), a.abs() @ b.abs().t(), gt.shape[1] // 128)


@pytest.mark.parametrize("sizes,N,K", [([3, 0, 200, 129], 144, 272), ([700, 0, 0, 1000], 2064, 1024)])
def test_grouped_wgrad(gpu, sizes, N, K):
    M = sum(sizes) + 7
    offs = torch.tensor(sizes, device=gpu).cumsum(0).int()
    gt, gs, pad = mxfp8gg.to_fp8_block_dim1(_x(gpu, M, N, seed=M), offs)
    xt, xs, _ = mxfp8gg.to_fp8_block_dim1(_x(gpu, M, K, seed=K), offs)
    dw = mxfp8gg.fp8_block_wgrad(gt, gs, xt, xs, pad)
    at = 0
    for e, n in enumerate(sizes):
        one = slice(at, at + (n + 127) // 128 * 128)
        blk = slice(one.start // 128, one.stop // 128)
        at = one.stop
        a, b = _wide(gt[:, one], gs[:, blk]), _wide(xt[:, one], xs[:, blk])
        if n == 0:
            assert not dw[e].any()
        _near(dw[e], a @ b.t(), a.abs() @ b.abs().t(), 1 + n // 128)
