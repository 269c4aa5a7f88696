"""GPU parity of the block-scaled e4m3 casts and products.

Casts are compared bit for bit with the definition: scale max(amax (1 / 448), 2^-126) in
fp32, payload the format's rounding of the fp32 quotient x / scale.

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
    s = torch.clamp(a * (torch.ones_like(a) / torch.full_like(a, 448.0)), min=2.0 ** -126)
    return (b / s).to(FP8), s


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


MM = [(300, 400, 4112), (1003, 2112, 1040), (70, 20, 8192), (1, 16, 16), (1, 4096, 7168), (5, 130, 144), (16, 256, 1024), (17, 48, 2064), (33, 100, 400),
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
                                       ([5] * 100, 64, 128), ([90, 0, 200, 33], 144, 2064)])
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


@pytest.mark.parametrize("M,N,K", [(1, 16, 16), (130, 144, 272), (1000, 256, 512), (300, 4096, 4112),
                                   (5000, 144, 160)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_wgrad(gpu, M, N, K, dtype):
    gt, gs, _ = mxfp8gg.to_fp8_block_dim1(_x(gpu, M, N, seed=M))
    xt, xs, _ = mxfp8gg.to_fp8_block_dim1(_x(gpu, M, K, seed=K))
    dw = mxfp8gg.fp8_block_wgrad(gt, gs, xt, xs, out_dtype=dtype)
    a, b = _wide(gt, gs), _wide(xt, xs)
    _near(dw, a @ b.t(), a.abs() @ b.abs().t(), gt.shape[1] // 128)


@pytest.mark.parametrize("sizes,N,K", [([3, 0, 200, 129], 144, 272), ([700, 0, 0, 1000], 2064, 1024), ([3000, 1, 0, 5000], 128, 272)])
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


def _dequant_rows(x):
    return _wide(*_ref_rows(x))


def _dequant_tokens(x):
    """Values of x [M, C] in blocks of 128 tokens, transposed: [C, M padded]."""
    return _wide(*_ref_rows(_pad(x.float(), 0).t()))


@pytest.mark.parametrize("sizes,N,K", [(None, 144, 272), (None, 256, 1024), ([40, 0, 129, 300], 272, 144),
                                       ([0, 0, 5], 128, 128)])
def test_linear_gradients(gpu, sizes, N, K):
    M = 333 if sizes is None else sum(sizes) + 4
    E = 1 if sizes is None else len(sizes)
    x, dy = _x(gpu, M, K, seed=1), _x(gpu, M, N, seed=2, scale=1e-2)
    w = _x(gpu, E, N, K, seed=3, scale=K ** -0.5)
    offs = None if sizes is None else torch.tensor(sizes, device=gpu).cumsum(0).int()
    leaves = [x.requires_grad_(True), (w[0] if sizes is None else w).detach().requires_grad_(True)]
    y = mxfp8gg.fp8_block_linear(*leaves, offs)
    dx, dw = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    dw = dw.view(E, N, K)
    at = 0
    for e, n in enumerate([M] if sizes is None else sizes):
        one = slice(at, at + n)
        at += n
        if n == 0:
            assert not dw[e].any()
            continue
        xe, ge = x.detach()[one], dy[one]
        wq = _wide(*_ref_tiles(w[e]), True)
        for got, a, b in ((y.detach()[one], _dequant_rows(xe), wq), (dx[one], _dequant_rows(ge), wq.t()),
                          (dw[e], _dequant_tokens(ge), _dequant_tokens(xe))):
            _near(got, a @ b.t(), a.abs() @ b.abs().t(), (a.shape[1] + 127) // 128)
    assert not y[at:].any() and not dx[at:].any()         # rows past the groups
    # each gradient alone: the same bits
    assert torch.equal(torch.autograd.grad(y, leaves[0], dy, retain_graph=True)[0], dx)
    assert torch.equal(torch.autograd.grad(y, leaves[1], dy)[0].view(E, N, K), dw)
    only = mxfp8gg.fp8_block_linear(leaves[0], leaves[1].detach(), offs)
    assert torch.equal(only, y) and torch.equal(torch.autograd.grad(only, leaves[0], dy)[0], dx)
    with torch.no_grad():
        assert torch.equal(mxfp8gg.fp8_block_linear(*leaves, offs), y)


def test_linear_shapes(gpu):
    x, w = _x(gpu, 12, 64, seed=1), _x(gpu, 32, 64, seed=2)
    y = mxfp8gg.fp8_block_linear(x, w)
    assert torch.equal(mxfp8gg.fp8_block_linear(x.view(2, 6, 64), w), y.view(2, 6, 32))
    assert torch.equal(mxfp8gg.fp8_block_linear(x[0], w), y[0])
    leaf, wl = x[:0].requires_grad_(True), w.detach().requires_grad_(True)
    e = mxfp8gg.fp8_block_linear(leaf, wl)
    dx, dw = torch.autograd.grad(e, (leaf, wl), torch.zeros_like(e))
    assert e.shape == (0, 32) and dx.shape == (0, 64) and dw.shape == (32, 64) and not dw.any()


def test_operand_layouts(gpu):
    """Row strides, unaligned starts, strided experts and scales of other layouts."""
    x = _x(gpu, 70, 272, seed=1)
    q, s = mxfp8gg.to_fp8_block_dim0(x)
    wq, ws = _weights(gpu, 3, 144, 272, seed=2)
    offs = torch.tensor([30, 30, 70], dtype=torch.int32, device=gpu)
    want = mxfp8gg.fp8_block_mm(q, s, wq, ws, offs)

    def bytes_of(t):
        return t.view(torch.uint8)

    wide = torch.zeros((70, 304), dtype=torch.uint8, device=gpu)
    wide[:, 16:288] = bytes_of(q)
    odd = torch.zeros((70, 273), dtype=torch.uint8, device=gpu)
    odd[:, 1:] = bytes_of(q)
    two = torch.zeros((6, 144, 272), dtype=torch.uint8, device=gpu)
    two[::2] = bytes_of(wq)
    for a in (wide[:, 16:288], odd[:, 1:], bytes_of(q)):
        for b in (two[::2], bytes_of(wq)):
            for sa in (s, s.contiguous()):
                assert torch.equal(mxfp8gg.fp8_block_mm(a, sa, b, ws, offs), want)
    sc = torch.zeros((3, *ws.shape[1:], 2), device=gpu)
    sc[..., 1] = ws
    assert torch.equal(mxfp8gg.fp8_block_mm(q, s, wq, sc[..., 1], offs), want)
    lead = torch.cat([offs.new_zeros(1), offs]).long()     # [E + 1] with a leading 0, int64
    assert torch.equal(mxfp8gg.fp8_block_mm(q, s, wq, ws, lead), want)


def test_rows_past_the_groups_stay(gpu):
    """Rows outside every group are not written, whatever their scales hold."""
    for M, K in ((20, 256), (400, 256), (400, 4096), (3000, 128)):
        x = _x(gpu, M, K, seed=M)
        q, s = mxfp8gg.to_fp8_block_dim0(x)
        s = s.clone()
        s[M // 2:] = float("nan")
        wq, ws = _weights(gpu, 2, 256, K, seed=2)
        offs = torch.tensor([M // 4, M // 2], dtype=torch.int32, device=gpu)
        out = torch.full((M, 256), 7.0, dtype=torch.bfloat16, device=gpu)
        lib = mxfp8gg.load_library()
        s = s.t().contiguous()
        ws_buf = torch.empty(lib.mxgg_block_mm_workspace_bytes(1, 2, M, 256, K), dtype=torch.uint8, device=gpu)
        assert lib.mxgg_block_mm(q.data_ptr(), K, s.data_ptr(), M, wq.data_ptr(), 256 * K, K, ws.data_ptr(),
                                 2 * ws.shape[2], ws.shape[2], offs.data_ptr(), 2, M, 256, K,
                                 out.data_ptr(), 256, 0, ws_buf.data_ptr(), ws_buf.numel(),
                                 torch.cuda.current_stream().cuda_stream) == 0
        assert (out[M // 2:] == 7).all() and torch.isfinite(out).all()


def test_non_finite_operands(gpu):
    x = _x(gpu, 40, 256, seed=1).abs()
    x[3, 200] = float("nan")
    x[5, 0] = float("inf")
    w = _x(gpu, 144, 256, seed=2)
    y = mxfp8gg.fp8_block_linear(x, w)
    ok = torch.ones(40, dtype=torch.bool, device=gpu)
    ok[3] = ok[5] = False
    assert torch.isnan(y[3]).all() and torch.isnan(y[5]).all() and torch.isfinite(y[ok]).all()


def test_graph_replays(gpu):
    x, w = _x(gpu, 30, 256, seed=1), _x(gpu, 144, 256, seed=2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        mxfp8gg.fp8_block_linear(x, w)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = mxfp8gg.fp8_block_linear(x, w)
    for i in range(3):
        x.copy_(_x(gpu, 30, 256, seed=i + 4))
        want = mxfp8gg.fp8_block_linear(x, w)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)


def test_refusals(gpu):
    m = mxfp8gg
    x, w = _x(gpu, 8, 64, seed=1), _x(gpu, 32, 64, seed=2)
    q, s = m.to_fp8_block_dim0(x)
    wq, ws = m.to_fp8_block_weight(w)
    offs = torch.tensor([8], dtype=torch.int32, device=gpu)
    for call in (lambda: m.to_fp8_block_dim0(x[:, :40]), lambda: m.to_fp8_block_weight(w[:, :40]),
                 lambda: m.to_fp8_block_dim1(x, offs[:0]),
                 lambda: m.fp8_block_mm(q, s, wq[:, :48].contiguous(), ws),
                 lambda: m.fp8_block_mm(q, s[:4], wq, ws), lambda: m.fp8_block_mm(q, s, wq, ws[:, :0]),
                 lambda: m.fp8_block_mm(q, s.double(), wq, ws), lambda: m.fp8_block_mm(q, s, wq, ws, offs),
                 lambda: m.fp8_block_mm(q, s, wq[None], ws[None]),
                 lambda: m.fp8_block_mm(q, s, wq, ws, out_dtype=torch.float16),
                 lambda: m.fp8_block_mm(q.cpu(), s, wq, ws),
                 lambda: m.fp8_block_linear(x, w[:20]), lambda: m.fp8_block_linear(x, w[:, :48]),
                 lambda: m.fp8_block_linear(x, w, offs), lambda: m.fp8_block_linear(x, w[None]),
                 lambda: m.fp8_block_wgrad(q, s, q, s)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: m.to_fp8_block_dim0(x.float()), lambda: m.to_fp8_block_dim0(x[0]),
                 lambda: m.to_fp8_block_weight(w.float()), lambda: m.fp8_block_linear(x.float(), w),
                 lambda: m.fp8_block_mm(x, s, wq, ws)):
        with pytest.raises(TypeError):
            call()
    leaf = x.clone().requires_grad_(True)
    with pytest.raises(RuntimeError, match="differentiated twice"):
        torch.autograd.grad(m.fp8_block_linear(leaf, w).sum(), leaf, create_graph=True)
