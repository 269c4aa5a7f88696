"""C ABI of the block-scaled products, the norms with residual, the log probabilities
and the gradient clipping without a GPU: bad arguments are refused on the host before
the device is touched, with a status and a message."""
import ctypes

import pytest

from mxfp8gg import _lib

P = 0x10000  # a 16-byte aligned address that is never read
INVALID, SHAPE = _lib.ERR_INVALID_ARGUMENT, _lib.ERR_SHAPE
UNSUPPORTED, ALIGNMENT = _lib.ERR_UNSUPPORTED, _lib.ERR_ALIGNMENT


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def _call(fn, defaults, kw):
    a = dict(defaults)
    assert set(kw) <= set(a)
    a.update(kw)
    return fn(*a.values())


DIM0 = dict(x=P, rows=8, cols=64, ldx=64, q=P, ldq=64, scales=P, lds=8, stream=None)


@pytest.mark.parametrize("status,kw", [
    (SHAPE, dict(rows=-1)), (SHAPE, dict(cols=-16)), (SHAPE, dict(cols=24)), (SHAPE, dict(ldx=63)),
    (SHAPE, dict(ldq=63)), (SHAPE, dict(lds=7)), (INVALID, dict(x=None)), (INVALID, dict(q=None)),
    (INVALID, dict(scales=None)), (ALIGNMENT, dict(x=P + 8)), (ALIGNMENT, dict(ldx=68)),
    (ALIGNMENT, dict(q=P + 4)), (ALIGNMENT, dict(ldq=68)), (UNSUPPORTED, dict(rows=1 << 31)),
    (UNSUPPORTED, dict(cols=(1 << 22) + 16)),
    (UNSUPPORTED, dict(rows=1 << 27, cols=1024, ldx=1024)),
    (_lib.OK, dict(rows=0, x=None, q=None)), (_lib.OK, dict(cols=0, x=None))])
def test_block_quant_dim0(lib, status, kw):
    assert _call(lib.mxgg_block_quant_dim0, DIM0, kw) == status
    assert status == _lib.OK or lib.mxgg_last_error()


DIM1 = dict(x=P, rows=200, cols=64, ldx=64, ends=P, groups=2, cap=512, q=P, ldq=64, scales=P,
            lds=200, qt=P, st=P, ldst=64, ends_pad=P, stream=None)


@pytest.mark.parametrize("status,kw", [
    (SHAPE, dict(rows=-1)), (SHAPE, dict(cols=40)), (SHAPE, dict(ldx=48)), (INVALID, dict(x=None)),
    (UNSUPPORTED, dict(groups=0)), (UNSUPPORTED, dict(groups=1025, cap=1 << 20)),
    (UNSUPPORTED, dict(ends=None)), (SHAPE, dict(cap=256)), (SHAPE, dict(cap=500)),
    (SHAPE, dict(cap=128, ends=None, groups=0)), (INVALID, dict(ends_pad=None)),
    (INVALID, dict(qt=None)), (INVALID, dict(st=None)), (SHAPE, dict(ldst=63)),
    (ALIGNMENT, dict(qt=P + 8)), (ALIGNMENT, dict(q=P + 4)), (INVALID, dict(scales=None)),
    (SHAPE, dict(lds=199)), (UNSUPPORTED, dict(cap=128 << 16)),
    (UNSUPPORTED, dict(cap=(1 << 22) + 128))])
def test_block_quant_dim1(lib, status, kw):
    assert _call(lib.mxgg_block_quant_dim1, DIM1, kw) == status
    assert lib.mxgg_last_error()


WEIGHT = dict(w=P, groups=2, N=64, K=64, q=P, scales=P, qt=P, st=P, stream=None)


@pytest.mark.parametrize("status,kw", [
    (SHAPE, dict(N=-1)), (SHAPE, dict(K=40)), (UNSUPPORTED, dict(groups=-1)),
    (UNSUPPORTED, dict(groups=1025)), (UNSUPPORTED, dict(N=1 << 23)), (INVALID, dict(w=None)),
    (INVALID, dict(q=None)), (INVALID, dict(scales=None)), (INVALID, dict(st=None)),
    (ALIGNMENT, dict(w=P + 8)), (ALIGNMENT, dict(q=P + 8)), (ALIGNMENT, dict(qt=P + 8)),
    (_lib.OK, dict(groups=0)), (_lib.OK, dict(N=0))])
def test_block_quant_weight(lib, status, kw):
    assert _call(lib.mxgg_block_quant_weight, WEIGHT, kw) == status
    assert status == _lib.OK or lib.mxgg_last_error()


MM = dict(a=P, lda=256, a_scales=P, ldas=100, w=P, w_gstride=64 * 256, ldw=256, w_scales=P,
          ws_gstride=2, ldws=2, ends=P, groups=3, M=100, N=64, K=256, out=P, ldo=64,
          out_type=_lib.OUT_BF16, workspace=P, workspace_bytes=1 << 40, stream=None)


@pytest.mark.parametrize("status,kw", [
    (INVALID, dict(out_type=9)), (SHAPE, dict(M=-1)), (SHAPE, dict(K=0)), (SHAPE, dict(K=200)),
    (UNSUPPORTED, dict(groups=0)), (UNSUPPORTED, dict(ends=None)), (UNSUPPORTED, dict(groups=1025)),
    (UNSUPPORTED, dict(M=1 << 31)), (UNSUPPORTED, dict(K=1 << 23)), (UNSUPPORTED, dict(N=1 << 23)),
    (UNSUPPORTED, dict(M=1 << 24, N=1 << 14)), (INVALID, dict(a=None)), (INVALID, dict(a_scales=None)),
    (INVALID, dict(w=None)), (INVALID, dict(w_scales=None)), (INVALID, dict(out=None)),
    (SHAPE, dict(lda=240)), (SHAPE, dict(ldw=240)), (SHAPE, dict(ldas=99)), (SHAPE, dict(ldws=1)),
    (SHAPE, dict(ldo=63)), (SHAPE, dict(w_gstride=0)), (SHAPE, dict(ws_gstride=-1)),
    (UNSUPPORTED, dict(lda=1 << 23)), (UNSUPPORTED, dict(ldas=1 << 30)),
    (ALIGNMENT, dict(a=P + 8)), (ALIGNMENT, dict(lda=264)), (ALIGNMENT, dict(w=P + 1)),
    (ALIGNMENT, dict(w_gstride=64 * 256 + 8)), (_lib.OK, dict(M=0)), (_lib.OK, dict(N=0))])
def test_block_mm(lib, status, kw):
    assert _call(lib.mxgg_block_mm, MM, kw) == status
    assert status == _lib.OK or lib.mxgg_last_error()


@pytest.mark.gpu  # how far a product is split depends on the card
def test_block_mm_workspace(gpu, lib):
    """What a call needs it refuses to go without; sizes that it refuses have none."""
    kw = dict(ends=None, groups=1, M=100, N=128, K=8192, lda=8192, ldw=8192, w_gstride=0, ldws=64,
              ldo=128)
    need = lib.mxgg_block_mm_workspace_bytes(0, 1, 100, 128, 8192)
    assert need > 0 and need % 4 == 0
    for status, more in ((SHAPE, dict(workspace_bytes=need - 1)), (INVALID, dict(workspace=None)),
                         (ALIGNMENT, dict(workspace=P + 4))):
        assert _call(lib.mxgg_block_mm, MM, {**kw, **more}) == status
    assert lib.mxgg_block_mm_workspace_bytes(0, 2, 100, 128, 8192) == -1
    assert lib.mxgg_block_mm_workspace_bytes(0, 1, 0, 128, 8192) == 0
    assert lib.mxgg_block_mm_workspace_bytes(0, 1, 4, 128, 24) == -1


WGRAD = dict(go=P, ldgo=256, go_scales=P, ldgos=64, ia=P, ldia=256, ia_scales=P, ldias=48, ends=P,
             groups=2, tokens=256, N=64, K=48, dw=P, out_type=_lib.OUT_BF16, workspace=P,
             workspace_bytes=1 << 40, stream=None)


@pytest.mark.parametrize("status,kw", [
    (INVALID, dict(out_type=9)), (SHAPE, dict(tokens=200)), (SHAPE, dict(tokens=-128)),
    (SHAPE, dict(N=-1)), (UNSUPPORTED, dict(groups=0)), (UNSUPPORTED, dict(ends=None)),
    (UNSUPPORTED, dict(groups=1025)), (UNSUPPORTED, dict(tokens=1 << 23)),
    (UNSUPPORTED, dict(N=1 << 20, K=1 << 20)), (INVALID, dict(dw=None)), (INVALID, dict(go=None)),
    (INVALID, dict(ia=None)), (INVALID, dict(go_scales=None)), (INVALID, dict(ia_scales=None)),
    (SHAPE, dict(ldgo=240)), (SHAPE, dict(ldia=240)), (SHAPE, dict(ldgos=63)),
    (SHAPE, dict(ldias=47)), (UNSUPPORTED, dict(ldgo=1 << 23)), (UNSUPPORTED, dict(ldgos=1 << 30)),
    (ALIGNMENT, dict(go=P + 8)), (ALIGNMENT, dict(ldia=264)), (_lib.OK, dict(N=0)),
    (_lib.OK, dict(K=0))])
def test_block_wgrad(lib, status, kw):
    assert _call(lib.mxgg_block_wgrad, WGRAD, kw) == status
    assert status == _lib.OK or lib.mxgg_last_error()


@pytest.mark.gpu
def test_block_wgrad_workspace(gpu, lib):
    need = lib.mxgg_block_wgrad_workspace_bytes(0, 1, 1 << 16, 128, 128)
    assert need > 0
    kw = dict(ends=None, groups=1, tokens=1 << 16, ldgo=1 << 16, ldia=1 << 16, N=128, K=128,
              ldgos=128, ldias=128)
    assert _call(lib.mxgg_block_wgrad, WGRAD, {**kw, "workspace_bytes": need - 4}) == SHAPE
    assert _call(lib.mxgg_block_wgrad, WGRAD, {**kw, "workspace": None}) == INVALID
    assert lib.mxgg_block_wgrad_workspace_bytes(0, 1, 100, 128, 128) == -1


def _norm(**kw):
    o = dict(rows=4, cols=64, dtype=_lib.OUT_F32, weight_dtype=_lib.OUT_F32,
             bias_dtype=_lib.OUT_F32, center=0, eps=1e-5)
    o.update(kw)
    return ctypes.byref(_lib.NormOptions(**o))


ADD = dict(x=P, ldx=64, residual=P, ldres=64, weight=P, options=_norm(), h=P, ldh=64, y=P, ldy=64,
           stats=P, stream=None)
ADD_GRAD = dict(dy=P, ldg=64, dh=P, ldgh=64, h=P, ldh=64, weight=P, stats=P, options=_norm(), dx=P,
                ldgx=64, dw=None, workspace=None, workspace_bytes=0, stream=None)
QUANT = dict(x=P, ldx=64, residual=P, ldres=64, weight=P, options=_norm(), h=P, ldh=64, q=P, ldq=64,
             scales=P, lds=4, format=_lib.QUANT_MX, mode=_lib.SCALE_RCEIL, stream=None)


@pytest.mark.parametrize("status,o", [
    (INVALID, dict(center=1)), (SHAPE, dict(rows=-1)), (SHAPE, dict(cols=0)),
    (UNSUPPORTED, dict(cols=32800)), (INVALID, dict(dtype=5)), (INVALID, dict(weight_dtype=5))])
def test_add_norm_options(lib, status, o):
    for fn, a in ((lib.mxgg_add_rms_norm, ADD), (lib.mxgg_add_rms_norm_grad, ADD_GRAD),
                  (lib.mxgg_rms_norm_quant, QUANT)):
        assert _call(fn, a, dict(options=_norm(**o))) == status
        assert _call(fn, a, dict(options=None)) == INVALID
        assert lib.mxgg_last_error()


@pytest.mark.parametrize("status,kw", [
    (INVALID, dict(x=None)), (INVALID, dict(residual=None)), (INVALID, dict(h=None)),
    (INVALID, dict(y=None)), (SHAPE, dict(ldx=63)), (SHAPE, dict(ldres=63)), (SHAPE, dict(ldh=63)),
    (SHAPE, dict(ldy=63)), (INVALID, dict(residual=None, h=None)),
    (_lib.OK, dict(options=_norm(rows=0), x=None))])
def test_add_norm(lib, status, kw):
    assert _call(lib.mxgg_add_rms_norm, ADD, kw) == status


@pytest.mark.parametrize("status,kw", [
    (INVALID, dict(dy=None)), (INVALID, dict(h=None)), (INVALID, dict(stats=None)),
    (SHAPE, dict(ldg=63)), (SHAPE, dict(ldgh=63)), (SHAPE, dict(ldh=63)), (SHAPE, dict(ldgx=63)),
    (SHAPE, dict(dw=P))])
def test_add_norm_gradient(lib, status, kw):
    assert _call(lib.mxgg_add_rms_norm_grad, ADD_GRAD, kw) == status


@pytest.mark.parametrize("status,kw", [
    (INVALID, dict(x=None)), (INVALID, dict(residual=None)), (INVALID, dict(q=None)),
    (INVALID, dict(scales=None)), (INVALID, dict(format=7)), (INVALID, dict(mode=7)),
    (SHAPE, dict(ldq=63)), (SHAPE, dict(lds=3)), (SHAPE, dict(options=_norm(cols=48))),
    (SHAPE, dict(options=_norm(cols=40), format=_lib.QUANT_BLOCK)),
    (ALIGNMENT, dict(q=P + 4)), (ALIGNMENT, dict(ldq=68)),
    (_lib.OK, dict(options=_norm(rows=0), x=None))])
def test_norm_quant(lib, status, kw):
    assert _call(lib.mxgg_rms_norm_quant, QUANT, kw) == status


def _grads(*entries):
    return (_lib.GradTensor * len(entries))(*[_lib.GradTensor(*e) for e in entries])


@pytest.mark.parametrize("status,entry", [
    (INVALID, (P, 10, 7)), (SHAPE, (P, -1, 0)), (SHAPE, (P, 1 << 49, 0)), (INVALID, (None, 10, 0)),
    (ALIGNMENT, (P + 2, 10, _lib.OUT_F32)), (ALIGNMENT, (P + 1, 10, _lib.OUT_BF16))])
def test_gradient_tensors(lib, status, entry):
    t = _grads((P, 10, _lib.OUT_F32), entry)
    opt = ctypes.byref(_lib.ClipOptions(max_norm=1.0, eps=1e-6))
    assert lib.mxgg_grad_norm(t, 2, P, P, 1 << 30, None) == status
    assert lib.mxgg_clip_grad_norm(t, 2, opt, P, P, 1 << 30, None) == status
    assert lib.mxgg_grad_norm_workspace_bytes(t, 2) == -1


def test_clip(lib):
    t = _grads((P, 10, _lib.OUT_F32))
    need = lib.mxgg_grad_norm_workspace_bytes(t, 1)
    assert need > 0 and need % 8 == 0
    opt = lambda m, e: ctypes.byref(_lib.ClipOptions(max_norm=m, eps=e))  # noqa: E731
    nan = float("nan")
    good = opt(1.0, 1e-6)
    for status, args in ((INVALID, (None, 1, good, P, P, need)), (SHAPE, (t, -1, good, P, P, need)),
                         (SHAPE, (t, 1 << 25, good, P, P, need)), (INVALID, (t, 1, None, P, P, need)),
                         (INVALID, (t, 1, opt(-1.0, 0.0), P, P, need)),
                         (INVALID, (t, 1, opt(nan, 0.0), P, P, need)),
                         (INVALID, (t, 1, opt(1.0, nan), P, P, need)),
                         (INVALID, (t, 1, good, None, P, need)), (SHAPE, (t, 1, good, P, P, need - 8)),
                         (INVALID, (t, 1, good, P, None, need)),
                         (ALIGNMENT, (t, 1, good, P, P + 4, need))):
        assert lib.mxgg_clip_grad_norm(*args, None) == status
        assert lib.mxgg_last_error()


def _logp(**kw):
    o = dict(tokens=4, vocab=1000, ldz=1000, ignore_index=-100, dtype=_lib.OUT_BF16,
             target_int64=1, topk=2, temperature=1.0)
    o.update(kw)
    return ctypes.byref(_lib.LogProbOptions(**o))


LOGP = dict(z=P, target=P, options=_logp(), log_probs=P, entropy=P, ids=P, top=P, stats=P,
            workspace=P, workspace_bytes=1 << 40, stream=None)
LOGP_GRAD = dict(g_lp=P, g_ent=P, g_top=P, z=P, target=P, ids=P, stats=P, options=_logp(), dz=P,
                 stream=None)


@pytest.mark.parametrize("status,o", [
    (INVALID, dict(dtype=7)), (INVALID, dict(temperature=0.0)), (INVALID, dict(temperature=-1.0)),
    (INVALID, dict(temperature=float("nan"))), (INVALID, dict(temperature=float("inf"))),
    (INVALID, dict(temperature=1e-39)), (SHAPE, dict(tokens=-1)), (SHAPE, dict(vocab=0)),
    (SHAPE, dict(topk=-1)), (SHAPE, dict(vocab=3, ldz=3, topk=4)), (SHAPE, dict(ldz=999)),
    (UNSUPPORTED, dict(topk=65)), (UNSUPPORTED, dict(vocab=(1 << 24) + 1, ldz=1 << 25)),
    (UNSUPPORTED, dict(tokens=1 << 40))])
def test_log_prob_options(lib, status, o):
    assert _call(lib.mxgg_token_log_probs, LOGP, dict(options=_logp(**o))) == status
    assert _call(lib.mxgg_token_log_probs_grad, LOGP_GRAD, dict(options=_logp(**o))) == status
    assert lib.mxgg_token_log_probs_workspace_bytes(_logp(**o)) == -1
    assert lib.mxgg_last_error()


def test_log_probs(lib):
    for kw in (dict(options=None), dict(z=None), dict(target=None), dict(ids=None), dict(top=None)):
        assert _call(lib.mxgg_token_log_probs, LOGP, kw) == INVALID
    for kw in (dict(options=None), dict(z=None), dict(target=None), dict(ids=None),
               dict(stats=None), dict(dz=None)):
        assert _call(lib.mxgg_token_log_probs_grad, LOGP_GRAD, kw) == INVALID
    none = _logp(tokens=0)
    assert _call(lib.mxgg_token_log_probs, LOGP, dict(options=none, z=None)) == _lib.OK
    assert _call(lib.mxgg_token_log_probs_grad, LOGP_GRAD, dict(options=none, z=None)) == _lib.OK
    assert lib.mxgg_token_log_probs_workspace_bytes(none) == 0


@pytest.mark.gpu  # which rows are shared out depends on the card
def test_log_probs_workspace(gpu, lib):
    long = dict(tokens=1, vocab=1 << 17, ldz=1 << 17)
    need = lib.mxgg_token_log_probs_workspace_bytes(_logp(**long))
    assert need > 0
    for status, kw in ((SHAPE, dict(workspace_bytes=need - 1)), (INVALID, dict(workspace=None)),
                       (ALIGNMENT, dict(workspace=P + 4))):
        assert _call(lib.mxgg_token_log_probs, LOGP, {"options": _logp(**long), **kw}) == status
