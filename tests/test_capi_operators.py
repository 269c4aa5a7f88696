"""C ABI of the operators around the expert FFN without a GPU: bad arguments are
refused on the host before the device is touched, with a status and a message."""
import ctypes

import pytest

from mxfp8gg import _lib

P = 0x10000  # a 16-byte aligned address that is never read


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def _route(lib, grad=False, tokens=4, logits=P, idx=P, weights=P, options=True, **kw):
    o = dict(experts=16, topk=2, groups=1, top_groups=1, score=_lib.SCORE_SIGMOID,
             dtype=_lib.OUT_F32, group_best=1, renormalize=1, scale=1.0)
    o.update(kw)
    opt = ctypes.byref(_lib.RouteOptions(**o)) if options else None
    if grad:
        return lib.mxgg_route_topk_grad(weights, idx, P, logits, tokens, opt, P, None)
    return lib.mxgg_route_topk(logits, tokens, None, opt, idx, weights, None, None)


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("status,kw", [
    (_lib.ERR_INVALID_ARGUMENT, dict(options=False)),
    (_lib.ERR_INVALID_ARGUMENT, dict(idx=None)),
    (_lib.ERR_INVALID_ARGUMENT, dict(weights=None)),
    (_lib.ERR_INVALID_ARGUMENT, dict(score=2)),
    (_lib.ERR_INVALID_ARGUMENT, dict(dtype=7)),
    (_lib.ERR_INVALID_ARGUMENT, dict(group_best=0)),
    (_lib.ERR_SHAPE, dict(tokens=-1)),
    (_lib.ERR_SHAPE, dict(topk=0)),
    (_lib.ERR_SHAPE, dict(topk=17)),
    (_lib.ERR_SHAPE, dict(experts=0)),
    (_lib.ERR_SHAPE, dict(groups=3)),
    (_lib.ERR_SHAPE, dict(groups=4, top_groups=5)),
    (_lib.ERR_SHAPE, dict(groups=4, top_groups=0)),
    (_lib.ERR_SHAPE, dict(experts=1024, groups=128)),
    (_lib.ERR_UNSUPPORTED, dict(experts=1025)),
    (_lib.ERR_UNSUPPORTED, dict(experts=64, topk=33)),
    (_lib.ERR_UNSUPPORTED, dict(tokens=1 << 24)),
])
def test_route_refusals(lib, grad, status, kw):
    assert _route(lib, grad, **kw) == status
    assert lib.mxgg_last_error()


def test_route_softmax_gradient_needs_the_logits(lib):
    kw = dict(score=_lib.SCORE_SOFTMAX, renormalize=0, logits=None)
    assert _route(lib, True, **kw) == _lib.ERR_INVALID_ARGUMENT
    assert _route(lib, False, tokens=0, logits=None, idx=None, weights=None) == _lib.OK


def _norm_options(**kw):
    o = dict(rows=4, cols=64, dtype=_lib.OUT_F32, weight_dtype=_lib.OUT_F32,
             bias_dtype=_lib.OUT_F32, center=1, eps=1e-5)
    o.update(kw)
    return ctypes.byref(_lib.NormOptions(**o))


@pytest.mark.parametrize("status,kw", [
    (_lib.ERR_SHAPE, dict(rows=-1)), (_lib.ERR_SHAPE, dict(cols=0)),
    (_lib.ERR_UNSUPPORTED, dict(cols=32769)), (_lib.ERR_INVALID_ARGUMENT, dict(dtype=3)),
    (_lib.ERR_INVALID_ARGUMENT, dict(weight_dtype=-1))])
def test_norm_option_refusals(lib, status, kw):
    o = _norm_options(**kw)
    assert lib.mxgg_norm(P, 64, None, None, o, P, 64, None, None) == status
    assert lib.mxgg_norm_grad(P, 64, P, 64, None, P, o, P, 64, None, None, None, 0, None) == status
    assert lib.mxgg_norm_grad_workspace_bytes(o) == -1


def test_norm_refusals(lib):
    o = _norm_options()
    assert lib.mxgg_norm(None, 64, None, None, o, P, 64, None, None) == _lib.ERR_INVALID_ARGUMENT
    assert lib.mxgg_norm(P, 64, None, None, None, P, 64, None, None) == _lib.ERR_INVALID_ARGUMENT
    assert lib.mxgg_norm(P, 63, None, None, o, P, 64, None, None) == _lib.ERR_SHAPE
    assert lib.mxgg_norm(P, 64, None, None, o, P, 63, None, None) == _lib.ERR_SHAPE
    need = lib.mxgg_norm_grad_workspace_bytes(o)
    assert need > 0 and need % (8 * 64) == 0
    f = lambda ws, n, dw=P: lib.mxgg_norm_grad(  # noqa: E731
        P, 64, P, 64, None, P, o, P, 64, dw, None, ws, n, None)
    assert f(P, need - 1) == _lib.ERR_SHAPE
    assert f(None, need) == _lib.ERR_INVALID_ARGUMENT
    assert f(P + 2, need) == _lib.ERR_ALIGNMENT
    assert lib.mxgg_norm_grad(P, 64, P, 64, None, P, o, P, 32, None, None, None, 0,
                              None) == _lib.ERR_SHAPE
    assert lib.mxgg_norm(None, 64, None, None, _norm_options(rows=0), None, 64, None,
                         None) == _lib.OK


def _adamw(lib, count=1, options=True, tensor=None, **kw):
    t = dict(param=P, grad=P, exp_avg=P, exp_avg_sq=P, n=8, param_dtype=_lib.OUT_F32,
             grad_dtype=_lib.OUT_F32)
    t.update(tensor or {})
    o = dict(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.0, step=1, state_bits=32)
    o.update(kw)
    table = (_lib.AdamwTensor * max(1, count))()
    table[max(0, count - 1)] = _lib.AdamwTensor(**t)  # the others are empty
    for i in range(count - 1):
        table[i].param_dtype = table[i].grad_dtype = _lib.OUT_F32
    return lib.mxgg_adamw_step(table, count, ctypes.byref(_lib.AdamwOptions(**o)) if options
                               else None, None)


@pytest.mark.parametrize("count", [1, 100])
@pytest.mark.parametrize("status,kw", [
    (_lib.ERR_INVALID_ARGUMENT, dict(options=False)),
    (_lib.ERR_SHAPE, dict(step=0)),
    (_lib.ERR_INVALID_ARGUMENT, dict(state_bits=16)),
    (_lib.ERR_INVALID_ARGUMENT, dict(beta1=1.0)),
    (_lib.ERR_INVALID_ARGUMENT, dict(beta2=-0.1)),
    (_lib.ERR_INVALID_ARGUMENT, dict(lr=float("nan"))),
    (_lib.ERR_INVALID_ARGUMENT, dict(eps=-1.0)),
    (_lib.ERR_INVALID_ARGUMENT, dict(weight_decay=-1.0)),
    (_lib.ERR_INVALID_ARGUMENT, dict(tensor=dict(grad=None))),
    (_lib.ERR_INVALID_ARGUMENT, dict(tensor=dict(param_dtype=5))),
    (_lib.ERR_INVALID_ARGUMENT, dict(state_bits=8)),            # no scales
    (_lib.ERR_SHAPE, dict(tensor=dict(n=-1))),
    (_lib.ERR_UNSUPPORTED, dict(tensor=dict(n=1 << 40))),
])
def test_adamw_refusals(lib, count, status, kw):
    """Also where only the last of many tensors is bad: nothing was launched."""
    assert _adamw(lib, count, **kw) == status


def test_adamw_of_nothing(lib):
    assert _adamw(lib, 0) == _lib.OK
    assert _adamw(lib, 3, tensor=dict(n=0, param=None)) == _lib.OK


def _loss_options(**kw):
    o = dict(tokens=4, vocab=100, hidden=64, ldx=64, ldw=64, ignore_index=-100, target_int64=1,
             reduction=_lib.REDUCE_MEAN)
    o.update(kw)
    return ctypes.byref(_lib.LossOptions(**o))


@pytest.mark.parametrize("status,kw", [
    (_lib.ERR_SHAPE, dict(tokens=-1)), (_lib.ERR_SHAPE, dict(vocab=0)),
    (_lib.ERR_SHAPE, dict(hidden=0)), (_lib.ERR_SHAPE, dict(hidden=60, ldx=64)),
    (_lib.ERR_SHAPE, dict(ldx=56)), (_lib.ERR_SHAPE, dict(ldw=56)),
    (_lib.ERR_ALIGNMENT, dict(ldx=68)), (_lib.ERR_ALIGNMENT, dict(ldw=68)),
    (_lib.ERR_INVALID_ARGUMENT, dict(reduction=3)),
    (_lib.ERR_UNSUPPORTED, dict(ldw=1 << 23)), (_lib.ERR_UNSUPPORTED, dict(tokens=1 << 22)),
    (_lib.ERR_UNSUPPORTED, dict(vocab=1 << 25)),
    (_lib.ERR_UNSUPPORTED, dict(vocab=1 << 24, tokens=1 << 21))])
def test_loss_option_refusals(lib, status, kw):
    o = _loss_options(**kw)
    assert lib.mxgg_linear_cross_entropy(P, P, P, o, P, P, P, 1 << 40, None) == status
    assert lib.mxgg_linear_cross_entropy_grad(P, P, P, P, P, o, P, P, P, 1 << 40, None) == status
    assert lib.mxgg_linear_cross_entropy_workspace_bytes(o) == -1
    assert lib.mxgg_linear_cross_entropy_grad_workspace_bytes(o, 1, 1) == -1


def test_loss_refusals(lib):
    o = _loss_options()
    f = lib.mxgg_linear_cross_entropy
    need = lib.mxgg_linear_cross_entropy_workspace_bytes(o)
    assert need > 0
    assert f(None, P, P, o, P, P, P, need, None) == _lib.ERR_INVALID_ARGUMENT
    assert f(P, None, P, o, P, P, P, need, None) == _lib.ERR_INVALID_ARGUMENT
    assert f(P, P, None, o, P, P, P, need, None) == _lib.ERR_INVALID_ARGUMENT
    assert f(P, P, P, o, None, P, P, need, None) == _lib.ERR_INVALID_ARGUMENT
    assert f(P, P, P, o, P, None, P, need, None) == _lib.ERR_INVALID_ARGUMENT
    assert f(P + 2, P, P, o, P, P, P, need, None) == _lib.ERR_ALIGNMENT
    assert f(P, P + 8, P, o, P, P, P, need, None) == _lib.ERR_ALIGNMENT
    assert f(P, P, P, o, P, P, P, need - 1, None) == _lib.ERR_SHAPE
    assert f(P, P, P, o, P, P, P + 8, need, None) == _lib.ERR_ALIGNMENT
    g = lib.mxgg_linear_cross_entropy_grad
    need = lib.mxgg_linear_cross_entropy_grad_workspace_bytes(o, 1, 1)
    assert need > 0
    assert g(None, P, P, P, P, o, P, P, P, need, None) == _lib.ERR_INVALID_ARGUMENT
    assert g(P, P, P, P, None, o, P, P, P, need, None) == _lib.ERR_INVALID_ARGUMENT
    assert g(P, P, P, P, P, o, P + 4, P, P, need, None) == _lib.ERR_ALIGNMENT
    assert g(P, P, P, P, P, o, P, P, P, need - 1, None) == _lib.ERR_SHAPE
    assert g(P, P, P, P, P, o, None, None, None, 0, None) == _lib.OK       # nothing wanted
    none = _loss_options(tokens=0)
    assert g(P, P, P, P, P, none, P, None, None, 0, None) == _lib.OK
    assert g(P, P, P, P, P, none, P, P, None, 0, None) == _lib.ERR_SHAPE
