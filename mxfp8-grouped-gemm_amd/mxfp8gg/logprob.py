"""Log probabilities of given tokens from logits, with entropy and top alternatives.

    r = token_log_probs(logits, tokens, temperature=0.7, topk=8)
    r.log_probs, r.entropy, r.top_ids, r.top_log_probs

is log_softmax(logits / temperature) at the tokens, the entropy of that distribution and
its most probable tokens, from one read of the logits and without a tensor of their
size; the gradient is one more read and one write.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import _lib
from .norm import _ld, _ptr, _rows
from .ops import _first_order, _native, _need_gpu, _no_tangent, _stream_ptr, _tensors, _took

__all__ = ["token_log_probs", "TokenLogProbs"]

_TYPES = {torch.float32: _lib.OUT_F32, torch.bfloat16: _lib.OUT_BF16}


class TokenLogProbs(NamedTuple):
    """What token_log_probs returns; None where it was not asked for."""

    log_probs: torch.Tensor | None
    entropy: torch.Tensor
    top_ids: torch.Tensor | None
    top_log_probs: torch.Tensor | None


def _forward(z, target, opt, keep):
    dev, T, k = z.device, opt.tokens, opt.topk
    f32 = lambda *shape: torch.empty(shape, dtype=torch.float32, device=dev)  # noqa: E731
    lp = f32(T) if target is not None else None
    ent = f32(T)
    ids = torch.empty((T, k), dtype=torch.int32, device=dev) if k else None
    top = f32(T, k) if k else None
    stats = f32(3, T) if keep else None
    lib = _lib.load()
    nbytes = lib.mxgg_token_log_probs_workspace_bytes(ctypes.byref(opt))
    ws = torch.empty(max(nbytes, 0), dtype=torch.uint8, device=dev)
    _lib.check(
        lib.mxgg_token_log_probs(z.data_ptr(), _ptr(target), ctypes.byref(opt), _ptr(lp),
                                 ent.data_ptr(), _ptr(ids), _ptr(top), _ptr(stats), ws.data_ptr(),
                                 nbytes, _stream_ptr(z)), "token_log_probs")
    return lp, ent, ids, top, stats


class _TokenLogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, target, opt):
        lp, ent, ids, top, stats = _forward(z, target, opt, True)
        ctx.save_for_backward(z, target, ids, stats)
        ctx.opt = opt
        ctx.set_materialize_grads(False)
        if ids is not None:
            ctx.mark_non_differentiable(ids)
        return lp, ent, ids, top

    @staticmethod
    def backward(ctx, glp, gent, _, gtop):
        _first_order("token_log_probs", glp, gent, gtop)
        z, target, ids, stats = ctx.saved_tensors
        g = [t.to(torch.float32).contiguous() if t is not None else None for t in (glp, gent, gtop)]
        dz = torch.empty(z.shape, dtype=z.dtype, device=z.device)
        _lib.check(
            _lib.load().mxgg_token_log_probs_grad(*map(_ptr, g), z.data_ptr(), _ptr(target),
                                                  _ptr(ids), stats.data_ptr(),
                                                  ctypes.byref(ctx.opt), dz.data_ptr(),
                                                  _stream_ptr(z)), "token_log_probs_grad")
        return dz, None, None


def token_log_probs(logits: torch.Tensor, targets: torch.Tensor | None = None,
                    temperature: float = 1.0, topk: int = 0,
                    ignore_index: int = -100) -> TokenLogProbs:
    """TokenLogProbs of p = softmax(logits / temperature) over the last dimension.

    logits: bf16 or fp32 [..., V], any row stride; targets: int32 or int64 of the leading
    dimensions, or None (log_probs is then None).
      log_probs      fp32 [...], log p[target]
      entropy        fp32 [...], -sum p log p
      top_ids, top_log_probs   int32 and fp32 [..., topk] (topk up to 64): the most
                     probable tokens in falling order, equal ones by their index
    Logits of -inf are masked: probability 0, never an alternative (-1 and -inf fill up).
    A row of nothing else has log_probs -inf and entropy 0.  A row with a NaN or +inf is
    NaN.  Rows whose target is ignore_index are left out: log_probs and entropy 0, no
    alternatives; any other target outside [0, V) has a NaN log probability.
    Differentiable in logits through log_probs, entropy and top_log_probs (the choice of
    alternatives held fixed); ignored and wholly masked rows have gradients of 0."""
    host = _native(logits)
    if host is not None and _tensors(targets) and topk.__class__ is int:
        r = host.log_probs(logits, targets, temperature, topk, ignore_index, _stream_ptr(logits))
        if _took(r, "token_log_probs"):
            return TokenLogProbs(*r)
    _need_gpu(logits, "logits")
    if logits.dtype not in _TYPES or logits.dim() < 1:
        raise TypeError("logits must be a float32 or bfloat16 tensor [..., V], got "
                        f"{logits.dtype} {tuple(logits.shape)}")
    V, lead = logits.shape[-1], logits.shape[:-1]
    if V < 1:
        raise ValueError(f"logits has rows of no elements: {tuple(logits.shape)}")
    if targets is not None:
        _need_gpu(targets, "targets")
        if targets.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"targets must be int32 or int64, got {targets.dtype}")
        if targets.shape != lead or targets.device != logits.device:
            raise ValueError(f"targets must have shape {tuple(lead)} on {logits.device}, got "
                             f"{tuple(targets.shape)} on {targets.device}")
    if isinstance(topk, bool) or not isinstance(topk, int) or not 0 <= topk <= min(64, V):
        raise ValueError(f"topk must be an integer from 0 to 64 and at most V={V}, got {topk!r}")
    _no_tangent("token_log_probs", logits)
    z = _rows(logits, V)
    t = targets.reshape(-1).contiguous() if targets is not None else None
    opt = _lib.LogProbOptions(z.shape[0], V, _ld(z), ignore_index, _TYPES[z.dtype],
                              t is not None and t.dtype == torch.int64, topk, temperature)
    if torch.is_grad_enabled() and logits.requires_grad:
        lp, ent, ids, top = _TokenLogProbs.apply(z, t, opt)
    else:
        lp, ent, ids, top, _ = _forward(z.detach(), t, opt, False)
    return TokenLogProbs(lp.view(lead) if lp is not None else None, ent.view(lead),
                         ids.view(*lead, topk) if topk else None,
                         top.view(*lead, topk) if topk else None)
