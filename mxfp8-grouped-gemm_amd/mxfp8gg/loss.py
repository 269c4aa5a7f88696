"""Softmax cross entropy of a linear layer over a large vocabulary.

    loss = linear_cross_entropy(x, weight, target)   # x [T, H], weight [V, H], target [T]
    loss.backward()

is cross_entropy(x @ weight.T, target) without the logits [T, V]: the forward
pass keeps two fp32 values a token, the backward pass computes the logits again
in pieces of the vocabulary.  While it runs it holds at most 1 GiB of bf16 [T, piece],
dx in fp32 where there are several pieces, and, where a product is split over the
compute units, fp32 partial sums of at most two tiles of 256 KB a unit for each of the
two gradients (128 MiB each on 256 units).  d loss / d logits is rounded to bf16 between
the products, which sum in fp32.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .ops import _first_order, _native, _need_gpu, _no_tangent, _stream_ptr, _tensors, _took

__all__ = ["linear_cross_entropy", "LinearCrossEntropy"]

_REDUCTIONS = {"none": _lib.REDUCE_NONE, "sum": _lib.REDUCE_SUM, "mean": _lib.REDUCE_MEAN}


def _operand(t: torch.Tensor):
    """(t, row stride) with the 16-byte aligned rows that the kernels read: a copy
    where t has none."""
    ld = t.stride(0) if t.shape[0] > 1 else t.shape[1]
    if t.stride(1) == 1 and ld >= t.shape[1] and ld % 8 == 0 and t.data_ptr() % 16 == 0:
        return t, ld
    return t.clone(memory_format=torch.contiguous_format), t.shape[1]


def _forward(x, w, target, opt):
    lib, dev = _lib.load(), x.device
    loss = torch.empty(opt.tokens if opt.reduction == _lib.REDUCE_NONE else (),
                       dtype=torch.float32, device=dev)
    stats = torch.empty(2 * opt.tokens + 1, dtype=torch.float32, device=dev)
    nbytes = lib.mxgg_linear_cross_entropy_workspace_bytes(ctypes.byref(opt))
    ws = torch.empty(max(nbytes, 0), dtype=torch.uint8, device=dev)
    _lib.check(
        lib.mxgg_linear_cross_entropy(x.data_ptr(), w.data_ptr(), target.data_ptr(),
                                      ctypes.byref(opt), loss.data_ptr(), stats.data_ptr(),
                                      ws.data_ptr(), nbytes, _stream_ptr(x)),
        "linear_cross_entropy",
    )
    return loss, stats


class LinearCrossEntropy(torch.autograd.Function):
    """linear_cross_entropy with the gradients of x and the weight."""

    @staticmethod
    def forward(ctx, x, weight, target, opt):
        (x2, opt.ldx), (w2, opt.ldw) = _operand(x), _operand(weight)
        loss, stats = _forward(x2, w2, target, opt)
        ctx.save_for_backward(x2, w2, target, stats)
        ctx.opt = opt
        return loss

    @staticmethod
    def backward(ctx, dloss):
        _first_order("linear_cross_entropy")
        x, w, target, stats = ctx.saved_tensors
        opt, dev = ctx.opt, x.device
        need_x, need_w = ctx.needs_input_grad[:2]
        dx = torch.empty(x.shape, dtype=x.dtype, device=dev) if need_x else None
        if opt.tokens == 0:
            return dx, torch.zeros(w.shape, dtype=w.dtype, device=dev) if need_w else None, None, None
        dw = torch.empty(w.shape, dtype=w.dtype, device=dev) if need_w else None
        d = dloss.to(torch.float32).contiguous()
        lib = _lib.load()
        nbytes = lib.mxgg_linear_cross_entropy_grad_workspace_bytes(ctypes.byref(opt), need_x,
                                                                    need_w)
        ws = torch.empty(max(nbytes, 0), dtype=torch.uint8, device=dev)
        _lib.check(
            lib.mxgg_linear_cross_entropy_grad(
                d.data_ptr(), x.data_ptr(), w.data_ptr(), target.data_ptr(), stats.data_ptr(),
                ctypes.byref(opt), dx.data_ptr() if need_x else None,
                dw.data_ptr() if need_w else None, ws.data_ptr(), nbytes, _stream_ptr(x)),
            "linear_cross_entropy_grad",
        )
        return dx, dw, None, None


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor,
                         ignore_index: int = -100, reduction: str = "mean") -> torch.Tensor:
    """cross_entropy(x @ weight.T, target), in fp32, without the logits.

    x: bf16 [..., H]; weight: bf16 [V, H] (H a multiple of 8); target: int32 or
    int64 of x's leading dimensions.  Tokens whose target is ignore_index have
    loss 0 and no gradient, and the mean is over the others (as torch's, NaN with
    gradients of 0 if there are none); any other target outside [0, V) gives a NaN
    loss.
    reduction: "mean", "sum" or "none" (target's shape).  Differentiable in x and
    weight; the same bits on every run."""
    host = _native(x)
    if host is not None and reduction in _REDUCTIONS and _tensors(weight, target) \
            and weight is not None and target is not None:
        r = host.linear_cross_entropy(x, weight, target, ignore_index, _REDUCTIONS[reduction],
                                      _stream_ptr(x))
        if _took(r, "linear_cross_entropy"):
            return r
    _need_gpu(x, "x")
    for name, t in (("weight", weight), ("target", target)):
        _need_gpu(t, name)
        if t.device != x.device:
            raise ValueError(f"{name} is on {t.device}, x on {x.device}")
    if x.dtype != torch.bfloat16 or weight.dtype != torch.bfloat16:
        raise TypeError(f"x and weight must be bfloat16, got {x.dtype} and {weight.dtype}")
    if target.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"target must be int32 or int64, got {target.dtype}")
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1] \
            or target.shape != x.shape[:-1]:
        raise ValueError(f"shapes must be x [..., H], weight [V, H], target [...], got "
                         f"{tuple(x.shape)}, {tuple(weight.shape)}, {tuple(target.shape)}")
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be one of {sorted(_REDUCTIONS)}, got {reduction!r}")
    _no_tangent("linear_cross_entropy", x, weight)
    H = x.shape[-1]
    x2 = x.reshape(-1, H) if H else x.new_empty((0, 0))
    t = target.reshape(-1).contiguous()
    opt = _lib.LossOptions(x2.shape[0], weight.shape[0], H, H, H, ignore_index,
                           target.dtype == torch.int64, _REDUCTIONS[reduction])
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad):
        loss = LinearCrossEntropy.apply(x2, weight, t, opt)
    else:
        (a, opt.ldx), (w, opt.ldw) = _operand(x2.detach()), _operand(weight.detach())
        loss, _ = _forward(a, w, t, opt)
    return loss.view(target.shape) if reduction == "none" else loss
