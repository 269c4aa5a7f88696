"""Layer norm and root-mean-square norm around the expert layer.

    y = layer_norm(x, weight, bias)     (x - mean) / sqrt(var + eps) * weight + bias
    y = rms_norm(x, weight)             x / sqrt(mean(x^2) + eps) * weight

Rows are the last dimension of x (bf16 or fp32, at most 32768 long, any length
and row stride).  Statistics are fp32; the backward pass keeps x and two fp32
values a row, and adds the weight's gradient over the rows in a fixed order, so
it is the same on every run.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .ops import _first_order, _native, _need_gpu, _no_tangent, _stream_ptr, _tensors, _took

__all__ = ["layer_norm", "rms_norm", "Norm"]

_TYPES = {torch.float32: _lib.OUT_F32, torch.bfloat16: _lib.OUT_BF16}


def _rows(t: torch.Tensor, cols: int) -> torch.Tensor:
    """t as [rows, cols] with contiguous rows (a copy only where it has none)."""
    t = t.reshape(-1, cols)
    if (cols > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < cols):
        t = t.contiguous()
    return t


def _ld(t: torch.Tensor) -> int:
    return max(t.stride(0), t.shape[1])


def _forward(x2, weight, bias, opt, keep):
    y = torch.empty(x2.shape, dtype=x2.dtype, device=x2.device)
    stats = torch.empty((2, x2.shape[0]), dtype=torch.float32, device=x2.device) if keep else None
    _lib.check(
        _lib.load().mxgg_norm(
            x2.data_ptr(), _ld(x2), weight.data_ptr() if weight is not None else None,
            bias.data_ptr() if bias is not None else None, ctypes.byref(opt), y.data_ptr(), _ld(y),
            stats.data_ptr() if keep else None, _stream_ptr(x2)),
        "norm",
    )
    return y, stats


class Norm(torch.autograd.Function):
    """layer_norm / rms_norm with their gradients."""

    @staticmethod
    def forward(ctx, x, weight, bias, opt):
        x2 = _rows(x, opt.cols)
        w = weight.contiguous() if weight is not None else None
        y, stats = _forward(x2, w, bias.contiguous() if bias is not None else None, opt, True)
        ctx.save_for_backward(x2, w, stats)
        ctx.opt = opt
        ctx.shape = x.shape
        ctx.param_types = [p.dtype if p is not None else None for p in (weight, bias)]
        return y.view(x.shape)

    @staticmethod
    def backward(ctx, dy):
        _first_order("norm")
        x2, w, stats = ctx.saved_tensors
        opt, dev = ctx.opt, x2.device
        dy2 = _rows(dy.to(x2.dtype), opt.cols)
        need = ctx.needs_input_grad
        dx = torch.empty(x2.shape, dtype=x2.dtype, device=dev) if need[0] else None
        dw, db = (torch.empty(opt.cols, dtype=t, device=dev) if n else None
                  for t, n in zip(ctx.param_types, need[1:3]))
        lib = _lib.load()
        ws = None
        if dw is not None or db is not None:
            ws = torch.empty(lib.mxgg_norm_grad_workspace_bytes(ctypes.byref(opt)),
                             dtype=torch.uint8, device=dev)
        ptr = lambda t: t.data_ptr() if t is not None else None  # noqa: E731
        _lib.check(
            lib.mxgg_norm_grad(dy2.data_ptr(), _ld(dy2), x2.data_ptr(), _ld(x2), ptr(w),
                               stats.data_ptr(), ctypes.byref(opt), ptr(dx),
                               _ld(dx) if dx is not None else 0, ptr(dw), ptr(db), ptr(ws),
                               ws.numel() if ws is not None else 0, _stream_ptr(x2)),
            "norm_grad",
        )
        return dx.view(ctx.shape) if dx is not None else None, dw, db, None


def _norm(x, weight, bias, eps, center):
    host = _native(x)
    if host is not None and _tensors(weight, bias):
        r = host.norm(x, weight, bias, eps, center, _stream_ptr(x))
        if _took(r, "norm"):
            return r
    _need_gpu(x, "x")
    if x.dtype not in _TYPES or x.dim() < 1:
        raise TypeError("x must be a float32 or bfloat16 tensor [..., cols]")
    cols = x.shape[-1]
    if cols < 1:
        raise ValueError(f"x has rows of no elements: {tuple(x.shape)}")
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        _need_gpu(p, name)
        if p.dtype not in _TYPES:
            raise TypeError(f"{name} must be float32 or bfloat16, got {p.dtype}")
        if p.shape != (cols,):
            raise ValueError(f"{name} must have shape ({cols},), got {tuple(p.shape)}")
        if p.device != x.device:
            raise ValueError(f"{name} is on {p.device}, x on {x.device}")
    _no_tangent("layer_norm" if center else "rms_norm", x, weight, bias)
    kind = lambda p: _lib.OUT_F32 if p is None else _TYPES[p.dtype]  # noqa: E731
    opt = _lib.NormOptions(x.numel() // cols, cols, _TYPES[x.dtype], kind(weight),
                           kind(bias), center, eps)
    if torch.is_grad_enabled() and any(
            t is not None and t.requires_grad for t in (x, weight, bias)):
        return Norm.apply(x, weight, bias, opt)
    y, _ = _forward(_rows(x.detach(), cols), *(p.detach().contiguous() if p is not None else None
                                               for p in (weight, bias)), opt, False)
    return y.view(x.shape)


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None,
               bias: torch.Tensor | None = None, eps: float = 1e-5) -> torch.Tensor:
    """Layer norm over the last dimension of x (bf16 or fp32, on the GPU), in x's
    type.  weight, bias: fp32 or bf16 [cols], or None.  Differentiable in x,
    weight and bias."""
    return _norm(x, weight, bias, eps, True)


def rms_norm(x: torch.Tensor, weight: torch.Tensor | None = None,
             eps: float = 1e-6) -> torch.Tensor:
    """Root-mean-square norm over the last dimension of x: x * weight /
    sqrt(mean(x^2) + eps).  Types and gradients as layer_norm."""
    return _norm(x, weight, None, eps, False)
