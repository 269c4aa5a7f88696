"""Layer norm and root-mean-square norm around the expert layer.

    y = layer_norm(x, weight, bias)     (x - mean) / sqrt(var + eps) * weight + bias
    y = rms_norm(x, weight)             x / sqrt(mean(x^2) + eps) * weight
    y, h = add_rms_norm(x, residual, weight)          h = x + residual, y = rms_norm(h)
    q, s, h = rms_norm_quant(x, weight, residual)     y in e4m3 with its scales

Rows are the last dimension of x (bf16 or fp32, at most 32768 long, any length
and row stride).  Statistics are fp32; the backward pass keeps x and two fp32
values a row, and adds the weight's gradient over the rows in a fixed order, so
it is the same on every run.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .ops import (_FP8, _MODES, _block_major_buffer, _first_order, _mode, _native, _need_gpu, _no_tangent,
                  _stream_ptr, _tensors, _took)

__all__ = ["layer_norm", "rms_norm", "Norm", "add_rms_norm", "AddRMSNorm", "rms_norm_quant"]

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
        _first_order("norm", dy)
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


_FORMATS = {"mxfp8": (_lib.QUANT_MX, 32), "fp8_block": (_lib.QUANT_BLOCK, 128)}


def _add_checks(x, residual, weight, eps):
    """Checks that add_rms_norm and rms_norm_quant share; the options of the call."""
    _need_gpu(x, "x")
    if x.dtype not in _TYPES or x.dim() < 1:
        raise TypeError("x must be a float32 or bfloat16 tensor [..., cols]")
    cols = x.shape[-1]
    if cols < 1:
        raise ValueError(f"x has rows of no elements: {tuple(x.shape)}")
    if residual is not None:
        _need_gpu(residual, "residual")
        if residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device:
            raise ValueError(f"residual must be {x.dtype} {tuple(x.shape)} on {x.device}, got "
                             f"{residual.dtype} {tuple(residual.shape)} on {residual.device}")
    if weight is not None:
        _need_gpu(weight, "weight")
        if weight.dtype not in _TYPES:
            raise TypeError(f"weight must be float32 or bfloat16, got {weight.dtype}")
        if weight.shape != (cols,) or weight.device != x.device:
            raise ValueError(f"weight must have shape ({cols},) on {x.device}, got "
                             f"{tuple(weight.shape)} on {weight.device}")
    return _lib.NormOptions(x.numel() // cols, cols, _TYPES[x.dtype],
                            _lib.OUT_F32 if weight is None else _TYPES[weight.dtype],
                            _lib.OUT_F32, 0, eps)


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _add_forward(x2, r2, w, opt, keep):
    h, y = (torch.empty(x2.shape, dtype=x2.dtype, device=x2.device) for _ in range(2))
    stats = torch.empty((2, x2.shape[0]), dtype=torch.float32, device=x2.device) if keep else None
    _lib.check(
        _lib.load().mxgg_add_rms_norm(x2.data_ptr(), _ld(x2), r2.data_ptr(), _ld(r2), _ptr(w),
                                      ctypes.byref(opt), h.data_ptr(), opt.cols, y.data_ptr(),
                                      opt.cols, _ptr(stats), _stream_ptr(x2)), "add_rms_norm")
    return y, h, stats


class AddRMSNorm(torch.autograd.Function):
    """add_rms_norm with its gradients; x and the residual share one."""

    @staticmethod
    def forward(ctx, x, residual, weight, opt):
        w = weight.contiguous() if weight is not None else None
        y, h, stats = _add_forward(_rows(x, opt.cols), _rows(residual, opt.cols), w, opt, True)
        ctx.opt, ctx.shape = opt, x.shape
        ctx.weight_type = weight.dtype if weight is not None else None
        ctx.set_materialize_grads(False)
        h = h.view(x.shape)
        ctx.save_for_backward(h, w, stats)
        return y.view(x.shape), h

    @staticmethod
    def backward(ctx, dy, dh):
        # where only h was used, dh passes through as it is
        _first_order("add_rms_norm", *((dy, dh) if dy is not None else ()))
        h, w, stats = ctx.saved_tensors
        opt, dev = ctx.opt, h.device
        need_w = ctx.needs_input_grad[2]
        need_x = ctx.needs_input_grad[0] or ctx.needs_input_grad[1]
        if dy is None:  # only h was used
            dw = torch.zeros(opt.cols, dtype=ctx.weight_type, device=dev) if need_w else None
            return dh, dh, dw, None
        h2, dy2 = _rows(h, opt.cols), _rows(dy.to(h.dtype), opt.cols)
        dh2 = _rows(dh.to(h.dtype), opt.cols) if dh is not None else None
        dx = torch.empty(h2.shape, dtype=h.dtype, device=dev) if need_x else None
        dw = torch.empty(opt.cols, dtype=ctx.weight_type, device=dev) if need_w else None
        lib = _lib.load()
        ws = None
        if need_w:
            ws = torch.empty(lib.mxgg_norm_grad_workspace_bytes(ctypes.byref(opt)),
                             dtype=torch.uint8, device=dev)
        _lib.check(
            lib.mxgg_add_rms_norm_grad(
                dy2.data_ptr(), _ld(dy2), _ptr(dh2), _ld(dh2) if dh2 is not None else 0,
                h2.data_ptr(), _ld(h2), _ptr(w), stats.data_ptr(), ctypes.byref(opt), _ptr(dx),
                opt.cols, _ptr(dw), _ptr(ws), ws.numel() if ws is not None else 0,
                _stream_ptr(h2)), "add_rms_norm_grad")
        dx = dx.view(ctx.shape) if need_x else None
        return dx, dx, dw, None


def add_rms_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor | None = None,
                 eps: float = 1e-6):
    """(y, h): h = x + residual, rounded to their type, and y = rms_norm(h, weight, eps), in
    one pass.  x, residual: bf16 or fp32 [..., cols] of one type and shape.  weight: fp32 or
    bf16 [cols], or None.  Differentiable in x, residual and weight, through y and h."""
    host = _native(x)
    if host is not None and residual is not None and _tensors(residual, weight):
        r = host.add_norm(x, residual, weight, eps, _stream_ptr(x))
        if _took(r, "add_rms_norm"):
            return r
    opt = _add_checks(x, residual, weight, eps)
    if residual is None:
        raise TypeError("residual must be a torch.Tensor")
    _no_tangent("add_rms_norm", x, residual, weight)
    if torch.is_grad_enabled() and any(
            t is not None and t.requires_grad for t in (x, residual, weight)):
        return AddRMSNorm.apply(x, residual, weight, opt)
    y, h, _ = _add_forward(_rows(x.detach(), opt.cols), _rows(residual.detach(), opt.cols),
                           weight.detach().contiguous() if weight is not None else None, opt,
                           False)
    return y.view(x.shape), h.view(x.shape)


def rms_norm_quant(x: torch.Tensor, weight: torch.Tensor | None = None,
                   residual: torch.Tensor | None = None, eps: float = 1e-6,
                   out_format: str = "mxfp8", scaling_mode: str = "rceil"):
    """(payload, scales, h): rms_norm of h = x + residual (of x without one; h is then None)
    with its result in e4m3, rounded once from fp32.

    out_format "mxfp8": an E8M0 scale for each 32, uint8 [M, cols / 32], the operand of
    grouped_mm, fused_grouped_fwd and fwd_ge (cols a multiple of 32; scaling_mode as
    to_mxfp8_dim0).  "fp8_block": an fp32 scale for each 128, [M, ceil(cols / 128)], the
    operand of fp8_block_mm (cols a multiple of 16).  M: x's leading dimensions together;
    the payload is [M, cols], h has x's shape.  The scales are views of storage laid out
    block by block.  Not differentiable: inputs that require grad are refused while grad
    mode is on."""
    if out_format not in _FORMATS:
        raise ValueError(f"out_format must be one of {sorted(_FORMATS)}, got {out_format!r}")
    host = _native(x, scaling_mode)
    if host is not None and _tensors(weight, residual):
        r = host.rms_quant(x, weight, residual, eps, _FORMATS[out_format][0],
                           _MODES[scaling_mode], _stream_ptr(x))
        if _took(r, "rms_norm_quant"):
            return r
    opt = _add_checks(x, residual, weight, eps)
    _no_tangent("rms_norm_quant", x, residual, weight)
    if torch.is_grad_enabled() and any(
            t is not None and t.requires_grad for t in (x, residual, weight)):
        raise RuntimeError("rms_norm_quant has no gradient: use add_rms_norm, or call it under "
                           "torch.no_grad()")
    code, width = _FORMATS[out_format]
    mode = _mode(scaling_mode)
    M, cols, dev = opt.rows, opt.cols, x.device
    x2 = _rows(x.detach(), cols)
    r2 = _rows(residual.detach(), cols) if residual is not None else None
    w = weight.detach().contiguous() if weight is not None else None
    h = torch.empty(x.shape, dtype=x.dtype, device=dev) if r2 is not None else None
    q = torch.empty((M, cols), dtype=_FP8, device=dev)
    blocks = (cols + width - 1) // width
    if code == _lib.QUANT_MX:
        s = _block_major_buffer(M, blocks, dev)
    else:
        s = torch.empty((blocks, (M + 3) // 4 * 4), dtype=torch.float32, device=dev)
    _lib.check(
        _lib.load().mxgg_rms_norm_quant(
            x2.data_ptr(), _ld(x2), _ptr(r2), _ld(r2) if r2 is not None else 0, _ptr(w),
            ctypes.byref(opt), _ptr(h), cols, q.data_ptr(), cols, s.data_ptr(), s.stride(0), code,
            mode, _stream_ptr(x)), "rms_norm_quant")
    return q, s[:, :M].t(), h
