"""Products in e4m3 with one fp32 scale for each block of 128.

The format of checkpoints and recipes whose scales are not powers of two: activations
in blocks of 1 x 128 along the contraction, weights in tiles of 128 x 128, operands of
the weight gradient in blocks of 128 tokens.

    q, s = to_fp8_block_dim0(x)                  # bf16 [M, K]
    y = fp8_block_mm(q, s, w, w_scales, offs)    # w e4m3 [N, K] or [E, N, K]
    y = fp8_block_linear(x, w, offs)             # bf16 in, differentiable

A scale is max(amax * (1 / 448), 2^-126) in fp32 and the payload e4m3(x / scale), to
nearest even.  Products are summed in fp32, but for each eight consecutive ones: the matrix
instruction cuts those 13 bits below the largest of the eight before it adds them, so that
a result, in fp32 too, is off by 2e-5 in the root mean square of normal data (an fp32 sum
by 7e-7), without a lean to either side.  Widths are multiples of 16; the last block of a
row may be narrower than 128.  With `offs` the rows are grouped by expert as in grouped_mm.  Inputs
that carry a tangent of forward-mode differentiation are refused; casts of inputs that
require grad are not recorded by autograd.
"""
from __future__ import annotations

import torch

from . import _lib
from .ops import (_FP8, _as_u8, _first_order, _group_ends, _mark_ends, _native, _need_gpu,
                  _no_tangent, _out_code, _stream_ptr, _tensors, _took, zero_rows_past_groups)

__all__ = ["to_fp8_block_dim0", "to_fp8_block_dim1", "to_fp8_block_weight", "fp8_block_mm",
           "fp8_block_wgrad", "fp8_block_linear", "FP8BlockLinear"]

_BLOCK = 128


def _blocks(n: int) -> int:
    return (n + _BLOCK - 1) // _BLOCK


def _bf16_rows(x: torch.Tensor, name: str) -> torch.Tensor:
    """x as 2-D bf16 with 16-byte aligned rows (a copy only where it has none)."""
    _need_gpu(x, name)
    if x.dtype != torch.bfloat16 or x.dim() != 2:
        raise TypeError(f"{name} must be a bfloat16 matrix, got {x.dtype} {tuple(x.shape)}")
    if x.shape[1] % 16 != 0:
        raise ValueError(f"{name} has rows of {x.shape[1]} elements, not a multiple of 16")
    x = x.detach()
    if x.stride(1) != 1 or (x.shape[0] > 1 and (x.stride(0) < x.shape[1] or x.stride(0) % 8)) \
            or x.data_ptr() % 16:
        x = x.clone(memory_format=torch.contiguous_format)
    return x


def _ld(t: torch.Tensor) -> int:
    return max(t.stride(0), t.shape[1]) if t.shape[0] > 1 else t.shape[1]


def _scale_buffer(blocks: int, rows: int, device) -> torch.Tensor:
    """Storage of a scale for each row and block, block by block."""
    return torch.empty((blocks, (rows + 3) // 4 * 4), dtype=torch.float32, device=device)


def to_fp8_block_dim0(x: torch.Tensor):
    """(payload e4m3 [M, K], scales fp32 [M, ceil(K / 128)]) of x bf16 [M, K] in blocks
    of 1 x 128 along each row.  The scales are a view of storage laid out block by block."""
    host = _native(x)
    if host is not None:
        r = host.block_dim0(x, _stream_ptr(x))
        if _took(r, "to_fp8_block_dim0"):
            return r
    _need_gpu(x, "x")
    _no_tangent("to_fp8_block_dim0", x)
    x = _bf16_rows(x, "x")
    M, K = x.shape
    q = torch.empty((M, K), dtype=_FP8, device=x.device)
    s = _scale_buffer(_blocks(K), M, x.device)
    _lib.check(_lib.load().mxgg_block_quant_dim0(x.data_ptr(), M, K, _ld(x), q.data_ptr(), K,
                                                 s.data_ptr(), s.stride(0), _stream_ptr(x)),
               "to_fp8_block_dim0")
    return q, s[:, :M].t()


def _dim1(x: torch.Tensor, ends, rows: bool):
    """(q, s, qt, st, ends_pad) of a matrix that _bf16_rows has passed."""
    M, C = x.shape
    E = 0 if ends is None else ends.numel()
    cap = _blocks(M + (_BLOCK - 1) * E) * _BLOCK
    dev = x.device
    qt, st = torch.empty((C, cap), dtype=_FP8, device=dev), _scale_buffer(cap // _BLOCK, C, dev)
    pad = torch.empty(E, dtype=torch.int32, device=dev) if E else None
    q = s = None
    if rows:
        q, s = torch.empty((M, C), dtype=_FP8, device=dev), _scale_buffer(_blocks(C), M, dev)
    _lib.check(
        _lib.load().mxgg_block_quant_dim1(
            x.data_ptr(), M, C, _ld(x), ends.data_ptr() if E else None, E, cap,
            q.data_ptr() if rows else None, C, s.data_ptr() if rows else None,
            s.stride(0) if rows else 0, qt.data_ptr(), st.data_ptr(), st.stride(0),
            pad.data_ptr() if E else None, _stream_ptr(x)), "to_fp8_block_dim1")
    return q, s[:, :M].t() if rows else None, qt, st[:, :C].t(), _mark_ends(pad)


def to_fp8_block_dim1(x: torch.Tensor, offs: torch.Tensor | None = None):
    """(payload e4m3 [C, T], scales fp32 [C, T / 128], padded ends or None) of x bf16
    [M, C] in blocks of 128 tokens of a column, transposed.  The tokens of every group of
    `offs` (all of them without) are padded with zeros to whole blocks."""
    _need_gpu(x, "x")
    _no_tangent("to_fp8_block_dim1", x)
    x = _bf16_rows(x, "x")
    ends = None if offs is None else _ends(offs, x)
    return _dim1(x, ends, False)[2:]


def _ends(offs, like: torch.Tensor) -> torch.Tensor:
    if not isinstance(offs, torch.Tensor) or offs.dim() != 1 or offs.numel() == 0:
        raise ValueError("offs must be a 1-D tensor of at least one group end")
    return _group_ends(offs, offs.numel(), like.device)


def to_fp8_block_weight(w: torch.Tensor, dual: bool = False):
    """(payload e4m3 [..., N, K], scales fp32 [..., ceil(N / 128), ceil(K / 128)]) of w bf16
    [N, K] or [E, N, K] in tiles of 128 x 128; with `dual` also the same payload and
    scales transposed, [..., K, N], the operand of the input gradient (N a multiple of 16)."""
    _need_gpu(w, "w")
    if w.dtype != torch.bfloat16 or w.dim() not in (2, 3):
        raise TypeError(f"w must be bfloat16 [N, K] or [E, N, K], got {w.dtype} {tuple(w.shape)}")
    E = w.shape[0] if w.dim() == 3 else 1
    N, K = w.shape[-2:]
    if K % 16 != 0 or (dual and N % 16 != 0):
        raise ValueError(f"w {tuple(w.shape)}: K (and N with dual) must be multiples of 16")
    _no_tangent("to_fp8_block_weight", w)
    w = w.detach().contiguous()
    if w.data_ptr() % 16:
        w = w.clone()
    batch, dev = tuple(w.shape[:-2]), w.device
    q = torch.empty(w.shape, dtype=_FP8, device=dev)
    s = torch.empty((*batch, _blocks(N), _blocks(K)), dtype=torch.float32, device=dev)
    qt = st = None
    if dual:
        qt = torch.empty((*batch, K, N), dtype=_FP8, device=dev)
        st = torch.empty((*batch, _blocks(K), _blocks(N)), dtype=torch.float32, device=dev)
    _lib.check(
        _lib.load().mxgg_block_quant_weight(w.data_ptr(), E, N, K, q.data_ptr(), s.data_ptr(),
                                            qt.data_ptr() if dual else None,
                                            st.data_ptr() if dual else None, _stream_ptr(w)),
        "to_fp8_block_weight")
    return (q, s, qt, st) if dual else (q, s)


def _payload(t: torch.Tensor, name: str, dims) -> torch.Tensor:
    """An e4m3 (or raw byte) operand with 16-byte aligned rows."""
    if t.dim() not in dims:
        raise ValueError(f"{name} must have {' or '.join(map(str, dims))} dimensions, "
                         f"got {tuple(t.shape)}")
    t = _as_u8(t.detach(), name)
    ok = t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and \
        (t.shape[-2] == 1 or (t.stride(-2) >= t.shape[-1] and t.stride(-2) % 16 == 0)) and \
        (t.dim() == 2 or t.shape[0] == 1
         or (t.stride(0) % 16 == 0 and t.stride(0) >= t.shape[1] * t.stride(1)))
    if not ok:
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def _row_scales(s: torch.Tensor, shape, name: str, device):
    """(scales of one a row and block, stride from block to block), rows consecutive."""
    if s.dtype != torch.float32 or tuple(s.shape) != shape or s.device != device:
        raise ValueError(f"{name} must be float32 {shape} on {device}, got {s.dtype} "
                         f"{tuple(s.shape)} on {s.device}")
    s = s.detach()
    rows, blocks = shape
    if (rows > 1 and s.stride(0) != 1) or (blocks > 1 and s.stride(1) < rows):
        s = s.t().contiguous().t()
    return s, max(s.stride(1), rows) if blocks > 1 else rows


def fp8_block_mm(a: torch.Tensor, a_scales: torch.Tensor, w: torch.Tensor,
                 w_scales: torch.Tensor, offs: torch.Tensor | None = None,
                 out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """a @ w.T for block-scaled e4m3 operands, [M, N] in out_dtype (bf16 or fp32).

    a [M, K] with fp32 scales [M, ceil(K / 128)] (to_fp8_block_dim0); w [N, K] with
    scales [ceil(N / 128), ceil(K / 128)], or [E, N, K] with [E, ...] and `offs`, the
    experts' cumulative row ends (rows past the last one are not written).  K is a
    multiple of 16."""
    out = _out_code(out_dtype)
    host = _native(a)
    if host is not None and isinstance(w, torch.Tensor) and isinstance(a_scales, torch.Tensor) \
            and isinstance(w_scales, torch.Tensor) and _tensors(offs):
        r = host.block_mm(a, a_scales, w, w_scales, offs, out == _lib.OUT_F32, _stream_ptr(a))
        if _took(r, "fp8_block_mm"):
            return r
    for t, name in ((a, "a"), (a_scales, "a_scales"), (w, "w"), (w_scales, "w_scales")):
        _need_gpu(t, name)
    _no_tangent("fp8_block_mm", a, a_scales, w, w_scales)
    a = _payload(a, "a", (2,))
    w = _payload(w, "w", (2, 3))
    M, K = a.shape
    N = w.shape[-2]
    E = w.shape[0] if w.dim() == 3 else 1
    if w.shape[-1] != K or w.device != a.device:
        raise ValueError(f"w {tuple(w.shape)} on {w.device} does not fit a {tuple(a.shape)} "
                         f"on {a.device}")
    if (offs is None) != (w.dim() == 2):
        raise ValueError("offs goes with weights [E, N, K]")
    a_s, ldas = _row_scales(a_scales, (M, _blocks(K)), "a_scales", a.device)
    shape = (*w.shape[:-2], _blocks(N), _blocks(K))
    if w_scales.dtype != torch.float32 or tuple(w_scales.shape) != shape \
            or w_scales.device != a.device:
        raise ValueError(f"w_scales must be float32 {shape} on {a.device}, got {w_scales.dtype} "
                         f"{tuple(w_scales.shape)} on {w_scales.device}")
    ws = w_scales.detach()
    if not ws.is_contiguous():
        ws = ws.contiguous()
    ends = None if offs is None else _group_ends(offs, E, a.device)
    y = torch.empty((M, N), dtype=out_dtype, device=a.device)
    lib = _lib.load()
    nbytes = lib.mxgg_block_mm_workspace_bytes(offs is not None, E, M, N, K)
    ws_buf = torch.empty(nbytes, dtype=torch.uint8, device=a.device) if nbytes > 0 else None
    _lib.check(
        lib.mxgg_block_mm(
            a.data_ptr(), _ld(a), a_s.data_ptr(), ldas, w.data_ptr(),
            w.stride(0) if w.dim() == 3 and E > 1 else N * K, _ld(w[0] if w.dim() == 3 else w),
            ws.data_ptr(), _blocks(N) * _blocks(K), _blocks(K),
            ends.data_ptr() if ends is not None else None, E, M, N, K, y.data_ptr(), N, out,
            ws_buf.data_ptr() if ws_buf is not None else None, max(nbytes, 0), _stream_ptr(a)),
        "fp8_block_mm")
    return y


def fp8_block_wgrad(go_t: torch.Tensor, go_scales: torch.Tensor, ia_t: torch.Tensor,
                    ia_scales: torch.Tensor, offs_pad: torch.Tensor | None = None,
                    out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """dY^T X for operands in blocks of 128 tokens (to_fp8_block_dim1): go_t [N, T] with
    scales [N, T / 128], ia_t [K, T] with [K, T / 128].  Returns [N, K], or [E, N, K] for
    the padded ends that the casts return (every entry a multiple of 128).  Sums as at the
    head of this file, in fp32 output as well."""
    out = _out_code(out_dtype)
    for t, name in ((go_t, "go_t"), (go_scales, "go_scales"), (ia_t, "ia_t"), (ia_scales, "ia_scales")):
        _need_gpu(t, name)
    _no_tangent("fp8_block_wgrad", go_t, go_scales, ia_t, ia_scales)
    go, ia = _payload(go_t, "go_t", (2,)), _payload(ia_t, "ia_t", (2,))
    N, T = go.shape
    K = ia.shape[0]
    if ia.shape[1] != T or T % _BLOCK or ia.device != go.device:
        raise ValueError(f"go_t {tuple(go.shape)} and ia_t {tuple(ia.shape)} must hold the same "
                         "tokens, a multiple of 128, on one device")
    gs, ldgs = _row_scales(go_scales, (N, T // _BLOCK), "go_scales", go.device)
    xs, ldxs = _row_scales(ia_scales, (K, T // _BLOCK), "ia_scales", go.device)
    ends = None if offs_pad is None else _ends(offs_pad, go)
    E = 1 if ends is None else ends.numel()
    dw = torch.empty((E, N, K), dtype=out_dtype, device=go.device)
    lib = _lib.load()
    nbytes = lib.mxgg_block_wgrad_workspace_bytes(ends is not None, E, T, N, K)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=go.device) if nbytes > 0 else None
    _lib.check(
        lib.mxgg_block_wgrad(go.data_ptr(), _ld(go), gs.data_ptr(), ldgs, ia.data_ptr(),
                                     _ld(ia), xs.data_ptr(), ldxs,
                                     ends.data_ptr() if ends is not None else None, E, T, N, K,
                                     dw.data_ptr(), out, ws.data_ptr() if ws is not None else None,
                                     max(nbytes, 0), _stream_ptr(go)), "fp8_block_wgrad")
    return dw if ends is not None else dw[0]


class FP8BlockLinear(torch.autograd.Function):
    """fp8_block_linear with both gradients.  Kept for the backward pass: the transposed
    casts of x (for w's gradient) and of w (for x's).  grad: grad mode where it is applied
    (needs_input_grad does not know it, and in here it is off)."""

    @staticmethod
    def forward(ctx, x, w, ends, grad=True):
        need_x, need_w = (grad and n for n in ctx.needs_input_grad[:2])
        x2 = _bf16_rows(x, "x")
        if need_w:
            q, s, qt, st, pad = _dim1(x2, ends, True)
        else:
            (q, s), qt, st, pad = to_fp8_block_dim0(x2), None, None, None
        wq = to_fp8_block_weight(w, dual=need_x)
        y = fp8_block_mm(q, s, wq[0], wq[1], ends)
        if ends is not None:
            zero_rows_past_groups(y, ends)
        ctx.save_for_backward(qt, st, pad, ends, *(wq[2:] if need_x else (None, None)))
        return y

    @staticmethod
    def backward(ctx, dy):
        _first_order("fp8_block_linear", dy)
        qt, st, pad, ends, wt, wts = ctx.saved_tensors
        need_x, need_w = ctx.needs_input_grad[:2]
        dy = _bf16_rows(dy.to(torch.bfloat16), "dy")
        dx = dw = None
        if need_w:
            q, s, gt, gs, _ = _dim1(dy, ends, need_x)
            dw = fp8_block_wgrad(gt, gs, qt, st, pad, out_dtype=torch.bfloat16)
        else:
            q, s = to_fp8_block_dim0(dy)
        if need_x:
            dx = fp8_block_mm(q, s, wt, wts, ends)
            if ends is not None:
                zero_rows_past_groups(dx, ends)
        return dx, dw, None, None


def fp8_block_linear(x: torch.Tensor, w: torch.Tensor,
                     offs: torch.Tensor | None = None) -> torch.Tensor:
    """x @ w.T with both operands cast to block-scaled e4m3: x bf16 [..., K]; w bf16 [N, K],
    or [E, N, K] with x [M, K] grouped by `offs` (rows past the last end are 0, with
    gradients of 0).  N and K are multiples of 16.  Differentiable in x and w: the
    gradients' products are block-scaled as well, dy in blocks along N for x's and in
    blocks of tokens, as x, for w's."""
    host = _native(x)
    if host is not None and isinstance(w, torch.Tensor) and _tensors(offs):
        r = host.block_linear(x, w, offs, _stream_ptr(x))
        if _took(r, "fp8_block_linear"):
            return r
    _need_gpu(x, "x")
    _need_gpu(w, "w")
    if x.dtype != torch.bfloat16 or w.dtype != torch.bfloat16:
        raise TypeError(f"x and w must be bfloat16, got {x.dtype} and {w.dtype}")
    if w.device != x.device:
        raise ValueError(f"w is on {w.device}, x on {x.device}")
    if w.dim() not in (2, 3) or x.dim() < 1 or x.shape[-1] != w.shape[-1]:
        raise ValueError(f"shapes must be x [..., K] and w [N, K] or [E, N, K], got "
                         f"{tuple(x.shape)} and {tuple(w.shape)}")
    if (offs is None) != (w.dim() == 2) or (w.dim() == 3 and x.dim() != 2):
        raise ValueError("offs and x [M, K] go with weights [E, N, K]")
    N, K = w.shape[-2:]
    if N % 16 or K % 16 or N == 0 or K == 0:
        raise ValueError(f"N={N} and K={K} must be positive multiples of 16")
    _no_tangent("fp8_block_linear", x, w)
    ends = None if offs is None else _group_ends(offs, w.shape[0], x.device)
    y = FP8BlockLinear.apply(x.reshape(-1, K), w, ends, torch.is_grad_enabled())
    return y.view(*x.shape[:-1], N)
