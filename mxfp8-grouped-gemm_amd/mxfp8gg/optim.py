"""AdamW over many tensors at once, with states in 32 or in 8 bits, and the clipping of
their gradients' global norm.

    opt = AdamW(model.parameters(), lr=1e-3, state_bits=8)
    loss.backward(); opt.clip_grad_norm_(1.0); opt.step()

One kernel launch updates up to 48 tensors (weights and gradients bf16 or fp32).
8-bit states are MXFP8 as the rest of this package uses it: e4m3 payloads with
one E8M0 scale for every 32 consecutive elements; the second moment is kept as
its root.  What is below about 2^-18 of its block's largest value is stored as 0, so a
weight whose gradients are that small beside its neighbours' has no second moment from
one step to the next.  The update marks the weights as modified (torch's version counter),
so a WeightCastCache casts them again.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .ops import _FP8, _native, _need_gpu, _no_tangent, _stream_ptr, _tensors, _took

__all__ = ["AdamW", "adamw_step", "adamw_state", "grad_norm", "clip_grad_norm_"]

_TYPES = {torch.float32: _lib.OUT_F32, torch.bfloat16: _lib.OUT_BF16}


def adamw_state(param: torch.Tensor, state_bits: int = 32):
    """A zero state for `param`: an fp32 tensor of its shape (32), or the pair
    (e4m3 payload of its shape, uint8 E8M0 scales [ceil(numel / 32)]) (8)."""
    if state_bits == 32:
        return torch.zeros(param.shape, dtype=torch.float32, device=param.device)
    if state_bits != 8:
        raise ValueError(f"state_bits must be 8 or 32, got {state_bits!r}")
    q = torch.zeros(param.shape, dtype=torch.uint8, device=param.device).view(_FP8)
    return q, torch.ones((param.numel() + 31) // 32, dtype=torch.uint8, device=param.device)


def _dense(t, name, like, types):
    if not isinstance(t, torch.Tensor) or t.device != like.device:
        raise ValueError(f"{name} must be a tensor on {like.device}")
    if t.dtype not in types:
        raise TypeError(f"{name} must be one of {[str(x) for x in types]}, got {t.dtype}")
    if not t.is_contiguous() or t.numel() != like.numel():
        raise ValueError(f"{name} must be contiguous with the weight's {like.numel()} elements, "
                         f"got {tuple(t.shape)} with strides {t.stride()}")
    return t


def _scales(t, name, like):
    if not isinstance(t, torch.Tensor) or t.device != like.device or t.dtype != torch.uint8 \
            or not t.is_contiguous() or t.numel() != (like.numel() + 31) // 32:
        raise ValueError(f"{name} must be contiguous uint8 [ceil(numel / 32)] on {like.device}")
    return t


def adamw_step(params, grads, exp_avg, exp_avg_sq, step: int, lr: float = 1e-3,
               betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.01,
               masters=None) -> None:
    """One AdamW step of every tensor of `params`, in place, on the current stream.

    params, grads: lists of contiguous fp32 or bf16 tensors (each its own type).
    exp_avg, exp_avg_sq: their states, all fp32 tensors or all (payload, scales)
    pairs as adamw_state makes them (8 bits; exp_avg_sq then holds the root).
    masters: fp32 copies of the weights, or None; with them the step is taken on
    the copies and `params` are written as their rounding.  step: the number of
    this update, from 1.  step, lr and the other numbers are arguments of the launch:
    a captured graph repeats the captured ones at every replay."""
    params, grads, exp_avg, exp_avg_sq = map(list, (params, grads, exp_avg, exp_avg_sq))
    masters = list(masters) if masters is not None else []
    n = len(params)
    if not len(grads) == len(exp_avg) == len(exp_avg_sq) == n or (masters and len(masters) != n):
        raise ValueError("params, grads, states and masters must be lists of one length")
    if n == 0:
        return
    _need_gpu(params[0], "params[0]")
    small = isinstance(exp_avg[0], (tuple, list))
    if any(isinstance(s, (tuple, list)) != small for s in exp_avg + exp_avg_sq):
        raise ValueError("the states of one step are all 32-bit tensors or all 8-bit pairs")
    if small:
        ms, vs = [s[1] for s in exp_avg], [s[1] for s in exp_avg_sq]
        exp_avg, exp_avg_sq = [s[0] for s in exp_avg], [s[0] for s in exp_avg_sq]
    else:
        ms = vs = []
    host = _native(params[0])
    if host is not None and _tensors(*params, *grads, *exp_avg, *exp_avg_sq, *ms, *vs, *masters):
        r = host.adamw(params, grads, exp_avg, exp_avg_sq, ms, vs, masters, step, lr, betas[0],
                       betas[1], eps, weight_decay, _stream_ptr(params[0]))
        if _took(r, "adamw_step"):
            return
    opt = _lib.AdamwOptions(lr, betas[0], betas[1], eps, weight_decay, step, 8 if small else 32)
    first = params[0]
    table = (_lib.AdamwTensor * n)()
    for i, p in enumerate(params):
        if not isinstance(p, torch.Tensor) or p.device != first.device:
            raise ValueError(f"params[{i}] must be a tensor on {first.device}")
        e = table[i]
        e.param = _dense(p, f"params[{i}]", p, _TYPES).data_ptr()
        e.grad = _dense(grads[i], f"grads[{i}]", p, _TYPES).data_ptr()
        types = (_FP8, torch.uint8) if small else (torch.float32,)
        e.exp_avg = _dense(exp_avg[i], f"exp_avg[{i}]", p, types).data_ptr()
        e.exp_avg_sq = _dense(exp_avg_sq[i], f"exp_avg_sq[{i}]", p, types).data_ptr()
        if small:
            e.exp_avg_scales = _scales(ms[i], f"exp_avg[{i}] scales", p).data_ptr()
            e.exp_avg_sq_scales = _scales(vs[i], f"exp_avg_sq[{i}] scales", p).data_ptr()
        if masters:
            e.master = _dense(masters[i], f"masters[{i}]", p, (torch.float32,)).data_ptr()
        e.n = p.numel()
        e.param_dtype = _TYPES[p.dtype]
        e.grad_dtype = _TYPES[grads[i].dtype]
    _lib.check(_lib.load().mxgg_adamw_step(table, n, ctypes.byref(opt), _stream_ptr(first)),
               "adamw_step")
    torch.autograd.graph.increment_version([*params, *exp_avg, *exp_avg_sq, *ms, *vs, *masters])


def _own_memory(t: torch.Tensor) -> bool:
    """Whether t's elements fill one stretch of memory, each once, in any order of its
    dimensions."""
    expect = 1
    for stride, size in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n > 1):
        if stride != expect:
            return False
        expect *= size
    return True


def _grad_table(grads, written):
    """The tensors' table for the library; written: it scales them."""
    table = (_lib.GradTensor * max(len(grads), 1))()
    seen = set()
    for i, g in enumerate(grads):
        _need_gpu(g, f"grads[{i}]")
        if g.device != grads[0].device:
            raise ValueError(f"grads[{i}] is on {g.device}, grads[0] on {grads[0].device}")
        if g.layout != torch.strided or g.dtype not in _TYPES:
            raise TypeError(f"grads[{i}] must be a dense float32 or bfloat16 tensor, got {g.dtype} "
                            f"({g.layout})")
        if written and g.requires_grad and g.is_leaf:
            raise ValueError(f"grads[{i}] is a parameter (a leaf that requires grad) and would be "
                             "scaled itself: pass the parameters' gradients")
        if not _own_memory(g):
            raise ValueError(f"grads[{i}] must fill its memory without gaps or overlap, got "
                             f"{tuple(g.shape)} with strides {g.stride()}")
        if g.numel() and g.data_ptr() in seen:
            raise ValueError(f"grads[{i}] is in the list twice")
        seen.add(g.data_ptr())
        table[i] = _lib.GradTensor(g.data_ptr(), g.numel(), _TYPES[g.dtype])
    if not grads:
        raise ValueError("grads is empty")
    return table


def _clip(grads, what, options=None):
    grads = [grads] if isinstance(grads, torch.Tensor) else list(grads)
    host = _native(grads[0]) if grads else None
    if host is not None and all(isinstance(g, torch.Tensor) for g in grads):
        r = host.clip(grads, -1.0 if options is None else options.max_norm,
                      0.0 if options is None else options.eps, _stream_ptr(grads[0]))
        if _took(r, what):
            return r
    table = _grad_table(grads, options is not None)
    _no_tangent(what, *grads)
    lib, n = _lib.load(), len(grads)
    dev = grads[0].device
    norm = torch.empty((), dtype=torch.float32, device=dev)
    nbytes = lib.mxgg_grad_norm_workspace_bytes(table, n)
    ws = torch.empty(max(nbytes, 0), dtype=torch.uint8, device=dev)
    rest = (norm.data_ptr(), ws.data_ptr(), nbytes, _stream_ptr(grads[0]))
    _lib.check(lib.mxgg_grad_norm(table, n, *rest) if options is None else
               lib.mxgg_clip_grad_norm(table, n, ctypes.byref(options), *rest), what)
    if options is not None:
        torch.autograd.graph.increment_version(grads)
    return norm


def grad_norm(grads) -> torch.Tensor:
    """sqrt(sum of g^2) over all tensors of the list (bf16 or fp32, on one device), fp32 on
    the device.  Squares and sums are fp64; the same bits on every run."""
    return _clip(grads, "grad_norm")


def clip_grad_norm_(grads, max_norm: float, eps: float = 1e-6) -> torch.Tensor:
    """Scale the gradients of the list in place by min(1, max_norm / (norm + eps)), norm being
    grad_norm(grads), which is returned.  Nothing waits for the device, and where nothing is
    clipped no gradient is written: nothing ever is where max_norm is infinite, whatever the
    norm short of NaN.  A norm that is NaN makes the gradients NaN, an infinite one makes
    the finite ones 0.  The tensors may be laid out in any order of
    their dimensions but must not overlap.  Parameters themselves (leaves that require
    grad, which torch's function of the name takes) are refused; the scaling is not
    recorded by autograd."""
    max_norm, eps = float(max_norm), float(eps)
    if not (max_norm >= 0 and eps >= 0):
        raise ValueError(f"max_norm and eps must not be negative, got {max_norm} and {eps}")
    return _clip(grads, "clip_grad_norm_", _lib.ClipOptions(max_norm, eps))


class AdamW(torch.optim.Optimizer):
    """AdamW (decoupled weight decay) on adamw_step: a torch optimizer with
    parameter groups, learning-rate schedulers and state_dict as torch's own.

    state_bits      32: fp32 moments; 8: MXFP8 moments, 2.06 bytes a weight
    master_weights  keep an fp32 copy of every bf16 weight and step on it

    Weights are fp32 or bf16 and contiguous; gradients fp32 or bf16 (a gradient
    of another layout is copied).  Parameters without a gradient are skipped.
    step() raises while the stream is captured into a graph, whose replays would repeat
    one step number and learning rate."""

    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 0.01, state_bits: int = 32, master_weights: bool = False):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {state_bits!r}")
        if lr < 0 or eps < 0 or weight_decay < 0 or not all(0 <= b < 1 for b in betas):
            raise ValueError(f"invalid lr={lr}, betas={betas}, eps={eps} or "
                             f"weight_decay={weight_decay}")
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay,
                                      state_bits=state_bits, master_weights=master_weights))

    def _state_of(self, p, group):
        state = self.state[p]
        if not state:
            state["step"] = 0
            for name in ("exp_avg", "exp_avg_sq"):
                s = adamw_state(p.detach(), group["state_bits"])
                if group["state_bits"] == 8:
                    state[name], state[name + "_scales"] = s
                else:
                    state[name] = s
            if group["master_weights"] and p.dtype != torch.float32:
                state["master"] = p.detach().to(torch.float32)
        return state

    def clip_grad_norm_(self, max_norm: float) -> torch.Tensor | None:
        """clip_grad_norm_ over every parameter's gradient, between backward() and step();
        None where there is no gradient."""
        grads = [p.grad for group in self.param_groups for p in group["params"]
                 if p.grad is not None]
        return clip_grad_norm_(grads, max_norm) if grads else None

    @torch.no_grad()
    def step(self, closure=None):
        if torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW.step in a graph capture: every replay would repeat this "
                               "step's number and learning rate")
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            runs = {}  # tensors that are at the same step and alike in having a master copy
            for p in group["params"]:
                if p.grad is None:
                    continue
                state = self._state_of(p, group)
                runs.setdefault((state["step"] + 1, "master" in state, p.device), []).append(
                    (p, state))
            for (step, master, _), run in runs.items():
                if group["state_bits"] == 8:
                    moments = [[(s[n], s[n + "_scales"]) for _, s in run]
                               for n in ("exp_avg", "exp_avg_sq")]
                else:
                    moments = [[s[n] for _, s in run] for n in ("exp_avg", "exp_avg_sq")]
                adamw_step([p.detach() for p, _ in run], [p.grad.contiguous() for p, _ in run],
                           *moments, step=step, lr=float(group["lr"]), betas=group["betas"],
                           eps=group["eps"], weight_decay=group["weight_decay"],
                           masters=[s["master"] for _, s in run] if master else None)
                for _, state in run:  # not of a step that was refused
                    state["step"] = step
        return loss

    def load_state_dict(self, state_dict):
        """As torch's, with every state in its own type: the base class would
        convert fp32 and e4m3 states to the type of their weight."""
        super().load_state_dict(state_dict)
        for saved, group in zip(state_dict["param_groups"], self.param_groups):
            for key, p in zip(saved["params"], group["params"]):
                if key in state_dict["state"]:
                    self.state[p] = {
                        k: v.to(p.device, copy=True) if isinstance(v, torch.Tensor) else v
                        for k, v in state_dict["state"][key].items()}
