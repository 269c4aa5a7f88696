"""More operators around the routed expert FFN, as measurable cases.

The dense layers around the experts, the residual stream between them, and what a
training step does before the optimizer's:

  `block`  products in e4m3 with an fp32 scale for each block of 128 (activations
           1 x 128 along the contraction, weights 128 x 128), dense or grouped by
           expert, with the activations' cast; in training both gradients
  `norm`   root-mean-square norm with the residual's addition, its result in the
           input's type (with gradients) or in 8 bits (MXFP8, or blocks of 128)
  `logp`   log probabilities of given tokens with entropy and top alternatives, and
           the gradient of the first two
  `clip`   the global gradient norm over many tensors, and clipping in place

Hidden size 7168, projections of 4096 x 7168 and 32 experts are the layer of this
repository's benchmark; the other sizes are generic.

With `own` false, `run` computes the plain form: elementary torch operations in
32 bits, rounded once at the end.
"""
import math
import sys
from pathlib import Path

import torch

own = False

DEV = "cuda"
NEG = float("-inf")
E4M3 = torch.float8_e4m3fn
BLOCK = 128


def _package():
    path = str(Path.cwd() / "mxfp8-grouped-gemm_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import mxfp8gg

    return mxfp8gg


def listed():
    return [
        # Serving: the gate+up projection of a dense layer for the one token of a
        # decode step, weights as a checkpoint holds them.  The weights' bytes count.
        dict(name="block_decode", kind="block", tokens=1, n=4096, k=7168, experts=0, train=False),
        # Serving: a prompt of odd length through a projection whose width is no
        # multiple of the block.
        dict(name="block_prompt", kind="block", tokens=1003, n=2112, k=7168, experts=0,
             train=False),
        # Serving a large batch: gate+up of the benchmark layer's 32 experts, uneven groups.
        dict(name="block_experts", kind="block", tokens=16384, n=4096, k=7168, experts=32,
             train=False),
        # Training: forward, input and weight gradient of a dense projection, the casts
        # of activations, weights and gradients among them.
        dict(name="block_train", kind="block", tokens=8192, n=4096, k=7168, experts=0, train=True),
        # Serving: residual, norm and MXFP8 cast in front of a layer for 64 decoded tokens.
        dict(name="norm_mxfp8_decode", kind="norm", rows=64, cols=7168, out="mxfp8",
             dtype="bfloat16", train=False),
        # Serving a large batch: the same into blocks of 128.
        dict(name="norm_block_prompt", kind="norm", rows=16384, cols=7168, out="fp8_block",
             dtype="bfloat16", train=False),
        # Training: residual and norm, forward and backward.
        dict(name="norm_train", kind="norm", rows=16384, cols=7168, out="same", dtype="bfloat16",
             train=True),
        # Serving: the decoded tokens of a batch of 16 with 8 alternatives each.
        dict(name="logp_decode", kind="logp", tokens=16, vocab=131072, topk=8, dtype="bfloat16",
             temperature=1.0, masked=False, ignored=False, train=False),
        # Evaluation of a policy: odd vocabulary in fp32, some words not allowed, prompt
        # tokens ignored, 20 alternatives.
        dict(name="logp_odd", kind="logp", tokens=1000, vocab=50021, topk=20, dtype="float32",
             temperature=0.7, masked=True, ignored=True, train=False),
        # Policy training: log probabilities and entropy of 4096 tokens with the gradient.
        dict(name="logp_train", kind="logp", tokens=4096, vocab=131072, topk=0, dtype="bfloat16",
             temperature=1.0, masked=False, ignored=False, train=True),
        # The small gradients of a model (norm weights, biases, router): 64 tensors of odd
        # sizes.  Launches, not bytes, set the time.
        dict(name="clip_small", kind="clip", tensors=64, largest=7169, dtype="float32"),
        # The gate+up gradients of 8 experts in bf16.
        dict(name="clip_experts", kind="clip", tensors=8, largest=4096 * 7168, dtype="bfloat16"),
    ]


def _log(rng, lo, hi, step=1):
    """A multiple of `step` in [lo, hi], spread over the logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def draw(rng):
    """One more case of the listed kinds: sizes from the smallest to the largest
    listed ones, odd ones among them."""
    most = {k: max(_cost(c) for c in listed() if c["kind"] == k)
            for k in ("block", "norm", "logp", "clip")}
    while True:
        kind = rng.choice(sorted(most))
        if kind == "block":
            c = dict(kind=kind, tokens=_log(rng, 1, 16384),
                     n=rng.choice([_log(rng, 128, 8192, 16), _log(rng, 128, 8192, 128)]),
                     k=rng.choice([_log(rng, 128, 8192, 16), _log(rng, 128, 8192, 128)]),
                     experts=rng.choice([0, 0, 1, 4, 8, 32]), train=rng.random() < 0.5)
        elif kind == "norm":
            out = rng.choice(["same", "mxfp8", "fp8_block"])
            step = {"same": 1, "mxfp8": 32, "fp8_block": 16}[out]
            c = dict(kind=kind, rows=_log(rng, 1, 65536), cols=_log(rng, 64, 16384, step), out=out,
                     dtype=rng.choice(["float32", "bfloat16", "bfloat16"]),
                     train=out == "same" and rng.random() < 0.7)
        elif kind == "logp":
            c = dict(kind=kind, tokens=_log(rng, 1, 4096),
                     vocab=rng.choice([_log(rng, 1000, 200000), _log(rng, 1024, 131072, 256)]),
                     topk=rng.choice([0, 1, 5, 8, 20, 32]),
                     dtype=rng.choice(["float32", "bfloat16"]),
                     temperature=rng.choice([1.0, 1.0, 0.6, 1.7]), masked=rng.random() < 0.3,
                     ignored=rng.random() < 0.4, train=rng.random() < 0.5)
            if c["topk"] and c["tokens"] * c["vocab"] > 1000 * 131072:
                continue
        else:
            c = dict(kind=kind, tensors=_log(rng, 1, 100), largest=_log(rng, 100, 3e7),
                     dtype=rng.choice(["float32", "bfloat16"]))
        if _cost(c) <= most[kind]:
            return c


# ---------------------------------------------------------------------------
# sizes and work
# ---------------------------------------------------------------------------
def _cost(case):
    """Seconds a pass cannot go below at nominal rates (for comparing cases)."""
    w = work(case)
    rate = 5e15 if case["kind"] == "block" else 2.5e15
    return max(w["bytes"] / 8e12, w["flops"] / rate)


def _sizes(case):
    """Elements of every gradient: the largest first, then odd fractions of it;
    equal ones where they are expert weights."""
    n, most = case["tensors"], case["largest"]
    if most % 4096 == 0:
        return [most] * n
    return [max(1, most * (n - i) // n - i % 7) for i in range(n)]


def _width(name):
    return {"float32": 4, "bfloat16": 2}[name]


def work(case):
    kind = case["kind"]
    if kind == "block":
        t, n, k, e = case["tokens"], case["n"], case["k"], max(1, case["experts"])
        if case["train"]:  # x, w, dy in and y, dx, dw out, all bf16
            return {"bytes": 2 * (2 * t * k + 2 * t * n + 2 * e * n * k), "flops": 6 * t * n * k}
        used = min(e, t)   # experts that have a token
        return {"bytes": 2 * t * k + 2 * t * n + used * (n * k + n * k // 4096),
                "flops": 2 * t * n * k}
    if kind == "norm":
        n, b = case["rows"] * case["cols"], _width(case["dtype"])
        out = {"same": b, "mxfp8": 1 + 1 / 32, "fp8_block": 1 + 4 / 128}[case["out"]]
        moved = n * (3 * b + out) + 4 * case["cols"]
        if case["train"]:
            moved += 4 * n * b + 8 * case["cols"]
        return {"bytes": int(moved), "flops": n * (20 if case["train"] else 6)}
    if kind == "logp":
        n, b = case["tokens"] * case["vocab"], _width(case["dtype"])
        return {"bytes": n * b * (3 if case["train"] else 1) + case["tokens"] * (16 + 8 * case["topk"]),
                "flops": n * (12 if case["train"] else 6)}
    n = sum(_sizes(case))
    return {"bytes": 3 * n * _width(case["dtype"]), "flops": 3 * n}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _normal(gen, shape, scale=1.0, dtype=torch.float32, shift=0.0):
    return torch.empty(shape, dtype=dtype, device=DEV).normal_(shift, scale, generator=gen)


def _uniform(gen, shape):
    return torch.rand(shape, generator=gen, device=DEV)


def _padded(x, *dims):
    """x with zeros up to whole blocks along the given dimensions."""
    size = list(x.shape)
    for d in dims:
        size[d] = (size[d] + BLOCK - 1) // BLOCK * BLOCK
    out = x.new_zeros(size)
    out[tuple(slice(0, s) for s in x.shape)] = x
    return out


def _prepare_block(gen, case):
    t, n, k, e = case["tokens"], case["n"], case["k"], case["experts"]
    x = _normal(gen, (t, k), 1.0, torch.bfloat16)
    x[:, :: 97] *= 8                       # the channels that stand out in activations
    w = _normal(gen, (e or 1, n, k), 1 / math.sqrt(k), torch.bfloat16)
    w *= 0.5 + _uniform(gen, (e or 1, n, 1)).to(w.dtype)
    s = dict(x=x, sizes=[t], offs=None)
    if e:  # uneven groups, some of them empty
        share = _uniform(gen, (e,)).pow(2).cpu()
        ends = (share.cumsum(0) / share.sum() * t).round().to(torch.int32)
        ends[-1] = t
        s["sizes"] = torch.diff(ends, prepend=ends.new_zeros(1)).tolist()
        s["offs"] = ends.to(DEV)
    if case["train"]:
        s["x"].requires_grad_(True)
        s["w"] = (w if e else w[0]).requires_grad_(True)
        s["dy"] = _normal(gen, (t, n), 1e-3, torch.bfloat16)
        return s
    # the checkpoint's weights: payload and scales [E, N / 128, K / 128]
    q, scale = [], []
    for i in range(e or 1):
        b = _padded(w[i].float(), 0, 1)
        b = b.view(b.shape[0] // BLOCK, BLOCK, b.shape[1] // BLOCK, BLOCK)
        sc = (b.abs().amax(dim=(1, 3), keepdim=True) / 448).clamp_min(2.0 ** -126)
        q.append((b / sc).reshape(sc.shape[0] * BLOCK, -1)[:n, :k].to(E4M3))
        scale.append(sc[:, 0, :, 0])
    if e:
        s["w"] = torch.stack([p.view(torch.uint8) for p in q]).view(E4M3)
        s["ws"] = torch.stack(scale)
    else:
        s["w"], s["ws"] = q[0].contiguous(), scale[0].contiguous()
    return s


def _prepare_norm(gen, case):
    shape, dtype = (case["rows"], case["cols"]), getattr(torch, case["dtype"])
    s = dict(x=_normal(gen, shape, 0.6, dtype), residual=_normal(gen, shape, 1.7, dtype, 0.1),
             w=_normal(gen, (case["cols"],), 0.1, shift=1.0))
    if case["train"]:
        s["dy"] = _normal(gen, shape, 1e-2, dtype)
        s["dh"] = _normal(gen, shape, 1e-2, dtype)
        for name in ("x", "residual", "w"):
            s[name].requires_grad_(True)
    return s


def _prepare_logp(gen, case):
    t, v = case["tokens"], case["vocab"]
    # frequent words score higher for every token, one stands out here and there
    lean = -1.2 * torch.log(1 + torch.arange(v, device=DEV, dtype=torch.float32) / 20)
    z = torch.empty((t, v), dtype=getattr(torch, case["dtype"]), device=DEV)
    for i in range(0, t, 512):
        z[i:i + 512] = _normal(gen, (min(512, t - i), v), 2.0) + lean
    target = (v ** _uniform(gen, (t,)) - 1).long().clamp_(0, v - 1)
    rows = torch.arange(t, device=DEV)
    z[rows, target] += (6 * _uniform(gen, (t,))).to(z.dtype)
    if case["masked"]:  # words that the sampler's grammar forbids, for every token alike
        dead = _uniform(gen, (v,)) < 0.2
        dead[0] = False
        z[:, dead] = NEG
        target = torch.where(dead[target], 0, target)
    if case["ignored"]:
        target[1:][_uniform(gen, (t - 1,)) < 0.3] = -100
    return dict(z=z.requires_grad_(case["train"]), target=target,
                dlogp=_normal(gen, (t,), 1e-2), dent=_normal(gen, (t,), 1e-3))


def _prepare_clip(gen, case):
    dtype = getattr(torch, case["dtype"])
    grads = [_normal(gen, (n,), 1e-3, dtype) for n in _sizes(case)]
    # the norm is about six times what is allowed
    most = 1e-3 * math.sqrt(sum(_sizes(case))) / 6
    return dict(grads=grads, max_norm=most)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    make = {"block": _prepare_block, "norm": _prepare_norm, "logp": _prepare_logp,
            "clip": _prepare_clip}
    return dict(make[case["kind"]](gen, case), case=dict(case))


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def _run_own(s):
    m, c = _package(), s["case"]
    if c["kind"] == "block":
        if c["train"]:
            y = m.fp8_block_linear(s["x"], s["w"], s["offs"])
            dx, dw = torch.autograd.grad(y, (s["x"], s["w"]), s["dy"])
            return dict(y=y.detach(), dx=dx, dw=dw)
        q, scale = m.to_fp8_block_dim0(s["x"])
        return dict(y=m.fp8_block_mm(q, scale, s["w"], s["ws"], s["offs"]))
    if c["kind"] == "norm":
        if c["out"] != "same":
            q, scale, h = m.rms_norm_quant(s["x"], s["w"], s["residual"], out_format=c["out"])
            return dict(q=q, scales=_scale_values(scale), h=h)
        y, h = m.add_rms_norm(s["x"], s["residual"], s["w"])
        if not c["train"]:
            return dict(y=y, h=h)
        names = ("x", "residual", "w")
        grads = torch.autograd.grad((y, h), [s[n] for n in names], (s["dy"], s["dh"]))
        return dict({"d" + n: g for n, g in zip(names, grads)}, y=y.detach(), h=h.detach())
    if c["kind"] == "logp":
        r = m.token_log_probs(s["z"], s["target"], temperature=c["temperature"], topk=c["topk"])
        out = dict(logp=r.log_probs.detach(), entropy=r.entropy.detach())
        if c["topk"]:
            out.update(ids=r.top_ids, top=r.top_log_probs.detach())
        if c["train"]:
            out["dz"], = torch.autograd.grad((r.log_probs, r.entropy), s["z"],
                                             (s["dlogp"], s["dent"]))
        return out
    norm = m.clip_grad_norm_(s["grads"], s["max_norm"])
    return _clip_outputs(s, norm)


def _scale_values(scale):
    """E8M0 bytes as the values that they stand for."""
    return scale.view(torch.float8_e8m0fnu) if scale.dtype == torch.uint8 else scale


def _clip_outputs(s, norm):
    """Many small gradients come joined."""
    g = s["grads"]
    return dict(norm=norm, grads=g if len(g) <= 8 else torch.cat(g))


def run(s):
    if own:
        return _run_own(s)
    with torch.no_grad():
        return {"block": _plain_block, "norm": _plain_norm, "logp": _plain_logp,
                "clip": _plain_clip}[s["case"]["kind"]](s)


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _quantised(b, dims):
    """The values that blocks keep in e4m3 under the scale amax / 448 of `dims`."""
    scale = (b.abs().amax(dim=dims, keepdim=True) / 448).clamp_min(2.0 ** -126)
    return (b / scale).to(E4M3).float() * scale


def _rows_of(x):
    """Values of x [M, K] in blocks of 1 x 128."""
    b = _padded(x.float(), 1)
    return _quantised(b.view(x.shape[0], -1, BLOCK), 2).view(b.shape)[:, :x.shape[1]]


def _tiles_of(w):
    """Values of w [N, K] in blocks of 128 x 128."""
    b = _padded(w.float(), 0, 1)
    v = _quantised(b.view(b.shape[0] // BLOCK, BLOCK, -1, BLOCK), (1, 3))
    return v.view(b.shape)[:w.shape[0], :w.shape[1]]


def _plain_block(s):
    c, n = s["case"], s["case"]["n"]
    x, w = s["x"], s["w"]
    y = torch.empty((x.shape[0], n), dtype=torch.bfloat16, device=DEV)
    if c["train"]:
        dx, dw = torch.empty_like(x), torch.empty_like(w)
    at = 0
    for e, size in enumerate(s["sizes"]):
        one = slice(at, at + size)
        at += size
        we = w[e] if c["experts"] else w
        if not c["train"]:
            if size == 0:
                continue
            scale = s["ws"][e] if c["experts"] else s["ws"]
            full = scale.repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :c["k"]]
            y[one] = (_rows_of(x[one]) @ (we.float() * full).t()).to(y.dtype)
            continue
        dwe = dw[e] if c["experts"] else dw
        if size == 0:
            dwe.zero_()
            continue
        we = _tiles_of(we)
        y[one] = (_rows_of(x[one]) @ we.t()).to(y.dtype)
        dx[one] = (_rows_of(s["dy"][one]) @ we).to(dx.dtype)
        dwe.copy_(_rows_of(s["dy"][one].t()) @ _rows_of(x[one].t()).t())
    return dict(y=y, dx=dx, dw=dw) if c["train"] else dict(y=y)


def _plain_norm(s):
    c = s["case"]
    h = (s["x"].float() + s["residual"].float()).to(s["x"].dtype)
    x = h.float()
    r = 1 / torch.sqrt((x * x).mean(dim=1, keepdim=True) + 1e-6)
    xhat = x * r
    y = xhat * s["w"]
    if c["out"] == "fp8_block":
        b = _padded(y, 1).view(y.shape[0], -1, BLOCK)
        scale = (b.abs().amax(dim=2, keepdim=True) / 448).clamp_min(2.0 ** -126)
        q = (b / scale).to(E4M3).view(y.shape[0], -1)[:, :y.shape[1]]
        return dict(q=q, scales=scale[:, :, 0], h=h)
    if c["out"] == "mxfp8":
        b = y.view(y.shape[0], -1, 32)
        amax = b.abs().amax(dim=2, keepdim=True)
        mant, exp = torch.frexp(amax)   # the least j with amax <= 448 * 2^j (448 = 0.875 * 2^9)
        j = torch.where(amax > 0, exp - 9 + (mant > 0.875), -127).clamp(-127, 127)
        q = torch.ldexp(b, -j.clamp_min(-126)).to(E4M3).view(y.shape)
        return dict(q=q, scales=(j + 127).to(torch.uint8)[:, :, 0].view(torch.float8_e8m0fnu), h=h)
    out = dict(y=y.to(h.dtype), h=h)
    if not c["train"]:
        return out
    dy = s["dy"].float()
    u = dy * s["w"]
    d = r * (u - xhat * (u * xhat).mean(dim=1, keepdim=True)) + s["dh"].float()
    d = d.to(h.dtype)
    return dict(out, dx=d, dresidual=d, dw=(dy * xhat).sum(dim=0))


def _plain_logp(s):
    c, target = s["case"], s["target"]
    t, k = target.numel(), c["topk"]
    z = s["z"].float() / c["temperature"]
    live = target >= 0
    at = torch.where(live, target, 0)[:, None]
    top = z.amax(dim=1, keepdim=True)
    d = z - top
    p = torch.exp(d)
    total = p.sum(dim=1, keepdim=True)
    logp = d.gather(1, at) - torch.log(total)
    p = p / total
    dead = d == NEG
    ent = torch.log(total) - (p * torch.where(dead, 0.0, d)).sum(dim=1, keepdim=True)
    out = dict(logp=torch.where(live, logp[:, 0], 0.0), entropy=torch.where(live, ent[:, 0], 0.0))
    if k:
        order = s["z"].float().sort(dim=1, descending=True, stable=True).indices[:, :k]
        best = d.gather(1, order) - torch.log(total)
        kept = live[:, None] & (best > NEG)
        out["ids"] = torch.where(kept, order, -1).to(torch.int32)
        out["top"] = torch.where(kept, best, NEG)
    if c["train"]:
        gl, gh = (s["dlogp"] * live)[:, None], (s["dent"] * live)[:, None]
        d = torch.where(dead, 0.0, d - torch.log(total) + ent)  # log p + H
        g = p * (-gl - gh * d)
        g.scatter_add_(1, at, gl)
        out["dz"] = (g / c["temperature"]).to(s["z"].dtype)
    return out


def _plain_clip(s):
    total = torch.stack([(g.float() * g.float()).sum() for g in s["grads"]]).sum()
    norm = torch.sqrt(total)
    coef = torch.clamp(s["max_norm"] / (norm + 1e-6), max=1.0)
    for g in s["grads"]:
        g.copy_(g.float() * coef)
    return _clip_outputs(s, norm)


# ---------------------------------------------------------------------------
# the same in 64 bits, from the definitions
# ---------------------------------------------------------------------------
def _kept(x, down):
    """What e4m3 blocks of `down` x 128 (from the first element on) keep of the
    2-D x: the scales are fp32, the payload is the rounding of the 64-bit quotient."""
    out = torch.empty(x.shape, dtype=torch.float64, device=DEV)
    for i in range(0, x.shape[1], BLOCK):
        part = x[:, i:i + BLOCK].double()
        amax = part.abs().amax(dim=1)
        if down > 1:
            amax = torch.stack([a.max() for a in amax.split(down)]).repeat_interleave(down)
            amax = amax[:x.shape[0]]
        scale = (amax.float() / 448).clamp_min(2.0 ** -126).double()[:, None]
        out[:, i:i + BLOCK] = (part / scale).to(E4M3).double() * scale
    return out


def _exact_block(s, c):
    n, k = c["n"], c["k"]
    x, w = s["x"].detach(), s["w"].detach().view(-1, n, k)
    y = torch.zeros((c["tokens"], n), dtype=torch.float64, device=DEV)
    dx, dw = torch.zeros_like(x, dtype=torch.float64), None
    if c["train"]:
        dw = torch.zeros(w.shape, dtype=torch.float64, device=DEV)
    ends = [sum(s["sizes"][:i + 1]) for i in range(len(s["sizes"]))]
    for e, (size, end) in enumerate(zip(s["sizes"], ends)):
        if size == 0:
            continue
        rows = slice(end - size, end)
        if c["train"]:
            we = _kept(w[e], BLOCK)
        else:
            we = w[e].double()
            ws = s["ws"].view(w.shape[0], -1, s["ws"].shape[-1])[e].double()
            for i in range(ws.shape[0]):
                for j in range(ws.shape[1]):
                    we[i * BLOCK:(i + 1) * BLOCK, j * BLOCK:(j + 1) * BLOCK] *= ws[i, j]
        y[rows] = torch.mm(_kept(x[rows], 1), we.t())
        if c["train"]:
            dx[rows] = torch.mm(_kept(s["dy"][rows], 1), we)
            dw[e] = torch.mm(_kept(s["dy"][rows].t(), 1), _kept(x[rows].t(), 1).t())
    if not c["train"]:
        return dict(y=y)
    return dict(y=y, dx=dx, dw=dw if c["experts"] else dw[0])


def _exact_norm(s, c):
    both = s["x"].detach().double() + s["residual"].detach().double()
    h = both.to(s["x"].dtype).double()     # the residual stream is kept in the input's type
    w = s["w"].detach().double()
    rms = (h.square().mean(dim=1, keepdim=True) + 1e-6).sqrt()
    y = h / rms * w
    rows, cols = h.shape
    if c["out"] == "fp8_block":
        q = torch.empty_like(y)
        scales = torch.empty((rows, (cols + BLOCK - 1) // BLOCK), dtype=torch.float64, device=DEV)
        for j in range(scales.shape[1]):
            part = y[:, j * BLOCK:(j + 1) * BLOCK]
            scales[:, j] = (part.abs().amax(dim=1) / 448).clamp_min(2.0 ** -126)
            q[:, j * BLOCK:(j + 1) * BLOCK] = (part / scales[:, j:j + 1]).to(E4M3).double()
        return dict(q=q, scales=scales, h=both)
    if c["out"] == "mxfp8":
        part = y.view(rows, -1, 32)
        amax = part.abs().amax(dim=2).clamp_min(2.0 ** -140)
        scales = torch.exp2(torch.ceil(torch.log2(amax / 448)).clamp(-127, 127))
        q = (part / scales.clamp_min(2.0 ** -126)[:, :, None]).to(E4M3).double().view(rows, cols)
        return dict(q=q, scales=scales, h=both)
    if not c["train"]:
        return dict(y=y, h=both)
    dy = s["dy"].double()
    u, xhat = dy * w, h / rms
    d = (u - xhat * (u * xhat).sum(dim=1, keepdim=True) / cols) / rms + s["dh"].double()
    return dict(y=y, h=both, dx=d, dresidual=d, dw=(dy * xhat).sum(dim=0))


def _exact_logp(s, c):
    z, target = s["z"].detach(), s["target"]
    t, k = target.numel(), c["topk"]
    got = dict(logp=torch.zeros(t, dtype=torch.float64, device=DEV),
               entropy=torch.zeros(t, dtype=torch.float64, device=DEV))
    if k:
        got["ids"] = torch.full((t, k), -1, dtype=torch.int32, device=DEV)
        got["top"] = torch.full((t, k), NEG, dtype=torch.float64, device=DEV)
    if c["train"]:
        got["dz"] = torch.zeros(z.shape, dtype=torch.float64, device=DEV)
    for i in range(0, t, 256):
        rows = torch.arange(i, min(t, i + 256), device=DEV)[target[i:i + 256] != -100]
        if rows.numel() == 0:
            continue
        lp = torch.log_softmax(z[rows].double() / c["temperature"], dim=1)
        p = lp.exp()
        fin = lp.masked_fill(lp == NEG, 0.0)
        ent = -(p * fin).sum(dim=1)
        here = torch.arange(rows.numel(), device=DEV)
        got["logp"][rows] = lp[here, target[rows]]
        got["entropy"][rows] = ent
        if k:
            order = torch.argsort(-z[rows].double(), dim=1, stable=True)[:, :k]
            best = lp.gather(1, order)
            got["ids"][rows] = torch.where(best > NEG, order, -1).int()
            got["top"][rows] = best
        if c["train"]:
            gl, gh = s["dlogp"][rows].double(), s["dent"][rows].double()
            one = torch.zeros_like(p)
            one[here, target[rows]] = 1.0
            g = gl[:, None] * (one - p) - gh[:, None] * p * (fin + ent[:, None])
            got["dz"][rows] = g / c["temperature"]
    return got


def _exact_clip(s, c):
    norm = math.sqrt(math.fsum(float(torch.linalg.vector_norm(g.double())) ** 2
                               for g in s["grads"]))
    coef = min(1.0, s["max_norm"] / (norm + 1e-6))
    grads = [g.double() * coef for g in s["grads"]]
    return dict(norm=torch.tensor(norm, dtype=torch.float64, device=DEV),
                grads=grads if len(grads) <= 8 else torch.cat(grads))


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"block": _exact_block, "norm": _exact_norm, "logp": _exact_logp,
                "clip": _exact_clip}[case["kind"]](s, case)
