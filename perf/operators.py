"""The operators around the routed expert FFN, as measurable cases.

One training step of an MoE layer normalises its input, decides which experts
every token goes to, runs them, takes the loss over a vocabulary and updates
the weights; serving does the first two for a few tokens at a time.  The cases
are those operators: `norm` (layer norm and root-mean-square norm), `route`
(softmax or sigmoid scores, balance bias, groups, top-k, renormalised
weights), `loss` (softmax cross entropy of a linear layer, the logits never
kept) and `adamw` (one step over many tensors, states in 32 or in 8 bits).
Hidden size 7168, expert weights of 4096 x 7168 and 32 experts with top-8 are
the layer of this repository's benchmark; the other sizes are generic.

With `own` false, `run` computes the plain form: elementary torch operations
in 32 bits, rounded once at the end.
"""
import math
import sys
from pathlib import Path

import torch

own = False

DEV = "cuda"
NEG = float("-inf")


def _package():
    path = str(Path.cwd() / "mxfp8-grouped-gemm_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import mxfp8gg

    return mxfp8gg


def listed():
    return [
        # Serving: the router's decision for the one token of a decode step,
        # 256 experts in 8 groups.  Latency of one launch and its host path.
        dict(name="route_decode", kind="route", tokens=1, experts=256, topk=8, score="sigmoid",
             groups=8, top_groups=4, best=2, bias=True, renorm=True, dtype="float32", masked=False,
             train=False),
        # Training, the benchmark layer's routing: 16384 tokens x top-8 of 32
        # experts, bf16 logits (many ties), softmax; decision and gradient.
        dict(name="route_softmax", kind="route", tokens=16384, experts=32, topk=8, score="softmax",
             groups=1, top_groups=1, best=1, bias=False, renorm=True, dtype="bfloat16",
             masked=False, train=True),
        # Training with a balance bias and groups: a large batch over 256
        # experts; decision and gradient.
        dict(name="route_groups", kind="route", tokens=131072, experts=256, topk=8,
             score="sigmoid", groups=8, top_groups=4, best=2, bias=True, renorm=True,
             dtype="float32", masked=False, train=True),
        # Serving: the norm in front of the layer for 64 decoded tokens.
        dict(name="norm_decode", kind="norm", rows=64, cols=7168, center=False, affine=True,
             dtype="bfloat16", train=False),
        # Training: layer norm forward and backward, 16384 tokens of 7168.
        dict(name="norm_train", kind="norm", rows=16384, cols=7168, center=True, affine=True,
             dtype="bfloat16", train=True),
        # Training in fp32 with an odd width: rows that start at any element.
        dict(name="norm_odd", kind="norm", rows=5003, cols=1001, center=True, affine=True,
             dtype="float32", train=True),
        # The small tensors of a model (norm weights, biases, router): 64
        # tensors of odd sizes in fp32.  Launches, not bytes, set the time.
        dict(name="adamw_small", kind="adamw", tensors=64, largest=7169, param="float32",
             grad="float32", bits=32, master=False),
        # The gate+up weights of 8 experts in bf16 with fp32 states and an fp32
        # master copy, as a trainer of bf16 weights keeps them.
        dict(name="adamw_experts", kind="adamw", tensors=8, largest=4096 * 7168,
             param="bfloat16", grad="bfloat16", bits=32, master=True),
        # The same weights without a master copy and with 8-bit states.
        dict(name="adamw_experts_8bit", kind="adamw", tensors=8, largest=4096 * 7168,
             param="bfloat16", grad="bfloat16", bits=8, master=False),
        # Evaluation: the loss of every token of a short text, no gradient.
        dict(name="loss_eval", kind="loss", tokens=128, vocab=32000, hidden=1024, ignored=False,
             train=False),
        # Training with an odd vocabulary and ignored (prompt) tokens.
        dict(name="loss_odd", kind="loss", tokens=1000, vocab=50021, hidden=2048, ignored=True,
             train=True),
        # Training: 4096 tokens of the benchmark's hidden size, 131072 words.
        dict(name="loss_train", kind="loss", tokens=4096, vocab=131072, hidden=7168, ignored=False,
             train=True),
    ]


def _log(rng, lo, hi, step=1):
    """A multiple of `step` in [lo, hi], spread over the logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def draw(rng):
    """One more case of the listed kinds: sizes from the smallest to the largest
    listed ones, odd ones among them."""
    most = {k: max(_cost(c) for c in listed() if c["kind"] == k)
            for k in ("route", "norm", "adamw", "loss")}
    while True:
        kind = rng.choice(sorted(most))
        if kind == "route":
            # the two forms that models use: softmax scores, ranked without a
            # bias, and sigmoid scores with one
            score = rng.choice(["softmax", "sigmoid"])
            groups = rng.choice([1, 1, 2, 4, 8])
            per = rng.choice([2, 4, 5, 8, 12, 16, 20, 32, 48, 64, 128])
            c = dict(kind=kind, tokens=_log(rng, 1, 131072), experts=groups * per, topk=0,
                     score=score, groups=groups, top_groups=rng.randint((groups + 1) // 2, groups),
                     best=2 if score == "sigmoid" else 1, bias=score == "sigmoid",
                     renorm=rng.random() < 0.75, dtype=rng.choice(["float32", "bfloat16"]),
                     masked=rng.random() < 0.3, train=rng.random() < 0.6)
            c["topk"] = rng.randint(1, min(10, per * c["top_groups"]))
            if c["experts"] > 512:
                continue
        elif kind == "norm":
            c = dict(kind=kind, rows=_log(rng, 1, 65536),
                     cols=rng.choice([_log(rng, 64, 16384), _log(rng, 64, 16384, 64)]),
                     center=rng.random() < 0.5, affine=rng.random() < 0.8,
                     dtype=rng.choice(["float32", "bfloat16"]), train=rng.random() < 0.6)
        elif kind == "adamw":
            bits = rng.choice([32, 8])
            param = rng.choice(["float32", "bfloat16"])
            c = dict(kind=kind, tensors=_log(rng, 1, 100), largest=_log(rng, 100, 3e7),
                     param=param, grad=rng.choice([param, "float32"]), bits=bits,
                     master=param == "bfloat16" and rng.random() < 0.5)
        else:
            c = dict(kind=kind, tokens=_log(rng, 1, 4096),
                     vocab=rng.choice([_log(rng, 1000, 131072), _log(rng, 1024, 131072, 256)]),
                     hidden=_log(rng, 64, 7168, 8), ignored=rng.random() < 0.4,
                     train=rng.random() < 0.6)
        if _cost(c) <= most[kind]:
            return c


# ---------------------------------------------------------------------------
# sizes and work
# ---------------------------------------------------------------------------
def _cost(case):
    """Seconds a pass cannot go below at nominal rates (for comparing cases)."""
    w = work(case)
    return max(w["bytes"] / 8e12, w["flops"] / 2.5e15)


def _sizes(case):
    """Elements of every tensor of an optimizer step: the largest first, then
    odd fractions of it; equal ones where they are expert weights."""
    n, most = case["tensors"], case["largest"]
    if most % 4096 == 0:
        return [most] * n
    return [max(1, most * (n - i) // n - i % 7) for i in range(n)]


def _width(name):
    return {"float32": 4, "bfloat16": 2}[name]


def work(case):
    kind = case["kind"]
    if kind == "route":
        t, e, k, b = case["tokens"], case["experts"], case["topk"], _width(case["dtype"])
        fwd = t * e * b + t * k * 8 + (4 * e if case["bias"] else 0)
        # gradient: the logits, the ids and the scores' gradient read again
        bwd = 2 * t * e * b + t * k * 8 if case["train"] else 0
        return {"bytes": fwd + bwd, "flops": t * e * (12 if case["train"] else 8)}
    if kind == "norm":
        n, b = case["rows"] * case["cols"], _width(case["dtype"])
        w = 4 * case["cols"] * (2 if case["center"] else 1) if case["affine"] else 0
        moved = 2 * n * b + w + ((3 * n * b + 2 * w) if case["train"] else 0)
        return {"bytes": moved, "flops": n * (22 if case["train"] else 8)}
    if kind == "adamw":
        n = sum(_sizes(case))
        per = 2 * _width(case["param"]) + _width(case["grad"]) + (16 if case["bits"] == 32 else 4.125)
        if case["master"]:  # the copy is read and written, the weight only written
            per += 8 - _width(case["param"])
        return {"bytes": n * per, "flops": n * 16}
    t, v, h = case["tokens"], case["vocab"], case["hidden"]
    moved = 2 * h * (t + v) * (2 if case["train"] else 1) + 12 * t
    return {"bytes": moved, "flops": (6 if case["train"] else 2) * t * v * h}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _normal(gen, shape, scale=1.0, dtype=torch.float32, shift=0.0):
    return torch.empty(shape, dtype=dtype, device=DEV).normal_(shift, scale, generator=gen)


def _uniform(gen, shape):
    return torch.rand(shape, generator=gen, device=DEV)


def _prepare_route(gen, case):
    t, e = case["tokens"], case["experts"]
    # popular experts score higher for every token, as routers learn it
    lean = 0.5 * _normal(gen, (e,))
    logits = (_normal(gen, (t, e), 1.5) + lean).to(getattr(torch, case["dtype"]))
    if case["masked"]:  # experts that are switched off, and padding tokens
        logits[_uniform(gen, (t, e)) < 0.1] = NEG
        logits[_uniform(gen, (t,)) < 0.05] = NEG
    bias = -0.1 * lean + 0.01 * _normal(gen, (e,)) if case["bias"] else None
    return dict(logits=logits.requires_grad_(case["train"]), bias=bias,
                dscores=_normal(gen, (t, case["topk"]), 1e-2))


def _prepare_norm(gen, case):
    shape, dtype = (case["rows"], case["cols"]), getattr(torch, case["dtype"])
    s = dict(x=_normal(gen, shape, 1.7, dtype, 0.3), w=None, b=None)
    if case["affine"]:
        s["w"] = _normal(gen, (case["cols"],), 0.1, shift=1.0)
        if case["center"]:
            s["b"] = _normal(gen, (case["cols"],), 0.1)
    if case["train"]:
        s["dy"] = _normal(gen, shape, 1e-2, dtype)
        for name in ("x", "w", "b"):
            if s[name] is not None:
                s[name].requires_grad_(True)
    return s


def _prepare_adamw(gen, case):
    s = dict(params=[], grads=[], m=[], v=[], masters=[] if case["master"] else None)
    for n in _sizes(case):
        full = _normal(gen, (n,), 0.02)
        g = _normal(gen, (n,), 1e-4)
        m = 0.3 * g + _normal(gen, (n,), 3e-5)
        r = (g * g + 1e-9 * _uniform(gen, (n,))).sqrt() * (0.5 + _uniform(gen, (n,)))
        # a run that no token has reached yet has no gradient and no history
        a = n // 3
        for x in (g, m, r):
            x[a:a + n // 20] = 0
        s["params"].append(full.to(getattr(torch, case["param"])))
        s["grads"].append(g.to(getattr(torch, case["grad"])))
        if case["master"]:
            s["masters"].append(full)
        if case["bits"] == 32:
            s["m"].append(m)
            s["v"].append(r * r)
        else:
            s["m"].append(_pack(m))
            s["v"].append(_pack(r))
    s["hyper"] = dict(step=25, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01)
    return s


def _prepare_loss(gen, case):
    t, v, h = case["tokens"], case["vocab"], case["hidden"]
    x = _normal(gen, (t, h), 1.0, torch.bfloat16)
    w = _normal(gen, (v, h), 2.0 / math.sqrt(h), torch.bfloat16)
    # frequent words more often than rare ones
    target = (v ** _uniform(gen, (t,)) - 1).long().clamp_(0, v - 1)
    if case["ignored"]:
        target[1:][_uniform(gen, (t - 1,)) < 0.3] = -100
    return dict(x=x.requires_grad_(case["train"]), w=w.requires_grad_(case["train"]), target=target)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    make = {"route": _prepare_route, "norm": _prepare_norm, "adamw": _prepare_adamw,
            "loss": _prepare_loss}
    return dict(make[case["kind"]](gen, case), case=dict(case))


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def _options(c):
    return dict(score=c["score"], num_groups=c["groups"], top_groups=c["top_groups"],
                group_best=c["best"], renormalize=c["renorm"], scale=2.5)


def _run_own(s):
    m, c = _package(), s["case"]
    if c["kind"] == "route":
        idx, scores = m.route_topk(s["logits"], c["topk"], bias=s["bias"], **_options(c))
        if not c["train"]:
            return dict(idx=idx, scores=scores)
        dlogits, = torch.autograd.grad(scores, s["logits"], s["dscores"])
        return dict(idx=idx, scores=scores.detach(), dlogits=dlogits)
    if c["kind"] == "norm":
        y = m.layer_norm(s["x"], s["w"], s["b"]) if c["center"] else m.rms_norm(s["x"], s["w"])
        if not c["train"]:
            return dict(y=y)
        names = [n for n in ("x", "w", "b") if s[n] is not None]
        grads = torch.autograd.grad(y, [s[n] for n in names], s["dy"])
        return dict({"d" + n: g for n, g in zip(names, grads)}, y=y.detach())
    if c["kind"] == "adamw":
        m.adamw_step(s["params"], s["grads"], s["m"], s["v"], masters=s["masters"], **s["hyper"])
        return _adamw_outputs(s)
    if not c["train"]:
        return dict(loss=m.linear_cross_entropy(s["x"], s["w"], s["target"], reduction="none"))
    loss = m.linear_cross_entropy(s["x"], s["w"], s["target"])
    dx, dw = torch.autograd.grad(loss, (s["x"], s["w"]))
    return dict(loss=loss.detach(), dx=dx, dw=dw)


def _adamw_outputs(s):
    """The updated tensors; 8-bit states as the values that their payload and
    their block scales stand for.  Many small tensors come joined."""
    out = dict(params=s["params"], m=s["m"], v=s["v"], masters=s["masters"] or [])
    if s["case"]["bits"] == 8:
        for n in ("m", "v"):
            out[n] = [q for q, _ in s[n]]
            out[n + "_scales"] = [e.view(torch.float8_e8m0fnu) for _, e in s[n]]
    if len(s["params"]) <= 8:
        return out
    return {n: torch.cat([x.view(torch.uint8) for x in v]).view(v[0].dtype) if v else None
            for n, v in out.items()}


def run(s):
    if own:
        return _run_own(s)
    with torch.no_grad():
        return {"route": _plain_route, "norm": _plain_norm, "adamw": _plain_adamw,
                "loss": _plain_loss}[s["case"]["kind"]](s)


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _plain_route(s):
    c, logits = s["case"], s["logits"]
    t, e, k, g = logits.shape[0], c["experts"], c["topk"], c["groups"]
    x = logits.float()
    if c["score"] == "sigmoid":
        score = 1 / (1 + torch.exp(-x))
    else:
        top = x.amax(dim=1, keepdim=True)
        num = torch.exp(x - torch.where(top == NEG, 0.0, top))
        total = num.sum(dim=1, keepdim=True)
        score = num / torch.where(total > 0, total, 1.0)
    # ranked by score + bias; without a bias by the logit, which orders alike
    choice = x if s["bias"] is None else torch.where(x == NEG, NEG, score + s["bias"])
    if g > 1:
        # a group's worth is its best choice, or its two best scores (+ bias) together
        value = choice if c["best"] == 1 or s["bias"] is not None else torch.where(x == NEG, NEG, score)
        best = value.view(t, g, e // g).sort(dim=2, descending=True).values[:, :, :c["best"]]
        rank = torch.where(best[:, :, 0] == NEG, NEG, torch.where(best == NEG, 0.0, best).sum(dim=2))
        keep = rank.sort(dim=1, descending=True, stable=True).indices[:, :c["top_groups"]]
        kept = torch.zeros((t, g), dtype=torch.bool, device=DEV).scatter_(1, keep, True)
        choice = torch.where(kept.repeat_interleave(e // g, dim=1), choice, NEG)
    order = choice.sort(dim=1, descending=True, stable=True).indices[:, :k]
    live = choice.gather(1, order) != NEG
    sel = torch.where(live, score.gather(1, order), 0.0)
    total = sel.sum(dim=1, keepdim=True)
    norm = torch.where(total > 0, 2.5 / torch.where(total > 0, total, 1.0), 0.0)
    scores = sel * norm if c["renorm"] else 2.5 * sel
    out = dict(idx=torch.where(live, order, -1).to(torch.int32), scores=scores)
    if not c["train"]:
        return out
    d = s["dscores"] * live
    if c["renorm"]:
        d = norm * (d - (d * scores).sum(dim=1, keepdim=True) / 2.5)
    else:
        d = 2.5 * d
    grad = torch.zeros((t, e), device=DEV)
    if c["score"] == "sigmoid":
        grad.scatter_(1, order, d * sel * (1 - sel))
    else:
        grad.scatter_(1, order, d)
        grad = score * (grad - (d * sel).sum(dim=1, keepdim=True))
    return dict(out, dlogits=grad.to(logits.dtype))


def _plain_norm(s):
    c = s["case"]
    x = s["x"].float()
    xc = x - x.mean(dim=1, keepdim=True) if c["center"] else x
    r = 1 / torch.sqrt((xc * xc).mean(dim=1, keepdim=True) + (1e-5 if c["center"] else 1e-6))
    xhat = xc * r
    y = xhat if s["w"] is None else xhat * s["w"]
    y = y if s["b"] is None else y + s["b"]
    out = dict(y=y.to(s["x"].dtype))
    if not c["train"]:
        return out
    dy = s["dy"].float()
    if s["w"] is not None:
        out["dw"] = (dy * xhat).sum(dim=0)
    if s["b"] is not None:
        out["db"] = dy.sum(dim=0)
    dxhat = dy if s["w"] is None else dy * s["w"]
    d = dxhat - xhat * (dxhat * xhat).mean(dim=1, keepdim=True)
    if c["center"]:
        d = d - dxhat.mean(dim=1, keepdim=True)
    return dict(out, dx=(d * r).to(s["x"].dtype))


def _blocks(x):
    return torch.nn.functional.pad(x, (0, -x.numel() % 32)).view(-1, 32)


def _block_exponent(b):
    """Exponent j in [-126, 127] of the block scale 2^j: the least with
    amax <= 448 * 2^j (448 = 0.875 * 2^9)."""
    amax = b.abs().amax(dim=1, keepdim=True)
    mant, exp = torch.frexp(amax)
    return torch.where(amax > 0, exp - 9 + (mant > 0.875), -126).clamp(-126, 127)


def _pack(x):
    """8-bit state: e4m3 payload and one E8M0 byte for every 32 elements."""
    b = _blocks(x)
    j = _block_exponent(b)
    q = (b * torch.exp2(-j.to(b.dtype))).to(torch.float8_e4m3fn)
    return q.view(-1)[:x.numel()].contiguous(), (j + 127).to(torch.uint8).view(-1)


def _unpack(state, dtype=torch.float32):
    q, e = state
    up = torch.exp2(e.to(dtype) - 127)
    return q.to(dtype) * up.repeat_interleave(32)[:q.numel()]


def _adamw_math(p, g, m, root, v, h):
    """New (p, m, root, v): the second moment v, or its root where that is kept."""
    (b1, b2), lr = h["betas"], h["lr"]
    p = p * (1 - lr * h["weight_decay"])
    m = m * b1 + g * (1 - b1)
    v = (root * root if v is None else v) * b2 + (g * g) * (1 - b2)
    root = torch.sqrt(v)
    denom = root / math.sqrt(1 - b2 ** h["step"]) + h["eps"]
    return p - (lr / (1 - b1 ** h["step"])) * (m / denom), m, root, v


def _plain_adamw(s):
    small = s["case"]["bits"] == 8
    for i, p in enumerate(s["params"]):
        full = s["masters"][i] if s["masters"] else p.float()
        m = _unpack(s["m"][i]) if small else s["m"][i]
        root, v = (_unpack(s["v"][i]), None) if small else (None, s["v"][i])
        new, m, root, v = _adamw_math(full, s["grads"][i].float(), m, root, v, s["hyper"])
        p.copy_(new)
        if s["masters"]:
            full.copy_(new)
        if small:
            for old, x in ((s["m"][i], m), (s["v"][i], root)):
                for o, n in zip(old, _pack(x)):
                    o.copy_(n)
        else:
            s["m"][i].copy_(m)
            s["v"][i].copy_(v)
    return _adamw_outputs(s)


def _plain_loss(s):
    c, target = s["case"], s["target"]
    x, w = s["x"].float(), s["w"].float()
    z = x @ w.t()
    top = z.amax(dim=1, keepdim=True)
    z = z - top
    live = target >= 0
    at = torch.where(live, target, 0)[:, None]
    picked = z.gather(1, at)
    p = torch.exp(z)
    del z
    total = p.sum(dim=1, keepdim=True)
    loss = torch.where(live, (torch.log(total) - picked)[:, 0], 0.0)
    if not c["train"]:
        return dict(loss=loss)
    n = live.sum()
    p = p * (live[:, None] / (total * n))
    p.scatter_add_(1, at, -(live / n)[:, None])
    return dict(loss=loss.sum() / n, dx=(p @ w).to(torch.bfloat16),
                dw=(p.t() @ x).to(torch.bfloat16))


# ---------------------------------------------------------------------------
# the same in 64 bits, from the definitions
# ---------------------------------------------------------------------------
def _exact_route(s, c):
    z, k, e = s["logits"].detach().double(), c["topk"], c["experts"]
    dead = z == NEG
    if c["score"] == "sigmoid":
        prob = torch.sigmoid(z)
    else:
        prob = torch.where(dead.all(dim=1, keepdim=True), 0.0, z).softmax(dim=1)
        prob = torch.where(dead, 0.0, prob)
    rank = z if s["bias"] is None else prob + s["bias"].double()
    rank = rank.masked_fill(dead, NEG)
    if c["groups"] > 1:
        parts = prob.masked_fill(dead, NEG) if c["best"] == 2 and s["bias"] is None else rank
        parts = parts.reshape(z.shape[0], c["groups"], -1)
        best = parts.topk(c["best"], dim=2).values
        total = best.masked_fill(best == NEG, 0.0).sum(dim=2).masked_fill(best[..., 0] == NEG, NEG)
        # lowest group first among equal ones: as many groups beat it as rank before it
        a, b = total[:, :, None], total[:, None, :]
        i = torch.arange(c["groups"], device=DEV)
        before = (b > a) | ((b == a) & (i[None, :] < i[:, None]))
        out = (before.sum(dim=2) >= c["top_groups"]).repeat_interleave(e // c["groups"], dim=1)
        rank = rank.masked_fill(out, NEG)
    order = torch.argsort(-rank, dim=1, stable=True)[:, :k]
    live = rank.gather(1, order) > NEG
    picked = prob.gather(1, order) * live
    total = picked.sum(dim=1, keepdim=True)
    total = torch.where(total > 0, total, 1.0) if c["renorm"] else torch.ones_like(total)
    w = 2.5 * picked / total
    got = dict(idx=torch.where(live, order, -1).int(), scores=w)
    if not c["train"]:
        return got
    up = s["dscores"].double() * live
    dp = 2.5 * up / total
    if c["renorm"]:
        dp = dp - (dp * picked).sum(dim=1, keepdim=True) / total * live
    full = torch.zeros_like(prob)
    full.scatter_(1, order, dp)
    if c["score"] == "sigmoid":
        return dict(got, dlogits=full * prob * torch.sigmoid(-z))
    return dict(got, dlogits=prob * (full - (full * prob).sum(dim=1, keepdim=True)))


def _exact_norm(s, c):
    x = s["x"].detach().double()
    if c["center"]:
        mu = x.mean(dim=1, keepdim=True)
        sd = (x.var(dim=1, unbiased=False, keepdim=True) + 1e-5).sqrt()
    else:
        mu, sd = 0.0, (x.square().mean(dim=1, keepdim=True) + 1e-6).sqrt()
    z = (x - mu) / sd
    one = torch.ones(x.shape[1], dtype=torch.float64, device=DEV)
    w = one if s["w"] is None else s["w"].detach().double()
    b = 0 * one if s["b"] is None else s["b"].detach().double()
    got = dict(y=z * w + b)
    if not c["train"]:
        return got
    dy = s["dy"].double()
    if s["w"] is not None:
        got["dw"] = (dy * z).sum(dim=0)
    if s["b"] is not None:
        got["db"] = dy.sum(dim=0)
    u = dy * w
    dx = u - z * (u * z).sum(dim=1, keepdim=True) / x.shape[1]
    if c["center"]:
        dx -= u.sum(dim=1, keepdim=True) / x.shape[1]
    return dict(got, dx=dx / sd)


def _exact_adamw(s, c):
    h = s["hyper"]
    (b1, b2), t = h["betas"], h["step"]
    got = dict(params=[], m=[], v=[], masters=[], m_scales=[], v_scales=[])
    for i, p in enumerate(s["params"]):
        g = s["grads"][i].double()
        small = c["bits"] == 8
        m = _unpack(s["m"][i], torch.float64) if small else s["m"][i].double()
        v = _unpack(s["v"][i], torch.float64).square() if small else s["v"][i].double()
        w = (s["masters"][i] if c["master"] else p).double()
        m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
        rate = (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + h["eps"])
        w = w - h["lr"] * (rate + h["weight_decay"] * w)
        got["params"].append(w)
        if c["master"]:
            got["masters"].append(w)
        if not small:
            got["m"].append(m)
            got["v"].append(v)
            continue
        for name, x in (("m", m), ("v", v.sqrt())):
            blocks = torch.nn.functional.pad(x, (0, -x.numel() % 32)).reshape(-1, 32)
            amax = blocks.abs().amax(dim=1, keepdim=True).clamp_min(2.0 ** -140)
            scale = torch.exp2(torch.ceil(torch.log2(amax / 448)).clamp(-126, 127))
            # the payload is the format's rounding of the 64-bit quotient
            q = (blocks / scale).to(torch.float8_e4m3fn).double()
            got[name].append(q.reshape(-1)[:x.numel()])
            got[name + "_scales"].append(scale.reshape(-1))
    if not small:
        del got["m_scales"], got["v_scales"]
    if len(s["params"]) <= 8:
        return got
    return {n: torch.cat(x) if x else None for n, x in got.items()}


def _exact_loss(s, c):
    x, w = s["x"].detach().double(), s["w"].detach().double()
    t = s["target"]
    live = t != -100
    rows = torch.arange(t.numel(), device=DEV)[live]
    z = x @ w.t()
    lse = torch.logsumexp(z, dim=1)
    loss = torch.zeros_like(lse)
    loss[live] = lse[live] - z[rows, t[live]]
    if not c["train"]:
        return dict(loss=loss)
    z.sub_(lse[:, None]).exp_()
    z[rows, t[live]] -= 1
    z[~live] = 0
    z /= live.sum()
    return dict(loss=loss.sum() / live.sum(), dx=z @ w, dw=z.t() @ x)


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"route": _exact_route, "norm": _exact_norm, "adamw": _exact_adamw,
                "loss": _exact_loss}[case["kind"]](s, case)
