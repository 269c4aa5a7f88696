"""The served policy of examples/policy_gradient.py, call by call: what each operator was
given is what the one before it returned (or the policy's own tensors), and what it
returned is its formula in 64 bits.  The same check on the CPU, with stand-ins for the
operators, has to find planted mistakes in the chain.

Tolerances.  A payload is the rounding of a quotient, 2^-4 of the value or half of e4m3's
smallest step, 2^-10 of the scale; the fp32 scale, quotient and norm before it are off by
less than 2^-16.  A product's bound is that of tests/test_gpu_block.py (7 * 2^-13 of the sum
of magnitudes in the matrix instruction, 2^-23 for each fp32 sum) and bf16's half step,
2^-8.  silu(gate) * up is rounded twice to bf16.  Log probabilities are fp32 sums of a few
hundred terms: 2^-20 of the value and 2^-18."""
import importlib.util
from pathlib import Path

import pytest
import torch

import mxfp8gg

FP8 = torch.float8_e4m3fn
BF16 = 2.0 ** -8
EPS = 1e-6


@pytest.fixture
def example():
    path = Path(__file__).resolve().parent.parent / "examples" / "policy_gradient.py"
    spec = importlib.util.spec_from_file_location("policy_gradient_served", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def _wide(q, s, rows):
    """Values of a payload under scales of `rows` x 128, in 64 bits."""
    s = s.double().repeat_interleave(128, 1)[:, :q.shape[1]]
    return q.double() * (s.repeat_interleave(rows, 0)[:q.shape[0]] if rows > 1 else s)


def _same(a, b):
    return a.dtype == b.dtype and a.shape == b.shape and torch.equal(a, b)


def _near(got, want, bound, what):
    assert got.shape == want.shape, what
    err = (got.double() - want).abs()
    assert bool((err <= bound).all()), (what, float((err - bound).max()))


def _cast(q, s, want, rows, what):
    """q and s hold `want`, each within its rounding."""
    assert q.dtype is FP8 and s.dtype is torch.float32, what
    step = s.double().repeat_interleave(128, 1)[:, :q.shape[1]]
    if rows > 1:
        step = step.repeat_interleave(rows, 0)[:q.shape[0]]
    _near(_wide(q, s, rows), want, (2.0 ** -4 + 2.0 ** -16) * want.abs() + 2.0 ** -10 * step, what)


def _product(y, q, s, wq, ws, what):
    a, w = _wide(q, s, 1), _wide(wq, ws, 128)
    want, size = a @ w.t(), a.abs() @ w.abs().t()
    bound = (7 * 2.0 ** -13 + (16 + s.shape[1] + 4) * 2.0 ** -23) * size
    _near(y, want, bound + BF16 * (want.abs() + bound), what)


def _norm(call, x, weight, residual, what):
    """The call took these, and its results are theirs; (payload, scales, sum)."""
    (gx, gw, gr), kw, (q, s, h) = call
    assert _same(gx, x) and gw is weight and _same(gr, residual), what
    assert kw == dict(out_format="fp8_block"), what
    total = (x.float() + residual.float()).bfloat16()
    assert _same(h, total), what
    t = total.double()
    _cast(q, s, t / (t.square().mean(1, keepdim=True) + EPS).sqrt() * weight.double(), 1, what)
    return q, s, h


def _check(calls, policy, tokens, at, topk, result):
    """Every seam of one served step; calls: (name, args, kwargs, result) in their order."""
    names = [c[0] for c in calls]
    assert names == ["to_fp8_block_weight"] * 3 + [
        "rms_norm_quant", "fp8_block_mm", "to_fp8_block_dim0", "fp8_block_mm", "rms_norm_quant",
        "fp8_block_mm", "token_log_probs"]
    calls = [c[1:] for c in calls]
    weights = []
    for call, w in zip(calls, (policy.up, policy.down, policy.head)):
        assert call[0][0] is w
        _cast(*call[2], w.detach().double(), 128, "weight")
        weights.append(call[2])

    def product(call, q, s, w, what):
        assert len(call[0]) == 4 and all(a is b for a, b in zip(call[0], (q, s, *w))), what
        _product(call[2], q, s, *w, what)
        return call[2]
    q, s, h = _norm(calls[3], policy.embedding[tokens], policy.norm_in, policy.position[at], "norm in")
    gate, up = (t.double() for t in product(calls[4], q, s, weights[0], "up").chunk(2, dim=-1))
    (a,), _, (q, s) = calls[5]
    want = gate / (1 + torch.exp(-gate)) * up
    _near(a, want, 2.02 * BF16 * want.abs() + 2.0 ** -130, "silu(gate) * up")
    _cast(q, s, a.double(), 1, "cast")
    out = product(calls[6], q, s, weights[1], "down")
    q, s, _ = _norm(calls[7], out, policy.norm_out, h, "norm out")
    logits = product(calls[8], q, s, weights[2], "head")
    (z,), kw, r = calls[9]
    assert z is logits and kw == dict(topk=topk) and r is result
    lp = z.double().log_softmax(1)
    order = z.float().sort(dim=1, descending=True, stable=True).indices[:, :topk]
    assert torch.equal(r.top_ids.long(), order) and r.log_probs is None
    top = lp.gather(1, order)
    _near(r.top_log_probs, top, 2.0 ** -20 * top.abs() + 2.0 ** -18, "top")
    ent = -(lp.exp() * lp).sum(1)
    _near(r.entropy, ent, 2.0 ** -20 * ent.abs() + 2.0 ** -18, "entropy")


NAMES = ("to_fp8_block_weight", "to_fp8_block_dim0", "rms_norm_quant", "fp8_block_mm",
         "token_log_probs")


def _record(monkeypatch, operators):
    """Calls of mxfp8gg's operators, which `operators` carry out, as they come."""
    calls = []

    def wrap(name):
        def call(*args, **kw):
            r = operators[name](*args, **kw)
            calls.append((name, args, kw, r))
            return r
        return call
    for name in NAMES:
        monkeypatch.setattr(mxfp8gg, name, wrap(name))
    return calls


@pytest.mark.gpu
@pytest.mark.parametrize("trained", [False, True])
@pytest.mark.parametrize("T", [1, 16, 17, 300])
def test_every_call_of_a_served_step(gpu, monkeypatch, example, T, trained):
    policy = example.train(steps=3, batch=256, device=gpu)[0] if trained else example.Policy(device=gpu)
    tokens = torch.arange(T, device=gpu) * 5 % 512
    calls = _record(monkeypatch, {n: getattr(mxfp8gg, n) for n in NAMES})
    result = example.Server(policy)(tokens, tokens % 64, topk=5)
    with torch.no_grad():
        _check(calls, policy, tokens, tokens % 64, 5, result)


# ---------------------------------------------------------------------------
# planted mistakes, on the CPU
# ---------------------------------------------------------------------------
def _blocks(x, rows):
    """(payload, scales) of x in blocks of rows x 128."""
    M, K = x.shape
    pad = torch.zeros(((M + rows - 1) // rows * rows, (K + 127) // 128 * 128))
    pad[:M, :K] = x
    b = pad.view(pad.shape[0] // rows, rows, -1, 128)
    s = (b.abs().amax(dim=(1, 3), keepdim=True) / 448).clamp_min(2.0 ** -126)
    return (b / s).to(FP8).view(pad.shape)[:M, :K], s[:, 0, :, 0]


def _plain_norm(x, weight, residual, out_format):
    h = (x.float() + residual.float()).bfloat16()
    f = h.float()
    return (*_blocks(f / (f.square().mean(1, keepdim=True) + EPS).sqrt() * weight, 1), h)


def _plain_log_probs(z, topk):
    lp = z.float().log_softmax(1)
    ids = z.float().sort(dim=1, descending=True, stable=True).indices[:, :topk]
    return mxfp8gg.TokenLogProbs(None, -(lp.exp() * lp).sum(1), ids.int(), lp.gather(1, ids))


PLAIN = {
    "to_fp8_block_weight": lambda w: _blocks(w.float(), 128),
    "to_fp8_block_dim0": lambda x: _blocks(x.float(), 1),
    "rms_norm_quant": _plain_norm,
    "fp8_block_mm": lambda q, s, wq, ws: (_wide(q, s, 1) @ _wide(wq, ws, 128).t()).bfloat16(),
    "token_log_probs": _plain_log_probs,
}


def _served(server, tokens, at, topk, wrong):
    """The server's step with one mistake in it (none for ""), written as the example's."""
    m, (up, down, head) = server.policy, (server.up, server.down, server.head)
    if wrong == "weights of another layer":
        head = (head[0].flip(0).clone(), head[1])
    if wrong == "next token":
        tokens = tokens + 1
    if wrong == "next position":
        at = at + 1
    position = m.position[at] * (wrong != "no position")
    norm_in, norm_out = (m.norm_out, m.norm_in) if wrong == "norms swapped" else (m.norm_in, m.norm_out)
    q, s, h = mxfp8gg.rms_norm_quant(m.embedding[tokens], norm_in, position, out_format="fp8_block")
    gate, up = mxfp8gg.fp8_block_mm(q, s, *up).chunk(2, dim=-1)
    if wrong == "gate and up swapped":
        gate, up = up, gate
    act = torch.sigmoid(gate) if wrong == "sigmoid" else torch.nn.functional.silu(gate)
    q, s = mxfp8gg.to_fp8_block_dim0(act * up * (wrong != "no inner product"))
    out = mxfp8gg.fp8_block_mm(q, s, *down)
    if wrong == "sum of the embedding":
        h = m.embedding[tokens].clone()
    if wrong == "no residual":
        h = torch.zeros_like(h)
    q, s, _ = mxfp8gg.rms_norm_quant(out, norm_out, h, out_format="fp8_block")
    z = mxfp8gg.fp8_block_mm(q, s, *head)
    if wrong == "logits of another row":
        z = z.roll(1, 0)
    return mxfp8gg.token_log_probs(z, topk=topk)


MISTAKES = ["weights of another layer", "next token", "next position", "no position", "norms swapped",
            "gate and up swapped", "sigmoid", "no inner product", "sum of the embedding", "no residual",
            "logits of another row"]


@pytest.mark.parametrize("wrong", ["example", "", *MISTAKES, "casts", "a product", "the norm",
                                   "the likeliest"])
def test_planted_mistakes_are_found(monkeypatch, example, wrong):
    operators = dict(PLAIN)
    if wrong == "casts":  # one payload byte two steps off
        def cast(x):
            q, s = _blocks(x.float(), 1)
            q = q.clone()
            q.view(torch.uint8)[2, 5] ^= 2
            return q, s
        operators["to_fp8_block_dim0"] = cast
    if wrong == "a product":  # the last sixteen of the contraction left out
        operators["fp8_block_mm"] = lambda q, s, wq, ws: (
            _wide(q, s, 1)[:, :-16] @ _wide(wq, ws, 128)[:, :-16].t()).bfloat16()
    if wrong == "the norm":  # without the mean
        def norm(x, weight, residual, out_format):
            h = (x.float() + residual.float()).bfloat16()
            return (*_blocks(h.float() / h.float().norm(dim=1, keepdim=True) * weight, 1), h)
        operators["rms_norm_quant"] = norm
    if wrong == "the likeliest":
        def top(z, topk):
            r = _plain_log_probs(z, topk)
            return r._replace(top_ids=r.top_ids.roll(1, 1))
        operators["token_log_probs"] = top
    policy = example.Policy(vocab=96, hidden=160, inter=144, positions=32, device="cpu")
    tokens = torch.arange(7) * 11 % 90
    calls = _record(monkeypatch, operators)
    server = example.Server(policy)
    with torch.no_grad():
        if wrong == "example":
            result = server(tokens, tokens % 30)
        else:
            result = _served(server, tokens, tokens % 30, 4, wrong)
        if wrong in ("", "example"):
            _check(calls, policy, tokens, tokens % 30, 4, result)
        else:
            with pytest.raises(AssertionError):
                _check(calls, policy, tokens, tokens % 30, 4, result)
