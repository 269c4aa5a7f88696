"""The norms with residual, the block-scaled products, the log probabilities and the
clipping in one run, as a policy is trained and served: each seam of a training step
against its formula in 64 bits, the served form against the trained one."""
import importlib.util
from pathlib import Path

import pytest
import torch

import mxfp8gg

pytestmark = pytest.mark.gpu
BF16 = 2.0 ** -8  # a rounding to bfloat16, relative


@pytest.fixture(scope="module")
def example():
    path = Path(__file__).resolve().parent.parent / "examples" / "policy_gradient.py"
    spec = importlib.util.spec_from_file_location("policy_gradient", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def test_the_example_runs(gpu, example):
    policy, rewards, norms = example.train(steps=6, batch=256, device=gpu)
    assert rewards.shape == norms.shape == (6,)
    assert torch.isfinite(norms).all() and (norms > 0).all()
    tokens = torch.arange(20, device=gpu)
    top = example.Server(policy)(tokens, tokens)
    assert top.top_ids.shape == (20, 4) and top.log_probs is None
    assert ((top.top_ids >= 0) & (top.top_ids < 512)).all()
    assert (top.top_log_probs[:, :-1] >= top.top_log_probs[:, 1:]).all()


def test_every_parameter_gets_a_gradient(gpu, example):
    policy = example.Policy(device=gpu)
    tokens = torch.arange(300, device=gpu)
    policy.loss(tokens, tokens % 64, (tokens * 7 + 1) % 512, torch.ones(300, device=gpu)).backward()
    for name, p in policy.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all(), name
        assert p.grad.abs().max() > 0, name


def _close(got, want, rounding, size=0.0):
    """Within `rounding` of the value itself, and of `size` (what the value is a sum of)."""
    err = (got.double() - want).abs()
    assert (err <= rounding * want.abs() + size + 1e-30).all(), float(
        (err / (rounding * want.abs() + size + 1e-30)).max())


@pytest.mark.parametrize("T", [1, 77, 300])
def test_seams_of_a_step(gpu, example, T):
    """The gradients that reach each seam, against the formulas applied to the seam before."""
    m = example.Policy(device=gpu)
    g = torch.Generator().manual_seed(T)
    tokens = torch.randint(0, 512, (T,), generator=g).to(gpu)
    actions = torch.randint(0, 512, (T,), generator=g).to(gpu)
    adv = torch.randn(T, generator=g).to(gpu)
    x, res = m.embedding[tokens], m.position[tokens % 64]
    y, h = mxfp8gg.add_rms_norm(x, res, m.norm_in)
    u = mxfp8gg.fp8_block_linear(y, m.up)
    gate, up = u.chunk(2, dim=-1)
    a = torch.nn.functional.silu(gate) * up
    o = mxfp8gg.fp8_block_linear(a, m.down)
    y2, h2 = mxfp8gg.add_rms_norm(o, h, m.norm_out)
    z = mxfp8gg.fp8_block_linear(y2, m.head)
    p = mxfp8gg.token_log_probs(z, actions)
    seams = (x, res, y, h, u, a, o, y2, z)
    for t in seams:
        t.retain_grad()
    (-(adv * p.log_probs + 0.01 * p.entropy).mean()).backward()

    # the loss: log p, entropy and their gradient
    lp = z.detach().double().log_softmax(1)
    pr = lp.exp()
    at = (torch.arange(T, device=gpu), actions)
    ent = -(pr * lp).sum(1)
    _close(p.log_probs.detach(), lp[at], 2.0 ** -20, 2.0 ** -18)
    _close(p.entropy.detach(), ent, 2.0 ** -20, 2.0 ** -18)
    one = torch.zeros_like(pr)
    one[at] = 1
    dz = -(adv.double()[:, None] * (one - pr) - 0.01 * pr * (lp + ent[:, None])) / T
    # the rounding to bf16; fp32's in the terms (each at most |adv| + 0.01 * 20, over T)
    _close(z.grad, dz, BF16 * 1.01, (float(adv.abs().max()) + 1) / T * 2.0 ** -18)

    # the products: the same casts and products called one by one
    for inp, w, out in ((y, m.up, u), (a, m.down, o), (y2, m.head, z)):
        wq, ws, wt, wts = mxfp8gg.to_fp8_block_weight(w.detach(), dual=True)
        q, s = mxfp8gg.to_fp8_block_dim0(inp.detach())
        assert torch.equal(mxfp8gg.fp8_block_mm(q, s, wq, ws), out.detach())
        q, s = mxfp8gg.to_fp8_block_dim0(out.grad)
        assert torch.equal(mxfp8gg.fp8_block_mm(q, s, wt, wts), inp.grad)
        gt, it = (mxfp8gg.to_fp8_block_dim1(t.detach()) for t in (out.grad, inp))
        assert torch.equal(mxfp8gg.fp8_block_wgrad(*gt[:2], *it[:2], out_dtype=torch.bfloat16),
                           w.grad)

    # the norms: h of both terms, and the stream's gradient joined with the norm's
    for xi, ri, w, yi, hi, dh in ((x, res, m.norm_in, y, h, None), (o, h, m.norm_out, y2, h2, 0)):
        hd = (xi.detach().float() + ri.detach().float()).bfloat16()
        assert torch.equal(hi.detach(), hd)
        hd, wd = hd.double(), w.detach().double()
        r = 1 / (hd.square().mean(1, keepdim=True) + 1e-6).sqrt()
        # three fp32 roundings, and a sum of 256 squares of one sign, before bf16's
        _close(yi.detach(), hd * r * wd, BF16 * 1.001)
        dy = yi.grad.double() * wd
        dx = r * (dy - hd * r * (dy * hd * r).mean(1, keepdim=True))
        if dh is None:
            dx = dx + hi.grad.double()
        # sums of 256 terms in fp32 against the size of their terms
        size = (r * (dy.abs() + (hd * r).abs() * (dy * hd * r).abs().mean(1, keepdim=True))
                + (hi.grad.double().abs() if dh is None else 0)) * 2.0 ** -18
        _close(xi.grad, dx, BF16 * 1.001, size)
        dw = yi.grad.double() * hd * r
        _close(w.grad, dw.sum(0), 0.0, dw.abs().sum(0) * 2.0 ** -16 + 2.0 ** -40)
    assert torch.equal(o.grad, h.grad)  # one gradient for both terms of the second sum

    # the clipping of what the step left
    grads = [t.grad for t in m.parameters()]
    want = torch.stack([t.double().square().sum() for t in grads]).sum().sqrt()
    before = [t.clone() for t in grads]
    opt = mxfp8gg.AdamW(m.parameters(), lr=1e-3)
    norm = opt.clip_grad_norm_(float(want) / 3)
    _close(norm, want, 2.0 ** -22)
    for t, b in zip(grads, before):
        _close(t, b.double() * (want / 3 / (want + 1e-6)), (BF16 if t.dtype == torch.bfloat16 else 2.0 ** -24) + 2.0 ** -18)
    opt.step()
    assert all(torch.isfinite(t).all() for t in m.parameters())


@pytest.mark.parametrize("T", [1, 16, 17, 300])
def test_served_as_trained(gpu, example, T):
    """The served policy differs from the trained one by where values are rounded: its
    norms' results go to e4m3 from fp32, the trained ones' from bf16.  A product's operand
    is then another by one e4m3 step where the quotient lies within bf16's rounding of a
    border: at most 2^-3 of the value, for 2^-8 / 2^-4 = 1/16 of the values.  In the root
    of the mean square that is 2^-3 * (1/16)^0.5 = 2^-5 of a product's result each, and
    three products follow one another, the last one with both errors of its inputs: 4 of
    2^-5 of the logits' root mean square, 6 times that for the largest."""
    m = example.Policy(device=gpu)
    tokens = torch.arange(T, device=gpu) * 5 % 512
    with torch.no_grad():
        z = m.logits(tokens, tokens % 64).float()
        want = mxfp8gg.token_log_probs(z, topk=4)
        got = example.Server(m)(tokens, tokens % 64)
    bound = 6 * 4 * 2.0 ** -5 * float(z.square().mean().sqrt())
    assert (got.top_log_probs - want.top_log_probs).abs().max() <= 2 * bound
    assert torch.isfinite(got.entropy).all() and (got.entropy >= 0).all()
