"""Operators on tensors of more than 2^31 elements: the last rows get what a small
call on them gets (offsets that pass 32 bits); and operators captured in a HIP graph
and replayed several times with new inputs, eager work in between."""
import pytest
import torch

import mxfp8gg

pytestmark = pytest.mark.gpu


def _free():
    torch.cuda.synchronize()
    torch.cuda.empty_cache()


def test_norm(gpu):
    rows, cols = (1 << 18) + 300, 8200
    x = torch.empty((rows, cols), dtype=torch.bfloat16, device=gpu).normal_().requires_grad_(True)
    w = torch.randn(cols, device=gpu)
    y = mxfp8gg.rms_norm(x, w)
    dx, = torch.autograd.grad(y, x, x.detach())
    tail = x.detach()[-200:].clone().requires_grad_(True)
    z = mxfp8gg.rms_norm(tail, w)
    dz, = torch.autograd.grad(z, tail, tail.detach())
    assert x.numel() > 1 << 31
    assert torch.equal(y[-200:], z) and torch.equal(dx[-200:], dz)
    del x, y, dx
    _free()


def test_route_topk(gpu):
    T, E = (1 << 21) + 1000, 1024
    x = torch.empty((T, E), dtype=torch.bfloat16, device=gpu).normal_().requires_grad_(True)
    idx, w = mxfp8gg.route_topk(x, 4, renormalize=False)
    dx, = torch.autograd.grad(w, x, w.detach())
    tail = x.detach()[-100:].clone().requires_grad_(True)
    i, v = mxfp8gg.route_topk(tail, 4, renormalize=False)
    dv, = torch.autograd.grad(v, tail, v.detach())
    assert x.numel() > 1 << 31
    assert torch.equal(idx[-100:], i)
    # a row's softmax sum is shared out over other lanes in a small call
    assert torch.allclose(w[-100:], v, rtol=1e-5, atol=0)
    assert torch.allclose(dx[-100:].float(), dv.float(), rtol=1e-2, atol=1e-6)
    del x, idx, w, dx
    _free()


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw(gpu, bits):
    n = (1 << 31) + 32 * 1000 + 5
    p = torch.empty(n, dtype=torch.bfloat16, device=gpu).normal_()
    g = torch.empty(n, dtype=torch.bfloat16, device=gpu).normal_()
    states = [mxfp8gg.adamw_state(p, bits) for _ in range(2)]
    cut = n - 32 * 1000 - 5                       # a whole block of the states
    tail = [p[cut:].clone(), [mxfp8gg.adamw_state(p[cut:], bits) for _ in range(2)]]
    for step in (1, 2):
        mxfp8gg.adamw_step([p], [g], [states[0]], [states[1]], step=step)
        mxfp8gg.adamw_step([tail[0]], [g[cut:]], [tail[1][0]], [tail[1][1]], step=step)
    assert torch.equal(p[cut:], tail[0])
    for s, t in zip(states, tail[1]):
        s, t = (s, t) if bits == 8 else ((s,), (t,))
        assert torch.equal(s[0][cut:].view(torch.uint8), t[0].view(torch.uint8))
        if bits == 8:
            assert torch.equal(s[1][cut // 32:], t[1])
    del p, g, states
    _free()


def test_linear_cross_entropy(gpu):
    T, V, H = 70, (1 << 18) + 500, 8192
    x = torch.empty((T, H), dtype=torch.bfloat16, device=gpu).normal_().requires_grad_(True)
    w = torch.empty((V, H), dtype=torch.bfloat16, device=gpu).normal_(0, H ** -0.5)
    w.requires_grad_(True)
    t = torch.arange(T, device=gpu) + V - T       # the last words
    loss = mxfp8gg.linear_cross_entropy(x, w, t, reduction="sum")
    dx, dw = torch.autograd.grad(loss, (x, w))
    assert w.numel() > 1 << 31
    z = torch.cat([x.detach().float() @ c.float().t() for c in w.detach().split(1 << 16)], dim=1)
    p = z.softmax(dim=1)
    want = -torch.log_softmax(z, dim=1)[torch.arange(T), t].sum()
    assert abs(float(loss.detach()) - float(want)) <= 1e-4 * float(want)
    p[torch.arange(T), t] -= 1
    tail = p[:, -300:].t() @ x.detach().float()
    size = p[:, -300:].abs().t() @ x.detach().float().abs()
    assert ((dw[-300:].float() - tail).abs() <= 2 ** -7 * size).all()
    full = sum(p[:, i:i + (1 << 16)] @ w.detach()[i:i + (1 << 16)].float()
               for i in range(0, V, 1 << 16))
    assert ((dx.float() - full).abs() <= 2 ** -7 * full.abs() + 2 ** -7 * full.abs().mean()).all()
    del x, w, dw, z, p
    _free()


def test_captured_in_a_graph(gpu):
    """A routing decision, a norm, the loss with its gradients and an optimizer step
    in one graph, three replays with new inputs against the eager results."""
    T, H, V, E = 300, 256, 1500, 32
    g = torch.Generator(device=gpu).manual_seed(0)
    rand = lambda *s: torch.randn(s, generator=g, device=gpu)  # noqa: E731
    x = rand(T, H).bfloat16()
    router, head = rand(E, H).bfloat16() / 16, (rand(V, H) / 16).bfloat16()
    gamma = torch.ones(H, device=gpu)
    target = torch.randint(0, V, (T,), generator=g, device=gpu)
    param, m, v = rand(5000), torch.zeros(5000, device=gpu), torch.zeros(5000, device=gpu)
    grad = torch.zeros(5000, device=gpu)

    def step():
        xs, hd = x.detach().requires_grad_(True), head.detach().requires_grad_(True)
        y = mxfp8gg.layer_norm(xs, gamma)
        idx, w = mxfp8gg.route_topk(y @ router.t(), 4, score="sigmoid")
        loss = mxfp8gg.linear_cross_entropy(y * w.sum(dim=1, keepdim=True).bfloat16(), hd, target)
        dx, dh = torch.autograd.grad(loss, (xs, hd))
        mxfp8gg.adamw_step([param], [grad], [m], [v], step=3)
        return idx, w.detach(), loss.detach(), dx, dh

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(3):
        x.copy_(rand(T, H).bfloat16())
        grad.copy_(rand(5000))
        target.copy_(torch.randint(0, V, (T,), generator=g, device=gpu))
        state = [t.clone() for t in (param, m, v)]
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (*out, param, m, v)]
        for t, s in zip((param, m, v), state):
            t.copy_(s)
        want = [*step(), param, m, v]
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
