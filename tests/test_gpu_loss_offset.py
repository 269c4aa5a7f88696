"""linear_cross_entropy of tokens that are sure of their target, with logits that share
a large offset: z = offset, and offset + 16 at the target, all exact in fp32.  The loss
log(1 + (V - 1) exp(-16)) and p - 1 are about 1e-4 to 2e-3, far below the spacing of
fp32 numbers at the offset.

Bounds: a sum of exponentials near 1 is added up in fewer than 64 steps, each off by at
most 2^-24: 64 * 2^-24, and 2^-20 of the value for the exponentials and the logarithm.
A gradient is p - 1 rounded to bf16 twice (d, and the result), 2^-7 of it."""
import numpy as np
import pytest
import torch

import mxfp8gg

pytestmark = pytest.mark.gpu


# few tokens, small tiles, large tiles
@pytest.mark.parametrize("T,V", [(5, 1000), (60, 20000), (130, 1000), (300, 20000)])
@pytest.mark.parametrize("offset", [0.0, 96.0, 1000.0, -1000.0, 20480.0])
def test_sure_of_the_target(gpu, T, V, offset):
    H = (T + 8) // 8 * 8
    x, w = torch.zeros((T, H)), torch.zeros((V, H))
    t = (7 * torch.arange(T) + 3) % V
    x[:, 0], w[:, 0] = offset, 1.0
    x[torch.arange(T), 1 + torch.arange(T)] = 16.0
    w[t, 1 + torch.arange(T)] = 1.0
    assert H > T and len(set(t.tolist())) == T and float(torch.tensor(offset).bfloat16()) == offset
    x, w, t = (a.to(gpu) for a in (x.bfloat16(), w.bfloat16(), t))
    x.requires_grad_(True), w.requires_grad_(True)
    loss = mxfp8gg.linear_cross_entropy(x, w, t, reduction="none")
    rest = (V - 1) * np.exp(-16.0)
    want, d = np.log1p(rest), -rest / (1 + rest)
    got = loss.detach().cpu().double().numpy()
    assert (got >= 0).all()
    assert (np.abs(got - want) <= 64 * 2.0 ** -24 + 2.0 ** -20 * want).all(), got - want
    dx, dw = torch.autograd.grad(loss.sum(), (x, w))
    rows = torch.arange(T, device=gpu)
    bound = 64 * 2.0 ** -24 + 2.0 ** -7 * abs(d)
    assert (np.abs(dx[rows, 1 + rows].cpu().double().numpy() - d) <= bound).all()
    assert (np.abs(dw[t, 1 + rows].cpu().double().numpy() - 16 * d) <= 16 * bound).all()
