"""AdamW without a GPU: a step of nothing is one, weights in host memory are refused."""
import pytest
import torch

import mxfp8gg


def test_step_without_a_gpu():
    p = torch.nn.Parameter(torch.ones(8))
    opt = mxfp8gg.AdamW([p])
    assert opt.step(lambda: 3.0) == 3.0 and not opt.state.get(p)
    p.grad = torch.ones(8)
    with pytest.raises(ValueError):
        opt.step()
    assert (p == 1).all() and opt.state[p]["step"] == 0  # a refused step is none
