"""token_log_probs for rows that one workgroup takes whole and rows shared out over
several, with few and with many alternatives: against 64 bits, where parts of a row hold
nothing, fewer logits than alternatives are left, or all are equal."""
import pytest
import torch

import mxfp8gg
from test_gpu_logprob import NEG, _check, _logits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("topk", [1, 32, 33, 64])
@pytest.mark.parametrize("T,V", [(1, 65536), (2, 65544), (3, 100003), (130, 90001), (300, 70000),
                                 (7, 300007)])
def test_shares(gpu, topk, T, V):
    z, t = _logits(gpu, T, V, torch.bfloat16, seed=3)
    _check(z, t, topk=topk, grads=False)


@pytest.mark.parametrize("topk", [8, 32, 40, 64])
@pytest.mark.parametrize("V", [3000, 100000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_parts_of_nothing(gpu, topk, V, dtype):
    z, t = _logits(gpu, 6, V, dtype, seed=4)
    z[0, 30:] = NEG                  # the first part alone, fewer than some topk
    z[1, :-30] = NEG                 # the last
    z[2, ::2] = NEG
    z[3] = NEG
    z[4] = 0.25                      # all equal
    z[5, 100:2000] = 9.0             # more equal ones at the top than alternatives
    t[1] = V - 1
    _check(z, t, topk=topk)


@pytest.mark.parametrize("topk", [8, 40])
@pytest.mark.parametrize("V", [3000, 100000])
def test_non_finite(gpu, topk, V):
    z, t = _logits(gpu, 4, V, torch.float32, seed=5)
    z[0, V - 7] = float("nan")
    z[1, 11] = float("inf")
    z[2] = float("nan")
    r = mxfp8gg.token_log_probs(z, t, topk=topk)
    for i in range(3):
        assert torch.isnan(r.entropy[i]) and torch.isnan(r.top_log_probs[i]).all()
        assert (r.top_ids[i] == -1).all()
    _check(z[3:], t[3:], topk=topk)
