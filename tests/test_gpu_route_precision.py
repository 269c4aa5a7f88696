"""route_topk where scores are close, saturated or taken on different paths."""
import pytest
import torch

import mxfp8gg

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("E,G,K", [(256, 8, 8), (32, 1, 8), (320, 8, 6), (1000, 1, 3), (24, 4, 4),
                                   (120, 3, 5)])
def test_softmax_scores_do_not_depend_on_the_batch(gpu, E, G, K, biased):
    """Scores that hold the row's whole sum, and choices that go by them: the same bits
    in a call that shares a token out over more lanes."""
    g = torch.Generator(device=gpu).manual_seed(E)
    T = 2_500_000 // E
    x = 1.5 * torch.randn((T, E), generator=g, device=gpu)
    bias = 0.01 * torch.randn(E, generator=g, device=gpu) if biased else None
    f = lambda z: mxfp8gg.route_topk(z, K, score="softmax", num_groups=G,  # noqa: E731
                                     top_groups=(G + 1) // 2, bias=bias, renormalize=False)
    idx, w = f(x)
    for a in (0, 777, T - 300):
        i, v = f(x[a:a + 300])
        assert torch.equal(i, idx[a:a + 300]) and torch.equal(v, w[a:a + 300])
