"""AdamW.step in a captured graph: the step number and the learning rate are arguments
of the launch, so every replay would repeat the captured ones.  It is refused, and the
optimizer is as before."""
import pytest
import torch

import mxfp8gg

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [32, 8])
def test_step_is_refused_under_capture(gpu, bits):
    p = torch.nn.Parameter(torch.randn(1000, device=gpu))
    p.grad = torch.ones_like(p)
    opt = mxfp8gg.AdamW([p], lr=0.1, state_bits=bits)
    opt.step()
    before, version = p.detach().clone(), p._version
    x = torch.zeros(8, device=gpu)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x += 1
        with pytest.raises(RuntimeError, match="capture"):
            opt.step()
    graph.replay()
    torch.cuda.synchronize()
    assert (x == 1).all()
    assert torch.equal(p, before) and p._version == version and opt.state[p]["step"] == 1
    opt.step()
    assert opt.state[p]["step"] == 2 and not torch.equal(p, before)
