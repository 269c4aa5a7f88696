"""fp8_block_linear's Python form (the one that int64 or [E + 1] offs, a weight that is not
contiguous and rows off the 16-byte grid take) where no gradient is wanted: no cast for a
backward pass, no memory for one, and none of its limits."""
import pytest
import torch

import mxfp8gg
from mxfp8gg import _lib

pytestmark = pytest.mark.gpu


def _allocations(f):
    """(result, allocations, bytes allocated) of f, once it has run before."""
    f()
    stats = torch.cuda.memory_stats
    keys = ("allocation.all.allocated", "requested_bytes.all.allocated")
    before = [stats()[k] for k in keys]
    r = f()
    return (r, *(stats()[k] - b for k, b in zip(keys, before)))


def _rand(shape, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).bfloat16().cuda()


@pytest.mark.parametrize("what", ["int64", "leading 0", "transposed", "stride", "python"])
def test_no_work_for_a_backward_pass(gpu, monkeypatch, what):
    _lib.load()
    if what == "python":
        monkeypatch.setattr(_lib, "_native", None)
    x, w, offs = _rand((300, 144), 0), _rand((80, 144), 1), None
    if what in ("int64", "leading 0"):
        w = _rand((3, 80, 144), 1)
        offs = torch.tensor([0, 100, 100, 250], device=gpu)
        offs = offs[1:] if what == "int64" else offs.int()
    elif what == "transposed":
        w = _rand((144, 80), 1).t()
    elif what == "stride":
        x = _rand((300, 148), 0)[:, :144]

    def call():
        return mxfp8gg.fp8_block_linear(x, w, offs)
    want, calls, size = _allocations(call)
    assert not want.requires_grad
    x, w = x.detach().requires_grad_(True), torch.nn.Parameter(w)
    with torch.no_grad():
        got, more, bigger = _allocations(call)
        with torch.inference_mode():
            assert torch.equal(call(), want)
    assert not got.requires_grad and torch.equal(got, want)
    assert (more, bigger) == (calls, size)
    # and with gradients on, they are there
    y = call()
    assert torch.equal(y.detach(), want)
    y.backward(torch.ones_like(y))
    assert x.grad.shape == x.shape and w.grad.shape == w.shape
    assert bool(x.grad.any()) and bool(w.grad.any())


def test_the_function_without_the_flag(gpu):
    """FP8BlockLinear.apply(x, w, ends), as before."""
    x, w = _rand((40, 64), 0).requires_grad_(True), _rand((32, 64), 1).requires_grad_(True)
    mxfp8gg.FP8BlockLinear.apply(x, w, None).sum().backward()
    got = x.grad.clone(), w.grad.clone()
    x.grad = w.grad = None
    mxfp8gg.fp8_block_linear(x, w).sum().backward()
    assert torch.equal(got[0], x.grad) and torch.equal(got[1], w.grad)


def test_more_tokens_than_a_weight_gradient_takes(gpu, monkeypatch):
    """2^22 tokens bound the token-axis casts, which only a weight's gradient needs."""
    M = (1 << 22) + 128
    x = _rand((64, 16), 0).repeat(M // 64, 1)
    w = torch.nn.Parameter(_rand((16, 16), 1))
    _lib.load()
    monkeypatch.setattr(_lib, "_native", None)
    with torch.no_grad():
        y = mxfp8gg.fp8_block_linear(x, w)
    few = mxfp8gg.fp8_block_linear(x[:64], w.detach())
    assert torch.equal(y.view(-1, 64, 16), few.expand(M // 64, 64, 16))
