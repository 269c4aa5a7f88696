"""The example model runs the routing decision, the norms, the expert FFN, the
vocabulary loss and the optimizer together, in training and one token at a time."""
import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    path = Path(__file__).resolve().parent.parent / "examples" / "moe_language_model.py"
    spec = importlib.util.spec_from_file_location("moe_language_model", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.mark.parametrize("bits", [32, 8])
def test_training_learns_the_next_word(gpu, example, bits):
    model, losses, follow = example.train(steps=60, state_bits=bits, vocab=500, device=gpu)
    assert torch.isfinite(losses).all()
    # a random guess costs log(500) = 6.2
    assert losses[0] > 4.0 and losses[-5:].mean() < 1.0
    tokens = torch.arange(500, device=gpu)
    with torch.no_grad():
        each, experts = model.loss(tokens, follow, reduction="none")
    assert each.shape == (500,) and each.mean() < 1.0
    # decoded one token at a time, it follows the table
    start = torch.tensor(3, device=gpu)
    want, t = [], 3
    for _ in range(6):
        t = int(follow[t])
        want.append(t)
    assert model.generate(start, 6).tolist() == want


def test_every_parameter_gets_a_gradient(gpu, example):
    model = example.MoELanguageModel(vocab=300, device=gpu)
    tokens = torch.randint(0, 300, (256,), device=gpu)
    loss, experts = model.loss(tokens, (tokens * 7 + 1) % 300)
    loss.backward()
    for name, p in model.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all(), name
        assert p.grad.abs().max() > 0, name
    assert experts.shape == (256, 4)
