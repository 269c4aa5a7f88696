"""A one-layer MoE language model, trained and then asked, on mxfp8gg alone.

    token embedding -> rms_norm -> router -> route_topk -> moe_routed_ffn (MXFP8)
    -> residual -> layer_norm -> linear_cross_entropy;  AdamW with 8-bit states

The data is synthetic: sequences of a fixed permutation of the vocabulary, so the
next word is a function of the current one and the loss can go to zero.

    python examples/moe_language_model.py [--steps 60] [--state-bits 8]
"""
import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "mxfp8-grouped-gemm_amd"))

import mxfp8gg  # noqa: E402


class MoELanguageModel(torch.nn.Module):
    def __init__(self, vocab=1000, hidden=256, inter=256, experts=16, topk=4, groups=4,
                 device="cuda", seed=0):
        super().__init__()
        gen = torch.Generator(device=device).manual_seed(seed)

        def weight(*shape, scale=None, dtype=torch.bfloat16):
            w = torch.randn(shape, generator=gen, device=device)
            return torch.nn.Parameter((w * (scale or shape[-1] ** -0.5)).to(dtype))

        self.topk, self.groups = topk, groups
        self.embedding = weight(vocab, hidden, scale=1.0)
        self.norm_in = torch.nn.Parameter(torch.ones(hidden, device=device))
        self.router = weight(experts, hidden)
        self.w_gate_up = weight(experts, 2 * inter, hidden)
        self.w_down = weight(experts, hidden, inter)
        self.norm_out = torch.nn.Parameter(torch.ones(hidden, device=device))
        self.norm_out_bias = torch.nn.Parameter(torch.zeros(hidden, device=device))
        self.head = weight(vocab, hidden)
        # balance bias of the routing: moved after every step, not trained
        self.register_buffer("balance", torch.zeros(experts, device=device))
        self.cache = mxfp8gg.WeightCastCache()  # casts of unchanged expert weights

    def hidden(self, tokens):
        """(final hidden states [T, H], expert ids [T, topk]) of int64 tokens [T]."""
        x = self.embedding[tokens]
        y = mxfp8gg.rms_norm(x, self.norm_in)
        logits = torch.nn.functional.linear(y, self.router)
        experts, scores = mxfp8gg.route_topk(
            logits, self.topk, score="sigmoid", bias=self.balance, num_groups=self.groups,
            top_groups=max(1, self.groups // 2), group_best=2)
        x = x + mxfp8gg.moe_routed_ffn(y, experts, scores, self.w_gate_up, self.w_down,
                                       weight_cache=self.cache)
        return mxfp8gg.layer_norm(x, self.norm_out, self.norm_out_bias), experts

    def loss(self, tokens, targets, **options):
        x, experts = self.hidden(tokens)
        return mxfp8gg.linear_cross_entropy(x, self.head, targets, **options), experts

    @torch.no_grad()
    def rebalance(self, experts, rate=1e-3):
        """Raise the bias of experts with fewer tokens than the mean, lower the others'."""
        counts = mxfp8gg.route_plan(experts, self.balance.numel()).counts.float()
        self.balance += rate * torch.sign(counts.mean() - counts)

    @torch.no_grad()
    def generate(self, token, length):
        """Greedy continuation, one token at a time."""
        out = [token]
        for _ in range(length):
            x, _ = self.hidden(out[-1].view(1))
            out.append((x @ self.head.t()).argmax(dim=1)[0])
        return torch.stack(out[1:])


def train(steps=60, batch=512, state_bits=8, lr=1e-2, vocab=1000, device="cuda", report=None):
    """(model, losses, next-word table) after `steps` steps on random positions."""
    model = MoELanguageModel(vocab=vocab, device=device)
    follow = torch.randperm(vocab, generator=torch.Generator().manual_seed(1)).to(device)
    decay, rest = [], []
    for p in model.parameters():
        (decay if p.dim() > 1 else rest).append(p)
    opt = mxfp8gg.AdamW([dict(params=decay), dict(params=rest, weight_decay=0.0)], lr=lr,
                        state_bits=state_bits, master_weights=True)
    gen = torch.Generator(device=device).manual_seed(2)
    losses = []
    for step in range(steps):
        tokens = torch.randint(0, vocab, (batch,), generator=gen, device=device)
        targets = follow[tokens]
        targets[::16] = -100                      # words that are not to be learnt from
        loss, experts = model.loss(tokens, targets)
        opt.zero_grad()
        loss.backward()
        opt.step()
        model.rebalance(experts)
        losses.append(loss.detach())
        if report and step % report == 0:
            print(f"step {step:4d}  loss {float(loss.detach()):.3f}", flush=True)
    return model, torch.stack(losses), follow


def main():
    ap = argparse.ArgumentParser(description=__doc__,
                                 formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--state-bits", type=int, default=8, choices=(8, 32))
    a = ap.parse_args()
    model, losses, follow = train(a.steps, state_bits=a.state_bits, report=10)
    tokens = torch.arange(follow.numel(), device=follow.device)
    with torch.no_grad():
        each, _ = model.loss(tokens, follow, reduction="none")
    first = torch.tensor(7, device=follow.device)
    got = model.generate(first, 8)
    print(f"loss {float(losses[0]):.3f} -> {float(each.mean()):.3f} over the whole vocabulary; "
          f"from word 7: {got.tolist()}")


if __name__ == "__main__":
    main()
