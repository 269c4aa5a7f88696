"""A policy over a vocabulary trained by its own rewards and then served, on mxfp8gg.

    token embedding + position -> add_rms_norm -> fp8_block_linear, SwiGLU, fp8_block_linear
    -> add_rms_norm -> fp8_block_linear (head) -> token_log_probs
    training: -(advantage * log_prob + entropy bonus), AdamW.clip_grad_norm_, AdamW
    serving:  the weights cast once, rms_norm_quant -> fp8_block_mm, the likeliest words

The reward is synthetic: 1 where the word chosen after a word is the one of a fixed table.

    python examples/policy_gradient.py [--steps 50]
"""
import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "mxfp8-grouped-gemm_amd"))

import mxfp8gg  # noqa: E402


class Policy(torch.nn.Module):
    def __init__(self, vocab=512, hidden=256, inter=384, positions=64, device="cuda", seed=0):
        super().__init__()
        gen = torch.Generator(device=device).manual_seed(seed)

        def weight(*shape, scale=None):
            w = torch.randn(shape, generator=gen, device=device)
            return torch.nn.Parameter((w * (scale or shape[-1] ** -0.5)).bfloat16())

        self.embedding = weight(vocab, hidden, scale=1.0)
        self.position = weight(positions, hidden, scale=0.1)
        self.norm_in = torch.nn.Parameter(torch.ones(hidden, device=device))
        self.up = weight(2 * inter, hidden)
        self.down = weight(hidden, inter)
        self.norm_out = torch.nn.Parameter(torch.ones(hidden, device=device))
        self.head = weight(vocab, hidden)

    def logits(self, tokens, at):
        """bf16 [..., vocab] for int64 tokens and positions of one shape."""
        y, h = mxfp8gg.add_rms_norm(self.embedding[tokens], self.position[at], self.norm_in)
        gate, up = mxfp8gg.fp8_block_linear(y, self.up).chunk(2, dim=-1)
        out = mxfp8gg.fp8_block_linear(torch.nn.functional.silu(gate) * up, self.down)
        y, _ = mxfp8gg.add_rms_norm(out, h, self.norm_out)
        return mxfp8gg.fp8_block_linear(y, self.head)

    def loss(self, tokens, at, actions, advantage, bonus=0.01):
        p = mxfp8gg.token_log_probs(self.logits(tokens, at), actions)
        return -(advantage * p.log_probs + bonus * p.entropy).mean()


class Server:
    """The policy with its weights cast once, for decoding."""

    def __init__(self, policy):
        self.policy = policy
        with torch.no_grad():
            self.up, self.down, self.head = (mxfp8gg.to_fp8_block_weight(w)
                                             for w in (policy.up, policy.down, policy.head))

    @torch.no_grad()
    def __call__(self, tokens, at, topk=4):
        """TokenLogProbs of the next word for int64 tokens and positions [T]."""
        m = self.policy
        q, s, h = mxfp8gg.rms_norm_quant(m.embedding[tokens], m.norm_in, m.position[at],
                                         out_format="fp8_block")
        gate, up = mxfp8gg.fp8_block_mm(q, s, *self.up).chunk(2, dim=-1)
        q, s = mxfp8gg.to_fp8_block_dim0(torch.nn.functional.silu(gate) * up)
        q, s, _ = mxfp8gg.rms_norm_quant(mxfp8gg.fp8_block_mm(q, s, *self.down), m.norm_out, h,
                                         out_format="fp8_block")
        return mxfp8gg.token_log_probs(mxfp8gg.fp8_block_mm(q, s, *self.head), topk=topk)


def train(steps=50, batch=2048, vocab=512, lr=3e-3, device="cuda", report=None):
    """(policy, mean reward of each step, gradient norm of each step)."""
    policy = Policy(vocab=vocab, device=device)
    table = torch.randperm(vocab, generator=torch.Generator().manual_seed(1)).to(device)
    opt = mxfp8gg.AdamW(policy.parameters(), lr=lr, weight_decay=0.0, master_weights=True)
    gen = torch.Generator(device=device).manual_seed(2)
    rewards, norms = [], []
    for step in range(steps):
        tokens = torch.randint(0, vocab, (batch,), generator=gen, device=device)
        at = torch.randint(0, 64, (batch,), generator=gen, device=device)
        with torch.no_grad():
            p = torch.softmax(policy.logits(tokens, at).float(), dim=-1)
            actions = torch.multinomial(p, 1, generator=gen)[:, 0]
            # half of the words are shown the right answer
            actions[::2] = table[tokens[::2]]
            reward = (actions == table[tokens]).float()
        loss = policy.loss(tokens, at, actions, reward - reward[1::2].mean())
        opt.zero_grad()
        loss.backward()
        norms.append(opt.clip_grad_norm_(1.0))
        opt.step()
        rewards.append(reward[1::2].mean())
        if report and step % report == 0:
            print(f"step {step:4d}  reward {float(rewards[-1]):.3f}  "
                  f"gradient {float(norms[-1]):.3f}", flush=True)
    return policy, torch.stack(rewards), torch.stack(norms)


def main():
    ap = argparse.ArgumentParser(description=__doc__,
                                 formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=50)
    a = ap.parse_args()
    policy, rewards, _ = train(a.steps, report=10)
    tokens = torch.arange(8, device=policy.embedding.device)
    top = Server(policy)(tokens, torch.zeros_like(tokens))
    print(f"reward {float(rewards[0]):.3f} -> {float(rewards[-1]):.3f}; after words 0..7: "
          f"{top.top_ids[:, 0].tolist()}")


if __name__ == "__main__":
    main()
