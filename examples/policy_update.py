"""A policy update in miniature, on one GPU: rollout, scoring under a frozen 8-bit reference, clipped update.

    python examples/policy_update.py [--steps 30]

The policy is a small residual network over a synthetic task: given a prompt
token, answer with a token of the same parity. Each step draws a group of
answers per prompt (sample_top_p), rewards them, scores them under the frozen
reference, whose weights were quantised once and whose layers run in 8 bits
(add_rmsnorm_fp8, linear_fp8, quantize_fp8), and trains the policy on them:
token_logprobs gives the reference's and the rollout's log-probabilities,
policy_loss the clipped loss with its KL term and, through backward, the
gradient that an optimiser takes. Prints the mean reward, the KL estimate and
the clipped share.
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from grpo_training_engine_b200 import ops  # noqa: E402

HIDDEN, INTER, VOCAB, EPS = 256, 512, 1000, 1e-6


class Policy(torch.nn.Module):
    """Embedding, one gated MLP block with its norm, a final norm and a head: bf16 modules of torch."""

    def __init__(self) -> None:
        super().__init__()
        self.embed = torch.nn.Embedding(VOCAB, HIDDEN)
        self.norms = torch.nn.ParameterList(torch.nn.Parameter(torch.ones(HIDDEN)) for _ in range(2))
        self.gate = torch.nn.Linear(HIDDEN, INTER, bias=False)
        self.up = torch.nn.Linear(HIDDEN, INTER, bias=False)
        self.down = torch.nn.Linear(INTER, HIDDEN, bias=False)
        self.head = torch.nn.Linear(HIDDEN, VOCAB, bias=False)

    def forward(self, tokens: torch.Tensor) -> torch.Tensor:
        x = self.embed(tokens)
        h = torch.nn.functional.rms_norm(x, (HIDDEN,), self.norms[0], EPS)
        x = x + self.down(torch.nn.functional.silu(self.gate(h)) * self.up(h))
        return self.head(torch.nn.functional.rms_norm(x, (HIDDEN,), self.norms[1], EPS))


class Reference8Bit:
    """The policy's weights as they were, in 8 bits: every projection is linear_fp8 of what a norm or a
    quantiser wrote."""

    def __init__(self, policy: Policy) -> None:
        self.embed = policy.embed.weight.detach().clone()
        self.norms = [w.detach().clone() for w in policy.norms]
        self.weights = {name: ops.quantize_fp8_weight(getattr(policy, name).weight.detach())
                        for name in ("gate", "up", "down", "head")}

    def logits(self, tokens: torch.Tensor) -> torch.Tensor:
        x = self.embed[tokens]
        q, scale, _ = ops.add_rmsnorm_fp8(x, self.norms[0], EPS)
        act = ops.silu_mul(ops.linear_fp8(q, scale, *self.weights["gate"]),
                           ops.linear_fp8(q, scale, *self.weights["up"]))
        mlp = ops.linear_fp8(*ops.quantize_fp8(act), *self.weights["down"])
        q, scale, _ = ops.add_rmsnorm_fp8(mlp, self.norms[1], EPS, x)
        return ops.linear_fp8(q, scale, *self.weights["head"])


def train(steps: int = 30, prompts: int = 64, group: int = 16, updates: int = 2, seed: int = 0) -> list[dict]:
    """Runs `steps` rollouts with `updates` policy updates each; returns what each step measured."""
    torch.manual_seed(seed)
    dev = torch.device("cuda")
    policy = Policy().to(dev, torch.bfloat16)
    reference = Reference8Bit(policy)
    optimiser = torch.optim.AdamW(policy.parameters(), lr=2e-3, weight_decay=0.0)
    draws = torch.Generator(device=dev).manual_seed(seed + 1)
    history = []
    for _ in range(steps):
        prompt = torch.randint(0, VOCAB, (prompts,), device=dev, generator=draws).repeat_interleave(group)
        with torch.no_grad():
            logits = policy(prompt)
            answer = ops.sample_top_p(logits, 1.0, 1.0, generator=draws)
            old = ops.token_logprobs(logits, answer)
            ref = ops.token_logprobs(reference.logits(prompt), answer)
        reward = (answer % 2 == prompt % 2).float()
        by_group = reward.view(prompts, group)
        advantage = ((by_group - by_group.mean(1, keepdim=True)) / (by_group.std(1, keepdim=True) + 1e-4)).view(-1)
        for _ in range(updates):
            out = ops.policy_loss(policy(prompt)[:, None], answer[:, None], old[:, None], advantage,
                                  ref_logprobs=ref[:, None], kl_coef=0.02, reduction="sequence")
            optimiser.zero_grad(set_to_none=True)
            out.loss.backward()
            optimiser.step()
        history.append({"reward": float(reward.mean()), "loss": float(out.loss.detach()), "kl": float(out.kl),
                        "clipped": float(out.clip_fraction)})
    return history


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--steps", type=int, default=30)
    for i, h in enumerate(train(parser.parse_args().steps)):
        print(f"step {i:3d}  reward {h['reward']:.3f}  loss {h['loss']:+.4f}  kl {h['kl']:.4f}  "
              f"clipped {h['clipped']:.3f}")


if __name__ == "__main__":
    main()
