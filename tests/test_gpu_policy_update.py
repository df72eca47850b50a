"""The scoring and update operators together: the 8-bit reference against the model it was made of, and a few
policy updates."""

from __future__ import annotations

import importlib.util

import pytest
import torch

from conftest import REPO

pytestmark = pytest.mark.gpu


def _example():
    spec = importlib.util.spec_from_file_location("policy_update", REPO / "examples" / "policy_update.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def test_reference_in_8_bits_scores_like_the_model():
    ex = _example()
    torch.manual_seed(0)
    policy = ex.Policy().to("cuda", torch.bfloat16)
    tokens = torch.randint(0, ex.VOCAB, (300,), device="cuda")
    with torch.no_grad():
        want = policy(tokens).float()
        got = ex.Reference8Bit(policy).logits(tokens).float()
    # five products, each of operands rounded to 3 bits (about 2.6% each in the mean square), mostly in the residual's
    # shadow
    assert float((got - want).norm() / want.norm()) < 0.1
    lp = [ex.ops.token_logprobs(x, tokens) for x in (got, want)]
    assert float((lp[0] - lp[1]).abs().mean()) < 0.1


def test_policy_updates_raise_the_reward():
    history = _example().train(steps=60)
    assert all(torch.isfinite(torch.tensor(list(h.values()))).all() for h in history)
    assert all(h["kl"] >= 0 and 0 <= h["clipped"] <= 1 for h in history)
    # the first rollouts answer by chance (1024 answers: 0.5 +- 0.016); the updates are on the rewarded parity
    assert sum(h["reward"] for h in history[:3]) / 3 < 0.6
    assert sum(h["reward"] for h in history[-3:]) / 3 > 0.75
