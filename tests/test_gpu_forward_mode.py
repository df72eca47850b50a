"""Forward-mode derivatives, which the loss operators do not have, are refused and not dropped."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwd

from grpo_training_engine_b200 import ops


def _refused(device, requires_grad):
    logits = torch.randn(2, 3, 20, device=device).requires_grad_(requires_grad)
    tokens = torch.zeros(2, 3, dtype=torch.int64, device=device)
    old, adv = torch.zeros(2, 3, device=device), torch.ones(2, device=device)
    with fwd.dual_level():
        dual = fwd.make_dual(logits, torch.ones_like(logits))
        for x in (dual, dual[:, :, :10]):
            with pytest.raises(RuntimeError, match="forward-mode"):
                ops.token_logprobs(x, tokens)
            with pytest.raises(RuntimeError, match="forward-mode"):
                ops.policy_loss(x, tokens, old, adv)
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                ops.policy_loss(x, tokens, old, adv)


@pytest.mark.parametrize("requires_grad", [False, True])
def test_tangents_are_refused(requires_grad):
    _refused("cpu", requires_grad)


@pytest.mark.gpu
@pytest.mark.parametrize("requires_grad", [False, True])
def test_tangents_are_refused_on_the_gpu(requires_grad):
    _refused("cuda", requires_grad)


@pytest.mark.gpu
def test_plain_tensors_run_within_a_dual_level():
    logits, tokens = torch.randn(4, 20, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    want = ops.token_logprobs(logits, tokens)
    with fwd.dual_level():
        assert torch.equal(ops.token_logprobs(logits, tokens), want)
