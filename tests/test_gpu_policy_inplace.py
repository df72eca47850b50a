"""The loss and its measures are tensors of their own."""

from __future__ import annotations

import pytest
import torch

from test_gpu_policy import _batch, _check_grad, _policy_formula

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from grpo_training_engine_b200 import ops


def test_loss_can_be_changed_in_place():
    logits, tokens, old, adv, mask, ref = _batch(2, 9, 500, torch.float32, 3)
    *_, d, bulk, _ = _policy_formula(logits, tokens, old, adv, mask, ref, 0.1)
    leaf = logits.requires_grad_()
    got = ops.policy_loss(leaf, tokens, old, adv, mask, ref_logprobs=ref, kl_coef=0.1)
    loss, kl, clipped = (float(v.detach()) for v in (got.loss, got.kl, got.clip_fraction))
    loss_t = got.loss
    loss_t += 1.0
    loss_t /= 4
    loss_t.backward()
    _check_grad(leaf.grad, d / 4, bulk / 4)
    got.kl.mul_(2)
    assert abs(float(got.loss.detach()) - (loss + 1) / 4) <= 1e-6 * (1 + abs(loss))
    assert float(got.kl) == 2 * kl and float(got.clip_fraction) == clipped


@pytest.mark.parametrize("grad", [False, True])
def test_results_are_no_views(grad):
    logits, tokens, old, adv, mask, _ = _batch(2, 3, 20, torch.float32, 6)
    got = ops.policy_loss(logits.requires_grad_(grad), tokens, old, adv, mask)
    assert not any(t._is_view() for t in got)
    versions = [t._version for t in got]
    with torch.no_grad():
        got.kl.add_(1)
    assert [t._version for t in got] == [v + (i == 2) for i, v in enumerate(versions)]
