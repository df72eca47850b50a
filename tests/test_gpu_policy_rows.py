"""The policy gradient where each block takes many rows in turn."""

from __future__ import annotations

import pytest
import torch

from test_gpu_policy import _batch, _check_policy, _policy_formula

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from grpo_training_engine_b200 import ops


@pytest.mark.parametrize("batch,length,vocab,dtype", [
    # rows held in shared memory, two blocks on an SM and one: five and more rows with a weight for each block
    (8, 301, 33001, torch.float32), (8, 301, 45003, torch.bfloat16), (5, 221, 110001, torch.bfloat16),
    (5, 221, 60001, torch.float32),
    # rows held in registers of a warp, of a small and of a larger block
    (40, 251, 1003, torch.float32), (20, 251, 9001, torch.float16), (10, 251, 16001, torch.float32)])
@pytest.mark.parametrize("shifted", [False, True])
def test_policy_loss_many_rows_per_block(batch, length, vocab, dtype, shifted):
    logits, tokens, old, adv, mask, ref = _batch(batch, length, vocab, dtype, vocab)
    cut = slice(None, -1) if shifted else slice(None)
    kw = dict(kl_coef=0.05, clip_low=0.2, clip_high=0.28, reduction="sequence")
    args = [t[:, cut] for t in (tokens, old)] + [adv, mask[:, cut]]
    want = _policy_formula(logits[:, cut], *args, ref[:, cut], **kw)
    leaf = logits.detach()[:, cut].requires_grad_()
    got = ops.policy_loss(leaf, *args, ref_logprobs=ref[:, cut], **kw)
    (grad,) = torch.autograd.grad(got.loss, leaf)
    _check_policy(got, grad, want)
    assert not grad[~args[-1]].any()
    plain = ops.policy_loss(logits[:, cut], *args, ref_logprobs=ref[:, cut], **kw)
    _check_policy(plain, None, want)
