"""The policy gradient under an upstream gradient: a scaled loss (fp16 training), a mean over accumulated batches."""

from __future__ import annotations

import pytest
import torch

from test_gpu_policy import DTYPES, _batch, _check_grad, _policy_formula

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from grpo_training_engine_b200 import _lib, ops


@pytest.mark.parametrize("upstream", [65536.0, 3.0, 1.0 / 3.0, -0.7, 1.0, 0.0])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("batch,length,vocab", [(3, 20, 1003), (900, 2, 64), (3, 70, 9001), (8, 40, 32003),
                                                (2, 200, 45001), (4, 70, 151936)])
def test_gradient_is_rounded_once_whatever_the_upstream(batch, length, vocab, dtype, upstream):
    """The formula times the upstream, rounded once to the logits' type: half a step of it, and half the smallest step
    (what a push-down element of an unscaled fp16 gradient is below)."""
    logits, tokens, old, adv, mask, ref = _batch(batch, length, vocab, dtype, vocab + 1)
    mask[0, 0] = True
    kw = dict(kl_coef=0.05, clip_low=0.2, clip_high=0.28, temperature=0.9)
    *_, d, bulk, _ = _policy_formula(logits, tokens, old, adv, mask, ref, **kw)
    leaf = logits.detach().requires_grad_()
    got = ops.policy_loss(leaf, tokens, old, adv, mask, ref_logprobs=ref, **kw)
    u = torch.tensor(upstream, device="cuda")
    (grad,) = torch.autograd.grad(got.loss, leaf, u)
    _check_grad(grad, d * u.double(), bulk * abs(u.double()))
    assert not grad[~mask].any()


def test_masked_rows_stay_unread_and_zero_under_an_upstream():
    logits, tokens, old, adv, mask, ref = _batch(4, 6, 300, torch.float16, 31)
    mask[1] = False
    mask[0, 2] = False
    *_, d, bulk, _ = _policy_formula(logits, tokens, old, adv, mask, ref, 0.1)
    for t in (logits, old, ref):
        t[1] = float("nan")
        t[0, 2] = float("inf")
    tokens[1] = -100
    tokens[0, 2] = 1 << 40
    leaf = logits.requires_grad_()
    got = ops.policy_loss(leaf, tokens, old, adv, mask, ref_logprobs=ref, kl_coef=0.1)
    (grad,) = torch.autograd.grad(got.loss * 1024.0, leaf)
    _check_grad(grad, d * 1024, bulk * 1024)
    assert not grad[1].any() and not grad[0, 2].any()


def test_shifted_view_under_an_upstream():
    """logits[:, :-1] of an odd vocabulary: rows of the logits and of the gradient begin at different alignments."""
    base, tokens, old, adv, mask, _ = _batch(3, 9, 2003, torch.bfloat16, 5)
    leaf = base.detach().requires_grad_()
    got = ops.policy_loss(leaf[:, :-1], tokens[:, :-1], old[:, :-1], adv, mask[:, :-1])
    (got.loss / 3).backward()
    *_, d, bulk, _ = _policy_formula(base[:, :-1], tokens[:, :-1], old[:, :-1], adv, mask[:, :-1])
    third = torch.tensor(1.0, device="cuda") / 3
    _check_grad(leaf.grad[:, :-1], d * third.double(), bulk / 3)
    assert not leaf.grad[:, -1].any()


def test_empty_batch_under_an_upstream():
    leaf = torch.empty(0, 4, 10, device="cuda", requires_grad=True)
    got = ops.policy_loss(leaf, torch.empty(0, 4, dtype=torch.int64, device="cuda"), torch.empty(0, 4, device="cuda"),
                          torch.empty(0, device="cuda"))
    (got.loss * 3).backward()
    assert leaf.grad.shape == (0, 4, 10)


@pytest.mark.parametrize("n", [1, 1000, 1 << 20])
def test_scale_grad_in_place(n):
    """The C entry point that multiplies a stored fp32 gradient; an upstream of 1 leaves it as it is."""
    grad = torch.randn(n, device="cuda")
    want = grad * 3
    for u, expect in ((1.0, grad.clone()), (3.0, want)):
        up = torch.tensor(u, device="cuda")
        rc = _lib.load().pkv_scale_grad(grad.data_ptr(), n, _lib.DTYPE_F32, up.data_ptr(),
                                        torch.cuda.current_stream().cuda_stream)
        assert rc == 0 and torch.equal(grad, expect)
