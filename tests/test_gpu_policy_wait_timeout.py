"""The policy gradient's bounded waits run out, report, and return.

The test flag PKV_POLICY_TEST_WAIT_TIMEOUT shortens every limit to 4096 polls and makes the first CTA's producer leave
out the last part of its second row: the consumers wait for a part that never comes, the producer for one that is never
freed. Nothing faults or traps; the waits run out. The launch ends promptly with the timeout bit, a loss of NaN, NaN in
the rows that were left out and right values in the others, and the next call on the stream is right.
"""

from __future__ import annotations

import time

import pytest
import torch

from grpo_training_engine_b200 import _lib, ops
from test_gpu_policy import _batch, _check_policy, _policy_formula

pytestmark = pytest.mark.gpu


# rows held by one CTA on an SM (148 of them) and by two (296): four and more rows each; two rows for the first alone
@pytest.mark.parametrize("batch,length,vocab,dtype,ctas", [
    (2, 300, 110001, torch.bfloat16, 148), (4, 300, 33001, torch.float32, 296), (1, 149, 110001, torch.float16, 148)])
@pytest.mark.parametrize("with_status", [True, False])
def test_wait_timeout_is_reported_and_the_context_stays_usable(batch, length, vocab, dtype, ctas, with_status):
    logits, tokens, old, adv, _, _ = _batch(batch, length, vocab, dtype, 9, kl=False)
    lib, rows, stream = _lib.load(), batch * length, torch.cuda.current_stream().cuda_stream
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out, logp = torch.empty(3, device="cuda"), torch.empty(batch, length, device="cuda")
    grad = torch.empty_like(logits)
    ws = torch.empty(lib.pkv_policy_loss_workspace_size(batch, length), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    t0 = time.monotonic()
    code = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16, torch.float32: _lib.DTYPE_F32}[dtype]
    rc = lib.pkv_policy_loss(logits.data_ptr(), code, tokens.data_ptr(), old.data_ptr(), None, adv.data_ptr(), 1, 0,
                             None, batch, length, vocab, length * vocab, vocab, 1.0, 0.2, 0.2, 0.0,
                             _lib.REDUCE_SUM | _lib.POLICY_TEST_WAIT_TIMEOUT, out.data_ptr(), logp.data_ptr(),
                             grad.data_ptr(), ws.data_ptr(), ws.numel(), status.data_ptr() if with_status else None,
                             stream)
    assert rc == 0, _lib.last_detail()
    torch.cuda.synchronize()
    assert time.monotonic() - t0 < 10.0
    assert int(status) == (_lib.DEV_WAIT_TIMEOUT if with_status else 0)
    assert torch.isnan(out).all()
    # the first CTA's rows after its first are left out; any other row is whole, or left out as well
    want = _policy_formula(logits, tokens, old, adv, reduction="sum")
    lost = torch.isnan(logp).view(-1)
    flat = grad.view(rows, vocab)
    assert lost[ctas::ctas].all() and torch.isnan(flat[lost, 0].float()).all()
    assert not lost[0] and int(lost.sum()) < rows
    assert torch.all((logp.double() - want[1]).abs().view(-1)[~lost] <= 3e-5 + 1e-6 * want[1].abs().view(-1)[~lost])
    assert torch.isfinite(flat[~lost].float()).all()
    # a scaled gradient of those rows is NaN throughout
    two = torch.full((), 2.0, device="cuda")
    rc = lib.pkv_policy_loss_grad(logits.data_ptr(), code, batch, length, vocab, length * vocab, vocab, 1.0,
                                  ws.data_ptr(), ws.numel(), two.data_ptr(), grad.data_ptr(), stream)
    assert rc == 0 and torch.isnan(flat[lost].float()).all() and torch.isfinite(flat[~lost].float()).all()

    leaf = logits.requires_grad_()
    status.zero_()
    got = ops.policy_loss(leaf, tokens, old, adv, reduction="sum", status=status)
    (grad,) = torch.autograd.grad(got.loss, leaf)
    assert int(status) == 0
    _check_policy(got, grad, want)
