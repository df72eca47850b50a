"""Token log-probabilities and the clipped policy loss against their formulas in 64 bits."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from grpo_training_engine_b200 import _lib, ops

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
# half a step of a value of p bits is 2^-p of it; half the smallest step
HALF = {torch.bfloat16: (2.0 ** -8, 2.0 ** -134), torch.float16: (2.0 ** -11, 2.0 ** -25),
        torch.float32: (2.0 ** -24, 2.0 ** -150)}
# The sum of a row's exponentials: each within 2^-22 (hardware exp2) and |t| 2^-23 of its exponent's rounding, added
# in at most about 300 steps of 2^-24 (a thread's share of the largest vocabulary) and 15 joins.
SUM = 3e-5


def _logits(shape, dtype, seed, sd=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=g) * sd).to(dtype)


def _formula(logits, tokens, temperature):
    logs = torch.log_softmax(logits.double() / temperature, -1)
    p = logs.exp()
    ent = -(p * torch.where(p > 0, logs, torch.zeros_like(logs))).sum(-1)
    return logs, p, logs.gather(-1, tokens[..., None].long())[..., 0], ent


def _check_logp(got, want):
    assert got.dtype == torch.float32 and got.shape == want.shape
    assert torch.all((got.double() - want).abs() <= SUM + 1e-6 * want.abs())


def _check_grad(got, want, bulk):
    """bulk: the magnitude that the terms of an element have before they cancel."""
    rel, tiny = HALF[got.dtype]
    assert torch.all((got.double() - want).abs() <= (1.01 * rel) * want.abs() + 2 * SUM * bulk + tiny)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows,vocab,temperature", [(1, 1, 1.0), (1, 151936, 0.7), (3, 2, 1.0), (5, 7, 1.3),
                                                    (4, 1000, 1.0), (9, 1001, 0.7), (40, 32003, 1.0),
                                                    (200, 151936, 1.0), (2, 300007, 1.0), (2000, 100, 1.0),
                                                    (1201, 2003, 1.0)])
def test_token_logprobs_and_gradient(rows, vocab, temperature, dtype):
    logits = _logits((rows, vocab), dtype, rows + vocab).requires_grad_()
    tokens = torch.randint(0, vocab, (rows,), device="cuda")
    logs, p, lp, ent = _formula(logits.detach(), tokens, temperature)
    _check_logp(ops.token_logprobs(logits.detach(), tokens, temperature=temperature), lp)
    got, got_ent = ops.token_logprobs(logits, tokens.int(), temperature=temperature, entropy=True)
    _check_logp(got.detach(), lp)
    # the entropy is a difference of two sums of magnitude up to log(vocab) and the mean exponent
    assert torch.all((got_ent.detach().double() - ent).abs() <= 20 * SUM)
    g, h = torch.randn(rows, device="cuda"), torch.randn(rows, device="cuda")
    (grad,) = torch.autograd.grad((got, got_ent), logits, (g, h))
    assert grad.dtype == dtype and grad.shape == logits.shape
    hot = torch.zeros_like(p).scatter_(-1, tokens[:, None], 1.0)
    gd, hd = g.double()[:, None], h.double()[:, None]
    inner = torch.where(p > 0, logs, torch.zeros_like(logs)) + ent[:, None]
    want = (gd * (hot - p) - hd * p * inner) / temperature
    bulk = (gd.abs() * (hot + p) + hd.abs() * p * (inner.abs() + 20)) / temperature
    _check_grad(grad, want, bulk)
    # one output alone
    got = ops.token_logprobs(logits, tokens, temperature=temperature)
    (grad,) = torch.autograd.grad(got.sum(), logits)
    _check_grad(grad, (hot - p) / temperature, (hot + p) / temperature)
    _, got_ent = ops.token_logprobs(logits, tokens, temperature=temperature, entropy=True)
    (grad,) = torch.autograd.grad(got_ent, logits, h)
    _check_grad(grad, -hd * p * inner / temperature, hd.abs() * p * (inner.abs() + 20) / temperature)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("vocab", [1000, 1003])
def test_token_logprobs_views(vocab, dtype):
    """The shifted view that a trainer takes, rows of a wider matrix, and a transposed vocabulary."""
    base = _logits((3, 6, vocab + 5), dtype, vocab)
    tokens = torch.randint(0, vocab, (3, 5), device="cuda")
    for view in (base[:, :-1, :vocab], base[:, 1:, 3:vocab + 3], base.flip(1)[:, :5, 5:],
                 base[..., :vocab].transpose(1, 2).contiguous().transpose(1, 2)[:, :5]):
        leaf = view.detach().requires_grad_()
        _, p, lp, _ = _formula(view, tokens, 1.0)
        got = ops.token_logprobs(leaf, tokens)
        _check_logp(got.detach(), lp)
        (grad,) = torch.autograd.grad(got.sum(), leaf)
        hot = torch.zeros_like(p).scatter_(-1, tokens[..., None], 1.0)
        _check_grad(grad, hot - p, hot + p)
    two = base.view(18, -1)[::2, :vocab]
    got = ops.token_logprobs(two, tokens.view(-1)[:9])
    _check_logp(got, _formula(two, tokens.view(-1)[:9], 1.0)[2])


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("vocab", [9, 1000, 151936])
def test_token_logprobs_masked_vocabularies(vocab, dtype):
    """Entries of -inf, of the type's lowest value, rows of nothing else, a single entry, and huge logits."""
    low, top = torch.finfo(dtype).min, torch.finfo(dtype).max
    logits = _logits((8, vocab), dtype, 3)
    tokens = torch.zeros(8, dtype=torch.int64, device="cuda")
    logits[0, 1::2] = float("-inf")
    logits[1, 1::2] = low
    logits[2] = low                    # a uniform distribution
    logits[3] = float("-inf")
    logits[3, 0] = 1.0                 # all of it on the token
    logits[4] = float("-inf")          # nothing: NaN
    logits[5, 0] = float("nan")        # NaN
    logits[6] = low
    logits[6, 0] = top                 # the widest range there is
    logits[7, -1] = float("-inf")
    tokens[7] = vocab - 1              # a token of probability 0
    leaf = logits.requires_grad_()
    got, ent = ops.token_logprobs(leaf, tokens, entropy=True)
    logs, p, lp, want_ent = _formula(logits.detach(), tokens, 1.0)
    finite = [0, 1, 2, 3, 6]
    _check_logp(got.detach()[finite], lp[finite])
    assert torch.isnan(got[[4, 5]]).all() and got[7] == float("-inf")
    assert torch.all((ent.detach().double() - want_ent)[finite].abs() <= 20 * SUM)
    (grad,) = torch.autograd.grad((got, ent), leaf, (torch.ones_like(got), torch.ones_like(ent)))
    hot = torch.zeros_like(p).scatter_(-1, tokens[:, None], 1.0)
    inner = torch.where(p > 0, logs, torch.zeros_like(logs)) + want_ent[:, None]
    for i in finite:
        _check_grad(grad[i], hot[i] - p[i] - p[i] * inner[i], hot[i] + p[i] * (1 + inner[i].abs() + 20))
    assert torch.isnan(grad[4].float()).all() and torch.isnan(grad[5].float()).all()


def test_token_logprobs_token_out_of_range():
    logits = _logits((4, 50), torch.float32, 1)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    tokens = torch.tensor([-1, 50, 2, 1 << 40], device="cuda")
    got = ops.token_logprobs(logits, tokens, status=status)
    assert torch.isnan(got[[0, 1, 3]]).all() and torch.isfinite(got[2])
    assert int(status) == _lib.DEV_TOKEN_OUT_OF_RANGE


def test_token_logprobs_empty():
    logits = torch.empty(0, 10, device="cuda", requires_grad=True)
    got = ops.token_logprobs(logits, torch.empty(0, dtype=torch.int64, device="cuda"))
    got.sum().backward()
    assert got.shape == (0,) and logits.grad.shape == (0, 10)


def test_offsets_past_32_bits():
    rows, vocab = 16384, 151936
    logits = torch.zeros(1, rows, vocab, device="cuda", dtype=torch.bfloat16)
    logits[0, -3:] = _logits((3, vocab), torch.bfloat16, 8)
    tokens = torch.randint(0, vocab, (1, rows), device="cuda")
    _check_logp(ops.token_logprobs(logits, tokens)[0, -3:], _formula(logits[0, -3:], tokens[0, -3:], 1.0)[2])
    old = torch.full((1, rows), -10.0, device="cuda")
    mask = torch.zeros(1, rows, dtype=torch.bool, device="cuda")
    mask[0, -3:] = True
    got = ops.policy_loss(logits.requires_grad_(), tokens, old, torch.full((1,), -1.0, device="cuda"), mask)
    (grad,) = torch.autograd.grad(got.loss, logits)
    want = _policy_formula(logits[:, -3:], tokens[:, -3:], old[:, -3:], torch.full((1,), -1.0, device="cuda"),
                           mask[:, -3:])
    _check_policy(got, grad, want, rows=slice(rows - 3, rows))
    assert not grad[0, ::1000].any()


# ---------------------------------------------------------------------------
# policy loss
# ---------------------------------------------------------------------------
def _policy_formula(logits, tokens, old, adv, mask=None, ref=None, kl_coef=0.0, clip_low=0.2, clip_high=0.2,
                    temperature=1.0, reduction="token"):
    """(loss, logprobs, kl, clip fraction, gradient, its bulk, the loss's bulk), by the formulas in 64 bits."""
    with torch.no_grad():
        mask = torch.ones_like(tokens, dtype=torch.bool) if mask is None else mask != 0
        seen = torch.where(mask[..., None], logits.double(), torch.zeros((), dtype=torch.float64, device="cuda"))
        safe = torch.where(mask, tokens.long(), 0)
        _, p, lp, _ = _formula(seen, safe, temperature)
        a = (adv if adv.ndim == 2 else adv[:, None]).double().expand_as(lp)
        m = mask.double()
        w = {"token": m / m.sum().clamp_min(1), "sum": m,
             "sequence": m / m.sum(1, keepdim=True).clamp_min(1) / m.shape[0]}[reduction]
        r = (lp - old.double()).exp()
        free, held = r * a, r.clamp(1 - clip_low, 1 + clip_high) * a
        value, slope = -torch.minimum(free, held), torch.where(free <= held, -free, 0.0)
        kl = torch.zeros_like(lp)
        bulk = r * a.abs()
        if ref is not None:
            d = ref.double() - lp
            kl = d.exp() - d - 1
            value, slope = value + kl_coef * kl, slope + kl_coef * (1 - d.exp())
            bulk = bulk + kl_coef * (1 + d.exp())
        hot = torch.zeros_like(p).scatter_(-1, safe[..., None], 1.0)
        s = (torch.where(mask, slope, 0.0) * w / temperature)[..., None]
        b = (torch.where(mask, bulk, 0.0) * w / temperature)[..., None]
        count = m.sum().clamp_min(1)
        zero = torch.zeros((), dtype=torch.float64, device="cuda")
        # an element is slope (hot - p); the slope is off by SUM of its terms, hot - p by SUM of p
        return ((torch.where(mask, value, zero) * w).sum(), torch.where(mask, lp, zero),
                torch.where(mask, kl, zero).sum() / count, ((held < free) & mask).double().sum() / count,
                s * (hot - p), b * (hot - p).abs() + s.abs() * (hot + p), (torch.where(mask, bulk + kl, zero) * w).sum())


def _check_policy(got, grad, want, rows=slice(None)):
    loss, lp, kl, clipped, d, bulk, loss_bulk = want
    assert abs(float(got.loss.detach()) - float(loss)) <= 2 * SUM * float(loss_bulk) + 1e-30
    _check_logp(got.logprobs[:, rows], lp)
    assert abs(float(got.kl) - float(kl)) <= 4 * SUM * (1 + float(kl))
    assert abs(float(got.clip_fraction) - float(clipped)) <= 1e-6
    if grad is not None:
        _check_grad(grad[:, rows], d, bulk)


def _batch(batch, length, vocab, dtype, seed, kl=True, per_token=False, temperature=1.0):
    logits = _logits((batch, length, vocab), dtype, seed)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    tokens = torch.randint(0, vocab, (batch, length), device="cuda", generator=g)
    lp = _formula(logits, tokens, temperature)[2].float()
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    old = lp + 0.3 * rand(batch, length)
    ref = lp + 0.5 * rand(batch, length) if kl else None
    adv = rand(batch, length) if per_token else rand(batch)
    mask = torch.rand(batch, length, device="cuda", generator=g) < 0.7
    return logits, tokens, old, adv, mask, ref


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("batch,length,vocab,reduction,temperature", [
    (1, 1, 1, "token", 1.0), (1, 1, 151936, "sequence", 1.0), (2, 9, 1000, "token", 1.0),
    (3, 5, 1003, "sequence", 0.7), (4, 33, 129, "sum", 1.3), (8, 40, 32003, "sequence", 1.0),
    (2, 100, 151936, "token", 1.0), (1, 1500, 64, "sequence", 1.0), (7, 3, 200001, "sum", 1.0),
    (3, 70, 9001, "token", 1.0), (2, 200, 45001, "sequence", 1.0)])
def test_policy_loss(batch, length, vocab, reduction, temperature, dtype):
    kl, per_token = bool((batch + length) % 2), length % 3 == 0
    logits, tokens, old, adv, mask, ref = _batch(batch, length, vocab, dtype, vocab, kl, per_token, temperature)
    kw = dict(kl_coef=0.05 if kl else 0.0, clip_low=0.2, clip_high=0.28, temperature=temperature, reduction=reduction)
    for m in (mask, None, mask.to(torch.int64)):
        want = _policy_formula(logits, tokens, old, adv, m, ref, **kw)
        plain = ops.policy_loss(logits, tokens, old, adv, m, ref_logprobs=ref, **kw)
        assert not plain.loss.requires_grad
        _check_policy(plain, None, want)
        leaf = logits.detach().requires_grad_()
        got = ops.policy_loss(leaf, tokens, old, adv, m, ref_logprobs=ref, **kw)
        (grad,) = torch.autograd.grad(got.loss, leaf)
        assert not got.logprobs.requires_grad and got.loss.shape == ()
        _check_policy(got, grad, want)
        again = ops.policy_loss(logits.detach().requires_grad_(), tokens, old, adv, m, ref_logprobs=ref, **kw)
        assert all(torch.equal(x, y) for x, y in zip(got, again))  # no result depends on timing


@pytest.mark.parametrize("vocab", [1000, 1003])
def test_policy_loss_shifted_view_through_a_layer(vocab):
    """logits[:, :-1] of a model's output, the loss scaled, the gradient arriving at the weight."""
    torch.manual_seed(0)
    hidden = torch.randn(3, 8, 16, device="cuda")
    weight = torch.randn(vocab, 16, device="cuda", requires_grad=True)
    logits = hidden @ weight.t()
    _, tokens, old, adv, mask, ref = _batch(3, 7, vocab, torch.float32, 4)
    old = _formula(logits.detach()[:, :-1], tokens, 1.0)[2].float() + 0.1
    got = ops.policy_loss(logits[:, :-1], tokens, old, adv, mask, ref_logprobs=ref, kl_coef=0.01)
    (got.loss * 3.0).backward()
    want = _policy_formula(logits.detach()[:, :-1], tokens, old, adv, mask, ref, 0.01)
    _check_policy(got, None, want)
    d = torch.einsum("btv,bth->vh", 3 * want[4], hidden[:, :-1].double())
    bulk = torch.einsum("btv,bth->vh", 3 * want[5], hidden[:, :-1].abs().double())
    assert torch.all((weight.grad.double() - d).abs() <= 4 * SUM * bulk + 1e-6 * d.abs() + 1e-9)


def test_policy_loss_gradient_against_differences():
    logits, tokens, old, adv, mask, ref = _batch(2, 6, 50, torch.float32, 12)
    kw = dict(ref_logprobs=ref, kl_coef=0.3, reduction="sum")
    leaf = logits.requires_grad_()
    (grad,) = torch.autograd.grad(ops.policy_loss(leaf, tokens, old, adv, mask, **kw).loss, leaf)
    g = torch.Generator(device="cuda").manual_seed(3)
    for _ in range(4):
        step = torch.randn(logits.shape, device="cuda", generator=g) * 1e-3
        up = ops.policy_loss(logits.detach() + step, tokens, old, adv, mask, **kw)
        down = ops.policy_loss(logits.detach() - step, tokens, old, adv, mask, **kw)
        if float(up.clip_fraction) != float(down.clip_fraction):
            continue  # a kink lies between the two
        slope = float(up.loss.double() - down.loss.double()) / 2
        want = float((grad.double() * step.double()).sum())
        # second-order terms of a step of 1e-3 and fp32 sums of about ten terms of order 1
        assert abs(slope - want) <= 1e-2 * abs(want) + 1e-5


def test_token_logprobs_gradient_against_differences():
    logits = _logits((5, 40), torch.float32, 2)
    tokens = torch.arange(5, device="cuda")
    leaf = logits.requires_grad_()
    lp, ent = ops.token_logprobs(leaf, tokens, entropy=True)
    (grad,) = torch.autograd.grad((lp.sum() + 2 * ent.sum()), leaf)
    step = torch.randn(logits.shape, device="cuda") * 1e-3
    vals = []
    for sign in (1, -1):
        lp, ent = ops.token_logprobs(logits.detach() + sign * step, tokens, entropy=True)
        vals.append(float(lp.double().sum() + 2 * ent.double().sum()))
    want = float((grad.double() * step.double()).sum())
    assert abs((vals[0] - vals[1]) / 2 - want) <= 1e-2 * abs(want) + 2e-5


@pytest.mark.parametrize("reduction", ["token", "sequence", "sum"])
def test_policy_loss_masks(reduction):
    """A sequence without tokens, a batch without any, and whatever lies under the mask."""
    logits, tokens, old, adv, mask, ref = _batch(4, 6, 300, torch.bfloat16, 31)
    mask[1] = False
    mask[0, 2] = False
    clean = _policy_formula(logits, tokens, old, adv, mask, ref, 0.1, reduction=reduction)
    for t in (logits, old, ref):
        t[1] = float("nan")
        t[0, 2] = float("inf")
    tokens[1] = -100
    tokens[0, 2] = 1 << 40
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    leaf = logits.requires_grad_()
    got = ops.policy_loss(leaf, tokens, old, adv, mask, ref_logprobs=ref, kl_coef=0.1, reduction=reduction,
                          status=status)
    (grad,) = torch.autograd.grad(got.loss, leaf)
    _check_policy(got, grad, clean)
    assert int(status) == 0 and not grad[1].any() and not grad[0, 2].any()
    got = ops.policy_loss(leaf, tokens, old, adv, torch.zeros_like(mask), ref_logprobs=ref, kl_coef=0.1,
                          reduction=reduction)
    (grad,) = torch.autograd.grad(got.loss, leaf)
    assert float(got.loss) == 0 and float(got.kl) == 0 and float(got.clip_fraction) == 0 and not grad.any()


def test_policy_loss_clip_cases():
    """Each side of each bound, for advantages of both signs and of zero."""
    vocab = 16
    logits = _logits((1, 10, vocab), torch.float32, 1)
    tokens = torch.randint(0, vocab, (1, 10), device="cuda")
    lp = _formula(logits, tokens, 1.0)[2]
    ratio = torch.tensor([0.5, 0.75, 1.0, 1.25, 1.5] * 2, device="cuda", dtype=torch.float64)
    old = (lp - ratio.log()).float()
    adv = torch.tensor([[1.0] * 5 + [-1.0] * 5], device="cuda")
    for a in (adv, 0 * adv):
        want = _policy_formula(logits, tokens, old, a, clip_low=0.3, clip_high=0.4, reduction="sum")
        leaf = logits.detach().requires_grad_()
        got = ops.policy_loss(leaf, tokens, old, a, clip_low=0.3, clip_high=0.4, reduction="sum")
        (grad,) = torch.autograd.grad(got.loss, leaf)
        _check_policy(got, grad, want)
    assert float(want[0]) == 0 and not grad.any()


def test_policy_loss_out_of_range_token_is_loud():
    logits, tokens, old, adv, _, _ = _batch(2, 3, 20, torch.float32, 6)
    tokens[1, 1] = 20
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = ops.policy_loss(logits, tokens, old, adv, status=status)
    assert torch.isnan(got.loss) and torch.isnan(got.logprobs[1, 1]) and int(status) == _lib.DEV_TOKEN_OUT_OF_RANGE
    assert int(torch.isnan(got.logprobs).sum()) == 1


def test_policy_loss_gradient_is_handed_out_once():
    logits, tokens, old, adv, mask, _ = _batch(2, 3, 20, torch.float32, 6)
    got = ops.policy_loss(logits.requires_grad_(), tokens, old, adv, mask)
    got.loss.backward(retain_graph=True)
    with pytest.raises(RuntimeError, match="handed out"):
        got.loss.backward()


def test_policy_loss_empty_and_other_stream():
    empty = ops.policy_loss(torch.empty(0, 4, 10, device="cuda", requires_grad=True),
                            torch.empty(0, 4, dtype=torch.int64, device="cuda"), torch.empty(0, 4, device="cuda"),
                            torch.empty(0, device="cuda"))
    assert float(empty.loss) == 0 and empty.logprobs.shape == (0, 4)
    logits, tokens, old, adv, mask, ref = _batch(4, 30, 5000, torch.bfloat16, 16)
    want = ops.policy_loss(logits, tokens, old, adv, mask, ref_logprobs=ref, kl_coef=0.1)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = ops.policy_loss(logits, tokens, old, adv, mask, ref_logprobs=ref, kl_coef=0.1)
    st.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_no_second_derivatives():
    logits, tokens, old, adv, mask, _ = _batch(2, 3, 20, torch.float32, 6)
    leaf = logits.requires_grad_()
    for loss in (ops.policy_loss(leaf, tokens, old, adv, mask).loss, ops.token_logprobs(leaf, tokens).sum()):
        with pytest.raises(RuntimeError, match="second derivative"):
            torch.autograd.grad(loss, leaf, create_graph=True)
