"""Measured cases of the scoring and policy-update operators.

A policy update scores the tokens of a rollout and trains on them. The frozen
reference model is scored in 8 bits: its norms write 8-bit activations with a
scale for each 128 values (add_rmsnorm_fp8), its projections and LM head
multiply them by 8-bit weights with a scale for each 128 x 128 block
(linear_fp8), and the logits become log-probabilities of the rollout's tokens
(token_logprobs). The trained policy's logits go into the clipped loss with a
KL term and come back as its gradient (policy_loss).

Each case runs one operator once, in its plain form (elementary torch
operations in 32 bits, rounded once at the end) or, with `own` set, as a user
calls the package. exact() gives the same outputs from the definitions in 64
bits. Geometries are the package's own: hidden 1536 / 3584, MLP 8960 / 18944,
a vocabulary of 151,936, rollouts of 128 sequences, responses of up to 512
tokens; the odd ones are generic.
"""

import math
import random

import torch

own = False

GROUP = 128        # values that share a scale (weights: blocks of 128 x 128)
E4M3_MAX = 448.0   # largest finite value of the 8-bit type
EPS = 1e-6
DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
BYTES = {"bfloat16": 2, "float16": 2, "float32": 4}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # the residual stream of one sequence's new token: latency only
        dict(name="norm one token", op="norm", rows=1, hidden=1536, dtype="bfloat16", residual=True),
        # an odd number of tokens, a hidden size that leaves a short last group, no residual (a first norm)
        dict(name="norm odd", op="norm", rows=777, hidden=1000, dtype="float16", residual=False),
        # a scoring batch: 32 sequences of 512 tokens of the larger model, bandwidth only
        dict(name="norm batch", op="norm", rows=16384, hidden=3584, dtype="bfloat16", residual=True),
        # stacked q/k/v projection of one new token: latency and the weight stream
        dict(name="linear one token", op="linear", rows=1, n=2048, k=1536, dtype="bfloat16", bias=True),
        # down projection of a rollout step of 128 sequences: few columns, long sums
        dict(name="linear rollout down", op="linear", rows=128, n=1536, k=8960, dtype="bfloat16", bias=False),
        # LM head on an odd handful of rows: the largest weight matrix, streamed once
        dict(name="linear head", op="linear", rows=37, n=151936, k=1536, dtype="float16", bias=False),
        # gate projection of a scoring batch of the larger model: bound by the tensor cores
        dict(name="linear batch gate", op="linear", rows=4096, n=18944, k=3584, dtype="bfloat16", bias=False),
        # log-probability of one sampled token: one row over the whole machine
        dict(name="logprob one token", op="logprob", rows=1, vocab=151936, dtype="bfloat16", temperature=0.7,
             entropy=False, grad=False),
        # scoring a batch of responses under the frozen model: one read of the logits
        dict(name="logprob batch", op="logprob", rows=4096, vocab=151936, dtype="bfloat16", temperature=1.0,
             entropy=False, grad=False),
        # log-probabilities and entropies with their gradient, an odd vocabulary whose rows are not aligned
        dict(name="logprob odd gradient", op="logprob", rows=515, vocab=32003, dtype="float32", temperature=1.0,
             entropy=True, grad=True),
        # a tiny model's update: two short responses, latency only
        dict(name="policy tiny", op="policy", batch=2, length=9, vocab=1000, dtype="float32", reduction="token",
             kl=True, per_token=False, shifted=False, temperature=1.0),
        # a GRPO group of 8 ragged responses of up to 512 tokens over the full vocabulary, with the KL term
        dict(name="policy group", op="policy", batch=8, length=512, vocab=151936, dtype="bfloat16",
             reduction="sequence", kl=True, per_token=False, shifted=True, temperature=1.0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _size(rng, lo, hi, step=8):
    """A size between lo and hi, spread over its logarithm: odd, or an odd multiple of `step`."""
    size = _log_int(rng, lo, hi)
    if rng.random() < 0.5 and size >= 2 * step:
        return (size // step - 1 | 1) * step
    return max(lo, min(size | 1, hi))


def draw(rng):
    op = rng.choice(["norm", "linear", "logprob", "policy"])
    if op == "norm":
        hidden = rng.choice([1536, 3584, _size(rng, 64, 8192), _size(rng, 64, 8192)])
        rows = min(_size(rng, 1, 16384), 16384 * 3584 // hidden)
        return dict(op=op, rows=rows, hidden=hidden, residual=rng.random() < 0.7,
                    dtype=rng.choice(["bfloat16", "float16", "float32"][: 3 if rows * hidden < 1 << 24 else 2]))
    if op == "linear":
        n, k = rng.choice([(2048, 1536), (1536, 8960), (8960, 1536), (3584, 18944), (18944, 3584),
                           (_size(rng, 64, 151936), 16 * (_log_int(rng, 8, 512) | 1)),
                           (_size(rng, 64, 20000), 16 * (_log_int(rng, 8, 1024) | 1))])
        rows = max(1, min(_size(rng, 1, 4096), 4096 * 18944 * 3584 // (n * k), 4096 * 18944 // n))
        return dict(op=op, rows=rows, n=n, k=k, dtype=rng.choice(["bfloat16", "float16"]),
                    bias=rng.random() < 0.4)
    vocab = rng.choice([151936, 1000, _size(rng, 100, 151936), _size(rng, 100, 151936)])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    most = max(4, min(4096, 4096 * 151936 * 2 // (vocab * BYTES[dtype])))
    temperature = rng.choice([1.0, 1.0, 0.7, 1.3])
    if op == "logprob":
        grad = rng.random() < 0.5
        return dict(op=op, rows=_size(rng, 1, most // 2 if grad else most), vocab=vocab, dtype=dtype,
                    temperature=temperature, entropy=rng.random() < 0.5, grad=grad)
    batch = _log_int(rng, 1, min(16, most))
    return dict(op=op, batch=batch, length=_size(rng, 2, max(2, most * 3 // (4 * batch))), vocab=vocab, dtype=dtype,
                reduction=rng.choice(["token", "sequence", "sum"]), kl=rng.random() < 0.7,
                per_token=rng.random() < 0.3, shifted=rng.random() < 0.5, temperature=temperature)


def _lengths(case):
    """Response lengths of a ragged batch, spread from a quarter of the longest to the longest."""
    b, t = case["batch"], case["length"]
    return [max(1, round(t * (0.25 + 0.75 * (i + 1) / b))) for i in range(b)]


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _quantize(v):
    """Rows of `v` (32 bits) as 8-bit values and a scale for each GROUP of them."""
    rows, k = v.shape
    groups = -(-k // GROUP)
    v = torch.nn.functional.pad(v, (0, groups * GROUP - k)).view(rows, groups, GROUP)
    scale = v.abs().amax(-1).clamp_min(2.0 ** -100) / E4M3_MAX
    q = (v / scale[..., None]).view(rows, groups * GROUP)[:, :k]
    return q.to(torch.float8_e4m3fn).contiguous(), scale


def _quantize_weight(w):
    """`w` [n, k] as 8-bit values and a scale for each GROUP x GROUP block."""
    n, k = w.shape
    bn, bk = -(-n // GROUP), -(-k // GROUP)
    pad = torch.nn.functional.pad(w, (0, bk * GROUP - k, 0, bn * GROUP - n)).view(bn, GROUP, bk, GROUP)
    scale = pad.abs().amax((1, 3)).clamp_min(2.0 ** -100) / E4M3_MAX
    q = (pad / scale[:, None, :, None]).view(bn * GROUP, bk * GROUP)[:n, :k]
    return q.to(torch.float8_e4m3fn).contiguous(), scale


def _logits(g, rows, vocab, dtype, tokens, temperature):
    """Logits of a trained model: a normal floor, and the sampled token anywhere from the floor's middle to well
    above all of it together (probabilities from 1 / vocab to about 0.9 at this temperature)."""
    out = torch.empty(rows, vocab, dtype=dtype, device="cuda")
    step = max(1, (1 << 28) // vocab)
    top = 1.1 * (temperature * math.log(vocab) + 2 / temperature)
    lift = torch.rand(rows, 1, generator=g, device="cuda") * top
    for r in range(0, rows, step):
        part = torch.randn(min(step, rows - r), vocab, generator=g, device="cuda") * 2
        part.scatter_(1, tokens[r:r + step, None], lift[r:r + step])
        out[r:r + step] = part
    return out


def _seen_logprobs(logits, tokens, temperature):
    """Log-probabilities of `tokens`, for inputs that lie near the policy's own."""
    rows = []
    step = max(1, (1 << 27) // logits.shape[-1])
    for r in range(0, logits.shape[0], step):
        z = logits[r:r + step].float() / temperature
        rows.append(z.gather(1, tokens[r:r + step, None])[:, 0] - torch.logsumexp(z, 1))
    return torch.cat(rows)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    dtype = DTYPES[case["dtype"]]
    st = dict(case)
    if case["op"] == "norm":
        rows, hidden = case["rows"], case["hidden"]
        channel = torch.exp(randn(hidden))  # a few channels of a residual stream are much wider than the rest
        st["x"] = (randn(rows, hidden) * channel).to(dtype)
        st["res"] = (randn(rows, hidden) * channel * 2).to(dtype) if case["residual"] else None
        st["weight"] = (1 + 0.3 * randn(hidden)).to(dtype)
        return st
    if case["op"] == "linear":
        rows, n, k = case["rows"], case["n"], case["k"]
        st["x"], st["x_scale"] = _quantize(randn(rows, k) * torch.exp(0.5 * randn(k)))
        parts = [_quantize_weight(randn(min(16384, n - i), k) * 0.02) for i in range(0, n, 16384)]
        st["w"], st["w_scale"] = torch.cat([p[0] for p in parts]), torch.cat([p[1] for p in parts])
        st["bias"] = randn(n).to(dtype) if case["bias"] else None
        return st
    vocab = case["vocab"]
    if case["op"] == "logprob":
        rows = case["rows"]
        st["tokens"] = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
        st["logits"] = _logits(g, rows, vocab, dtype, st["tokens"], case["temperature"]).requires_grad_(case["grad"])
        # upstream gradients: those of a loss on the log-probabilities with an entropy bonus
        st["d_logp"] = randn(rows) if case["grad"] else None
        st["d_entropy"] = -0.1 * torch.rand(rows, generator=g, device="cuda") if case["grad"] and case["entropy"] \
            else None
        return st
    b, t = case["batch"], case["length"]
    width = t + 1 if case["shifted"] else t  # the logits of position i score token i + 1: the last are cut off
    tokens = torch.randint(0, vocab, (b, width), generator=g, device="cuda")
    logits = _logits(g, b * width, vocab, dtype, tokens.view(-1), case["temperature"])
    seen = _seen_logprobs(logits, tokens.view(-1), case["temperature"]).view(b, width)[:, :t].contiguous()
    st["logits"] = logits.view(b, width, vocab)[:, :t].requires_grad_()
    st["tokens"] = tokens[:, :t].contiguous()
    order = list(range(b))
    random.Random(seed).shuffle(order)
    spread = _lengths(case)
    lens = torch.tensor([spread[i] for i in order], device="cuda")
    st["mask"] = torch.arange(t, device="cuda")[None, :] < lens[:, None]
    st["old"] = seen + 0.15 * randn(b, t)   # the rollout's policy, some updates ago: some ratios are clipped
    st["ref"] = seen + 0.3 * randn(b, t) if case["kl"] else None
    st["adv"] = randn(b, t) if case["per_token"] else randn(b)
    return st


CLIP_LOW, CLIP_HIGH, KL_COEF = 0.2, 0.28, 0.04


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _plain_norm(st):
    x = st["x"].float()
    if st["res"] is not None:
        x = x + st["res"].float()
    rows, hidden = x.shape
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * st["weight"].float()
    groups = -(-hidden // GROUP)
    padded = torch.zeros(rows, groups * GROUP, device=y.device)
    padded[:, :hidden] = y
    blocks = padded.view(rows, groups, GROUP)
    scale = blocks.abs().amax(-1).clamp_min(2.0 ** -100) / E4M3_MAX
    q = (blocks / scale[..., None]).view(rows, -1)[:, :hidden].to(torch.float8_e4m3fn)
    return {"q": q, "scale": scale, "sum": None if st["res"] is None else x.to(st["x"].dtype)}


def _plain_linear(st):
    k, n = st["k"], st["n"]
    x = st["x"].float() * st["x_scale"].repeat_interleave(GROUP, 1)[:, :k]
    w = st["w"].float() * st["w_scale"].repeat_interleave(GROUP, 0)[:n].repeat_interleave(GROUP, 1)[:, :k]
    y = x @ w.t()
    if st["bias"] is not None:
        y = y + st["bias"].float()
    return {"y": y.to(DTYPES[st["dtype"]])}


def _softmax_parts(logits, tokens, temperature):
    z = logits.float() / temperature
    z = z - z.amax(-1, keepdim=True)
    e = torch.exp(z)
    total = e.sum(-1, keepdim=True)
    logp = z.gather(-1, tokens[..., None])[..., 0] - torch.log(total[..., 0])
    return z, e, total, logp


def _plain_logprob(st):
    z, e, total, logp = _softmax_parts(st["logits"], st["tokens"], st["temperature"])
    out = {"logp": logp}
    p = e / total
    if st["entropy"]:
        out["entropy"] = torch.log(total[..., 0]) - (p * z).sum(-1)
    if st["grad"]:
        d = -p * st["d_logp"][:, None]
        d.scatter_add_(1, st["tokens"][:, None], st["d_logp"][:, None])
        if st["entropy"]:
            logs = z - torch.log(total)
            d = d - st["d_entropy"][:, None] * p * (logs + out["entropy"][:, None])
        out["d_logits"] = (d / st["temperature"]).to(st["logits"].dtype)
    return out


def _plain_policy(st):
    z, e, total, logp = _softmax_parts(st["logits"], st["tokens"], st["temperature"])
    del z
    mask = st["mask"].float()
    if st["reduction"] == "token":
        weight = mask / mask.sum().clamp_min(1)
    elif st["reduction"] == "sequence":
        weight = mask / mask.sum(1, keepdim=True).clamp_min(1) / mask.shape[0]
    else:
        weight = mask
    adv = st["adv"] if st["adv"].ndim == 2 else st["adv"][:, None]
    ratio = torch.exp(logp - st["old"])
    free, held = ratio * adv, ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH) * adv
    loss = -torch.minimum(free, held)
    slope = torch.where(free <= held, -free, torch.zeros_like(free))
    count = mask.sum().clamp_min(1)
    kl = torch.zeros_like(count)
    if st["ref"] is not None:
        d = st["ref"] - logp
        k3 = torch.expm1(d) - d
        loss = loss + KL_COEF * k3
        slope = slope - KL_COEF * torch.expm1(d)
        kl = (k3 * mask).sum() / count
    slope = slope * weight / st["temperature"]
    grad = e.mul_(-(slope / total[..., 0])[..., None])
    grad.scatter_add_(-1, st["tokens"][..., None], slope[..., None])
    return {"loss": (loss * weight).sum(), "logp": logp * mask, "kl": kl,
            "clipped": ((held < free) * mask).sum() / count, "d_logits": grad.to(st["logits"].dtype)}


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(st):
    if not own:
        with torch.no_grad():
            return {"norm": _plain_norm, "linear": _plain_linear, "logprob": _plain_logprob,
                    "policy": _plain_policy}[st["op"]](st)
    from grpo_training_engine_b200 import ops

    if st["op"] == "norm":
        q, scale, total = ops.add_rmsnorm_fp8(st["x"], st["weight"], EPS, st["res"])
        return {"q": q, "scale": scale, "sum": total}
    if st["op"] == "linear":
        return {"y": ops.linear_fp8(st["x"], st["x_scale"], st["w"], st["w_scale"], st["bias"],
                                    out_dtype=DTYPES[st["dtype"]])}
    if st["op"] == "logprob":
        got = ops.token_logprobs(st["logits"], st["tokens"], temperature=st["temperature"], entropy=st["entropy"])
        outs = got if st["entropy"] else (got,)
        out = dict(zip(("logp", "entropy"), (o.detach() for o in outs)))
        if st["grad"]:
            ups = (st["d_logp"], st["d_entropy"])[: len(outs)]
            out["d_logits"] = torch.autograd.grad(outs, st["logits"], ups)[0]
        return out
    got = ops.policy_loss(st["logits"], st["tokens"], st["old"], st["adv"], st["mask"], ref_logprobs=st["ref"],
                          kl_coef=KL_COEF if st["kl"] else 0.0, clip_low=CLIP_LOW, clip_high=CLIP_HIGH,
                          temperature=st["temperature"], reduction=st["reduction"])
    return {"loss": got.loss.detach(), "logp": got.logprobs, "kl": got.kl, "clipped": got.clip_fraction,
            "d_logits": torch.autograd.grad(got.loss, st["logits"])[0]}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    size = BYTES[case["dtype"]]
    if case["op"] == "norm":
        rows, hidden = case["rows"], case["hidden"]
        streams = 3 if case["residual"] else 1  # x, and the residual in and out
        return {"bytes": rows * hidden * (streams * size + 1) + rows * -(-hidden // GROUP) * 4 + hidden * size,
                "flops": rows * hidden * 6}
    if case["op"] == "linear":
        rows, n, k = case["rows"], case["n"], case["k"]
        kb, nb = -(-k // GROUP), -(-n // GROUP)
        return {"bytes": rows * k + n * k + 4 * (rows * kb + nb * kb) + rows * n * size + case["bias"] * n * size,
                "flops": 2 * rows * n * k}
    vocab = case["vocab"]
    if case["op"] == "logprob":
        rows = case["rows"]
        return {"bytes": rows * vocab * size * (2 if case["grad"] else 1) + rows * 16,
                "flops": rows * vocab * (10 if case["grad"] else 4)}
    rows, active = case["batch"] * case["length"], sum(_lengths(case))
    # the logits of the response tokens are read, a gradient (zero at the others) is written for all
    return {"bytes": (active + rows) * vocab * size + rows * 25, "flops": active * vocab * 8}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _exact_rows(logits, tokens, temperature):
    """Per row: probabilities, their logarithms, the token's log-probability."""
    logs = torch.log_softmax(logits.double() / temperature, -1)
    return logs, logs.gather(-1, tokens[..., None]).squeeze(-1)


def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "norm":
            s = st["x"].double() + (0 if st["res"] is None else st["res"].double())
            y = st["weight"].double() * s / torch.sqrt(s.pow(2).sum(1, keepdim=True) / s.shape[1] + EPS)
            scale = torch.stack([part.abs().max(1).values.clamp_min(2.0 ** -100) / E4M3_MAX
                                 for part in y.split(GROUP, 1)], 1)
            q = torch.cat([part / scale[:, i:i + 1] for i, part in enumerate(y.split(GROUP, 1))], 1)
            return {"q": q, "scale": scale, "sum": None if st["res"] is None else s}
        if case["op"] == "linear":
            n, k = case["n"], case["k"]
            spread = lambda scale, rows: scale.double().repeat_interleave(GROUP, 1)[:rows, :k]  # noqa: E731
            x = st["x"].double() * spread(st["x_scale"], case["rows"])
            y = torch.empty(case["rows"], n, dtype=torch.float64, device="cuda")
            for i in range(0, n, 8 * GROUP):
                w = st["w"][i:i + 8 * GROUP].double()
                scale = st["w_scale"][i // GROUP:i // GROUP + 8].repeat_interleave(GROUP, 0)
                y[:, i:i + 8 * GROUP] = x @ (w * spread(scale, w.shape[0])).t()
            return {"y": y if st["bias"] is None else y + st["bias"].double()}
        vocab, t = case["vocab"], case["temperature"]
        if case["op"] == "logprob":
            rows = case["rows"]
            out = {"logp": torch.empty(rows, dtype=torch.float64, device="cuda")}
            if case["entropy"]:
                out["entropy"] = torch.empty(rows, dtype=torch.float64, device="cuda")
            if case["grad"]:
                out["d_logits"] = torch.empty(rows, vocab, dtype=torch.float64, device="cuda")
            step = max(1, (1 << 26) // vocab)
            for r in range(0, rows, step):
                cut = slice(r, r + step)
                logs, out["logp"][cut] = _exact_rows(st["logits"][cut], st["tokens"][cut], t)
                p = logs.exp()
                if case["entropy"]:
                    h = -(p * logs).nan_to_num(0).sum(1)
                    out["entropy"][cut] = h
                if case["grad"]:
                    hot = torch.zeros_like(p).scatter_(1, st["tokens"][cut, None], 1.0)
                    d = st["d_logp"][cut, None].double() * (hot - p)
                    if case["entropy"]:
                        d -= st["d_entropy"][cut, None].double() * p * (logs + h[:, None])
                    out["d_logits"][cut] = d / t
            return out
        b, length = case["batch"], case["length"]
        mask, adv = st["mask"], st["adv"].double()
        adv = adv[:, None].expand(b, length) if adv.ndim == 1 else adv
        lens = mask.sum(1).double()
        share = {"token": 1 / lens.sum(), "sum": torch.ones(()).cuda().double(),
                 "sequence": (1 / (b * lens))[:, None]}[case["reduction"]]
        share = share * mask
        out = {"loss": 0.0, "logp": torch.zeros(b, length, dtype=torch.float64, device="cuda"), "kl": 0.0,
               "clipped": 0.0, "d_logits": torch.zeros(b, length, vocab, dtype=torch.float64, device="cuda")}
        step = max(1, (1 << 26) // vocab)
        for i in range(b):
            for j in range(0, int(lens[i]), step):
                cut = slice(j, min(j + step, int(lens[i])))
                logs, lp = _exact_rows(st["logits"][i, cut], st["tokens"][i, cut], t)
                ratio = (lp - st["old"][i, cut].double()).exp()
                a = adv[i, cut]
                best = torch.where(a > 0, 1.0 + CLIP_HIGH, 1.0 - CLIP_LOW)
                clipped = torch.where(a > 0, ratio > best, ratio < best) & (a != 0)
                value = -torch.where(clipped, best, ratio) * a
                slope = -torch.where(clipped, 0.0, ratio) * a
                if case["kl"]:
                    gap = st["ref"][i, cut].double() - lp
                    value = value + KL_COEF * (gap.exp() - gap - 1)
                    slope = slope + KL_COEF * (1 - gap.exp())
                    out["kl"] = out["kl"] + (gap.exp() - gap - 1).sum() / lens.sum()
                out["clipped"] = out["clipped"] + clipped.sum() / lens.sum()
                out["loss"] = out["loss"] + (value * share[i, cut]).sum()
                out["logp"][i, cut] = lp
                d = -logs.exp_() * (slope * share[i, cut])[:, None]
                d.scatter_add_(1, st["tokens"][i, cut, None], (slope * share[i, cut])[:, None])
                out["d_logits"][i, cut] = d / t
        return {name: v if torch.is_tensor(v) else torch.tensor(v, dtype=torch.float64) for name, v in out.items()}
