"""What the 8-bit and policy entry points refuse, in the C ABI and on tensors; nothing reaches a GPU."""

from __future__ import annotations

import ctypes as C

import pytest
import torch

from grpo_training_engine_b200 import _lib, ops

A, B, D, E = (C.c_void_p(1 << s) for s in (20, 21, 22, 23))  # aligned addresses that nothing reads
OFF = C.c_void_p((1 << 20) + 1)
BF16, F32 = _lib.DTYPE_BF16, _lib.DTYPE_F32


def test_add_rmsnorm_fp8_refuses():
    lib = _lib.load()

    def call(x=A, res=None, w=B, total=None, q=D, scales=E, rows=4, hidden=256, dtype=BF16):
        return lib.pkv_add_rmsnorm_fp8(x, res, w, total, q, scales, rows, hidden, hidden, hidden, hidden, hidden, 2,
                                       1e-6, dtype, None)

    assert call(rows=0) == _lib.OK
    assert call(dtype=7) == _lib.ERR_UNSUPPORTED
    assert call(rows=-1) == _lib.ERR_INVALID_ARG
    assert call(hidden=0) == _lib.ERR_INVALID_ARG
    for name in ("x", "w", "q", "scales"):
        assert call(**{name: None}) == _lib.ERR_INVALID_ARG, name
    assert call(res=A) == _lib.ERR_INVALID_ARG            # a residual without a place for the sum
    assert call(total=A) == _lib.ERR_INVALID_ARG          # and the other way round
    assert call(x=OFF) == _lib.ERR_ALIGNMENT
    assert "pkv_add_rmsnorm_fp8" in _lib.last_detail()


def test_quantize_fp8_refuses():
    lib = _lib.load()

    def call(x=A, q=B, scales=D, rows=4, cols=256, block=1, dtype=BF16):
        return lib.pkv_quantize_fp8(x, q, scales, rows, cols, block, cols, cols, 2, dtype, None)

    assert call(rows=0) == _lib.OK
    assert call(dtype=-1) == _lib.ERR_UNSUPPORTED
    assert call(block=64) == _lib.ERR_INVALID_ARG
    assert call(cols=0) == _lib.ERR_INVALID_ARG
    assert call(q=None) == _lib.ERR_INVALID_ARG
    assert call(x=OFF) == _lib.ERR_ALIGNMENT


def test_linear_fp8_refuses():
    lib = _lib.load()

    def call(x=A, xs=B, w=D, ws=E, bias=None, out=A, rows=40, n=256, k=256, x_stride=256, xs_stride=2, w_stride=256,
             ws_stride=2, out_stride=256, dtype=BF16):
        return lib.pkv_linear_fp8(x, xs, w, ws, bias, out, rows, n, k, x_stride, xs_stride, w_stride, ws_stride,
                                  out_stride, dtype, None, None)

    assert call(rows=0) == _lib.OK
    assert call(dtype=F32) == _lib.ERR_UNSUPPORTED
    assert call(rows=-1) == _lib.ERR_INVALID_ARG
    assert call(n=0) == _lib.ERR_INVALID_ARG
    assert call(k=0) == _lib.ERR_INVALID_ARG
    for name in ("x", "xs", "w", "ws", "out"):
        assert call(**{name: None}) == _lib.ERR_INVALID_ARG, name
    assert call(xs_stride=1) == _lib.ERR_INVALID_ARG
    assert call(ws_stride=1) == _lib.ERR_INVALID_ARG
    assert call(out_stride=255) == _lib.ERR_INVALID_ARG
    assert call(x=C.c_void_p((1 << 20) + 8)) == _lib.ERR_ALIGNMENT
    assert call(x_stride=264) == _lib.ERR_ALIGNMENT
    assert call(w_stride=240) == _lib.ERR_ALIGNMENT       # below k
    # every check passes: only the tensor-map encoder, which needs the driver, is left
    assert call() == _lib.ERR_TENSOR_MAP


def test_token_logprobs_refuses():
    lib = _lib.load()

    def call(logits=A, dtype=BF16, tokens=B, rows=4, vocab=100, inner=4, temperature=1.0, out=D):
        return lib.pkv_token_logprobs(logits, dtype, tokens, rows, vocab, inner, 0, vocab, temperature, out, None, None,
                                      None, None)

    assert call(rows=0) == _lib.OK
    assert call(dtype=5) == _lib.ERR_UNSUPPORTED
    for bad in (dict(vocab=0), dict(inner=0), dict(temperature=0.0), dict(temperature=float("nan")), dict(rows=-1),
                dict(logits=None), dict(tokens=None), dict(out=None), dict(logits=OFF), dict(rows=1 << 33)):
        assert call(**bad) == _lib.ERR_INVALID_ARG, bad
    grad = lib.pkv_token_logprobs_grad
    assert grad(A, BF16, B, 4, 100, 4, 0, 100, 1.0, None, None, D, None, E, None) == _lib.ERR_INVALID_ARG  # no stats
    assert grad(A, BF16, B, 4, 100, 4, 0, 100, 1.0, D, None, None, D, E, None) == _lib.ERR_INVALID_ARG  # no entropies


def test_policy_loss_refuses():
    lib = _lib.load()
    need = lib.pkv_policy_loss_workspace_size(2, 3)
    assert need > 0 and lib.pkv_policy_loss_workspace_size(1 << 20, 1 << 20) == 0

    def call(logits=A, dtype=BF16, tokens=B, old=D, adv=E, batch=2, length=3, vocab=100, temperature=1.0, low=0.2,
             high=0.2, reduction=0, out=A, logp=B, ws=D, ws_bytes=need):
        return lib.pkv_policy_loss(logits, dtype, tokens, old, None, adv, 1, 0, None, batch, length, vocab, 300, 100,
                                   temperature, low, high, 0.0, reduction, out, logp, None, ws, ws_bytes, None, None)

    assert call(dtype=5) == _lib.ERR_UNSUPPORTED
    for bad in (dict(batch=-1), dict(vocab=0), dict(temperature=-1.0), dict(low=-0.1), dict(high=float("nan")),
                dict(reduction=3), dict(tokens=None), dict(old=None), dict(adv=None), dict(out=None), dict(logp=None),
                dict(logits=None), dict(batch=1 << 30, length=1 << 30)):
        assert call(**bad) == _lib.ERR_INVALID_ARG, bad
    assert call(ws=None) == _lib.ERR_WORKSPACE
    assert call(ws_bytes=need - 1) == _lib.ERR_WORKSPACE
    assert call(ws=C.c_void_p((1 << 20) + 4)) == _lib.ERR_WORKSPACE
    assert lib.pkv_scale_grad(None, 5, BF16, None, None) == _lib.ERR_INVALID_ARG
    assert lib.pkv_scale_grad(None, 0, BF16, None, None) == _lib.OK


def test_tensors_are_checked():
    x = torch.zeros(4, 256, dtype=torch.bfloat16)
    w = torch.ones(256, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.add_rmsnorm_fp8(x, w, 1e-6)
    with pytest.raises(ValueError, match="CUDA"):
        ops.quantize_fp8(x)
    for bad, match in (((x[0], w), "rows, hidden"), ((x.t(), w), "contiguous rows"), ((x, w[:5]), "weight"),
                       ((x, w.float()), "weight"), ((x[:, :0], w[:0]), "column")):
        with pytest.raises(ValueError, match=match):
            ops.add_rmsnorm_fp8(*bad, 1e-6)
    with pytest.raises(ValueError, match="residual"):
        ops.add_rmsnorm_fp8(x, w, 1e-6, x[:2])
    with pytest.raises(ValueError, match="must be float32, bfloat16 or float16"):
        ops.add_rmsnorm_fp8(x.double(), w.double(), 1e-6)

    q = torch.zeros(4, 256).to(torch.float8_e4m3fn)
    wq = torch.zeros(300, 256).to(torch.float8_e4m3fn)
    xs, ws = torch.ones(4, 2), torch.ones(3, 2)
    for args, kw, match in (((x, xs, wq, ws), {}, "float8"), ((q[:, :128], xs, wq, ws), {}, "one K"),
                            ((q, xs[:, :1], wq, ws), {}, "x_scale"), ((q, xs, wq, ws[:2]), {}, "weight_scale"),
                            ((q, xs.double(), wq, ws), {}, "fp32"),
                            ((q, xs, wq, ws), {"out_dtype": torch.float32}, "out_dtype"),
                            ((q, xs, wq, ws, torch.zeros(300)), {}, "bias"), ((q, xs, wq, ws), {}, "CUDA")):
        with pytest.raises(ValueError, match=match):
            ops.linear_fp8(*args, **kw)

    logits, tokens = torch.zeros(2, 3, 10), torch.zeros(2, 3, dtype=torch.int64)
    for args, kw, match in (((logits[0, 0], tokens), {}, "logits must be"), ((logits, tokens[:1]), {}, "tokens must"),
                            ((logits, tokens.float()), {}, "tokens must"), ((logits[..., :0], tokens), {}, "logits"),
                            ((logits, tokens), {"temperature": 0.0}, "temperature"), ((logits, tokens), {}, "CUDA"),
                            ((logits.int(), tokens), {}, "float32, bfloat16")):
        with pytest.raises(ValueError, match=match):
            ops.token_logprobs(*args, **kw)

    old, adv = torch.zeros(2, 3), torch.zeros(2)
    ok = (logits, tokens, old, adv)
    for args, kw, match in (((logits[0], tokens[0], old[0], adv), {}, "logits must be"),
                            ((logits, tokens, old[:1], adv), {}, "old_logprobs"),
                            ((logits, tokens, old, adv[:1]), {}, "advantages"),
                            (ok + (old > 1,), {"ref_logprobs": old[:, :1]}, "ref_logprobs"),
                            (ok + ((old > 1)[:, :2],), {}, "mask"), (ok + (old,), {}, "mask must be bool"),
                            (ok, {"reduction": "mean"}, "reduction"), (ok, {"clip_low": -1.0}, "clip_low"),
                            (ok, {"temperature": -1.0}, "temperature"), (ok, {}, "CUDA")):
        with pytest.raises(ValueError, match=match):
            ops.policy_loss(*args, **kw)


def test_package_exports():
    import grpo_training_engine_b200 as pkg

    for name in ("add_rmsnorm_fp8", "quantize_fp8", "quantize_fp8_weight", "linear_fp8", "token_logprobs",
                 "policy_loss", "PolicyLoss"):
        assert name in pkg.__all__ and getattr(pkg, name) is getattr(ops, name)
