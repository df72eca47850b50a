"""What the scaled policy gradient's C entry point refuses; nothing reaches a GPU."""

from __future__ import annotations

import ctypes as C

from grpo_training_engine_b200 import _lib

A, B, D = (C.c_void_p(1 << s) for s in (20, 21, 22))  # aligned addresses that nothing reads


def test_policy_loss_grad_refuses():
    lib = _lib.load()
    need = lib.pkv_policy_loss_workspace_size(2, 3)

    def call(logits=A, dtype=_lib.DTYPE_BF16, batch=2, length=3, vocab=100, temperature=1.0, ws=D, ws_bytes=need,
             upstream=B, grad=A):
        return lib.pkv_policy_loss_grad(logits, dtype, batch, length, vocab, 300, 100, temperature, ws, ws_bytes,
                                        upstream, grad, None)

    assert call(batch=0) == _lib.OK
    assert call(dtype=5) == _lib.ERR_UNSUPPORTED
    for bad in (dict(batch=-1), dict(length=-1), dict(vocab=0), dict(temperature=0.0), dict(logits=None),
                dict(upstream=None), dict(grad=None), dict(batch=1 << 30, length=1 << 30),
                dict(upstream=C.c_void_p((1 << 20) + 2)), dict(grad=C.c_void_p((1 << 20) + 1))):
        assert call(**bad) == _lib.ERR_INVALID_ARG, bad
    assert call(ws=None) == _lib.ERR_WORKSPACE
    assert call(ws_bytes=need - 1) == _lib.ERR_WORKSPACE
    assert call(ws=C.c_void_p((1 << 20) + 8)) == _lib.ERR_WORKSPACE
