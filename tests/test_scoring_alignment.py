"""The 8-bit and policy entry points refuse every pointer that is not aligned to its elements; nothing reaches a GPU."""

from __future__ import annotations

import ctypes as C

import pytest

from grpo_training_engine_b200 import _lib

BASE = 1 << 20  # an aligned address that nothing reads
BF16, F32 = _lib.DTYPE_BF16, _lib.DTYPE_F32


def _ptr(off: int = 0) -> C.c_void_p:
    return C.c_void_p(BASE + off)


def _calls():
    lib = _lib.load()
    need = lib.pkv_policy_loss_workspace_size(2, 3)

    def norm(scales=0, total=0):
        return lib.pkv_add_rmsnorm_fp8(_ptr(), _ptr(), _ptr(), _ptr(total), _ptr(), _ptr(scales), 4, 256, 256, 256, 256,
                                       256, 2, 1e-6, BF16, None)

    def quantize(scales=0):
        return lib.pkv_quantize_fp8(_ptr(), _ptr(), _ptr(scales), 4, 256, 1, 256, 256, 2, BF16, None)

    def linear(status=0):
        return lib.pkv_linear_fp8(_ptr(), _ptr(), _ptr(), _ptr(), None, _ptr(), 40, 256, 256, 256, 2, 256, 2, 256, BF16,
                                  _ptr(status), None)

    def logprobs(tokens=0, out=0, entropy=0, stats=0, status=0):
        return lib.pkv_token_logprobs(_ptr(), BF16, _ptr(tokens), 4, 100, 4, 0, 100, 1.0, _ptr(out), _ptr(entropy),
                                      _ptr(stats), _ptr(status), None)

    def logprobs_grad(tokens=0, stats=0, entropy=0, d_logp=0, d_entropy=0):
        return lib.pkv_token_logprobs_grad(_ptr(), BF16, _ptr(tokens), 4, 100, 4, 0, 100, 1.0, _ptr(stats),
                                           _ptr(entropy), _ptr(d_logp), _ptr(d_entropy), _ptr(), None)

    def policy(tokens=0, old=0, ref=0, adv=0, out=0, logp=0, status=0):
        return lib.pkv_policy_loss(_ptr(), BF16, _ptr(tokens), _ptr(old), _ptr(ref), _ptr(adv), 1, 0, None, 2, 3, 100,
                                   300, 100, 1.0, 0.2, 0.2, 0.0, 0, _ptr(out), _ptr(logp), None, _ptr(), need,
                                   _ptr(status), None)

    def scale(grad=0, upstream=0):
        return lib.pkv_scale_grad(_ptr(grad), 5, F32, _ptr(upstream), None)

    return {f.__name__: f for f in (norm, quantize, linear, logprobs, logprobs_grad, policy, scale)}


CASES = [(name, arg, off) for name, args in {
    "norm": {"scales": 2, "total": 1}, "quantize": {"scales": 2}, "linear": {"status": 2},
    "logprobs": {"tokens": 4, "out": 2, "entropy": 2, "stats": 4, "status": 2},
    "logprobs_grad": {"tokens": 4, "stats": 4, "entropy": 2, "d_logp": 2, "d_entropy": 2},
    "policy": {"tokens": 4, "old": 2, "ref": 2, "adv": 2, "out": 2, "logp": 2, "status": 2},
    "scale": {"grad": 2, "upstream": 2}}.items() for arg, off in args.items()]


@pytest.mark.parametrize("name,arg,off", CASES)
def test_misaligned_pointers_are_refused(name, arg, off):
    assert _calls()[name](**{arg: off}) in (_lib.ERR_ALIGNMENT, _lib.ERR_INVALID_ARG)
