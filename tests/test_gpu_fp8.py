"""8-bit norm, quantisers and projection against their definitions in 64 bits."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from grpo_training_engine_b200 import ops

GROUP, TOP, FLOOR = 128, 448.0, 2.0 ** -100
# half a step of each type, relative to a value of p bits (2^-p), and half the smallest step
HALF = {torch.bfloat16: (2.0 ** -8, 2.0 ** -134), torch.float16: (2.0 ** -11, 2.0 ** -25),
        torch.float32: (2.0 ** -24, 2.0 ** -150)}


def _groups(v: torch.Tensor) -> torch.Tensor:
    rows, k = v.shape
    return torch.nn.functional.pad(v, (0, -k % GROUP)).view(rows, -1, GROUP)


def _spread(scale: torch.Tensor, k: int) -> torch.Tensor:
    return scale.double().repeat_interleave(GROUP, 1)[:, :k]


def _check_q(q, scale, y, slack):
    """q * scale against y (64 bits): the scale, then each value to half a step of the 8-bit type."""
    want = _groups(y).abs().amax(-1).clamp_min(FLOOR) / TOP
    assert scale.dtype == torch.float32 and scale.shape == want.shape
    assert torch.all((scale.double() - want).abs() <= slack * want)
    s = _spread(scale, y.shape[1])
    # 3 mantissa bits: half a step is 2^-4 of a normal value, 2^-10 of the scale below 2^-6
    assert torch.all((q.double() * s - y).abs() <= (2.0 ** -4 + 2 * slack) * y.abs() + 2.0 ** -10 * s)


# fp32 sums of up to 8192 squares by 256 or more threads: at most 32 + 13 roundings of 2^-24, halved by the
# root, and about ten more in rsqrt, products and quotient
SLACK = 4e-6


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("rows,hidden", [(1, 1), (1, 1536), (3, 127), (2, 128), (5, 129), (7, 1000), (64, 3584),
                                         (33, 1001), (4, 8192), (2, 8200), (1, 20001), (300, 104)])
def test_add_rmsnorm_fp8(rows, hidden, residual, dtype):
    g = torch.Generator(device="cuda").manual_seed(rows * 100003 + hidden)
    wide = torch.randn(rows, hidden + 8, device="cuda", generator=g) * torch.exp(torch.randn(hidden + 8, device="cuda"))
    x = wide.to(dtype)[:, :hidden]
    r = torch.randn(rows, hidden, device="cuda", generator=g).to(dtype) if residual else None
    w = (1 + 0.3 * torch.randn(hidden, device="cuda", generator=g)).to(dtype)
    q, scale, total = ops.add_rmsnorm_fp8(x, w, 1e-6, r)
    assert q.dtype == torch.float8_e4m3fn and q.shape == x.shape and q.stride(0) % 16 == 0
    s = x.double() + (0 if r is None else r.double())
    if r is None:
        assert total is None
    else:
        rel, tiny = HALF[dtype]
        # fp32 + fp32 rounds once to fp32 and once more to the type
        assert total.dtype == dtype
        assert torch.all((total.double() - s).abs() <= (rel * 1.001 + 2.0 ** -24) * s.abs() + tiny)
    y = s * torch.rsqrt(s.pow(2).mean(-1, keepdim=True) + 1e-6) * w.double()
    _check_q(q, scale, y, SLACK * (1 + hidden / 8192))


def test_add_rmsnorm_fp8_zero_group_row_and_nan():
    x = torch.randn(4, 300, device="cuda")
    x[0, 128:256] = 0          # a group of zeros
    x[1] = 0                   # a row of zeros
    x[2, 5] = float("nan")     # a NaN reaches its whole row through the mean
    q, scale, _ = ops.add_rmsnorm_fp8(x, torch.ones(300, device="cuda"), 1e-6)
    assert torch.all(q[0, 128:256].float() == 0) and torch.all(q[1].float() == 0)
    assert torch.all(scale[:2] > 0) and torch.isfinite(scale[:2]).all()
    assert torch.isnan(q[2].float()).all() and torch.isnan(scale[2]).all()
    assert torch.isfinite(q[3].float()).all()


def test_add_rmsnorm_fp8_empty_and_other_stream():
    w = torch.ones(256, device="cuda", dtype=torch.bfloat16)
    q, scale, total = ops.add_rmsnorm_fp8(torch.empty(0, 256, device="cuda", dtype=torch.bfloat16), w, 1e-6)
    assert q.shape == (0, 256) and scale.shape == (0, 2) and total is None
    x = torch.randn(64, 256, device="cuda").to(torch.bfloat16)
    want = ops.add_rmsnorm_fp8(x, w, 1e-6)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = ops.add_rmsnorm_fp8(x, w, 1e-6)
    st.synchronize()
    assert torch.equal(got[0].view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(got[1], want[1])


def test_add_rmsnorm_fp8_offsets_past_32_bits():
    rows, hidden = 600_000, 3584
    x = torch.zeros(rows, hidden, device="cuda", dtype=torch.bfloat16)
    x[-2:] = torch.randn(2, hidden, device="cuda").to(torch.bfloat16)
    w = torch.ones(hidden, device="cuda", dtype=torch.bfloat16)
    q, scale, _ = ops.add_rmsnorm_fp8(x, w, 1e-6)
    y = x[-2:].double()
    y = y * torch.rsqrt(y.pow(2).mean(-1, keepdim=True) + 1e-6)
    _check_q(q[-2:], scale[-2:], y, SLACK)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 128), (5, 129), (130, 257), (300, 1000)])
def test_quantizers(rows, cols, dtype):
    x = (torch.randn(rows, cols + 3, device="cuda") * 5).to(dtype)[:, 1:cols + 1]
    q, scale = ops.quantize_fp8(x)
    _check_q(q, scale, x.double(), 4e-7)
    q, scale = ops.quantize_fp8_weight(x)
    assert scale.shape == (-(-rows // GROUP), -(-cols // GROUP)) and q.stride(0) % 16 == 0
    for i in range(scale.shape[0]):
        block = x[i * GROUP:(i + 1) * GROUP].double()
        want = _groups(block).abs().amax((0, 2)).clamp_min(FLOOR) / TOP
        assert torch.all((scale[i].double() - want).abs() <= 4e-7 * want)
        s = _spread(scale[i:i + 1], cols)
        err = (q[i * GROUP:(i + 1) * GROUP].double() * s - block).abs()
        assert torch.all(err <= (2.0 ** -4 + 1e-6) * block.abs() + 2.0 ** -10 * s)


def _operands(rows, n, k, seed, wide=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, k, device="cuda", generator=g) * torch.exp(wide * torch.randn(k, device="cuda", generator=g))
    w = torch.randn(n, k, device="cuda", generator=g) * 0.05
    return (*ops.quantize_fp8(x), *ops.quantize_fp8_weight(w))


def _check_linear(out, x, xs, w, ws, bias=None):
    rows, k = x.shape
    n, kb = w.shape[0], -(-k // GROUP)
    xd = x.double() * _spread(xs, k)
    wd = w.double() * _spread(ws, k).repeat_interleave(GROUP, 0)[:n]
    y = xd @ wd.t()
    # a block of 128 products takes at most 16 roundings of 2^-23 inside the tensor core (4 MMAs of 32), the
    # blocks are added with one each, and a split of k adds 8
    slack = (16 + kb + 8) * 2.0 ** -23 * (xd.abs() @ wd.abs().t())
    if bias is not None:
        y = y + bias.double()
        slack = slack + 2.0 ** -24 * y.abs()
    rel, tiny = HALF[out.dtype]
    assert out.shape == (rows, n)
    assert torch.all((out.double() - y).abs() <= rel * 1.01 * y.abs() + tiny + 1.01 * slack)


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("rows,n,k", [(1, 1, 1), (1, 2048, 1536), (1, 64, 16), (7, 130, 129), (16, 128, 128),
                                      (17, 1000, 1000), (37, 5001, 1536), (64, 1536, 8960), (128, 1536, 8960),
                                      (129, 257, 384), (200, 8960, 1536), (257, 3584, 18944), (300, 1003, 2064),
                                      (1024, 2048, 1536), (1500, 5000, 640)])
def test_linear_fp8(rows, n, k, out_dtype):
    x, xs, w, ws = _operands(rows, n, k, rows + n + k)
    bias = torch.randn(n, device="cuda").to(out_dtype) if n % 2 else None
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = ops.linear_fp8(x, xs, w, ws, bias, out_dtype=out_dtype, status=status)
    assert out.dtype == out_dtype and int(status) == 0
    _check_linear(out, x, xs, w, ws, bias)
    # the same bits again: no result depends on which block or split finishes first
    assert torch.equal(out, ops.linear_fp8(x, xs, w, ws, bias, out_dtype=out_dtype))


def test_linear_fp8_strided_out_and_scales():
    x, xs, w, ws = _operands(50, 200, 300, 5)
    xs2 = torch.full((50, 7), float("nan"), device="cuda")
    xs2[:, 2:5] = xs
    buf = torch.full((50, 333), 7.0, device="cuda", dtype=torch.bfloat16)
    out = ops.linear_fp8(x, xs2[:, 2:5], w, ws, out=buf[:, 101:301])
    assert out.data_ptr() == buf[:, 101:].data_ptr()
    _check_linear(out, x, xs, w, ws)
    assert torch.all(buf[:, :101] == 7) and torch.all(buf[:, 301:] == 7)


def test_linear_fp8_rows_do_not_mix():
    """A row's NaN (and a row of zeros) stays in that row; rows past the last one are not read as values."""
    x, xs, w, ws = _operands(5, 256, 256, 9)
    xs[2, 1] = float("nan")
    x[3] = 0
    out = ops.linear_fp8(x, xs, w, ws)
    assert torch.isnan(out[2].float()).all() and torch.all(out[3] == 0)
    keep = [0, 1, 4]
    _check_linear(out[keep], x[keep], xs[keep], w, ws)


def test_linear_fp8_each_block_has_its_scales():
    """One block of k at a time is not zero: every (row, k) and (n, k) scale is the one that is used."""
    rows, n, k = 140, 300, 520
    x, xs, w, ws = _operands(rows, n, k, 11)
    xs = torch.exp(torch.randn(xs.shape, device="cuda") * 3)
    ws = torch.exp(torch.randn(ws.shape, device="cuda") * 3)
    for b in range(xs.shape[1]):
        one = torch.zeros(rows, 528, device="cuda").to(x.dtype)[:, :k]  # rows on 16-byte boundaries
        one[:, b * GROUP:(b + 1) * GROUP] = x[:, b * GROUP:(b + 1) * GROUP]
        _check_linear(ops.linear_fp8(one, xs, w, ws), one, xs, w, ws)


def test_linear_fp8_empty_and_other_stream():
    x, xs, w, ws = _operands(40, 2048, 1536, 3)
    assert ops.linear_fp8(x[:0], xs[:0], w, ws).shape == (0, 2048)
    want = ops.linear_fp8(x, xs, w, ws)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = ops.linear_fp8(x, xs, w, ws)
    st.synchronize()
    assert torch.equal(got, want)


def test_linear_fp8_offsets_past_32_bits():
    rows, n, k = 16384, 151936, 128
    x, xs, w, ws = _operands(rows, n, k, 21)
    out = ops.linear_fp8(x, xs, w, ws)
    for cut in (slice(0, 3), slice(rows - 3, rows)):
        _check_linear(out[cut], x[cut], xs[cut], w, ws)


def test_norm_then_linear_is_the_projection():
    """The two together against the 64-bit norm and product: the 8-bit rounding of both operands is all."""
    rows, hidden, n = 48, 1536, 640
    x = torch.randn(rows, hidden, device="cuda").to(torch.bfloat16)
    w = (torch.randn(n, hidden, device="cuda") * 0.02).to(torch.bfloat16)
    norm = torch.ones(hidden, device="cuda", dtype=torch.bfloat16)
    q, scale, _ = ops.add_rmsnorm_fp8(x, norm, 1e-6)
    out = ops.linear_fp8(q, scale, *ops.quantize_fp8_weight(w))
    y = x.double() * torch.rsqrt(x.double().pow(2).mean(-1, keepdim=True) + 1e-6) @ w.double().t()
    # independent roundings of up to 2^-4 (about 2^-4 / sqrt(3) / 1.5 each in the mean square) on both sides
    assert float((out.double() - y).norm() / y.norm()) < 0.06
