"""8-bit projections at the sizes that choose each kernel and each of its edges."""

from __future__ import annotations

import pytest
import torch

from test_gpu_fp8 import _check_linear, _operands

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from grpo_training_engine_b200 import ops


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("rows,n,k", [
    # up to 16 rows on warp-level MMAs: one warp, four and eight per 16 rows of W (n from 37,873 and 9,457 on), one
    # and two groups of 8 activation rows, short last blocks of k, warps without a block, one block on an SM
    (1, 151936, 1536), (5, 37889, 1040), (16, 37889, 1536), (16, 9473, 1536), (8, 9475, 400), (3, 1001, 1104),
    (16, 200, 400), (9, 33, 272), (8, 2048, 18944),
    # wide matrices: 256-column tiles, by TMA stores and by element
    (37, 151936, 1536), (128, 76000, 272), (100, 80001, 400),
    # pairs: the second CTA's rows beyond the last, short last blocks of k, both ways to store
    (1281, 6001, 2064), (1400, 6001, 648), (1400, 6008, 648), (300, 5000, 1000), (513, 12345, 130),
    # k split over a cluster, more tiles than SMs without a split
    (20, 1544, 8976), (129, 1536, 1537), (64, 20000, 300)])
def test_linear_fp8_sizes(rows, n, k, out_dtype):
    x, xs, w, ws = _operands(rows, n, k, rows + n + k)
    bias = torch.randn(n, device="cuda").to(out_dtype)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = ops.linear_fp8(x, xs, w, ws, bias, out_dtype=out_dtype, status=status)
    assert int(status) == 0
    _check_linear(out, x, xs, w, ws, bias)
    assert torch.equal(out, ops.linear_fp8(x, xs, w, ws, bias, out_dtype=out_dtype))
    # into rows of a wider tensor, whose other elements stay
    buf = torch.full((rows + 1, n + 24), 7.0, device="cuda", dtype=out_dtype)
    ops.linear_fp8(x, xs, w, ws, bias, out=buf[:rows, 8:n + 8])
    assert torch.equal(buf[:rows, 8:n + 8], out)
    assert torch.all(buf[:, :8] == 7) and torch.all(buf[:, n + 8:] == 7) and torch.all(buf[rows] == 7)
