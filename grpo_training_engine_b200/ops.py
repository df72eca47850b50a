"""Kernel-level paged-KV operations on torch tensors, calling libpkv.so.

Each function validates its tensors, passes raw device pointers, element
strides and the current CUDA stream through the C ABI (include/pkv.h) and
returns without synchronising. There is no non-CUDA implementation: CPU
tensors are rejected with the reference's ValueError, and a missing
libpkv.so raises ImportError.

Reference correspondence (src/triton_kernels/paged_kv.py):
  paged_kv_append        _paged_kv_update_kernel launch   :253-319, :730-752
  paged_attention_decode _paged_attention_decode_kernel   :63-251,  :754-783
  paged_kv_append_prompt _prefill_paged_cache scatter     :572-586
  gather_kv              the kernel's block-table addressing written densely :98-131
"""

from __future__ import annotations

import contextlib
import functools
import math
from dataclasses import dataclass
from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad

from . import _lib


@functools.lru_cache(maxsize=512)
def _strides(values: tuple) -> object:
    """ctypes int64 array of a stride tuple, built once per distinct tuple (the
    library only reads it; the arrays are kept alive by the cache)."""
    return _lib.i64_array(values)


_NULL_CTX = contextlib.nullcontext()


def _device_ctx(dev: torch.device):
    """torch.cuda.device(dev) only when dev is not already the current device."""
    return _NULL_CTX if dev.index == torch.cuda.current_device() else torch.cuda.device(dev)

_DTYPES = {
    torch.float32: _lib.DTYPE_F32,
    torch.bfloat16: _lib.DTYPE_BF16,
    torch.float16: _lib.DTYPE_F16,
}


def _dtype_code(t: torch.Tensor, what: str) -> int:
    try:
        return _DTYPES[t.dtype]
    except KeyError:
        raise ValueError(f"{what} must be float32, bfloat16 or float16, got {t.dtype}.") from None


def _require_cuda(*tensors: Optional[torch.Tensor]) -> torch.device:
    dev, index = None, -1
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise ValueError("inputs and caches must be on CUDA device.")
        if dev is None:
            dev, index = t.device, t.get_device()
        elif t.get_device() != index:
            raise ValueError(f"all tensors must be on one device, got {dev} and {t.device}.")
    assert dev is not None
    return dev


def _as_i32(t: torch.Tensor) -> torch.Tensor:
    return t if t.dtype == torch.int32 else t.to(torch.int32)


def _stream(dev: torch.device) -> int:
    # the handle alone: a Stream object per call takes 2 us of host time
    return torch._C._cuda_getCurrentRawStream(dev.index)


def _check_cache_pair(k_cache: torch.Tensor, v_cache: torch.Tensor) -> None:
    if k_cache.ndim != 4 or v_cache.ndim != 4:
        raise ValueError("k_cache/v_cache must be [num_blocks, heads, block, head_dim].")
    if k_cache.shape != v_cache.shape:
        raise ValueError("k_cache and v_cache must have identical shapes.")
    if k_cache.dtype != v_cache.dtype:
        raise ValueError("k_cache and v_cache must have the same dtype.")
    if k_cache.stride() != v_cache.stride():
        raise ValueError("k_cache and v_cache must have identical strides.")


def _check_tables(block_tables: torch.Tensor, context_lens: torch.Tensor, batch: int) -> None:
    if block_tables.ndim != 2:
        raise ValueError(f"block_tables must be [batch, max_blocks], got {tuple(block_tables.shape)}.")
    if context_lens.ndim != 1:
        raise ValueError(f"context_lens must be [batch], got {tuple(context_lens.shape)}.")
    if block_tables.shape[0] != batch:
        raise ValueError("block_tables batch dimension must match input_ids batch.")
    if context_lens.shape[0] != batch:
        raise ValueError("context_lens batch dimension must match input_ids batch.")


def _status_ptr(status: Optional[torch.Tensor]) -> Optional[int]:
    if status is None:
        return None
    if status.dtype != torch.int32 or status.numel() < 1 or not status.is_cuda:
        raise ValueError("status must be a CUDA int32 tensor with at least one element.")
    return status.data_ptr()


# ---------------------------------------------------------------------------
# append / prompt append / gather
# ---------------------------------------------------------------------------
def paged_kv_append(
    k_new: torch.Tensor,
    v_new: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_tables: torch.Tensor,
    context_lens: torch.Tensor,
    *,
    status: Optional[torch.Tensor] = None,
) -> None:
    """Write k_new/v_new [B, H, D] at position context_lens[b] (pre-append) in place.

    Same slot rule as the reference update kernel (paged_kv.py:277-284); the
    payload is copied bit for bit.
    """
    _check_cache_pair(k_cache, v_cache)
    if k_new.ndim != 3 or k_new.shape != v_new.shape:
        raise ValueError("k_new/v_new must be matching [batch, heads, head_dim] tensors.")
    if k_new.stride() != v_new.stride():
        raise ValueError("k_new and v_new must have identical strides.")
    batch, heads, head_dim = k_new.shape
    num_blocks, cache_heads, block_size, cache_dim = k_cache.shape
    if heads != cache_heads or head_dim != cache_dim:
        raise ValueError(
            f"k_new {tuple(k_new.shape)} does not match cache heads/head_dim ({cache_heads}, {cache_dim})."
        )
    if k_new.dtype != k_cache.dtype or v_new.dtype != k_cache.dtype:
        raise ValueError("k_new/v_new must have the cache dtype.")
    _check_tables(block_tables, context_lens, batch)
    dev = _require_cuda(k_new, v_new, k_cache, v_cache, block_tables, context_lens, status)
    bt = _as_i32(block_tables)
    ctx = _as_i32(context_lens)
    lib = _lib.load()
    with _device_ctx(dev):
        _lib.check(
            "pkv_append",
            lib.pkv_append(
                k_new.data_ptr(), v_new.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
                bt.data_ptr(), ctx.data_ptr(), batch, heads, head_dim, block_size, num_blocks,
                bt.shape[1], _strides(k_new.stride()), _strides(k_cache.stride()),
                _strides(bt.stride()), _dtype_code(k_cache, "k_cache"), _status_ptr(status),
                _stream(dev),
            ),
        )


def paged_kv_append_prompt(
    k: torch.Tensor,
    v: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_tables: torch.Tensor,
    start_pos: Optional[torch.Tensor] = None,
    lens: Optional[torch.Tensor] = None,
    *,
    status: Optional[torch.Tensor] = None,
) -> None:
    """Bulk prompt write: k/v [B, H, T, D] (HF past_key_values layout) into pages.

    Position start_pos[b] + t for t < lens[b] (defaults 0 and T), the
    addressing of the reference prefill scatter (paged_kv.py:576-586) done
    in one launch instead of B x T x L slice assignments.
    """
    _check_cache_pair(k_cache, v_cache)
    if k.ndim != 4 or k.shape != v.shape or k.stride() != v.stride():
        raise ValueError("k/v must be matching [batch, heads, seq_len, head_dim] tensors.")
    batch, heads, seq_len, head_dim = k.shape
    num_blocks, cache_heads, block_size, cache_dim = k_cache.shape
    if heads != cache_heads or head_dim != cache_dim:
        raise ValueError(f"k {tuple(k.shape)} does not match cache heads/head_dim ({cache_heads}, {cache_dim}).")
    if k.dtype != k_cache.dtype or v.dtype != k_cache.dtype:
        raise ValueError("k/v must have the cache dtype.")
    if block_tables.ndim != 2 or block_tables.shape[0] != batch:
        raise ValueError("block_tables must be [batch, max_blocks].")
    for name, t in (("start_pos", start_pos), ("lens", lens)):
        if t is not None and (t.ndim != 1 or t.shape[0] != batch):
            raise ValueError(f"{name} must be [batch].")
    dev = _require_cuda(k, v, k_cache, v_cache, block_tables, start_pos, lens, status)
    bt = _as_i32(block_tables)
    sp = None if start_pos is None else _as_i32(start_pos)
    ln = None if lens is None else _as_i32(lens)
    lib = _lib.load()
    with _device_ctx(dev):
        _lib.check(
            "pkv_append_prompt",
            lib.pkv_append_prompt(
                k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), bt.data_ptr(),
                _lib.ptr(sp), _lib.ptr(ln), batch, heads, seq_len, head_dim, block_size, num_blocks,
                bt.shape[1], _strides(k.stride()), _strides(k_cache.stride()),
                _strides(bt.stride()), _dtype_code(k_cache, "k_cache"), _status_ptr(status),
                _stream(dev),
            ),
        )


def gather_kv(
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_tables: torch.Tensor,
    context_lens: torch.Tensor,
    max_tokens: Optional[int] = None,
    *,
    status: Optional[torch.Tensor] = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Dense K, V [B, H, T, D] of the paged cache; positions >= context_lens[b] are zero.

    max_tokens defaults to the block-table capacity max_blocks * block_size.
    """
    _check_cache_pair(k_cache, v_cache)
    batch = block_tables.shape[0] if block_tables.ndim == 2 else -1
    _check_tables(block_tables, context_lens, batch)
    dev = _require_cuda(k_cache, v_cache, block_tables, context_lens, status)
    num_blocks, heads, block_size, head_dim = k_cache.shape
    bt = _as_i32(block_tables)
    ctx = _as_i32(context_lens)
    if max_tokens is None:
        max_tokens = bt.shape[1] * block_size
    k_out = torch.empty((batch, heads, max_tokens, head_dim), dtype=k_cache.dtype, device=dev)
    v_out = torch.empty_like(k_out)
    lib = _lib.load()
    with _device_ctx(dev):
        _lib.check(
            "pkv_gather",
            lib.pkv_gather(
                k_cache.data_ptr(), v_cache.data_ptr(), bt.data_ptr(), ctx.data_ptr(),
                k_out.data_ptr(), v_out.data_ptr(), batch, heads, head_dim, block_size, num_blocks,
                bt.shape[1], max_tokens, _strides(k_cache.stride()),
                _strides(bt.stride()), _strides(k_out.stride()),
                _dtype_code(k_cache, "k_cache"), _status_ptr(status), _stream(dev),
            ),
        )
    return k_out, v_out


# ---------------------------------------------------------------------------
# decode attention
# ---------------------------------------------------------------------------
@dataclass
class DecodePlan:
    """A decode work plan in a device workspace, valid for one context_lens.

    A plan depends only on context_lens and the sizes, so a caller that runs
    several layers with the same context_lens (one decode step of a model)
    makes one plan and calls ``paged_attention_decode(..., plan=plan)`` per
    layer. The workspace is also the split-K scratch of every call that uses
    the plan: calls sharing a plan must be ordered on one stream.
    ``pages_per_split`` is the split-length argument every call of the plan
    passes (0: the library's heuristic); ``chosen_pages_per_split()`` reads the
    length the plan kernel used back from the workspace (a device sync).
    """

    batch: int
    num_q_heads: int
    num_kv_heads: int
    head_dim: int
    block_size: int
    max_blocks: int
    pages_per_split: int
    workspace: torch.Tensor
    context_lens: torch.Tensor

    def chosen_pages_per_split(self) -> int:
        """The split length the plan kernel wrote into the workspace header."""
        return int(self.workspace[:8].view(torch.int32)[1].item())

    def matches(self, batch, num_q_heads, num_kv_heads, head_dim, block_size, max_blocks) -> bool:
        return (self.batch, self.num_q_heads, self.num_kv_heads, self.head_dim, self.block_size, self.max_blocks) == (
            batch, num_q_heads, num_kv_heads, head_dim, block_size, max_blocks)


def decode_workspace_bytes(batch, num_q_heads, num_kv_heads, head_dim, max_blocks, pages_per_split=0) -> int:
    n = _lib.load().pkv_decode_workspace_size(batch, num_q_heads, num_kv_heads, head_dim, max_blocks, pages_per_split)
    if n == 0:
        raise ValueError("invalid decode geometry for the workspace size query.")
    return int(n)


def _pages_per_split(batch, num_q_heads, num_kv_heads, head_dim, max_blocks, num_splits, pages_per_split) -> int:
    """The split-length argument of the C ABI: pages_per_split, or the length
    that caps the splits per sequence at num_splits, or 0 (the library's
    heuristic, which lets the plan kernel pick the length from the actual
    context lengths when the batch has fewer units than SMs)."""
    if pages_per_split <= 0 and num_splits and num_splits > 0:
        pages_per_split = max(1, math.ceil(max(max_blocks, 1) / num_splits))
    pages_per_split = max(0, int(pages_per_split))
    _lib.check(
        "pkv_decode_pages_per_split",
        _lib.load().pkv_decode_pages_per_split(batch, num_q_heads, num_kv_heads, head_dim, max_blocks, pages_per_split),
    )
    return pages_per_split


def plan_decode(
    context_lens: torch.Tensor,
    num_q_heads: int,
    num_kv_heads: int,
    head_dim: int,
    block_size: int,
    max_blocks: int,
    num_splits: int = 0,
    *,
    pages_per_split: int = 0,
    workspace: Optional[torch.Tensor] = None,
    status: Optional[torch.Tensor] = None,
) -> DecodePlan:
    """Plan the split-K decode of all sequences for one context_lens (post-append lengths)."""
    if context_lens.ndim != 1:
        raise ValueError(f"context_lens must be [batch], got {tuple(context_lens.shape)}.")
    if num_q_heads % num_kv_heads != 0:
        raise ValueError(f"num_heads ({num_q_heads}) must be divisible by num_kv_heads ({num_kv_heads}).")
    dev = _require_cuda(context_lens, workspace, status)
    batch = context_lens.shape[0]
    ctx = _as_i32(context_lens)
    pps = _pages_per_split(batch, num_q_heads, num_kv_heads, head_dim, max_blocks, num_splits, pages_per_split)
    need = decode_workspace_bytes(batch, num_q_heads, num_kv_heads, head_dim, max_blocks, pps)
    if workspace is None or workspace.numel() * workspace.element_size() < need:
        workspace = torch.empty(need, dtype=torch.uint8, device=dev)
    lib = _lib.load()
    with _device_ctx(dev):
        _lib.check(
            "pkv_decode_plan",
            lib.pkv_decode_plan(
                ctx.data_ptr(), batch, num_q_heads, num_kv_heads, head_dim, block_size, max_blocks, pps,
                workspace.data_ptr(), workspace.numel() * workspace.element_size(), _status_ptr(status),
                _stream(dev),
            ),
        )
    return DecodePlan(batch, num_q_heads, num_kv_heads, head_dim, block_size, max_blocks, pps, workspace, ctx)


def paged_attention_decode(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_tables: torch.Tensor,
    context_lens: torch.Tensor,
    scale: Optional[float] = None,
    out: Optional[torch.Tensor] = None,
    num_splits: int = 0,
    *,
    pages_per_split: int = 0,
    plan: Optional[DecodePlan] = None,
    force_generic: bool = False,
    exact: bool = False,
    status: Optional[torch.Tensor] = None,
    k_new: Optional[torch.Tensor] = None,
    v_new: Optional[torch.Tensor] = None,
    out_dtype: Optional[torch.dtype] = None,
    rope: Optional[tuple[torch.Tensor, torch.Tensor]] = None,
    early_start: bool = False,
) -> torch.Tensor:
    """Single-query attention over the paged cache; returns fp32 [B, Hq, D].

    q is [B, Hq, D]; the caches are [num_blocks, Hkv, block_size, D] with
    Hq a multiple of Hkv (query head h reads cache head h // (Hq // Hkv),
    the grouped-query mapping of HF repeat_kv). Hq == Hkv is the reference's
    head-replicated layout. context_lens are POST-append lengths
    (paged_kv.py:697,761,938); scale defaults to 1/sqrt(D) (paged_kv.py:681,900).
    num_splits > 0 caps the number of split-K chunks per sequence;
    pages_per_split > 0 sets the chunk length directly; both 0 = heuristic.
    The tensor-core kernel multiplies the softmax weights by V in 16 bits
    (max-abs error a few 1e-3 for N(0,1) data); exact=True keeps ~17
    significant bits of the weights at some speed cost. The CUDA-core kernel
    (fp32 caches, force_generic=True) is fp32 throughout.

    With k_new / v_new ([B, Hkv, D], cache dtype) the call is one decode step
    of a layer including the append: the new token is written at position
    context_lens[b] - 1 (context_lens stay POST-append) and attended to, in
    a single launch on the tensor-core kernel (C ABI pkv_append_decode_run).
    It writes the cache bytes paged_kv_append(..., context_lens - 1) writes.

    With rope=(cos, sin) ([B, D], q's dtype) and k_new / v_new, q and k_new
    are the rows before RoPE and the launch rotates them as rope_qk does (C ABI
    pkv_rope_append_decode_run; tensor-core kernel only, PkvError otherwise).

    out_dtype=q.dtype (bf16 / fp16 q) returns the output in q's dtype, each
    fp32 result rounded to nearest: the values of ``.to(q.dtype)`` of the fp32
    output, without a separate conversion launch.

    early_start=True promises that the previous kernel queued on the stream
    wrote none of the plan, the block tables, the context lengths and the
    caches, and that the kernels before it are complete once it lets this
    launch start: true for every layer's decode launch of a step after the
    first (each follows an earlier decode launch, which lets the next launch
    start only after its own wait), not for the first (behind the plan) nor
    one behind a separate append. The tensor-core launch then schedules its
    first unit and starts loading its pages before that kernel has finished;
    q, the new rows and cos / sin are still read after it. Results are
    unchanged.
    """
    _check_cache_pair(k_cache, v_cache)
    if q.ndim != 3:
        raise ValueError(f"q must be [batch, heads, head_dim], got {tuple(q.shape)}.")
    batch, hq, head_dim = q.shape
    num_blocks, hkv, block_size, cache_dim = k_cache.shape
    if cache_dim != head_dim:
        raise ValueError(f"q head_dim {head_dim} does not match cache head_dim {cache_dim}.")
    if hq % hkv != 0:
        raise ValueError(f"num_heads ({hq}) must be divisible by num_kv_heads ({hkv}).")
    _check_tables(block_tables, context_lens, batch)
    dev = _require_cuda(q, k_cache, v_cache, block_tables, context_lens, out, status)
    if out_dtype is None:
        out_dtype = out.dtype if out is not None else torch.float32
    if out_dtype not in (torch.float32, q.dtype):
        raise ValueError(f"out_dtype must be float32 or q's dtype ({q.dtype}), got {out_dtype}.")
    if out is None:
        out = torch.empty((batch, hq, head_dim), dtype=out_dtype, device=dev)
    elif out.dtype != out_dtype or tuple(out.shape) != (batch, hq, head_dim):
        raise ValueError(f"out must be a {out_dtype} [batch, heads, head_dim] tensor.")
    if scale is None:
        scale = 1.0 / math.sqrt(head_dim)
    bt = _as_i32(block_tables)
    max_blocks = bt.shape[1]
    if plan is None:
        plan = plan_decode(context_lens, hq, hkv, head_dim, block_size, max_blocks, num_splits,
                           pages_per_split=pages_per_split, status=status)
    elif not plan.matches(batch, hq, hkv, head_dim, block_size, max_blocks):
        raise ValueError("decode plan was made for a different geometry.")
    lib = _lib.load()
    ws = plan.workspace
    if rope is not None and k_new is None:
        raise ValueError("rope needs k_new / v_new (RoPE runs with the fused append).")
    flags = (_lib.DECODE_FORCE_GENERIC if force_generic else 0) | (_lib.DECODE_EXACT_P if exact else 0)
    if early_start:
        flags |= _lib.DECODE_EARLY_START
    if out.dtype != torch.float32:
        flags |= _lib.DECODE_OUT_Q_DTYPE
    if k_new is not None or v_new is not None:
        if k_new is None or v_new is None:
            raise ValueError("k_new and v_new must be given together.")
        if k_new.ndim != 3 or k_new.shape != v_new.shape or tuple(k_new.shape) != (batch, hkv, head_dim):
            raise ValueError(f"k_new/v_new must be matching [batch, num_kv_heads, head_dim] = "
                             f"{(batch, hkv, head_dim)} tensors.")
        if k_new.stride() != v_new.stride():
            raise ValueError("k_new and v_new must have identical strides.")
        if k_new.dtype != k_cache.dtype or v_new.dtype != k_cache.dtype:
            raise ValueError("k_new/v_new must have the cache dtype.")
        _require_cuda(k_new, v_new, k_cache)
        if rope is not None:
            cos, sin = rope
            if cos.shape != (batch, head_dim) or sin.shape != cos.shape or cos.stride() != sin.stride() \
                    or cos.stride(1) != 1 or cos.dtype != q.dtype or sin.dtype != q.dtype:
                raise ValueError("rope cos / sin must be matching [batch, head_dim] tensors of q's dtype "
                                 "with contiguous rows.")
            _require_cuda(cos, sin)
            with _device_ctx(dev):
                _lib.check(
                    "pkv_rope_append_decode_run",
                    lib.pkv_rope_append_decode_run(
                        q.data_ptr(), k_new.data_ptr(), v_new.data_ptr(), cos.data_ptr(), sin.data_ptr(),
                        cos.stride(0), k_cache.data_ptr(), v_cache.data_ptr(), bt.data_ptr(),
                        plan.context_lens.data_ptr(), out.data_ptr(), batch, hq, hkv, head_dim, block_size,
                        num_blocks, max_blocks, _strides(q.stride()), _strides(k_new.stride()),
                        _strides(k_cache.stride()), _strides(bt.stride()), _strides(out.stride()),
                        _dtype_code(q, "q"), _dtype_code(k_cache, "k_cache"), float(scale), plan.pages_per_split,
                        flags, ws.data_ptr(), ws.numel() * ws.element_size(), _status_ptr(status), _stream(dev),
                    ),
                )
            return out
        with _device_ctx(dev):
            _lib.check(
                "pkv_append_decode_run",
                lib.pkv_append_decode_run(
                    q.data_ptr(), k_new.data_ptr(), v_new.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
                    bt.data_ptr(), plan.context_lens.data_ptr(), out.data_ptr(), batch, hq, hkv, head_dim,
                    block_size, num_blocks, max_blocks, _strides(q.stride()), _strides(k_new.stride()),
                    _strides(k_cache.stride()), _strides(bt.stride()), _strides(out.stride()),
                    _dtype_code(q, "q"), _dtype_code(k_cache, "k_cache"), float(scale), plan.pages_per_split,
                    flags, ws.data_ptr(), ws.numel() * ws.element_size(), _status_ptr(status), _stream(dev),
                ),
            )
        return out
    with _device_ctx(dev):
        _lib.check(
            "pkv_decode_run",
            lib.pkv_decode_run(
                q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), bt.data_ptr(), plan.context_lens.data_ptr(),
                out.data_ptr(), batch, hq, hkv, head_dim, block_size, num_blocks, max_blocks,
                _strides(q.stride()), _strides(k_cache.stride()), _strides(bt.stride()),
                _strides(out.stride()), _dtype_code(q, "q"), _dtype_code(k_cache, "k_cache"),
                float(scale), plan.pages_per_split, flags, ws.data_ptr(), ws.numel() * ws.element_size(),
                _status_ptr(status), _stream(dev),
            ),
        )
    return out


# ---------------------------------------------------------------------------
# decode-step element-wise steps
# ---------------------------------------------------------------------------
def add_rmsnorm(
    x: torch.Tensor,
    weight: torch.Tensor,
    eps: float,
    residual: Optional[torch.Tensor] = None,
) -> tuple[torch.Tensor, Optional[torch.Tensor]]:
    """RMSNorm of x [rows, hidden] (after adding residual, if given) in one launch.

    Returns (normed, x + residual or None), with the rounding points of HF's
    Qwen2RMSNorm: the sum rounded to the dtype, fp32 statistics,
    dtype(s * rsqrt(mean(s^2) + eps)) scaled by weight (C ABI pkv_add_rmsnorm).
    """
    if x.ndim != 2 or x.stride(1) != 1:
        raise ValueError("x must be [rows, hidden] with contiguous rows.")
    rows, hidden = x.shape
    if weight.shape != (hidden,) or weight.dtype != x.dtype or not weight.is_contiguous():
        raise ValueError("weight must be a contiguous [hidden] tensor of x's dtype.")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype or residual.stride(1) != 1):
        raise ValueError("residual must match x.")
    dev = _require_cuda(x, weight, residual)
    out = torch.empty_like(x, memory_format=torch.contiguous_format)
    total = torch.empty_like(out) if residual is not None else None
    with _device_ctx(dev):
        _lib.check(
            "pkv_add_rmsnorm",
            _lib.load().pkv_add_rmsnorm(
                x.data_ptr(), residual.data_ptr() if residual is not None else None, weight.data_ptr(),
                total.data_ptr() if total is not None else None, out.data_ptr(), rows, hidden, x.stride(0),
                residual.stride(0) if residual is not None else 0, hidden, hidden, float(eps),
                _dtype_code(x, "x"), _stream(dev)),
        )
    return out, total


def silu_mul(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    """dtype(dtype(silu(gate)) * up) for [rows, cols] tensors in one launch (C ABI pkv_silu_mul):
    the gated activation of a Qwen2 MLP with the rounding of F.silu(gate) * up."""
    if gate.ndim != 2 or gate.shape != up.shape or gate.dtype != up.dtype or gate.stride(1) != 1 or up.stride(1) != 1:
        raise ValueError("gate and up must be matching [rows, cols] tensors with contiguous rows.")
    dev = _require_cuda(gate, up)
    out = torch.empty(gate.shape, dtype=gate.dtype, device=dev)
    with _device_ctx(dev):
        _lib.check(
            "pkv_silu_mul",
            _lib.load().pkv_silu_mul(gate.data_ptr(), up.data_ptr(), out.data_ptr(), gate.shape[0], gate.shape[1],
                                     gate.stride(0), up.stride(0), _dtype_code(gate, "gate"), _stream(dev)),
        )
    return out


def rope_qk(
    q: torch.Tensor,
    k: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
    num_q_heads: int,
    num_kv_heads: int,
    head_dim: int,
    k_out: Optional[torch.Tensor] = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """RoPE of one new query / key row per sequence, one launch.

    q [rows, Hq * D], k [rows, Hkv * D] (the projections' outputs), cos / sin
    [rows, D]; returns q [rows, Hq, D] (contiguous) and k [rows, Hkv, D] equal to
    HF's apply_rotary_pos_emb of the same rows (C ABI pkv_rope_qk). With k_out
    ([rows, Hkv * D], contiguous rows; k itself rotates k in place) the keys are
    written there and the returned k is its [rows, Hkv, D] view.
    """
    rows = q.shape[0]
    if (q.shape != (rows, num_q_heads * head_dim) or k.shape != (rows, num_kv_heads * head_dim)
            or q.stride(1) != 1 or k.stride(1) != 1):
        raise ValueError("q / k must be [rows, heads * head_dim] with contiguous rows.")
    if cos.shape != (rows, head_dim) or sin.shape != cos.shape or cos.stride() != sin.stride() or cos.stride(1) != 1:
        raise ValueError("cos / sin must be matching [rows, head_dim] tensors with contiguous rows.")
    if not (q.dtype == k.dtype == cos.dtype == sin.dtype):
        raise ValueError("q, k, cos and sin must share one dtype.")
    dev = _require_cuda(q, k, cos, sin)
    qo = torch.empty(rows, num_q_heads, head_dim, dtype=q.dtype, device=dev)
    if k_out is None:
        ko = torch.empty(rows, num_kv_heads, head_dim, dtype=k.dtype, device=dev)
        k_rows = num_kv_heads * head_dim
    else:
        if k_out.shape != k.shape or k_out.dtype != k.dtype or k_out.stride(1) != 1:
            raise ValueError("k_out must match k: [rows, heads * head_dim] with contiguous rows.")
        _require_cuda(k_out)
        ko, k_rows = k_out.view(rows, num_kv_heads, head_dim), k_out.stride(0)
    with _device_ctx(dev):
        _lib.check(
            "pkv_rope_qk",
            _lib.load().pkv_rope_qk(q.data_ptr(), k.data_ptr(), cos.data_ptr(), sin.data_ptr(), qo.data_ptr(),
                                    ko.data_ptr(), rows, num_q_heads, num_kv_heads, head_dim, q.stride(0),
                                    k.stride(0), cos.stride(0), num_q_heads * head_dim, k_rows,
                                    _dtype_code(q, "q"), _stream(dev)),
        )
    return qo, ko


# ---------------------------------------------------------------------------
# sampling
# ---------------------------------------------------------------------------
# ---------------------------------------------------------------------------
# projections of the decode step (tcgen05 GEMM)
# ---------------------------------------------------------------------------
def linear_supported(x: torch.Tensor, weight: torch.Tensor) -> bool:
    """Whether linear() serves these operands: CUDA bf16 / fp16 x and weight of
    one dtype, in_features a multiple of 64, 16-byte aligned rows with
    contiguous columns."""
    return (x.is_cuda and weight.is_cuda and x.dtype == weight.dtype and x.dtype in (torch.bfloat16, torch.float16)
            and x.ndim == 2 and weight.ndim == 2 and x.shape[1] == weight.shape[1] and x.shape[1] % 64 == 0
            and x.stride(1) == 1 and weight.stride(1) == 1 and x.stride(0) % 8 == 0 and weight.stride(0) % 8 == 0
            and x.data_ptr() % 16 == 0 and weight.data_ptr() % 16 == 0)


def linear(
    x: torch.Tensor,
    weight: torch.Tensor,
    bias: Optional[torch.Tensor] = None,
    *,
    out: Optional[torch.Tensor] = None,
    silu_gate: bool = False,
    weight_up: Optional[torch.Tensor] = None,
    status: Optional[torch.Tensor] = None,
    weights_static: bool = False,
) -> torch.Tensor:
    """``x @ weight.T (+ bias)`` for the few activation rows of a decode step,
    on the tcgen05 tensor cores (C ABI pkv_linear): x [rows, K], weight in
    nn.Linear's [N, K] layout, fp32 accumulation, output in x's dtype.

    silu_gate=True: weight is the gate_proj weight [n, K] and weight_up the
    up_proj weight (or, without weight_up, weight is the two stacked, [2 n, K]);
    the result [rows, n] is ``silu(x @ gate.T) * (x @ up.T)`` with the rounding
    of HF Qwen2MLP (each GEMM output, the activation and the product rounded to
    the dtype). Rows beyond 128 run as further launches of 128 rows.

    weights_static=True promises that no kernel still queued on the stream
    writes weight / weight_up (model weights during generation): the launch
    then streams its first weight tiles while the previous kernel finishes.
    """
    if not linear_supported(x, weight):
        raise ValueError("linear needs CUDA bf16/fp16 x [rows, K] and weight [N, K] of one dtype, K a multiple of "
                         "64, contiguous 16-byte aligned rows.")
    dev = _require_cuda(x, weight, bias, out, status, weight_up)
    rows, k = x.shape
    if weight_up is not None:
        if not silu_gate or weight_up.shape != weight.shape or weight_up.stride() != weight.stride() \
                or weight_up.dtype != weight.dtype or weight_up.data_ptr() % 16 != 0:
            raise ValueError("weight_up must match weight (shape, strides, dtype) and needs silu_gate.")
        n = weight.shape[0]
    else:
        n = weight.shape[0] // 2 if silu_gate else weight.shape[0]
    if silu_gate and ((weight_up is None and weight.shape[0] % 2 != 0) or bias is not None):
        raise ValueError("silu_gate needs gate / up weights (separate, or stacked [2 n, K]) and no bias.")
    if bias is not None and (bias.dtype != x.dtype or bias.numel() != n or bias.stride(0) != 1):
        raise ValueError("bias must be a contiguous [N] tensor of x's dtype.")
    if out is None:
        out = torch.empty(rows, n, dtype=x.dtype, device=dev)
    elif out.dtype != x.dtype or tuple(out.shape) != (rows, n) or out.stride(1) != 1:
        raise ValueError(f"out must be a [rows, {n}] tensor of x's dtype with contiguous rows.")
    lib = _lib.load()
    act = _lib.LINEAR_SILU_GATE if silu_gate else _lib.LINEAR_NONE
    if weights_static:
        act |= _lib.LINEAR_WEIGHTS_STATIC
    code = _dtype_code(x, "x")
    with _device_ctx(dev):
        st = _stream(dev)
        for r0 in range(0, rows, 128):
            r = min(128, rows - r0)
            _lib.check("pkv_linear", lib.pkv_linear(
                x[r0:].data_ptr(), weight.data_ptr(), _lib.ptr(weight_up), _lib.ptr(bias), out[r0:].data_ptr(), r, n,
                k, x.stride(0), weight.stride(0), out.stride(0), code, act, _status_ptr(status), st))
    return out


def sample_top_p(
    logits: torch.Tensor,
    temperature: float,
    top_p: float,
    generator: Optional[torch.Generator] = None,
    force_radix: bool = False,
) -> torch.Tensor:
    """One token per row of logits [B, V]: temperature + nucleus (top-p) sampling.

    The nucleus is the reference's (paged_kv.py:418-450): softmax(logits / T)
    in descending order, tokens kept while their running probability stays
    <= top_p, the most likely token always kept; top_p >= 1 keeps all. One
    launch per call (C ABI pkv_sample_top_p) instead of a sort of the whole
    vocabulary. The draw uses one uniform per row from ``generator`` (so a
    seeded generator reproduces the tokens) and the inverse CDF of the kept
    tokens in index order. Returns int64 [B]. ``force_radix`` selects the
    radix-select path for 16-bit logits (the same tokens, slower).
    """
    if logits.ndim != 2:
        raise ValueError(f"logits must be [batch, vocab], got {tuple(logits.shape)}.")
    if not temperature > 0.0 or not top_p > 0.0:
        raise ValueError("temperature and top_p must be > 0 for sampling.")
    dev = _require_cuda(logits)
    if logits.stride(1) != 1:
        logits = logits.contiguous()
    batch, vocab = logits.shape
    u = torch.rand(batch, device=dev, dtype=torch.float32, generator=generator)
    out = torch.empty(batch, dtype=torch.int64, device=dev)
    lib = _lib.load()
    with _device_ctx(dev):
        _lib.check(
            "pkv_sample_top_p",
            lib.pkv_sample_top_p(logits.data_ptr(), _dtype_code(logits, "logits"), batch, vocab, logits.stride(0),
                                 float(max(temperature, 1e-6)), float(top_p if top_p < 1.0 else 2.0),
                                 u.data_ptr(), out.data_ptr(), _lib.SAMPLE_FORCE_RADIX if force_radix else 0,
                                 _stream(dev)),
        )
    return out


# ---------------------------------------------------------------------------
# 8-bit activations and weights
# ---------------------------------------------------------------------------
def _call(dev: torch.device, name: str, *args) -> None:
    """One entry point of libpkv.so on `dev`'s current stream (the last argument)."""
    fn = getattr(_lib.load(), name)
    if dev.index == torch._C._cuda_getDevice():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev.index))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev.index))
    if rc < 0:
        raise _lib.PkvError(name, rc, _lib.last_detail())


FP8_GROUP = 128  # values that share a scale


def _empty2(rows: int, cols: int, dtype: torch.dtype, dev: torch.device, stride: int = 0) -> torch.Tensor:
    """torch.empty((rows, cols)), with rows `stride` elements apart (empty_strided takes 1 us less per call)."""
    return torch.empty_strided((rows, cols), (stride or cols, 1), dtype=dtype, device=dev)


def _fp8_rows(rows: int, cols: int, dev: torch.device) -> torch.Tensor:
    """An e4m3 [rows, cols] tensor whose rows begin on 16-byte boundaries, as linear_fp8 reads them."""
    return _empty2(rows, cols, torch.float8_e4m3fn, dev, (cols + 15) // 16 * 16)


def _groups(n: int) -> int:
    return (n + FP8_GROUP - 1) // FP8_GROUP


def add_rmsnorm_fp8(
    x: torch.Tensor,
    weight: torch.Tensor,
    eps: float,
    residual: Optional[torch.Tensor] = None,
) -> tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
    """RMSNorm of x [rows, hidden] (after adding residual, if given) as 8-bit values, in one launch.

    Returns (q, scales, x + residual or None): q float8_e4m3fn [rows, hidden]
    and scales fp32 [rows, ceil(hidden / 128)], the norm being q times the
    scale of its group of 128; the two are linear_fp8's x and x_scale. The norm
    is fp32 from the unrounded sum up to q (add_rmsnorm rounds the sum and the
    norm to x's dtype on the way); the returned sum is rounded to x's dtype.
    Any hidden size and row strides (C ABI pkv_add_rmsnorm_fp8).
    """
    if x.ndim != 2 or x.stride(1) != 1:
        raise ValueError("x must be [rows, hidden] with contiguous rows.")
    rows, hidden = x.shape
    if hidden == 0:
        raise ValueError("x must have at least one column.")
    if weight.shape != (hidden,) or weight.dtype != x.dtype or not weight.is_contiguous():
        raise ValueError("weight must be a contiguous [hidden] tensor of x's dtype.")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype or residual.stride(1) != 1):
        raise ValueError("residual must match x.")
    code = _dtype_code(x, "x")
    dev = _require_cuda(x, weight, residual)
    q = _fp8_rows(rows, hidden, dev)
    scales = _empty2(rows, _groups(hidden), torch.float32, dev)
    total = _empty2(rows, hidden, x.dtype, dev) if residual is not None else None
    _call(dev, "pkv_add_rmsnorm_fp8", x.data_ptr(), _lib.ptr(residual), weight.data_ptr(), _lib.ptr(total),
          q.data_ptr(), scales.data_ptr(), rows, hidden, x.stride(0),
          residual.stride(0) if residual is not None else 0, hidden, q.stride(0), scales.stride(0), eps, code)
    return q, scales, total


def _quantize_fp8(x: torch.Tensor, block_rows: int) -> tuple[torch.Tensor, torch.Tensor]:
    if x.ndim != 2 or x.shape[1] == 0 or x.stride(1) != 1:
        raise ValueError("x must be [rows, cols] with contiguous rows and at least one column.")
    code = _dtype_code(x, "x")
    dev = _require_cuda(x)
    rows, cols = x.shape
    q = _fp8_rows(rows, cols, dev)
    scales = torch.empty(((rows + block_rows - 1) // block_rows, _groups(cols)), dtype=torch.float32, device=dev)
    _call(dev, "pkv_quantize_fp8", x.data_ptr(), q.data_ptr(), scales.data_ptr(), rows, cols, block_rows,
          x.stride(0), q.stride(0), scales.stride(0), code)
    return q, scales


def quantize_fp8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x [rows, cols] as (q float8_e4m3fn, scales fp32 [rows, ceil(cols / 128)]), a scale for each 128
    values of a row: activations for linear_fp8 that no norm wrote."""
    return _quantize_fp8(x, 1)


def quantize_fp8_weight(weight: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """weight [n, k] as (q float8_e4m3fn, scales fp32 [ceil(n / 128), ceil(k / 128)]), a scale for each
    128 x 128 block: what linear_fp8 takes. Done once when a model is loaded."""
    return _quantize_fp8(weight, FP8_GROUP)


def linear_fp8(
    x: torch.Tensor,
    x_scale: torch.Tensor,
    weight: torch.Tensor,
    weight_scale: torch.Tensor,
    bias: Optional[torch.Tensor] = None,
    *,
    out: Optional[torch.Tensor] = None,
    out_dtype: torch.dtype = torch.bfloat16,
    status: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """``x @ weight.T (+ bias)`` of 8-bit x [rows, K] and weight [N, K] with a scale for each 128 values of
    a row of x and each 128 x 128 block of weight (add_rmsnorm_fp8, quantize_fp8, quantize_fp8_weight).

    Any rows, N and K; fp32 accumulation, one rounding to out_dtype (bf16 or
    fp16, also the bias's). x and weight need rows on 16-byte boundaries, as the
    functions named lay them out (C ABI pkv_linear_fp8).
    """
    fp8 = torch.float8_e4m3fn
    if x.ndim != 2 or weight.ndim != 2 or x.dtype != fp8 or weight.dtype != fp8 or x.shape[1] != weight.shape[1] \
            or x.shape[1] == 0 or weight.shape[0] == 0:
        raise ValueError("x [rows, K] and weight [N, K] must be float8_e4m3fn matrices of one K >= 1.")
    rows, k = x.shape
    n = weight.shape[0]
    kb = _groups(k)
    if x_scale.shape != (rows, kb) or weight_scale.shape != (_groups(n), kb) or x_scale.dtype != torch.float32 \
            or weight_scale.dtype != torch.float32 or x_scale.stride(1) != 1 or weight_scale.stride(1) != 1:
        raise ValueError(f"x_scale must be fp32 [rows, ceil(K / 128)] = {(rows, kb)} and weight_scale fp32 "
                         f"[ceil(N / 128), ceil(K / 128)] = {(_groups(n), kb)}, with contiguous rows.")
    if out is not None:
        out_dtype = out.dtype
    if out_dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"out_dtype must be bfloat16 or float16, got {out_dtype}.")
    if bias is not None and (bias.shape != (n,) or bias.dtype != out_dtype or bias.stride(0) != 1):
        raise ValueError("bias must be a contiguous [N] tensor of out_dtype.")
    dev = _require_cuda(x, x_scale, weight, weight_scale, bias, out, status)
    # (a single row has no stride to keep)
    x_stride = x.stride(0) if rows > 1 else (k + 15) // 16 * 16
    w_stride = weight.stride(0) if n > 1 else (k + 15) // 16 * 16
    if x.stride(1) != 1 or weight.stride(1) != 1 or x_stride % 16 or w_stride % 16 or x_stride < k or w_stride < k \
            or x.data_ptr() % 16 or weight.data_ptr() % 16:
        raise ValueError("x and weight need contiguous rows that begin on 16-byte boundaries.")
    if out is None:
        out = _empty2(rows, n, out_dtype, dev)
    elif out.shape != (rows, n) or out.stride(1) != 1 or (rows > 1 and out.stride(0) < n):
        raise ValueError(f"out must be a [rows, {n}] tensor with contiguous rows that do not overlap.")
    _call(dev, "pkv_linear_fp8", x.data_ptr(), x_scale.data_ptr(), weight.data_ptr(), weight_scale.data_ptr(),
          _lib.ptr(bias), out.data_ptr(), rows, n, k, x_stride, x_scale.stride(0) if rows > 1 else kb, w_stride,
          weight_scale.stride(0) if n > FP8_GROUP else kb, out.stride(0) if rows > 1 else n, _DTYPES[out_dtype],
          _status_ptr(status))
    return out


# ---------------------------------------------------------------------------
# from logits to the policy update
# ---------------------------------------------------------------------------
def _logit_rows(logits: torch.Tensor) -> tuple[torch.Tensor, int, int, int, int]:
    """(logits, rows, inner, outer stride, row stride) of [rows, vocab] or [batch, length, vocab] logits
    whose vocabulary is contiguous (copied only where it is not)."""
    if logits.stride(-1) != 1 and logits.shape[-1] > 1:
        logits = logits.contiguous()
    if logits.ndim == 2:
        return logits, logits.shape[0], max(1, logits.shape[0]), 0, logits.stride(0)
    return logits, logits.shape[0] * logits.shape[1], max(1, logits.shape[1]), logits.stride(0), logits.stride(1)


def _check_logits(logits: torch.Tensor, tokens: torch.Tensor, temperature: float, ndims: tuple) -> None:
    if logits.ndim not in ndims or logits.shape[-1] == 0:
        want = " or ".join({2: "[rows, vocab]", 3: "[batch, length, vocab]"}[d] for d in ndims)
        raise ValueError(f"logits must be {want}, got {tuple(logits.shape)}.")
    if tokens.shape != logits.shape[:-1] or tokens.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"tokens must be int64 or int32 {tuple(logits.shape[:-1])}, got {tokens.dtype} "
                         f"{tuple(tokens.shape)}.")
    if not temperature > 0.0:
        raise ValueError("temperature must be > 0.")
    if forward_ad.unpack_dual(logits).tangent is not None:
        raise RuntimeError("logits carry a forward-mode tangent; only backward derivatives are implemented.")


def _tokens64(tokens: torch.Tensor) -> torch.Tensor:
    return (tokens if tokens.dtype == torch.int64 else tokens.to(torch.int64)).contiguous()


def _f32(t: torch.Tensor) -> torch.Tensor:
    """t as an fp32 constant."""
    if t.requires_grad:
        t = t.detach()
    return t if t.dtype == torch.float32 else t.to(torch.float32)


def _first_order(what: str) -> None:
    # (grad mode is on in a backward pass under create_graph; once_differentiable says the same, 20 us later)
    if torch.is_grad_enabled():
        raise RuntimeError(f"{what} has no second derivative (create_graph=True).")


def _logprobs_forward(logits, tokens, temperature, entropy, want_stats, status):
    logits, rows, inner, outer_stride, row_stride = _logit_rows(logits)
    dev = logits.device
    logp = torch.empty_like(tokens, dtype=torch.float32)
    ent = torch.empty_like(logp) if entropy else None
    stats = _empty2(rows, 2, torch.float32, dev) if want_stats else None
    _call(dev, "pkv_token_logprobs", logits.data_ptr(), _DTYPES[logits.dtype], tokens.data_ptr(), rows,
          logits.shape[-1], inner, outer_stride, row_stride, temperature, logp.data_ptr(), _lib.ptr(ent),
          _lib.ptr(stats), _status_ptr(status))
    return logp, ent, stats


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, temperature, entropy, status):
        logp, ent, stats = _logprobs_forward(logits, tokens, temperature, entropy, True, status)
        ctx.save_for_backward(logits, tokens, stats, ent)
        ctx.temperature = temperature
        ctx.set_materialize_grads(False)
        return (logp, ent) if entropy else logp

    @staticmethod
    def backward(ctx, d_logp, d_ent=None):
        _first_order("token_logprobs")
        logits, tokens, stats, ent = ctx.saved_tensors
        if d_logp is None and d_ent is None:
            return None, None, None, None, None
        src, rows, inner, outer_stride, row_stride = _logit_rows(logits)
        dev = src.device
        grad = torch.empty(logits.shape, dtype=logits.dtype, device=dev)
        d_logp, d_ent = (None if d is None else d.contiguous() for d in (d_logp, d_ent))
        _call(dev, "pkv_token_logprobs_grad", src.data_ptr(), _DTYPES[src.dtype], tokens.data_ptr(), rows,
              src.shape[-1], inner, outer_stride, row_stride, ctx.temperature, stats.data_ptr(), _lib.ptr(ent),
              _lib.ptr(d_logp), _lib.ptr(d_ent), grad.data_ptr())
        return grad, None, None, None, None


def token_logprobs(
    logits: torch.Tensor,
    tokens: torch.Tensor,
    *,
    temperature: float = 1.0,
    entropy: bool = False,
    status: Optional[torch.Tensor] = None,
):
    """Log-probability of each token under softmax(logits / temperature): fp32, tokens' shape.

    logits are [rows, vocab] or [batch, length, vocab] (a ``logits[:, :-1]`` view
    is read in place), tokens their leading shape. entropy=True returns
    (logprobs, entropies). Differentiable in the logits through both outputs.
    The logits are read once (and once more, with one write, for the gradient);
    the softmax itself is never stored. A token outside [0, vocab) gives NaN and
    sets PKV_DEV_TOKEN_OUT_OF_RANGE in status (C ABI pkv_token_logprobs).
    """
    _check_logits(logits, tokens, temperature, (2, 3))
    _dtype_code(logits, "logits")
    _require_cuda(logits, tokens, status)
    tokens = _tokens64(tokens)
    if logits.requires_grad and torch.is_grad_enabled():
        return _TokenLogprobs.apply(logits, tokens, float(temperature), bool(entropy), status)
    logp, ent, _ = _logprobs_forward(logits, tokens, float(temperature), entropy, False, status)
    return (logp, ent) if entropy else logp


class PolicyLoss(NamedTuple):
    """What policy_loss returns; only ``loss`` carries a gradient."""

    loss: torch.Tensor           # scalar
    logprobs: torch.Tensor       # [batch, length], 0 where the mask is 0
    kl: torch.Tensor             # scalar: mean KL estimate over the unmasked tokens (0 without ref_logprobs)
    clip_fraction: torch.Tensor  # scalar: share of the unmasked tokens whose ratio the clip decides


_REDUCTIONS = {"token": _lib.REDUCE_TOKEN, "sequence": _lib.REDUCE_SEQUENCE, "sum": _lib.REDUCE_SUM}


def _policy_forward(logits, tokens, old, ref, adv, mask, kl_coef, clip_low, clip_high, temperature, reduction,
                    status, want_grad):
    src, rows, _, batch_stride, row_stride = _logit_rows(logits)
    batch, length, vocab = logits.shape
    dev = logits.device
    out = torch.empty_strided((3,), (1,), dtype=torch.float32, device=dev)
    logp = _empty2(batch, length, torch.float32, dev)
    ws_bytes = _lib.load().pkv_policy_loss_workspace_size(batch, length)
    ws = torch.empty_strided((ws_bytes,), (1,), dtype=torch.uint8, device=dev)
    grad = None
    if want_grad:
        grad = torch.empty_strided((batch, length, vocab), (length * vocab, vocab, 1), dtype=logits.dtype, device=dev)
    _call(dev, "pkv_policy_loss", src.data_ptr(), _DTYPES[src.dtype], tokens.data_ptr(), old.data_ptr(),
          _lib.ptr(ref), adv.data_ptr(), adv.stride(0), adv.stride(1) if adv.ndim == 2 else 0, _lib.ptr(mask), batch,
          length, vocab, batch_stride, row_stride, temperature, clip_low, clip_high, kl_coef, reduction,
          out.data_ptr(), logp.data_ptr(), _lib.ptr(grad), ws.data_ptr(), ws_bytes, _status_ptr(status))
    # .data: tensors of their own, not views of one (a Function's output that is a view cannot be changed in place)
    loss, kl, clipped = out.unbind()
    return loss.data, logp, kl.data, clipped.data, src, grad, ws, (batch, length, vocab, batch_stride, row_stride)


class _PolicyLossFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, args):  # (one argument for all constants: apply looks at each)
        loss, logp, kl, clipped, src, ctx.d_logits, ctx.workspace, ctx.layout = _policy_forward(logits, *args, True)
        ctx.save_for_backward(src)
        ctx.temperature = args[-3]
        ctx.mark_non_differentiable(logp, kl, clipped)
        ctx.set_materialize_grads(False)  # (no zeros for the outputs without a gradient)
        return loss, logp, kl, clipped

    @staticmethod
    def backward(ctx, d_loss, *unused):
        _first_order("policy_loss")
        if d_loss is None:
            return None, None
        (src,) = ctx.saved_tensors
        grad, ctx.d_logits = ctx.d_logits, None
        if grad is None:
            raise RuntimeError("policy_loss: its gradient was computed with the loss and has been handed out; call "
                               "policy_loss again for another backward pass.")
        ws, ctx.workspace = ctx.workspace, None
        # for an upstream gradient other than 1: read on the device, so nothing waits for it here
        _call(grad.device, "pkv_policy_loss_grad", src.data_ptr(), _DTYPES[src.dtype], *ctx.layout, ctx.temperature,
              ws.data_ptr(), ws.numel(), d_loss.data_ptr(), grad.data_ptr())
        return grad, None


def policy_loss(
    logits: torch.Tensor,
    tokens: torch.Tensor,
    old_logprobs: torch.Tensor,
    advantages: torch.Tensor,
    mask: Optional[torch.Tensor] = None,
    *,
    ref_logprobs: Optional[torch.Tensor] = None,
    kl_coef: float = 0.0,
    clip_low: float = 0.2,
    clip_high: float = 0.2,
    temperature: float = 1.0,
    reduction: str = "token",
    status: Optional[torch.Tensor] = None,
) -> PolicyLoss:
    """Clipped policy loss with a KL term on the logits [batch, length, vocab] of the trained policy.

    Per token with lp its log-probability under softmax(logits / temperature),
    r = exp(lp - old_logprobs) and A its advantage ([batch] or [batch, length]):

        -min(r A, clip(r, 1 - clip_low, 1 + clip_high) A)
            + kl_coef (exp(ref - lp) - (ref - lp) - 1)

    the KL term with ref_logprobs only. mask [batch, length] (bool or integer)
    leaves tokens out: their logits are not read, whatever they hold, and get a
    zero gradient. reduction: "token" (mean over the unmasked tokens),
    "sequence" (mean over the batch of each sequence's mean, 0 for one without
    tokens) or "sum".

    Where the logits require grad, the same launch that computes the loss
    writes their gradient (read once, written once), and backward hands it out,
    so it can run once per call. Where the upstream gradient is not 1 (a scaled
    loss, a mean over accumulated batches), backward computes it again from the
    logits, which are kept until then, with the upstream in fp32: one rounding
    to the logits' dtype either way. The other tensors are constants (C ABI
    pkv_policy_loss, pkv_policy_loss_grad).
    """
    _check_logits(logits, tokens, temperature, (3,))
    _dtype_code(logits, "logits")
    shape = tokens.shape
    for name, t in (("old_logprobs", old_logprobs), ("ref_logprobs", ref_logprobs), ("mask", mask)):
        if t is not None and t.shape != shape:
            raise ValueError(f"{name} must be {tuple(shape)}, got {tuple(t.shape)}.")
    if advantages.shape not in (shape, shape[:1]):
        raise ValueError(f"advantages must be {tuple(shape[:1])} or {tuple(shape)}, got {tuple(advantages.shape)}.")
    if mask is not None and mask.is_floating_point():
        raise ValueError("mask must be bool or integer.")
    if not (clip_low >= 0.0 and clip_high >= 0.0):
        raise ValueError("clip_low and clip_high must be >= 0.")
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be one of {sorted(_REDUCTIONS)}, got {reduction!r}.")
    _require_cuda(logits, tokens, old_logprobs, advantages, mask, ref_logprobs, status)
    if mask is not None:
        mask = (mask if mask.dtype in (torch.bool, torch.uint8) else mask != 0).contiguous()
    args = (
        _tokens64(tokens),
        _f32(old_logprobs).contiguous(),
        None if ref_logprobs is None else _f32(ref_logprobs).contiguous(),
        _f32(advantages),
        mask, float(kl_coef), float(clip_low), float(clip_high), float(temperature), _REDUCTIONS[reduction], status,
    )
    if logits.requires_grad and torch.is_grad_enabled():
        return PolicyLoss(*_PolicyLossFn.apply(logits, args))
    return PolicyLoss(*_policy_forward(logits, *args, False)[:4])


def decode_kernel_kind(q: torch.Tensor, k_cache: torch.Tensor, force_generic: bool = False) -> str:
    """'tensor_core' or 'cuda_core': which decode kernel these tensors select."""
    hq, head_dim = q.shape[1], q.shape[2]
    _, hkv, block_size, _ = k_cache.shape
    kind = _lib.check(
        "pkv_decode_kernel_kind",
        _lib.load().pkv_decode_kernel_kind(
            k_cache.data_ptr(), hq, hkv, head_dim, block_size, _strides(k_cache.stride()),
            _dtype_code(q, "q"), _dtype_code(k_cache, "k_cache"),
            _lib.DECODE_FORCE_GENERIC if force_generic else 0,
        ),
    )
    return "tensor_core" if kind == 1 else "cuda_core"
