"""Paged serving operators on torch CUDA tensors: page planning, the K/V append and attention over the pages.

The batched decode of :mod:`.qwen3` gives every member of a fixed batch a contiguous cache of the full context.  These
operators serve requests that come and go: the caches are pages, a block table says which pages hold a request, and one
step takes any mix of prompts' chunks and single decoded tokens.  One step calls, in this order::

    step = paged.plan(lens, new_lens, block_table, free_ring, ring_state, page_size, token_capacity)
    q = paged.append(k, v, k_cache, v_cache, step.positions, step.slots, rope_cos, rope_sin, q=q, ...)   # per layer
    out = paged.attention(q, k_cache, v_cache, block_table, step.lens, step.cu_new, workspace)           # per layer

Every call checks its arguments, enqueues on torch's current stream of the tensors' device and returns without waiting;
errors raise :class:`.gpu.GpuError` with the library's message.  No call reads device values on the host, so a step can
be captured into a CUDA graph (with all outputs given).  ``include/minicpmo_gpu.h`` documents the C entry points.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional

import torch

from . import BF16, F16, F32, lib
from .gpu import ERR_CAP, GpuError, PagedCache

WORKSPACE_BYTES = 64 << 20  # MINICPMO_PAGED_WORKSPACE_BYTES
MAX_REQUESTS = 8192  # MINICPMO_PAGED_MAX_REQUESTS

_DTYPES = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}


def _check(cond: bool, msg: str) -> None:
    if not cond:
        raise GpuError("error: " + msg)


def _call(fn, device: torch.device, *args) -> None:
    err = C.create_string_buffer(ERR_CAP)
    if torch.cuda.current_device() == device.index:
        ok = fn(*args, torch.cuda.current_stream(device).cuda_stream, err, ERR_CAP)
    else:
        with torch.cuda.device(device):
            ok = fn(*args, torch.cuda.current_stream(device).cuda_stream, err, ERR_CAP)
    if not ok:
        raise GpuError(err.value.decode())


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _tensor(op: str, name: str, t: torch.Tensor, device: torch.device, dtype, shape) -> None:
    """t: a contiguous tensor of that type and shape on `device`."""
    if t.dtype != dtype or t.device != device or tuple(t.shape) != tuple(shape) or not t.is_contiguous():
        raise GpuError(f"error: {op}: {name} must be a contiguous {dtype} tensor {tuple(shape)} on {device}, got "
                       f"{t.dtype} {tuple(t.shape)} on {t.device}")


def _rows(op: str, name: str, t: torch.Tensor, device: torch.device, hd: int) -> int:
    """t: [tokens, heads, hd] with contiguous heads; the elements between two tokens."""
    st = t.stride()
    if t.dim() != 3 or t.device != device or t.shape[2] != hd or st[2] != 1 or (st[1] != hd and t.shape[1] > 1):
        raise GpuError(f"error: {op}: {name} must be [tokens, heads, {hd}] on {device} with contiguous heads, got "
                       f"{tuple(t.shape)} with strides {tuple(st)} on {t.device}")
    # the stride of a single token says nothing, and may be anything
    return st[0] if t.shape[0] > 1 else max(st[0], t.shape[1] * hd)


def _cache(op: str, k: torch.Tensor, v: torch.Tensor) -> PagedCache:
    """The C description of one layer's K and V pages, [pages, page_size, kv_heads, head_dim] views of any layout."""
    if k.dim() != 4 or k.shape != v.shape or k.stride() != v.stride() or k.dtype != v.dtype or k.device != v.device:
        raise GpuError(f"error: {op}: k_cache and v_cache must be [pages, page_size, kv_heads, head_dim] tensors alike")
    if not k.is_cuda or k.dtype not in _DTYPES or k.stride(3) != 1:
        raise GpuError(f"error: {op}: caches must be f32, f16 or bf16 CUDA tensors with contiguous rows, got {k.dtype} "
                       f"on {k.device}")
    n, ps, kv, hd = k.shape
    sp, st, sh, _ = k.stride()
    # a dimension of one has no stride of its own: take the contiguous one
    if kv == 1:
        sh = hd
    if n == 1:
        sp = max(st * ps, sh * kv)
    return PagedCache(k.data_ptr(), v.data_ptr(), _DTYPES[k.dtype], ps, kv, hd, n, sp, st, sh)


class PagedPlan(NamedTuple):
    """What one scheduler step does; ``status`` is [flags, free pages]: flags 0, or why the step was refused."""

    lens: torch.Tensor        # int32 [requests]: positions cached after the step
    ring_state: torch.Tensor  # int64 [2]: head and tail of the ring of free pages after the step
    cu_new: torch.Tensor      # int32 [requests + 1]: prefix sums of the new tokens
    positions: torch.Tensor   # int32 [token_capacity]
    slots: torch.Tensor       # int64 [token_capacity]: page * page_size + offset; -1 behind the last token
    status: torch.Tensor      # int32 [2]


def plan(lens: torch.Tensor, new_lens: torch.Tensor, block_table: torch.Tensor, free_ring: torch.Tensor,
         ring_state: torch.Tensor, page_size: int, token_capacity: int, out: Optional[PagedPlan] = None) -> PagedPlan:
    """Give every request's new tokens their pages, positions and cache slots (``minicpmo_gpu_paged_plan``).

    lens int32 [requests]: cached positions; new_lens int32: tokens to add, -1 for a finished request; block_table int32
    [requests, max_pages] and free_ring int32 [capacity] are updated in place.  out's lens and ring_state may be the
    inputs themselves.  A step that does not fit (see status) changes nothing and plans no token.
    """
    op = "paged plan"
    dev, n = lens.device, lens.shape[0] if lens.dim() == 1 else 0
    _check(lens.is_cuda and n > 0, f"{op}: lens must be a CUDA tensor [requests]")
    i32, i64 = torch.int32, torch.int64
    _tensor(op, "lens", lens, dev, i32, (n,))
    _tensor(op, "new_lens", new_lens, dev, i32, (n,))
    _tensor(op, "ring_state", ring_state, dev, i64, (2,))
    _check(free_ring.dim() == 1, f"{op}: free_ring must be [capacity]")
    _tensor(op, "free_ring", free_ring, dev, i32, free_ring.shape)
    if (block_table.dim() != 2 or block_table.shape[0] != n or block_table.dtype != i32 or block_table.device != dev
            or block_table.stride(1) != 1):
        raise GpuError(f"error: {op}: block_table must be an int32 tensor [{n}, max_pages] on {dev} with contiguous rows")
    _check(token_capacity >= 0 and page_size > 0, f"{op}: token_capacity {token_capacity}, page_size {page_size}")
    if out is None:
        with torch.cuda.device(dev):
            out = PagedPlan(torch.empty_like(lens), torch.empty_like(ring_state), lens.new_empty(n + 1),
                            lens.new_empty(token_capacity), ring_state.new_empty(token_capacity), lens.new_empty(2))
    else:
        _tensor(op, "out.lens", out.lens, dev, i32, (n,))
        _tensor(op, "out.ring_state", out.ring_state, dev, i64, (2,))
        _tensor(op, "out.cu_new", out.cu_new, dev, i32, (n + 1,))
        _tensor(op, "out.positions", out.positions, dev, i32, (token_capacity,))
        _tensor(op, "out.slots", out.slots, dev, i64, (token_capacity,))
        _tensor(op, "out.status", out.status, dev, i32, (2,))
    max_pages = block_table.shape[1]
    _call(lib().minicpmo_gpu_paged_plan, dev, lens.data_ptr(), new_lens.data_ptr(), n, block_table.data_ptr(), max_pages,
          block_table.stride(0) if n > 1 else max_pages, free_ring.data_ptr(), free_ring.shape[0], ring_state.data_ptr(),
          page_size, token_capacity, out.lens.data_ptr(), out.ring_state.data_ptr(), out.cu_new.data_ptr(),
          out.positions.data_ptr(), out.slots.data_ptr(), out.status.data_ptr())
    return out


def append(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, positions: torch.Tensor,
           slots: torch.Tensor, rope_cos: torch.Tensor, rope_sin: torch.Tensor, q: Optional[torch.Tensor] = None,
           q_norm: Optional[torch.Tensor] = None, k_norm: Optional[torch.Tensor] = None, eps: float = 1e-6,
           q_out: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """QK-norm, RoPE and the cache write of new tokens (``minicpmo_gpu_paged_append``); returns the rotated q.

    k, v [tokens, kv_heads, head_dim] and q [tokens, q_heads, head_dim] (views into one projection's output are fine) in
    f32, f16 or bf16; k_cache, v_cache [pages, page_size, kv_heads, head_dim] views; rope tables f32 [context,
    head_dim / 2]; norm weights f32 [head_dim] or None.  q_out (default: zeros) has the cache's type; its rows of tokens
    with a negative slot stay as they are.  status int32 [1] gets 1 by OR for a position outside the tables, 2 for a
    slot outside the cache.
    """
    op = "paged append"
    cache = _cache(op, k_cache, v_cache)
    dev, hd, n = k_cache.device, k_cache.shape[3], k.shape[0]
    ks, vs = _rows(op, "k", k, dev, hd), _rows(op, "v", v, dev, hd)
    _check(k.dtype in _DTYPES and v.dtype == k.dtype and k.shape == v.shape and k.shape[1] == k_cache.shape[2],
           f"{op}: k and v must be alike, with the cache's {k_cache.shape[2]} heads")
    _tensor(op, "positions", positions, dev, torch.int32, (n,))
    _tensor(op, "slots", slots, dev, torch.int64, (n,))
    _check(rope_cos.dim() == 2, f"{op}: rope tables must be [context, head_dim / 2]")
    _tensor(op, "rope_cos", rope_cos, dev, torch.float32, (rope_cos.shape[0], hd // 2))
    _tensor(op, "rope_sin", rope_sin, dev, torch.float32, rope_cos.shape)
    for name, w in (("q_norm", q_norm), ("k_norm", k_norm)):
        if w is not None:
            _tensor(op, name, w, dev, torch.float32, (hd,))
    heads = qs = os = 0
    if q is not None:
        heads, qs = q.shape[1], _rows(op, "q", q, dev, hd)
        _check(q.dtype == k.dtype and q.shape[0] == n, f"{op}: q must have k's type and tokens")
        if q_out is None:
            q_out = torch.zeros(n, heads, hd, dtype=k_cache.dtype, device=dev)
        os = _rows(op, "q_out", q_out, dev, hd)
        _check(q_out.dtype == k_cache.dtype and q_out.shape == q.shape, f"{op}: q_out must have the cache's type and q's shape")
    else:
        _check(q_out is None, f"{op}: q_out without q")
    if status is not None:
        _tensor(op, "status", status, dev, torch.int32, (1,))
    _call(lib().minicpmo_gpu_paged_append, dev, C.byref(cache), _ptr(q), k.data_ptr(), v.data_ptr(), _DTYPES[k.dtype], n,
          heads, qs, ks, vs, _ptr(q_norm), _ptr(k_norm), eps, rope_cos.data_ptr(), rope_sin.data_ptr(), rope_cos.shape[0],
          positions.data_ptr(), slots.data_ptr(), _ptr(q_out), os, _ptr(status))
    return q_out


def workspace(device=None) -> torch.Tensor:
    """A workspace for :func:`attention`: one for each set of calls that may overlap on the GPU."""
    return torch.zeros(WORKSPACE_BYTES, dtype=torch.uint8, device="cuda" if device is None else device)


def attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
              lens: torch.Tensor, cu_new: torch.Tensor, workspace: torch.Tensor, scale: Optional[float] = None,
              out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of every request's new tokens over its pages (``minicpmo_gpu_paged_attention``).

    q [tokens, q_heads, head_dim] in the cache's type, q_heads a multiple of the cache's kv_heads (at most 16 each);
    block_table int32 [requests, max_pages]; lens int32 [requests], the new tokens included; cu_new int32 [requests + 1].
    scale defaults to head_dim ** -0.5.  out (default: zeros) keeps its rows behind the last token; lse, if given, is
    f32 [tokens, q_heads] and gets the natural logarithm of every softmax's denominator.
    """
    op = "paged attention"
    cache = _cache(op, k_cache, v_cache)
    dev, hd, n = k_cache.device, k_cache.shape[3], lens.shape[0]
    qs = _rows(op, "q", q, dev, hd)
    _check(q.dtype == k_cache.dtype, f"{op}: q must have the cache's type {k_cache.dtype}, got {q.dtype}")
    _tensor(op, "lens", lens, dev, torch.int32, (n,))
    _tensor(op, "cu_new", cu_new, dev, torch.int32, (n + 1,))
    if (block_table.dim() != 2 or block_table.shape[0] != n or block_table.dtype != torch.int32
            or block_table.device != dev or block_table.stride(1) != 1):
        raise GpuError(f"error: {op}: block_table must be an int32 tensor [{n}, max_pages] on {dev} with contiguous rows")
    _check(workspace.device == dev and workspace.is_contiguous()
           and workspace.numel() * workspace.element_size() >= WORKSPACE_BYTES,
           f"{op}: the workspace must be {WORKSPACE_BYTES} contiguous bytes on {dev}")
    if out is None:
        out = torch.zeros(q.shape, dtype=q.dtype, device=dev)
    os = _rows(op, "out", out, dev, hd)
    _check(out.dtype == q.dtype and out.shape == q.shape, f"{op}: out must have q's type and shape")
    if lse is not None:
        _tensor(op, "lse", lse, dev, torch.float32, q.shape[:2])
    max_pages = block_table.shape[1]
    _call(lib().minicpmo_gpu_paged_attention, dev, C.byref(cache), q.data_ptr(), q.shape[0], q.shape[1], qs,
          block_table.data_ptr(), max_pages, block_table.stride(0) if n > 1 else max_pages, lens.data_ptr(),
          cu_new.data_ptr(), n, hd ** -0.5 if scale is None else scale, out.data_ptr(), os, _ptr(lse),
          workspace.data_ptr())
    return out


class Sampled(NamedTuple):
    token: torch.Tensor  # int32 [rows]
    prob: torch.Tensor   # f32 [rows]: the token's share of the kept weights
    kept: torch.Tensor   # int32 [rows]: tokens that the filters kept


def sample(logits: torch.Tensor, uniform: torch.Tensor, temperature: Optional[torch.Tensor] = None,
           top_k: Optional[torch.Tensor] = None, top_p: Optional[torch.Tensor] = None,
           min_p: Optional[torch.Tensor] = None, out: Optional[Sampled] = None) -> Sampled:
    """One token per row of logits [rows, vocab] (f32, f16 or bf16) from uniform random numbers f32 [rows]
    (``minicpmo_gpu_sample``): temperature, top_p, min_p f32 [rows] and top_k int32 [rows], each None for off."""
    op = "sample"
    if not logits.is_cuda or logits.dim() != 2 or logits.dtype not in _DTYPES or logits.stride(1) != 1:
        raise GpuError(f"error: {op}: logits must be a [rows, vocab] f32, f16 or bf16 CUDA tensor with contiguous rows")
    dev, (n, vocab) = logits.device, logits.shape
    f32 = torch.float32
    _tensor(op, "uniform", uniform, dev, f32, (n,))
    for name, t, dtype in (("temperature", temperature, f32), ("top_k", top_k, torch.int32), ("top_p", top_p, f32),
                           ("min_p", min_p, f32)):
        if t is not None:
            _tensor(op, name, t, dev, dtype, (n,))
    if out is None:
        words = torch.empty(3, n, dtype=torch.int32, device=dev)
        out = Sampled(words[0], words[1].view(f32), words[2])
    else:
        _tensor(op, "out.token", out.token, dev, torch.int32, (n,))
        _tensor(op, "out.prob", out.prob, dev, f32, (n,))
        _tensor(op, "out.kept", out.kept, dev, torch.int32, (n,))
    _call(lib().minicpmo_gpu_sample, dev, logits.data_ptr(), _DTYPES[logits.dtype], n, vocab,
          logits.stride(0) if n > 1 else vocab, _ptr(temperature), _ptr(top_k), _ptr(top_p), _ptr(min_p),
          uniform.data_ptr(), out.token.data_ptr(), out.prob.data_ptr(), out.kept.data_ptr())
    return out
