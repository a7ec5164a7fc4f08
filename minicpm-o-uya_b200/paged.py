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
import threading
from typing import NamedTuple, Optional

import torch

from . import BF16, F16, F32, lib
from .gpu import ERR_CAP, GpuError, PagedCache

WORKSPACE_BYTES = 64 << 20  # MINICPMO_PAGED_WORKSPACE_BYTES
MAX_REQUESTS = 8192  # MINICPMO_PAGED_MAX_REQUESTS

_DTYPES = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}
_I32, _I64, _F32 = torch.int32, torch.int64, torch.float32
_local = threading.local()  # this thread's error buffer
_entry: dict = {}  # the library's entry points by name


def _check(cond: bool, msg: str) -> None:
    if not cond:
        raise GpuError("error: " + msg)


def _call(name: str, index: int, *args) -> None:
    """The library's entry point with the device current and its current stream, the message raised on refusal."""
    try:
        err = _local.err
    except AttributeError:
        err = _local.err = C.create_string_buffer(ERR_CAP)
    fn = _entry.get(name)
    if fn is None:
        fn = _entry[name] = getattr(lib(), name)
    if torch._C._cuda_getDevice() == index:
        ok = fn(*args, torch._C._cuda_getCurrentRawStream(index), err, ERR_CAP)
    else:
        with torch.cuda.device(index):
            ok = fn(*args, torch._C._cuda_getCurrentRawStream(index), err, ERR_CAP)
    if not ok:
        raise GpuError(err.value.decode())


def _tensor(op: str, name: str, t: torch.Tensor, index: int, dtype, shape) -> int:
    """The address of t, a contiguous tensor of that type and shape on device `index`."""
    if t.dtype is not dtype or t.get_device() != index or t.shape != shape or not t.is_contiguous():
        raise GpuError(f"error: {op}: {name} must be a contiguous {dtype} tensor {tuple(shape)} on cuda:{index}, got "
                       f"{t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _rows(op: str, name: str, t: torch.Tensor, index: int, hd: int) -> int:
    """t: [tokens, heads, hd] with contiguous heads; the elements between two tokens."""
    st, shape = t.stride(), t.shape
    if len(shape) != 3 or t.get_device() != index or shape[2] != hd or st[2] != 1 or (st[1] != hd and shape[1] > 1):
        raise GpuError(f"error: {op}: {name} must be [tokens, heads, {hd}] on cuda:{index} with contiguous heads, got "
                       f"{tuple(shape)} with strides {tuple(st)} on {t.device}")
    # the stride of a single token says nothing, and may be anything
    return st[0] if shape[0] > 1 else max(st[0], shape[1] * hd)


def _cache(op: str, k: torch.Tensor, v: torch.Tensor) -> PagedCache:
    """The C description of one layer's K and V pages, [pages, page_size, kv_heads, head_dim] views of any layout."""
    shape, st = k.shape, k.stride()
    if len(shape) != 4 or shape != v.shape or st != v.stride() or k.dtype is not v.dtype or k.get_device() != v.get_device():
        raise GpuError(f"error: {op}: k_cache and v_cache must be [pages, page_size, kv_heads, head_dim] tensors alike")
    dtype = _DTYPES.get(k.dtype)
    if k.get_device() < 0 or dtype is None or st[3] != 1:
        raise GpuError(f"error: {op}: caches must be f32, f16 or bf16 CUDA tensors with contiguous rows, got {k.dtype} "
                       f"on {k.device}")
    n, ps, kv, hd = shape
    sp, st, sh, _ = st
    # a dimension of one has no stride of its own: take the contiguous one
    if kv == 1:
        sh = hd
    if n == 1:
        sp = max(st * ps, sh * kv)
    return PagedCache(k.data_ptr(), v.data_ptr(), dtype, ps, kv, hd, n, sp, st, sh)


def _table(op: str, t: torch.Tensor, n: int, index: int) -> int:
    """The entries between two rows of a block table [n, max_pages]."""
    shape, st = t.shape, t.stride()
    if len(shape) != 2 or shape[0] != n or t.dtype is not _I32 or t.get_device() != index or st[1] != 1:
        raise GpuError(f"error: {op}: block_table must be an int32 tensor [{n}, max_pages] on cuda:{index} with "
                       f"contiguous rows")
    return st[0] if n > 1 else shape[1]


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
    dev, n = lens.get_device(), lens.numel()
    _check(dev >= 0 and n > 0, f"{op}: lens must be a CUDA tensor [requests]")
    _check(token_capacity >= 0 and page_size > 0, f"{op}: token_capacity {token_capacity}, page_size {page_size}")
    stride, ring = _table(op, block_table, n, dev), free_ring.numel()
    inputs = (_tensor(op, "lens", lens, dev, _I32, (n,)), _tensor(op, "new_lens", new_lens, dev, _I32, (n,)), n,
              block_table.data_ptr(), block_table.shape[1], stride, _tensor(op, "free_ring", free_ring, dev, _I32, (ring,)),
              ring, _tensor(op, "ring_state", ring_state, dev, _I64, (2,)), page_size, token_capacity)
    if out is None:
        a, b, c, d = lens.new_empty(2 * n + 3 + token_capacity).split((n, n + 1, token_capacity, 2))
        e, f = ring_state.new_empty(2 + token_capacity).split((2, token_capacity))
        out = PagedPlan(a, e, b, c, f, d)
    else:
        _tensor(op, "out.lens", out.lens, dev, _I32, (n,))
        _tensor(op, "out.ring_state", out.ring_state, dev, _I64, (2,))
        _tensor(op, "out.cu_new", out.cu_new, dev, _I32, (n + 1,))
        _tensor(op, "out.positions", out.positions, dev, _I32, (token_capacity,))
        _tensor(op, "out.slots", out.slots, dev, _I64, (token_capacity,))
        _tensor(op, "out.status", out.status, dev, _I32, (2,))
    _call("minicpmo_gpu_paged_plan", dev, *inputs, *(t.data_ptr() for t in out))
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
    dev, hd, n, ctype = k_cache.get_device(), k_cache.shape[3], k.shape[0], k_cache.dtype
    ks, vs = _rows(op, "k", k, dev, hd), _rows(op, "v", v, dev, hd)
    dtype = _DTYPES.get(k.dtype)
    if dtype is None or v.dtype is not k.dtype or k.shape != v.shape or k.shape[1] != k_cache.shape[2]:
        raise GpuError(f"error: {op}: k and v must be alike, with the cache's {k_cache.shape[2]} heads")
    _check(rope_cos.dim() == 2, f"{op}: rope tables must be [context, head_dim / 2]")
    context = rope_cos.shape[0]
    heads = qs = os = 0
    if q is not None:
        heads, qs = q.shape[1], _rows(op, "q", q, dev, hd)
        if q.dtype is not k.dtype or q.shape[0] != n:
            raise GpuError(f"error: {op}: q must have k's type and tokens")
        if q_out is None:
            q_out = torch.zeros(n, heads, hd, dtype=ctype, device=k_cache.device)
        os = _rows(op, "q_out", q_out, dev, hd)
        if q_out.dtype is not ctype or q_out.shape != q.shape:
            raise GpuError(f"error: {op}: q_out must have the cache's type and q's shape")
    else:
        _check(q_out is None, f"{op}: q_out without q")
    _call("minicpmo_gpu_paged_append", dev, C.byref(cache), None if q is None else q.data_ptr(), k.data_ptr(),
          v.data_ptr(), dtype, n, heads, qs, ks, vs,
          None if q_norm is None else _tensor(op, "q_norm", q_norm, dev, _F32, (hd,)),
          None if k_norm is None else _tensor(op, "k_norm", k_norm, dev, _F32, (hd,)), eps,
          _tensor(op, "rope_cos", rope_cos, dev, _F32, (context, hd // 2)),
          _tensor(op, "rope_sin", rope_sin, dev, _F32, (context, hd // 2)), context,
          _tensor(op, "positions", positions, dev, _I32, (n,)), _tensor(op, "slots", slots, dev, _I64, (n,)),
          None if q_out is None else q_out.data_ptr(), os,
          None if status is None else _tensor(op, "status", status, dev, _I32, (1,)))
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
    dev, hd, n = k_cache.get_device(), k_cache.shape[3], lens.numel()
    qs, stride = _rows(op, "q", q, dev, hd), _table(op, block_table, n, dev)
    if q.dtype is not k_cache.dtype:
        raise GpuError(f"error: {op}: q must have the cache's type {k_cache.dtype}, got {q.dtype}")
    if workspace.get_device() != dev or not workspace.is_contiguous() or workspace.nbytes < WORKSPACE_BYTES:
        raise GpuError(f"error: {op}: the workspace must be {WORKSPACE_BYTES} contiguous bytes on cuda:{dev}")
    if out is None:
        out = torch.zeros(q.shape, dtype=q.dtype, device=q.device)
    os = _rows(op, "out", out, dev, hd)
    if out.dtype is not q.dtype or out.shape != q.shape:
        raise GpuError(f"error: {op}: out must have q's type and shape")
    tokens, heads, _ = q.shape
    _call("minicpmo_gpu_paged_attention", dev, C.byref(cache), q.data_ptr(), tokens, heads, qs, block_table.data_ptr(),
          block_table.shape[1], stride, _tensor(op, "lens", lens, dev, _I32, (n,)),
          _tensor(op, "cu_new", cu_new, dev, _I32, (n + 1,)), n, hd ** -0.5 if scale is None else scale, out.data_ptr(),
          os, None if lse is None else _tensor(op, "lse", lse, dev, _F32, (tokens, heads)), workspace.data_ptr())
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
    shape, dev, dtype = logits.shape, logits.get_device(), _DTYPES.get(logits.dtype)
    if dev < 0 or len(shape) != 2 or dtype is None or logits.stride(1) != 1:
        raise GpuError(f"error: {op}: logits must be a [rows, vocab] f32, f16 or bf16 CUDA tensor with contiguous rows")
    n, vocab = shape
    rows = (n,)
    if out is None:
        token, prob, kept = torch.empty(3, n, dtype=_I32, device=logits.device).unbind()
        out = Sampled(token, prob.view(_F32), kept)
    _call("minicpmo_gpu_sample", dev, logits.data_ptr(), dtype, n, vocab, logits.stride(0) if n > 1 else vocab,
          None if temperature is None else _tensor(op, "temperature", temperature, dev, _F32, rows),
          None if top_k is None else _tensor(op, "top_k", top_k, dev, _I32, rows),
          None if top_p is None else _tensor(op, "top_p", top_p, dev, _F32, rows),
          None if min_p is None else _tensor(op, "min_p", min_p, dev, _F32, rows),
          _tensor(op, "uniform", uniform, dev, _F32, rows), _tensor(op, "out.token", out.token, dev, _I32, rows),
          _tensor(op, "out.prob", out.prob, dev, _F32, rows), _tensor(op, "out.kept", out.kept, dev, _I32, rows))
    return out
