"""Many sequences on one device: a paged key-value cache and the operators of
a batched step (mlq_paged_* and mlq_qk_norm_rope, include/mlq.h). The
reference serves one sequence; this has no counterpart there.

A step of a serving loop, all stream-ordered and with no host round trip:

    plan(batch, batch.lengths, n_new, free_pages, n_free, cache.page_size)
    per layer, with the rows' fused q | k | v projection in `qkv`:
        qk_norm_rope(rotary, q, k, v, batch.positions, q_out=q, cache=cache, layer=i,
                     slots=batch.slots)
        attention_decode(cache, i, batch, q, max_len=...)    # one new token each, or
        attention_prefill(cache, i, batch, q)                # any numbers of them

Activations are float32, the cache float32, float16 or bfloat16. Tensors are
passed as they are: q, k, v and outputs are [rows, heads, head_dim] with any
row stride (views of a fused projection), heads contiguous. There is no CPU
fallback. Tensors of a call live on one device; it need not be the current
one. Given a `stream`, the call's work is ordered on it and so must be the
tensors.
"""
from __future__ import annotations

import contextlib
import ctypes

import numpy as np

from . import (ROPE_NEOX, ROPE_NORMAL, MlqAttentionRule, MlqPagedBatch, MlqPagedCache, MlqRotary,
               _check, _stream, lib)

__all__ = ["ROPE_NEOX", "ROPE_NORMAL", "PLAN_STATUS", "PagedCache", "PagedBatch", "Rotary",
           "AttentionRule", "plan", "rope_frequencies", "qk_norm_rope", "attention_decode",
           "attention_prefill", "attention_workspace_bytes"]

PLAN_STATUS = {0: "ok", 1: "count out of range", 2: "more rows than the batch holds",
               3: "not enough free pages"}
SCALINGS = {"none": 0, "linear": 1, "parts": 2}


def _kv_type(dtype) -> int:
    import torch
    types = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
    if dtype not in types:
        raise ValueError("the cache must be float32, float16 or bfloat16")
    return types[dtype]


def _ints(name: str, t, dtype, shape, device):
    """t itself, checked: a contiguous device tensor of that type and shape
    (None in shape: any size)."""
    if t.dtype != dtype or not t.is_cuda or not t.is_contiguous() or t.device != device or \
       t.dim() != len(shape) or any(s is not None and s != n for s, n in zip(shape, t.shape)):
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {list(shape)} on "
                         f"{device}")
    return t


def _rows(name: str, t, heads, head_dim: int, device):
    """Row stride of a [rows, heads, head_dim] float32 tensor whose heads are
    contiguous."""
    import torch
    if t.dtype != torch.float32 or t.device != device or t.dim() != 3 or \
       t.shape[2] != head_dim or (heads is not None and t.shape[1] != heads):
        raise ValueError(f"{name} must be float32 [rows, {heads or 'heads'}, {head_dim}] on "
                         f"{device}")
    if t.stride(2) != 1 or (t.shape[1] > 1 and t.stride(1) != head_dim):
        raise ValueError(f"the heads of {name} must lie side by side")
    # (a single row's stride says nothing)
    return t.stride(0) if t.shape[0] > 1 else t.shape[1] * head_dim


@contextlib.contextmanager
def _switched(device):
    import torch
    with torch.cuda.device(device):
        yield


def _on(device):
    """The call's device made current where it is not."""
    import torch
    if device.index is None or device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return _switched(device)


class PagedCache:
    """keys and values [n_layers, n_pages, n_kv_heads, page_size, head_dim]."""

    def __init__(self, keys, values):
        if keys.dim() != 5 or keys.shape != values.shape or keys.dtype != values.dtype or \
           keys.device != values.device or not keys.is_cuda or not keys.is_contiguous() or \
           not values.is_contiguous():
            raise ValueError("keys and values must be contiguous device tensors [n_layers, "
                             "n_pages, n_kv_heads, page_size, head_dim] of one type and device")
        self.keys, self.values, self.device = keys, values, keys.device
        self.n_layers, self.n_pages, self.n_kv_heads, self.page_size, self.head_dim = keys.shape
        self.struct = MlqPagedCache(keys.data_ptr(), values.data_ptr(), _kv_type(keys.dtype),
                                    self.n_layers, self.n_pages, self.page_size, self.n_kv_heads,
                                    self.head_dim)
        nbytes = ctypes.c_size_t()
        _check(lib().mlq_paged_cache_bytes(ctypes.byref(self.struct), ctypes.byref(nbytes)),
               "mlq_paged_cache_bytes")
        self.nbytes = 2 * nbytes.value

    @classmethod
    def empty(cls, n_layers: int, n_pages: int, page_size: int, n_kv_heads: int, head_dim: int,
              dtype=None, device: str = "cuda") -> "PagedCache":
        """Uninitialised pages: what lies behind a sequence's end is never used."""
        import torch
        shape = (n_layers, n_pages, n_kv_heads, page_size, head_dim)
        dtype = torch.float32 if dtype is None else dtype
        return cls(torch.empty(shape, dtype=dtype, device=device),
                   torch.empty(shape, dtype=dtype, device=device))


class PagedBatch:
    """The device arrays of a batch (mlq_paged_batch): block_table int32
    [n_seqs, max_pages], lengths int32 [n_seqs], row_start int32 [n_seqs + 1]
    (None for a decode batch whose row i is sequence i), and for plan():
    positions int32 and slots int64 [max_rows], status int32 [1]."""

    def __init__(self, block_table, lengths, row_start=None, positions=None, slots=None,
                 status=None, max_rows: int | None = None):
        import torch
        dev = block_table.device
        n_seqs, max_pages = block_table.shape
        i32, i64 = torch.int32, torch.int64
        _ints("block_table", block_table, i32, (None, None), dev)
        _ints("lengths", lengths, i32, (n_seqs,), dev)
        if row_start is not None:
            _ints("row_start", row_start, i32, (n_seqs + 1,), dev)
        if positions is not None:
            _ints("positions", positions, i32, (max_rows,), dev)
            max_rows = positions.shape[0]
        if slots is not None:
            _ints("slots", slots, i64, (max_rows,), dev)
        if status is not None:
            _ints("status", status, i32, (1,), dev)
        self.block_table, self.lengths, self.row_start = block_table, lengths, row_start
        self.positions, self.slots, self.status = positions, slots, status
        self.device, self.n_seqs, self.max_pages, self.max_rows = dev, n_seqs, max_pages, max_rows
        ptr = [t.data_ptr() if t is not None else None
               for t in (block_table, lengths, row_start, positions, slots, status)]
        self.struct = MlqPagedBatch(n_seqs, max_pages, max_rows or 0, *ptr)

    @classmethod
    def empty(cls, n_seqs: int, max_pages: int, max_rows: int,
              device: str = "cuda") -> "PagedBatch":
        """A batch of sequences without tokens; every table entry -1."""
        import torch
        i32 = dict(dtype=torch.int32, device=device)
        return cls(torch.full((n_seqs, max_pages), -1, **i32), torch.zeros(n_seqs, **i32),
                   torch.zeros(n_seqs + 1, **i32), torch.full((max_rows,), -1, **i32),
                   torch.full((max_rows,), -1, dtype=torch.int64, device=device),
                   torch.zeros(1, **i32))


def plan(batch: PagedBatch, lengths, n_new, free_pages, n_free, page_size: int, n_free_out=None,
         stream=None) -> None:
    """One step's pages, positions and slots (mlq_paged_plan). lengths: before
    the step (batch.lengths itself in a serving loop); n_new: new tokens of
    each sequence, -1 ends it; free_pages: the stack of free pages, its size
    the number of pages of the cache; n_free int32 [1]: its height, updated in
    place unless n_free_out is given. batch.status says whether the step was
    planned (PLAN_STATUS)."""
    import torch
    dev, i32 = batch.device, torch.int32
    if batch.row_start is None or batch.positions is None or batch.slots is None or \
       batch.status is None:
        raise ValueError("plan needs a batch with row_start, positions, slots and status")
    _ints("lengths", lengths, i32, (batch.n_seqs,), dev)
    _ints("n_new", n_new, i32, (batch.n_seqs,), dev)
    _ints("free_pages", free_pages, i32, (None,), dev)
    _ints("n_free", n_free, i32, (1,), dev)
    out = n_free if n_free_out is None else _ints("n_free_out", n_free_out, i32, (1,), dev)
    with _on(dev):
        _check(lib().mlq_paged_plan(ctypes.byref(batch.struct), page_size, free_pages.shape[0],
                                    lengths.data_ptr(), n_new.data_ptr(), free_pages.data_ptr(),
                                    n_free.data_ptr(), out.data_ptr(), _stream(stream)),
               "mlq_paged_plan")


def rope_frequencies(theta: float, rot_dim: int, scaling: str = "none", factor: float = 1.0,
                     original_len: int = 0, beta_fast: float = 32.0, beta_slow: float = 1.0):
    """(radians per position of each rotated pair as float64 [rot_dim / 2],
    magnitude) of mlq_rope_frequencies; scaling "none", "linear" or "parts"
    (YaRN)."""
    if scaling not in SCALINGS:
        raise ValueError(f"scaling must be one of {sorted(SCALINGS)}")
    freqs = np.zeros(max(rot_dim // 2, 1), np.float64)
    magnitude = ctypes.c_float()
    _check(lib().mlq_rope_frequencies(theta, rot_dim, SCALINGS[scaling], factor, original_len,
                                      beta_fast, beta_slow,
                                      freqs.ctypes.data_as(ctypes.POINTER(ctypes.c_double)),
                                      ctypes.byref(magnitude)), "mlq_rope_frequencies")
    return freqs, magnitude.value


class Rotary:
    """What a model does to each query and key head (mlq_rotary): freqs, a
    float64 device tensor [rot_dim / 2] of radians per position (None: no
    rotation), and the float32 norm weights [head_dim] of queries and keys."""

    def __init__(self, head_dim: int, freqs=None, rope_type: int = ROPE_NEOX,
                 magnitude: float = 1.0, q_norm=None, k_norm=None, eps: float = 1e-6):
        import torch
        for name, t, dtype in (("freqs", freqs, torch.float64), ("q_norm", q_norm, torch.float32),
                               ("k_norm", k_norm, torch.float32)):
            if t is None:
                continue
            if t.dtype != dtype or not t.is_cuda or t.dim() != 1 or not t.is_contiguous() or \
               (name != "freqs" and t.shape[0] != head_dim):
                raise ValueError(f"{name} must be a contiguous {dtype} device vector" +
                                 ("" if name == "freqs" else f" of {head_dim}"))
        given = [t for t in (freqs, q_norm, k_norm) if t is not None]
        if len({t.device for t in given}) > 1:
            raise ValueError("freqs and norms must be on one device")
        self.device = given[0].device if given else None
        self.head_dim = head_dim
        self.rot_dim = 2 * freqs.shape[0] if freqs is not None else 0
        self._keep = given
        self.struct = MlqRotary(head_dim, self.rot_dim, rope_type, magnitude, eps,
                                *(t.data_ptr() if t is not None else None
                                  for t in (freqs, q_norm, k_norm)))


def qk_norm_rope(rotary: Rotary, q, k, v, positions, q_out=None, k_out=None, cache=None,
                 layer: int = 0, slots=None, stream=None):
    """Queries and keys normalised per head and rotated to their positions;
    with a cache, keys and values stored at their slots (mlq_qk_norm_rope).
    Returns (q_out, k_out): q_out (a new tensor unless given; q itself for in
    place) and k_out (new only where there is no cache). Rows whose position
    is negative are left as they were in every output."""
    import torch
    dev, hd = q.device, rotary.head_dim
    if not q.is_cuda or (rotary.device is not None and rotary.device != dev):
        raise ValueError("q must be a device tensor, on the device of the rotary")
    qs = _rows("q", q, None, hd, dev)
    n, heads = q.shape[:2]
    ks = _rows("k", k, None, hd, dev)
    kv = k.shape[1]
    if k.shape[0] != n:
        raise ValueError("q and k must have the same rows")
    _ints("positions", positions, torch.int32, (None,), dev)
    if positions.shape[0] < n:
        raise ValueError("a position for each row is needed")
    vs = 0
    if cache is not None:
        vs = _rows("v", v, kv, hd, dev)
        if cache.device != dev or v.shape[0] != n or slots is None:
            raise ValueError("v and slots of every row, on the cache's device, are needed")
        _ints("slots", slots, torch.int64, (None,), dev)
        if slots.shape[0] < n:
            raise ValueError("a slot for each row is needed")
    with _on(dev), _allocating(stream):
        if q_out is None:
            q_out = torch.empty((n, heads, hd), dtype=torch.float32, device=dev)
        if k_out is None and cache is None:
            k_out = torch.empty((n, kv, hd), dtype=torch.float32, device=dev)
        qos = _rows("q_out", q_out, heads, hd, dev)
        kos = _rows("k_out", k_out, kv, hd, dev) if k_out is not None else 0
        if q_out.shape[0] != n or (k_out is not None and k_out.shape[0] != n):
            raise ValueError("the outputs must have the rows of q")
        if n == 0:
            return q_out, k_out
        _check(lib().mlq_qk_norm_rope(
            ctypes.byref(rotary.struct), n, positions.data_ptr(), heads, kv, q.data_ptr(), qs,
            k.data_ptr(), ks, v.data_ptr() if cache is not None else None, vs, q_out.data_ptr(),
            qos, k_out.data_ptr() if k_out is not None else None, kos,
            ctypes.byref(cache.struct) if cache is not None else None, layer,
            slots.data_ptr() if cache is not None else None, _stream(stream)),
               "mlq_qk_norm_rope")
    return q_out, k_out


class AttentionRule:
    """How scores enter the softmax (mlq_attention_rule): scale (None:
    1 / sqrt(head_dim)), softcap, window and slopes, a float32 device tensor
    [n_heads] of biases per token of distance."""

    def __init__(self, scale: float | None = None, softcap: float = 0.0, window: int = 0,
                 slopes=None):
        import torch
        if scale == 0.0:
            raise ValueError("a scale of 0 would weigh every key alike")
        if slopes is not None and (slopes.dtype != torch.float32 or not slopes.is_cuda or
                                   slopes.dim() != 1 or not slopes.is_contiguous()):
            raise ValueError("slopes must be a contiguous float32 device vector")
        self.slopes = slopes
        self.struct = MlqAttentionRule(scale or 0.0, softcap, window,
                                       slopes.data_ptr() if slopes is not None else None)


def attention_workspace_bytes(cache: PagedCache, n_heads: int, n_seqs: int, max_len: int) -> int:
    """Workspace of attention_decode for any lengths up to max_len."""
    nbytes = ctypes.c_size_t()
    _check(lib().mlq_paged_attention_workspace(ctypes.byref(cache.struct), n_heads, n_seqs,
                                               max_len, ctypes.byref(nbytes)),
           "mlq_paged_attention_workspace")
    return nbytes.value


def _allocating(stream):
    """What is allocated inside belongs to `stream` (the current one if None):
    the allocator reuses it in that stream's order."""
    import torch
    return contextlib.nullcontext() if stream is None else torch.cuda.stream(stream)


def _attention_args(cache, batch, q, out, rule):
    import torch
    dev, hd = cache.device, cache.head_dim
    if batch.device != dev:
        raise ValueError("the batch must be on the cache's device")
    qs = _rows("q", q, None, hd, dev)
    heads = q.shape[1]
    if rule is not None and rule.slopes is not None and \
       (rule.slopes.shape[0] != heads or rule.slopes.device != dev):
        raise ValueError("slopes must have a value for each head, on the cache's device")
    if out is None:
        # (rows that the call does not compute keep zeros)
        out = torch.zeros((q.shape[0], heads, hd), dtype=torch.float32, device=dev)
    os = _rows("out", out, heads, hd, dev)
    if out.shape[0] != q.shape[0]:
        raise ValueError("out must have the rows of q")
    return heads, qs, out, os


def _bounded(batch, rows: int):
    """The batch's struct with max_rows held to the rows that q has."""
    s = batch.struct
    if s.max_rows == rows:
        return s
    most = min(s.max_rows, rows) if batch.max_rows is not None else rows
    return MlqPagedBatch(s.n_seqs, s.max_pages, most, s.block_table, s.lengths, s.row_start,
                         s.positions, s.slots, s.status)


def attention_decode(cache: PagedCache, layer: int, batch: PagedBatch, q, out=None,
                     rule: AttentionRule | None = None, max_len: int | None = None,
                     workspace=None, stream=None):
    """out [rows, n_heads, head_dim]: attention of each sequence's last row
    over its pages (mlq_paged_attention_decode). max_len bounds the lengths
    (None: what the block table can hold; a longer sequence gives NaN).
    workspace: a uint8 device tensor of attention_workspace_bytes, or None for
    one of the call's own."""
    import torch
    with _on(cache.device), _allocating(stream):
        heads, qs, out, os = _attention_args(cache, batch, q, out, rule)
        if batch.row_start is None and q.shape[0] < batch.n_seqs:
            raise ValueError("a row for each sequence is needed")
        max_len = batch.max_pages * cache.page_size if max_len is None else int(max_len)
        if workspace is None:
            need = attention_workspace_bytes(cache, heads, batch.n_seqs, max_len)
            if need:
                workspace = torch.empty(need, dtype=torch.uint8, device=cache.device)
        if q.shape[0]:
            _check(lib().mlq_paged_attention_decode(
                ctypes.byref(cache.struct), layer, ctypes.byref(_bounded(batch, q.shape[0])),
                ctypes.byref(rule.struct) if rule is not None else None, heads, q.data_ptr(), qs,
                out.data_ptr(), os, max_len,
                workspace.data_ptr() if workspace is not None else None,
                workspace.numel() * workspace.element_size() if workspace is not None else 0,
                _stream(stream)), "mlq_paged_attention_decode")
    return out


def attention_prefill(cache: PagedCache, layer: int, batch: PagedBatch, q, out=None,
                      rule: AttentionRule | None = None, stream=None):
    """out [rows, n_heads, head_dim]: causal attention of every new row of
    every sequence over its pages (mlq_paged_attention_prefill)."""
    with _on(cache.device), _allocating(stream):
        heads, qs, out, os = _attention_args(cache, batch, q, out, rule)
        if batch.row_start is None:
            raise ValueError("attention_prefill needs a batch with row_start")
        if q.shape[0]:
            _check(lib().mlq_paged_attention_prefill(
                ctypes.byref(cache.struct), layer, ctypes.byref(_bounded(batch, q.shape[0])),
                ctypes.byref(rule.struct) if rule is not None else None, heads, q.data_ptr(), qs,
                out.data_ptr(), os, _stream(stream)), "mlq_paged_attention_prefill")
    return out
