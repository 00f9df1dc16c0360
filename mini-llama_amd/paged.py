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

Where some sequences bring one token and others a prompt, a batch whose
sequences are in that order is two: PagedBatch of block_table[:n], lengths[:n]
and row_start[:n + 1] for attention_decode, of [n:] of each for
attention_prefill, both with the whole step's q and out. attention_prefill alone
takes any mixture, but a workgroup walks all keys of a sequence if the batch has
rows enough to fill the chip: long contexts belong to attention_decode.

Activations are float32, the cache float32, float16 or bfloat16. Tensors are
passed as they are: q, k, v and outputs are [rows, heads, head_dim] with any
row stride (views of a fused projection), heads contiguous. There is no CPU
fallback. Tensors of a call live on one device; it need not be the current
one. Given a `stream`, the call's work is ordered on it and so must be the
tensors. Forward only: outputs carry no gradients.
"""
from __future__ import annotations

import ctypes

import numpy as np
import torch

from . import (ROPE_NEOX, ROPE_NORMAL, MlqAttentionRule, MlqPagedBatch, MlqPagedCache, MlqRotary,
               _check, lib)

__all__ = ["ROPE_NEOX", "ROPE_NORMAL", "PLAN_STATUS", "PagedCache", "PagedBatch", "Rotary",
           "AttentionRule", "plan", "rope_frequencies", "qk_norm_rope", "attention_decode",
           "attention_prefill", "attention_workspace_bytes"]

PLAN_STATUS = {0: "ok", 1: "count out of range", 2: "more rows than the batch holds",
               3: "not enough free pages"}
SCALINGS = {"none": 0, "linear": 1, "parts": 2}
_KV_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_F32, _I32, _I64 = torch.float32, torch.int32, torch.int64

# A step's calls are a few microseconds each: the checks below ask a tensor for
# as little as they can, and the stream's handle is taken without a Stream
# object where torch gives it.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _elsewhere(call, index: int, stream):
    """call() with the tensors' device current, and `stream` (if given) the
    current stream: what it allocates then belongs to that stream."""
    if stream is None:
        with torch.cuda.device(index):
            return call()
    if stream.device.index != index:
        raise ValueError("the stream must be on the tensors' device")
    with torch.cuda.stream(stream):
        return call()


def _int32(name: str, value) -> int:
    """value, if a C int holds it (ctypes keeps the low 32 bits of any other)."""
    if not -(1 << 31) <= value < 1 << 31:
        raise ValueError(f"{name} does not fit 32 bits")
    return value


def _ints(name: str, t, dtype, index: int, n=None, least: int = 0):
    """Address of a contiguous 1-D device tensor of that type with n elements
    (or at least `least`)."""
    size = t.shape
    if t.dtype is dtype and len(size) == 1 and t.get_device() == index and t.is_contiguous():
        if size[0] == n or (n is None and size[0] >= least):
            return t.data_ptr()
    size = n if n is not None else f"at least {least}" if least else "any number of"
    raise ValueError(f"{name} must be a contiguous {dtype} tensor of {size} elements on "
                     f"cuda:{index}")


def _rows(name: str, t, rows, heads, head_dim: int, index: int):
    """(address, row stride) of a [rows, heads, head_dim] float32 tensor whose
    heads lie side by side; rows, heads None: any."""
    if t.dtype is _F32 and t.dim() == 3 and t.get_device() == index:
        n, h, d = t.shape
        if d == head_dim and (h == heads or heads is None) and (n == rows or rows is None):
            s0, s1, s2 = t.stride()
            if s2 == 1 and (s1 == d or h <= 1):
                # (a single row's stride says nothing)
                return t.data_ptr(), s0 if n > 1 else h * d
            raise ValueError(f"the heads of {name} must lie side by side")
    raise ValueError(f"{name} must be float32 [{'rows' if rows is None else rows}, "
                     f"{'heads' if heads is None else heads}, {head_dim}] on cuda:{index}")


class _Fixed:
    """Attributes that are set once. The C structs hold the tensors' addresses:
    another tensor in a tensor's place would not reach the device, and the old
    one's memory could be given away under the kernels' writes."""

    def __setattr__(self, name, value):
        if name in self.__dict__:
            raise AttributeError(f"{type(self).__name__}.{name} cannot be replaced: write into the "
                                 "tensor, or make another object")
        self.__dict__[name] = value

    def __delattr__(self, name):
        raise AttributeError(f"{type(self).__name__}.{name} cannot be deleted")


class PagedCache(_Fixed):
    """keys and values [n_layers, n_pages, n_kv_heads, page_size, head_dim]."""

    def __init__(self, keys, values):
        if keys.dtype not in _KV_TYPES:
            raise ValueError("the cache must be float32, float16 or bfloat16")
        if keys.dim() != 5 or keys.shape != values.shape or keys.dtype != values.dtype or \
           keys.device != values.device or not keys.is_cuda or not keys.is_contiguous() or \
           not values.is_contiguous():
            raise ValueError("keys and values must be contiguous device tensors [n_layers, "
                             "n_pages, n_kv_heads, page_size, head_dim] of one type and device")
        self.keys, self.values, self.device = keys, values, keys.device
        self.n_layers, self.n_pages, self.n_kv_heads, self.page_size, self.head_dim = keys.shape
        self.struct = MlqPagedCache(keys.data_ptr(), values.data_ptr(), _KV_TYPES[keys.dtype],
                                    self.n_layers, self.n_pages, self.page_size, self.n_kv_heads,
                                    self.head_dim)
        self.ref = ctypes.byref(self.struct)
        self.index = keys.get_device()
        self._workspaces = {}  # bytes by (n_heads, n_seqs, rows, max_len)
        nbytes = ctypes.c_size_t()
        _check(lib().mlq_paged_cache_bytes(self.ref, ctypes.byref(nbytes)),
               "mlq_paged_cache_bytes")
        self.nbytes = 2 * nbytes.value

    @classmethod
    def empty(cls, n_layers: int, n_pages: int, page_size: int, n_kv_heads: int, head_dim: int,
              dtype=None, device: str = "cuda") -> "PagedCache":
        """Uninitialised pages: what lies behind a sequence's end is never used."""
        shape = (n_layers, n_pages, n_kv_heads, page_size, head_dim)
        dtype = torch.float32 if dtype is None else dtype
        return cls(torch.empty(shape, dtype=dtype, device=device),
                   torch.empty(shape, dtype=dtype, device=device))


class PagedBatch(_Fixed):
    """The device arrays of a batch (mlq_paged_batch): block_table int32
    [n_seqs, max_pages], lengths int32 [n_seqs], row_start int32 [n_seqs + 1]
    (None for a decode batch whose row i is sequence i), and for plan():
    positions int32 and slots int64 [max_rows], status int32 [1]. What they hold
    may change, the tensors themselves are the batch's for good."""

    def __init__(self, block_table, lengths, row_start=None, positions=None, slots=None,
                 status=None):
        if block_table.dim() != 2 or block_table.dtype is not _I32 or not block_table.is_cuda or \
           not block_table.is_contiguous():
            raise ValueError("block_table must be a contiguous int32 device tensor [n_seqs, "
                             "max_pages]")
        n_seqs, max_pages = block_table.shape
        index = block_table.get_device()
        max_rows = positions.shape[0] if positions is not None else None
        ptr = [block_table.data_ptr()]
        for name, x, dtype, n in (("lengths", lengths, _I32, n_seqs),
                                  ("row_start", row_start, _I32, n_seqs + 1),
                                  ("positions", positions, _I32, None),
                                  ("slots", slots, _I64, max_rows), ("status", status, _I32, 1)):
            ptr.append(_ints(name, x, dtype, index, n) if x is not None else None)
        self.block_table, self.lengths, self.row_start = block_table, lengths, row_start
        self.positions, self.slots, self.status = positions, slots, status
        self.device, self.index = block_table.device, index
        self.n_seqs, self.max_pages, self.max_rows = n_seqs, max_pages, max_rows
        self.struct = MlqPagedBatch(n_seqs, max_pages, max_rows or 0, *ptr)
        self.ref = ctypes.byref(self.struct)
        self._bounded = {}  # the struct with max_rows held to a number of rows

    def bounded(self, rows: int):
        """The struct's reference with max_rows held to the rows that q has."""
        most = rows if self.max_rows is None else min(self.max_rows, rows)
        if most == self.struct.max_rows:
            return self.ref
        ref = self._bounded.get(most)
        if ref is None:
            s = self.struct
            ref = ctypes.byref(MlqPagedBatch(s.n_seqs, s.max_pages, most, s.block_table, s.lengths,
                                             s.row_start, s.positions, s.slots, s.status))
            if len(self._bounded) >= 64:
                self._bounded.clear()
            self._bounded[most] = ref
        return ref

    @classmethod
    def empty(cls, n_seqs: int, max_pages: int, max_rows: int,
              device: str = "cuda") -> "PagedBatch":
        """A batch of sequences without tokens; every table entry -1."""
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
    index, n = batch.index, batch.n_seqs
    if stream is not None or index != _current_device():
        return _elsewhere(lambda: plan(batch, lengths, n_new, free_pages, n_free, page_size,
                                       n_free_out), index, stream)
    if batch.row_start is None or batch.positions is None or batch.slots is None or \
       batch.status is None:
        raise ValueError("plan needs a batch with row_start, positions, slots and status")
    height = _ints("n_free", n_free, _I32, index, 1)
    stack = _ints("free_pages", free_pages, _I32, index)
    _check(lib().mlq_paged_plan(
        batch.ref, _int32("page_size", page_size), _int32("the size of free_pages", free_pages.shape[0]),
        _ints("lengths", lengths, _I32, index, n), _ints("n_new", n_new, _I32, index, n), stack, height,
        height if n_free_out is None else _ints("n_free_out", n_free_out, _I32, index, 1),
        _raw_stream(index)), "mlq_paged_plan")


def rope_frequencies(theta: float, rot_dim: int, scaling: str = "none", factor: float = 1.0,
                     original_len: int = 0, beta_fast: float = 32.0, beta_slow: float = 1.0):
    """(radians per position of each rotated pair as float64 [rot_dim / 2],
    magnitude) of mlq_rope_frequencies; scaling "none", "linear" or "parts"
    (YaRN)."""
    if scaling not in SCALINGS:
        raise ValueError(f"scaling must be one of {sorted(SCALINGS)}")
    _int32("original_len", original_len)
    freqs = np.zeros(max(_int32("rot_dim", rot_dim) // 2, 1), np.float64)
    magnitude = ctypes.c_float()
    _check(lib().mlq_rope_frequencies(theta, rot_dim, SCALINGS[scaling], factor, original_len,
                                      beta_fast, beta_slow,
                                      freqs.ctypes.data_as(ctypes.POINTER(ctypes.c_double)),
                                      ctypes.byref(magnitude)), "mlq_rope_frequencies")
    return freqs, magnitude.value


class Rotary(_Fixed):
    """What a model does to each query and key head (mlq_rotary): freqs, a
    float64 device tensor [rot_dim / 2] of radians per position (None: no
    rotation), and the float32 norm weights [head_dim] of queries and keys."""

    def __init__(self, head_dim: int, freqs=None, rope_type: int = ROPE_NEOX,
                 magnitude: float = 1.0, q_norm=None, k_norm=None, eps: float = 1e-6):
        for name, t, dtype in (("freqs", freqs, torch.float64), ("q_norm", q_norm, torch.float32),
                               ("k_norm", k_norm, torch.float32)):
            if t is None:
                continue
            if t.dtype != dtype or not t.is_cuda or t.dim() != 1 or not t.is_contiguous() or \
               (name != "freqs" and t.shape[0] != head_dim):
                raise ValueError(f"{name} must be a contiguous {dtype} device vector" +
                                 ("" if name == "freqs" else f" of {head_dim}"))
        _int32("rope_type", rope_type)
        given = [t for t in (freqs, q_norm, k_norm) if t is not None]
        if len({t.device for t in given}) > 1:
            raise ValueError("freqs and norms must be on one device")
        self.index = given[0].get_device() if given else None
        self.head_dim = head_dim
        self.rot_dim = 2 * freqs.shape[0] if freqs is not None else 0
        self._keep = given
        self.struct = MlqRotary(head_dim, self.rot_dim, rope_type, magnitude, eps,
                                *(t.data_ptr() if t is not None else None
                                  for t in (freqs, q_norm, k_norm)))
        self.ref = ctypes.byref(self.struct)


def qk_norm_rope(rotary: Rotary, q, k, v, positions, q_out=None, k_out=None, cache=None,
                 layer: int = 0, slots=None, stream=None):
    """Queries and keys normalised per head and rotated to their positions;
    with a cache, keys and values stored at their slots (mlq_qk_norm_rope).
    Returns (q_out, k_out): q_out (a new tensor unless given; q itself for in
    place) and k_out (new only where there is no cache). Rows whose position
    is negative are left as they were in every output."""
    index, hd = q.get_device(), rotary.head_dim
    if index < 0 or (rotary.index is not None and rotary.index != index):
        raise ValueError("q must be a device tensor, on the device of the rotary")
    if stream is not None or index != _current_device():
        return _elsewhere(lambda: qk_norm_rope(rotary, q, k, v, positions, q_out, k_out, cache, layer,
                                               slots), index, stream)
    qp, qs = _rows("q", q, None, None, hd, index)
    q_shape = q.shape
    n, heads = q_shape[0], q_shape[1]
    kp, ks = _rows("k", k, n, None, hd, index)
    k_shape = k.shape
    kv = k_shape[1]
    vp = sp = cp = kop = None
    vs = kos = 0
    if cache is not None:
        if cache.index != index or v is None or slots is None:
            raise ValueError("v and slots, on the cache's device, are needed")
        _int32("layer", layer)
        vp, vs = _rows("v", v, n, kv, hd, index)
        sp, cp = _ints("slots", slots, _I64, index, None, n), cache.ref
    elif k_out is None:
        k_out = torch.empty(k_shape, dtype=_F32, device=q.device)
    if q_out is None:
        q_out = torch.empty(q_shape, dtype=_F32, device=q.device)
    qop, qos = (qp, qs) if q_out is q else _rows("q_out", q_out, n, heads, hd, index)
    if k_out is not None:
        kop, kos = _rows("k_out", k_out, n, kv, hd, index)
    pp = _ints("positions", positions, _I32, index, None, n)
    if n:
        _check(lib().mlq_qk_norm_rope(rotary.ref, n, pp, heads, kv, qp, qs, kp, ks, vp, vs, qop, qos,
                                      kop, kos, cp, layer, sp, _raw_stream(index)),
               "mlq_qk_norm_rope")
    return q_out, k_out


class AttentionRule(_Fixed):
    """How scores enter the softmax (mlq_attention_rule): scale (None:
    1 / sqrt(head_dim)), softcap, window and slopes, a float32 device tensor
    [n_heads] of biases per token of distance."""

    def __init__(self, scale: float | None = None, softcap: float = 0.0, window: int = 0,
                 slopes=None):
        if scale is not None and ctypes.c_float(scale).value == 0.0:
            raise ValueError("a scale of 0 (in float32) would weigh every key alike")
        if softcap != 0.0 and ctypes.c_float(softcap).value == 0.0:
            raise ValueError("a softcap that is 0 in float32 would be none")
        if not 0 <= window < 1 << 31:
            raise ValueError("a window is a number of keys below 2^31 (0: none)")
        if slopes is not None and (slopes.dtype != torch.float32 or not slopes.is_cuda or
                                   slopes.dim() != 1 or not slopes.is_contiguous()):
            raise ValueError("slopes must be a contiguous float32 device vector")
        self.slopes = slopes
        self.struct = MlqAttentionRule(scale or 0.0, softcap, window,
                                       slopes.data_ptr() if slopes is not None else None)
        self.ref = ctypes.byref(self.struct)


def attention_workspace_bytes(cache: PagedCache, n_heads: int, n_seqs: int, max_len: int,
                              rows: int = 0) -> int:
    """Workspace of attention_decode for any lengths up to max_len, with rows
    that of attention_prefill for so many rows."""
    key = (n_heads, n_seqs, rows, max_len)
    need = cache._workspaces.get(key)
    if need is None:
        for name, value in zip(("n_heads", "n_seqs", "rows", "max_len"), key):
            _int32(name, value)
        nbytes = ctypes.c_size_t()
        _check(lib().mlq_paged_attention_workspace(cache.ref, n_heads, n_seqs, rows, max_len,
                                                   ctypes.byref(nbytes)),
               "mlq_paged_attention_workspace")
        need = nbytes.value
        if len(cache._workspaces) >= 256:
            cache._workspaces.clear()
        cache._workspaces[key] = need
    return need


def _workspace(cache, workspace, n_heads: int, n_seqs: int, max_len: int, rows: int):
    """(tensor, address, bytes): the caller's workspace, or one of the call's
    own, which the allocator reuses in the current stream's order."""
    if workspace is None:
        size = attention_workspace_bytes(cache, n_heads, n_seqs, max_len, rows)
        if size == 0:
            return None, None, 0
        workspace = torch.empty(size, dtype=torch.uint8, device=cache.device)
        return workspace, workspace.data_ptr(), size
    _int32("max_len", max_len)
    if workspace.get_device() != cache.index or not workspace.is_contiguous():
        raise ValueError("the workspace must be a contiguous tensor on the cache's device")
    return workspace, workspace.data_ptr(), workspace.numel() * workspace.element_size()


def _attention_args(cache, layer, batch, q, out, rule):
    """(heads, q's address and stride, out, its address and stride, the rule's
    reference), checked."""
    index, hd = cache.index, cache.head_dim
    if batch.index != index:
        raise ValueError("the batch must be on the cache's device")
    _int32("layer", layer)
    qp, qs = _rows("q", q, None, None, hd, index)
    n, heads = q.shape[:2]
    ref = None
    if rule is not None:
        if rule.slopes is not None and (rule.slopes.shape[0] != heads or
                                        rule.slopes.get_device() != index):
            raise ValueError("slopes must have a value for each head, on the cache's device")
        ref = rule.ref
    if out is None:
        # (rows that the call does not compute keep zeros)
        out = torch.zeros((n, heads, hd), dtype=_F32, device=q.device)
    op, os = _rows("out", out, n, heads, hd, index)
    return heads, qp, qs, out, op, os, ref


def attention_decode(cache: PagedCache, layer: int, batch: PagedBatch, q, out=None,
                     rule: AttentionRule | None = None, max_len: int | None = None,
                     workspace=None, stream=None):
    """out [rows, n_heads, head_dim]: attention of each sequence's last row
    over its pages (mlq_paged_attention_decode). max_len bounds the lengths
    (None: what the block table can hold; a longer sequence gives NaN).
    workspace: a uint8 device tensor of attention_workspace_bytes, or None for
    one of the call's own."""
    index = cache.index
    if stream is not None or index != _current_device():
        return _elsewhere(lambda: attention_decode(cache, layer, batch, q, out, rule, max_len,
                                                   workspace), index, stream)
    heads, qp, qs, out, op, os, ref = _attention_args(cache, layer, batch, q, out, rule)
    n = q.shape[0]
    if batch.row_start is None and n < batch.n_seqs:
        raise ValueError("a row for each sequence is needed")
    if max_len is None:
        max_len = batch.max_pages * cache.page_size
    workspace, wp, size = _workspace(cache, workspace, heads, batch.n_seqs, max_len, 0)
    if n:
        _check(lib().mlq_paged_attention_decode(cache.ref, layer, batch.bounded(n), ref, heads, qp, qs,
                                                op, os, max_len, wp, size, _raw_stream(index)),
               "mlq_paged_attention_decode")
    return out


def attention_prefill(cache: PagedCache, layer: int, batch: PagedBatch, q, out=None,
                      rule: AttentionRule | None = None, max_len: int | None = None,
                      workspace=None, stream=None):
    """out [rows, n_heads, head_dim]: causal attention of every new row of
    every sequence over its pages (mlq_paged_attention_prefill). max_len and
    workspace as in attention_decode, the workspace of
    attention_workspace_bytes(..., rows) for the rows that q has, or the batch
    if it holds fewer (batch.max_rows)."""
    index = cache.index
    if stream is not None or index != _current_device():
        return _elsewhere(lambda: attention_prefill(cache, layer, batch, q, out, rule, max_len,
                                                    workspace), index, stream)
    heads, qp, qs, out, op, os, ref = _attention_args(cache, layer, batch, q, out, rule)
    if batch.row_start is None:
        raise ValueError("attention_prefill needs a batch with row_start")
    n = q.shape[0]
    if n:
        if max_len is None:
            max_len = batch.max_pages * cache.page_size
        rows = n if batch.max_rows is None else min(n, batch.max_rows)
        workspace, wp, size = _workspace(cache, workspace, heads, batch.n_seqs, max_len, rows)
        _check(lib().mlq_paged_attention_prefill(cache.ref, layer, batch.bounded(n), ref, heads, qp, qs,
                                                 op, os, max_len, wp, size, _raw_stream(index)),
               "mlq_paged_attention_prefill")
    return out
