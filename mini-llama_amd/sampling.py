"""The tokens of a batched step from its logits (mlq_sample, include/mlq.h):
temperature, top-k, top-p and min-p of each row, from given random numbers. The
reference samples one sequence on the host; the greedy choice of one
sequence is mlq_greedy_next.

    rule = Sampling(temperature, top_k, top_p, min_p)     # device vectors, one value a row
    tokens = sample(rule, logits, uniform)                # int32 [rows]

There is no CPU fallback, and nothing comes back to the host: a step with its
sampling can be captured in a graph and replayed while settings and random
numbers change on the device.
"""
from __future__ import annotations

import ctypes

import torch

from . import MlqSampling, _check, lib
from .paged import _F32, _I32, _Fixed, _current_device, _elsewhere, _int32, _ints, _raw_stream

__all__ = ["Sampling", "sample", "sample_workspace_bytes"]


class Sampling(_Fixed):
    """Settings of each row (mlq_sampling): temperature, top_p and min_p float32,
    top_k int32, device vectors of one length or None (temperature 1, and no
    filter). What they hold may change, the tensors are the rule's for good."""

    def __init__(self, temperature=None, top_k=None, top_p=None, min_p=None):
        given = [(n, t, d) for n, t, d in (("temperature", temperature, _F32), ("top_k", top_k, _I32),
                                           ("top_p", top_p, _F32), ("min_p", min_p, _F32))
                 if t is not None]
        for name, t, dtype in given:
            if t.dtype is not dtype or not t.is_cuda or t.dim() != 1 or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous {dtype} device vector")
        if len({(t.get_device(), t.shape[0]) for _, t, _ in given}) > 1:
            raise ValueError("the settings must have one length and device")
        self.index = given[0][1].get_device() if given else None
        self.rows = given[0][1].shape[0] if given else None
        self.temperature, self.top_k, self.top_p, self.min_p = temperature, top_k, top_p, min_p
        self.struct = MlqSampling(*(t.data_ptr() if t is not None else None
                                    for t in (temperature, top_k, top_p, min_p)))
        self.ref = ctypes.byref(self.struct)


_workspaces = {}  # bytes by (rows, vocab)


def sample_workspace_bytes(rows: int, vocab: int) -> int:
    need = _workspaces.get((rows, vocab))
    if need is None:
        nbytes = ctypes.c_size_t()
        _check(lib().mlq_sample_workspace(_int32("rows", rows), _int32("vocab", vocab),
                                          ctypes.byref(nbytes)), "mlq_sample_workspace")
        need = nbytes.value
        if len(_workspaces) >= 256:
            _workspaces.clear()
        _workspaces[(rows, vocab)] = need
    return need


def sample(rule, logits, uniform, out=None, workspace=None, stream=None):
    """Tokens int32 [rows] (out, a new tensor unless given) of logits float32
    [rows, vocab], whose rows may have any stride, by rule (a Sampling, or None:
    temperature 1 without filters) and uniform, float32 [rows] in [0, 1).
    workspace: a uint8 device tensor of sample_workspace_bytes (of these rows and
    vocab, or larger ones), or None for one of the call's own."""
    index = logits.get_device()
    if index < 0 or (rule is not None and rule.index is not None and rule.index != index):
        raise ValueError("logits must be a device tensor, on the device of the settings")
    if stream is not None or index != _current_device():
        return _elsewhere(lambda: sample(rule, logits, uniform, out, workspace), index, stream)
    if logits.dtype is not _F32 or logits.dim() != 2 or logits.shape[1] == 0 or \
       (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise ValueError("logits must be float32 [rows, vocab], the vocabulary side by side")
    n, vocab = logits.shape
    if rule is not None and rule.rows is not None and rule.rows != n:
        raise ValueError(f"the settings have {rule.rows} rows, the logits {n}")
    up = _ints("uniform", uniform, _F32, index, n)
    if out is None:
        out = torch.empty(n, dtype=_I32, device=logits.device)
    op = _ints("out", out, _I32, index, n)
    wp, size = None, 0
    if workspace is None:
        size = sample_workspace_bytes(n, vocab)
        if size:
            workspace = torch.empty(size, dtype=torch.uint8, device=logits.device)
            wp = workspace.data_ptr()
    else:
        if workspace.get_device() != index or not workspace.is_contiguous():
            raise ValueError("the workspace must be a contiguous tensor on the logits' device")
        wp, size = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    if n:
        _check(lib().mlq_sample(rule.ref if rule is not None else None, _int32("rows", n),
                                _int32("vocab", vocab), logits.data_ptr(),
                                logits.stride(0) if n > 1 else vocab, up, op, wp, size,
                                _raw_stream(index)), "mlq_sample")
    return out
