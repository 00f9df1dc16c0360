"""CPU: argument checks of the sampling entry points (every case returns
before a launch) and properties of the definition that the GPU tests use."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

import sampling_ref as ref

FAKE = 1 << 20
OK, ARG, SHAPE, SMALL, UNSUPPORTED = 0, -1, -2, -4, -5


def test_refusals(pkg):
    lib = pkg.lib()
    n = ctypes.c_size_t(7)
    for rows, vocab, want in [(0, 10, OK), (1, 1, OK), (64, 152064, OK), (-1, 10, SHAPE), (1, 0, SHAPE), (1, -3, SHAPE),
                              (1, (1 << 19) + 1, UNSUPPORTED), ((1 << 20) + 1, 5, UNSUPPORTED), (1 << 20, 1 << 19, OK)]:
        assert lib.mlq_sample_workspace(rows, vocab, ctypes.byref(n)) == want
    assert lib.mlq_sample_workspace(1, 1, None) == ARG

    def call(rows=2, vocab=100, logits=FAKE, stride=100, uniform=FAKE, tokens=FAKE, ws=FAKE, size=1 << 40):
        s = pkg.MlqSampling(None, None, None, None)
        return lib.mlq_sample(ctypes.byref(s), rows, vocab, logits, stride, uniform, tokens, ws, size, None)
    for kw, want in [(dict(logits=None), ARG), (dict(uniform=None), ARG), (dict(tokens=None), ARG), (dict(stride=-1), SHAPE),
                     (dict(stride=-100), SHAPE), (dict(vocab=0), SHAPE), (dict(rows=-1), SHAPE), (dict(ws=FAKE + 128), ARG),
                     (dict(vocab=(1 << 19) + 1, stride=1 << 20), UNSUPPORTED), (dict(rows=0), OK)]:
        assert call(**kw) == want, kw
    big = ctypes.c_size_t()
    assert lib.mlq_sample_workspace(64, 152064, ctypes.byref(big)) == OK
    if big.value:
        kw = dict(rows=64, vocab=152064, stride=152064)
        assert call(size=big.value - 1, **kw) == SMALL and call(ws=None, size=0, **kw) == SMALL


def test_front_end_refusals(pkg):
    import torch
    from mini_llama_amd import sampling
    for kw in (dict(temperature=torch.ones(3)), dict(top_k=torch.ones(3, dtype=torch.int64)), dict(top_p=torch.ones(3, 1)),
               dict(min_p=torch.ones(6)[::2])):
        with pytest.raises(ValueError):
            sampling.Sampling(**kw)
    with pytest.raises(ValueError):
        sampling.sample(None, torch.zeros(2, 5), torch.zeros(2))
    for rows, vocab in ((1 << 32, 10), (1, 1 << 32)):
        with pytest.raises(ValueError):
            sampling.sample_workspace_bytes(rows, vocab)


def test_definition():
    """By hand: weights 4, 2, 1, 1 of 8."""
    x = np.log(np.array([1, 4, 1, 2], np.float64)).astype(np.float32)
    got = lambda u, **kw: ref.token(x, u, **kw)[0]  # noqa: E731
    assert [got(u) for u in (0.0, 0.49, 0.51, 0.74, 0.76, 0.87, 0.88, 1.0)] == [1, 1, 3, 3, 0, 0, 2, 2]
    assert [got(u, top_k=2) for u in (0.0, 0.66, 0.67, 0.99)] == [1, 1, 3, 3]
    assert [got(u, top_p=0.7) for u in (0.6, 0.67, 0.99)] == [1, 3, 3] and got(0.99, top_p=0.49) == 1
    assert [got(u, min_p=0.4) for u in (0.66, 0.99)] == [1, 3] and got(0.99, min_p=2.0) == 1
    assert got(0.99, temperature=0.0) == 1 and got(0.9, temperature=1e-3) == 1 and got(0.76, temperature=1e6) == 2
    assert ref.token([np.nan, -np.inf], 0.3)[0] == -1 and ref.token([np.nan, 3, np.inf, np.inf], 0.6)[0] == 3


@pytest.mark.parametrize("vocab", [1025, 5000, 32000, 152064, 1 << 19])
def test_a_workspace_serves_smaller_calls(pkg, vocab):
    """Bytes do not fall as rows or the vocabulary grow."""
    n = ctypes.c_size_t()

    def need(rows, vocab):
        assert pkg.lib().mlq_sample_workspace(rows, vocab, ctypes.byref(n)) == OK
        return n.value
    sizes = [need(rows, vocab) for rows in range(1, 1100)]
    assert sizes == sorted(sizes) and sizes[-1] == need(1 << 20, vocab)
    for rows in (1, 3, 100, 257, 2000):
        assert need(rows, 1024) == 0 < need(rows, vocab - 1 if vocab > 1025 else vocab) <= need(rows, vocab)
