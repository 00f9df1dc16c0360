"""CPU: argument checks of what a paged cache of 4 or 8 bits adds to the C ABI
(every case returns before a launch), its sizes, and the definition's own
properties that the GPU tests rely on."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

import kv_quant_ref as kvq

FAKE = 1 << 20  # a non-null, aligned pointer that no check dereferences
OK, ARG, SHAPE, SMALL, UNSUPPORTED = 0, -1, -2, -4, -5
TYPE = {"q4": 4, "q8": 8}


def cache(pkg, **kw):
    f = dict(keys=FAKE, values=FAKE, type=4, n_layers=2, n_pages=9, page_size=16, n_kv_heads=4, head_dim=128)
    f.update(kw)
    return pkg.MlqPagedCache(*(f[n] for n, _ in pkg.MlqPagedCache._fields_))


def test_the_definition_at_a_border():
    """A block of -8.5 .. 6.5 has d = 1 and m = -0.5: 0 is halfway from code 8 to 9, what is below it has code 8."""
    x = np.full((1, 32), 1.0, np.float32)
    x[0, :6] = -8.5, 6.5, 0.0, -1e-30, -2.0 ** -149, -1e-3
    row = kvq.quantise(x, "q4")[0]
    codes = np.stack([row[:32:2] & 15, row[:32:2] >> 4], -1).reshape(-1)
    assert list(codes[:7]) == [0, 15, 9, 8, 8, 8, 10]
    assert list(row[32:36].view(np.float16)) == [1.0, -0.5]


@pytest.mark.parametrize("kind", ["q4", "q8"])
@pytest.mark.parametrize("hd", [8, 64, 72, 128, 136, 256])
def test_cache_bytes(pkg, kind, hd):
    n = ctypes.c_size_t(7)
    c = cache(pkg, keys=None, values=None, type=TYPE[kind], head_dim=hd)
    assert pkg.lib().mlq_paged_cache_bytes(ctypes.byref(c), ctypes.byref(n)) == OK
    assert n.value == 2 * 9 * 4 * 16 * kvq.row_bytes(hd, kind)


@pytest.mark.parametrize("kw,want", [(dict(type=5), ARG), (dict(type=7), ARG), (dict(type=9), ARG), (dict(head_dim=100), UNSUPPORTED),
                                     (dict(head_dim=264), UNSUPPORTED), (dict(page_size=8), UNSUPPORTED), (dict(n_pages=0), SHAPE)])
def test_geometry(pkg, kw, want):
    n = ctypes.c_size_t()
    c = cache(pkg, **kw)
    assert pkg.lib().mlq_paged_cache_bytes(ctypes.byref(c), ctypes.byref(n)) == want


def test_write_and_read_refusals(pkg):
    def write(c=None, layer=0, rows=3, slots=FAKE, k=FAKE, ks=512, v=FAKE, vs=512, ko=None, kos=0, vo=None, vos=0):
        c = cache(pkg) if c is None else c
        return pkg.lib().mlq_paged_write(ctypes.byref(c), layer, rows, slots, k, ks, v, vs, ko, kos, vo, vos, None)

    def read(c=None, layer=0, rows=3, slots=FAKE, k=FAKE, ks=512, v=FAKE, vs=512):
        c = cache(pkg) if c is None else c
        return pkg.lib().mlq_paged_read(ctypes.byref(c), layer, rows, slots, k, ks, v, vs, None)

    for call in (write, read):
        for kw, want in [(dict(layer=2), SHAPE), (dict(layer=-1), SHAPE), (dict(rows=-1), SHAPE), (dict(slots=None), ARG), (dict(k=None), ARG),
                         (dict(v=None), ARG), (dict(k=FAKE + 4), ARG), (dict(v=FAKE + 8), ARG), (dict(ks=510), ARG), (dict(ks=508), SHAPE),
                         (dict(vs=508), SHAPE), (dict(vs=-512), SHAPE), (dict(rows=1 << 26), UNSUPPORTED), (dict(rows=2 ** 31 - 1), UNSUPPORTED),
                         (dict(rows=0), OK)]:
            assert call(**kw) == want, (call, kw)
        for kw, want in [(dict(keys=None), ARG), (dict(values=FAKE + 8), ARG), (dict(type=3), ARG), (dict(head_dim=12), UNSUPPORTED)]:
            assert call(c=cache(pkg, **kw)) == want, (call, kw)
    assert pkg.lib().mlq_paged_write(None, 0, 3, FAKE, FAKE, 512, FAKE, 512, None, 0, None, 0, None) == ARG
    assert pkg.lib().mlq_paged_read(None, 0, 3, FAKE, FAKE, 512, FAKE, 512, None) == ARG
    other = 2 * FAKE
    for kw, want in [(dict(ko=other, kos=508), SHAPE), (dict(vo=other, vos=508), SHAPE), (dict(ko=other + 4, kos=512), ARG),
                     (dict(ko=FAKE, kos=516), ARG), (dict(vo=FAKE, vos=516), ARG), (dict(vo=other, vos=514), ARG),
                     (dict(rows=0, ko=other, kos=512, vo=other, vos=512), OK)]:
        assert write(**kw) == want, kw
    # (the largest number of rows that a launch of this cache holds is checked, not launched)
    assert write(rows=0) == OK and read(rows=0) == OK


def test_front_end_refusals(pkg):
    import torch
    from mini_llama_amd import paged
    rows = torch.zeros((1, 2, 4, 16, 80), dtype=torch.uint8)
    for kw in (dict(), dict(quant="q5"), dict(quant="q4"), dict(quant="q8", head_dim=128)):  # (a CPU tensor is refused last)
        with pytest.raises(ValueError):
            paged.PagedCache(rows, rows, **kw)
    with pytest.raises(ValueError):
        paged.PagedCache(rows.float(), rows.float(), quant="q4")
    with pytest.raises(ValueError):
        paged.PagedCache.empty(1, 2, 16, 4, 128, "q6", device="cpu")
    with pytest.raises(ValueError):
        paged.PagedCache.empty(1, 2, 16, 4, 264, "q4", device="cpu")
    assert [paged.quant_row_bytes(k, hd) for k in ("q4", "q8") for hd in (8, 64, 128, 256)] == [40, 40, 80, 160, 72, 72, 144, 288]


@pytest.mark.parametrize("kind", ["q4", "q8"])
@pytest.mark.parametrize("hd", [8, 40, 64, 80, 128, 200, 256])
def test_definition(kind, hd):
    """Values lie within half a step of what was quantised, and a little more
    at the ends: m is off by half an fp16 step, d by half of its own a level."""
    r = np.random.default_rng(hd)
    x = (r.standard_normal((40, 3, hd)) * np.exp(r.uniform(-3, 3, (40, 3, 1)))).astype(np.float32)
    levels, middle, _ = kvq.KINDS[kind]
    rows = kvq.quantise(x, kind)
    assert rows.shape == (40, 3, kvq.row_bytes(hd, kind))
    y = kvq.values(rows, kind, hd)
    for b in range(0, hd, 32):
        e, f = x[..., b:b + 32].astype(np.float64), y[..., b:b + 32]
        d = (e.max(-1) - e.min(-1)) / levels
        big = np.abs(e).max(-1) + levels * d
        bound = 0.5 * d * (1 + 2.0 ** -10) + big * 2.0 ** -11 + levels * (d * 2.0 ** -11 + 2.0 ** -25) + 1e-12
        assert (np.abs(e - f).max(-1) <= bound).all()
    # what was read is written back as it was, but for m and d: both ends have their codes, so lo, hi
    # and d come back to half an fp16 step each, 2^-11 (|m| + levels d) in all, at most three times max |y|
    again = kvq.values(kvq.quantise(y.astype(np.float32), kind), kind, hd)
    assert np.abs(again - y).max() <= np.abs(y).max() * 2.0 ** -9


def test_more_rows_than_a_c_int_holds(pkg, monkeypatch):
    """2^32 + 5 rows would be taken as 5 (tensors without memory: what is not refused fails as a null address)."""
    from types import SimpleNamespace

    import torch
    from mini_llama_amd import paged

    def tensor(*shape, dtype=torch.float32):
        strides = tuple(int(np.prod(shape[i + 1:], dtype=np.int64)) for i in range(len(shape)))
        return SimpleNamespace(shape=shape, dtype=dtype, device="cuda:0", get_device=lambda: 0, dim=lambda: len(shape), stride=lambda: strides,
                               is_contiguous=lambda: True, data_ptr=lambda: None)
    c = SimpleNamespace(index=0, device="cuda:0", head_dim=128, n_kv_heads=4, ref=ctypes.byref(cache(pkg)))
    r = SimpleNamespace(index=0, head_dim=128, ref=ctypes.byref(pkg.MlqRotary(128, 0, 0, 1.0, 1e-6, None, None, None)))
    monkeypatch.setattr(paged, "_current_device", lambda: 0)
    monkeypatch.setattr(paged, "_raw_stream", lambda index: None)
    for n, error in ((5, pkg.MLQError), ((1 << 32) + 5, ValueError), (1 << 31, ValueError)):
        x, slots, positions = tensor(n, 4, 128), tensor(n, dtype=torch.int64), tensor(n, dtype=torch.int32)
        with pytest.raises(error):
            paged.write(c, 0, x, x, slots)
        with pytest.raises(error):
            paged.read(c, 0, slots, x, x)
        with pytest.raises(error):
            paged.qk_norm_rope(r, x, x, x, positions, q_out=x, k_out=x)
    b = SimpleNamespace(max_rows=None, struct=pkg.MlqPagedBatch(1, 1, 0, None, None, None, None, None, None), _bounded={})
    assert paged.PagedBatch.bounded(b, 5)._obj.max_rows == 5
    for n in ((1 << 32) + 5, 1 << 31):
        with pytest.raises(ValueError):
            paged.PagedBatch.bounded(b, n)
