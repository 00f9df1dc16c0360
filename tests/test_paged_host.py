"""CPU: argument checks of the paged-cache C ABI (every case returns before a
launch), its sizes, the rotation frequencies, and the 64-bit definitions'
own properties that the GPU tests rely on."""
from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest

import paged_ref

FAKE = 1 << 20  # a non-null, aligned pointer that no check dereferences
OK, ARG, SHAPE, SMALL, UNSUPPORTED = 0, -1, -2, -4, -5


def cache(pkg, **kw):
    f = dict(keys=FAKE, values=FAKE, type=0, n_layers=2, n_pages=9, page_size=16, n_kv_heads=4,
             head_dim=128)
    f.update(kw)
    return pkg.MlqPagedCache(*(f[n] for n, _ in pkg.MlqPagedCache._fields_))


def batch(pkg, **kw):
    f = dict(n_seqs=3, max_pages=8, max_rows=5, block_table=FAKE, lengths=FAKE, row_start=FAKE,
             positions=FAKE, slots=FAKE, status=FAKE)
    f.update(kw)
    return pkg.MlqPagedBatch(*(f[n] for n, _ in pkg.MlqPagedBatch._fields_))


@pytest.mark.parametrize("kw,want", [
    (dict(type=3), ARG), (dict(type=-1), ARG), (dict(n_layers=0), SHAPE), (dict(n_pages=0), SHAPE),
    (dict(n_kv_heads=-1), SHAPE), (dict(head_dim=0), SHAPE), (dict(page_size=0), SHAPE),
    (dict(page_size=8), UNSUPPORTED), (dict(page_size=48), UNSUPPORTED),
    (dict(page_size=8192), UNSUPPORTED), (dict(head_dim=100), UNSUPPORTED),
    (dict(head_dim=264), UNSUPPORTED), (dict(), OK), (dict(head_dim=8, page_size=4096), OK)])
def test_cache_geometry(pkg, kw, want):
    n = ctypes.c_size_t(7)
    c = cache(pkg, keys=None, values=None, **kw)
    assert pkg.lib().mlq_paged_cache_bytes(ctypes.byref(c), ctypes.byref(n)) == want
    if want == OK:
        assert n.value == c.n_layers * c.n_pages * c.n_kv_heads * c.page_size * c.head_dim * 4
        c.type = 2
        assert pkg.lib().mlq_paged_cache_bytes(ctypes.byref(c), ctypes.byref(n)) == OK
        assert n.value == c.n_layers * c.n_pages * c.n_kv_heads * c.page_size * c.head_dim * 2
    assert pkg.lib().mlq_paged_cache_bytes(None, ctypes.byref(n)) == ARG


def test_plan_refusals(pkg):
    def call(b=None, page=16, pages=10, lengths=FAKE, n_new=FAKE, free=FAKE, n_free=FAKE, out=FAKE):
        b = batch(pkg) if b is None else b
        return pkg.lib().mlq_paged_plan(ctypes.byref(b), page, pages, lengths, n_new, free, n_free,
                                        out, None)
    for name in ("block_table", "lengths", "row_start", "positions", "slots", "status"):
        assert call(batch(pkg, **{name: None})) == ARG
    for name in ("lengths", "n_new", "free", "n_free", "out"):
        assert call(**{name: None}) == ARG
    for name in ("n_seqs", "max_pages", "max_rows"):
        assert call(batch(pkg, **{name: 0})) == SHAPE
    assert call(page=0) == SHAPE and call(pages=0) == SHAPE
    assert call(page=24) == UNSUPPORTED
    assert call(batch(pkg, max_pages=1 << 30)) == UNSUPPORTED
    assert pkg.lib().mlq_paged_plan(None, 16, 10, FAKE, FAKE, FAKE, FAKE, FAKE, None) == ARG


def test_rotary_refusals(pkg):
    def call(r=None, rows=2, positions=FAKE, heads=8, kv=4, q=FAKE, qs=1024, k=FAKE, ks=512, v=FAKE,
             vs=512, qo=FAKE, qos=1024, ko=None, kos=0, c=True, layer=0, slots=FAKE, **kw):
        f = dict(head_dim=128, rot_dim=128, rope_type=1, magnitude=1.0, eps=1e-6, freqs=FAKE,
                 q_norm=None, k_norm=None)
        f.update(kw)
        r = pkg.MlqRotary(*(f[n] for n, _ in pkg.MlqRotary._fields_))
        c = cache(pkg) if c is True else c
        return pkg.lib().mlq_qk_norm_rope(ctypes.byref(r), rows, positions, heads, kv, q, qs, k, ks,
                                          v, vs, qo, qos, ko, kos,
                                          ctypes.byref(c) if c is not None else None, layer, slots,
                                          None)
    assert call(rows=0) == OK  # nothing to do, checked all the same
    for kw, want in [(dict(positions=None), ARG), (dict(rows=-1), SHAPE), (dict(heads=0), SHAPE),
                     (dict(kv=0), SHAPE), (dict(rot_dim=130), SHAPE), (dict(rot_dim=7), SHAPE),
                     (dict(rot_dim=-2), SHAPE), (dict(head_dim=100, rot_dim=100), UNSUPPORTED),
                     (dict(head_dim=512, qs=4096, ks=2048, qos=4096), UNSUPPORTED),
                     (dict(rope_type=2), ARG), (dict(freqs=None), ARG),
                     (dict(magnitude=math.inf), ARG), (dict(q_norm=FAKE, eps=0.0), ARG),
                     (dict(k_norm=FAKE, eps=math.nan), ARG), (dict(q_norm=FAKE + 4), ARG),
                     (dict(q=None), ARG), (dict(k=None), ARG), (dict(v=None), ARG),
                     (dict(qo=None), ARG), (dict(q=FAKE + 4), ARG), (dict(qs=1022), ARG),
                     (dict(qs=1020), SHAPE), (dict(ks=508), SHAPE), (dict(vs=508), SHAPE),
                     (dict(qos=1028), ARG), (dict(ko=FAKE + 8, kos=512), ARG),
                     (dict(k=FAKE + 16, ko=FAKE + 16, kos=516), ARG), (dict(slots=None), ARG),
                     (dict(layer=2), SHAPE), (dict(layer=-1), SHAPE),
                     (dict(c=cache(pkg, n_kv_heads=2)), SHAPE),
                     (dict(c=cache(pkg, head_dim=64)), SHAPE),
                     (dict(c=cache(pkg, keys=None)), ARG), (dict(c=cache(pkg, keys=FAKE + 2)), ARG),
                     (dict(c=None), ARG), (dict(rows=1 << 24), UNSUPPORTED),
                     (dict(heads=2049, qs=2049 * 128, qos=2049 * 128), UNSUPPORTED),
                     (dict(kv=2049, ks=2049 * 128, vs=2049 * 128), UNSUPPORTED)]:
        assert call(**kw) == want, kw
    assert call(rows=0, c=None, ko=FAKE + 4096, kos=512, v=None, slots=None) == OK
    assert call(rows=0, rot_dim=0, freqs=None) == OK


@pytest.mark.parametrize("prefill", [False, True])
def test_attention_refusals(pkg, prefill):
    def call(c=None, layer=0, b=None, rule=(), heads=28, q=FAKE, qs=3584, out=FAKE, os=3584,
             max_len=128, ws=FAKE, ws_bytes=1 << 40):
        c = cache(pkg) if c is None else c
        b = batch(pkg) if b is None else b
        r = pkg.MlqAttentionRule(*rule) if rule else None
        args = [ctypes.byref(c), layer, ctypes.byref(b), ctypes.byref(r) if r else None, heads, q, qs,
                out, os]
        if prefill:
            return pkg.lib().mlq_paged_attention_prefill(*args, max_len, ws, ws_bytes, None)
        return pkg.lib().mlq_paged_attention_decode(*args, max_len, ws, ws_bytes, None)
    for kw, want in [(dict(c=cache(pkg, keys=None)), ARG), (dict(c=cache(pkg, values=FAKE + 8)), ARG),
                     (dict(c=cache(pkg, head_dim=12)), UNSUPPORTED), (dict(layer=2), SHAPE),
                     (dict(layer=-1), SHAPE), (dict(b=batch(pkg, block_table=None)), ARG),
                     (dict(b=batch(pkg, lengths=None)), ARG), (dict(b=batch(pkg, n_seqs=0)), SHAPE),
                     (dict(b=batch(pkg, max_pages=0)), SHAPE), (dict(b=batch(pkg, max_rows=0)), SHAPE),
                     (dict(b=batch(pkg, max_pages=1 << 28)), UNSUPPORTED), (dict(heads=0), SHAPE),
                     (dict(heads=30), SHAPE), (dict(q=None), ARG), (dict(out=None), ARG),
                     (dict(q=FAKE + 4), ARG), (dict(out=FAKE + 8), ARG), (dict(qs=3586), ARG),
                     (dict(os=3580), SHAPE), (dict(rule=(math.nan, 0.0, 0, None)), ARG),
                     (dict(rule=(0.0, -1.0, 0, None)), ARG), (dict(rule=(0.0, math.inf, 0, None)), ARG),
                     (dict(rule=(0.0, 0.0, -1, None)), ARG)]:
        assert call(**kw) == want, kw
    assert call(heads=2052, qs=2052 * 128, os=2052 * 128) == UNSUPPORTED
    if prefill:
        assert call(b=batch(pkg, row_start=None)) == ARG
        assert call(b=batch(pkg, n_seqs=1 << 22)) == UNSUPPORTED
        assert call(b=batch(pkg, max_rows=2 ** 31 - 1)) == UNSUPPORTED
    assert call(max_len=0) == SHAPE and call(max_len=129) == SHAPE
    assert call(ws=FAKE + 16) == ARG
    # the keys of one sequence of 100000 are shared by workgroups: it needs their partials
    n = ctypes.c_size_t()
    c = cache(pkg, n_pages=10000)
    assert pkg.lib().mlq_paged_attention_workspace(ctypes.byref(c), 28, 1, 5 if prefill else 0, 100000,
                                                   ctypes.byref(n)) == OK
    assert n.value > 0
    long = dict(c=c, b=batch(pkg, n_seqs=1, max_pages=6250), max_len=100000)
    assert call(ws_bytes=n.value - 1, **long) == SMALL
    assert call(ws=None, **long) == SMALL
    assert call(**long) == ARG  # out is q


def test_attention_workspace(pkg):
    lib, n = pkg.lib(), ctypes.c_size_t()
    c = cache(pkg, keys=None, values=None)
    for heads, seqs, rows, max_len, want in [(0, 1, 0, 1, SHAPE), (30, 1, 0, 1, SHAPE), (28, 0, 0, 1, SHAPE),
                                             (28, 1, 0, 0, SHAPE), (28, 1, -1, 1, SHAPE), (28, 1, 7, 1, OK),
                                             (2052, 1, 0, 1, UNSUPPORTED), (28, 1 << 22, 1, 1, UNSUPPORTED),
                                             (28, 1, 0, 1, OK)]:
        n.value = 77
        assert lib.mlq_paged_attention_workspace(ctypes.byref(c), heads, seqs, rows, max_len,
                                                 ctypes.byref(n)) == want
        assert n.value == (0 if want == OK else 77)  # a single key is never split
    sizes = []
    for max_len in (16, 100, 1000, 10000, 100000, 1000000):
        assert lib.mlq_paged_attention_workspace(ctypes.byref(c), 28, 4, 0, max_len, ctypes.byref(n)) == OK
        sizes.append(n.value)
    assert sizes == sorted(sizes)  # one sized for the longest serves the shorter ones
    # many rows fill the chip by themselves
    assert lib.mlq_paged_attention_workspace(ctypes.byref(c), 28, 4, 20000, 100000, ctypes.byref(n)) == OK
    assert n.value == 0


@pytest.mark.parametrize("theta,rot,factor,original,fast,slow", [
    (1e4, 128, 4.0, 4096, 32.0, 1.0), (1e6, 64, 8.0, 32768, 32.0, 1.0), (5e5, 20, 2.0, 1000, 16.0, 2.0),
    (1e4, 2, 4.0, 4096, 32.0, 1.0)])
def test_frequencies(pkg, theta, rot, factor, original, fast, slow):
    from mini_llama_amd import paged
    plain = np.array([theta ** (-2 * i / rot) for i in range(rot // 2)])
    f, m = paged.rope_frequencies(theta, rot)
    np.testing.assert_allclose(f, plain, rtol=1e-14)
    assert m == 1.0
    f, m = paged.rope_frequencies(theta, rot, "linear", factor)
    np.testing.assert_allclose(f, plain / factor, rtol=1e-14)
    assert m == 1.0
    f, m = paged.rope_frequencies(theta, rot, "parts", factor, original, fast, slow)
    np.testing.assert_allclose(f, paged_ref.rope_parts(theta, rot, factor, original, fast, slow), rtol=1e-12)
    assert m == np.float32(0.1 * math.log(factor) + 1)
    assert np.all(f <= plain * (1 + 1e-14)) and np.all(f >= plain / factor * (1 - 1e-14))


def test_frequency_refusals(pkg):
    from mini_llama_amd import paged
    bad = [(dict(theta=0.0), ARG), (dict(theta=math.inf), ARG), (dict(rot_dim=3), SHAPE), (dict(rot_dim=0), SHAPE),
           (dict(scaling="linear", factor=0.5), ARG), (dict(scaling="parts", factor=2.0), ARG),
           (dict(scaling="parts", factor=2.0, original_len=10, beta_fast=1.0), ARG),
           (dict(scaling="parts", factor=2.0, original_len=10, beta_slow=0.0), ARG),
           (dict(scaling="parts", factor=math.nan, original_len=10), ARG),
           (dict(scaling="parts", factor=2.0, original_len=10, theta=1.0), ARG)]
    for kw, want in bad:
        with pytest.raises(pkg.MLQError) as e:
            paged.rope_frequencies(**{**dict(theta=1e4, rot_dim=8), **kw})
        assert e.value.status == want, kw
    with pytest.raises(ValueError):
        paged.rope_frequencies(1e4, 8, "other")
    out = (ctypes.c_double * 4)()
    assert pkg.lib().mlq_rope_frequencies(1e4, 8, 7, 1.0, 0, 1.0, 1.0, out, ctypes.byref(ctypes.c_float())) == ARG
    assert pkg.lib().mlq_rope_frequencies(1e4, 8, 0, 1.0, 0, 1.0, 1.0, out, None) == ARG


def test_python_refusals(pkg):
    """What the front end refuses before the library is called."""
    import torch
    from mini_llama_amd import paged
    z = torch.zeros(2, 3, 4, 16, 64)
    for keys, values in ((z, z), (z, z[:, :2]), (z.to(torch.float64), z.to(torch.float64))):
        with pytest.raises(ValueError):
            paged.PagedCache(keys, values)  # not on a device, or unlike
    with pytest.raises(ValueError):
        paged.Rotary(64, torch.zeros(32, dtype=torch.float64))
    with pytest.raises(ValueError):
        paged.AttentionRule(scale=0.0)
    for window in (-1, 1 << 31, (1 << 32) + 5):  # (a C int would hold another number)
        with pytest.raises(ValueError):
            paged.AttentionRule(window=window)
    with pytest.raises(ValueError):
        paged.AttentionRule(slopes=torch.zeros(4))
    with pytest.raises(ValueError):
        paged.PagedBatch(torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32))


def test_reference_plan_is_a_loop_over_sequences():
    """Two steps by hand: pages of 4, prompts of 5 and 3, then one token each, the first ended."""
    table = np.full((2, 4), -1, np.int32)
    stack = np.array([7, 3, 9, 5, 1], np.int32)
    st, length, table, stack, free, start, pos, slots = paged_ref.plan(
        np.zeros(2, np.int32), np.array([5, 3]), table, stack, 5, 4, 10, 9)
    assert st == 0 and free == 2 and list(start) == [0, 5, 8]
    assert table.tolist() == [[1, 5, -1, -1], [9, -1, -1, -1]]
    assert pos.tolist() == [0, 1, 2, 3, 4, 0, 1, 2, -1]
    assert slots.tolist() == [4, 5, 6, 7, 20, 36, 37, 38, -1]
    stack = np.concatenate([stack, np.zeros(5, np.int32)])
    st, length, table, stack, free, start, pos, slots = paged_ref.plan(
        length, np.array([-1, 2]), table, stack, free, 4, 10, 3)
    assert st == 0 and list(length) == [0, 5] and free == 3
    assert stack[:4].tolist() == [7, 3, 1, 5] and table[1].tolist() == [9, 5, -1, -1]
    assert pos.tolist() == [3, 4, -1] and slots.tolist() == [39, 20, -1]


def test_reference_attention_matches_a_softmax():
    rng = np.random.default_rng(1)
    q, k, v = rng.standard_normal((4, 8)), rng.standard_normal((2, 9, 8)), rng.standard_normal((2, 9, 8))
    out, bound = paged_ref.attention(q, k, v, 8, 0.3, softcap=5.0, window=4, slopes=[0.1, 0.2, 0.0, 0.4])
    for h in range(4):
        s = np.array([5 * math.tanh(0.3 * (q[h] @ k[h // 2, t]) / 5) + [0.1, 0.2, 0.0, 0.4][h] * (t - 8)
                      for t in range(5, 9)])
        p = np.exp(s) / np.exp(s).sum()
        np.testing.assert_allclose(out[h], p @ v[h // 2, 5:9], rtol=1e-12)
    assert np.all(bound < 1e-4) and np.all(bound > 0)
    assert np.all(paged_ref.attention(q, k, v, -1, 0.3)[0] == 0)


@pytest.mark.parametrize("kind", [0, 1, 2])
@pytest.mark.parametrize("heads,kv,hd,seqs", [(16, 16, 64, 200), (40, 8, 64, 5000), (8, 8, 8, 190), (2, 1, 64, 4096), (28, 4, 128, 3000),
                                              (16, 1, 256, 700), (16, 16, 64, 1)])
def test_a_decode_workspace_serves_every_smaller_bound(pkg, heads, kv, hd, seqs, kind):
    """Up to the longest bound, where a launch takes fewer sequences than the batch has."""
    lib, n, sizes = pkg.lib(), ctypes.c_size_t(), []
    c = cache(pkg, keys=None, values=None, type=kind, n_kv_heads=kv, head_dim=hd)
    for max_len in sorted({max(1, (1 << s) + d) for s in range(3, 31) for d in (-1, 0)} | {300, 700, 10000, 5 * 10 ** 8}):
        assert lib.mlq_paged_attention_workspace(ctypes.byref(c), heads, seqs, 0, max_len, ctypes.byref(n)) == OK
        sizes.append(n.value)
    assert sizes == sorted(sizes)


def test_handles_keep_what_they_were_made_of(pkg):
    """Their addresses are taken once: another tensor in a tensor's place is refused, not passed by."""
    import torch
    from mini_llama_amd import paged
    rule, rotary = paged.AttentionRule(window=7), paged.Rotary(64)
    for obj, names in ((rule, ("slopes", "struct", "ref")), (rotary, ("head_dim", "rot_dim", "struct"))):
        for name in names:
            was = getattr(obj, name)
            with pytest.raises(AttributeError):
                setattr(obj, name, torch.zeros(4))
            with pytest.raises(AttributeError):
                delattr(obj, name)
            assert getattr(obj, name) is was
    for cls in (paged.PagedCache, paged.PagedBatch):  # (made of device tensors only)
        obj = object.__new__(cls)
        obj.lengths = 1
        with pytest.raises(AttributeError):
            obj.lengths = 2
        assert obj.lengths == 1


def test_numbers_that_a_c_type_would_hold_as_others(pkg):
    """A float that fp32 rounds to 0 is another rule, an int past 32 bits another number."""
    from types import SimpleNamespace

    from mini_llama_amd import paged
    for kw in (dict(scale=1e-60), dict(scale=-1e-60), dict(softcap=1e-60), dict(softcap=-1e-60)):
        with pytest.raises(ValueError):
            paged.AttentionRule(**kw)
    assert paged.AttentionRule(scale=1e-30, softcap=0.0).struct.scale == np.float32(1e-30)
    wrap = 1 << 32
    for kw in (dict(rot_dim=wrap + 8), dict(rot_dim=8 - wrap), dict(original_len=wrap + 4096), dict(original_len=4096 - wrap)):
        with pytest.raises(ValueError):
            paged.rope_frequencies(**{**dict(theta=1e4, rot_dim=8, scaling="parts", factor=2.0, original_len=4096), **kw})
    for rope_type in (wrap, wrap + 1, -wrap):
        with pytest.raises(ValueError):
            paged.Rotary(64, rope_type=rope_type)
    c = SimpleNamespace(ref=ctypes.byref(cache(pkg)), _workspaces={})
    for n in (wrap + 100, 100 - wrap):
        for args in ((28, 1, n, 0), (28, n, 100, 0), (28, 1, 100, n), (n, 1, 100, 0)):
            with pytest.raises(ValueError):
                paged.attention_workspace_bytes(c, *args)
        with pytest.raises(ValueError):
            paged._workspace(c, object(), 28, 1, n, 0)


def test_a_cap_that_no_score_can_be_divided_by(pkg):
    """scale / softcap past fp32 would make a score of 0 NaN."""
    n = ctypes.c_size_t()
    c, b = cache(pkg), batch(pkg)
    for call in (pkg.lib().mlq_paged_attention_decode, pkg.lib().mlq_paged_attention_prefill):
        for scale, cap in ((0.0, 1e-42), (1e30, 1e-10), (-1e30, 1e-10)):
            rule = pkg.MlqAttentionRule(scale, cap, 0, None)
            assert call(ctypes.byref(c), 0, ctypes.byref(b), ctypes.byref(rule), 28, FAKE, 3584, FAKE + 4096, 3584, 0, FAKE, 1 << 40,
                        None) == ARG, (scale, cap)  # (max_len 0: nothing is launched if the rule passes)
