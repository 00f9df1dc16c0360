"""GPU: the paged cache of 4 and 8 bits against its definition
(tests/kv_quant_ref.py) and attention over it against its own in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

import kv_quant_ref as kvq
import paged_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def paged(pkg):
    from mini_llama_amd import paged
    return paged


def dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).to("cuda")


# ---- rows written and read ---------------------------------------------------------
ROWS = [  # rows, kv heads, head dim, page
    (1, 1, 128, 16), (33, 4, 128, 16), (7, 8, 64, 32), (21, 2, 8, 16), (5, 3, 24, 64), (19, 2, 40, 16), (30, 4, 80, 16), (12, 1, 200, 128),
    (40, 1, 256, 16), (18, 3, 32, 16), (18, 2, 72, 16), (300, 16, 64, 16), (1000, 5, 128, 64)]


def rows_problem(paged, kind, rows, kv, hd, page, seed):
    """Strided k and v, slots in random order with some outside, a cache of
    0xA5 bytes of two layers."""
    import torch
    r = np.random.default_rng(seed)
    n_pages = (rows + page - 1) // page + 2
    k, v = kvq.heads(r, rows, kv, hd), kvq.heads(r, rows, kv, hd)
    slots = r.permutation(n_pages * page)[:rows].astype(np.int64)
    slots[r.random(rows) < 0.1] = -1
    if rows > 5:
        slots[3], slots[4] = n_pages * page, 1 << 40
    fused = torch.zeros(rows, 2 * kv * hd + 4, device="cuda")
    fused[:, :kv * hd], fused[:, kv * hd:2 * kv * hd] = dev(k).view(rows, -1), dev(v).view(rows, -1)
    kd, vd = fused[:, :kv * hd].view(rows, kv, hd), fused[:, kv * hd:2 * kv * hd].view(rows, kv, hd)
    cache = paged.PagedCache.empty(2, n_pages, page, kv, hd, kind)
    cache.keys.fill_(0xA5 if isinstance(kind, str) else 3.0)
    cache.values.fill_(0xA5 if isinstance(kind, str) else 3.0)
    return k, v, kd, vd, slots, cache



@pytest.mark.parametrize("kind", ["q4", "q8"])
@pytest.mark.parametrize("rows,kv,hd,page", ROWS)
def test_write_and_read(paged, kind, rows, kv, hd, page):
    import torch
    k, v, kd, vd, slots, cache = rows_problem(paged, kind, rows, kv, hd, page, rows + hd)
    live = (slots >= 0) & (slots < cache.n_pages * page)
    ko = torch.full((rows, kv, hd), 7.0, device="cuda")
    vo = torch.full((rows, kv * hd + 8), 7.0, device="cuda")[:, :kv * hd].view(rows, kv, hd)
    paged.write(cache, 1, kd, vd, dev(slots), k_out=ko, v_out=vo)
    got_k, got_v = paged.read(cache, 1, dev(slots))
    for x, pool, out, got in ((k, cache.keys, ko, got_k), (v, cache.values, vo, got_v)):
        want = np.full(tuple(cache.keys.shape[1:]), 0xA5, np.uint8)
        q = kvq.quantise(x, kind)
        want[slots[live] // page, :, slots[live] % page] = q[live]
        pool = pool.cpu().numpy()
        assert (pool[0] == 0xA5).all()
        assert kvq.same_rows(pool[1], want, hd, kind)
        y = np.where(live[:, None, None], kvq.values(q, kind, hd), 7.0).astype(np.float32)
        assert np.array_equal(out.cpu().numpy(), y, equal_nan=True)
        y = np.where(live[:, None, None], y, 0.0)
        assert np.array_equal(got.cpu().numpy(), y, equal_nan=True)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("rows,kv,hd,page", ROWS[:9])
def test_write_and_read_of_other_types(paged, dtype, rows, kv, hd, page):
    import torch
    t = getattr(torch, dtype)
    k, v, kd, vd, slots, cache = rows_problem(paged, t, rows, kv, hd, page, rows + hd)
    live = (slots >= 0) & (slots < cache.n_pages * page)
    ko = torch.full((rows, kv, hd), 7.0, device="cuda")
    paged.write(cache, 1, kd, vd, dev(slots), k_out=ko)
    got = paged.read(cache, 1, dev(slots))
    for x, pool, y in ((k, cache.keys, got[0]), (v, cache.values, got[1])):
        want = torch.full(tuple(cache.keys.shape[1:]), 3.0, dtype=t)
        rounded = torch.from_numpy(x).to(t)
        want[slots[live] // page, :, slots[live] % page] = rounded[live]
        assert (pool[0].cpu() == 3.0).all()
        assert np.array_equal(pool[1].cpu().float().numpy(), want.float().numpy(), equal_nan=True)
        assert np.array_equal(y.cpu().numpy(), np.where(live[:, None, None], rounded.float().numpy(), 0.0), equal_nan=True)
    want = np.where(live[:, None, None], torch.from_numpy(k).to(t).float().numpy(), 7.0)
    assert np.array_equal(ko.cpu().numpy(), want, equal_nan=True)


@pytest.mark.parametrize("kind", ["q4", "q8", "f16"])
def test_write_in_place_and_read_of_one_slot_twice(paged, kind):
    import torch
    k, v, kd, vd, slots, cache = rows_problem(paged, torch.float16 if kind == "f16" else kind, 40, 2, 128, 16, 5)
    at = dev(slots)
    paged.write(cache, 0, kd.clone(), vd.clone(), at, k_out=(a := torch.zeros_like(kd)), v_out=(b := torch.zeros_like(vd)))
    live = ((at >= 0) & (at < cache.n_pages * 16))[:, None, None]
    a, b = torch.where(live, a, kd), torch.where(live, b, vd)
    paged.write(cache, 0, kd, vd, at, k_out=kd, v_out=vd)
    assert torch.equal(a.nan_to_num(5.5), kd.nan_to_num(5.5)) and torch.equal(b.nan_to_num(5.5), vd.nan_to_num(5.5))
    twice = torch.cat([at[20:], at[20:]])
    x, y = paged.read(cache, 0, twice)
    assert torch.equal(x[:20].nan_to_num(5.5), x[20:].nan_to_num(5.5)) and torch.equal(y[:20].nan_to_num(5.5), y[20:].nan_to_num(5.5))
    paged.write(cache, 0, kd[:0], vd[:0], at[:0])
    assert paged.read(cache, 0, at[:0])[0].shape == (0, 2, 128)


@pytest.mark.parametrize("kind", ["q4", "q8"])
def test_rows_on_another_stream_and_in_a_graph(paged, kind):
    import torch
    rows, kv, hd, page = 65, 4, 128, 16
    cache = paged.PagedCache.empty(1, 8, page, kv, hd, kind)
    slots = torch.randperm(8 * page, device="cuda")[:rows].contiguous()
    k, v, ko, vo = (torch.zeros(rows, kv, hd, device="cuda") for _ in range(4))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        k.normal_()
        v.normal_()
    paged.write(cache, 0, k, v, slots, stream=side)
    got = paged.read(cache, 0, slots, stream=side)
    side.synchronize()
    assert kvq.same_rows(cache.keys[0].cpu().numpy()[slots.cpu() // page, :, slots.cpu() % page], kvq.quantise(k.cpu().numpy(), kind), hd, kind)
    assert np.array_equal(got[1].cpu().numpy(), kvq.values(kvq.quantise(v.cpu().numpy(), kind), kind, hd).astype(np.float32))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        paged.write(cache, 0, k, v, slots)
        paged.read(cache, 0, slots, k_out=ko, v_out=vo)
    for _ in range(3):
        k.normal_()
        v.normal_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for x, out in ((k, ko), (v, vo)):
            assert np.array_equal(out.cpu().numpy(), kvq.values(kvq.quantise(x.cpu().numpy(), kind), kind, hd).astype(np.float32))


# ---- the write of rotated rows -------------------------------------------------------
@pytest.mark.parametrize("kind", ["q4", "q8"])
@pytest.mark.parametrize("heads,kv,hd,rot,neox,rows,page,norm", [
    (28, 4, 128, 128, True, 9, 16, False), (8, 8, 64, 32, False, 33, 32, True), (12, 4, 80, 20, True, 7, 16, True), (3, 1, 8, 8, True, 5, 16, False),
    (5, 5, 24, 6, False, 3, 64, True), (16, 1, 256, 64, True, 40, 16, True), (2, 2, 40, 0, True, 4, 16, False), (40, 8, 200, 100, True, 11, 16, True),
    (64, 8, 128, 64, True, 700, 64, True)])
def test_qk_norm_rope_stores_what_write_does(paged, kind, heads, kv, hd, rot, neox, rows, page, norm):
    """The cache holds k_out and v quantised; q_out and k_out are within the
    bounds of the definition (which of two products of a rotation is rounded
    before their sum is the compiler's choice, and not the same in a call
    without a cache: the bounds count both)."""
    import torch
    r = np.random.default_rng(rows)
    k, v, kd, vd, slots, cache = rows_problem(paged, kind, rows, kv, hd, page, rows + hd)
    live = (slots >= 0) & (slots < cache.n_pages * page)
    q = torch.randn(rows, heads, hd, device="cuda")
    positions = dev(r.integers(0, 5000, rows).astype(np.int32))
    positions[rows // 2] = -1
    live[rows // 2] = False
    weights = [torch.rand(hd, device="cuda") + 0.5 if norm else None for _ in range(2)]
    freqs = torch.rand(rot // 2, dtype=torch.float64, device="cuda") if rot else None
    rotary = paged.Rotary(hd, freqs, paged.ROPE_NEOX if neox else paged.ROPE_NORMAL, q_norm=weights[0], k_norm=weights[1])
    k1 = torch.zeros(rows, kv, hd, device="cuda")
    q1, _ = paged.qk_norm_rope(rotary, q, kd, vd, positions, k_out=k1, cache=cache, layer=1, slots=dev(slots))
    keep = (positions >= 0).cpu().numpy()
    f = freqs.cpu().numpy() if rot else np.zeros(0)
    for x, y, w in ((q.cpu().numpy(), q1, weights[0]), (k, k1, weights[1])):
        fine = keep[:, None] & np.isfinite(x).all(-1) & (np.abs(x).max(-1) < 1e15)  # (others: infinities and NaN)
        with np.errstate(all="ignore"):
            want, bound = ref.turn(x, w.cpu().numpy() if norm else None, 1e-6, positions.cpu().numpy(), f, 1.0, rot, neox)
            ok = np.abs(y.cpu().numpy() - want) <= bound
        assert ok[fine].all()
    for x, pool in ((k1.cpu().numpy(), cache.keys), (v, cache.values)):
        want = np.full(tuple(cache.keys.shape[1:]), 0xA5, np.uint8)
        want[slots[live] // page, :, slots[live] % page] = kvq.quantise(x, kind)[live]
        assert (pool[0].cpu().numpy() == 0xA5).all()
        assert kvq.same_rows(pool[1].cpu().numpy(), want, hd, kind)
