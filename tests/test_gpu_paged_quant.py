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


@pytest.mark.parametrize("kind", ["q4", "q8"])
def test_elements_next_to_a_border(paged, kind):
    """x = m + (c + 1/2) d is rounded up, the float below it down, also where the border is 0 and x - m rounds to it."""
    levels, middle, _ = kvq.KINDS[kind]
    x = np.zeros((40, 1, 64), np.float32)
    r = np.random.default_rng(2)
    for i in range(40):
        d = np.float32(2.0 ** r.integers(-12, 6))
        m = np.float32(-(r.integers(-6, 6) + 0.5)) * d if i % 2 else np.float32(r.integers(-40, 40)) * d
        for b in range(2):
            border = m + (r.integers(0, levels, 32).astype(np.float32) - middle + np.float32(0.5)) * d
            near = np.where(r.random(32) < 0.5, border, np.nextafter(border, np.float32(-np.inf), dtype=np.float32))
            near = np.where((r.random(32) < 0.3) & (border == 0), np.float32(-1e-30), near)
            if i % 2:
                near[5:8] = -1e-30, -2.0 ** -149, 0.0
            near[:2] = m - middle * d, m + (levels - middle) * d  # (the block's ends: they give d and m back)
            x[i, 0, 32 * b:32 * b + 32] = near
    rows = kvq.quantise(x, kind)
    assert len(np.unique(rows[..., :16 * 2 * kvq.KINDS[kind][2]])) > 10
    slots = np.arange(40, dtype=np.int64)
    cache = paged.PagedCache.empty(1, 3, 16, 1, 64, kind)
    paged.write(cache, 0, dev(x), dev(x), dev(slots))
    for pool in (cache.keys, cache.values):
        assert np.array_equal(pool[0].cpu().numpy()[slots // 16, :, slots % 16], rows)


@pytest.mark.parametrize("kind", ["q4", "q8"])
def test_scales_are_rounded_twice(paged, kind):
    """m = lo + z d is rounded to fp32 and then to fp16: 1 + 2^-11 + 2^-30 becomes 1 + 2^-11, a tie, and that 1."""
    levels, middle, _ = kvq.KINDS[kind]
    lo = np.float32(2.0 ** -11 + 2.0 ** -30)
    x = np.full((16, 1, 64), lo, np.float32)
    x[:, 0, 1::2] = lo + np.float32(levels / middle)
    rows = kvq.quantise(x, kind)
    scales = rows[0, 0, 16 * 2 * kvq.KINDS[kind][2]:].view(np.float16)
    assert list(scales[:2]) == [1.0 / middle, 1.0]
    slots = np.arange(16, dtype=np.int64)
    cache = paged.PagedCache.empty(1, 1, 16, 1, 64, kind)
    paged.write(cache, 0, dev(x), dev(x), dev(slots))
    assert np.array_equal(cache.keys[0, 0, 0].cpu().numpy(), rows[:, 0])
    # (and rotated by nothing, a position of 0)
    cache.keys.zero_()
    rotary = paged.Rotary(64, dev(paged.rope_frequencies(1e4, 64)[0]))
    paged.qk_norm_rope(rotary, dev(x), dev(x), dev(x), dev(np.zeros(16, np.int32)), cache=cache, slots=dev(slots))
    assert np.array_equal(cache.keys[0, 0, 0].cpu().numpy(), rows[:, 0])
    assert np.array_equal(cache.values[0, 0, 0].cpu().numpy(), rows[:, 0])


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


# ---- attention -----------------------------------------------------------------------
class Problem:
    """A cache with sequences of `lengths`; what nobody owns holds any bytes, NaN
    and infinite scales among them."""

    def __init__(self, paged, kind, lengths, heads, kv, hd, page, seed=0, layers=1, q_scale=1.5, new=None, extra_pages=0, size=1.0):
        import torch
        r = np.random.default_rng(seed + 17 * len(lengths) + hd)
        lengths = np.asarray(lengths)
        self.new = np.ones(len(lengths), np.int64) if new is None else np.asarray(new)
        pages = -(-lengths // page)
        n_pages = int(pages.sum()) + 2
        order = r.permutation(n_pages)
        most = max(1, int(pages.max())) + extra_pages
        self.table = np.full((len(lengths), most), -1, np.int32)
        used = np.zeros((n_pages, page), bool)
        at = 0
        for i, p in enumerate(pages):
            self.table[i, :p] = order[at:at + p]
            at += p
            for j in range(p):
                used[self.table[i, j], :max(0, min(page, lengths[i] - j * page))] = True
        width = kvq.row_bytes(hd, kind)
        self.k, self.v = (r.integers(0, 256, (layers, n_pages, kv, page, width)).astype(np.uint8) for _ in range(2))
        for pool in (self.k, self.v):
            pool[..., -4:][r.random(pool.shape[:-1]) < 0.3] = 255
            for layer in range(layers):
                x = (r.standard_normal((int(used.sum()), kv, hd)) * np.exp(0.5 * r.standard_normal((kv, hd))) * size).astype(np.float32)
                x[r.random(x.shape[:2]) < 0.02] *= 20  # (a token that stands out, as the first ones of a text do)
                a, b = np.nonzero(used)
                pool[layer][a, :, b] = kvq.quantise(x, kind)
        self.cache = paged.PagedCache(dev(self.k), dev(self.v), quant=kind, head_dim=hd)
        self.start = np.concatenate([[0], np.cumsum(self.new)]).astype(np.int32)
        rows = int(self.start[-1])
        self.q = (q_scale * r.standard_normal((rows, heads, hd))).astype(np.float32)
        wide = np.zeros((rows, (heads + 2 * kv) * hd), np.float32)
        wide[:, :heads * hd] = self.q.reshape(rows, -1)
        self.qd = dev(wide)[:, :heads * hd].view(rows, heads, hd) if rows else torch.zeros((0, heads, hd), device="cuda")
        self.lengths, self.kind, self.heads, self.kv, self.hd, self.page, self.rows = lengths, kind, heads, kv, hd, page, rows
        self.batch = paged.PagedBatch(dev(self.table), dev(lengths.astype(np.int32)), dev(self.start))

    def want(self, layer=0, rows=None, **rule):
        """{row: (out, bound)}"""
        got = {}
        scale = rule.pop("scale", None) or self.hd ** -0.5
        for i, n in enumerate(self.lengths):
            if rows is not None and not rows & set(range(self.start[i], self.start[i + 1])):
                continue
            ids = self.table[i, :-(-int(n) // self.page)]
            k, v = (np.concatenate([p[layer, j] for j in ids], axis=1)[:, :n] if n else p[layer, 0, :, :0] for p in (self.k, self.v))
            for r in range(self.start[i], self.start[i + 1]):
                if rows is None or r in rows:
                    pos = int(n) - (self.start[i + 1] - r)
                    got[r] = kvq.attention(self.q[r], k, v, pos, scale, kind=self.kind, **rule)
        return got

    def compare(self, out, want, what=""):
        out = out.double().cpu().numpy()
        for r, (y, bound) in want.items():
            # (a block past fp16's range reads as NaN, and so do the rows that see it)
            bad = ~((np.abs(out[r] - y) <= bound) | (np.isnan(out[r]) & np.isnan(y)))
            assert not bad.any(), (what, r, int(bad.sum()), float(np.nanmax(np.abs(out[r] - y) / bound)), out[r][bad][:3], y[bad][:3])

    def some(self, n):
        """About n rows, first and last ones of the sequences among them."""
        edges = {int(s) + d for s in self.start for d in (-1, 0) if 0 <= s + d < self.rows}
        return set(range(0, self.rows, max(1, self.rows // n))) | (edges if len(edges) < 40 else set())


def rule_of(paged, heads, softcap=0.0, window=0, slopes=False, scale=None):
    s = np.array([2.0 ** (-8.0 * (i + 1) / heads) for i in range(heads)], np.float32) if slopes else None
    return (paged.AttentionRule(scale, softcap, window, dev(s) if slopes else None),
            dict(softcap=softcap, window=window, slopes=s, scale=scale))


KINDS = ["q4", "q8"]
SHAPES = [(28, 4, 128), (8, 8, 64), (16, 1, 256), (12, 4, 80), (3, 1, 8), (40, 2, 64), (33, 1, 128), (4, 4, 200), (5, 5, 96), (6, 2, 32)]
EDGES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65, 100, 127, 128, 129, 255, 257, 600]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("heads,kv,hd", SHAPES)
def test_decode_edges(paged, heads, kv, hd, page, kind):
    p = Problem(paged, kind, EDGES, heads, kv, hd, page)
    out = paged.attention_decode(p.cache, 0, p.batch, p.qd)
    p.compare(out, p.want())


RULES = [dict(softcap=20.0), dict(window=1), dict(window=37), dict(slopes=True), dict(scale=0.3), dict(softcap=30.0, window=100, slopes=True),
         dict(scale=-0.2, softcap=2.0)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rule", RULES)
@pytest.mark.parametrize("heads,kv,hd", [(28, 4, 128), (16, 16, 64), (4, 1, 256), (40, 2, 72)])
def test_decode_rules(paged, heads, kv, hd, rule, kind):
    p = Problem(paged, kind, EDGES, heads, kv, hd, 32, seed=3)
    own, plain = rule_of(paged, heads, **rule)
    out = paged.attention_decode(p.cache, 0, p.batch, p.qd, rule=own)
    p.compare(out, p.want(**plain), rule)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv,hd,page,lengths", [
    (28, 4, 128, 16, [9001]), (28, 4, 128, 128, [5000, 1, 4097, 300]), (8, 8, 64, 64, [20000, 0, 7]), (16, 1, 256, 16, [4500, 6001]),
    (12, 4, 80, 32, [7777, 12]), (32, 8, 128, 4096, [10000, 8192, 8193])])
def test_decode_long(paged, heads, kv, hd, page, lengths, kind):
    import torch
    p = Problem(paged, kind, lengths, heads, kv, hd, page, seed=5)
    for rule in (dict(), dict(window=2500, softcap=50.0)):
        own, plain = rule_of(paged, heads, **rule)
        out = paged.attention_decode(p.cache, 0, p.batch, p.qd, rule=own)
        again = paged.attention_decode(p.cache, 0, p.batch, p.qd, rule=own)
        p.compare(out, p.want(**plain), rule)
        assert torch.equal(out, again)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("seqs", [1, 3, 40, 300])
def test_decode_result_does_not_depend_on_the_bound(paged, seqs, kind):
    """A tight max_len and a loose one split the keys differently: the same results within the bounds; rows past are left."""
    import torch
    r = np.random.default_rng(seqs)
    p = Problem(paged, kind, r.integers(1, 900, seqs), 28, 4, 128, 16, seed=7, extra_pages=2800)
    want = p.want(rows=set(range(0, p.rows, 7)))
    for max_len in (900, 4000, None):
        out = torch.full((p.rows + 2, 28, 128), 9.0, device="cuda")
        q = torch.cat([p.qd, p.qd[:1], p.qd[:1]])
        paged.attention_decode(p.cache, 0, p.batch, q, out=out, max_len=max_len)
        p.compare(out, want, max_len)
        assert torch.all(out[p.rows:] == 9.0)


def test_decode_of_more_sequences_than_a_launch_takes(paged):
    import torch
    r = np.random.default_rng(8)
    n = 4150
    lengths = r.integers(0, 40, n)
    lengths[[7, 4090, 4096, n - 1]] = [500, 200, 470, 129]
    p = Problem(paged, "q4", lengths, 4, 2, 64, 16, seed=19, new=(r.random(n) < 0.9).astype(int))
    want = p.want(rows=set(range(0, p.rows, 50)) | set(range(p.rows - 60, p.rows)))
    for max_len in (None, 500):
        out = paged.attention_decode(p.cache, 0, p.batch, p.qd, max_len=max_len)
        p.compare(out, want)
    p = Problem(paged, "q8", [40, 50, 60, 70, 0], 8, 4, 64, 16, new=[1, 0, 3, 1, 0])
    out = torch.full((p.rows, 8, 64), 9.0, device="cuda")
    paged.attention_decode(p.cache, 0, p.batch, p.qd, out=out)
    p.compare(out, p.want(rows={0, 3, 4}))
    assert torch.all(out[1:3] == 9.0)  # (of several new rows the last one is computed)


PREFILL = [  # lengths, new
    ([0, 1, 1, 2, 17], [0, 1, 1, 2, 17]), ([16, 33, 64, 100, 31], [16, 1, 32, 33, 31]), ([300], [300]), ([700, 5, 129], [1, 5, 64]),
    ([130] * 9, [15, 16, 17, 31, 32, 33, 0, 130, 127]), ([513, 400], [513, 200])]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("lengths,new", PREFILL)
@pytest.mark.parametrize("heads,kv,hd", SHAPES)
def test_prefill(paged, heads, kv, hd, lengths, new, kind):
    import torch
    p = Problem(paged, kind, lengths, heads, kv, hd, 16, seed=21, new=new)
    out = torch.full((p.rows + 3, heads, hd), 9.0, device="cuda")
    q = torch.cat([p.qd, p.qd[:1], p.qd[:1], p.qd[:1]])
    paged.attention_prefill(p.cache, 0, p.batch, q, out=out)
    p.compare(out, p.want(rows=p.some(40)))
    assert torch.all(out[p.rows:] == 9.0)  # rows behind the last sequence


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rule", RULES[:4] + RULES[5:])
@pytest.mark.parametrize("heads,kv,hd", [(28, 4, 128), (4, 4, 64), (16, 1, 256), (6, 2, 80)])
def test_prefill_rules(paged, heads, kv, hd, rule, kind):
    p = Problem(paged, kind, [400, 90, 1, 350], heads, kv, hd, 32, seed=23, new=[250, 90, 1, 3])
    own, plain = rule_of(paged, heads, **rule)
    out = paged.attention_prefill(p.cache, 0, p.batch, p.qd, rule=own)
    p.compare(out, p.want(rows=p.some(60), **plain), rule)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv,hd,lengths,new", [(28, 4, 128, [2100, 1500, 60], [1900, 800, 60]), (8, 8, 64, [3000], [1537]), (16, 1, 256, [1300], [700])])
def test_prefill_long(paged, heads, kv, hd, lengths, new, kind):
    import torch
    p = Problem(paged, kind, lengths, heads, kv, hd, 64, seed=25, new=new, layers=2)
    out = paged.attention_prefill(p.cache, 1, p.batch, p.qd)
    again = paged.attention_prefill(p.cache, 1, p.batch, p.qd)
    p.compare(out, p.want(layer=1, rows=p.some(20)))
    assert torch.equal(out, again)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [256, 257])
def test_prefill_of_many_sequences(paged, n, kind):
    """Tiles are given out in another way from 257 sequences on; some have no rows, one has several tiles."""
    import torch
    r = np.random.default_rng(n)
    lengths = r.integers(0, 50, n)
    lengths[n // 2] = 300
    new = np.minimum(r.choice([0, 1, 1, 2, 40], n), lengths)
    new[n // 2], new[-1], new[0] = 290, 0, 0
    p = Problem(paged, kind, lengths, 12, 4, 128, 16, seed=31, new=new)
    out = torch.full((p.rows + 3, 12, 128), 9.0, device="cuda")
    paged.attention_prefill(p.cache, 0, p.batch, torch.cat([p.qd, p.qd[:3]]), out=out)
    p.compare(out, p.want(rows=set(range(0, p.rows, 7)) | {p.rows - 1}))
    assert torch.all(torch.isfinite(out)) and torch.all(out[p.rows:] == 9.0)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv,hd,lengths,new", [
    (28, 4, 128, [5000], [3]), (8, 8, 64, [3000, 10, 900, 0], [20, 10, 1, 0]), (16, 1, 256, [1300, 2000], [5, 4]), (12, 4, 80, [4000, 130, 2000, 20], [1, 2, 40, 20])])
def test_prefill_of_few_rows_behind_long_contexts(pkg, paged, heads, kv, hd, lengths, new, kind):
    """Their keys are shared by several workgroups and joined."""
    import torch
    p = Problem(paged, kind, lengths, heads, kv, hd, 16, seed=27, new=new)
    need = paged.attention_workspace_bytes(p.cache, heads, len(lengths), p.table.shape[1] * 16, rows=p.rows)
    assert need > 0
    ws = torch.full((need,), 255, dtype=torch.uint8, device="cuda")  # (NaN wherever nothing is written)
    for rule in (dict(), dict(softcap=20.0, slopes=True), dict(window=300), dict(scale=-0.1)):
        own, plain = rule_of(paged, heads, **rule)
        out = paged.attention_prefill(p.cache, 0, p.batch, p.qd, rule=own, workspace=ws)
        again = paged.attention_prefill(p.cache, 0, p.batch, p.qd, rule=own)
        p.compare(out, p.want(rows=p.some(30), **plain), rule)
        assert torch.equal(out, again)
    with pytest.raises(pkg.MLQError):
        paged.attention_prefill(p.cache, 0, p.batch, p.qd, workspace=ws[:need - 256])


@pytest.mark.parametrize("kind", KINDS)
def test_prefill_rows_before_the_first_key(paged, kind):
    """More rows than tokens: the first ones see nothing and are zeros."""
    import torch
    p = Problem(paged, kind, [150, 40, 90], 8, 2, 64, 16, seed=33, new=[150, 40, 90])
    kept = p.lengths = np.array([30, 0, 89])
    p.batch.lengths.copy_(dev(kept.astype(np.int32)))
    out = paged.attention_prefill(p.cache, 0, p.batch, p.qd, rule=paged.AttentionRule(window=64))
    lost = {int(p.start[i]) + j for i, n in enumerate(kept) for j in range(int(p.new[i] - n))}
    assert torch.all(out[sorted(lost)] == 0.0)
    p.compare(out, p.want(rows=set(range(p.rows)) - lost, window=64))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("prefill", [False, True])
def test_bad_device_numbers_give_nan_rows_alone(paged, prefill, kind):
    """A page outside the cache or a length past the table: that sequence's rows are NaN, the others' are right."""
    p = Problem(paged, kind, [100, 333, 70, 200, 500, 90], 8, 2, 128, 16, seed=9, new=None if not prefill else [3, 2, 5, 1, 4, 90])
    want = p.want(rows=p.some(30))
    call = paged.attention_prefill if prefill else paged.attention_decode
    table, n = p.batch.block_table, p.batch.lengths
    table[1, 5], table[3, 0], table[4, 31] = p.cache.n_pages, -1, 2 ** 31 - 1
    n[2] = p.batch.max_pages * 16 + 1
    out = call(p.cache, 0, p.batch, p.qd)
    bad = {r for i in (1, 2, 3, 4) for r in range(p.start[i], p.start[i + 1])}
    o = out.cpu().numpy()
    assert all(np.all(np.isnan(o[r])) for r in bad)
    p.compare(out, {r: w for r, w in want.items() if r not in bad})
    for length, value in ((-5, 0.0), (-2 ** 31, 0.0), (2 ** 31 - 1, np.nan)):  # negative: nothing to see
        n.fill_(length)
        out = call(p.cache, 0, p.batch, p.qd)
        assert np.array_equal(out.cpu().numpy(), np.full(out.shape, value), equal_nan=True), length


def set_scale(pool, p, kind, i, t, kvh, block, which, value):
    """Overwrites d (0) or m (1) of a block of token t of sequence i."""
    nb = kvq.blocks(p.hd)
    at = 16 * nb * kvq.KINDS[kind][2] + 4 * block + 2 * which
    pool[0, int(p.table[i, t // p.page]), kvh, t % p.page, at:at + 2] = np.array([value], np.float16).view(np.uint8)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("prefill", [False, True])
@pytest.mark.parametrize("value", [np.nan, np.inf])
def test_blocks_that_are_not_finite(paged, prefill, value, kind):
    """A block that reads as NaN or infinities makes the heads that see it non-finite (of a value: in its dims), and no
    other's; behind the window or the row's position it is not seen."""
    p = Problem(paged, kind, [200, 200, 200], 8, 4, 128, 16, seed=11, new=None if not prefill else [150, 150, 150])
    own, plain = rule_of(paged, 8, window=100)
    want = p.want(rows=p.some(90), **plain)
    keys, vals = p.k.copy(), p.v.copy()
    set_scale(keys, p, kind, 0, 120, 1, 2, 0, value)
    set_scale(vals, p, kind, 1, 120, 2, 1, 1, value)
    set_scale(vals, p, kind, 2, 20, 0, 3, 0, value)
    p.cache.keys.copy_(dev(keys))
    p.cache.values.copy_(dev(vals))
    out = (paged.attention_prefill if prefill else paged.attention_decode)(p.cache, 0, p.batch, p.qd, rule=own).cpu().numpy()
    for r, (y, bound) in want.items():
        i = int(np.searchsorted(p.start, r, side="right")) - 1
        pos = 200 - (p.start[i + 1] - r)
        for h in range(8):
            sees = lambda t: t <= pos < t + 100  # noqa: E731
            free = np.ones(128, bool)
            if i == 0 and h // 2 == 1 and sees(120):
                # (a NaN score takes all; an infinite one has the sign of a sum of q, and may weigh 0)
                assert np.all(np.isnan(out[r, h])) or value == np.inf
                continue
            if i == 1 and h // 2 == 2 and sees(120):
                free[32:64] = False
            if i == 2 and h // 2 == 0 and sees(20):
                free[96:] = False
            # (an infinite d times a code of 0 is NaN, others infinite: none is finite)
            assert not np.isfinite(out[r, h, ~free]).any(), (r, h)
            assert np.all(np.abs(out[r, h, free] - y[h, free]) <= bound[h, free]), (r, h)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size", [1e-6, 1e-4, 1e-2, 100.0, 2000.0])
def test_values_of_other_sizes(paged, size, kind):
    """Cached keys and values far from 1, fp16 subnormals among their scales."""
    p = Problem(paged, kind, [1, 70, 300, 40], 8, 4, 64, 16, seed=15, new=[1, 70, 9, 0], size=size)
    own, plain = rule_of(paged, 8, scale=0.2 / max(size, 1.0))
    want = p.want(**plain)
    p.compare(paged.attention_decode(p.cache, 0, p.batch, p.qd, rule=own), {int(s) - 1: want[int(s) - 1] for s in p.start[1:]}, size)
    p.compare(paged.attention_prefill(p.cache, 0, p.batch, p.qd, rule=own), want, size)


@pytest.mark.parametrize("kind", KINDS)
def test_values_of_very_different_sizes(paged, kind):
    """Tokens and blocks whose values differ by factors of up to 10^6: each output to the bound of the largest that it holds."""
    for order in (1, -1):
        p = Problem(paged, kind, [700, 33], 8, 2, 128, 16, seed=35, new=[200, 33])
        nb = kvq.blocks(128)
        at = 16 * nb * kvq.KINDS[kind][2]
        for j, t in enumerate(range(0, 700, 5)):
            s = p.v[0, int(p.table[0, t // 16]), :, t % 16, at:].copy().view(np.float16)
            s[:, 2 * (j % nb):2 * (j % nb) + 2] *= np.float16(10.0 ** (order * (t // 140 - 2)))
            p.v[0, int(p.table[0, t // 16]), :, t % 16, at:] = s.view(np.uint8)
        p.cache.values.copy_(dev(p.v))
        want = p.want(rows=p.some(50))
        p.compare(paged.attention_prefill(p.cache, 0, p.batch, p.qd), want, order)
        p.compare(paged.attention_decode(p.cache, 0, p.batch, p.qd), {int(s) - 1: want[int(s) - 1] for s in p.start[1:]}, order)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("scale", [1e-30, 1e-6, 3e3, 1e6])
def test_large_and_tiny_queries(paged, scale, kind):
    p = Problem(paged, kind, [1, 70, 300], 8, 4, 64, 16, seed=13, q_scale=scale)
    own, plain = rule_of(paged, 8, scale=0.125 / max(scale, 1.0) * 10)
    for call in (paged.attention_decode, paged.attention_prefill):
        p.compare(call(p.cache, 0, p.batch, p.qd, rule=own), p.want(**plain), scale)


@pytest.mark.parametrize("kind", KINDS)
def test_a_query_that_is_not_finite_stays_alone(paged, kind):
    import torch
    p = Problem(paged, kind, [150, 200, 90], 8, 2, 64, 16, seed=17, new=[60, 1, 90])
    for call, rows in ((paged.attention_prefill, None), (paged.attention_decode, [59, 60, 150])):
        clean = call(p.cache, 0, p.batch, p.qd)
        q = p.qd.clone()
        hit = torch.zeros(p.rows, 8, dtype=torch.bool, device="cuda")
        for r, h, d, x in ((59, 2, 5, np.nan), (60, 4, 0, np.inf), (150, 7, 63, -np.inf)):
            q[r, h, d] = x
            hit[r, h] = True
        out = call(p.cache, 0, p.batch, q)
        assert torch.all(torch.isnan(out[hit])) and torch.equal(out[~hit], clean[~hit])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv,hd,page", [(8, 2, 64, 16), (28, 4, 128, 32), (4, 1, 256, 64)])
def test_pages_behind_the_window_are_not_asked_for(paged, heads, kv, hd, page, kind):
    import torch
    window = 50
    ends = [1, 50, 51, 65, 66, 67, 81, 82, 83, 97, 98, 99, 113, 114, 130, 200, 1003, 2000]
    for new in (None, [min(n, 1 + 7 * i % 40) for i, n in enumerate(ends)]):
        p = Problem(paged, kind, ends, heads, kv, hd, page, seed=61, new=new)
        own, plain = rule_of(paged, heads, window=window)
        call = paged.attention_decode if new is None else paged.attention_prefill
        whole = call(p.cache, 0, p.batch, p.qd, rule=own)
        p.compare(whole, p.want(rows=p.some(30), **plain))
        for junk in (-1, p.cache.n_pages, 2 ** 31 - 1):
            table = p.table.copy()
            for i, f in enumerate(p.lengths - p.new + 1 - window):
                table[i, :max(0, int(f)) // page] = junk
            p.batch.block_table.copy_(dev(table))
            assert torch.equal(call(p.cache, 0, p.batch, p.qd, rule=own), whole), junk


@pytest.mark.parametrize("kind", KINDS)
def test_offsets_past_32_bits(paged, kind):
    """Rows whose bytes lie past 2^32 of a layer: written, read back and attended to."""
    import torch
    kv, page, hd = 4, 64, 256
    n_pages = 2 ** 32 // (kv * page * kvq.row_bytes(hd, kind)) + 50
    keys, vals = (torch.zeros((1, n_pages, kv, page, kvq.row_bytes(hd, kind)), dtype=torch.uint8, device="cuda") for _ in range(2))
    cache = paged.PagedCache(keys, vals, quant=kind, head_dim=hd)
    table = np.array([[n_pages - 1, 3, n_pages - 40, n_pages - 2]], np.int32)
    rows, heads = 200, 8
    q, k, v = (torch.randn(rows, n, hd, device="cuda") for n in (heads, kv, kv))
    positions = np.arange(rows)
    slots = dev(table[0, positions // page].astype(np.int64) * page + positions % page)
    paged.write(cache, 0, k, v, slots)
    bytes_ = [kvq.quantise(x.cpu().numpy(), kind) for x in (k, v)]
    for got, b in zip(paged.read(cache, 0, slots), bytes_):
        assert np.array_equal(got.cpu().numpy(), kvq.values(b, kind, hd).astype(np.float32))
    batch = paged.PagedBatch(dev(table), dev(np.array([rows], np.int32)), dev(np.array([0, rows], np.int32)))
    out, one = paged.attention_prefill(cache, 0, batch, q).cpu().numpy(), paged.attention_decode(cache, 0, batch, q).cpu().numpy()
    kk, vv = (b.transpose(1, 0, 2) for b in bytes_)
    for r, o in ((0, out), (63, out), (64, out), (150, out), (199, out), (199, one)):
        y, bound = kvq.attention(q[r].cpu().numpy(), kk, vv, r, hd ** -0.5, kind=kind)
        assert np.all(np.abs(o[r] - y) <= bound), r


# ---- streams, graphs, the operators together --------------------------------------------
@pytest.mark.parametrize("kind", KINDS)
def test_two_captured_calls_at_once(paged, kind):
    """Attention of two batches captured apart, replayed on two streams at once while lengths change between the replays."""
    import torch
    problems = [Problem(paged, kind, [4000, 2100, 900, 30], 28, 4, 128, 16, seed=51, new=[1, 3, 2, 0]),
                Problem(paged, "q8", [3000, 5000, 77], 8, 8, 64, 32, seed=53, new=[2, 1, 1])]
    calls = []
    for p in problems:
        outs = [torch.zeros_like(p.qd).contiguous() for _ in range(2)]
        both = lambda p=p, outs=outs: (paged.attention_decode(p.cache, 0, p.batch, p.qd, out=outs[0]),  # noqa: E731
                                       paged.attention_prefill(p.cache, 0, p.batch, p.qd, out=outs[1]))
        both()
        torch.cuda.synchronize()
        g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(g):
            both()
        calls.append((both, outs, g, s))
    for step in range(5):
        want = []
        for p, (both, outs, g, s) in zip(problems, calls):
            p.batch.lengths.copy_(dev(np.maximum(p.lengths - 17 * step, 0).astype(np.int32)))
            for o in outs:
                o.fill_(9.0)
            both()
            want.append([o.clone() for o in outs])
            for o in outs:
                o.fill_(9.0)
        torch.cuda.synchronize()
        for both, outs, g, s in calls:
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for w, (both, outs, g, s) in zip(want, calls):
            assert all(torch.equal(a, b) for a, b in zip(w, outs)), step


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("graph", [False, True])
def test_serving_loop(paged, kind, graph):
    """Plan, rotate and store, attend: prompts, steps of one token, sequences that end and come back on pages of others. The
    attention is held to the bytes that the cache has, those to the rotated keys and the values."""
    import torch
    heads, kv, hd, page, seqs, most = 8, 2, 64, 16, 5, 200
    cache = paged.PagedCache.empty(1, 40, page, kv, hd, kind)
    cache.keys.fill_(255)
    cache.values.fill_(255)
    batch = paged.PagedBatch.empty(seqs, 12, most)
    free = dev(np.random.default_rng(3).permutation(40).astype(np.int32))
    n_free = torch.full((1,), 40, dtype=torch.int32, device="cuda")
    n_new = torch.zeros(seqs, dtype=torch.int32, device="cuda")
    freqs, _ = paged.rope_frequencies(1e4, hd // 2)
    rotary = paged.Rotary(hd, dev(freqs))
    qkv = torch.zeros((most, (heads + 2 * kv) * hd), device="cuda")
    k_out, out = torch.zeros((most, kv, hd), device="cuda"), torch.zeros((most, heads, hd), device="cuda")
    q_out = torch.zeros((most, heads, hd), device="cuda")

    def launch(rows, decode):
        paged.plan(batch, batch.lengths, n_new, free, n_free, page)
        q, k, v = (t.view(rows, -1, hd) for t in qkv[:rows].split([heads * hd, kv * hd, kv * hd], 1))
        paged.qk_norm_rope(rotary, q, k, v, batch.positions, q_out=q_out[:rows], k_out=k_out[:rows], cache=cache, slots=batch.slots)
        (paged.attention_decode if decode else paged.attention_prefill)(cache, 0, batch, q_out[:rows], out=out[:rows])

    steps = [[20, 33, 0, 1, 16], [1, 1, 50, 1, 1], [1, 1, 1, 1, 1], [-1, 1, 1, 0, -1], [70, 1, 1, 1, 0], [1, 1, 1, 1, 0], [1, -1, 17, 1, 40],
             [1, 0, 1, 1, 1], [1, 0, 1, 1, 1], [-1, -1, -1, -1, -1], [100, 2, 3, 60, 5], [1, 1, 1, 1, 1]]
    captured = None
    for i, new in enumerate(steps):
        rows = max(1, sum(max(0, n) for n in new))
        one = max(new) <= 1
        qkv[:rows].normal_()
        n_new.copy_(dev(np.array(new, np.int32)))
        if one and graph:
            if captured is None:
                captured = torch.cuda.CUDAGraph()
                torch.cuda.synchronize()
                with torch.cuda.graph(captured):
                    launch(seqs, True)
            captured.replay()
            torch.zeros(1000, device="cuda").sum().item()
        else:
            launch(rows, one)
        torch.cuda.synchronize()
        assert int(batch.status.item()) == 0
        slots, start, lengths = (t.cpu().numpy() for t in (batch.slots, batch.row_start, batch.lengths))
        table, keys, vals = (t.cpu().numpy() for t in (batch.block_table, cache.keys[0], cache.values[0]))
        n = int(start[-1])
        if n == 0:
            continue
        at = (slots[:n] // page, slice(None), slots[:n] % page)
        assert kvq.same_rows(keys[at], kvq.quantise(k_out[:n].cpu().numpy(), kind), hd, kind)
        v = qkv[:n, (heads + kv) * hd:].view(n, kv, hd).cpu().numpy()
        assert kvq.same_rows(vals[at], kvq.quantise(v, kind), hd, kind)
        for s in range(seqs):
            if start[s + 1] == start[s]:
                continue
            kk, vv = (np.concatenate([p[j] for j in table[s, :-(-lengths[s] // page)]], axis=1)[:, :lengths[s]] for p in (keys, vals))
            for r in range(start[s], start[s + 1]):
                y, bound = kvq.attention(q_out[r].cpu().numpy(), kk, vv, int(lengths[s]) - (start[s + 1] - r), hd ** -0.5, kind=kind)
                assert np.all(np.abs(out[r].double().cpu().numpy() - y) <= bound), (i, r)


# ---- what values a row's weights are held beside ------------------------------------------
def small_weights(paged, kind, heads, kv, hd, lengths, new, size, sink, seed):
    """Values of `size`, and in each sequence a token `sink` (from its end) that weighs e^12 times what others do: what the
    others add has to come out of weights far below the largest, which is the sink's, of a value a million times smaller."""
    p = Problem(paged, kind, lengths, heads, kv, hd, 16, seed=seed, new=new, size=size)
    r = np.random.default_rng(seed)
    p.q = (0.3 * r.standard_normal(p.q.shape) + 4 * hd ** -0.5).astype(np.float32)
    p.qd.copy_(dev(p.q))
    for i, n in enumerate(lengths):
        put(p.k, p, i, np.arange(n), (1.5 * r.standard_normal((n, kv, hd))).astype(np.float32))
        put(p.k, p, i, n - sink, np.full((kv, hd), 3.0, np.float32))
        put(p.v, p, i, n - sink, (1e-6 * size * r.standard_normal((kv, hd))).astype(np.float32))
    return p


def put(pool, p, i, t, x):
    """Heads x in the place of token t, or of several, of sequence i."""
    pool[0, p.table[i, t // p.page], :, t % p.page] = kvq.quantise(x, p.kind)


def compare_prefill(paged, p, what, **rule):
    """Both attentions against the definition. Prefill holds a weight beside its value row's bound |m| + middle d: a part's
    last bit, 2^-24, is off by half of it, of weights lifted to 2^11 at least for the largest bound among the seen rows,
    2^14 to 2^15 in the parts' own units: 2^-25 2^15 / 2^11 / 2^14 = 2^-35 of that bound a key."""
    own, plain = rule_of(paged, p.heads, **rule)
    p.cache.keys.copy_(dev(p.k))
    p.cache.values.copy_(dev(p.v))
    want = p.want(**plain)
    p.compare(paged.attention_decode(p.cache, 0, p.batch, p.qd, rule=own), {int(s) - 1: want[int(s) - 1] for s in p.start[1:]}, what)
    levels, middle, unit = kvq.KINDS[p.kind]
    nb, window = kvq.blocks(p.hd), plain["window"]
    for row, (y, bound) in want.items():
        i = int(np.searchsorted(p.start, row, side="right")) - 1
        pos = int(p.lengths[i]) - (p.start[i + 1] - row)
        t = np.arange(max(0, pos + 1 - window) if window else 0, pos + 1)
        s = np.ascontiguousarray(p.v[0, p.table[i, t // p.page], :, t % p.page][..., 16 * nb * unit:]).view(np.float16).astype(np.float64)
        most = (np.abs(s[..., 1::2]) + middle * s[..., ::2]).max((0, 2))
        bound += len(t) * 2.0 ** -35 * np.repeat(most, p.heads // p.kv)[:, None]
    p.compare(paged.attention_prefill(p.cache, 0, p.batch, p.qd, rule=own), want, what)


FEW_AND_SPLIT = [([170, 90], [150, 90]), ([1500], [3])]  # (the second one's keys are shared by workgroups)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size", [1e-2, 1e-3])
@pytest.mark.parametrize("lengths,new", FEW_AND_SPLIT)
@pytest.mark.parametrize("heads,kv,hd", [(8, 2, 128), (4, 4, 64), (4, 1, 256), (6, 2, 80)])
def test_value_rows_of_zeros_take_nothing_from_others(paged, heads, kv, hd, lengths, new, size, kind):
    """A value row of zeros, first, in the middle, last or everywhere but in a few places: the weights of the others keep their
    bits."""
    for at in ([0], [lengths[0] // 2], [-1], "most", "all"):
        p = small_weights(paged, kind, heads, kv, hd, lengths, new, size, sink=70, seed=71)
        r = np.random.default_rng(5)
        for i, n in enumerate(lengths):
            t = np.flatnonzero(r.random(n) < (0.9 if at == "most" else 2.0)) if isinstance(at, str) else np.array(at) % n
            put(p.v, p, i, t, np.zeros((len(t), kv, hd), np.float32))
        compare_prefill(paged, p, at)
        if at == "all":
            assert not paged.attention_prefill(p.cache, 0, p.batch, p.qd).any()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv,hd", [(8, 2, 128), (4, 4, 64), (4, 1, 256)])
def test_a_value_row_that_is_nan_among_zeros(paged, heads, kv, hd, kind):
    """All values zero but for one row without a number: who sees it gets NaN, others zeros."""
    p = Problem(paged, kind, [150, 700], heads, kv, hd, 16, seed=73, new=[150, 5])
    for i, n in enumerate(p.lengths):
        put(p.v, p, i, np.arange(n), np.zeros((n, kv, hd), np.float32))
        put(p.v, p, i, 77, np.full((kv, hd), np.nan, np.float32))
    p.cache.values.copy_(dev(p.v))
    own, _ = rule_of(paged, heads, window=60)
    for rule, last in ((None, 10 ** 9), (own, 60)):
        out = paged.attention_prefill(p.cache, 0, p.batch, p.qd, rule=rule).cpu().numpy()
        for row in range(p.rows):
            i = int(np.searchsorted(p.start, row, side="right")) - 1
            pos = int(p.lengths[i]) - (p.start[i + 1] - row)
            assert np.isnan(out[row]).all() if 77 <= pos < 77 + last else (out[row] == 0.0).all(), (row, pos)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("big", [1e2, 1e4])
@pytest.mark.parametrize("heads,kv,hd,softcap", [(8, 2, 128, 0.0), (4, 4, 64, 0.0), (4, 1, 256, 0.0), (6, 2, 80, 0.0), (8, 2, 128, 50.0)])
def test_large_value_rows_that_are_not_seen(paged, heads, kv, hd, softcap, big, kind):
    """A later token's values in the same tile, and a token's just before the window: a row's bits do not hang on them."""
    p = small_weights(paged, kind, heads, kv, hd, [170, 90], [150, 90], 1e-2, sink=70, seed=75)
    r = np.random.default_rng(9)
    for i, n in enumerate(p.lengths):
        for t in [n - 1, n - 2] + ([95] if n > 95 else []):  # (95 is the last of its tile: 64 .. 94 do not see it)
            put(p.v, p, i, t, (big * r.standard_normal((kv, hd))).astype(np.float32))
    compare_prefill(paged, p, "later", softcap=softcap)
    # the windows of the last rows begin in the tile of a large row, behind it
    for n, window in ((170, 76), (1511, 100), (1511, 90)):
        p = small_weights(paged, kind, heads, kv, hd, [n, n - 1], [4, 1], 1e-2, sink=40, seed=77)
        for i, m in enumerate(p.lengths):
            put(p.v, p, i, np.arange(m - 3 - window, m - window), (big * r.standard_normal((3, kv, hd))).astype(np.float32))
        compare_prefill(paged, p, (n, window), window=window, softcap=softcap)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv,hd", [(8, 2, 128), (28, 4, 128), (24, 2, 128), (4, 4, 64), (16, 1, 64), (4, 1, 256), (12, 1, 256), (6, 2, 80)])
def test_steps_below_zero(paged, heads, kv, hd, kind):
    """Rows from elsewhere may have a negative d: some blocks, or all of them, in keys and values."""
    for share in (0.02, 0.5, 1.0):
        p = Problem(paged, kind, [700, 33, 1], heads, kv, hd, 16, seed=81, new=[40, 33, 1])
        r = np.random.default_rng(7)
        at = 16 * kvq.blocks(hd) * kvq.KINDS[kind][2]
        for pool in (p.k, p.v):
            s = np.ascontiguousarray(pool[..., at:]).view(np.float16)
            s[..., ::2] *= np.where(r.random(s[..., ::2].shape) < share, -1, 1).astype(np.float16)
            pool[..., at:] = s.view(np.uint8)
        p.cache.keys.copy_(dev(p.k))
        p.cache.values.copy_(dev(p.v))
        want = p.want(rows=p.some(20))
        p.compare(paged.attention_decode(p.cache, 0, p.batch, p.qd), {int(s) - 1: want[int(s) - 1] for s in p.start[1:]}, share)
        p.compare(paged.attention_prefill(p.cache, 0, p.batch, p.qd), want, share)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv,hd", [(8, 2, 128), (28, 4, 128), (24, 2, 128), (8, 2, 64), (16, 1, 64), (4, 1, 256)])
@pytest.mark.parametrize("bits", [0x7c01, 0xfd55, 0x7e00, 0xffff])
def test_any_nan_stays_in_its_block(paged, heads, kv, hd, bits, kind):
    """A d that is NaN, quiet or signalling, beside one large value row of its tile among small ones: the other blocks are as
    they were."""
    p = Problem(paged, kind, [70, 64, 33], heads, kv, hd, 16, seed=83, new=[1, 40, 33], size=1e-2)
    r = np.random.default_rng(3)
    nb = kvq.blocks(hd)
    at = 16 * nb * kvq.KINDS[kind][2]
    for large, bad in ((0, 2), (1, 3), (17, 16), (5, 7), (12, 30), (31, 28)):
        v = p.v.copy()
        for i in range(3):
            put(v, p, i, large, (1e3 * r.standard_normal((kv, hd))).astype(np.float32))
            v[0, p.table[i, bad // 16], :, bad % 16, at + 4:at + 6] = np.array([bits], np.uint16).view(np.uint8)
        p.cache.values.copy_(dev(v))
        kept, p.v = p.v, v
        with np.errstate(invalid="ignore"):
            want = p.want(rows=p.some(20))
        p.v = kept
        for call, rows in ((paged.attention_decode, {int(s) - 1 for s in p.start[1:]}), (paged.attention_prefill, set(want))):
            out = call(p.cache, 0, p.batch, p.qd).double().cpu().numpy()
            for row in rows:
                y, bound = want[row]
                fine = ~np.isnan(y)
                assert np.array_equal(np.isnan(out[row]), ~fine), (large, bad, row)
                assert (np.abs(out[row] - y)[fine] <= bound[fine]).all(), (large, bad, row)
