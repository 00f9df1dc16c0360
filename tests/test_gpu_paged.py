"""GPU: the paged-cache operators against their definitions in 64 bits
(tests/paged_ref.py, whose bounds count the roundings of an fp32 kernel and,
for a cache of 16 bits, half a step of its type).

Unused slots of the pages hold NaN and infinities: nothing behind a
sequence's end may reach a result. Sequences' pages lie in random order
among pages of nobody."""
from __future__ import annotations

import math

import numpy as np
import pytest

import paged_ref as ref

pytestmark = pytest.mark.gpu

KINDS = ["f32", "f16", "bf16"]


@pytest.fixture(scope="module")
def paged(pkg):
    from mini_llama_amd import paged
    return paged


def dtype(kind):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[kind]


def dev(a, t=None):
    import torch
    x = torch.from_numpy(np.ascontiguousarray(a)).to("cuda")
    return x if t is None else x.to(t)


def host(t):
    return t.detach().double().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


def check(got, want, bound, what):
    bad = ~((np.abs(got - want) <= bound) | (got == want))
    assert not bad.any(), (what, int(bad.sum()), np.argwhere(bad)[:3].tolist(),
                           float(np.nanmax(np.abs(got - want) / bound)), got[bad][:3], want[bad][:3])


# ---- the plan --------------------------------------------------------------------
def run_plan(paged, lengths, n_new, page, max_pages, max_rows, n_pages, n_free, table, stack,
             in_place=False):
    import torch
    n = len(lengths)
    b = paged.PagedBatch.empty(n, max_pages, max_rows)
    b.block_table.copy_(dev(table))
    b.positions.fill_(77)
    b.slots.fill_(77)
    b.status.fill_(77)
    free, top = dev(stack), dev(np.array([n_free], np.int32))
    ins, top_out = dev(np.asarray(lengths, np.int32)), None
    if in_place:
        b.lengths.copy_(ins)
        ins = b.lengths
    else:
        top_out = torch.full((1,), 77, dtype=torch.int32, device="cuda")
    paged.plan(b, ins, dev(np.asarray(n_new, np.int32)), free, top, page, n_free_out=top_out)
    torch.cuda.synchronize()
    return (int(b.status.item()), host(b.lengths), host(b.block_table), host(free),
            int((top if in_place else top_out).item()), host(b.row_start), host(b.positions), host(b.slots))


def plan_problem(seed, n, page, longest, what, spare=5):
    r = np.random.default_rng(seed)
    lengths = r.integers(0, longest + 1, n)
    n_new = {"decode": np.ones(n, np.int64), "mixed": r.choice([-1, 0, 1, 1, 1, 7, longest], n),
             "prompts": r.integers(0, longest + 1, n), "end": np.full(n, -1)}[what]
    held = (lengths + page - 1) // page
    after = (lengths + np.maximum(n_new, 0) + page - 1) // page
    max_pages, need = int(after.max()) + 1, int((after - held).sum())
    n_pages = int(held.sum()) + need + spare
    pool = r.permutation(n_pages).astype(np.int32)
    table = r.integers(-5, n_pages, (n, max_pages)).astype(np.int32)  # unused entries: anything
    at = 0
    for i, h in enumerate(held):
        table[i, :h] = pool[at:at + h]
        at += h
    stack = np.full(n_pages, -9, np.int32)
    stack[:n_pages - at] = pool[at:]
    return lengths, n_new, table, stack, n_pages, n_pages - at, max_pages, int(np.maximum(n_new, 0).sum())


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("n,page,longest,what", [
    (1, 16, 1, "decode"), (1, 16, 100, "prompts"), (48, 16, 300, "decode"), (300, 32, 200, "mixed"),
    (300, 16, 40, "end"), (1023, 16, 30, "mixed"), (1024, 16, 30, "decode"), (1025, 64, 30, "mixed"),
    (2500, 16, 20, "prompts"), (3, 4096, 9000, "prompts"), (17, 16, 5000, "mixed"), (5000, 16, 3, "mixed")])
def test_plan(paged, n, page, longest, what, in_place):
    for seed in (1, 2):
        lengths, n_new, table, stack, n_pages, n_free, max_pages, rows = plan_problem(seed, n, page, longest, what)
        for extra in (0, 9):
            if rows + extra == 0:
                continue
            got = run_plan(paged, lengths, n_new, page, max_pages, rows + extra, n_pages, n_free, table, stack, in_place)
            want = ref.plan(lengths, n_new, table, stack, n_free, page, n_pages, rows + extra)
            for name, g, w in zip(("status", "lengths", "table", "free_pages", "n_free", "row_start", "positions", "slots"),
                                  got, want):
                assert np.array_equal(g, w), (name, seed, extra)
            assert got[0] == 0


def test_plan_that_cannot_be_met_changes_nothing(paged):
    lengths, n_new, table, stack, n_pages, n_free, max_pages, rows = plan_problem(3, 40, 16, 90, "mixed")
    for change, status in [(dict(max_rows=rows - 1), 2), (dict(n_free=3), 3), (dict(bad=-2), 1), (dict(length=-1), 1),
                           (dict(length=max_pages * 16 + 1), 1), (dict(n_free=-1), 1), (dict(n_free=n_pages), 1),
                           (dict(new=2 ** 31 - 1), 1)]:
        L, N, m, f = lengths.copy(), n_new.copy(), change.get("max_rows", rows), change.get("n_free", n_free)
        i = int(np.argmax(N == 1))
        if "bad" in change:
            N[i] = change["bad"]
        if "length" in change:
            L[i] = change["length"]
        if "new" in change:
            N[i] = change["new"]
        if status == 3:  # (so few free pages that even the released ones do not make up for them)
            N[N < 0] = 0
        want = ref.plan(L, N, table, stack, f, 16, n_pages, m)
        assert want[0] == status, change
        got = run_plan(paged, L, N, 16, max_pages, m, n_pages, f, table, stack)
        for name, g, w in zip(("status", "lengths", "table", "free_pages", "n_free", "row_start", "positions", "slots"),
                              got, want):
            assert np.array_equal(g, w), (name, change)


# ---- norm, rotation, cache write ---------------------------------------------------
ROTARY = [  # heads, kv heads, head dim, rot, neox, rows, page, far
    (28, 4, 128, 128, True, 9, 16, 4000), (28, 4, 128, 128, False, 1, 16, 4000), (8, 8, 64, 32, False, 33, 32, 3000),
    (8, 8, 64, 32, True, 33, 32, 3000), (12, 4, 80, 20, True, 7, 16, 100000), (12, 4, 80, 20, False, 7, 16, 100000),
    (3, 1, 8, 8, True, 5, 16, 50), (5, 5, 24, 6, False, 3, 64, 9), (16, 1, 256, 256, True, 300, 128, 2 ** 31 - 1),
    (16, 1, 256, 64, False, 6, 16, 1 << 20), (2, 2, 40, 0, True, 4, 16, 10), (64, 8, 128, 64, True, 700, 64, 250000),
    (1, 1, 128, 2, True, 2, 16, 10), (2, 1, 128, 2, False, 2, 16, 10), (40, 8, 200, 100, True, 11, 16, 5000)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("heads,kv,hd,rot,neox,rows,page,far", ROTARY)
def test_qk_norm_rope(paged, heads, kv, hd, rot, neox, rows, page, far, norm, kind):
    import torch
    r = np.random.default_rng(heads * 1000 + hd + rows)
    qkv = r.standard_normal((rows, (heads + 2 * kv) * hd)).astype(np.float32) * np.exp(r.standard_normal((rows, 1)) * 3).astype(np.float32)
    positions = r.integers(0, far, rows).astype(np.int32)
    n_pages = -(-rows // page) + 2
    slots = r.permutation(n_pages * page)[:rows].astype(np.int64)
    if rows > 3:
        positions[1] = -1                      # a padding row
        slots[2] = -1                          # a row that is not stored
        slots[3] = n_pages * page              # outside the cache
    freqs, _ = paged.rope_frequencies(1e4, rot) if rot else (None, 1.0)
    magnitude = 1.25 if rot else 1.0
    w = [(1 + 0.3 * r.standard_normal(hd)).astype(np.float32) if norm else None for _ in range(2)]
    ro = paged.Rotary(hd, dev(freqs) if rot else None, paged.ROPE_NEOX if neox else paged.ROPE_NORMAL, magnitude,
                      *(dev(x) if norm else None for x in w), eps=1e-5)
    flat = dev(qkv)
    q, k, v = (t.view(rows, -1, hd) for t in flat.split([heads * hd, kv * hd, kv * hd], 1))
    cache = paged.PagedCache.empty(2, n_pages, page, kv, hd, dtype(kind))
    cache.keys.fill_(3.0)
    cache.values.fill_(-3.0)
    k_out = torch.full((rows, kv, hd), 5.0, device="cuda")
    q_out = torch.full((rows, heads, hd), 5.0, device="cuda")
    paged.qk_norm_rope(ro, q, k, v, dev(positions), q_out=q_out, k_out=k_out, cache=cache, layer=1, slots=dev(slots))
    torch.cuda.synchronize()
    parts = [x.reshape(rows, -1, hd) for x in np.split(qkv, [heads * hd, (heads + kv) * hd], 1)]
    f = freqs if rot else np.zeros(0)
    live = positions >= 0
    want = {}
    for name, got, x, g in (("q", q_out, parts[0], w[0]), ("k", k_out, parts[1], w[1])):
        y, bound = ref.turn(x, g, 1e-5, np.maximum(positions, 0), f, magnitude, rot, neox)
        want[name] = y, bound
        check(host(got)[live], y[live], bound[live], name)
        assert np.all(host(got)[~live] == 5.0)
    assert np.all(host(cache.keys)[0] == 3.0) and np.all(host(cache.values)[0] == -3.0)
    pool = {n: host(t)[1].transpose(0, 2, 1, 3).reshape(-1, kv, hd) for n, t in (("k", cache.keys), ("v", cache.values))}
    put = live & (slots >= 0) & (slots < n_pages * page)
    check(pool["k"][slots[put]], ref.in_range(want["k"][0][put], kind), ref.stored(*want["k"], kind)[put], "keys")
    y = parts[2][put].astype(np.float64)
    rel, small = ref.STEP[kind]
    if kind == "f32":
        assert np.array_equal(pool["v"][slots[put]], y)
    else:
        check(pool["v"][slots[put]], ref.in_range(y, kind), np.abs(y) * rel + small, "values")
    rest = np.ones(n_pages * page, bool)
    rest[slots[put]] = False
    assert np.all(pool["k"][rest] == 3.0) and np.all(pool["v"][rest] == -3.0)
    # without a cache, and in place: the same values
    q2, k2 = paged.qk_norm_rope(ro, q, k, None, dev(np.maximum(positions, 0)))
    paged.qk_norm_rope(ro, q, k, v, dev(positions), q_out=q, k_out=k, cache=cache, layer=0, slots=dev(slots))
    for a, b, c, orig in ((q_out, q2, q, parts[0]), (k_out, k2, k, parts[1])):
        assert np.array_equal(host(a)[live], host(b)[live]) and np.array_equal(host(a)[live], host(c)[live])
        assert np.array_equal(host(c)[~live], orig[~live])


def test_rotary_matches_the_single_sequence_operators(pkg, paged):
    """The same head through mlq_rope and mlq_rmsnorm, within both bounds (mlq_rope's angles are fp32: its own 2.4e-7 pos)."""
    import torch
    r = np.random.default_rng(5)
    q, k = (r.standard_normal((n, 128)).astype(np.float32) for n in (28, 4))
    for rope_type in (paged.ROPE_NORMAL, paged.ROPE_NEOX):
        pos = 300
        qd, kd = dev(q), dev(k)
        pkg._check(pkg.lib().mlq_rope(qd.data_ptr(), kd.data_ptr(), 28, 4, 128, pos, 1e4, rope_type, pkg._stream()), "mlq_rope")
        f, _ = paged.rope_frequencies(1e4, 128)
        qo, ko = paged.qk_norm_rope(paged.Rotary(128, dev(f), rope_type), dev(q)[None], dev(k)[None], None,
                                    dev(np.array([pos], np.int32)))
        torch.cuda.synchronize()
        for a, b, x in ((qo[0], qd, q), (ko[0], kd, k)):
            assert np.all(np.abs(host(a) - host(b)) <= 1e-5 + 2.4e-7 * pos * np.abs(x).max())


# ---- attention -----------------------------------------------------------------------
class Problem:
    """A cache with sequences of `lengths`, everything nobody owns NaN or inf."""

    def __init__(self, paged, kind, lengths, heads, kv, hd, page, seed=0, layers=1, q_scale=1.5, new=None, extra_pages=0):
        import torch
        r = np.random.default_rng(seed + 17 * len(lengths) + hd)
        lengths = np.asarray(lengths)
        self.new = np.ones(len(lengths), np.int64) if new is None else np.asarray(new)
        pages = -(-lengths // page)
        n_pages = int(pages.sum()) + 2
        order = r.permutation(n_pages)
        most = max(1, int(pages.max())) + extra_pages
        self.table = np.full((len(lengths), most), -1, np.int32)
        at = 0
        for i, p in enumerate(pages):
            self.table[i, :p] = order[at:at + p]
            at += p
        shape = (layers, n_pages, kv, page, hd)
        pools = [r.standard_normal(shape).astype(np.float32) for _ in range(2)]
        used = np.zeros((n_pages, page), bool)
        for i, n in enumerate(lengths):
            for t in range(n):
                used[self.table[i, t // page], t % page] = True
        for p, junk in zip(pools, (np.nan, np.inf)):
            hole = np.broadcast_to(~used[None, :, None, :, None], shape)
            p[hole] = np.where(r.random(int(hole.sum())) < 0.5, junk, np.nan)
        self.cache = paged.PagedCache(*(dev(p, dtype(kind)) for p in pools))
        self.k, self.v = host(self.cache.keys), host(self.cache.values)
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
        scale = rule.pop("scale", None) or 1 / math.sqrt(self.hd)
        for i, n in enumerate(self.lengths):
            k, v = (ref.gather(p[layer], self.table[i], int(n)) for p in (self.k, self.v))
            for r in range(self.start[i], self.start[i + 1]):
                if rows is None or r in rows:
                    pos = int(n) - (self.start[i + 1] - r)
                    got[r] = ref.attention(self.q[r], k, v, pos, scale, kind=self.kind, **rule)
        return got

    def compare(self, out, want, what=""):
        out = host(out)
        for r, (y, bound) in want.items():
            check(out[r], y, bound, (what, r))


def rule_of(paged, heads, softcap=0.0, window=0, slopes=False, scale=None):
    s = np.array([2.0 ** (-8.0 * (i + 1) / heads) for i in range(heads)], np.float32) if slopes else None
    return (paged.AttentionRule(scale, softcap, window, dev(s) if slopes else None),
            dict(softcap=softcap, window=window, slopes=s, scale=scale))


SHAPES = [(28, 4, 128), (8, 8, 64), (16, 1, 256), (12, 4, 80), (3, 1, 8), (40, 2, 64), (33, 1, 128), (4, 4, 200), (24, 2, 128), (5, 5, 96)]
EDGES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65, 100, 127, 128, 129, 255, 257, 600]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("heads,kv,hd", SHAPES)
def test_decode_edges(paged, heads, kv, hd, page, kind):
    import torch
    p = Problem(paged, kind, EDGES, heads, kv, hd, page)
    out = paged.attention_decode(p.cache, 0, p.batch, p.qd)
    torch.cuda.synchronize()
    p.compare(out, p.want())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rule", [dict(softcap=20.0), dict(window=1), dict(window=37), dict(slopes=True), dict(scale=0.3),
                                  dict(softcap=30.0, window=100, slopes=True), dict(scale=-0.2, softcap=2.0)])
@pytest.mark.parametrize("heads,kv,hd", [(28, 4, 128), (16, 16, 64), (4, 1, 256), (40, 2, 72)])
def test_decode_rules(paged, heads, kv, hd, rule, kind):
    import torch
    p = Problem(paged, kind, EDGES, heads, kv, hd, 32, seed=3)
    own, plain = rule_of(paged, heads, **rule)
    out = paged.attention_decode(p.cache, 0, p.batch, p.qd, rule=own)
    torch.cuda.synchronize()
    p.compare(out, p.want(**plain), rule)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv,hd,page,lengths", [
    (28, 4, 128, 16, [9001]), (28, 4, 128, 128, [5000, 1, 4097, 300]), (8, 8, 64, 64, [20000, 0, 7]), (16, 1, 256, 16, [3000, 6001]),
    (12, 4, 80, 32, [7777, 12]), (32, 8, 128, 4096, [10000, 8192, 8193])])
def test_decode_long(paged, heads, kv, hd, page, lengths, kind):
    import torch
    p = Problem(paged, kind, lengths, heads, kv, hd, page, seed=5)
    for rule in (dict(), dict(window=2500, softcap=50.0)):
        own, plain = rule_of(paged, heads, **rule)
        out = paged.attention_decode(p.cache, 0, p.batch, p.qd, rule=own)
        again = paged.attention_decode(p.cache, 0, p.batch, p.qd, rule=own)
        torch.cuda.synchronize()
        p.compare(out, p.want(**plain), rule)
        assert torch.equal(out, again)


@pytest.mark.parametrize("seqs", [1, 3, 40, 300])
def test_decode_result_does_not_depend_on_the_bound(paged, seqs):
    """A tight max_len and a loose one split the keys differently: the same results within the bounds; rows past are left."""
    import torch
    r = np.random.default_rng(seqs)
    p = Problem(paged, "bf16", r.integers(1, 900, seqs), 28, 4, 128, 16, seed=7, extra_pages=3000)
    want = p.want(rows=set(range(0, p.rows, 7)))
    for max_len in (900, 3000, None):
        out = torch.full((p.rows + 2, 28, 128), 9.0, device="cuda")
        q = torch.cat([p.qd, p.qd[:1], p.qd[:1]])
        paged.attention_decode(p.cache, 0, p.batch, q, out=out, max_len=max_len)
        torch.cuda.synchronize()
        p.compare(out, want, max_len)
        assert torch.all(out[p.rows:] == 9.0)


@pytest.mark.parametrize("row_start", [False, True])
def test_decode_of_more_sequences_than_a_launch_takes(paged, row_start):
    import torch
    r = np.random.default_rng(8)
    n = 4100
    p = Problem(paged, "bf16", r.integers(0, 40, n), 4, 2, 64, 16, seed=19, new=(r.random(n) < 0.9).astype(int) if row_start else None)
    if not row_start:
        p.batch = paged.PagedBatch(p.batch.block_table, p.batch.lengths)
    out = paged.attention_decode(p.cache, 0, p.batch, p.qd)
    long = paged.attention_decode(p.cache, 0, p.batch, p.qd, max_len=p.table.shape[1] * 16)
    torch.cuda.synchronize()
    p.compare(out, p.want(rows=set(range(0, p.rows, 50)) | set(range(p.rows - 40, p.rows))))
    assert torch.equal(out, long)


def test_decode_rows_of_sequences_without_a_new_token(paged):
    """row_start names the rows: sequences that wait have none; of several new rows the last one is computed."""
    import torch
    p = Problem(paged, "f32", [40, 50, 60, 70, 0], 8, 4, 64, 16, new=[1, 0, 3, 1, 0])
    out = torch.full((p.rows, 8, 64), 9.0, device="cuda")
    paged.attention_decode(p.cache, 0, p.batch, p.qd, out=out)
    torch.cuda.synchronize()
    p.compare(out, p.want(rows={0, 3, 4}))
    assert torch.all(out[1:3] == 9.0)
    # no row_start: row i is sequence i
    p = Problem(paged, "f32", [40, 0, 60], 8, 4, 64, 16)
    b = paged.PagedBatch(p.batch.block_table, p.batch.lengths)
    out = paged.attention_decode(p.cache, 0, b, p.qd)
    torch.cuda.synchronize()
    p.compare(out, p.want())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("prefill", [False, True])
def test_bad_device_numbers_give_nan_rows_alone(paged, prefill, kind):
    """A page outside the cache or a length past the table: that sequence's rows are NaN, the others' are right."""
    import torch
    lengths = [100, 333, 70, 200, 500, 90]
    p = Problem(paged, kind, lengths, 8, 2, 128, 16, seed=9, new=None if not prefill else [3, 2, 5, 1, 4, 90])
    want = p.want()
    call = paged.attention_prefill if prefill else paged.attention_decode
    table, n = p.batch.block_table, p.batch.lengths
    table[1, 5] = p.cache.n_pages
    table[3, 0] = -1
    table[4, 31] = 2 ** 31 - 1
    n[2] = p.batch.max_pages * 16 + 1
    out = call(p.cache, 0, p.batch, p.qd)
    torch.cuda.synchronize()
    bad = {r for i in (1, 2, 3, 4) for r in range(p.start[i], p.start[i + 1])}
    o = host(out)
    for r in range(p.rows):
        if r in bad:
            assert np.all(np.isnan(o[r])), r
    p.compare(out, {r: w for r, w in want.items() if r not in bad})
    for length, value in ((-5, 0.0), (-2 ** 31, 0.0), (2 ** 31 - 1, math.nan)):  # negative: nothing to see
        n.fill_(length)
        out = call(p.cache, 0, p.batch, p.qd)
        torch.cuda.synchronize()
        assert np.array_equal(host(out), np.full(out.shape, value), equal_nan=True), length


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("prefill", [False, True])
def test_non_finite_values(paged, prefill, kind):
    """A NaN key or an infinite value that a row sees makes its heads' outputs non-finite, and no other's; behind the
    window or the row's position they are not seen."""
    import torch
    p = Problem(paged, kind, [200, 200, 200], 8, 4, 128, 16, seed=11, new=None if not prefill else [150, 150, 150])
    at = lambda i, t: (0, int(p.table[i, t // 16]), slice(None), t % 16)  # noqa: E731
    for pool, (i, t), kvh, value in ((p.cache.keys, (0, 120), 1, math.nan), (p.cache.values, (1, 120), 2, math.inf),
                                     (p.cache.values, (2, 20), 0, math.nan)):
        l, page, _, off = at(i, t)
        pool[l, page, kvh, off, 5] = value
    p.k, p.v = host(p.cache.keys), host(p.cache.values)
    own, plain = rule_of(paged, 8, window=100)
    call = paged.attention_prefill if prefill else paged.attention_decode
    out = call(p.cache, 0, p.batch, p.qd, rule=own)
    torch.cuda.synchronize()
    out = host(out)
    k, v = np.nan_to_num(p.k, nan=0, posinf=0), np.nan_to_num(p.v, nan=0, posinf=0)
    p.k, p.v = k, v
    for r, (y, bound) in p.want(**plain).items():
        i = int(np.searchsorted(p.start, r, side="right")) - 1
        pos = 200 - (p.start[i + 1] - r)
        for h in range(8):
            sees = lambda t: t <= pos < t + 100  # noqa: E731
            if i == 0 and h // 2 == 1 and sees(120):
                assert np.all(np.isnan(out[r, h]))
            elif i == 1 and h // 2 == 2 and sees(120):
                assert not np.isfinite(out[r, h, 5])
                rest = np.arange(128) != 5
                check(out[r, h, rest], y[h, rest], bound[h, rest], (r, h))
            elif i == 2 and h // 2 == 0 and sees(20):
                assert np.isnan(out[r, h, 5])
            else:
                check(out[r, h], y[h], bound[h], (r, h))


@pytest.mark.parametrize("kind", KINDS)
def test_large_and_tiny_queries(paged, kind):
    """Queries whose size is far from 1: scores that overflow an fp16 product, weights that underflow, a single winner."""
    import torch
    for scale in (1e-30, 1e-6, 3e3, 1e6):
        p = Problem(paged, kind, [1, 70, 300], 8, 4, 64, 16, seed=13, q_scale=scale)
        own, plain = rule_of(paged, 8, scale=0.125 / max(scale, 1.0) * 10)
        for call in (paged.attention_decode, paged.attention_prefill):
            out = call(p.cache, 0, p.batch, p.qd, rule=own)
            torch.cuda.synchronize()
            p.compare(out, p.want(**plain), scale)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size", [1e-6, 1e-3, 1e3])
def test_values_of_other_sizes(paged, size, kind):
    """Cached keys and values far from 1, for fp16 subnormals among them: as they are stored."""
    import torch
    p = Problem(paged, kind, [1, 70, 300, 40], 8, 4, 64, 16, seed=15, new=[1, 70, 9, 0])
    for pool in (p.cache.keys, p.cache.values):
        pool.copy_((pool.float() * size).to(pool.dtype))
    p.k, p.v = host(p.cache.keys), host(p.cache.values)
    own, plain = rule_of(paged, 8, scale=0.2 / max(size, 1.0))
    out = paged.attention_prefill(p.cache, 0, p.batch, p.qd, rule=own)
    last = paged.attention_decode(p.cache, 0, p.batch, p.qd, rule=own)
    torch.cuda.synchronize()
    want = p.want(**plain)
    p.compare(out, want, size)
    p.compare(last, {int(s) - 1: want[int(s) - 1] for s in p.start[1:]}, size)


@pytest.mark.parametrize("kind", KINDS)
def test_a_query_that_is_not_finite_stays_alone(paged, kind):
    import torch
    p = Problem(paged, kind, [150, 200, 90], 8, 2, 64, 16, seed=17, new=[60, 1, 90])
    clean = paged.attention_prefill(p.cache, 0, p.batch, p.qd)
    last = paged.attention_decode(p.cache, 0, p.batch, p.qd)
    q = p.qd.clone()
    q[30, 2, 5], q[60, 4, 0], q[100, 7, 63] = math.nan, math.inf, -math.inf
    out = paged.attention_prefill(p.cache, 0, p.batch, q)
    one = paged.attention_decode(p.cache, 0, p.batch, q)
    torch.cuda.synchronize()
    hit = torch.zeros(p.rows, 8, dtype=torch.bool, device="cuda")
    for r, h in ((30, 2), (60, 4), (100, 7)):
        hit[r, h] = True
    assert torch.all(torch.isnan(out[hit])) and torch.equal(out[~hit], clean[~hit])
    assert torch.all(torch.isnan(one[60, 4]))
    hit[30, 2] = hit[100, 7] = False  # (not the last rows of their sequences)
    assert torch.equal(one[~hit], last[~hit])


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
    torch.cuda.synchronize()
    step = max(1, p.rows // 60)
    rows = set(range(0, p.rows, step)) | {int(s) + d for s in p.start for d in (-1, 0) if 0 <= s + d < p.rows}
    p.compare(out, p.want(rows=rows))
    assert torch.all(out[p.rows:] == 9.0)  # rows behind the last sequence


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rule", [dict(softcap=20.0), dict(window=1), dict(window=50), dict(slopes=True), dict(scale=0.3, window=200, softcap=30.0, slopes=True)])
@pytest.mark.parametrize("heads,kv,hd", [(28, 4, 128), (4, 4, 64), (16, 1, 256), (6, 2, 80)])
def test_prefill_rules(paged, heads, kv, hd, rule, kind):
    import torch
    p = Problem(paged, kind, [400, 90, 1, 350], heads, kv, hd, 32, seed=23, new=[250, 90, 1, 3])
    own, plain = rule_of(paged, heads, **rule)
    out = paged.attention_prefill(p.cache, 0, p.batch, p.qd, rule=own)
    torch.cuda.synchronize()
    p.compare(out, p.want(rows=set(range(0, p.rows, 6)), **plain), rule)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("window", [64, 2 ** 31 - 1])
def test_prefill_rows_before_the_first_key(paged, window, kind):
    """More rows than tokens: the first ones see nothing and are zeros, the last ones what they would."""
    import torch
    p = Problem(paged, kind, [150, 40, 90], 8, 2, 64, 16, seed=33, new=[150, 40, 90])
    kept = p.lengths = np.array([30, 0, 89])
    p.batch.lengths.copy_(dev(kept.astype(np.int32)))
    out = paged.attention_prefill(p.cache, 0, p.batch, p.qd, rule=paged.AttentionRule(window=window))
    torch.cuda.synchronize()
    lost = {int(p.start[i]) + j for i, n in enumerate(kept) for j in range(int(p.new[i] - n))}
    assert torch.all(out[sorted(lost)] == 0.0)
    p.compare(out, p.want(rows=set(range(p.rows)) - lost, window=window))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv,hd,lengths,new", [(28, 4, 128, [2100, 1500, 60], [1900, 800, 60]), (8, 8, 64, [3000], [1537]), (16, 1, 256, [1300], [700])])
def test_prefill_long(paged, heads, kv, hd, lengths, new, kind):
    import torch
    p = Problem(paged, kind, lengths, heads, kv, hd, 64, seed=25, new=new, layers=2)
    out = paged.attention_prefill(p.cache, 1, p.batch, p.qd)
    again = paged.attention_prefill(p.cache, 1, p.batch, p.qd)
    torch.cuda.synchronize()
    p.compare(out, p.want(layer=1, rows=set(range(0, p.rows, 131)) | {p.rows - 1}))
    assert torch.equal(out, again)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [255, 256, 257, 700])
@pytest.mark.parametrize("heads,kv,hd", [(28, 4, 128), (4, 4, 64), (5, 1, 80)])
def test_prefill_of_many_sequences(paged, heads, kv, hd, n, kind):
    """Tiles are given out in another way from 257 sequences on; some have no rows, one has several tiles."""
    import torch
    r = np.random.default_rng(n)
    lengths = r.integers(0, 50, n)
    lengths[n // 2] = 300
    new = np.minimum(r.choice([0, 1, 1, 2, 40], n), lengths)
    new[n // 2], new[-1], new[0] = 290, 0, 0
    p = Problem(paged, kind, lengths, heads, kv, hd, 16, seed=31, new=new)
    out = torch.full((p.rows + 3, heads, hd), 9.0, device="cuda")
    q = torch.cat([p.qd, p.qd[:1], p.qd[:1], p.qd[:1]])
    paged.attention_prefill(p.cache, 0, p.batch, q, out=out)
    torch.cuda.synchronize()
    p.compare(out, p.want(rows=set(range(0, p.rows, 7)) | {p.rows - 1}))
    assert torch.all(torch.isfinite(out)) and torch.all(out[p.rows:] == 9.0)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv,hd,lengths,new", [
    (28, 4, 128, [5000], [3]), (8, 8, 64, [3000, 10, 900, 0], [20, 10, 1, 0]), (16, 1, 256, [1300, 2000], [5, 4]), (33, 1, 128, [700], [9]),
    (12, 4, 80, [4000, 130, 2000, 20], [1, 2, 40, 20]), (4, 4, 128, [600, 600], [300, 5])])
def test_prefill_of_few_rows_behind_long_contexts(pkg, paged, heads, kv, hd, lengths, new, kind):
    """Their keys are shared by several workgroups and joined: plain, with a rule, with a bad page, with a NaN that some rows see."""
    import torch
    p = Problem(paged, kind, lengths, heads, kv, hd, 16, seed=27, new=new)
    need = paged.attention_workspace_bytes(p.cache, heads, len(lengths), p.table.shape[1] * 16, rows=p.rows)
    assert need > 0
    ws = torch.full((need,), 255, dtype=torch.uint8, device="cuda")  # (NaN wherever nothing is written)
    rows = set(range(0, p.rows, max(1, p.rows // 40))) | {p.rows - 1}
    for rule in (dict(), dict(softcap=20.0, slopes=True), dict(window=300), dict(scale=-0.1)):
        own, plain = rule_of(paged, heads, **rule)
        out = paged.attention_prefill(p.cache, 0, p.batch, p.qd, rule=own, workspace=ws)
        again = paged.attention_prefill(p.cache, 0, p.batch, p.qd, rule=own)
        torch.cuda.synchronize()
        p.compare(out, p.want(rows=rows, **plain), rule)
        assert torch.equal(out, again)
    with pytest.raises(pkg.MLQError):
        paged.attention_prefill(p.cache, 0, p.batch, p.qd, workspace=ws[:need - 256])
    # the first sequence's key 100 holds an infinite value, key 300 lies on a page outside the cache
    clean = out.clone()
    page = int(p.table[0, 100 // 16])
    p.cache.values[0, page, kv - 1, 100 % 16, 3] = math.inf
    out = paged.attention_prefill(p.cache, 0, p.batch, p.qd, rule=own, workspace=ws)
    torch.cuda.synchronize()
    hit = heads - heads // kv
    n0 = int(p.start[1])
    assert torch.equal(out[n0:], clean[n0:]) and torch.equal(out[:n0, :hit], clean[:n0, :hit])
    first = int(p.lengths[0]) - n0  # (rows before key 100 do not see it)
    assert torch.all(~torch.isfinite(out[max(0, 100 - first):n0, hit:, 3]))
    assert torch.all(torch.isfinite(out[:max(0, 100 - first)]))
    p.batch.block_table[0, 300 // 16] = -7
    out = paged.attention_prefill(p.cache, 0, p.batch, p.qd, rule=own, workspace=ws)
    torch.cuda.synchronize()
    assert torch.equal(out[n0:], clean[n0:])
    assert torch.all(torch.isnan(out[max(0, 304 - first):n0]))
    assert torch.all(torch.isfinite(out[:max(0, 100 - first)]))


def test_decode_matches_the_single_sequence_attention(pkg, paged):
    """One sequence's attention through mlq_attention_decode over its own layout."""
    import ctypes

    import torch
    p = Problem(paged, "f32", [1234], 28, 4, 128, 16, seed=31)
    k, v = (dev(ref.gather(x[0], p.table[0], 1234).transpose(1, 0, 2).astype(np.float32)) for x in (p.k, p.v))
    c = pkg.MlqKvCache(k.data_ptr(), v.data_ptr(), 1, 1234, 4, 128)
    need = ctypes.c_size_t()
    pkg._check(pkg.lib().mlq_attention_workspace(ctypes.byref(c), 28, ctypes.byref(need)), "workspace")
    ws = torch.empty(need.value, dtype=torch.uint8, device="cuda")
    one = torch.empty((28, 128), device="cuda")
    q = dev(p.q[0])
    pkg._check(pkg.lib().mlq_attention_decode(ctypes.byref(c), 0, 1233, q.data_ptr(), 28, one.data_ptr(), ws.data_ptr(),
                                              ws.numel(), pkg._stream()), "mlq_attention_decode")
    out = paged.attention_decode(p.cache, 0, p.batch, p.qd)
    torch.cuda.synchronize()
    bound = p.want()[0][1]
    check(host(out[0]), host(one), 2 * bound, "single")


# ---- streams, graphs, the operators together --------------------------------------------
def test_another_stream_and_a_workspace_of_the_callers(pkg, paged):
    import torch
    p = Problem(paged, "bf16", [3000, 2000], 28, 4, 128, 16, seed=33)
    plain = paged.attention_decode(p.cache, 0, p.batch, p.qd)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    need = paged.attention_workspace_bytes(p.cache, 28, 2, p.batch.max_pages * 16)
    ws = torch.empty(max(need, 256), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    outs = [paged.attention_decode(p.cache, 0, p.batch, p.qd, stream=s, workspace=ws) for _ in range(3)]
    outs += [paged.attention_decode(p.cache, 0, p.batch, p.qd, stream=s) for _ in range(3)]
    with torch.cuda.stream(s):
        outs.append(paged.attention_decode(p.cache, 0, p.batch, p.qd))
    s.synchronize()
    assert all(torch.equal(o, plain) for o in outs)
    if need:
        with pytest.raises(pkg.MLQError):
            paged.attention_decode(p.cache, 0, p.batch, p.qd, workspace=ws[:need - 256])


class Loop:
    """A serving loop's layer: plan, rotate and store, attend; and the same in 64 bits from the plain history."""

    def __init__(self, paged, kind, heads=8, kv=2, hd=64, page=16, seqs=5, max_pages=12, max_rows=200, n_pages=40):
        import torch
        self.paged, self.kind, self.heads, self.kv, self.hd, self.seqs = paged, kind, heads, kv, hd, seqs
        self.cache = paged.PagedCache.empty(1, n_pages, page, kv, hd, dtype(kind))
        for t in (self.cache.keys, self.cache.values):
            t.fill_(math.nan)
        self.batch = paged.PagedBatch.empty(seqs, max_pages, max_rows)
        self.free = dev(np.random.default_rng(3).permutation(n_pages).astype(np.int32))
        self.n_free = torch.full((1,), n_pages, dtype=torch.int32, device="cuda")
        self.n_new = torch.zeros(seqs, dtype=torch.int32, device="cuda")
        self.freqs, _ = paged.rope_frequencies(1e4, hd // 2)
        self.w = [(1 + 0.2 * np.random.default_rng(i).standard_normal(hd)).astype(np.float32) for i in range(2)]
        self.rotary = paged.Rotary(hd, dev(self.freqs), paged.ROPE_NEOX, 1.0, dev(self.w[0]), dev(self.w[1]), 1e-6)
        self.rule, self.plain = rule_of(paged, heads, softcap=30.0)
        self.qkv = torch.zeros((max_rows, (heads + 2 * kv) * hd), device="cuda")
        self.q_out = torch.zeros((max_rows, heads, hd), device="cuda")
        self.out = torch.zeros((max_rows, heads, hd), device="cuda")
        self.k, self.v = [np.zeros((0, kv, hd)) for _ in range(seqs)], [np.zeros((0, kv, hd)) for _ in range(seqs)]

    def launch(self, rows, decode):
        paged, h, kv, hd = self.paged, self.heads, self.kv, self.hd
        paged.plan(self.batch, self.batch.lengths, self.n_new, self.free, self.n_free, self.cache.page_size)
        q, k, v = (t.view(rows, -1, hd) for t in self.qkv[:rows].split([h * hd, kv * hd, kv * hd], 1))
        paged.qk_norm_rope(self.rotary, q, k, v, self.batch.positions, q_out=self.q_out[:rows], cache=self.cache,
                           slots=self.batch.slots)
        call = paged.attention_decode if decode else paged.attention_prefill
        call(self.cache, 0, self.batch, self.q_out[:rows], out=self.out[:rows], rule=self.rule)

    def expect(self, n_new, qkv):
        """{row: (out, bound)} after the step, from histories of keys and values as the cache holds them."""
        h, kv, hd = self.heads, self.kv, self.hd
        got, r = {}, 0
        for i, n in enumerate(n_new):
            if n < 0:
                self.k[i], self.v[i] = np.zeros((0, kv, hd)), np.zeros((0, kv, hd))
            for _ in range(max(0, n)):
                pos = len(self.k[i])
                q, k, v = (x.reshape(1, -1, hd) for x in np.split(qkv[r].astype(np.float64), [h * hd, (h + kv) * hd]))
                (q, qb), (k, kb) = (ref.turn(x, w, 1e-6, [pos], self.freqs, 1.0, hd // 2, True) for x, w in ((q, self.w[0]), (k, self.w[1])))
                self.k[i] = np.concatenate([self.k[i], k])
                self.v[i] = np.concatenate([self.v[i], v])
                got[r] = (i, pos, q[0])
                r += 1
        want = {}
        rel = max(ref.STEP[self.kind][0], 1e-6)  # what keys, values and queries may be off by
        for r, (i, pos, q) in got.items():
            k, v = self.k[i].transpose(1, 0, 2), self.v[i].transpose(1, 0, 2)
            y, bound = ref.attention(q, k, v, pos, 1 / math.sqrt(hd), softcap=30.0)
            size = np.abs(q).sum(1).max() * np.abs(k[:, :pos + 1]).max() / math.sqrt(hd)
            want[r] = y, bound + 2 * (rel * size * 2 + rel) * np.abs(v[:, :pos + 1]).max()
        return want

    def feed(self, n_new, seed):
        rows = int(np.maximum(n_new, 0).sum())
        qkv = np.random.default_rng(seed).standard_normal((rows, self.qkv.shape[1])).astype(np.float32)
        self.qkv[:rows].copy_(dev(qkv))
        self.n_new.copy_(dev(np.asarray(n_new, np.int32)))
        return self.expect(n_new, qkv)

    def compare(self, want, what):
        import torch
        torch.cuda.synchronize()
        assert int(self.batch.status.item()) == 0
        assert host(self.batch.lengths).tolist() == [len(k) for k in self.k]
        out = host(self.out)
        for r, (y, bound) in want.items():
            check(out[r], y, bound, (what, r))


@pytest.mark.parametrize("kind", KINDS)
def test_serving_loop(paged, kind):
    """Prompts, steps of one token, sequences that end, wait and come back on pages of others."""
    loop = Loop(paged, kind)
    steps = [[20, 33, 0, 1, 16], [1, 1, 50, 1, 1], [1, 1, 1, 1, 1], [-1, 1, 1, 0, -1], [70, 1, 1, 1, 0], [1, -1, 17, 1, 40], [1, 12, 1, 1, 1],
             [1, 1, 1, 1, 1], [-1, -1, -1, -1, -1], [100, 2, 3, 60, 5], [1, 1, 1, 1, 1]]
    for i, n_new in enumerate(steps):
        want = loop.feed(n_new, i)
        rows = max(1, int(np.maximum(n_new, 0).sum()))
        loop.launch(rows, decode=max(n_new) <= 1)
        loop.compare(want, i)
    import torch
    held = sum(-(-len(k) // 16) for k in loop.k)
    assert int(loop.n_free.item()) == 40 - held
    left = set(host(loop.free)[:40 - held].tolist())
    used = {int(p) for i, k in enumerate(loop.k) for p in host(loop.batch.block_table)[i, :-(-len(k) // 16)]}
    assert len(left) == 40 - held and not left & used and torch.all(loop.batch.status == 0)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_serving_step_in_a_graph(paged, kind):
    """The decode step captured once and replayed while lengths, pages and rows change, with eager work between the
    replays; a second graph of another loop with a workspace of its own replays in between."""
    import torch
    loops = [Loop(paged, kind), Loop(paged, kind, heads=6, kv=6)]
    graphs = []
    for loop in loops:
        loop.compare(_prompts(loop), "prompts")
        state = [t.clone() for t in (loop.batch.lengths, loop.batch.block_table, loop.free, loop.n_free)]
        loop.n_new.fill_(1)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            loop.launch(5, decode=True)  # (once before the capture, then taken back)
        torch.cuda.current_stream().wait_stream(s)
        for t, was in zip((loop.batch.lengths, loop.batch.block_table, loop.free, loop.n_free), state):
            t.copy_(was)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            loop.launch(5, decode=True)
        graphs.append(g)
    for step in range(6):
        for j, (loop, g) in enumerate(zip(loops, graphs)):
            n_new = [1, 1, 1, 0 if step == 2 else 1, -1 if step == 4 else 1]
            want = loop.feed(n_new, 100 * j + step)
            g.replay()
            loop.compare(want, (j, step))
            torch.zeros(1000, device="cuda").sum().item()


def test_two_captured_calls_at_once(paged):
    """Attention of two batches captured apart, replayed on two streams at once while lengths change between the replays."""
    import torch
    problems = [Problem(paged, "bf16", [4000, 2100, 900], 28, 4, 128, 16, seed=51, new=[1, 3, 2]),
                Problem(paged, "f32", [3000, 5000], 8, 8, 64, 32, seed=53, new=[2, 1])]
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
            p.batch.lengths.copy_(dev((p.lengths - 17 * step).astype(np.int32)))
            both()
            want.append([o.clone() for o in outs])
            for o in outs:
                o.zero_()
        torch.cuda.synchronize()
        for both, outs, g, s in calls:
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for w, (both, outs, g, s) in zip(want, calls):
            n = [torch.equal(a, b) for a, b in zip(w, outs)]
            assert n[1] and torch.equal(w[0][outs[0] != 0], outs[0][outs[0] != 0]), step
            assert bool((outs[0] != 0).any())


def _prompts(loop):
    n_new = [20, 33, 5, 1, 16]
    want = loop.feed(n_new, 99)
    loop.launch(75, decode=False)
    return want


def test_one_page_used_by_two_sequences(paged):
    """A prefix shared by two sequences: the same pages in both tables."""
    import torch
    p = Problem(paged, "f16", [100, 100], 8, 2, 64, 16, seed=41)
    p.table[1, :4] = p.table[0, :4]
    p.batch.block_table.copy_(dev(p.table))
    out = paged.attention_decode(p.cache, 0, p.batch, p.qd)
    torch.cuda.synchronize()
    p.compare(out, p.want())


def test_offsets_past_32_bits(paged):
    """Pages whose elements lie past 2^31 (and whose bytes past 2^32) of one layer."""
    import torch
    n_pages, kv, page, hd = 70000, 4, 64, 128  # 2.29e9 elements an array
    cache = paged.PagedCache(torch.zeros((1, n_pages, kv, page, hd), dtype=torch.bfloat16, device="cuda"),
                             torch.zeros((1, n_pages, kv, page, hd), dtype=torch.bfloat16, device="cuda"))
    r = np.random.default_rng(43)
    table = np.array([[69999, 3, 65537, 69998]], np.int32)
    rows, heads = 200, 8
    qkv = r.standard_normal((rows, (heads + 2 * kv) * hd)).astype(np.float32)
    q, k, v = (t.view(rows, -1, hd) for t in dev(qkv).split([heads * hd, kv * hd, kv * hd], 1))
    positions = np.arange(rows)
    slots = table[0, positions // page].astype(np.int64) * page + positions % page
    paged.qk_norm_rope(paged.Rotary(hd), q, k, v, dev(positions.astype(np.int32)), cache=cache, slots=dev(slots))
    batch = paged.PagedBatch(dev(table), dev(np.array([rows], np.int32)), dev(np.array([0, rows], np.int32)))
    out = paged.attention_prefill(cache, 0, batch, q)
    one = paged.attention_decode(cache, 0, batch, q)
    torch.cuda.synchronize()
    kk, vv = (host(t.to(torch.bfloat16)).transpose(1, 0, 2) for t in (k, v))
    for r_ in (0, 63, 64, 150, 199):
        y, bound = ref.attention(host(q)[r_], kk, vv, r_, 1 / math.sqrt(hd))
        check(host(out[r_]), y, bound, r_)
    check(host(one[199]), y, bound, "decode")


# ---- pages behind a window ---------------------------------------------------------------
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("heads,kv,hd", [(8, 2, 64), (28, 4, 128), (4, 1, 256)])
def test_pages_behind_the_window_are_not_asked_for(paged, heads, kv, hd, page, kind):
    """Wherever the window begins in a tile of keys or a page: a table entry of a page wholly behind the window of the
    sequence's first new row may be anything, and the results are those of a whole table, bit for bit."""
    import torch
    window = 50
    ends = [1, 50, 51, 65, 66, 67, 81, 82, 83, 97, 98, 99, 113, 114, 130, 200, 1003, 2000]
    for new in (None, [min(n, 1 + 7 * i % 40) for i, n in enumerate(ends)]):
        p = Problem(paged, kind, ends, heads, kv, hd, page, seed=61, new=new)
        own, plain = rule_of(paged, heads, window=window)
        call = paged.attention_decode if new is None else paged.attention_prefill
        whole = call(p.cache, 0, p.batch, p.qd, rule=own)
        torch.cuda.synchronize()
        p.compare(whole, p.want(rows=set(range(0, p.rows, 3)) | {int(s) - 1 for s in p.start[1:]}, **plain))
        first = p.lengths - p.new + 1 - window  # the first key that a row sees
        for junk in (-1, p.cache.n_pages, 2 ** 31 - 1):
            table = p.table.copy()
            for i, f in enumerate(first):
                table[i, :max(0, int(f)) // page] = junk
            assert (table != p.table).any()
            p.batch.block_table.copy_(dev(table))
            out = call(p.cache, 0, p.batch, p.qd, rule=own)
            torch.cuda.synchronize()
            bad = [int(n) for i, n in enumerate(p.lengths)
                   if not torch.equal(out[p.start[i]:p.start[i + 1]], whole[p.start[i]:p.start[i + 1]])]
            assert not bad, (junk, bad)


@pytest.mark.parametrize("kind", KINDS)
def test_decode_of_many_short_pieces_in_a_workspace_of_the_longest_bound(paged, kind):
    """Small heads, many of them: twice the ranges a CU, several pieces each; a workspace sized for the longest bound
    that a table can have serves a call with a small one."""
    import torch
    r = np.random.default_rng(12)
    lengths = np.concatenate([[0, 1, 899], r.integers(1, 900, 117)])
    p = Problem(paged, kind, lengths, 16, 16, 64, 16, seed=63)
    bound = p.batch.max_pages * 16
    need = [paged.attention_workspace_bytes(p.cache, 16, len(lengths), n) for n in (bound, 2 ** 30)]
    assert 0 < need[0] <= need[1]
    ws = torch.full((need[1],), 255, dtype=torch.uint8, device="cuda")
    out = paged.attention_decode(p.cache, 0, p.batch, p.qd, workspace=ws)
    again = paged.attention_decode(p.cache, 0, p.batch, p.qd)
    torch.cuda.synchronize()
    p.compare(out, p.want(rows={0, 1, 2} | set(range(3, p.rows, 4))))
    assert torch.equal(out, again)


def test_tensors_of_a_batch_and_a_cache_are_not_replaced(paged):
    """Their contents change in place; another tensor in a tensor's place is refused."""
    import torch
    p = Problem(paged, "bf16", [40, 90], 8, 2, 64, 16, seed=65)
    for obj, names in ((p.batch, ("block_table", "lengths", "row_start", "positions", "max_rows", "n_seqs")),
                       (p.cache, ("keys", "values", "n_pages"))):
        for name in names:
            was = getattr(obj, name)
            with pytest.raises(AttributeError):
                setattr(obj, name, torch.zeros(2, dtype=torch.int32, device="cuda"))
            assert getattr(obj, name) is was
    p.lengths = np.array([33, 71])
    p.batch.lengths.copy_(dev(p.lengths.astype(np.int32)))
    out = paged.attention_decode(p.cache, 0, p.batch, p.qd)
    torch.cuda.synchronize()
    p.compare(out, p.want())


def test_a_layer_or_page_size_past_32_bits_is_refused(pkg, paged):
    """(ctypes would pass the low 32 bits: layer 0, pages of 16)"""
    import torch
    p = Problem(paged, "bf16", [40, 90], 8, 2, 64, 16, seed=67)
    at = torch.zeros(2, dtype=torch.int32, device="cuda")
    rotary, v = paged.Rotary(64), torch.zeros((2, 2, 64), device="cuda")
    calls = [lambda n: paged.attention_decode(p.cache, n, p.batch, p.qd), lambda n: paged.attention_prefill(p.cache, n, p.batch, p.qd),
             lambda n: paged.qk_norm_rope(rotary, p.qd, v, v, at, cache=p.cache, layer=n, slots=at.long())]
    for call in calls:
        for n in (1 << 32, -1 << 32):
            with pytest.raises(ValueError):
                call(n)
        for n in (1, -1):
            with pytest.raises(pkg.MLQError):
                call(n)
    batch = paged.PagedBatch.empty(2, 4, 8)
    for n in (16 + (1 << 32), 16 - (1 << 32)):
        with pytest.raises(ValueError):
            paged.plan(batch, batch.lengths, at, at, at[:1], n)


def test_prefill_workspace_of_a_batch_that_holds_fewer_rows_than_q(paged):
    """The rows that count are the batch's: few of them share their keys, whatever q is padded to."""
    import torch
    p = Problem(paged, "bf16", [3000, 900], 8, 2, 64, 16, seed=69, new=[5, 3])
    rows = torch.full((8,), -1, dtype=torch.int32, device="cuda")
    p.batch = paged.PagedBatch(p.batch.block_table, p.batch.lengths, p.batch.row_start, rows, rows.long())
    q = torch.cat([p.qd, torch.zeros((9000, 8, 64), device="cuda")])
    bound = p.batch.max_pages * 16
    need = [paged.attention_workspace_bytes(p.cache, 8, 2, bound, rows=n) for n in (p.batch.max_rows, q.shape[0])]
    assert need[0] > need[1] == 0  # (so many rows would fill the chip)
    out = paged.attention_prefill(p.cache, 0, p.batch, q, workspace=torch.empty(need[0], dtype=torch.uint8, device="cuda"))
    torch.cuda.synchronize()
    p.compare(out, p.want())
    assert torch.all(out[p.rows:] == 0.0)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv,hd,lengths,new", [(8, 2, 64, [400, 90], [400, 30]), (6, 2, 128, [700, 90], [650, 30]), (4, 1, 256, [300, 500], [300, 100]),
                                                     (12, 4, 80, [3000, 40], [40, 3]), (4, 2, 128, [2500], [60]),
                                                     (4, 2, 64, [200] + [9] * 300, [200] + [3] * 300)])
def test_prefill_where_values_are_not_finite(paged, heads, kv, hd, lengths, new, kind):
    """A value that overflowed early, a channel of infinite values, a last token of NaN, infinite keys: NaN or infinite where
    they are seen, and the right numbers everywhere else, in one piece and where workgroups share the keys."""
    import torch
    n = lengths[0]
    where = {"early": ("values", [5], 3, math.inf), "late": ("values", [n - 2], 1, -math.inf), "channel": ("values", range(n), 2, math.inf),
             "middle": ("values", [n // 2, n // 2 + 1, n - 20], 7, math.nan), "token": ("values", [n - 1], slice(None), math.nan),
             "key": ("keys", [n - 40], 4, math.nan), "far key": ("keys", [n // 3], slice(None), math.inf)}
    for name, (pool, tokens, dim, value) in where.items():
        p = Problem(paged, kind, lengths, heads, kv, hd, 16, seed=71, new=new)
        t = getattr(p.cache, pool)
        for k in tokens:
            t[0, int(p.table[0, k // 16]), kv - 1, k % 16, dim] = value
        clean_k, clean_v = (np.nan_to_num(x, nan=0, posinf=0, neginf=0) for x in (p.k, p.v))
        p.k, p.v = clean_k, clean_v
        hurt = np.zeros(hd, bool)
        hurt[dim] = True
        if pool == "values":  # (their dims, not the others)
            for k in tokens:
                p.v[0, int(p.table[0, k // 16]), kv - 1, k % 16, hurt] = 0
        for rule in (dict(), dict(window=100, softcap=20.0), dict(window=33)):
            own, plain = rule_of(paged, heads, **rule)
            out = paged.attention_prefill(p.cache, 0, p.batch, p.qd, rule=own)
            torch.cuda.synchronize()
            out = host(out)
            rows = set(range(0, p.rows, max(1, p.rows // 60))) | set(range(max(0, p.start[1] - 44), p.rows)) | set(range(12))
            for r, (y, bound) in p.want(rows=rows, **plain).items():
                pos = n - (p.start[1] - r) if r < p.start[1] else -1
                first = max(0, pos + 1 - rule["window"]) if rule else 0
                sees = any(first <= k <= pos for k in tokens)
                for h in range(heads):
                    whole = sees and h * kv // heads == kv - 1
                    if whole and pool == "keys":
                        assert np.all(np.isnan(out[r, h])) if value != value else True, (name, r, h)
                        continue
                    bad = hurt & whole
                    assert not np.isfinite(out[r, h, bad]).any(), (name, rule, r, h)
                    check(out[r, h, ~bad], y[h, ~bad], bound[h, ~bad], (name, rule, r, h))


@pytest.mark.parametrize("row_start", [False, True])
@pytest.mark.parametrize("n", [4100, 4200])
def test_decode_cut_into_ranges_over_several_launches(paged, n, row_start):
    """A loose bound cuts the sequences, a tight one does not; the second launch has fewer sequences than a wave has lanes
    (4100) or more (4200), in the first one's workspace."""
    import torch
    r = np.random.default_rng(n)
    lengths = r.integers(0, 40, n)
    lengths[[7, 2000, 4090, 4095, 4096, 4098, n - 1]] = [500, 333, 200, 480, 470, 350, 129]
    p = Problem(paged, "bf16", lengths, 4, 2, 64, 16, seed=73, new=(r.random(n) < 0.9).astype(int) if row_start else None, extra_pages=100)
    if not row_start:
        p.batch = paged.PagedBatch(p.batch.block_table, p.batch.lengths)
    loose = p.batch.max_pages * 16
    assert paged.attention_workspace_bytes(p.cache, 4, n, loose) > 0
    assert paged.attention_workspace_bytes(p.cache, 4, n, 500) == 0
    want = p.want(rows=set(range(0, p.rows, 40)) | set(range(p.rows - (n - 4080), p.rows)) |
                  {int(p.start[i]) for i in np.flatnonzero(lengths > 100) if p.new[i]})
    for bound in (loose, 500):
        out = torch.full((p.rows, 4, 64), 9.0, device="cuda")
        paged.attention_decode(p.cache, 0, p.batch, p.qd, out=out, max_len=bound)
        torch.cuda.synchronize()
        p.compare(out, want, bound)
        assert not torch.any(out == 9.0)


@pytest.mark.parametrize("decode", [True, False])
def test_replays_at_once_write_what_the_eager_calls_do(paged, decode):
    """Two batches' calls captured apart and replayed on two streams at once: all of each output, rows that the call leaves
    among it, bit for bit."""
    import torch
    problems = [Problem(paged, "bf16", [4000, 2100, 900, 30], 28, 4, 128, 16, seed=75, new=[1, 3, 2, 0]),
                Problem(paged, "f16", [3000, 5000, 77], 8, 8, 64, 32, seed=77, new=[2, 1, 1])]
    call = paged.attention_decode if decode else paged.attention_prefill
    jobs = []
    for p in problems:
        out = torch.zeros_like(p.qd).contiguous()
        run = lambda p=p, out=out: call(p.cache, 0, p.batch, p.qd, out=out)  # noqa: E731
        run()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            run()
        jobs.append((p, run, out, g, torch.cuda.Stream()))
    for step in range(6):
        want = []
        for p, run, out, g, s in jobs:
            p.batch.lengths.copy_(dev(np.maximum(p.lengths - 13 * step, 0).astype(np.int32)))
            out.fill_(9.0)
            run()
            want.append(out.clone())
            out.fill_(9.0)
        torch.cuda.synchronize()
        for p, run, out, g, s in jobs:
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for w, (p, run, out, g, s) in zip(want, jobs):
            assert torch.equal(out, w), step
            last = sorted({int(b) - 1 for a, b in zip(p.start, p.start[1:]) if b > a}) if decode else list(range(p.rows))
            assert not torch.any(out[last] == 9.0)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size", [1e3, 1e6, 1e10])
def test_a_query_element_far_above_the_others(paged, size, kind):
    """One element of q is huge where every key is 0. The others' scores are right to fp32's last bits, and for an fp16 cache
    to the 2^-39 of the head's largest |q| that an element may be off by: e = 2^-39 max|q| sum|k| scale in a score, which
    moves a weight p by at most 2 e p."""
    import torch
    p = Problem(paged, kind, [1, 70, 300], 8, 4, 64, 16, seed=79, new=[1, 50, 9])
    p.cache.keys[..., 5] = 0
    p.k = host(p.cache.keys)
    p.q[..., 5] = size
    p.qd = dev(p.q)
    keys = np.abs(np.nan_to_num(p.k)).sum(-1).max()
    more = 2 * 2.0 ** -39 * size * keys / 8 * np.abs(p.v[np.isfinite(p.v)]).max() if kind == "f16" else 0.0
    want = {r: (y, bound + more) for r, (y, bound) in p.want().items()}
    out, last = paged.attention_prefill(p.cache, 0, p.batch, p.qd), paged.attention_decode(p.cache, 0, p.batch, p.qd)
    torch.cuda.synchronize()
    p.compare(out, want, size)
    p.compare(last, {int(s) - 1: want[int(s) - 1] for s in p.start[1:]}, size)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("seqs,prompts", [(5, 2), (400, 90), (300, 290)])
def test_decode_for_some_sequences_and_prefill_for_the_others(paged, seqs, prompts, kind):
    """A step of both: views of the batch's arrays are batches of their own, with the whole step's q and out."""
    import torch
    r = np.random.default_rng(seqs)
    ones = seqs - prompts
    lengths = np.concatenate([r.integers(1, 200, ones), r.integers(10, 150, prompts)])
    lengths[0], lengths[ones] = 3000, 700
    new = np.concatenate([np.ones(ones, int), r.integers(1, 10, prompts)])
    new[ones], new[-1] = 650, lengths[-1]
    p = Problem(paged, kind, lengths, 8, 2, 64, 16, seed=81, new=new)
    b = p.batch
    first = paged.PagedBatch(b.block_table[:ones], b.lengths[:ones], b.row_start[:ones + 1])
    rest = paged.PagedBatch(b.block_table[ones:], b.lengths[ones:], b.row_start[ones:])
    out = torch.full((p.rows, 8, 64), 9.0, device="cuda")
    paged.attention_decode(p.cache, 0, first, p.qd, out=out)
    torch.cuda.synchronize()
    assert torch.all(out[ones:] == 9.0) and not torch.any(out[:ones] == 9.0)
    paged.attention_prefill(p.cache, 0, rest, p.qd, out=out)
    torch.cuda.synchronize()
    p.compare(out, p.want(rows=set(range(0, p.rows, max(1, p.rows // 150))) | {ones - 1, ones, p.rows - 1}))
    assert not torch.any(out == 9.0)
