"""GPU: sampling against its definition in 64 bits (tests/sampling_ref.py).
Tokens have to be equal; a row whose token hangs on a border nearer than
2^-38 of the sum (units of 2^-44 for up to 2^19 tokens, half of one each, and
64 bits' own roundings) says nothing and is left out."""
from __future__ import annotations

import numpy as np
import pytest

import sampling_ref as ref

pytestmark = pytest.mark.gpu
NEAR = 2.0 ** -38


@pytest.fixture(scope="module")
def sampling(pkg):
    from mini_llama_amd import sampling
    return sampling


def dev(a, t=None):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a if t is None else np.asarray(a, t))).to("cuda")


def check(sampling, x, u, stride=None, **settings):
    """Rows x [rows, vocab] with a setting for each row or one for all."""
    import torch
    rows, vocab = x.shape
    wide = torch.full((rows, stride or vocab), float("inf"), device="cuda")
    logits = wide[:, :vocab]
    logits.copy_(dev(x))
    full = {k: np.broadcast_to(np.asarray(v), (rows,)) for k, v in settings.items()}
    rule = sampling.Sampling(**{k: dev(v, np.int32 if k == "top_k" else np.float32) for k, v in full.items()})
    u = np.broadcast_to(np.asarray(u, np.float32), (rows,))
    out = torch.full((rows,), -7, dtype=torch.int32, device="cuda")
    sampling.sample(rule, logits, dev(u), out=out)
    got, left = out.cpu().numpy(), 0
    for r in range(rows):
        want, margin = ref.token(x[r], u[r], **{k: v[r] for k, v in full.items()})
        if margin < NEAR:
            left += 1
            continue
        assert got[r] == want, (r, got[r], want, margin, {k: v[r] for k, v in full.items()}, u[r])
    assert left <= 1 + rows // 50
    return got


def settings(r, rows):
    return dict(temperature=np.where(r.random(rows) < 0.1, 0.0, r.uniform(0.2, 2.0, rows)),
                top_k=np.where(r.random(rows) < 0.4, 0, r.integers(1, 300, rows)), top_p=np.where(r.random(rows) < 0.3, 1.0, r.uniform(0.05, 0.999, rows)),
                min_p=np.where(r.random(rows) < 0.5, 0.0, r.uniform(0.0, 0.3, rows)))


@pytest.mark.parametrize("vocab", [1, 2, 3, 63, 64, 65, 200, 1023, 1024, 1025, 4095, 4096, 4097, 5000, 8191, 32000, 50257, 128256, 152064, 1 << 19])
@pytest.mark.parametrize("sharp", [0.3, 2.0, 8.0])
def test_rows_of_their_own_settings(sampling, vocab, sharp):
    r = np.random.default_rng(vocab)
    rows = 40 if vocab < 100000 else 12
    x = (r.standard_normal((rows, vocab)) * sharp).astype(np.float32)
    check(sampling, x, r.random(rows), stride=vocab + 3, **settings(r, rows))


@pytest.mark.parametrize("rows,vocab", [(1, 152064), (3, 40000), (130, 20000), (700, 5000), (1500, 4500), (3000, 700)])
def test_numbers_of_rows(sampling, rows, vocab):
    r = np.random.default_rng(rows)
    x = (r.standard_normal((rows, vocab)) * 3).astype(np.float32)
    check(sampling, x, r.random(rows), **settings(r, rows))


@pytest.mark.parametrize("vocab", [100, 6000, 152064])
@pytest.mark.parametrize("step", [0.0, 1.0, 0.125, 0.01])
def test_equal_logits(sampling, vocab, step):
    """Ties go by index: all equal, a few values, as coarse as 16-bit logits."""
    r = np.random.default_rng(vocab)
    rows = 16
    x = r.standard_normal((rows, vocab)) * 2
    x = (np.round(x / step) * step if step else np.zeros((rows, vocab))).astype(np.float32)
    x[:, ::7] *= -1  # (zeros of both signs are equal)
    check(sampling, x, r.random(rows), **settings(r, rows))
    check(sampling, x, [0.0, 0.25, 0.5, 0.75] * 4, top_p=np.repeat([1.0, 0.5, 0.25, 0.75], 4))


def test_masked_rows(sampling):
    """-inf, NaN, the type's lowest value, +inf; a row that has nothing left."""
    r = np.random.default_rng(4)
    for vocab in (50, 3000, 40000):
        x = (r.standard_normal((24, vocab)) * 2).astype(np.float32)
        x[:4, r.random(vocab) < 0.9] = -np.inf
        x[4:8, r.random(vocab) < 0.9] = np.nan
        x[8:12, r.random(vocab) < 0.9] = np.finfo(np.float32).min
        x[12:14, r.integers(0, vocab, 3)] = np.inf
        x[14] = -np.inf
        x[15] = np.nan
        x[16] = np.finfo(np.float32).min
        x[17] = -np.inf
        x[17, vocab - 1] = -3.0
        x[18] = np.finfo(np.float32).min
        x[18, 7] = np.finfo(np.float32).max
        x[19] = np.inf
        x[20, :] = np.nan
        x[20, [3, vocab // 2]] = -1e30
        got = check(sampling, x, r.random(24), temperature=r.uniform(0.5, 1.5, 24), top_k=r.choice([0, 5, 100], 24), top_p=r.choice([1.0, 0.9], 24))
        assert got[14] == got[15] == -1 and got[17] == vocab - 1
        got = check(sampling, x, 0.3, temperature=0.0)
        assert got[14] == -1 and got[16] == 0 and got[19] == 0


@pytest.mark.parametrize("vocab", [900, 2000, 6000, 40000])
@pytest.mark.parametrize("low", [np.finfo(np.float32).min, -3.1e38, 3.3e38, np.finfo(np.float32).max, 0.0, -1e-45])
def test_equal_logits_at_the_type_s_ends(sampling, vocab, low):
    """A few thousand equal candidates among masked ones, and some neighbours of theirs."""
    r = np.random.default_rng(6)
    x = np.full((12, vocab), -np.inf, np.float32)
    for row in range(12):
        at = r.permutation(vocab)[:r.integers(1, min(vocab, 3500))]
        x[row, at] = low
        if row % 3 == 2:
            x[row, at[:len(at) // 2]] = np.nextafter(np.float32(low), np.float32(0.0 if low else 1.0))
    check(sampling, x, r.random(12), temperature=r.uniform(0.3, 2.0, 12), top_k=r.choice([0, 5, 900, 3000], 12), top_p=r.choice([1.0, 0.9], 12),
          min_p=r.choice([0.0, 0.2], 12))


@pytest.mark.parametrize("vocab", [300, 9000])
def test_settings_at_their_ends(sampling, vocab):
    r = np.random.default_rng(5)
    x = (r.standard_normal((20, vocab)) * 3).astype(np.float32)
    for kw in (dict(temperature=1e-30), dict(temperature=1e-45), dict(temperature=np.inf), dict(temperature=1e30), dict(temperature=-1.0), dict(temperature=np.nan),
               dict(top_k=1), dict(top_k=-5), dict(top_k=vocab), dict(top_k=vocab - 1), dict(top_k=2 ** 31 - 1), dict(top_k=-2 ** 31), dict(top_p=0.0),
               dict(top_p=-1.0), dict(top_p=np.nan), dict(top_p=2.0), dict(top_p=1 - 2.0 ** -24), dict(top_p=1e-30), dict(min_p=1.0), dict(min_p=5.0),
               dict(min_p=np.nan), dict(min_p=-1.0), dict(min_p=1e-30), dict(top_k=50, top_p=0.5, min_p=0.2), dict(top_k=2, top_p=0.999)):
        check(sampling, x, r.random(20), **kw)
    for u in (0.0, -0.5, -np.inf, np.nan, 1 - 2.0 ** -24, 2.0 ** -24, 1e-30):
        check(sampling, x, u, top_k=30)
        check(sampling, x, u)
    for u in (1.0, 2.0, np.inf):  # the last of those that stay
        check(sampling, x, u, top_k=30)
        check(sampling, x, u, top_p=0.9)


def test_logits_of_large_size(sampling):
    """Differences are exact in 64 bits, wherever the logits lie."""
    r = np.random.default_rng(6)
    for vocab in (500, 20000):
        for at, sharp in ((1e6, 2.0), (-3e7, 20.0), (1e30, 1e29), (1e-20, 1e-20)):
            x = (at + r.standard_normal((12, vocab)) * sharp).astype(np.float32)
            check(sampling, x, r.random(12), temperature=max(sharp, 1e-20), top_k=r.choice([0, 40], 12), top_p=r.choice([1.0, 0.8], 12))


def test_distribution(sampling):
    """2^17 draws of one row at evenly spaced u: each token as often as it should be, to one draw."""
    import torch
    x = np.linspace(-2, 2, 40).astype(np.float32)
    n = 1 << 17
    u = dev((np.arange(n) + 0.5) / n, np.float32)
    out = sampling.sample(None, dev(x)[None].expand(n, 40), u).cpu().numpy()
    p = np.exp(x.astype(np.float64)) / np.exp(x.astype(np.float64)).sum()
    assert np.all(np.abs(np.bincount(out, minlength=40) - p * n) <= 1.0)
    assert torch.all(u < 1)


def test_streams_graphs_and_workspaces(pkg, sampling):
    """Another stream, a workspace of the caller's, two captured steps replayed at once while everything changes."""
    import torch
    jobs = []
    for rows, vocab in ((5, 152064), (70, 30000), (300, 900)):
        g = torch.Generator(device="cuda")
        g.manual_seed(rows)
        x, u = torch.empty(rows, vocab, device="cuda"), torch.empty(rows, device="cuda")
        t, k, p, m = torch.ones(rows, device="cuda"), torch.zeros(rows, dtype=torch.int32, device="cuda"), torch.ones(rows, device="cuda"), torch.zeros(rows, device="cuda")

        def fill(x=x, u=u, t=t, k=k, p=p, m=m, g=g):
            x.normal_(generator=g).mul_(2.5)
            u.uniform_(generator=g)
            t.uniform_(0.4, 1.5, generator=g)
            t[::9] = 0
            k.random_(0, 60, generator=g)
            p.uniform_(0.5, 1.1, generator=g)
            m.uniform_(0, 0.1, generator=g)
        fill()
        rule, out = sampling.Sampling(t, k, p, m), torch.zeros(rows, dtype=torch.int32, device="cuda")
        eager = sampling.sample(rule, x, u)
        side = torch.cuda.Stream()
        torch.cuda.synchronize()
        other = sampling.sample(rule, x, u, stream=side)
        need = sampling.sample_workspace_bytes(rows, vocab)
        ws = torch.full((max(need, 1),), 255, dtype=torch.uint8, device="cuda")
        mine = sampling.sample(rule, x, u, workspace=ws)
        torch.cuda.synchronize()
        assert torch.equal(eager, other) and torch.equal(eager, mine)
        if need:
            with pytest.raises(pkg.MLQError):
                sampling.sample(rule, x, u, workspace=ws[:need - 1])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            sampling.sample(rule, x, u, out=out)
        jobs.append((fill, rule, x, u, out, graph, side))
    for _ in range(4):
        want = []
        for fill, rule, x, u, out, graph, side in jobs:
            fill()
            want.append(sampling.sample(rule, x, u))
            out.fill_(-9)
        torch.cuda.synchronize()
        for fill, rule, x, u, out, graph, side in jobs:
            with torch.cuda.stream(side):
                graph.replay()
        torch.cuda.synchronize()
        for w, (fill, rule, x, u, out, graph, side) in zip(want, jobs):
            assert torch.equal(w, out)
            r = int(u.argmax())
            settings_ = {n: float(getattr(rule, n)[r]) for n in ("temperature", "top_p", "min_p")}
            token, margin = ref.token(x[r].cpu().numpy(), float(u[r]), top_k=int(rule.top_k[r]), **settings_)
            assert margin < NEAR or token == int(out[r])


def test_refusals_on_the_device(pkg, sampling):
    import torch
    x, u = torch.zeros(4, 10, device="cuda"), torch.zeros(4, device="cuda")
    for bad in (dict(logits=x.double()), dict(logits=x.t()), dict(logits=x[0]), dict(uniform=u[:3]), dict(uniform=u.double()),
                dict(out=torch.zeros(4, device="cuda")), dict(out=torch.zeros(5, dtype=torch.int32, device="cuda")),
                dict(rule=sampling.Sampling(temperature=torch.ones(3, device="cuda")))):
        with pytest.raises(ValueError):
            sampling.sample(**{**dict(rule=None, logits=x, uniform=u), **bad})
    with pytest.raises(ValueError):
        sampling.Sampling(torch.ones(3, device="cuda"), torch.ones(4, dtype=torch.int32, device="cuda"))
    rule = sampling.Sampling(torch.ones(4, device="cuda"))
    with pytest.raises(AttributeError):
        rule.temperature = u
    assert sampling.sample(None, x[:0], u[:0]).shape == (0,)
    assert sampling.sample(None, x, u).tolist() == [0] * 4


@pytest.mark.parametrize("vocab", [900, 9000, 152064])
@pytest.mark.parametrize("temperature", [np.inf, 1e30, 1e20])
def test_min_p_at_temperatures_that_weigh_all_alike(sampling, vocab, temperature):
    """Every weight is 1 in 64 bits: min_p leaves all tokens up to 1, and the first for more."""
    r = np.random.default_rng(vocab)
    rows = 6
    x = (r.standard_normal((rows, vocab)) * 3).astype(np.float32)
    for least in (1.0, 0.5, 1e-30):
        for kw in (dict(), dict(top_k=[0, 5, 1500, 1024, 1025, 0], top_p=[0.9, 0.9, 1.0, 1.0, 0.5, 1.0])):
            check(sampling, x, r.random(rows), temperature=temperature, min_p=least, **kw)


@pytest.mark.parametrize("rows,vocab", [(177, 900), (3, 9000), (177, 152064), (8, 152064), (600, 152064), (5, 1 << 19)])
@pytest.mark.parametrize("units", [0.4, 0.6, 300.5, 1000.5, 2000.4])
def test_long_tails_of_equal_weights(sampling, rows, vocab, units):
    """One token of weight 1 and all others of a few units of 2^-44, half of one rounded each: sums are off by up to
    vocab 2^-45, and 2^-45 for each of 16 parts' 1024 bins, at the token and in the whole sum, and by 64 bits' roundings.
    What uniform points at lies within that of the token."""
    x = np.full(vocab, np.log(units * 2.0 ** -44), np.float32)
    x[vocab // 3] = 0.0
    w = np.exp(x.astype(np.float64)[0])
    whole = 1.0 + (vocab - 1) * w
    # from the peak's end to the last step of fp32 before 1
    u = np.float32(1.0) - np.float32(2.0 ** -24) * np.arange(1, rows + 1, dtype=np.float32)
    u[::2] = 1.0 - (np.linspace(0.01, 0.99, rows)[::2] * (vocab - 1) * w / whole)
    u = np.minimum(u, np.float32(1 - 2.0 ** -24))
    out = sampling.sample(None, dev(x)[None].expand(rows, vocab), dev(u)).cpu().numpy()
    assert ((out >= 0) & (out < vocab)).all()
    rank = np.where(out == vocab // 3, 0, out + (out < vocab // 3))
    lo, hi = np.where(rank == 0, 0.0, 1.0 + (rank - 1) * w), 1.0 + rank * w
    target = u.astype(np.float64) * whole
    assert (np.maximum(lo - target, target - hi) <= (vocab + 2 ** 14) * 2.0 ** -44 + 2.0 ** -40 * whole).all()


def test_a_workspace_of_the_largest_batch(sampling):
    """One workspace for every batch size of a server, other rows' numbers in it."""
    import torch
    vocab, most = 20000, 257
    ws = torch.full((sampling.sample_workspace_bytes(most, vocab),), 255, dtype=torch.uint8, device="cuda")
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    x, u = torch.randn(most, vocab, device="cuda", generator=g) * 3, torch.rand(most, device="cuda", generator=g)
    k, p = torch.randint(0, 2000, (most,), device="cuda", generator=g).int(), torch.rand(most, device="cuda", generator=g) + 0.3
    for rows in (257, 256, 255, 171, 128, 86, 33, 16, 1, 257):
        rule = sampling.Sampling(top_k=k[:rows].contiguous(), top_p=p[:rows].contiguous())
        for n in (vocab, 17000, 1025, 900):
            got = sampling.sample(rule, x[:rows, :n], u[:rows].contiguous(), workspace=ws)
            assert torch.equal(got, sampling.sample(rule, x[:rows, :n], u[:rows].contiguous())), (rows, n)
