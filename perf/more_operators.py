"""A serving step over a cache of 4 or 8 bits: its operators as cases whose time and results can be measured.

  write      keys and values of new tokens, already rotated, quantised to their slots; the values that the cache then stands for are
             given back: paged.write()
  read       tokens of the cache as the values that they stand for, to move a sequence elsewhere: paged.read()
  decode     attention of one new token of each sequence over its pages: paged.attention_decode()
  prefill    attention of many new tokens of each sequence, causal, over its pages: paged.attention_prefill()
  sample     the step's tokens from its logits with each sequence's temperature, top-k, top-p and min-p: sampling.sample()

Activations are fp32. A head's elements are quantised in blocks of 32: d = (largest - least) / 15 (q8: 255) and m = least + 8 d (128 d) in fp16, an
element the nearest d (c - 8) + m (d (c - 128) + m). A head takes up a row of 2, 4 or 8 blocks (head dims up to 64, 128, 256): unit 16 i of
them, i * blocks + b, holds dims 2 i and 2 i + 1 of block b (q4: a byte, the lower dim in its low half; q8: two bytes), then come d and m of every
block. Keys are N(0, 1) with channels of different sizes, as rotated keys have them, values N(0, 1); pages lie in the pool in random order. Heads
and head dims are those of the 7B- and 8B-class shapes that the benchmark and the tests use, the largest vocabulary the benchmark's.
"""
import importlib
import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
#: levels, middle, bytes of a unit of two elements
KINDS = {"q4": (15, 8, 1), "q8": (255, 128, 2)}
#: query heads, kv heads, head dim
SHAPES = [(28, 4, 128), (32, 8, 128), (64, 8, 128), (32, 32, 128), (24, 2, 128), (16, 16, 64), (40, 8, 64), (16, 1, 256), (12, 4, 80)]
VOCAB = 152064


def listed():
    return [
        # One new token for each of 48 users of a 7B shape: launch latency is all of it.
        {"name": "write_48_7b", "kind": "write", "type": "q4", "rows": 48, "kv_heads": 4, "hd": 128, "page": 16},
        # A full prefill batch of an 8B shape.
        {"name": "write_8000_8b", "kind": "write", "type": "q4", "rows": 8000, "kv_heads": 8, "hd": 128, "page": 64},
        # One conversation of a model with small heads taken out of the cache.
        {"name": "read_901_small", "kind": "read", "type": "q8", "rows": 901, "kv_heads": 16, "hd": 64, "page": 16},
        # A shared document's pages read back to be kept elsewhere.
        {"name": "read_16000_8b", "kind": "read", "type": "q4", "rows": 16000, "kv_heads": 8, "hd": 128, "page": 64},
        # A single user early in a conversation: the smallest call.
        {"name": "decode_1x700_7b", "kind": "decode", "type": "q4", "seqs": 1, "longest": 700, "spread": False, "heads": 28, "kv_heads": 4, "hd": 128,
         "page": 16, "softcap": 0.0, "window": 0, "slopes": False},
        # 64 users at all stages of their conversations on a 7B shape.
        {"name": "decode_64x8000_7b", "kind": "decode", "type": "q4", "seqs": 64, "longest": 8000, "spread": True, "heads": 28, "kv_heads": 4, "hd": 128,
         "page": 64, "softcap": 0.0, "window": 0, "slopes": False},
        # Users with whole books in their contexts, scores capped.
        {"name": "decode_8x100000_8b", "kind": "decode", "type": "q4", "seqs": 8, "longest": 100000, "spread": False, "heads": 32, "kv_heads": 8, "hd": 128,
         "page": 128, "softcap": 50.0, "window": 0, "slopes": False},
        # Many users of a small model in 8 bits, a kv head for each head, a sliding window and biases by distance.
        {"name": "decode_180x2500_window", "kind": "decode", "type": "q8", "seqs": 180, "longest": 2500, "spread": True, "heads": 16, "kv_heads": 16, "hd": 64,
         "page": 16, "softcap": 0.0, "window": 1000, "slopes": True},
        # Three prompts of odd lengths, the last one long, on a 7B shape in 8 bits.
        {"name": "prefill_3_7b", "kind": "prefill", "type": "q8", "seqs": 3, "rows": 700, "context": 100, "heads": 28, "kv_heads": 4, "hd": 128,
         "page": 16, "softcap": 0.0, "window": 0, "slopes": False},
        # A full prefill batch of an 8B shape: pieces of six prompts behind what is cached of them.
        {"name": "prefill_6_8b", "kind": "prefill", "type": "q4", "seqs": 6, "rows": 8000, "context": 2000, "heads": 32, "kv_heads": 8, "hd": 128,
         "page": 64, "softcap": 0.0, "window": 0, "slopes": False},
        # A single user's next token from the benchmark's vocabulary.
        {"name": "sample_1", "kind": "sample", "rows": 1, "vocab": VOCAB, "sharp": 2.0, "coarse": False},
        # 64 users, each with settings of their own, some of them greedy.
        {"name": "sample_64", "kind": "sample", "rows": 64, "vocab": VOCAB, "sharp": 2.5, "coarse": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["write", "read", "decode", "decode", "prefill", "prefill", "sample", "sample"])
    if kind == "sample":
        rows = _log(rng, 1, 400)
        # (logits of a head that multiplies in 16 bits are coarse: many of them are equal)
        return {"kind": kind, "rows": rows, "vocab": min(_log(rng, 300, VOCAB), 64 * VOCAB // rows), "sharp": round(rng.uniform(0.5, 4.0), 2),
                "coarse": rng.random() < 0.3}
    page = rng.choice([16, 32, 64, 128])
    heads, kv_heads, hd = rng.choice(SHAPES)
    case = {"kind": kind, "type": rng.choice(["q4", "q4", "q8"])}
    if kind in ("write", "read"):
        most = 8000 if kind == "write" else 16000
        return dict(case, rows=min(_log(rng, 1, most), most * 8 * 128 // (kv_heads * hd)), kv_heads=kv_heads, hd=hd, page=page)
    rule = {"heads": heads, "kv_heads": kv_heads, "hd": hd, "page": page, "softcap": rng.choice([0.0, 0.0, 30.0, 50.0]),
            "window": rng.choice([0, 0, 0, rng.randint(1, 2900)]), "slopes": rng.random() < 0.25}
    if kind == "decode":
        while True:
            seqs, longest = _log(rng, 1, 200), _log(rng, 1, 100000)
            # (the plain form holds every sequence, padded to the longest, in 32 bits)
            if seqs * longest * kv_heads * hd <= 4 * 100000 * 8 * 128:
                return dict(case, seqs=seqs, longest=longest, spread=rng.random() < 0.6, **rule)
    while True:
        seqs, rows, context = _log(rng, 1, 24), _log(rng, 24, 8000), rng.choice([0, 0, _log(rng, 10, 4000)])
        if rows * (1 + context + 2 * rows // seqs) * heads * hd <= 8000 * 4700 * 32 * 128 and \
           seqs * (2 * rows // seqs + 1) * (context + 2 * rows // seqs + 1) * heads <= 3 * 10**9:
            return dict(case, seqs=seqs, rows=rows, context=context, **rule)


# ---- the cache of 4 or 8 bits -----------------------------------------------------------------------------------------------------


def _blocks(hd):
    return 2 if hd <= 64 else 4 if hd <= 128 else 8


def _row_bytes(case):
    return _blocks(case["hd"]) * (16 * KINDS[case["type"]][2] + 4)


def _quantised(x, kind):
    """(row bytes, the values that they stand for) of heads x [..., hd] in 32 bits."""
    levels, middle, unit = KINDS[kind]
    hd, nb = x.shape[-1], _blocks(x.shape[-1])
    lead = x.shape[:-1]
    real = (torch.arange(32 * nb, device=x.device) < hd).view(nb, 32)
    x = torch.nn.functional.pad(x, (0, 32 * nb - hd)).view(*lead, nb, 32)
    any_real = real.any(-1)
    lo = torch.where(any_real, torch.where(real, x, math.inf).amin(-1), 0.0)
    hi = torch.where(any_real, torch.where(real, x, -math.inf).amax(-1), 0.0)
    # (a tensor of divisors: a number would be turned into its reciprocal)
    d = ((hi - lo) / torch.full_like(lo, levels)).half()
    m = (lo + middle * d.float()).half()
    d64, m64 = d.double()[..., None], m.double()[..., None]
    # (in 64 bits: the border between two codes is often as near as 32 bits round)
    c = torch.floor((x.double() - m64) / torch.where(d64 == 0, 1.0, d64) + 0.5) + middle
    c = torch.where((d64 == 0) | ~real, float(middle), c.clamp(0, levels)).to(torch.uint8)
    values = (d64 * (c.double() - middle) + m64).float().view(*lead, -1)[..., :hd]
    pairs = c.view(*lead, nb, 16, 2).transpose(-3, -2)
    codes = (pairs[..., 0] | (pairs[..., 1] << 4)) if unit == 1 else pairs
    scales = torch.stack([d, m], -1).contiguous().view(torch.uint8)
    return torch.cat([codes.reshape(*lead, -1), scales.reshape(*lead, -1)], -1), values


def _values(rows, kind, hd):
    """The values [..., hd] in 32 bits that row bytes stand for."""
    levels, middle, unit = KINDS[kind]
    nb = _blocks(hd)
    codes, scales = rows[..., :16 * nb * unit], rows[..., 16 * nb * unit:].contiguous().view(torch.float16).float()
    lead = rows.shape[:-1]
    pairs = torch.stack([codes & 15, codes >> 4], -1) if unit == 1 else codes
    c = pairs.reshape(*lead, 16, nb, 2).transpose(-3, -2).reshape(*lead, nb, 32).float() - middle
    scales = scales.view(*lead, nb, 2)
    return (scales[..., :1] * c + scales[..., 1:]).view(*lead, -1)[..., :hd]


# ---- inputs -------------------------------------------------------------------------------------------------------------------


def _lengths(case):
    """Cached lengths after the step and counts of new rows of an attention case, the same for every seed."""
    r = np.random.default_rng(case["seqs"] * 1000003 + case["hd"])
    n = case["seqs"]
    if case["kind"] == "decode":
        longest = case["longest"]
        lengths = np.exp(r.uniform(math.log(max(1, longest / 50)), math.log(longest), n)) if case["spread"] else r.uniform(0.9 * longest, longest, n)
        lengths = np.clip(np.rint(lengths).astype(np.int64), 1, longest)
        lengths[r.integers(n)] = longest
        return lengths, np.ones(n, np.int64)
    share = r.uniform(0.2, 2.0, n)
    share = np.minimum(share / share.sum(), 2.0 / n)
    rows = np.maximum(1, (share * case["rows"]).astype(np.int64))
    return rows + r.integers(0, case["context"] + 1, n), rows


def _starts(counts):
    return np.concatenate([[0], np.cumsum(counts)])


def _pages(case):
    return (_lengths(case)[0] + case["page"] - 1) // case["page"]


def _randn(g, *shape):
    return torch.randn(*shape, device=DEVICE, generator=g)


def _channels(g, kv, hd):
    return torch.exp(0.5 * _randn(g, kv, 1, hd))


def _pool(g, case, n_pages, sizes):
    """A layer's pages of quantised N(0, 1) times `sizes`."""
    kv, page = case["kv_heads"], case["page"]
    pool = torch.empty(1, n_pages, kv, page, _row_bytes(case), dtype=torch.uint8, device=DEVICE)
    step = max(1, (1 << 25) // (kv * page * case["hd"]))
    for p in range(0, n_pages, step):
        n = min(step, n_pages - p)
        pool[0, p:p + n] = _quantised(_randn(g, n, kv, page, case["hd"]) * sizes, case["type"])[0]
    return pool


def _prepare_sample(case, g):
    rows, vocab = case["rows"], case["vocab"]
    logits = _randn(g, rows, vocab) * case["sharp"]
    # a few dozen tokens stand out, as they do where a text goes on
    out = torch.randint(0, vocab, (rows, 24), device=DEVICE, generator=g)
    logits.scatter_add_(1, out, torch.rand(rows, 24, device=DEVICE, generator=g) * 4 * case["sharp"])
    if case["coarse"]:
        logits = logits.bfloat16().float()
    r = torch.rand(6, rows, device=DEVICE, generator=g)
    return {"case": case, "logits": logits, "uniform": torch.rand(rows, device=DEVICE, generator=g),
            "temperature": torch.where(r[0] < 0.1, 0.0, 0.3 + 1.2 * r[1]),
            "top_k": torch.where(r[2] < 0.4, 0, 1 + (200 * r[2] * r[2]).int()).int(),
            "top_p": torch.where(r[3] < 0.3, 1.0, 0.5 + 0.49 * r[3]),
            "min_p": torch.where(r[4] < 0.5, 0.0, 0.1 * r[5]), "tokens": torch.zeros(rows, dtype=torch.int32, device=DEVICE)}


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(int(seed) * 7919 + 29)
    if case["kind"] == "sample":
        return _prepare_sample(case, g)
    ints = dict(dtype=torch.int32, device=DEVICE)
    s = {"case": case}
    kv, hd, page = case["kv_heads"], case["hd"], case["page"]
    sizes = _channels(g, kv, hd)
    if case["kind"] in ("write", "read"):
        rows = case["rows"]
        n_pages = (rows + page - 1) // page + 2
        s["slots"] = torch.randperm(n_pages * page, device=DEVICE, generator=g)[:rows].contiguous()
        s["k_out"], s["v_out"] = (torch.zeros(rows, kv, hd, device=DEVICE) for _ in range(2))
        if case["kind"] == "write":
            kv_rows = _randn(g, rows, 2 * kv * hd)
            s["k"] = kv_rows[:, :kv * hd].view(rows, kv, hd)
            s["v"] = kv_rows[:, kv * hd:].view(rows, kv, hd)
            s["k"].mul_(sizes[:, 0])
            s["keys"], s["values"] = (torch.zeros(1, n_pages, kv, page, _row_bytes(case), dtype=torch.uint8, device=DEVICE) for _ in range(2))
            return s
        s["keys"], s["values"] = _pool(g, case, n_pages, sizes), _pool(g, case, n_pages, 1.0)
        return s
    heads = case["heads"]
    lengths, new = _lengths(case)
    pages = _pages(case)
    n_pages = int(pages.sum()) + 3
    order = torch.randperm(n_pages, device=DEVICE, generator=g).to(torch.int32)
    table = torch.full((case["seqs"], int(pages.max())), -1, **ints)
    table[torch.arange(int(pages.max()), device=DEVICE)[None] < torch.from_numpy(pages).to(DEVICE)[:, None]] = order[:int(pages.sum())]
    qkv = _randn(g, int(new.sum()), (heads + 2 * kv) * hd)
    s.update(keys=_pool(g, case, n_pages, sizes), values=_pool(g, case, n_pages, 1.0),
             block_table=table, lengths=torch.from_numpy(lengths).to(**ints), row_start=torch.from_numpy(_starts(new)).to(**ints),
             q=qkv[:, :heads * hd].view(-1, heads, hd), out=torch.zeros(int(new.sum()), heads, hd, device=DEVICE),
             # (what the program knows of its batch without asking the device)
             max_len=int(pages.max()) * page, max_new=int(new.max()),
             slopes=torch.tensor([2.0 ** (-8.0 * (i + 1) / heads) for i in range(heads)], device=DEVICE) if case["slopes"] else None)
    return s


# ---- the plain forms ------------------------------------------------------------------------------------------------------------


def _plain_write(s):
    page = s["case"]["page"]
    at = (s["slots"] // page, s["slots"] % page)
    for x, out, pool in (("k", "k_out", "keys"), ("v", "v_out", "values")):
        rows, values = _quantised(s[x], s["case"]["type"])
        s[pool][0][at[0], :, at[1]] = rows
        s[out].copy_(values)


def _plain_read(s):
    page = s["case"]["page"]
    at = (s["slots"] // page, s["slots"] % page)
    for out, pool in (("k_out", "keys"), ("v_out", "values")):
        s[out].copy_(_values(s[pool][0][at[0], :, at[1]], s["case"]["type"], s["case"]["hd"]))


def _plain_cached(s, pool):
    """[seqs, kv heads, longest, hd] in 32 bits: every sequence's pages, padded to the longest."""
    table = s["block_table"].long().clamp(min=0)
    x = _values(pool[0][table], s["case"]["type"], s["case"]["hd"])  # [seqs, pages, kv, page, hd]
    return x.permute(0, 2, 1, 3, 4).reshape(table.shape[0], pool.shape[2], -1, x.shape[-1])


def _plain_attention(s, q, qpos):
    """q [seqs, n, heads, hd] at positions qpos [seqs, n] (negative: no row) over the cache."""
    case = s["case"]
    seqs, n, heads, hd = q.shape
    kv = case["kv_heads"]
    k, v = _plain_cached(s, s["keys"]), _plain_cached(s, s["values"])
    t = torch.arange(k.shape[2], device=q.device)
    seen = t <= qpos[..., None]                                            # [seqs, n, t]
    if case["window"]:
        seen &= t > qpos[..., None] - case["window"]
    v = torch.where((t < s["lengths"][:, None])[:, None, :, None], v, 0.0)  # (whatever lies behind a sequence's end)
    q = q.reshape(seqs, n, kv, heads // kv, hd).permute(0, 2, 3, 1, 4).reshape(seqs, kv, -1, hd)
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()).view(seqs, heads, n, -1) / math.sqrt(hd)
    if case["softcap"]:
        scores = case["softcap"] * torch.tanh(scores / case["softcap"])
    if s["slopes"] is not None:
        scores = scores + s["slopes"][None, :, None, None] * (t - qpos[..., None]).float()[:, None]
    scores = scores.masked_fill_(~seen[:, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=-1e30)
    p = torch.exp(scores - top)
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
    out = torch.matmul(p.view(seqs, kv, -1, p.shape[-1]), v)
    return out.view(seqs, heads, n, hd).permute(0, 2, 1, 3)


def _plain_decode(s):
    s["out"].copy_(_plain_attention(s, s["q"][:, None], s["lengths"].long()[:, None] - 1)[:, 0])


def _plain_prefill(s):
    start = s["row_start"].long()
    new = start[1:] - start[:-1]
    n = torch.arange(s["max_new"], device=s["q"].device)
    live = n < new[:, None]
    row = (start[:-1, None] + n).clamp(max=s["q"].shape[0] - 1)
    qpos = torch.where(live, s["lengths"].long()[:, None] - new[:, None] + n, -1)
    out = _plain_attention(s, s["q"][row], qpos)
    whole = torch.cat([s["out"], s["out"][:1]])  # (padding rows go to a row behind the others)
    whole[torch.where(live, row, s["out"].shape[0])] = out
    s["out"].copy_(whole[:-1])


def _plain_sample(s):
    # (weights and their running sums in 64 bits: the token hangs on which of two near numbers is larger)
    logits, order = torch.sort(s["logits"].double(), dim=-1, descending=True, stable=True)
    rank = torch.arange(logits.shape[1], device=logits.device)
    t = s["temperature"].double()[:, None]
    w = torch.exp((logits - logits[:, :1]) / torch.where(t > 0, t, 1.0))
    k = torch.where(t > 0, torch.where(s["top_k"] > 0, s["top_k"], logits.shape[1])[:, None], 1)
    w = torch.where(rank < k, w, 0.0)
    sums = w.cumsum(-1)
    p, least = s["top_p"].double()[:, None], s["min_p"].double()[:, None]
    n = torch.where(p < 1, (sums < p * sums[:, -1:]).sum(-1, keepdim=True) + 1, logits.shape[1])
    n = torch.minimum(torch.minimum(n, k), (w >= least).sum(-1, keepdim=True)).clamp(min=1)
    kept = sums.gather(1, n - 1)
    at = torch.minimum((sums <= s["uniform"].double()[:, None] * kept).sum(-1, keepdim=True), n - 1)
    s["tokens"].copy_(order.gather(1, at)[:, 0])


# ---- one pass ---------------------------------------------------------------------------------------------------------------------


def _handles(s):
    """What a program makes once of its buffers: the cache, the batch and the rule of the attention or the sampling."""
    if "module" not in s:
        case = s["case"]
        if case["kind"] == "sample":
            s["module"] = m = importlib.import_module("mini-llama_amd.sampling")
            s["rule"] = m.Sampling(temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
            return m
        s["module"] = m = importlib.import_module("mini-llama_amd.paged")
        s["cache"] = m.PagedCache(s["keys"], s["values"], quant=case["type"], head_dim=case["hd"])
        if "block_table" in s:
            s["batch"] = m.PagedBatch(s["block_table"], s["lengths"], s["row_start"])
            s["rule"] = m.AttentionRule(softcap=case["softcap"], window=case["window"], slopes=s["slopes"])
    return s["module"]


PLAIN = {"write": _plain_write, "read": _plain_read, "decode": _plain_decode, "prefill": _plain_prefill, "sample": _plain_sample}
OUTPUTS = {"write": ("k_out", "v_out", "keys", "values"), "read": ("k_out", "v_out"), "decode": ("out",), "prefill": ("out",), "sample": ("tokens",)}


def run(s):
    kind = s["case"]["kind"]
    if own:
        m = _handles(s)
        if kind == "write":
            m.write(s["cache"], 0, s["k"], s["v"], s["slots"], k_out=s["k_out"], v_out=s["v_out"])
        elif kind == "read":
            m.read(s["cache"], 0, s["slots"], k_out=s["k_out"], v_out=s["v_out"])
        elif kind == "decode":
            m.attention_decode(s["cache"], 0, s["batch"], s["q"], out=s["out"], rule=s["rule"], max_len=s["max_len"])
        elif kind == "prefill":
            m.attention_prefill(s["cache"], 0, s["batch"], s["q"], out=s["out"], rule=s["rule"])
        else:
            m.sample(s["rule"], s["logits"], s["uniform"], out=s["tokens"])
    else:
        PLAIN[kind](s)
    return {k: s[k] for k in OUTPUTS[kind]}


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------------------


def _seen(case):
    """For each sequence: how many keys some row sees, and how many (row, key) pairs there are."""
    lengths, new = _lengths(case)
    w = case["window"] or 10**9
    keys = np.minimum(lengths, new + w - 1)
    first, last = lengths - new + 1, lengths  # keys that the first and the last row would see without a window
    a, b = np.minimum(first, w), np.minimum(last, w)
    short = np.maximum(b - a + 1, 0)  # rows whose view still grows
    pairs = np.where(first >= w, new * w, (a + b) * short // 2 + (new - short) * w)
    return int(keys.sum()), int(pairs.sum())


def work(case):
    if case["kind"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * 4 + case["rows"] * 24, "flops": n * 4}
    kv, hd = case["kv_heads"], case["hd"]
    # (what the blocks in use hold: a row may be wider)
    row = (hd + 31) // 32 * (16 * KINDS[case["type"]][2] + 4)
    if case["kind"] in ("write", "read"):
        rows = case["rows"] * kv * 2
        return {"bytes": rows * (row + hd * (8 if case["kind"] == "write" else 4)) + case["rows"] * 8, "flops": rows * hd * (6 if case["kind"] == "write" else 2)}
    keys, pairs = _seen(case)
    rows = int(_lengths(case)[1].sum())
    return {"bytes": keys * kv * 2 * row + rows * case["heads"] * hd * 8 + int(_pages(case).sum()) * 4, "flops": pairs * case["heads"] * 4 * hd}


# ---- the definition in 64 bits ----------------------------------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "sample":
        return {"tokens": _exact_sample(s)}
    if case["kind"] == "write":
        return _exact_write(s)
    if case["kind"] == "read":
        page = case["page"]
        return {out: _exact_values(s[pool][0].permute(0, 2, 1, 3).flatten(0, 1)[s["slots"]], case) for out, pool in (("k_out", "keys"), ("v_out", "values"))}
    return {"out": _exact_attention(s)}


def _exact_values(rows, case):
    """Row bytes [..., bytes] as values in 64 bits, a block at a time."""
    levels, middle, unit = KINDS[case["type"]]
    nb = _blocks(case["hd"])
    out = torch.zeros(*rows.shape[:-1], 32 * nb, dtype=torch.float64, device=rows.device)
    for b in range(nb):
        at = 16 * nb * unit + 4 * b
        d, m = (rows[..., at + i:at + i + 2].contiguous().view(torch.float16).double() for i in (0, 2))
        for i in range(16):
            first = rows[..., (i * nb + b) * unit].long()
            pair = (first % 16, first // 16) if unit == 1 else (first, rows[..., (i * nb + b) * unit + 1].long())
            for j in range(2):
                out[..., 32 * b + 2 * i + j] = d[..., 0] * (pair[j] - middle) + m[..., 0]
    return out[..., :case["hd"]]


def _exact_write(s):
    case = s["case"]
    levels, middle, unit = KINDS[case["type"]]
    hd, page, nb = case["hd"], case["page"], _blocks(case["hd"])
    slots = s["slots"].cpu().numpy()
    found = {}
    for x, out, pool in (("k", "k_out", "keys"), ("v", "v_out", "values")):
        a = s[x].cpu().numpy()
        bytes_ = np.zeros(a.shape[:2] + (_row_bytes(case),), np.uint8)
        values = np.zeros(a.shape)
        for b in range(nb):
            block = a[..., 32 * b:32 * b + 32]
            codes = np.full(a.shape[:2] + (32,), middle, np.uint8)
            n = block.shape[-1]
            if n:
                # (d and m are by definition quotient and sum in 32 bits, each rounded to 16)
                lo, hi = block.min(-1), block.max(-1)
                d = ((hi - lo) / np.float32(levels)).astype(np.float16)
                m = (lo + np.float32(middle) * d.astype(np.float32)).astype(np.float16)
                d64, m64 = d.astype(np.float64)[..., None], m.astype(np.float64)[..., None]
                with np.errstate(divide="ignore", invalid="ignore"):
                    c = np.where(d64 > 0, np.clip(np.floor((block - m64) / d64 + 0.5) + middle, 0, levels), middle)
                values[..., 32 * b:32 * b + 32] = d64 * (c - middle) + m64
                codes[..., :n] = c
                at = 16 * nb * unit + 4 * b
                bytes_[..., at:at + 2] = d[..., None].view(np.uint8)
                bytes_[..., at + 2:at + 4] = m[..., None].view(np.uint8)
            for i in range(16):
                at = (i * nb + b) * unit
                if unit == 1:
                    bytes_[..., at] = codes[..., 2 * i] | codes[..., 2 * i + 1] << 4
                else:
                    bytes_[..., at], bytes_[..., at + 1] = codes[..., 2 * i], codes[..., 2 * i + 1]
        whole = s[pool].cpu().numpy().copy()
        whole[0, slots // page, :, slots % page] = bytes_
        found.update({out: values, pool: whole})
    return found


def _exact_attention(s):
    case = s["case"]
    start, lengths = s["row_start"].tolist(), s["lengths"].tolist()
    heads, kv, hd, page = case["heads"], case["kv_heads"], case["hd"], case["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    for i, n in enumerate(lengths):
        ids = s["block_table"][i, :-(-n // page)].long()
        k, v = (_exact_values(s[x][0][ids], case).permute(1, 0, 2, 3).reshape(kv, -1, hd)[:, :n] for x in ("keys", "values"))
        t = torch.arange(n, device=DEVICE)
        for r0 in range(start[i], start[i + 1], 512):  # (512 rows at a time keep the scores small)
            r1 = min(r0 + 512, start[i + 1])
            pos = n - start[i + 1] + torch.arange(r0, r1, device=DEVICE)
            away = pos[:, None] - t
            hidden = away < 0
            if case["window"]:
                hidden |= away >= case["window"]
            for h in range(heads):
                x = s["q"][r0:r1, h].double() @ k[h * kv // heads].T * hd ** -0.5
                if case["softcap"]:
                    x = torch.tanh(x / case["softcap"]) * case["softcap"]
                if s["slopes"] is not None:
                    x = x - s["slopes"][h].double() * away
                out[r0:r1, h] = torch.softmax(x.masked_fill(hidden, -math.inf), -1) @ v[h * kv // heads]
    return out


def _exact_sample(s):
    logits = s["logits"].cpu().numpy().astype(np.float64)
    tokens = np.zeros(len(logits), np.int32)
    given = {k: s[k].cpu().numpy() for k in ("temperature", "top_k", "top_p", "min_p", "uniform")}
    for r, x in enumerate(logits):
        t, k, p, least, u = (float(given[n][r]) for n in ("temperature", "top_k", "top_p", "min_p", "uniform"))
        order = np.lexsort((np.arange(len(x)), -x))
        if not t > 0:
            tokens[r] = order[0]
            continue
        if k > 0:
            order = order[:int(k)]
        w = np.exp((x[order] - x[order[0]]) / t)
        if p < 1:
            enough = np.flatnonzero(np.cumsum(w) >= p * w.sum())
            w = w[:enough[0] + 1] if len(enough) else w
        w = w[:max(1, int((w >= least).sum()))]
        past = np.flatnonzero(np.cumsum(w) > u * w.sum())
        tokens[r] = order[past[0] if len(past) else len(w) - 1]
    return tokens
