"""GPU: a serving loop of all its operators together, from qkv to the next
tokens: plan, rotated keys quantised into a paged cache, attention, logits,
sampling, the tokens fed back; eagerly and replayed from a graph."""
from __future__ import annotations

import numpy as np
import pytest

import kv_quant_ref as kvq
import sampling_ref

pytestmark = pytest.mark.gpu

HEADS, KV, HD, PAGE, SEQS, LAYERS = 8, 2, 64, 16, 6, 2


class Server:
    """A small model of random weights: an embedding that gives each layer's qkv, two attention layers, a head."""

    def __init__(self, pkg, kind, vocab, most):
        import torch
        from mini_llama_amd import paged, sampling
        self.torch, self.paged, self.sampling = torch, paged, sampling
        g = torch.Generator(device="cuda").manual_seed(11)
        rand = lambda *s: torch.randn(*s, generator=g, device="cuda")
        self.embed = rand(vocab, LAYERS, (HEADS + 2 * KV) * HD)
        self.mix = rand(HEADS * HD, (HEADS + 2 * KV) * HD) * 0.2
        self.head = rand(HEADS * HD, vocab) * 0.3
        self.cache = paged.PagedCache.empty(LAYERS, 80, PAGE, KV, HD, kind)
        self.cache.keys.fill_(255)
        self.cache.values.fill_(255)
        self.batch = paged.PagedBatch.empty(SEQS, 16, most)
        i32 = dict(dtype=torch.int32, device="cuda")
        self.free = torch.randperm(80, generator=g, device="cuda").int()
        self.n_free, self.n_new = torch.full((1,), 80, **i32), torch.zeros(SEQS, **i32)
        self.rotary = paged.Rotary(HD, torch.from_numpy(np.asarray(paged.rope_frequencies(1e4, HD // 2)[0])).cuda())
        self.tokens, self.last = torch.zeros(most, **i32), torch.zeros(SEQS, dtype=torch.int64, device="cuda")
        self.next = torch.zeros(SEQS, **i32)
        self.uniform = torch.zeros(SEQS, device="cuda")
        self.rule = sampling.Sampling(temperature=torch.tensor([0.0, 0.7, 1.0, 1.3, 0.9, 1.0], device="cuda"),
                                      top_k=torch.tensor([0, 40, 0, 7, 0, 1], **i32),
                                      top_p=torch.tensor([1.0, 0.9, 0.95, 1.0, 1.0, 0.5], device="cuda"),
                                      min_p=torch.tensor([0.0, 0.0, 0.0, 0.02, 0.1, 0.0], device="cuda"))
        self.work = torch.empty(max(1, sampling.sample_workspace_bytes(SEQS, vocab)), dtype=torch.uint8, device="cuda")
        self.rows = {}

    def launch(self, rows, decode):
        torch, paged = self.torch, self.paged
        paged.plan(self.batch, self.batch.lengths, self.n_new, self.free, self.n_free, PAGE)
        x = self.embed.index_select(0, self.tokens[:rows])
        out = None
        for layer in range(LAYERS):
            qkv = x[:, layer] if out is None else x[:, layer] + out.view(rows, -1) @ self.mix
            q, k, v = (t.view(rows, -1, HD) for t in qkv.split([HEADS * HD, KV * HD, KV * HD], 1))
            q_out, _ = paged.qk_norm_rope(self.rotary, q, k, v, self.batch.positions, q_out=torch.empty(rows, HEADS, HD, device="cuda"),
                                          cache=self.cache, slots=self.batch.slots, layer=layer)
            attend = paged.attention_decode if decode else paged.attention_prefill
            out = attend(self.cache, layer, self.batch, q_out)
        # (the last row of each sequence; an idle one has another's)
        torch.sub(self.batch.row_start[1:], 1, out=self.last)
        hidden = out.view(rows, -1).index_select(0, self.last.clamp_(min=0))
        logits = hidden @ self.head
        self.sampling.sample(self.rule, logits, self.uniform, out=self.next, workspace=self.work)
        self.rows = dict(q=q_out, out=out, logits=logits)


@pytest.mark.parametrize("kind", ["q4", "q8"])
@pytest.mark.parametrize("vocab", [700, 9001])
def test_serving(pkg, kind, vocab):
    import torch
    r = np.random.default_rng(5)
    prompts = [r.integers(0, vocab, n) for n in (1, 20, 77, 16, 130, 33)]
    steps, most = 12, sum(map(len, prompts))
    uniform = r.random((steps, SEQS)).astype(np.float32)
    ends = {5: 2}  # (a sequence that ends at a step, and stays away)
    seen = []
    for graph in (False, True):
        s = Server(pkg, kind, vocab, most)
        captured, kept, alive, said = None, None, np.ones(SEQS, bool), []
        for step in range(steps):
            s.uniform.copy_(torch.from_numpy(uniform[step]))
            if step == 0:
                rows = most
                s.tokens[:rows] = torch.from_numpy(np.concatenate(prompts)).int()
                new = np.array([len(p) for p in prompts], np.int32)
            else:
                rows, new = SEQS, np.where(alive, 1, 0).astype(np.int32)
                if step in ends:
                    new[ends[step]], alive[ends[step]] = -1, False
                # rows go to the sequences that have one, in order
                given = torch.from_numpy(np.flatnonzero(new == 1)).cuda()
                s.tokens[:len(given)] = s.next[given]
            s.n_new.copy_(torch.from_numpy(new))
            if step and graph:
                if captured is None:
                    captured = torch.cuda.CUDAGraph()
                    torch.cuda.synchronize()
                    with torch.cuda.graph(captured):
                        s.launch(SEQS, True)
                    kept = s.rows
                captured.replay()
                torch.zeros(1000, device="cuda").sum().item()
                s.rows = kept
            else:
                s.launch(rows, step > 0)
            torch.cuda.synchronize()
            assert int(s.batch.status.item()) == 0
            live = alive.copy()
            tokens = s.next.cpu().numpy()
            said.append(np.where(live, tokens, -1))
            if graph:
                continue
            logits, q, out = (s.rows[n].cpu().numpy() for n in ("logits", "q", "out"))
            assert np.isfinite(logits).all()
            for i in np.flatnonzero(live):
                want, margin = sampling_ref.token(logits[i], uniform[step, i], *(float(t[i]) if j != 1 else int(t[i]) for j, t in enumerate(
                    (s.rule.temperature, s.rule.top_k, s.rule.top_p, s.rule.min_p))))
                # (sums of 2^19 weights at most, each off by half a unit of 2^-44 and by a double's roundings)
                assert margin < 2.0 ** -34 or tokens[i] == want, (step, i)
            # the last layer's attention against its cache
            start, lengths = s.batch.row_start.cpu().numpy(), s.batch.lengths.cpu().numpy()
            table, keys, vals = (t.cpu().numpy() for t in (s.batch.block_table, s.cache.keys[-1], s.cache.values[-1]))
            for i in np.flatnonzero(live):
                kk, vv = (np.concatenate([p[j] for j in table[i, :-(-lengths[i] // PAGE)]], axis=1)[:, :lengths[i]] for p in (keys, vals))
                row = start[i + 1] - 1
                y, bound = kvq.attention(q[row], kk, vv, int(lengths[i]) - 1, HD ** -0.5, kind=kind)
                assert np.all(np.abs(out[row].astype(np.float64) - y) <= bound), (step, i)
        seen.append(np.array(said))
    assert np.array_equal(*seen)
    assert len(np.unique(seen[0])) > 10
