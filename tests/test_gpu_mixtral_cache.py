"""The decoder with this library's cache, attention and sampling (ember_moe/mixtral.py, kv_type): the operators as a prompt and
several sampled continuations of it run them, each call against its definition in 64 bits on the rows that it got."""
import numpy as np
import pytest
import torch

import ember_moe as em
from attn_util import check, plain_attention, quantise
from ember_moe import mixtral
from test_gpu_sample import plain


def spec(**kw):
    return mixtral.MixtralSpec(**{**dict(n_layers=2, d=256, n_heads=4, n_kv=2, head_dim=64, E=4, k=2, d_ff=512, vocab=1000, expert_type=em.Q4_K,
                                         expert_sets=2, seed=1, kv_type=em.BF16, kv_page=16, max_seqs=5), **kw})


def build(s, max_ctx):
    return mixtral.Mixtral(s, max_ctx=max_ctx, log=lambda *a: None)


def tokens(n, vocab=1000):
    return torch.from_numpy(np.random.default_rng(n).integers(0, vocab, n)).cuda()


class Seen:
    """The rows that one layer's cache holds, per sequence, as attn_util.plain_attention asks for them."""

    def __init__(self, s, n):
        self.type, self.n_kv, self.D = s.kv_type, s.n_kv, s.head_dim
        self.held = [[torch.zeros(0, s.n_kv, s.head_dim, dtype=torch.float64)] * 2 for _ in range(n)]

    def add(self, news):
        """news: per sequence (k, v) of its new rows."""
        self.seqs, self.starts = [], [0]
        for b, kv in enumerate(news):
            for i, x in enumerate(kv):
                x = x.cpu()
                if self.type == em.Q8_0:
                    code, d = quantise(x)
                    x = code.double() * d.double().repeat_interleave(32, -1)
                self.held[b] = [*self.held[b][:i], torch.cat([self.held[b][i], x.double()]), *self.held[b][i + 1:]]
            self.seqs.append((self.held[b][0].shape[0], kv[0].shape[0]))
            self.starts.append(self.starts[-1] + kv[0].shape[0])
        self.n = self.starts[-1]
        return self

    def rows(self, b, which):
        return self.held[b][which]


@pytest.mark.gpu
@pytest.mark.parametrize("kv_type", [em.BF16, em.Q8_0])
@pytest.mark.parametrize("T,n", [(37, 5), (32, 3), (7, 2), (21, 1)])
def test_every_call_of_a_sampled_batch(gpu, monkeypatch, kv_type, T, n):
    """The prompt's pages shared, its last partial page copied, steps of n tokens, tokens drawn: what each call gave."""
    s = spec(kv_type=kv_type)
    model = build(s, 64)
    n_new, kw = 11, dict(temperature=0.8, top_k=50, top_p=0.95)
    u = torch.rand(n_new + 1, n, generator=torch.Generator().manual_seed(T))
    layers, calls, draws = {}, [0], []
    attention, draw = model._cached_attention, mixtral.sample

    def attend(l, batch, q, k, v):
        a = attention(l, batch, q, k, v)
        if batch.n_seqs == 1 and batch.n_tokens == T and l not in layers:
            seen = layers[l] = Seen(s, n)
            seen.add([(k, v)])
            first = seen.held[0]
        else:
            seen = layers[l].add([(k[b:b + 1], v[b:b + 1]) for b in range(n)])
            first = None
        want, bound = plain_attention(seen, q.cpu(), s.n_heads, s.head_dim ** -0.5)
        check(a, want, bound, (l, calls[0]))
        if first is not None:
            seen.held = [list(first) for _ in range(n)]
        calls[0] += 1
        return a

    def drawn(sampler, z, u_, *a):
        ids, probs = draw(sampler, z, u_, *a)
        draws.append((z.float().cpu().numpy(), u_.cpu().numpy(), ids.cpu(), probs.cpu()))
        return ids, probs

    monkeypatch.setattr(model, "_cached_attention", attend)
    monkeypatch.setattr(mixtral, "sample", drawn)
    first, out, _, _ = model.sample_many(tokens(T), n_new, u.cuda(), em.Sampler(**kw), use_graph=False)
    assert calls[0] == s.n_layers * (n_new + 1) and len(draws) == n_new + 1
    for i, (z, uu, ids, probs) in enumerate(draws):
        assert np.array_equal(uu, u[i].numpy())
        assert torch.equal(ids.long(), (first if i == 0 else out[i - 1]).cpu())
        for b in range(n):
            j, p, slack = plain(z[b], uu[b], **kw)
            if slack > 1e-9:
                assert int(ids[b]) == j and abs(float(probs[b]) - p) <= 2e-7 * max(p, 1e-9) + 1e-12


@pytest.mark.gpu
@pytest.mark.parametrize("kv_type", [em.BF16, em.Q8_0])
@pytest.mark.parametrize("T", [37, 48])
def test_captured_steps_draw_the_same(gpu, kv_type, T):
    s = spec(kv_type=kv_type)
    u = torch.rand(13, 4, generator=torch.Generator().manual_seed(1)).cuda()
    sampler = em.Sampler(temperature=1.1, min_p=0.01)
    runs = []
    model = build(s, 64)
    for use_graph in (False, True, False):  # (one model: what a run leaves in the cache and the page table does not matter to the next)
        first, out, _, _ = model.sample_many(tokens(T), 12, u, sampler, use_graph=use_graph)
        runs.append((first.cpu(), out.cpu()))
    for r in runs[1:]:
        assert torch.equal(r[0], runs[0][0]) and torch.equal(r[1], runs[0][1])
    assert int(runs[0][1].min()) >= 0 and int(runs[0][1].max()) < s.vocab


@pytest.mark.gpu
@pytest.mark.parametrize("kv_type", [em.BF16, em.Q8_0])
def test_greedy_steps_captured_and_not(gpu, kv_type):
    s = spec(kv_type=kv_type, max_seqs=1)
    runs = [build(s, 50).generate(tokens(24), 16, use_graph=g) for g in (False, True)]  # (50: the last page is partial)
    assert torch.equal(runs[0][0], runs[1][0]) and torch.equal(runs[0][1], runs[1][1])
    # sampling without choice is greedy decoding of one sequence
    first, out, _, _ = build(s, 50).sample_many(tokens(24), 16, torch.rand(17, 1).cuda(), em.Sampler(temperature=0.0))
    assert torch.equal(first, runs[0][0]) and torch.equal(out[:, 0], runs[0][1])


@pytest.mark.parametrize("kw", [dict(kv_type=None), dict(n=3), dict(n=0), dict(T=0), dict(T=10, n_new=7), dict(rows=4)], ids=str)
def test_refusals(kw):
    m = mixtral.Mixtral.__new__(mixtral.Mixtral)  # (the checks come before anything that the model holds)
    m.s, m.max_ctx = spec(kv_type=kw.get("kv_type", em.BF16), max_seqs=2), 16
    n_new = kw.get("n_new", 4)
    with pytest.raises(em.EmberError):
        m.sample_many(torch.zeros(kw.get("T", 5), dtype=torch.int64), n_new, torch.zeros(kw.get("rows", n_new + 1), kw.get("n", 2)), em.Sampler())
