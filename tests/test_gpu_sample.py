"""ember_sample on the GPU against the definition in 64 bits, token for token."""
import numpy as np
import pytest
import torch

import ember_moe as em

pytestmark = pytest.mark.gpu


def plain(z, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(id, probability, slack) of one row by the definition in include/ember_sample.h; slack: how near u times the sum comes to the
    border of the drawn token, relative to the sum (a draw nearer than the weights' rounding may go either way)."""
    z = z.astype(np.float64)
    V = z.size
    ok = ~(np.isnan(z) | (z == -np.inf))
    if not ok.any():
        return -1, 0.0, 1.0
    zv = np.where(ok, z, -np.inf)
    top = zv.max()
    if temperature <= 0 or top_k == 1 or top_p <= 0:
        return int(np.argmax(zv)), 1.0, 1.0
    with np.errstate(all="ignore"):
        w = np.where(zv == top, 1.0, np.exp((zv - top) / np.float64(np.float32(temperature))))
    w[~ok] = 0.0
    order = np.argsort(-zv, kind="stable")
    ws = w[order].copy()
    if 0 < top_k < V:
        ws[top_k:] = 0.0
    c = np.cumsum(ws)
    keep = ws > 0
    if top_p < 1:
        keep &= (c - ws) < np.float64(np.float32(top_p)) * c[-1]
        keep[0] = True
    keep &= ws >= min(np.float64(np.float32(min_p)), 1.0)
    kept = np.zeros(V, bool)
    kept[order[keep]] = True
    c = np.cumsum(np.where(kept, w, 0.0))
    x = np.float64(np.float32(u)) * c[-1]
    i = int(np.searchsorted(c, x, side="right"))
    lo = c[i - 1] if i else -np.inf
    return i, w[i] / c[-1], min(c[i] - x, x - lo) / c[-1]


def compare(z, u, **kw):
    ids, probs = em.sample(em.Sampler(**kw), z.cuda(), u.cuda())
    zn, un = z.float().numpy(), u.numpy()
    for r in range(z.shape[0]):
        i, p, slack = plain(zn[r], un[r], **kw)
        if slack > 1e-9:  # (the weights' rounding shifts a border by at most V 2^-(61 - log2 V), under 1e-9 at these sizes)
            assert int(ids[r]) == i, (r, kw, int(ids[r]), i)
            assert abs(float(probs[r]) - p) <= 2e-7 * max(p, 1e-9) + 1e-12, (r, float(probs[r]), p)


FILTERS = [{}, dict(top_k=40), dict(top_p=0.9), dict(min_p=0.05), dict(top_k=100, top_p=0.95, min_p=0.02), dict(top_k=5, top_p=0.2),
           dict(temperature=0.3, top_p=0.99), dict(temperature=4.0, top_k=1000), dict(top_p=1e-6), dict(min_p=1.0), dict(min_p=7.0, top_k=3)]


@pytest.mark.parametrize("V", [1, 2, 63, 64, 1000, 1025, 32000, 50257])
@pytest.mark.parametrize("kw", FILTERS, ids=str)
def test_draws(gpu, V, kw):
    g = torch.Generator().manual_seed(V)
    n = 6
    z = torch.randn(n, V, generator=g) * 3
    compare(z, torch.rand(n, generator=g), **kw)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kw", FILTERS, ids=str)
def test_halves_have_many_ties(gpu, dtype, kw):
    g = torch.Generator().manual_seed(9)
    z = (torch.randn(8, 5000, generator=g)).to(dtype)
    compare(z, torch.rand(8, generator=g), **kw)
    compare((z * 2).round(), torch.rand(8, generator=g), **kw)  # some twenty values in all


@pytest.mark.parametrize("kw", FILTERS, ids=str)
def test_all_equal(gpu, kw):
    u = torch.tensor([0.0, 0.3, 0.999999, 0.5])
    compare(torch.full((4, 3000), -7.25), u, **kw)
    z = torch.zeros(4, 777)
    z[:, ::2] = -0.0  # equal to +0
    compare(z, u, **kw)


@pytest.mark.parametrize("kw", FILTERS + [dict(temperature=0.0), dict(temperature=-1.0), dict(top_k=1), dict(top_p=0.0)], ids=str)
def test_what_is_never_drawn(gpu, kw):
    g = torch.Generator().manual_seed(4)
    z = torch.randn(7, 900, generator=g)
    z[0] = float("-inf")
    z[1] = float("nan")
    z[2, ::2] = float("-inf")
    z[3, 1::2] = float("nan")
    z[4, 5], z[4, 800] = float("inf"), float("inf")
    z[5] = float("-inf")
    z[5, 899] = -3e38
    z[6] = torch.finfo(torch.float32).min
    z[6, 17] = torch.finfo(torch.float32).max
    u = torch.rand(7, generator=g)
    compare(z, u, **kw)
    ids, probs = em.sample(em.Sampler(**kw), z.cuda(), u.cuda())
    assert ids[:2].tolist() == [-1, -1] and probs[:2].tolist() == [0, 0]
    assert int(ids[4]) in (5, 800) and int(ids[5]) == 899 and int(ids[6]) == 17


def test_random_numbers_at_the_borders(gpu):
    """u of 0 draws the first token of any weight, the largest below 1 the last; numbers outside count as the nearest."""
    z = torch.full((6, 500), float("-inf"))
    z[:, 100:300] = 0.0
    u = torch.tensor([0.0, 1.0 - 2.0 ** -24, 1.0, 5.0, -1.0, float("nan")])
    ids, probs = em.sample(em.Sampler(), z.cuda(), u.cuda())
    assert ids.tolist() == [100, 299, 299, 299, 100, 100]
    assert (probs.cpu() - 1 / 200).abs().max() < 1e-9


def test_settings_by_row(gpu):
    g = torch.Generator().manual_seed(2)
    n = len(FILTERS) + 3
    z, u = torch.randn(n, 2000, generator=g) * 2, torch.rand(n, generator=g)
    rows = FILTERS + [dict(temperature=float("nan")), dict(top_p=float("nan")), dict(min_p=float("nan"))]
    get = lambda name, off, dt: torch.tensor([f.get(name, off) for f in rows], dtype=dt).cuda()  # noqa: E731
    s = em.Sampler.per_row(n, get("temperature", 1.0, torch.float32), get("top_k", 0, torch.int32), get("top_p", 1.0, torch.float32),
                           get("min_p", 0.0, torch.float32))
    ids, probs = em.sample(s, z.cuda(), u.cuda())
    for r, kw in enumerate(rows):
        kw = {k: v for k, v in kw.items() if v == v}
        i, p, slack = plain(z[r].numpy(), u[r].item(), **kw)
        assert slack < 1e-9 or (int(ids[r]) == i and abs(float(probs[r]) - p) < 1e-6), (r, kw)
    with pytest.raises(em.EmberError):
        em.sample(s, torch.cat([z, z]).cuda(), torch.cat([u, u]).cuda())


def test_rows_apart_and_unaligned(gpu):
    g = torch.Generator().manual_seed(6)
    for dtype in (torch.float32, torch.bfloat16):
        wide = torch.randn(5, 1301, generator=g).to(dtype)
        u = torch.rand(5, generator=g)
        z = wide.cuda()[:, 3:1200]
        a, _ = em.sample(em.Sampler(top_k=50), z, u.cuda())
        b, _ = em.sample(em.Sampler(top_k=50), z.contiguous(), u.cuda())
        assert torch.equal(a, b)
        compare(wide[:, 3:1200].contiguous(), u, top_k=50)


def test_large_vocabulary(gpu):
    g = torch.Generator().manual_seed(8)
    z = torch.randn(3, 200001, generator=g) * 2
    u = torch.rand(3, generator=g)
    for kw in FILTERS:
        compare(z, u, **kw)


def test_frequencies(gpu):
    """Draws over evenly spread random numbers come as often as their probability says, to one draw."""
    n = 4096
    z = torch.tensor([0.0, 1.0, 2.0, -1.0, 2.0]).expand(n, 5).contiguous()
    u = (torch.arange(n) + 0.5) / n
    ids, _ = em.sample(em.Sampler(temperature=0.7, top_k=4), z.cuda(), u.cuda())
    p = torch.softmax(torch.tensor([0.0, 1.0, 2.0, float("-inf"), 2.0]).double() / 0.7, 0)
    seen = torch.bincount(ids.cpu().long(), minlength=5).double()
    assert (seen - n * p).abs().max() <= 1.0


def test_replayed_from_a_graph(gpu):
    z, u = torch.randn(4, 5000, device="cuda"), torch.rand(4, device="cuda")
    ids, probs = torch.zeros(4, dtype=torch.int32, device="cuda"), torch.zeros(4, device="cuda")
    s = em.Sampler(top_k=300, top_p=0.9)
    em.sample(s, z, u, ids, probs)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        em.sample(s, z, u, ids, probs)
    for _ in range(4):
        z.copy_(torch.randn(4, 5000))
        u.copy_(torch.rand(4))
        graph.replay()
        torch.cuda.synchronize()
        a, p = em.sample(s, z, u)
        assert torch.equal(a, ids) and torch.equal(p, probs)


def test_binding_refuses(gpu):
    z, u = torch.randn(2, 10, device="cuda"), torch.rand(2, device="cuda")
    for bad in [(z.double(), u), (z[0], u), (z.t(), u), (z, u[:1]), (z, u.double()), (z.cpu(), u)]:
        with pytest.raises(em.EmberError):
            em.sample(em.Sampler(), *bad)
