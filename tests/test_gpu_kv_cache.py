"""The paged cache on the GPU: stored rows bit by bit against the definition, rows read back, the places that are left
alone, and calls that the entries refuse."""
import numpy as np
import pytest
import torch

import ember_moe as em
from attn_util import TORCH, Setup, quantise

pytestmark = pytest.mark.gpu

SEQS = {
    "one": [(1, 1)],
    "steps": [(5, 1), (64, 1), (65, 1), (200, 1), (1, 1)],
    "prompts": [(70, 70), (1, 1), (130, 33), (64, 64)],
    "none": [(7, 0), (40, 40), (9, 0), (33, 2)],
    "many": [(3 + b % 5, 1 + b % 3) for b in range(150)],
}


def _bits(t):
    return t.contiguous().view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[t.element_size()])


@pytest.mark.parametrize("seqs", sorted(SEQS))
@pytest.mark.parametrize("type_,io", [(em.Q8_0, em.BF16), (em.Q8_0, em.F32), (em.BF16, em.BF16), (em.F16, em.F32), (em.Q8_0, em.F16),
                                      (em.F16, em.BF16), (em.BF16, em.F32)])
@pytest.mark.parametrize("n_kv,D,page", [(8, 128, 64), (1, 32, 7), (3, 96, 0), (2, 256, 100)])
def test_store_and_load(gpu, seqs, type_, io, n_kv, D, page):
    s = Setup(type_, SEQS[seqs], n_kv, D, page, seed=len(seqs), behind=3).up()
    g = torch.Generator().manual_seed(7)
    # rows as slices of a joint projection: apart, and K and V by different strides
    wide = torch.randn(s.n, 3 * n_kv, D, generator=g) * torch.exp2(torch.randint(-6, 4, (s.n, 1, 1), generator=g).float())
    wide = wide.to(TORCH[io]).cuda()
    k, v = wide[:, n_kv:2 * n_kv], wide[:, 2 * n_kv:].contiguous()
    want = [t.clone() for t in (s.k, s.v)]
    want_sc = [None if t is None else t.clone() for t in s.scales]
    for which, x in ((0, k.cpu()), (1, v.cpu())):
        for b, (kv, q) in enumerate(s.seqs):
            for i in range(q):
                p, r = s.place(b, kv - q + i)
                row = x[s.starts[b] + i]
                if type_ == em.Q8_0:
                    want[which][p, :, r], want_sc[which][p, :, r] = quantise(row)
                else:
                    want[which][p, :, r] = row.to(TORCH[type_])
    s.cache.store(s.batch, k, v)
    for which, t, sc in ((0, s.cache.k, s.cache.k_scale), (1, s.cache.v, s.cache.v_scale)):
        assert torch.equal(_bits(t.cpu()), _bits(want[which])), which  # (what no row goes to stays as it was)
        if sc is not None:
            assert torch.equal(_bits(sc.cpu()), _bits(want_sc[which]))
    # and back, in each type; rows behind the last sequence's are not written
    s.k, s.v, s.scales = want[0], want[1], tuple(want_sc)
    for back in (em.F32, em.F16, em.BF16):
        ko, vo = (torch.full((s.n, n_kv, D), 7.0, dtype=TORCH[back], device="cuda") for _ in range(2))
        s.cache.load(s.batch, ko, vo)
        for which, t in ((0, ko), (1, vo)):
            ref = torch.full((s.n, n_kv, D), 7.0, dtype=TORCH[back])
            for b, (kv, q) in enumerate(s.seqs):
                ref[s.starts[b]:s.starts[b] + q] = s.rows(b, which, kv - q, kv).float().to(TORCH[back])
            assert torch.equal(t.cpu(), ref), (back, which)


def test_blocks_at_the_edge(gpu):
    """Q8_0 blocks of zeros, subnormals, one huge value, infinities, NaN, exact ties, and values that round to the
    scale's neighbours."""
    D, n = 64, 64
    x = torch.zeros(n, 1, D)
    g = torch.Generator().manual_seed(3)
    for i in range(n):
        x[i, 0] = torch.randn(D, generator=g) * 2.0 ** (i - 40)
    x[0] = 0
    x[1, 0, :32] = 1e-30
    x[2, 0, 3], x[2, 0, 40] = float("inf"), float("-inf")
    x[3, 0, 5] = float("nan")
    x[4, 0, :32] = torch.arange(32) * 0.5  # ties of codes
    x[4, 0, 31] = 127.0
    x[5, 0, 0], x[5, 0, 32] = 3e38, 65504.0
    x[6, 0] = -0.0
    x[7, 0, :32] = torch.linspace(-6.5e4, 6.5e4, 32)
    s = Setup(em.Q8_0, [(n, n)], 1, D, 16).up()
    s.cache.store(s.batch, x.cuda(), x.cuda())
    k, v = (torch.empty(n, 1, D, device="cuda") for _ in range(2))
    s.cache.load(s.batch, k, v)
    codes, d = quantise(x)
    want = codes.float() * d.float().repeat_interleave(32, -1)
    assert torch.equal(torch.isnan(k.cpu()), torch.isnan(want)) and torch.isnan(want).sum() == 32
    assert torch.equal(torch.nan_to_num(k.cpu()), torch.nan_to_num(want)) and torch.equal(torch.nan_to_num(v.cpu()), torch.nan_to_num(want))


def test_values_stay_within_half_a_step(gpu):
    """What is read back is within half a code of what was stored, for every block whose scale is a normal fp16 number."""
    s = Setup(em.Q8_0, [(300, 300)], 4, 128, 64).up()
    x = torch.randn(300, 4, 128, generator=torch.Generator().manual_seed(5)).cuda()
    k, v = torch.empty_like(x), torch.empty_like(x)
    s.cache.store(s.batch, x, x * 3)
    s.cache.load(s.batch, k, v)
    for got, ref in ((k, x), (v, x * 3)):
        b = ref.unflatten(-1, (-1, 32)).double()
        # half a code, and the most that 127 codes fall short of the largest value by the scale's rounding (2^-11 of it)
        step = b.abs().amax(-1, keepdim=True) / 127 * (1 + 2.0 ** -11)
        over = b.abs().amax(-1, keepdim=True) * 2.0 ** -11
        assert ((got.double().unflatten(-1, (-1, 32)) - b).abs() <= torch.maximum(step / 2, over) * (1 + 1e-6)).all()


def test_sequence_in_the_last_page_row(gpu):
    """A token whose table entry is past the pages, one at a negative position, and one past the table are not stored, and
    read as zeros."""
    s = Setup(em.BF16, [(20, 4), (2, 4), (64, 2)], 2, 32, 16).up()
    s.batch.max_kv = 64
    table = s.table.clone()
    table[0, 1] = s.n_pages          # positions 16 .. 19 of sequence 0
    table[2, 3] = -1                 # positions 48 .. 63 of sequence 2
    dev = table.cuda()
    s.batch.pages = dev.data_ptr()
    before = s.cache.k.clone()
    x = torch.randn(s.n, 2, 32, dtype=torch.bfloat16, device="cuda")
    s.cache.store(s.batch, x, x)
    k, v = (torch.full((s.n, 2, 32), 9.0, device="cuda") for _ in range(2))
    s.cache.load(s.batch, k, v)
    stored = [6, 7]                  # positions 0 and 1 of sequence 1
    for i in range(s.n):
        assert torch.equal(k[i].cpu(), x[i].float().cpu() if i in stored else torch.zeros(2, 32)), i
    changed = (s.cache.k != before).flatten(2).any(-1).any(-1).nonzero().flatten().tolist()
    assert changed == [int(table[1, 0])]


def test_replayed_from_a_graph(gpu):
    """Captured once and replayed with other rows and lengths in the same buffers: each replay as the eager call."""
    s = Setup(em.Q8_0, [(40, 1), (17, 1), (90, 1)], 2, 64, 16).up()
    x = torch.randn(3, 2, 64, device="cuda")
    k, v = torch.empty_like(x), torch.empty_like(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        s.cache.store(s.batch, x, x)
        s.cache.load(s.batch, k, v)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.cache.store(s.batch, x, x)
        s.cache.load(s.batch, k, v)
    for step in range(4):
        x.copy_(torch.randn(3, 2, 64))
        s.kv_len.copy_(torch.tensor([40 - step, 17 + step, 90 - 3 * step]))
        graph.replay()
        torch.cuda.synchronize()
        codes, d = quantise(x.cpu())
        want = codes.float() * d.float().repeat_interleave(32, -1)
        assert torch.equal(k.cpu(), want) and torch.equal(v.cpu(), want)


def test_another_stream(gpu):
    s = Setup(em.F16, [(30, 30)], 2, 64, 16).up()
    x = torch.randn(30, 2, 64, device="cuda")
    k, v = torch.zeros_like(x), torch.zeros_like(x)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    s.cache.store(s.batch, x, x, stream=st.cuda_stream)
    s.cache.load(s.batch, k, v, stream=st.cuda_stream)
    torch.cuda.current_stream().wait_stream(st)
    assert torch.equal(k, x.half().float()) and torch.equal(v, k)


def test_far_offsets(gpu):
    """A cache of over 2^32 values: pages at its far end."""
    n_kv, D, page, n_pages = 2, 256, 1 << 16, 130  # 4.4e9 values, 4.4 GB of codes in K, and scales
    cache = em.DeviceKvCache.create(em.Q8_0, n_pages, n_kv, page, D)
    assert cache.k.numel() > 1 << 32
    table = torch.tensor([[129, 0, 128]], dtype=torch.int32, device="cuda")
    kv_len = torch.tensor([3 * page], dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, page + 5], dtype=torch.int32, device="cuda")
    b = em.kv_batch(kv_len, starts, n_tokens=page + 5, max_q=page + 5, max_kv=3 * page, pages=table)
    x = torch.randn(page + 5, n_kv, D, device="cuda", dtype=torch.bfloat16)
    cache.store(b, x, x)
    k, v = torch.empty_like(x), torch.empty_like(x)
    cache.load(b, k, v)
    codes, d = quantise(x[:8].cpu())
    want = (codes.float() * d.float().repeat_interleave(32, -1)).bfloat16()
    assert torch.equal(k[:8].cpu(), want)
    assert (k.float() - x.float()).abs().max() < 0.1 and torch.equal(k, v)
    assert int((cache.k[128] != 0).any(-1).sum()) == n_kv * page and not cache.k[1:128].any()


def test_binding_refuses(gpu):
    s = Setup(em.Q8_0, [(4, 4)], 2, 64, 16).up()
    x = torch.zeros(4, 2, 64, device="cuda")
    for k, v, status in [(x[:3], x, em.ERR_SHAPE), (x, x.half(), em.ERR_TYPE), (x.double(), x.double(), em.ERR_TYPE),
                         (x[:, :1], x, em.ERR_SHAPE), (x.cpu(), x, em.ERR_LAUNCH), (x.transpose(1, 2), x, em.ERR_SHAPE)]:
        with pytest.raises(em.EmberError) as e:
            s.cache.store(s.batch, k, v)
        assert e.value.status == status
    with pytest.raises(em.EmberError):
        em.DeviceKvCache(em.Q8_0, s.cache.k, s.cache.v)
    with pytest.raises(em.EmberError):
        em.DeviceKvCache(em.Q4_K, s.cache.k, s.cache.v)
    with pytest.raises(em.EmberError):
        em.kv_batch(s.kv_len.long())
    assert np.isfinite(s.scales[0].float().numpy()).all()
