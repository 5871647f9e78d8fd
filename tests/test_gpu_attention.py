"""ember_attn on the GPU against the plain attention in 64 bits (attn_util), each element within the bound that the
kernel's roundings add up to."""
import pytest
import torch

import ember_moe as em
from attn_util import TORCH, Setup, check, plain_attention

pytestmark = pytest.mark.gpu


def run(s, q, H, out=None, **opts):
    a = em.attn_options(H, s.D, **opts)
    out = s.cache.attend(a, s.batch, q, out)
    torch.cuda.synchronize()
    return out


def rows(s, H, dtype, std=2.0, seed=1):
    return (torch.randn(s.n, H, s.D, generator=torch.Generator().manual_seed(seed)) * std).to(dtype)


def case(type_, io, seqs, H, n_kv, D, page, seed=0, shared=0, std=2.0, behind=0, q_start=True, **opts):
    s = Setup(type_, seqs, n_kv, D, page, seed=seed, shared=shared, behind=behind, q_start=q_start).up()
    q = rows(s, H, TORCH[io], std)
    dev = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in opts.items()}
    out = torch.full((s.n, H, D), 5.0, dtype=TORCH[io], device="cuda")
    got = run(s, q.cuda(), H, out, **dev)
    want, bound = plain_attention(s, q, H, opts.pop("scale", D ** -0.5), **opts)
    n = s.starts[-1]
    w = check(got[:n], want[:n], bound[:n])
    assert (got[n:] == 5.0).all()  # rows behind the last sequence's
    return s, got, w


TYPES = [(em.BF16, em.BF16), (em.F16, em.F16), (em.Q8_0, em.BF16), (em.Q8_0, em.F16)]


@pytest.mark.parametrize("type_,io", TYPES)
@pytest.mark.parametrize("H,n_kv,D", [(32, 8, 128), (4, 4, 64), (8, 1, 96), (3, 1, 32), (2, 2, 256), (16, 2, 160)])
@pytest.mark.parametrize("page", [0, 64, 48, 5])
def test_steps(gpu, type_, io, H, n_kv, D, page):
    """One new token each, from one key to several splits' worth, without and with row starts."""
    seqs = [(1, 1), (700, 1), (64, 1), (65, 1), (2, 1), (257, 1)]
    case(type_, io, seqs, H, n_kv, D, page, q_start=False)
    case(type_, io, seqs, H, n_kv, D, page, seed=2, behind=2)


@pytest.mark.parametrize("type_,io", TYPES)
@pytest.mark.parametrize("H,n_kv,D", [(8, 2, 128), (4, 4, 64), (6, 1, 96), (2, 1, 256), (3, 3, 32), (20, 2, 192)])
@pytest.mark.parametrize("page", [0, 64, 48])
def test_prompts(gpu, type_, io, H, n_kv, D, page):
    """Whole prompts, parts of them behind what is cached, single tokens and sequences without new ones, together."""
    case(type_, io, [(130, 130), (1, 1), (300, 37), (64, 64), (9, 0), (77, 1), (191, 190)], H, n_kv, D, page, behind=3)


OPTS = {
    "cap": dict(softcap=5.0),
    "window": dict(window=50),
    "window1": dict(window=1),
    "scale": dict(scale=0.5),
    "slopes": dict(slopes=True),
    "prefix": dict(prefix=True),
    "all": dict(softcap=20.0, window=70, slopes=True, prefix=True, scale=0.3),
}


@pytest.mark.parametrize("opts", sorted(OPTS))
@pytest.mark.parametrize("type_,io", [(em.BF16, em.BF16), (em.Q8_0, em.F16)])
@pytest.mark.parametrize("seqs", [[(150, 150), (40, 40), (203, 60)], [(150, 1), (40, 1), (1000, 1), (1, 1)], [(90, 3), (400, 4), (2, 2)]])
def test_options(gpu, opts, type_, io, seqs):
    o = dict(OPTS[opts])
    if "slopes" in o:
        o["slopes"] = torch.tensor([0.5 ** (h + 1) for h in range(8)])
    if "prefix" in o:
        o["prefix"] = torch.tensor([100, 5, 1 << 20, 0][:len(seqs)], dtype=torch.int32)
    case(type_, io, seqs, 8, 2, 64, 48, **o)
    case(type_, io, seqs, 8, 2, 128, 0, **o)


@pytest.mark.parametrize("q_len,H", [(2, 8), (3, 4), (4, 16), (5, 32), (7, 8), (16, 4), (17, 8)])
def test_a_few_new_tokens(gpu, q_len, H):
    """A draft's tokens checked at once, at the borders of what the kernels for single tokens take."""
    case(em.BF16, em.BF16, [(500, q_len), (q_len, q_len), (64, q_len)], H, 4 if H > 4 else 1, 128, 64)
    case(em.Q8_0, em.BF16, [(500, q_len), (q_len, q_len), (64, q_len)], H, 4 if H > 4 else 1, 64, 64)


@pytest.mark.parametrize("G", [1, 5, 16, 17, 32, 40, 128])
def test_heads_per_kv_head(gpu, G):
    case(em.BF16, em.BF16, [(300, 1), (31, 1)], G, 1, 64, 64)
    case(em.Q8_0, em.BF16, [(300, 2), (70, 70)], 2 * G, 2, 64, 64)


@pytest.mark.parametrize("q_len", [1, 40])
def test_long(gpu, q_len):
    case(em.Q8_0, em.BF16, [(30000, q_len), (100, min(q_len, 100))], 8, 2, 128, 64, std=3.0)
    case(em.F16, em.F16, [(20001, q_len)], 4, 1, 64, 0, std=0.1)


def test_rows_that_see_nothing(gpu):
    """Sequences of no length and queries before the first position give zeros."""
    for q_len, kvs in ((1, (0, 5)), (6, (0, 3)), (40, (0, 30))):
        s = Setup(em.BF16, [(8, q_len), (50, q_len)], 2, 64, 16).up()
        s.kv_len.copy_(torch.tensor(kvs))
        q = rows(s, 4, torch.bfloat16)
        got = run(s, q.cuda(), 4)
        s.seqs = [(kvs[0], q_len), (kvs[1], q_len)]
        want, bound = plain_attention(s, q, 4, 0.125)
        check(got, want, bound)
        assert (got[:q_len] == 0).all()
        blind = max(0, q_len - kvs[1])
        assert (got[q_len:q_len + blind] == 0).all()


@pytest.mark.parametrize("type_", [em.BF16, em.F16])
@pytest.mark.parametrize("q_len,window,D", [(1, 0, 64), (1, 20, 128), (3, 20, 64), (100, 0, 64), (100, 30, 128), (100, 30, 256)])
def test_what_is_masked_has_no_effect(gpu, type_, q_len, window, D):
    """Infinities and NaN in the cache behind a sequence's end, before its window and in rows' later keys: a row is NaN exactly
    if it sees one."""
    n = 150
    s = Setup(type_, [(n, q_len), (n - 7, q_len)], 1, D, 64)
    poison = [float("nan"), float("inf"), float("-inf")]
    for b, (kv, _) in enumerate(s.seqs):
        p, r = s.place(b, kv - 1)
        for row in range(r + 1, s.page):  # the rest of the last page
            s.k[p, :, row] = poison[row % 3]
            s.v[p, :, row] = poison[row % 3]
        if q_len > 1:  # a key that the last rows see and the others do not
            p, r = s.place(b, kv - 2)
            s.v[p, 0, r, 3] = poison[b]
        if window:
            p, r = s.place(b, kv - q_len - window - 2)
            s.k[p, 0, r] = float("nan")
            s.v[p, 0, r] = float("inf")
    s.up()
    q = rows(s, 2, TORCH[type_])
    got = run(s, q.cuda(), 2, window=window)
    want, bound = plain_attention(s, q, 2, D ** -0.5, window=window)
    nan = torch.isnan(want).any(-1).any(-1)
    assert int(nan.sum()) == (4 if q_len > 1 else 0)
    g = got.double().cpu()
    # (of a row that sees one only the columns that hold it are lost, or, where weights are NaN, all)
    assert not torch.isnan(g[~nan]).any() and torch.isfinite(g[~nan]).all()
    assert (~torch.isfinite(g[nan])).any(-1).all()
    check(got[~nan.cuda()], want[~nan], bound[~nan])


def test_a_page_out_of_range(gpu):
    """Rows that see a key in such a page are NaN, the others are right."""
    s = Setup(em.Q8_0, [(100, 50), (100, 1), (40, 1)], 2, 64, 16)
    table = s.table.clone()
    table[0, 5], table[1, 0], table[2, 3:] = s.n_pages + 7, -3, 1 << 30
    s.up()
    dev = table.cuda()
    s.batch.pages = dev.data_ptr()
    q = rows(s, 4, torch.bfloat16)
    got = run(s, q.cuda(), 4).double().cpu()
    want, bound = plain_attention(s, q, 4, 0.125)
    sees = torch.tensor([p >= 80 for p in range(50, 100)] + [True, False])
    assert torch.isnan(got[sees]).all()
    check(got[~sees], want[~sees], bound[~sees])


@pytest.mark.parametrize("type_,io", [(em.BF16, em.BF16), (em.F16, em.F16), (em.Q8_0, em.BF16)])
@pytest.mark.parametrize("seqs,shared,page", [([(70, 1), (64, 1), (150, 1), (66, 1)], 64, 16), ([(130, 1)] * 5, 128, 64),
                                              ([(400 + 9 * b, 1) for b in range(33)], 384, 48), ([(210, 3), (199, 1), (230, 30)], 192, 64)])
@pytest.mark.parametrize("opts", ["plain", "all"])
def test_shared(gpu, type_, io, seqs, shared, page, opts):
    """A batch over the same first pages: as without the hint, and within the bound."""
    o = {}
    if opts == "all":
        o = dict(softcap=20.0, window=90, slopes=torch.tensor([0.5 ** (h + 1) for h in range(8)]),
                 prefix=torch.tensor([30] * len(seqs), dtype=torch.int32))
    for D, n_kv in ((128, 2), (64, 8), (256, 1)):
        case(type_, io, seqs, 8, n_kv, D, page, shared=shared, behind=1, **o)


@pytest.mark.parametrize("type_", [em.BF16, em.Q8_0])
@pytest.mark.parametrize("D,opts", [(128, "plain"), (128, "all"), (64, "plain"), (256, "all")])
def test_shared_pages_read_once(gpu, type_, D, opts):
    """Enough sequences behind enough tokens that the shared pages are taken on their own (the scratch says so), some of them
    shorter than these; q rows of some sequences are several."""
    n = 220
    seqs = [(1300, 1)] + [(1280 + (7 * b) % 50, 1 + (b % 9 == 3)) for b in range(1, n)]
    n_kv, H = (4, 8) if D < 256 else (2, 8)
    o = {}
    if opts == "all":
        o = dict(softcap=20.0, window=700, slopes=torch.tensor([0.5 ** (h + 1) for h in range(H)]), prefix=torch.tensor([30] * n, dtype=torch.int32))
    s = Setup(type_, seqs, n_kv, D, 64, shared=1216, behind=1).up()
    short = {5: 1200, 9: 64, 17: 0, 140: 700}
    lens = [short.get(b, kv) for b, (kv, _) in enumerate(seqs)]
    s.kv_len.copy_(torch.tensor(lens))
    dev = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in o.items()}
    a = em.attn_options(H, D, **dev)
    with_, alone = s.cache.attn_scratch_bytes(a, s.batch), None
    s.batch.shared = 0
    alone = s.cache.attn_scratch_bytes(a, s.batch)
    s.batch.shared = 1216
    assert with_ > alone
    q = rows(s, H, torch.bfloat16)
    out = torch.full((s.n, H, D), 5.0, dtype=torch.bfloat16, device="cuda")
    got = run(s, q.cuda(), H, out, **dev)
    s.seqs = [(lens[b], nq) for b, (_, nq) in enumerate(seqs)]
    want, bound = plain_attention(s, q, H, D ** -0.5, heads=[0, H - 1], **o)
    k = s.starts[-1]
    check(got[:k, [0, H - 1]], want[:k, [0, H - 1]], bound[:k, [0, H - 1]])
    assert (got[k:] == 5.0).all()


def test_sequences_shorter_than_the_shared_part(gpu):
    s = Setup(em.BF16, [(100, 1), (100, 2), (70, 70)], 2, 64, 16, shared=64)
    s.up()
    kv = [100, 30, 70]  # the second sequence has only a part of the shared tokens
    s.kv_len.copy_(torch.tensor(kv))
    s.seqs = [(n, q) for n, (_, q) in zip(kv, s.seqs)]
    q = rows(s, 4, torch.bfloat16)
    got = run(s, q.cuda(), 4)
    want, bound = plain_attention(s, q, 4, 0.125)
    check(got, want, bound)


@pytest.mark.parametrize("std", [0.01, 30.0])
def test_flat_and_sharp_scores(gpu, std):
    for seqs in ([(900, 1), (50, 1)], [(200, 200)]):
        case(em.Q8_0, em.F16, seqs, 8, 2, 128, 64, std=std)
        case(em.BF16, em.BF16, seqs, 8, 2, 128, 64, std=std)


def test_queries_past_half_precision_range(gpu):
    """bf16 queries far over 65504 and far under fp16's smallest number, over a quantised cache."""
    s = Setup(em.Q8_0, [(64, 1), (80, 30)], 2, 64, 16)
    s.up()
    for f in (1e8, 1e-12):
        q = (rows(s, 4, torch.float32) * f).bfloat16()
        got = run(s, q.cuda(), 4, scale=0.2 / f)
        want, bound = plain_attention(s, q, 4, 0.2 / f)
        check(got, want, bound)


@pytest.mark.parametrize("q_len", [1, 20])
def test_joint_projection_and_in_place(gpu, q_len):
    """q as a slice of a joint projection, the output into a slice, and over q itself."""
    s = Setup(em.BF16, [(90, q_len), (300, q_len)], 2, 64, 16).up()
    wide = torch.randn(s.n, 12, 64, device="cuda").bfloat16()
    q = wide[:, 2:10]
    want, bound = plain_attention(s, q.cpu(), 8, 0.125)
    out = torch.zeros(s.n, 16, 64, device="cuda", dtype=torch.bfloat16)
    run(s, q, 8, out[:, 4:12])
    check(out[:, 4:12], want, bound)
    assert (out[:, :4] == 0).all() and (out[:, 12:] == 0).all()
    keep = wide.clone()
    got = run(s, q, 8, q)
    check(got, want, bound)
    assert torch.equal(wide[:, :2], keep[:, :2]) and torch.equal(wide[:, 10:], keep[:, 10:])


@pytest.mark.parametrize("seqs,shared", [([(40, 1), (500, 1), (90, 1)], 0), ([(90, 30), (200, 40)], 0), ([(140, 1)] * 6, 128)])
def test_replayed_from_a_graph(gpu, seqs, shared):
    """Captured once; replayed with new queries and lengths, with eager work between: every replay as the eager call, bit for
    bit, and the same again."""
    s = Setup(em.Q8_0, seqs, 2, 128, 16, shared=shared).up()
    q = rows(s, 8, torch.bfloat16).cuda()
    a = em.attn_options(8, 128)
    out, eager = torch.empty_like(q), torch.empty_like(q)
    scratch = torch.empty(max(1, s.cache.attn_scratch_bytes(a, s.batch)), dtype=torch.uint8, device="cuda")
    other = torch.empty_like(scratch)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        s.cache.attend(a, s.batch, q, out, scratch)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.cache.attend(a, s.batch, q, out, scratch)
    for step in range(4):
        q.copy_(torch.randn(q.shape))
        s.kv_len.copy_(torch.tensor([kv - step for kv, _ in seqs]))
        scratch.fill_(255)  # NaN where it is read before it is written
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        s.cache.attend(a, s.batch, q, eager, other)
        assert torch.equal(out.view(torch.int16), eager.view(torch.int16)), step
    s.seqs = [(kv - 3, n) for kv, n in seqs]
    want, bound = plain_attention(s, q.cpu(), 8, 128 ** -0.5)
    check(out, want, bound)


def test_two_streams(gpu):
    """Two calls over one cache on two streams, each with its own scratch."""
    s = Setup(em.BF16, [(3000, 1), (2000, 1)], 2, 128, 64).up()
    a = em.attn_options(8, 128)
    qs = [rows(s, 8, torch.bfloat16, seed=i).cuda() for i in range(2)]
    want = [s.cache.attend(a, s.batch, q) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    outs = [torch.zeros_like(q) for q in qs]
    for st, q, o in zip(streams, qs, outs):
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            for _ in range(5):
                s.cache.attend(a, s.batch, q, o)
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o, w)


def test_scratch_is_checked(gpu):
    s = Setup(em.BF16, [(5000, 1)], 2, 128, 64).up()
    a = em.attn_options(8, 128)
    need = s.cache.attn_scratch_bytes(a, s.batch)
    q = rows(s, 8, torch.bfloat16).cuda()
    out = torch.full_like(q, 3.0)
    if need:
        with pytest.raises(em.EmberError) as e:
            s.cache.attend(a, s.batch, q, out, torch.empty(need - 1, dtype=torch.uint8, device="cuda"))
        assert e.value.status == em.ERR_SCRATCH
        assert (out == 3.0).all()


def test_binding_refuses(gpu):
    s = Setup(em.BF16, [(5, 5)], 2, 64, 16).up()
    q = rows(s, 4, torch.bfloat16).cuda()
    for bad, status in [(q.half(), em.ERR_TYPE), (q.float(), em.ERR_TYPE), (q[:, :3], em.ERR_SHAPE), (q[:4], em.ERR_SHAPE), (q.cpu(), em.ERR_LAUNCH)]:
        with pytest.raises(em.EmberError) as e:
            s.cache.attend(em.attn_options(4, 64), s.batch, bad)
        assert e.value.status == status
    with pytest.raises(em.EmberError):
        s.cache.attend(em.attn_options(4, 64, prefix=torch.zeros(0, dtype=torch.int32, device="cuda")), s.batch, q)
    with pytest.raises(em.EmberError):
        em.attn_options(4, 64, slopes=torch.zeros(3, device="cuda"))


def test_binding_refuses_what_another_stream_may_not_have(gpu):
    """Memory that the binding allocates is the current stream's: a call on another one brings its own."""
    s = Setup(em.BF16, [(5000, 1)], 2, 128, 64).up()
    a, q, side = em.attn_options(8, 128), rows(s, 8, torch.bfloat16).cuda(), torch.cuda.Stream()
    out, scratch = torch.empty_like(q), torch.empty(max(1, s.cache.attn_scratch_bytes(a, s.batch)), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    for kw in (dict(), dict(out=out), dict(scratch=scratch)):
        with pytest.raises(em.EmberError) as e:
            s.cache.attend(a, s.batch, q, stream=side.cuda_stream, **kw)
        assert e.value.status == em.ERR_NULL
    with pytest.raises(em.EmberError):
        s.cache.attend(a, s.batch, q, out, scratch[:1].expand(scratch.numel()))
    with pytest.raises(em.EmberError):
        em.sample(em.Sampler(), torch.zeros(1, 10, device="cuda"), torch.zeros(1, device="cuda"), stream=side.cuda_stream)
    s.cache.attend(a, s.batch, q, out, scratch, stream=side.cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(out, s.cache.attend(a, s.batch, q, stream=torch.cuda.current_stream().cuda_stream))


@pytest.mark.parametrize("type_,io", TYPES[1:])
@pytest.mark.parametrize("page", [4096, 4000])
def test_far_pages(gpu, type_, io, page):
    """Pages past 2^32 values (of Q8_0: bytes) of the cache give what the same rows give at its start."""
    n_kv, D, n_pages = 2, 256, (1 << 32) // (2 * 256 * page) + 4
    cache = em.DeviceKvCache.create(type_, n_pages, n_kv, page, D)
    assert cache.k.numel() > 1 << 32
    near, far = torch.tensor([[1, 0]], dtype=torch.int32).cuda(), torch.tensor([[n_pages - 1, n_pages - 3]], dtype=torch.int32).cuda()
    kv = torch.tensor([page + 100], dtype=torch.int32).cuda()
    x, y = (torch.randn(page + 100, n_kv, D, generator=torch.Generator().manual_seed(i)).to(TORCH[io]).cuda() for i in range(2))
    starts = torch.tensor([0, page + 100], dtype=torch.int32).cuda()
    for table in (near, far):
        cache.store(em.kv_batch(kv, starts, n_tokens=page + 100, max_q=page + 100, max_kv=2 * page, pages=table), x, y)
    a = em.attn_options(8, D)
    for q_len in (1, 200):
        q = torch.randn(q_len, 8, D, generator=torch.Generator().manual_seed(q_len)).to(TORCH[io]).cuda()
        at = torch.tensor([0, q_len], dtype=torch.int32).cuda()
        got = [cache.attend(a, em.kv_batch(kv, at, n_tokens=q_len, max_q=q_len, max_kv=2 * page, pages=t), q) for t in (near, far)]
        assert torch.isfinite(got[0]).all() and torch.equal(got[0], got[1]) and got[0].float().abs().max() > 0.01
