"""CPU checks of the cache, attention and sampling entries of the C ABI: every declared function is exported, and calls that
are refused return the documented status before any GPU work."""
import ctypes
import os
import subprocess

import pytest

import ember_moe as em
from test_capi import declared, exported


def test_library_exports_every_declared_symbol():
    for header, some in (("ember_attn.h", {"ember_kv_store", "ember_kv_load", "ember_attn", "ember_attn_scratch_bytes"}),
                         ("ember_sample.h", {"ember_sample"})):
        names = set(declared(header))
        assert some <= names
        assert names <= exported(em.lib_path())


def cache(**kw):
    c = em.KvCache(type=em.Q8_0, n_kv=2, head_dim=64, page=16, n_pages=10, k=0x10000, v=0x20000, k_scale=0x30000, v_scale=0x40000)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def batch(**kw):
    b = em.KvBatch(n_seqs=3, n_tokens=3, max_q=1, max_kv=100, q_start=0, kv_len=0x50000, pages=0x60000, max_pages=7, shared=0)
    for k, v in kw.items():
        setattr(b, k, v)
    return b


def opts(**kw):
    a = em.AttnOpts(n_heads=4, scale=0.125, softcap=0.0, window=0, slopes=0, prefix=0)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


BAD_CACHE = [(dict(type=em.F32), em.ERR_TYPE), (dict(type=em.Q4_K), em.ERR_TYPE), (dict(head_dim=48), em.ERR_SHAPE),
             (dict(head_dim=288), em.ERR_SHAPE), (dict(head_dim=0), em.ERR_SHAPE), (dict(n_kv=0), em.ERR_SHAPE), (dict(n_kv=257), em.ERR_SHAPE),
             (dict(page=0), em.ERR_SHAPE), (dict(n_pages=0), em.ERR_SHAPE), (dict(n_pages=2**31 - 1, page=2**31 - 1), em.ERR_SHAPE),
             (dict(k=0), em.ERR_NULL), (dict(v=0), em.ERR_NULL), (dict(k_scale=0), em.ERR_NULL), (dict(v=0x20008), em.ERR_ALIGN),
             (dict(v_scale=0x40002), em.ERR_ALIGN)]
BAD_BATCH = [(dict(n_seqs=-1), em.ERR_SHAPE), (dict(n_seqs=65536, n_tokens=65536), em.ERR_SHAPE), (dict(n_tokens=2), em.ERR_SHAPE),
             (dict(n_tokens=-1), em.ERR_SHAPE), (dict(max_q=0), em.ERR_SHAPE), (dict(max_kv=-1), em.ERR_SHAPE), (dict(max_kv=2**30 + 1), em.ERR_SHAPE),
             (dict(kv_len=0), em.ERR_NULL), (dict(max_pages=0), em.ERR_SHAPE), (dict(pages=0, n_seqs=11, n_tokens=11), em.ERR_SHAPE),
             (dict(shared=-16), em.ERR_SHAPE), (dict(shared=8), em.ERR_SHAPE), (dict(shared=128), em.ERR_SHAPE), (dict(pages=0, shared=16), em.ERR_SHAPE),
             (dict(kv_len=0x50002), em.ERR_ALIGN), (dict(pages=0x60001), em.ERR_ALIGN), (dict(q_start=0x70002), em.ERR_ALIGN)]


def _store(fn, c, b, k=0x100000, ks=128, v=0x200000, vs=128, type_=em.F16):
    p = ctypes.byref
    return getattr(em.lib(), fn)(p(c) if c else None, p(b) if b else None, k, ks, v, vs, type_, None)


@pytest.mark.parametrize("fn", ["ember_kv_store", "ember_kv_load"])
def test_rows_are_checked(fn):
    for kw, status in BAD_CACHE:
        assert _store(fn, cache(**kw), batch()) == status, kw
    for kw, status in BAD_BATCH:
        assert _store(fn, cache(), batch(**kw)) == status, kw
    assert _store(fn, None, batch()) == em.ERR_NULL and _store(fn, cache(), None) == em.ERR_NULL
    for kw, status in [(dict(type_=em.Q8_0), em.ERR_TYPE), (dict(k=0), em.ERR_NULL), (dict(v=0), em.ERR_NULL), (dict(ks=127), em.ERR_SHAPE),
                       (dict(vs=-128), em.ERR_SHAPE), (dict(k=0x100008), em.ERR_ALIGN), (dict(vs=132), em.ERR_ALIGN),
                       (dict(vs=2**41), em.ERR_SHAPE), (dict(ks=130, type_=em.F32), em.ERR_ALIGN)]:
        assert _store(fn, cache(), batch(), **kw) == status, kw
    assert _store(fn, cache(), batch(n_seqs=0, n_tokens=0), k=0, v=0) == em.OK
    assert _store(fn, cache(), batch(n_seqs=0, n_tokens=0, kv_len=0), k=0, v=0) == em.OK


def _attn(a, c, b, q=0x100000, qs=256, out=0x200000, os_=256, type_=em.BF16, scratch=0x300000, n=1 << 40):
    p = ctypes.byref
    return em.lib().ember_attn(p(a) if a else None, p(c) if c else None, p(b) if b else None, q, qs, out, os_, type_, scratch, n, None)


def test_attention_is_checked():
    for kw, status in BAD_CACHE:
        assert _attn(opts(), cache(**kw), batch()) == status, kw
    for kw, status in BAD_BATCH:
        assert _attn(opts(), cache(), batch(**kw)) == status, kw
    nan = float("nan")
    for kw, status in [(dict(n_heads=3), em.ERR_SHAPE), (dict(n_heads=0), em.ERR_SHAPE), (dict(n_heads=258), em.ERR_SHAPE), (dict(scale=0.0), em.ERR_SHAPE),
                       (dict(scale=-1.0), em.ERR_SHAPE), (dict(scale=nan), em.ERR_SHAPE), (dict(scale=float("inf")), em.ERR_SHAPE),
                       (dict(softcap=-1.0), em.ERR_SHAPE), (dict(softcap=nan), em.ERR_SHAPE), (dict(window=-1), em.ERR_SHAPE),
                       (dict(slopes=0x70001), em.ERR_ALIGN), (dict(prefix=0x70002), em.ERR_ALIGN)]:
        assert _attn(opts(**kw), cache(), batch()) == status, kw
        assert em.lib().ember_attn_scratch_bytes(ctypes.byref(opts(**kw)), ctypes.byref(cache()), ctypes.byref(batch())) == 0
    assert _attn(None, cache(), batch()) == em.ERR_NULL
    for kw, status in [(dict(type_=em.F32), em.ERR_TYPE), (dict(q=0), em.ERR_NULL), (dict(out=0), em.ERR_NULL), (dict(qs=255), em.ERR_SHAPE),
                       (dict(os_=260), em.ERR_ALIGN), (dict(out=0x200008), em.ERR_ALIGN)]:
        assert _attn(opts(), cache(), batch(), **kw) == status, kw
    assert _attn(opts(), cache(type=em.BF16), batch(), type_=em.F16) == em.ERR_TYPE
    assert _attn(opts(), cache(type=em.F16), batch(), type_=em.BF16) == em.ERR_TYPE
    assert _attn(opts(), cache(), batch(n_seqs=0, n_tokens=0), q=0, out=0) == em.OK


def test_scratch_is_checked():
    a, c, b = opts(n_heads=8), cache(n_pages=10000), batch(max_pages=9000, max_kv=100000)
    need = em.lib().ember_attn_scratch_bytes(ctypes.byref(a), ctypes.byref(c), ctypes.byref(b))
    if need:
        assert _attn(a, c, b, qs=512, os_=512, n=need - 1) == em.ERR_SCRATCH
        assert _attn(a, c, b, qs=512, os_=512, scratch=0) == em.ERR_SCRATCH
        assert _attn(a, c, b, qs=512, os_=512, scratch=0x300080) == em.ERR_ALIGN


def test_sampling_is_checked():
    def call(s=True, z=0x100000, type_=em.F32, n=2, V=100, stride=100, u=0x200000, ids=0x300000, probs=0, **kw):
        smp = em.Sampler()
        for k, v in kw.items():
            setattr(smp, k, v)
        return em.lib().ember_sample(ctypes.byref(smp) if s else None, z, type_, n, V, stride, u, ids, probs, None)

    for kw, status in [(dict(s=False), em.ERR_NULL), (dict(type_=em.Q8_0), em.ERR_TYPE), (dict(n=-1), em.ERR_SHAPE), (dict(V=0), em.ERR_SHAPE),
                       (dict(V=(1 << 24) + 1, stride=1 << 25), em.ERR_SHAPE), (dict(stride=99), em.ERR_SHAPE), (dict(stride=2**41), em.ERR_SHAPE),
                       (dict(z=0), em.ERR_NULL), (dict(u=0), em.ERR_NULL), (dict(ids=0), em.ERR_NULL), (dict(z=0x100002), em.ERR_ALIGN),
                       (dict(z=0x100001, type_=em.F16), em.ERR_ALIGN), (dict(ids=0x300001), em.ERR_ALIGN), (dict(probs=0x300002), em.ERR_ALIGN),
                       (dict(temperatures=0x400002), em.ERR_ALIGN), (dict(top_ks=0x400001), em.ERR_ALIGN)]:
        assert call(**kw) == status, kw
    assert call(n=0, z=0, u=0, ids=0) == em.OK


def test_calls_too_large_for_a_launch():
    """More blocks than a launch can have: refused before anything runs."""
    big = batch(n_tokens=2**31 - 1, max_q=2**31 - 1, q_start=0x70000, max_kv=112)
    wide = cache(n_kv=256, head_dim=256, n_pages=16)
    for fn in ("ember_kv_store", "ember_kv_load"):
        assert _store(fn, wide, big, ks=65536, vs=65536) == em.ERR_SHAPE
    assert _attn(opts(n_heads=256), cache(), big, qs=256 * 64, os_=256 * 64) == em.ERR_SHAPE
    a = em.Sampler()
    assert em.lib().ember_sample(ctypes.byref(a), 0x100000, em.F32, 1 << 23, 100, 100, 0x200000, 0x300000, 0, None) == em.ERR_SHAPE


def test_places_and_plans():
    """The native check of what keeps the kernels inside their buffers: places of tokens for device arrays of any content, and the
    parts that a call is split into."""
    exe = os.path.join(os.path.dirname(__file__), "native", "attn_host_check")
    if not os.path.exists(exe):
        lib = os.path.dirname(em.lib_path())
        subprocess.run(["make", "-C", lib, os.path.relpath(exe, lib)], check=True, capture_output=True, timeout=600)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and r.stdout.startswith("ok"), r.stdout + r.stderr


def test_a_cap_far_under_the_scale_is_refused():
    assert _attn(opts(softcap=1e-39), cache(), batch()) == em.ERR_SHAPE
    assert _attn(opts(softcap=1e-35, scale=1.0), cache(), batch()) == em.ERR_SHAPE


def test_a_batch_needs_its_sizes():
    torch = pytest.importorskip("torch")
    for kw in (dict(), dict(max_kv=5, q_start=torch.zeros(2, dtype=torch.int32))):
        with pytest.raises(em.EmberError) as e:
            em.kv_batch(torch.ones(1, dtype=torch.int32), **kw)
        assert e.value.status == em.ERR_SHAPE
