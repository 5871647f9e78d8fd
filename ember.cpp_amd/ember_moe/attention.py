"""Python binding of the paged cache and the attention over it (include/ember_attn.h), on torch tensors.

A decoder layer keeps its keys and values in a `DeviceKvCache`; `kv_batch` says which sequences a step works on and where
their tokens lie; `store` puts the step's new rows into the cache, `attend` computes the attention of the new tokens over
all of it, `load` reads rows back. Errors raise EmberError with the status that the C entry gives (or would give, for what
only the binding can see: tensor types, shapes and devices).
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass, field
from typing import Optional

import ember_moe as em


class KvCache(ctypes.Structure):
    """ember_kv_cache (include/ember_attn.h)."""

    _fields_ = [("type", ctypes.c_int), ("n_kv", ctypes.c_int), ("head_dim", ctypes.c_int), ("page", ctypes.c_int),
                ("n_pages", ctypes.c_int), ("k", ctypes.c_void_p), ("v", ctypes.c_void_p),
                ("k_scale", ctypes.c_void_p), ("v_scale", ctypes.c_void_p)]


class KvBatch(ctypes.Structure):
    """ember_kv_batch (include/ember_attn.h)."""

    device = None  # of its arrays, set by kv_batch
    _fields_ = [("n_seqs", ctypes.c_int), ("n_tokens", ctypes.c_int), ("max_q", ctypes.c_int), ("max_kv", ctypes.c_int),
                ("q_start", ctypes.c_void_p), ("kv_len", ctypes.c_void_p), ("pages", ctypes.c_void_p),
                ("max_pages", ctypes.c_int), ("shared", ctypes.c_int)]


class AttnOpts(ctypes.Structure):
    """ember_attn_opts (include/ember_attn.h)."""

    device = None  # of its arrays, set by attn_options
    _fields_ = [("n_heads", ctypes.c_int), ("scale", ctypes.c_float), ("softcap", ctypes.c_float),
                ("window", ctypes.c_int), ("slopes", ctypes.c_void_p), ("prefix", ctypes.c_void_p)]


def declare(L: ctypes.CDLL) -> None:
    vp, i, i64, sz = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_size_t
    cp, bp, ap = ctypes.POINTER(KvCache), ctypes.POINTER(KvBatch), ctypes.POINTER(AttnOpts)
    for f in (L.ember_kv_store, L.ember_kv_load):
        f.argtypes, f.restype = [cp, bp, vp, i64, vp, i64, i, vp], i
    L.ember_attn_scratch_bytes.argtypes, L.ember_attn_scratch_bytes.restype = [ap, cp, bp], sz
    L.ember_attn.argtypes, L.ember_attn.restype = [ap, cp, bp, vp, i64, vp, i64, i, vp, sz, vp], i


_IDS: dict = {}


def type_id(t) -> int:
    """The ggml type id of a tensor's dtype (F32, F16, BF16)."""
    if not _IDS:
        import torch

        _IDS.update({torch.float32: em.F32, torch.float16: em.F16, torch.bfloat16: em.BF16})
    ty = _IDS.get(t.dtype)
    if ty is None:
        raise em.EmberError(em.ERR_TYPE, f"dtype {t.dtype}")
    return ty


def on_current_device(*tensors, made=()) -> int:
    """Refuses tensors, and descriptors `made` of some, that are not on the current device, where the library launches; its index."""
    import torch

    here = torch.cuda.current_device()
    for t in tensors:
        if t.get_device() != here:  # (-1 for a CPU tensor)
            raise em.EmberError(em.ERR_LAUNCH, f"tensor on {t.device}, the current device is cuda:{here}")
    for d in made:
        if d.device is not None and d.device != here:
            raise em.EmberError(em.ERR_LAUNCH, f"{type(d).__name__} on cuda:{d.device}, the current device is cuda:{here}")
    return here


def own_stream(stream, here: int, what: str) -> None:
    """Refuses a stream other than torch's current one for a call that would allocate `what`: the memory is the current stream's, and
    may be in use there, before the call and after it."""
    if stream is not None and int(stream) != em._stream(None, here):
        raise em.EmberError(em.ERR_NULL, f"{what}: needed on a stream other than the current one")


def _array(t, n: int, dtype, what: str) -> int:
    """The address of a caller's device array of n values, or 0 for None."""
    if t is None:
        return 0
    if t.dtype != dtype or t.numel() < n or not t.is_contiguous():
        raise em.EmberError(em.ERR_SHAPE, f"{what}: a contiguous {dtype} tensor of {n} values is needed")
    return t.data_ptr()


def kv_batch(kv_len, q_start=None, n_tokens: Optional[int] = None, max_q: Optional[int] = None, max_kv: Optional[int] = None,
             pages=None, shared: int = 0) -> KvBatch:
    """A batch's descriptor from int32 device tensors: kv_len [n_seqs], q_start [n_seqs + 1] (None: one new token
    each), pages [n_seqs, max_pages] (None: sequence b lies in page b). max_kv, the most tokens that a sequence has, is needed, and with
    q_start n_tokens; max_q None: n_tokens (of one sequence). Keeps the tensors."""
    import torch

    n = kv_len.numel()
    if max_kv is None or (q_start is not None and n_tokens is None):
        raise em.EmberError(em.ERR_SHAPE, "max_kv, and n_tokens with q_start, are needed")
    n_tokens = n if n_tokens is None else n_tokens
    if max_q is None:
        max_q = 1 if q_start is None else max(n_tokens, 1)
    b = KvBatch(n_seqs=n, n_tokens=n_tokens, max_q=max_q, max_kv=max_kv, shared=shared)
    b.kv_len = _array(kv_len, n, torch.int32, "kv_len")
    b.q_start = _array(q_start, n + 1, torch.int32, "q_start")
    if pages is not None:
        if pages.dim() != 2 or pages.shape[0] < n:
            raise em.EmberError(em.ERR_SHAPE, "pages: [n_seqs, max_pages] is needed")
        b.pages, b.max_pages = _array(pages, pages.numel(), torch.int32, "pages"), pages.shape[1]
    b.device = on_current_device(*(t for t in (kv_len, q_start, pages) if t is not None))
    b._owner = (kv_len, q_start, pages)
    return b


def attn_options(n_heads: int, head_dim: int, scale: Optional[float] = None, softcap: float = 0.0, window: int = 0,
                 slopes=None, prefix=None) -> AttnOpts:
    """Attention options; scale None: 1 / sqrt(head_dim). slopes f32 [n_heads], prefix int32 [n_seqs]. Keeps the tensors."""
    import torch

    a = AttnOpts(n_heads=n_heads, scale=head_dim ** -0.5 if scale is None else scale, softcap=softcap, window=window)
    a.slopes = _array(slopes, n_heads, torch.float32, "slopes")
    a.prefix = _array(prefix, 0, torch.int32, "prefix")
    if slopes is not None or prefix is not None:
        a.device = on_current_device(*(t for t in (slopes, prefix) if t is not None))
    a._owner = (slopes, prefix)
    return a


def _rows(t, n: int, heads: int, dim: int, what: str) -> int:
    """Checks a [n, heads, dim] tensor whose rows may be apart (a slice of a joint projection); its row stride."""
    shape, stride = t.shape, t.stride()
    if len(shape) != 3 or shape[0] < n or shape[1] != heads or shape[2] != dim or (heads > 1 and stride[1] != dim) or stride[2] != 1:
        raise em.EmberError(em.ERR_SHAPE, f"{what}: [{n}, {heads}, {dim}] with whole rows is needed, got {tuple(shape)}")
    # (a single row's stride is anyone's: torch may give 1)
    return max(stride[0], heads * dim) if n <= 1 else stride[0]


@dataclass
class DeviceKvCache:
    """One layer's cache on the device: k, v [n_pages, n_kv, page, head_dim] (int8 with fp16 k_scale, v_scale [n_pages,
    n_kv, page, head_dim / 32] for Q8_0) and the C descriptor pointing at them."""

    type: int
    k: object
    v: object
    k_scale: object = None
    v_scale: object = None
    desc: KvCache = field(default_factory=KvCache)

    def __post_init__(self):
        import torch

        want = {em.F16: torch.float16, em.BF16: torch.bfloat16, em.Q8_0: torch.int8}.get(self.type)
        if want is None:
            raise em.EmberError(em.ERR_TYPE, "a cache is F16, BF16 or Q8_0")
        shape = tuple(self.k.shape)
        if len(shape) != 4 or tuple(self.v.shape) != shape or not self.k.is_contiguous() or not self.v.is_contiguous():
            raise em.EmberError(em.ERR_SHAPE, "k, v: contiguous [n_pages, n_kv, page, head_dim] are needed")
        if self.k.dtype != want or self.v.dtype != want:
            raise em.EmberError(em.ERR_TYPE, f"k, v of a {em.TYPE_NAMES[self.type]} cache are {want}")
        d = self.desc
        d.type, (d.n_pages, d.n_kv, d.page, d.head_dim) = self.type, shape
        d.k, d.v = self.k.data_ptr(), self.v.data_ptr()
        self.device = on_current_device(self.k, self.v)
        if self.type == em.Q8_0:
            for t in (self.k_scale, self.v_scale):
                if t is None or tuple(t.shape) != shape[:3] + (shape[3] // 32,) or t.dtype != torch.float16 or not t.is_contiguous():
                    raise em.EmberError(em.ERR_SHAPE, "k_scale, v_scale: contiguous fp16 [n_pages, n_kv, page, head_dim / 32] are needed")
                on_current_device(t)
            d.k_scale, d.v_scale = self.k_scale.data_ptr(), self.v_scale.data_ptr()

    @staticmethod
    def create(type_: int, n_pages: int, n_kv: int, page: int, head_dim: int, device="cuda") -> "DeviceKvCache":
        import torch

        dt = {em.F16: torch.float16, em.BF16: torch.bfloat16, em.Q8_0: torch.int8}.get(type_)
        if dt is None:
            raise em.EmberError(em.ERR_TYPE, "a cache is F16, BF16 or Q8_0")
        shape = (n_pages, n_kv, page, head_dim)
        k, v = (torch.zeros(shape, dtype=dt, device=device) for _ in range(2))
        if type_ != em.Q8_0:
            return DeviceKvCache(type_, k, v)
        return DeviceKvCache(type_, k, v, *(torch.zeros(shape[:3] + (head_dim // 32,), dtype=torch.float16, device=device) for _ in range(2)))

    def _kv(self, fn: str, batch: KvBatch, k, v, stream):
        d, n = self.desc, batch.n_tokens
        heads, dim = d.n_kv, d.head_dim
        ks, vs = _rows(k, n, heads, dim, "k"), _rows(v, n, heads, dim, "v")
        ty = type_id(k)
        if k.dtype != v.dtype:
            raise em.EmberError(em.ERR_TYPE, "k and v of one type are needed")
        here = on_current_device(k, v, made=(self, batch))
        st = getattr(em.lib(), fn)(ctypes.byref(d), ctypes.byref(batch), k.data_ptr(), ks, v.data_ptr(), vs, ty, em._stream(stream, here))
        if st:
            raise em.EmberError(st, fn)
        return k, v

    def store(self, batch: KvBatch, k, v, stream=None) -> None:
        """Stores rows k, v [n_tokens, n_kv, head_dim] (f32, f16 or bf16) at the batch's places (ember_kv_store)."""
        self._kv("ember_kv_store", batch, k, v, stream)

    def load(self, batch: KvBatch, k, v, stream=None):
        """Reads the rows at the batch's places into k, v (ember_kv_load); returns them."""
        return self._kv("ember_kv_load", batch, k, v, stream)

    def attn_scratch_bytes(self, opts: AttnOpts, batch: KvBatch) -> int:
        return int(em.lib().ember_attn_scratch_bytes(ctypes.byref(opts), ctypes.byref(self.desc), ctypes.byref(batch)))

    def attend(self, opts: AttnOpts, batch: KvBatch, q, out=None, scratch=None, stream=None):
        """Attention of the rows q [n_tokens, n_heads, head_dim] over the cache (ember_attn); returns out."""
        import torch

        d = self.desc
        qs = _rows(q, batch.n_tokens, opts.n_heads, d.head_dim, "q")
        here = torch.cuda.current_device()
        if out is None:
            own_stream(stream, here, "out")
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        os_ = _rows(out, batch.n_tokens, opts.n_heads, d.head_dim, "out")
        if out.dtype != q.dtype:
            raise em.EmberError(em.ERR_TYPE, "q and out of one type are needed")
        prefix = getattr(opts, "_owner", (None, None))[1]
        if prefix is not None and prefix.numel() < batch.n_seqs:
            raise em.EmberError(em.ERR_SHAPE, "prefix: one length per sequence is needed")
        if scratch is None:
            need = self.attn_scratch_bytes(opts, batch)
            if need:
                own_stream(stream, here, "scratch")
            scratch = torch.empty(max(1, need), dtype=torch.uint8, device=q.device)
        elif not scratch.is_contiguous():
            raise em.EmberError(em.ERR_SCRATCH, "scratch: contiguous memory is needed")
        on_current_device(q, out, scratch, made=(self, batch, opts))
        st = em.lib().ember_attn(ctypes.byref(opts), ctypes.byref(d), ctypes.byref(batch), q.data_ptr(), qs, out.data_ptr(), os_,
                                 type_id(q), scratch.data_ptr(), scratch.numel() * scratch.element_size(), em._stream(stream, here))
        if st:
            raise em.EmberError(st, "ember_attn")
        return out
