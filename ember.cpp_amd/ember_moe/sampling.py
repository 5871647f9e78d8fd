"""Python binding of the pick of the next token (include/ember_sample.h), on torch tensors."""
from __future__ import annotations

import ctypes

import ember_moe as em

from .attention import _array, on_current_device, own_stream, type_id


class Sampler(ctypes.Structure):
    """ember_sampler (include/ember_sample.h): temperature, top_k, top_p, min_p of every row, or per row by `sampler`."""

    _fields_ = [("temperature", ctypes.c_float), ("top_k", ctypes.c_int), ("top_p", ctypes.c_float),
                ("min_p", ctypes.c_float), ("temperatures", ctypes.c_void_p), ("top_ks", ctypes.c_void_p),
                ("top_ps", ctypes.c_void_p), ("min_ps", ctypes.c_void_p)]

    def __init__(self, temperature: float = 1.0, top_k: int = 0, top_p: float = 1.0, min_p: float = 0.0):
        super().__init__(temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
        self._rows, self._owner = None, ()

    @staticmethod
    def per_row(n: int, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0) -> "Sampler":
        """Settings for n rows, each a number or a device tensor [n] (f32; top_k int32). Keeps the tensors."""
        import torch

        s, kept = Sampler(), []
        s._rows = n
        for name, value, dtype in (("temperature", temperature, torch.float32), ("top_k", top_k, torch.int32),
                                   ("top_p", top_p, torch.float32), ("min_p", min_p, torch.float32)):
            if isinstance(value, torch.Tensor):
                setattr(s, name + "s", _array(value, n, dtype, name))
                on_current_device(value)
                kept.append(value)
            else:
                setattr(s, name, value)
        s._owner = tuple(kept)
        return s


def declare(L: ctypes.CDLL) -> None:
    vp, i = ctypes.c_void_p, ctypes.c_int
    L.ember_sample.argtypes, L.ember_sample.restype = [ctypes.POINTER(Sampler), vp, i, i, i, ctypes.c_int64, vp, vp, vp, vp], i


def sample(sampler: Sampler, logits, u, ids=None, probs=None, stream=None):
    """Draws one token per row of logits [n, V] (f32, f16 or bf16; rows may be apart) by u f32 [n] in [0, 1)
    (ember_sample); returns (ids int32 [n], probs f32 [n])."""
    import torch

    if logits.dim() != 2 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise em.EmberError(em.ERR_SHAPE, "logits: [n, V] with whole rows are needed")
    n, V = logits.shape
    if getattr(sampler, "_rows", None) is not None and sampler._rows < n:
        raise em.EmberError(em.ERR_SHAPE, f"settings of {sampler._rows} rows for {n}")
    here = on_current_device(logits, u, *getattr(sampler, "_owner", ()))
    if ids is None or probs is None:
        own_stream(stream, here, "ids and probs")
    if ids is None:
        ids = torch.empty(n, dtype=torch.int32, device=logits.device)
    if probs is None:
        probs = torch.empty(n, dtype=torch.float32, device=logits.device)
    stride = logits.stride(0) if n > 1 else max(logits.stride(0), V)
    a = (_array(u, n, torch.float32, "u"), _array(ids, n, torch.int32, "ids"), _array(probs, n, torch.float32, "probs"))
    on_current_device(ids, probs)
    st = em.lib().ember_sample(ctypes.byref(sampler), logits.data_ptr(), type_id(logits), n, V, stride, *a, em._stream(stream, here))
    if st:
        raise em.EmberError(st, "ember_sample")
    return ids, probs
