"""Helpers of the cache and attention tests: a batch of ragged sequences in a scattered paged cache, the plain
attention in 64 bits, and the bound on a kernel's error that its roundings add up to."""
import random

import numpy as np
import torch

import ember_moe as em

TORCH = {em.F32: torch.float32, em.F16: torch.float16, em.BF16: torch.bfloat16}


def quantise(x):
    """x [.., D] (torch, CPU) -> int8 codes, fp16 scales [.., D / 32], by the definition of include/ember_attn.h: the
    nearest code of the exact quotient by the stored scale, ties to even."""
    b = x.double().numpy().reshape(x.shape[:-1] + (-1, 32))
    with np.errstate(all="ignore"):
        q = np.abs(b).max(-1).astype(np.float32) / np.float32(127.0)  # (f32, as the scale is defined on f32 rows)
        d = np.where(q > 515.5, np.float32(515.5), q).astype(np.float16)
        dd = d.astype(np.float64)[..., None]
        code = np.where(dd > 0, np.clip(np.rint(b / np.where(dd > 0, dd, 1.0)), -127, 127), 0.0)
    code = np.nan_to_num(code)
    return torch.from_numpy(code.astype(np.int8)).reshape(x.shape), torch.from_numpy(d)


class Setup:
    """Sequences of (kv, q) tokens in a cache whose pages are scattered (page 0: one page per sequence), on the CPU; up() puts
    everything on the GPU. `behind`: rows after the last sequence's; `shared`: tokens that all sequences have in common."""

    def __init__(self, type_, seqs, n_kv, D, page, seed=0, shared=0, behind=0, spare=2, q_start=True):
        g = torch.Generator().manual_seed(seed)
        self.type, self.seqs, self.n_kv, self.D, self.shared = type_, seqs, n_kv, D, shared
        self.paged = page > 0
        self.page = page or max(1, max(kv for kv, _ in seqs))
        starts = [0]
        for _, q in seqs:
            starts.append(starts[-1] + q)
        self.starts, self.n = starts, starts[-1] + behind
        self.given_starts = q_start
        if self.paged:
            head = shared // self.page
            counts = [-(-kv // self.page) - (head if b else 0) for b, (kv, _) in enumerate(seqs)]
            self.n_pages = sum(max(c, 0) for c in counts) + spare
            order = list(range(self.n_pages))
            random.Random(seed).shuffle(order)
            width = max(1, max(-(-kv // self.page) for kv, _ in seqs))
            self.table = torch.zeros(len(seqs), width, dtype=torch.int32)
            for b, c in enumerate(counts):
                mine, order = order[:max(c, 0)], order[max(c, 0):]
                row = (self.table[0, :head].tolist() if b else []) + mine
                self.table[b, :len(row)] = torch.tensor(row, dtype=torch.int32)
        else:
            self.n_pages, self.table = len(seqs), None
        shape = (self.n_pages, n_kv, self.page, D)
        self.scales = (None, None)
        if type_ == em.Q8_0:
            self.k, self.v = (torch.randint(-127, 128, shape, generator=g, dtype=torch.int8) for _ in range(2))
            self.scales = tuple((torch.rand(*shape[:3], D // 32, generator=g) * 0.03 + 0.002).half() for _ in range(2))
        else:
            self.k, self.v = (torch.randn(*shape, generator=g).to(TORCH[type_]) for _ in range(2))
        self.g = g

    def place(self, b, j):
        """(page, row) of sequence b's position j."""
        return (int(self.table[b, j // self.page]), j % self.page) if self.paged else (b, j)

    def rows(self, b, which, lo=0, hi=None):
        """[n, n_kv, D] in 64 bits: positions lo .. hi - 1 of sequence b."""
        hi = self.seqs[b][0] if hi is None else hi
        x, sc = (self.k, self.v)[which], self.scales[which]
        j = torch.arange(lo, hi)
        p = self.table[b].long()[j // self.page] if self.paged else torch.full_like(j, b)
        out = x[p, :, j % self.page].double()
        return out if sc is None else out * sc[p, :, j % self.page].double().repeat_interleave(32, -1)

    def up(self):
        c = lambda t: None if t is None else t.cuda()  # noqa: E731
        self.cache = em.DeviceKvCache(self.type, c(self.k), c(self.v), c(self.scales[0]), c(self.scales[1]))
        self.kv_len = torch.tensor([kv for kv, _ in self.seqs], dtype=torch.int32).cuda()
        self.q_start = torch.tensor(self.starts, dtype=torch.int32).cuda() if self.given_starts else None
        self.batch = em.kv_batch(self.kv_len, self.q_start, n_tokens=self.n, max_q=max(1, max(q for _, q in self.seqs)),
                                 max_kv=max(kv for kv, _ in self.seqs), pages=c(self.table), shared=self.shared)
        return self


def plain_attention(s, q, H, scale, softcap=0.0, window=0, slopes=None, prefix=None, heads=None):
    """(out, bound) in 64 bits [n, H, D] for the rows q (CPU): the definition row by row, and what a kernel may be off by.

    The bound adds up, relative to A = sum p |v| / sum p: the rounding of the weights to the operand type (half a step); for Q8_0
    the rounding of a key's and a value's code * scale to fp16 (2^-11 each); scores in f32 (D products, each step 2^-24 of the sum of
    magnitudes, and the exponent's argument, a few 2^-24 of the largest score), where an error of ds in every score changes a weight by
    2 ds relatively; then the rounding of the result to its type. What a weight or a result that is subnormal in fp16 loses is
    absolute: 2^-25, of the weight's scale at least 2^8 below."""
    S, D = s, s.D
    G = H // S.n_kv
    out = torch.zeros(S.n, H, D, dtype=torch.float64)
    bound = torch.zeros_like(out)
    io = torch.finfo(q.dtype)
    op = 2.0 ** -8 if S.type == em.BF16 else 2.0 ** -11
    q8 = 2.0 ** -11 if S.type == em.Q8_0 else 0.0
    for b, (kv, nq) in enumerate(S.seqs):
        if nq == 0 or kv == 0:
            continue
        K, V = S.rows(b, 0), S.rows(b, 1)
        pos = torch.arange(kv - nq, kv)[:, None]
        j = torch.arange(kv)[None]
        seen = j <= pos
        if prefix is not None:
            seen = seen | (j < int(prefix[b]))
        if window:
            seen = seen & (pos - j < window)
        seen = seen & (pos >= 0)
        for h in heads if heads is not None else range(H):
            qq = q[S.starts[b]:S.starts[b] + nq, h].double()
            k, v = K[:, h // G], V[:, h // G]
            sc = scale * (qq @ torch.nan_to_num(k).t())
            mag = scale * (qq.abs() @ torch.nan_to_num(k).abs().t())
            hurt = torch.isfinite(k).all(1).logical_not()[None]  # keys that make a row NaN if it sees them
            if softcap:
                sc = softcap * torch.tanh(sc / softcap)
            if slopes is not None:
                sc = sc - float(slopes[h]) * (pos - j).abs()
            sc = sc.masked_fill(~seen, float("-inf"))
            top = sc.amax(1, keepdim=True) if kv else torch.zeros(nq, 1, dtype=torch.float64)
            top = torch.where(torch.isfinite(top), top, torch.zeros_like(top))
            w = torch.exp(sc - top)
            tot = w.sum(1, keepdim=True)
            w = torch.where(tot > 0, w / tot, torch.zeros_like(w))
            vz = torch.nan_to_num(v, nan=0.0, posinf=0.0, neginf=0.0)
            o, A = w @ vz, w @ vz.abs()
            big = torch.where(seen, sc.abs(), torch.zeros_like(sc)).amax(1, keepdim=True) if kv else top
            ds = torch.where(seen, mag, torch.zeros_like(mag)).amax(1, keepdim=True) * (q8 + (D + 8) * 2.0 ** -24) + (big + 16.0) * 2.0 ** -21
            e = A * (op + q8 + 2 * ds + 2.0 ** -16) + o.abs() * io.eps / 2 + 2.0 ** -24 * float(vz.abs().max() if kv else 0)
            bad = (hurt & seen).any(1, keepdim=True) | ((~torch.isfinite(v)).double()[None] * seen[:, :, None]).any(1)
            o = torch.where(bad.expand_as(o), torch.full_like(o, float("nan")), o)
            out[S.starts[b]:S.starts[b] + nq, h] = o
            bound[S.starts[b]:S.starts[b] + nq, h] = e
    return out, bound


def check(got, want, bound, what=""):
    got = got.double().cpu()
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan), (what, "NaN at other places", int((torch.isnan(got) != nan).sum()))
    off = torch.where(nan, torch.zeros_like(want), (got - want).abs())
    worst = (off / bound.clamp(min=1e-30)).max().item() if off.numel() else 0.0
    assert worst <= 1.0, (what, "error over its bound", worst, off.max().item())
    return worst
