"""The operators of a decode step around the MoE layer, as cases to be timed: K and V rows stored into a paged cache and
read back (`ember_kv_store`, `ember_kv_load`), attention over that cache for prompts and single tokens (`ember_attn`), the
same where a batch shares its first pages, and the pick of the next token and its probability (`ember_sample`); each beside its plain form in
elementary torch operations.

A case: `op` (store, load, attn, sample), and for the first three the cache's `type`, `io` (the type of q, k, v and the
outputs), KV heads, head width, page size (0: one page per sequence), the sequences: `seqs` of them, the longest with `kv`
tokens in the cache of which `q` are new; `ragged` 0 makes all alike, other values draw the lengths. `shared` tokens at
their head lie in the same pages."""
import math
import os
import random
import sys

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    mixtral = dict(heads=32, n_kv=8, dim=128)  # the attention of the end-to-end model
    return [
        # a server's decode step: one new token of each of 64 sequences into their quantised pages, and back
        dict(name="store_step", op="store", type="q8_0", io="bf16", n_kv=8, dim=128, page=64, seqs=64, kv=4000, q=1, ragged=1),
        # prompts of a batch, as they are prefilled together; a page size that no tile divides
        dict(name="store_prompts", op="store", type="q8_0", io="f16", n_kv=8, dim=128, page=48, seqs=9, kv=4000, q=4000, ragged=2),
        # whole sequences read back, to be moved to other pages
        dict(name="load_long", op="load", type="q8_0", io="bf16", n_kv=8, dim=128, page=64, seqs=5, kv=20000, q=20000, ragged=3),
        # the end-to-end model's decode: one user, the 512-token prompt and what was generated, a plain contiguous cache
        dict(name="attn_token", op="attn", type="bf16", io="bf16", page=0, seqs=1, kv=640, q=1, ragged=0, **mixtral),
        # a server's decode step over quantised pages
        dict(name="attn_step_q8", op="attn", type="q8_0", io="bf16", page=64, seqs=48, kv=6000, q=1, ragged=4, **mixtral),
        # one user deep in a long document
        dict(name="attn_token_long", op="attn", type="bf16", io="bf16", page=256, seqs=1, kv=131000, q=1, ragged=0, **mixtral),
        # a long prompt: the matrix cores' case
        dict(name="attn_prompt", op="attn", type="bf16", io="bf16", page=128, seqs=1, kv=8192, q=8192, ragged=0, **mixtral),
        # ragged prompts through every score option
        dict(name="attn_prompts_capped", op="attn", type="f16", io="f16", heads=16, n_kv=4, dim=64, page=64, seqs=7, kv=1500, q=1500,
             ragged=5, cap=30.0, window=1024, slopes=True, prefix=200),
        # a few answers to one short prompt
        dict(name="shared_few", op="attn", type="bf16", io="bf16", page=64, seqs=8, kv=640, q=1, ragged=6, shared=512, **mixtral),
        # many users behind one long system prompt
        dict(name="shared_many", op="attn", type="q8_0", io="bf16", page=64, seqs=96, kv=8900, q=1, ragged=7, shared=8192, **mixtral),
        # one user's next token at the end-to-end model's vocabulary
        dict(name="sample_one", op="sample", io="f32", rows=1, vocab=32000, temperature=0.8, top_k=0, top_p=0.95, min_p=0.0),
        # a server's step at a large vocabulary, every filter
        dict(name="sample_batch", op="sample", io="f32", rows=128, vocab=131072, temperature=1.0, top_k=1000, top_p=0.9, min_p=0.02),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["store", "load", "step", "step", "prompt", "prompt", "shared", "sample", "sample"])
    if kind == "sample":
        rows = _log(rng, 1, 256)
        return dict(op="sample", io=rng.choice(["f32", "f32", "bf16", "f16"]), rows=rows, vocab=_log(rng, 50, min(160000, (1 << 24) // rows)),
                    temperature=round(rng.uniform(0.3, 1.6), 3), top_k=rng.choice([0, 1, 40, _log(rng, 2, 20000)]),
                    top_p=rng.choice([1.0, round(rng.uniform(0.2, 0.99), 3)]), min_p=rng.choice([0.0, round(rng.uniform(0.001, 0.3), 4)]))
    t = rng.choice(["f16", "bf16", "q8_0", "q8_0"])
    io = t if t != "q8_0" else rng.choice(["f16", "bf16"])
    c = dict(op="attn", type=t, io=io, n_kv=rng.choice([1, 2, 4, 8]), dim=rng.choice([64, 64, 96, 128, 128, 128, 160, 256]), page=rng.choice([0, 16, 48, 64, 100, 256]),
             ragged=rng.randrange(1, 1 << 20))
    if kind in ("store", "load"):
        c["op"] = kind
        c["seqs"] = _log(rng, 1, 64)
        c["kv"] = _log(rng, 1, 40000 // c["seqs"])
        c["q"] = c["kv"] if kind == "load" or rng.random() < 0.5 else rng.randrange(1, c["kv"] + 1)
        return c
    c["heads"] = c["n_kv"] * rng.choice([1, 2, 4, 4, 8] if c["n_kv"] < 8 else [1, 2, 4])
    if kind == "step":
        c["seqs"] = _log(rng, 1, 96)
        c["kv"] = _log(rng, 1, min(60000, 200000 // c["seqs"]))
        c["q"] = min(c["kv"], rng.choice([1, 1, 1, 2, 5]))
    elif kind == "prompt":
        c["seqs"] = _log(rng, 1, 8)
        c["kv"] = _log(rng, 2, 5000 // c["seqs"])
        c["q"] = c["kv"] if rng.random() < 0.6 else rng.randrange(1, c["kv"] + 1)
    else:
        c["page"] = rng.choice([16, 48, 64, 256])
        c["seqs"] = _log(rng, 2, 96)
        c["shared"] = c["page"] * _log(rng, 1, 6000 // c["page"])
        c["kv"] = c["shared"] + _log(rng, 1, 500)
        c["q"] = 1
    if rng.random() < 0.4:
        c["cap"] = rng.choice([20.0, 50.0])
    if rng.random() < 0.4:
        c["window"] = _log(rng, 1, 3000)
    if rng.random() < 0.3:
        c["slopes"] = True
    if kind != "shared" and rng.random() < 0.3:
        c["prefix"] = rng.randrange(1, c["kv"] + 1)
    return c


# ---- a case's sequences, by the case alone

def _sequences(case):
    """Per sequence (tokens in the cache, new tokens among them): the first the longest, the others between a tenth of it and it."""
    rng, got = random.Random(case["ragged"]), []
    for b in range(case["seqs"]):
        kv, q = case["kv"], case["q"]
        if case["ragged"] and b:
            low = case.get("shared", 0)
            kv = low + rng.randint(max(1, (kv - low) // 10), kv - low)
            q = kv if case["q"] == case["kv"] else min(kv, rng.randint(max(1, q // 2), q))
        got.append((kv, q))
    return got


def _page(case):
    return case["page"] or case["kv"]


def _values(case):
    """Values of K (and as many of V) that the new tokens hold."""
    return sum(q for _, q in _sequences(case)) * case["n_kv"] * case["dim"]


def _visible(case, kv, q):
    """(pairs of a new token and a key that it sees, keys that any of them sees) of one sequence."""
    window, prefix = case.get("window", 0), case.get("prefix", 0)
    pairs, first, last = 0, kv, 0
    for p in range(kv - q, kv):
        lo = max(0, p - window + 1) if window else 0
        hi = min(kv, max(p + 1, prefix))
        pairs += max(0, hi - lo)
        first, last = min(first, lo), max(last, hi)
    return pairs, max(0, last - first)


def work(case):
    if case["op"] == "sample":
        size = 4 if case["io"] == "f32" else 2
        return {"bytes": case["rows"] * (case["vocab"] * size + 4 + 8), "flops": case["rows"] * case["vocab"] * 20.0}
    held = {"q8_0": 34 / 32}.get(case["type"], 2.0)  # bytes of a value in the cache
    if case["op"] == "store":  # rows in, into the cache, out of the cache, rows out
        return {"bytes": 2 * _values(case) * (2 + held + held + 2), "flops": 6.0 * _values(case)}
    if case["op"] == "load":
        return {"bytes": 2 * _values(case) * (held + 2), "flops": 2.0 * _values(case)}
    pairs = keys = new = 0
    shared = case.get("shared", 0)
    for b, (kv, q) in enumerate(_sequences(case)):
        p, k = _visible(case, kv, q)
        new += q
        pairs += p
        keys += k if b == 0 else max(0, min(k, kv - shared))
    return {"bytes": 2 * keys * case["n_kv"] * case["dim"] * held + 4 * new * case["heads"] * case["dim"],
            "flops": 4.0 * pairs * case["heads"] * case["dim"]}


# ---- inputs

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(1000003 * (seed + 1))

    def normal(*n, std=1.0, dtype=torch.float32):
        return (torch.randn(*n, generator=g, device="cuda", dtype=torch.float32) * std).to(dtype)

    if case["op"] == "sample":
        n = case["rows"]
        # a model's logits: a bell with a few tokens far above it
        z = normal(n, case["vocab"], std=2.0)
        z += 6.0 * (torch.rand(z.shape, generator=g, device="cuda") < 12.0 / case["vocab"])
        return dict(case=case, z=z.to(TYPES[case["io"]]), u=torch.rand(n, generator=g, device="cuda"))
    io, D, n_kv, page = TYPES[case["io"]], case["dim"], case["n_kv"], _page(case)
    seqs = _sequences(case)
    q_start = [0]
    for _, q in seqs:
        q_start.append(q_start[-1] + q)
    n = q_start[-1]
    # every sequence's pages, scattered over the cache; the shared ones are the first sequence's
    table = None
    n_pages = len(seqs)
    if case["page"]:
        wide, head = -(-max(kv for kv, _ in seqs) // page), case.get("shared", 0) // page
        own_pages = [-(-kv // page) - (head if b else 0) for b, (kv, _) in enumerate(seqs)]
        n_pages = sum(own_pages) + 1
        order = list(range(n_pages))
        random.Random(seed).shuffle(order)
        rows = []
        for b, m in enumerate(own_pages):
            mine, order = order[:m], order[m:]
            row = (rows[0][:head] if b else []) + mine
            rows.append(row + [0] * (wide - len(row)))
        table = torch.tensor(rows, dtype=torch.int32, device="cuda")
    s = dict(case=case, n=n, table=table, n_pages=n_pages, q_start=torch.tensor(q_start, dtype=torch.int32, device="cuda"),
             kv_len=torch.tensor([kv for kv, _ in seqs], dtype=torch.int32, device="cuda"),
             max_q=max(q for _, q in seqs), max_kv=max(kv for kv, _ in seqs))
    shape = (n_pages, n_kv, page, D)
    if case["type"] == "q8_0":
        for name in ("k", "v"):
            s[name] = torch.randint(-127, 128, shape, generator=g, device="cuda", dtype=torch.int8)
            s[name + "_scale"] = (torch.rand(*shape[:3], D // 32, generator=g, device="cuda") * 0.02 + 0.005).half()
    else:
        s["k"], s["v"] = (normal(*shape, dtype=TYPES[case["type"]]) for _ in range(2))
    if case["op"] == "store":
        s["k_new"], s["v_new"] = (normal(n, n_kv, D, dtype=io) for _ in range(2))
    if case["op"] == "attn":
        s["q"] = normal(n, case["heads"], D, std=2.0, dtype=io)
        if case.get("slopes"):
            s["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / case["heads"]) for h in range(case["heads"])], device="cuda")
        if case.get("prefix"):
            s["prefix"] = torch.full((len(seqs),), case["prefix"], dtype=torch.int32, device="cuda")
    return s


# ---- the framework's calls

def _em():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ember.cpp_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import ember_moe

    return ember_moe


def _plan(s):
    """The descriptors and buffers that a program keeps beside its cache."""
    em, case = _em(), s["case"]
    if case["op"] == "sample":
        smp = em.Sampler(temperature=case["temperature"], top_k=case["top_k"], top_p=case["top_p"], min_p=case["min_p"])
        ids, probs = (torch.empty(case["rows"], dtype=t, device="cuda") for t in (torch.int32, torch.float32))
        return dict(em=em, sampler=smp, ids=ids, probs=probs)
    cache = em.DeviceKvCache(em.TYPE_IDS[case["type"]], s["k"], s["v"], s.get("k_scale"), s.get("v_scale"))
    batch = em.kv_batch(s["kv_len"], q_start=s["q_start"], n_tokens=s["n"], max_q=s["max_q"], max_kv=s["max_kv"], pages=s["table"],
                        shared=case.get("shared", 0))
    p = dict(em=em, cache=cache, batch=batch)
    if case["op"] == "attn":
        p["attn"] = em.attn_options(case["heads"], case["dim"], softcap=case.get("cap", 0.0), window=case.get("window", 0),
                                    slopes=s.get("slopes"), prefix=s.get("prefix"))
        p["out"] = torch.empty_like(s["q"])
        p["scratch"] = torch.empty(max(1, cache.attn_scratch_bytes(p["attn"], batch)), dtype=torch.uint8, device="cuda")
    else:
        shape = (s["n"], case["n_kv"], case["dim"])
        p["k"], p["v"] = (torch.empty(shape, dtype=TYPES[case["io"]], device="cuda") for _ in range(2))
    return p


def _run_own(s):
    if "plan" not in s:
        s["plan"] = _plan(s)
    p, op = s["plan"], s["case"]["op"]
    if op == "sample":
        return p["em"].sample(p["sampler"], s["z"], s["u"], p["ids"], p["probs"])
    if op == "attn":
        return p["cache"].attend(p["attn"], p["batch"], s["q"], p["out"], p["scratch"])
    if op == "store":
        p["cache"].store(p["batch"], s["k_new"], s["v_new"])
    return p["cache"].load(p["batch"], p["k"], p["v"])


# ---- the plain forms

def _places(s):
    """Sequence, position, page and row in the page of every new token."""
    tok = torch.arange(s["n"], device="cuda")
    b = torch.searchsorted(s["q_start"][1:].long(), tok, right=True)
    pos = s["kv_len"].long()[b] - s["q_start"].long()[b + 1] + tok
    page = _page(s["case"])
    pid = b if s["table"] is None else s["table"].long()[b, pos // page]
    return b, pos, pid, pos % page


def _quantise(x):
    """[.., D] -> codes and fp16 scales of its blocks of 32: the nearest code of each value at the stored scale."""
    b = x.float().unflatten(-1, (-1, 32))
    d = (b.abs().amax(-1) / 127.0).clamp(max=515.5).half()
    dd = d.double().unsqueeze(-1)
    code = torch.where(dd > 0, torch.round(b.double() / torch.where(dd > 0, dd, torch.ones_like(dd))), torch.zeros_like(dd)).clamp(-127, 127)
    return code.to(torch.int8).flatten(-2), d


def _held(codes, scale):
    return codes.float() if scale is None else (codes.float().unflatten(-1, (-1, 32)) * scale.float().unsqueeze(-1)).flatten(-2)


def _store(s):
    _, _, pid, row = _places(s)
    for name in ("k", "v"):
        x = s[name + "_new"]
        if s["case"]["type"] == "q8_0":
            codes, d = _quantise(x)
            s[name][pid, :, row] = codes
            s[name + "_scale"][pid, :, row] = d
        else:
            s[name][pid, :, row] = x.to(s[name].dtype)


def _load(s):
    _, _, pid, row = _places(s)
    io = TYPES[s["case"]["io"]]
    return tuple(_held(s[n][pid, :, row], s[n + "_scale"][pid, :, row] if n + "_scale" in s else None).to(io) for n in ("k", "v"))


def _attend(s):
    case = s["case"]
    H, n_kv, D = case["heads"], case["n_kv"], case["dim"]
    G, B, L, Q, page = H // n_kv, case["seqs"], s["max_kv"], s["max_q"], _page(case)
    j = torch.arange(L, device="cuda")
    pid = torch.arange(B, device="cuda")[:, None].expand(B, L) if s["table"] is None else s["table"].long()[:, j // page]
    row = (j % page).expand(B, L)

    def rows(name):  # [B, n_kv, L, D] in 32 bits
        sc = s[name + "_scale"][pid, :, row] if name + "_scale" in s else None
        return _held(s[name][pid, :, row], sc).transpose(1, 2)

    b, pos, _, _ = _places(s)
    i = torch.arange(s["n"], device="cuda") - s["q_start"].long()[b]
    q = torch.zeros(B, Q, H, D, device="cuda")
    q[b, i] = s["q"].float()
    p = torch.full((B, Q), -1, device="cuda")
    p[b, i] = pos
    q = q.view(B, Q, n_kv, G, D).permute(0, 2, 3, 1, 4).reshape(B, n_kv, G * Q, D)
    sc = torch.matmul(q, rows("k").transpose(2, 3)).view(B, n_kv, G, Q, L)
    sc.mul_(1.0 / math.sqrt(D))
    if case.get("cap"):
        sc.div_(case["cap"]).tanh_().mul_(case["cap"])
    far = j - p[:, :, None]  # [B, Q, L]
    if case.get("slopes"):
        sc -= s["slopes"].view(n_kv, G, 1, 1) * far[:, None, None].abs().float()
    seen = far <= 0
    if case.get("prefix"):
        seen |= j < s["prefix"].long()[:, None, None]
    seen &= (j < s["kv_len"].long()[:, None, None]) & (p >= 0)[:, :, None]
    if case.get("window"):
        seen &= far > -case["window"]
    sc.masked_fill_(~seen[:, None, None], float("-inf"))
    top = sc.amax(-1, keepdim=True)
    w = torch.exp_(sc.sub_(torch.where(top == float("-inf"), torch.zeros_like(top), top)))
    total = w.sum(-1, keepdim=True)
    o = torch.matmul(w.view(B, n_kv, G * Q, L), rows("v")).view(B, n_kv, G, Q, D)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    return o.permute(0, 3, 1, 2, 4).reshape(B, Q, H, D)[b, i].to(TYPES[case["io"]])


def _sample(s):
    case, V = s["case"], s["case"]["vocab"]
    z = s["z"].double()
    order = torch.sort(z, dim=1, descending=True, stable=True).indices
    x = torch.gather(z, 1, order)
    w = torch.exp((x - x[:, :1]) / float(torch.tensor(case["temperature"], dtype=torch.float32)))
    if 0 < case["top_k"] < V:
        w[:, case["top_k"]:] = 0.0
    before = torch.cumsum(w, 1) - w
    kept = w > 0
    if case["top_p"] < 1.0:
        kept &= before < float(torch.tensor(case["top_p"], dtype=torch.float32)) * w.sum(1, keepdim=True)
    kept &= w >= float(torch.tensor(case["min_p"], dtype=torch.float32))
    w = torch.zeros_like(w).scatter_(1, order, torch.where(kept, w, torch.zeros_like(w)))
    c = torch.cumsum(w, 1)
    ids = (c <= s["u"].double()[:, None] * c[:, -1:]).sum(1, keepdim=True)
    return ids[:, 0].to(torch.int32), (torch.gather(w, 1, ids) / c[:, -1:])[:, 0].float()


def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    if op == "sample":
        return _sample(state)
    if op == "attn":
        return _attend(state)
    if op == "store":
        _store(state)
    return _load(state)


# ---- the definitions in 64 bits, a sequence (or row) at a time

def _exact_sample(s):
    case, ids, probs = s["case"], [], []
    T, top_p, min_p = (float(torch.tensor(case[n], dtype=torch.float32)) for n in ("temperature", "top_p", "min_p"))
    for z, u in zip(s["z"].double(), s["u"].double().tolist()):
        V = z.numel()
        rank = torch.argsort(-z, stable=True)
        e = torch.exp((z[rank] - z.max()) / T)
        k = case["top_k"] if 0 < case["top_k"] < V else V
        e = e[:k]
        run_ = torch.cumsum(e, 0)
        n = k if top_p >= 1.0 else min(k, int(torch.searchsorted(run_, top_p * run_[-1]).item()) + 1)
        n = min(n, int((e >= max(min_p, 1e-300)).sum()))
        places, at = torch.sort(rank[:n])
        c = torch.cumsum(e[:n][at], 0)
        drawn = int(torch.searchsorted(c, (u * c[-1]).reshape(1), right=True))
        ids.append(int(places[drawn]))
        probs.append(float(e[at[drawn]] / c[-1]))
    return torch.tensor(ids, dtype=torch.int32), torch.tensor(probs, dtype=torch.float64)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "sample":
        return _exact_sample(s)
    n_kv, D, page = case["n_kv"], case["dim"], _page(case)
    out_k, out_v, out = [], [], []
    at = 0

    def cached(name, b, lo, hi):  # [hi - lo, n_kv, D] of sequence b, page by page
        parts = []
        for first in range(lo // page * page, hi, page):
            pid = b if s["table"] is None else table[b][first // page]
            x = s[name][pid].double()
            if name + "_scale" in s:
                x = x * s[name + "_scale"][pid].double().repeat_interleave(32, dim=-1)
            parts.append(x[:, max(lo - first, 0):min(page, hi - first)])
        return torch.cat(parts, 1).transpose(0, 1)

    def codes(x):  # the values that the quantised rows stand for
        b = x.double().reshape(x.shape[0], n_kv, D // 32, 32)
        d = torch.minimum(b.abs().max(-1, keepdim=True).values / 127, torch.tensor(515.5, dtype=torch.float64, device="cuda")).half().double()
        t = b.abs() / d
        low = torch.floor(t)
        up = (t - low > 0.5) | ((t - low == 0.5) & (low % 2 == 1))
        return (torch.sign(b) * torch.clamp(low + up, max=127) * d).reshape(x.shape)

    table = None if s["table"] is None else s["table"].tolist()
    for b, (kv, q) in enumerate(_sequences(case)):
        if case["op"] == "store":
            for name, to in (("k_new", out_k), ("v_new", out_v)):
                x = s[name][at:at + q]
                to.append(codes(x) if case["type"] == "q8_0" else x.double())
        elif case["op"] == "load":
            out_k.append(cached("k", b, kv - q, kv))
            out_v.append(cached("v", b, kv - q, kv))
        else:
            K, Vv = cached("k", b, 0, kv), cached("v", b, 0, kv)
            pos = torch.arange(kv - q, kv, device="cuda")[:, None]
            key = torch.arange(kv, device="cuda")[None]
            gap = pos - key
            hide = (gap < 0) & (key >= case.get("prefix", 0))
            if case.get("window"):
                hide = hide | (gap >= case["window"])
            heads = []
            for h in range(case["heads"]):
                kv_head = h // (case["heads"] // n_kv)
                a = s["q"][at:at + q, h].double() @ K[:, kv_head].t().contiguous() / math.sqrt(D)
                if case.get("cap"):
                    a = case["cap"] * torch.tanh(a / case["cap"])
                if case.get("slopes"):
                    a = a - float(s["slopes"][h]) * gap.abs()
                a = torch.softmax(a.masked_fill(hide, float("-inf")), -1)
                heads.append(torch.nan_to_num(a) @ Vv[:, kv_head].contiguous())
            out.append(torch.stack(heads, 1))
        at += q
    return torch.cat(out) if case["op"] == "attn" else (torch.cat(out_k), torch.cat(out_v))
