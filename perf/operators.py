"""Operators of batched serving behind a shared prompt, with drafted tokens: what is measured.

    append     QK-norm and rotation of new tokens, their K and V written into a paged cache
    attention  causal attention of new tokens over the paged cache; a leading part of the positions
               may be shared by the whole batch
    probs      probabilities of rows of logits at a temperature
    verify     drafted tokens accepted or replaced against the target's probabilities, from given
               uniform numbers

`run` computes each in its plain form (torch, 32 bits) or, with `own`, through large_model_b200.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

EPS, ROPE_BASE = 1e-6, 1e6
# (q heads, kv heads, head size) of the framework's three model configurations
HEADS = {"235b": (64, 4, 128), "30b": (32, 4, 128), "tiny": (8, 2, 64)}
VOCAB = 151936


def listed():
    return [
        # one sequence decoding: the smallest append, a launch's latency
        dict(name="append one token", op="append", heads="235b", kv="f16", page=16, seqs=1, q=1, prefix=0, kv_new=1100, ragged=False),
        # 64 sequences, each with a token and up to four drafted ones, some idle
        dict(name="append drafts of 64", op="append", heads="235b", kv="f16", page=16, seqs=64, q=5, prefix=1024, kv_new=333, ragged=True),
        # prompts of different lengths entering the default fp32 cache
        dict(name="append prompts", op="append", heads="30b", kv="f32", page=64, seqs=9, q=500, prefix=0, kv_new=700, ragged=True),
        # one sequence decoding over the default fp32 cache
        dict(name="attend one token", op="attention", heads="235b", kv="f32", page=16, seqs=1, q=1, prefix=0, kv_new=1100, ragged=False),
        # the batched benchmark: 64 sequences behind one prompt of 1024 positions, a token each
        dict(name="attend 64 one prompt", op="attention", heads="235b", kv="f16", page=16, seqs=64, q=1, prefix=1024, kv_new=376, ragged=True),
        # the same behind a long prompt with four drafted tokens each: the largest
        dict(name="attend drafts long prompt", op="attention", heads="235b", kv="f16", page=64, seqs=64, q=5, prefix=8192, kv_new=640, ragged=False),
        # fp32 cache, an odd number of sequences and a prompt that ends inside a page, some idle
        dict(name="attend odd fp32", op="attention", heads="30b", kv="f32", page=16, seqs=23, q=3, prefix=1001, kv_new=701, ragged=True),
        # a chunk of a long prompt against what is cached
        dict(name="attend prompt chunk", op="attention", heads="235b", kv="f16", page=64, seqs=1, q=256, prefix=0, kv_new=4096, ragged=False),
        # one row of logits, as one sequence samples
        dict(name="probs one row", op="probs", rows=1, vocab=VOCAB, temp=0.8),
        # the rows that 64 sequences of five tokens produce
        dict(name="probs 320 rows", op="probs", rows=320, vocab=VOCAB, temp=0.8),
        # one sequence with tokens drafted by lookup (no draft probabilities)
        dict(name="verify one", op="verify", seqs=1, draft=4, vocab=VOCAB, with_q=False, ragged=False),
        # 64 sequences with a draft model's tokens and probabilities, drafts of different lengths
        dict(name="verify 64", op="verify", seqs=64, draft=4, vocab=VOCAB, with_q=True, ragged=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def _size(c):
    """What a case costs in its plain form: (values gathered from the cache, scores)."""
    H, Hk, D = HEADS[c["heads"]]
    n = c["prefix"] + c["kv_new"]
    return c["seqs"] * n * Hk * D, c["seqs"] * c["q"] * H * n


def draw(rng):
    op = rng.choice(["append", "append", "attention", "attention", "attention", "attention", "probs", "verify"])
    if op == "probs":
        return dict(op=op, rows=_log(rng, 1, 320), vocab=rng.choice([4096, 32003, VOCAB]), temp=rng.choice([0.6, 0.8, 1.0, 1.3]))
    if op == "verify":
        return dict(op=op, seqs=_log(rng, 1, 64), draft=rng.randint(1, 4), vocab=rng.choice([4096, 32003, VOCAB]), with_q=rng.random() < 0.5,
                    ragged=rng.random() < 0.5)
    most = _size(dict(heads="235b", seqs=64, q=5, prefix=8192, kv_new=640))
    if op == "append":
        most = (64 * 2048 * 4 * 128, most[1])       # the pools come back whole
    while True:
        seqs = _log(rng, 1, 64)
        q = rng.choice([1, 1, rng.randint(2, 8), _log(rng, 9, 512)])
        c = dict(op=op, heads=rng.choice(["235b", "30b", "tiny"]), kv=rng.choice(["f16", "f32"]), page=rng.choice([16, 32, 64, 128]), seqs=seqs, q=q,
                 prefix=rng.choice([0, _log(rng, 1, 8192)]), kv_new=q + _log(rng, 1, 8000), ragged=rng.random() < 0.6)
        if all(x <= y for x, y in zip(_size(c), most)):
            return c


# ---- lengths: from the case alone ------------------------------------------------------------------

def _lengths(c):
    """Per sequence: new tokens and positions in the cache with them. A ragged batch has idle sequences."""
    qs, kv = [], []
    for b in range(c["seqs"]):
        n = c["q"] if not c["ragged"] or b == 0 else (5 * b + 2) % (c["q"] + 1)
        qs.append(n)
        kv.append(c["prefix"] + (c["kv_new"] if not c["ragged"] or b == 0 else n + (7919 * b + 13) % (c["kv_new"] - n + 1)))
    return qs, kv


def _drafts(c):
    return [c["draft"] if not c["ragged"] or b == 0 else (3 * b + 1) % (c["draft"] + 1) for b in range(c["seqs"])]


def work(case):
    c = case
    if c["op"] == "probs":
        return {"bytes": 8 * c["rows"] * c["vocab"], "flops": 4 * c["rows"] * c["vocab"]}
    if c["op"] == "verify":
        # the row that the last token comes from, and the draft's where that token replaces one
        # (at most one of the two is read for a sequence whose drafts are all accepted)
        return {"bytes": c["seqs"] * c["vocab"] * (8 if c["with_q"] else 4), "flops": 3 * c["seqs"] * c["vocab"]}
    H, Hk, D = HEADS[c["heads"]]
    es = 2 if c["kv"] == "f16" else 4
    qs, kv = _lengths(c)
    if c["op"] == "append":
        return {"bytes": sum(qs) * D * (4 * (H + 2 * Hk) + 4 * H + 2 * Hk * es + 4), "flops": 10 * sum(qs) * (H + Hk) * D}
    rows = c["prefix"] + sum(n - c["prefix"] for n, t in zip(kv, qs) if t)
    pairs = sum(t * (n - t) + t * (t + 1) // 2 for n, t in zip(kv, qs))
    return {"bytes": rows * Hk * D * es * 2 + 8 * sum(qs) * H * D, "flops": 4 * pairs * H * D}


# ---- inputs -----------------------------------------------------------------------------------------

def _paged(c, seed):
    """A paged cache and a batch: the prompt's full pages are shared, every sequence has its own pages after them."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    H, Hk, D = HEADS[c["heads"]]
    P, dt = c["page"], torch.float16 if c["kv"] == "f16" else torch.float32
    qs, kv = _lengths(c)
    T, B, shared = sum(qs), c["seqs"], c["prefix"] // P
    need = [max(0, -(-n // P) - shared) for n in kv]
    order = np.random.default_rng(seed).permutation(shared + sum(need) + 3).astype(np.int32)    # three pages nobody uses
    table = np.zeros((B, max(1, shared + max(need))), np.int32)
    table[:, :shared] = order[:shared]
    at = shared
    for b in range(B):
        table[b, shared:shared + need[b]] = order[at:at + need[b]]
        at += need[b]
    table = torch.from_numpy(table).cuda()
    k = torch.randn((len(order), P, Hk, D), generator=g, device="cuda").to(dt)
    v = torch.randn((len(order), P, Hk, D), generator=g, device="cuda").to(dt)
    tail = c["prefix"] - shared * P
    if tail:                                        # the prompt ends inside a page: each sequence has a copy of its end
        k[table[:, shared].long(), :tail] = k[table[0, shared].long(), :tail].clone()
        v[table[:, shared].long(), :tail] = v[table[0, shared].long(), :tail].clone()
    start = torch.tensor([0] + np.cumsum(qs).tolist(), dtype=torch.int32, device="cuda")
    return g, dict(case=c, k=k, v=v, table=table, q_start=start, kv_len=torch.tensor(kv, dtype=torch.int32, device="cuda"), n_tok=T, max_q=max(qs), max_kv=max(kv))


def _rope(n, D):
    ang = np.arange(n)[:, None] * ROPE_BASE ** (-2.0 * np.arange(D // 2) / D)[None, :]
    return torch.from_numpy(np.cos(ang).astype(np.float32)).cuda(), torch.from_numpy(np.sin(ang).astype(np.float32)).cuda()


def prepare(case, seed):
    c = case
    if c["op"] in ("append", "attention"):
        g, s = _paged(c, seed)
        H, Hk, D = HEADS[c["heads"]]
        if c["op"] == "append":
            s["qkv"] = torch.randn((s["n_tok"], (H + 2 * Hk) * D), generator=g, device="cuda")
            s["q_norm"] = 1 + 0.2 * torch.randn((D,), generator=g, device="cuda")
            s["k_norm"] = 1 + 0.2 * torch.randn((D,), generator=g, device="cuda")
            s["cos"], s["sin"] = _rope(s["max_kv"], D)
        else:                                       # q as it leaves the norm: rows of length about sqrt(D)
            s["q"] = 1.2 * torch.randn((s["n_tok"], H * D), generator=g, device="cuda")
        s["out"] = torch.empty((s["n_tok"], H * D), device="cuda")
        return s
    g = torch.Generator(device="cuda").manual_seed(seed)
    if c["op"] == "probs":
        x = 2.5 * torch.randn((c["rows"], c["vocab"]), generator=g, device="cuda")
        return dict(case=c, logits=x, out=torch.empty_like(x))
    B, n, V = c["seqs"], c["draft"], c["vocab"]
    logits = 3.0 * torch.randn((B, n + 1, V), generator=g, device="cuda")
    p = torch.softmax(logits, -1)
    q = torch.softmax(logits[:, :n] + 0.7 * torch.randn((B, n, V), generator=g, device="cuda"), -1)
    # a draft model draws from its own probabilities; a lookup proposes a token of some weight
    race = (q if c["with_q"] else p[:, :n].sqrt()) / torch.empty((B, n, V), device="cuda").exponential_(generator=g)
    return dict(case=c, p=p.view(B * (n + 1), V), q=q.contiguous() if c["with_q"] else None, draft=race.argmax(-1).int(),
                n_draft=torch.tensor(_drafts(c), dtype=torch.int32, device="cuda"), u=torch.rand((B, n + 1), generator=g, device="cuda"),
                n_accept=torch.empty((B,), dtype=torch.int32, device="cuda"), tokens=torch.empty((B, n + 1), dtype=torch.int32, device="cuda"))


# ---- plain forms ------------------------------------------------------------------------------------

def _where(s):
    """Per new token: its sequence, its index there and its position."""
    t = torch.arange(s["n_tok"], device="cuda")
    b = (t[:, None] >= s["q_start"][None, 1:]).sum(1)
    i = t - s["q_start"][b]
    n = s["q_start"][b + 1] - s["q_start"][b]
    return b, i, s["kv_len"][b] - n + i


def _append_plain(s):
    c = s["case"]
    H, Hk, D = HEADS[c["heads"]]
    b, _, pos = _where(s)
    x = s["qkv"].view(-1, H + 2 * Hk, D)
    qk = x[:, :H + Hk]
    qk = qk / torch.sqrt((qk * qk).mean(-1, keepdim=True) + EPS)
    qk = qk * torch.cat([s["q_norm"].expand(H, D), s["k_norm"].expand(Hk, D)])
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    lo, hi = qk[..., :D // 2], qk[..., D // 2:]
    qk = torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1)
    page, off = s["table"][b, pos // c["page"]].long(), pos % c["page"]
    s["k"][page, off] = qk[:, H:].to(s["k"].dtype)
    s["v"][page, off] = x[:, H + Hk:].to(s["v"].dtype)
    return qk[:, :H].reshape(s["n_tok"], H * D), s["k"], s["v"]


def _attention_plain(s):
    c = s["case"]
    H, Hk, D = HEADS[c["heads"]]
    B, Q, G = c["seqs"], s["max_q"], H // Hk
    k, v = (s[x][s["table"].long()].flatten(1, 2).float().transpose(1, 2) for x in "kv")        # [B, Hk, L, D]
    at = torch.arange(k.shape[2], device="cuda")
    i = torch.arange(Q, device="cuda")
    n = s["q_start"][1:] - s["q_start"][:-1]
    rows = (s["q_start"][:-1, None] + i).clamp(max=max(0, s["n_tok"] - 1))
    q = s["q"].view(-1, Hk, G, D)[rows].permute(0, 2, 1, 3, 4).reshape(B, Hk, Q * G, D)
    pos = torch.where(i < n[:, None], s["kv_len"][:, None] - n[:, None] + i, -1)                # [B, Q]
    seen = (at <= pos[:, :, None]).repeat_interleave(G, 1)[:, None]                             # [B, 1, Q * G, L]
    x = torch.where(seen, q @ k.transpose(2, 3) * (1 / math.sqrt(D)), -math.inf)
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    o = e @ torch.where((at < s["kv_len"][:, None])[:, None, :, None], v, 0.0) / e.sum(-1, keepdim=True)
    b, i, _ = _where(s)
    return o.view(B, Hk, Q, G, D).permute(0, 2, 1, 3, 4)[b, i].reshape(s["n_tok"], H * D)


def _probs_plain(s):
    x = s["logits"] / s["case"]["temp"]
    e = torch.exp(x - x.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


def _verify_plain(s):
    c = s["case"]
    B, n, V = c["seqs"], c["draft"], c["vocab"]
    p, draft, i = s["p"].view(B, n + 1, V), s["draft"].long(), torch.arange(n, device="cuda")
    px = p[:, :n].gather(2, draft[..., None])[..., 0]
    qx = s["q"].gather(2, draft[..., None])[..., 0] if c["with_q"] else torch.ones_like(px)
    ok = (s["u"][:, :n] * qx < px) & (i < s["n_draft"][:, None])
    took = ok.int().cumprod(1).sum(1)                                                           # [B]
    b, last = torch.arange(B, device="cuda"), took.clamp(max=n - 1)
    row = p[b, took]
    replaced = (took < s["n_draft"])[:, None]
    if c["with_q"]:
        rest = row - torch.where(replaced, s["q"][b, last], 0.0)
    else:
        rest = torch.where(replaced & (torch.arange(V, device="cuda") == draft[b, last][:, None]), 0.0, row)
    # weights in units of 2^-40: their sums are whole numbers, the same in any order
    whole = lambda x: (torch.where(x > 0, x, 0.0).clamp(max=1.0) * 2.0 ** 40).round().long()    # noqa: E731
    w = whole(rest)
    w = torch.where(w.sum(1, keepdim=True) > 0, w, whole(row))
    total, u = w.sum(1), (s["u"][:, n] * 2.0 ** 24).floor().long()
    want = (total >> 24) * u + (((total & 0xFFFFFF) * u) >> 24)                                 # floor(total u / 2^24)
    pick = torch.searchsorted(w.cumsum(1), want[:, None], right=True)[:, 0]
    j = torch.arange(n + 1, device="cuda")
    kept = torch.where(j[:n] < took[:, None], draft, -1)
    tokens = torch.where(j == took[:, None], pick[:, None], torch.cat([kept, torch.full((B, 1), -1, device="cuda")], 1))
    return took.int(), tokens.int()


_PLAIN = {"append": _append_plain, "attention": _attention_plain, "probs": _probs_plain, "verify": _verify_plain}


# ---- the framework's calls ----------------------------------------------------------------------------

def _handles(s):
    """The cache's and the batch's descriptors, which a program keeps beside its buffers."""
    import large_model_b200 as m
    if "pages" not in s:
        s["pages"] = m.KvPages(s["k"], s["v"])
        s["batch"] = m.PagedBatch(s["q_start"], s["kv_len"], s["table"], s["n_tok"], s["max_q"], s["max_kv"], s["case"]["prefix"])
    return m, s["pages"], s["batch"], HEADS[s["case"]["heads"]][0]


def _append_own(s):
    m, pages, batch, H = _handles(s)
    return m.paged_append(pages, batch, s["qkv"], H, s["q_norm"], s["k_norm"], EPS, (s["cos"], s["sin"]), q=s["out"]), s["k"], s["v"]


def _attention_own(s):
    m, pages, batch, H = _handles(s)
    return m.paged_attention(pages, batch, s["q"], H, out=s["out"])


def _probs_own(s):
    import large_model_b200 as m
    return m.probs(s["logits"], s["case"]["temp"], out=s["out"])


def _verify_own(s):
    import large_model_b200 as m
    return m.verify(s["p"], s["draft"], s["u"], q=s["q"], n_draft=s["n_draft"], n_accept=s["n_accept"], tokens=s["tokens"])


_OWN = {"append": _append_own, "attention": _attention_own, "probs": _probs_own, "verify": _verify_own}


def run(state):
    return (_OWN if own else _PLAIN)[state["case"]["op"]](state)


# ---- from the definitions, in 64 bits -----------------------------------------------------------------

def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["op"] == "verify":
        return None                                 # whole numbers
    if c["op"] == "probs":
        x = s["logits"].double() / c["temp"]
        return torch.stack([torch.exp(r - torch.logsumexp(r, 0)) for r in x])
    H, Hk, D = HEADS[c["heads"]]
    qs, kv = _lengths(c)
    ends = np.cumsum(qs)
    if c["op"] == "append":
        k, v, out = s["k"].double(), s["v"].double(), torch.empty((s["n_tok"], H, D), dtype=torch.float64, device="cuda")
        turn = ROPE_BASE ** (-2.0 * torch.arange(D // 2, dtype=torch.float64, device="cuda") / D)
        for b, (n, end, t1) in enumerate(zip(qs, kv, ends)):
            x = s["qkv"][t1 - n:t1].double().view(n, H + 2 * Hk, D)
            at = torch.arange(end - n, end, device="cuda")
            z = torch.polar(torch.ones(n, D // 2, dtype=torch.float64, device="cuda"), at[:, None].double() * turn)[:, None]

            def turned(y, w):
                y = y * torch.rsqrt(y.pow(2).mean(-1, keepdim=True) + EPS) * w.double()
                r = torch.complex(y[..., :D // 2].contiguous(), y[..., D // 2:].contiguous()) * z
                return torch.cat([r.real, r.imag], -1)
            out[t1 - n:t1] = turned(x[:, :H], s["q_norm"])
            page = s["table"][b, at // c["page"]].long()
            k[page, at % c["page"]] = turned(x[:, H:H + Hk], s["k_norm"])
            v[page, at % c["page"]] = x[:, H + Hk:]
        return out.view(s["n_tok"], H * D), k, v
    out = torch.zeros((s["n_tok"], H, D), dtype=torch.float64, device="cuda")
    for b, (n, end, t1) in enumerate(zip(qs, kv, ends)):
        if n == 0:
            continue
        at = torch.arange(end, device="cuda")
        page = s["table"][b, at // c["page"]].long()
        k, v = (s[x][page, at % c["page"]].double() for x in "kv")                              # [end, Hk, D]
        q = s["q"][t1 - n:t1].double().view(n, Hk, H // Hk, D)
        late = at > torch.arange(end - n, end, device="cuda")[:, None]
        for h in range(Hk):
            x = torch.einsum("igd,jd->gij", q[:, h], k[:, h]) / math.sqrt(D)
            w = torch.softmax(x.masked_fill(late, -math.inf), -1)
            out[t1 - n:t1, h * (H // Hk):(h + 1) * (H // Hk)] = torch.einsum("gij,jd->igd", w, v[:, h])
    return out.view(s["n_tok"], H * D)
