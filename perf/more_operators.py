"""Operators of long prompts and small caches: what is measured.

    prompt     causal attention over whole prompts, packed one after another, in 16 bits
    append     QK-norm and rotation of new tokens, their K and V written into a cache held in 4 bits
               (and, for prompts, the heads' rows in 16 bits, as the prompt attention reads them)
    attend     causal attention of new tokens over a paged cache held in 4 bits
    logprobs   log probabilities of given tokens, with the entropy of their row and its likeliest tokens

`run` computes each in its plain form (torch, 32 or 64 bits) or, with `own`, through large_model_b200.

A cache in 4 bits: 32 values x of a K or V row have one scale d, the value of largest magnitude (the first of
equals) over -8, rounded to 8 significant bits, so that every value it stands for is exact in fp16; x is held as
n = floor(x / d + 8.5), 0 .. 15, and read back as d (n - 8). Of a page and kv head lie first the positions'
n, head_dim / 2 bytes each, value i of 8 in bits 4 (i / 2) + 16 (i % 2) of a 32-bit word, then their scales, fp16.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

EPS, ROPE_BASE = 1e-6, 1e6
# (q heads, kv heads, head size) of the framework's three model configurations
HEADS = {"235b": (64, 4, 128), "30b": (32, 4, 128), "tiny": (8, 2, 64)}
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
VOCAB = 151936
SHIFTS = (0, 16, 4, 20, 8, 24, 12, 28)          # of the 8 values in a word of the cache


def listed():
    return [
        # one short prompt, before its first token can be drawn: latency
        dict(name="prompt short", op="prompt", heads="235b", type="f16", seqs=1, longest=100, ragged=False, pad=0),
        # prompts of different lengths that arrive together, one of them empty
        dict(name="prompts packed", op="prompt", heads="30b", type="bf16", seqs=17, longest=1500, ragged=True, pad=3),
        # heads of 64 values, many short texts to be scored
        dict(name="prompts small heads", op="prompt", heads="tiny", type="bf16", seqs=64, longest=333, ragged=True, pad=0),
        # one long prompt: the largest
        dict(name="prompt long", op="prompt", heads="235b", type="f16", seqs=1, longest=8192, ragged=False, pad=0),
        # a token each of 64 sequences, as they decode (early on: the pool that comes back is small)
        dict(name="append tokens of 64", op="append", heads="235b", rows="", page=16, seqs=64, q=1, kv_new=45, ragged=True),
        # prompts entering the cache, their rows left for the prompt attention
        dict(name="append prompts", op="append", heads="30b", rows="bf16", page=64, seqs=9, q=700, kv_new=700, ragged=True),
        # one sequence decoding
        dict(name="attend one token", op="attend", heads="235b", page=16, seqs=1, q=1, prefix=0, kv_new=1100, ragged=False),
        # one sequence decoding far into a long text, which a small cache is for
        dict(name="attend long text", op="attend", heads="30b", page=64, seqs=1, q=1, prefix=0, kv_new=131072, ragged=False),
        # 64 sequences of different lengths, a token each
        dict(name="attend 64", op="attend", heads="235b", page=32, seqs=64, q=1, prefix=0, kv_new=4096, ragged=True),
        # 64 sequences of four drafted tokens behind one long prompt
        dict(name="attend drafts long prompt", op="attend", heads="235b", page=64, seqs=64, q=5, prefix=8192, kv_new=640, ragged=False),
        # the row that a token is drawn from, with its ten likeliest tokens
        dict(name="logprobs one row", op="logprobs", rows=1, vocab=VOCAB, ids=1, top=10, temp=1.0),
        # the rows of a prompt of 512 tokens that is being scored
        dict(name="logprobs 512 rows", op="logprobs", rows=512, vocab=VOCAB, ids=1, top=10, temp=1.0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def _cost(c):
    """What a case costs: (values gathered or stored, scores)."""
    H, Hk, D = HEADS[c["heads"]]
    if c["op"] == "prompt":
        n = _prompts(c)
        return sum(n) * H * D, sum(x * x for x in n) * H * D
    n = c.get("prefix", 0) + c["kv_new"]
    return c["seqs"] * n * Hk * D, c["seqs"] * c["q"] * H * n * D


def draw(rng):
    op = rng.choice(["prompt", "prompt", "prompt", "append", "attend", "attend", "attend", "logprobs"])
    if op == "logprobs":
        return dict(op=op, rows=_log(rng, 1, 512), vocab=rng.choice([4096, 32003, VOCAB]), ids=rng.choice([1, 1, rng.randint(2, 5)]),
                    top=rng.choice([0, 1, rng.randint(2, 20)]), temp=rng.choice([0.7, 1.0, 1.3]))
    while True:
        heads = rng.choice(["235b", "30b", "tiny"])
        if op == "prompt":
            c = dict(op=op, heads=heads, type=rng.choice(["f16", "bf16"]), seqs=rng.choice([1, _log(rng, 1, 64)]), longest=_log(rng, 1, 8192),
                     ragged=rng.random() < 0.6, pad=rng.choice([0, 0, rng.randint(1, 9)]))
            most = (1 << 62, _cost(dict(op=op, heads="235b", seqs=1, longest=8192, ragged=False))[1])
        elif op == "append":
            q = rng.choice([1, rng.randint(2, 8), _log(rng, 9, 1000)])
            c = dict(op=op, heads=heads, rows=rng.choice(["", "f16", "bf16"]), page=rng.choice([16, 32, 64, 128]), seqs=_log(rng, 1, 64), q=q,
                     kv_new=q + rng.choice([0, _log(rng, 1, 500)]), ragged=rng.random() < 0.6)
            most = (64 * 250 * 4 * 128, 1 << 62)
        else:
            q = rng.choice([1, 1, rng.randint(2, 8), _log(rng, 9, 400)])
            c = dict(op=op, heads=heads, page=rng.choice([16, 32, 64, 128]), seqs=_log(rng, 1, 64), q=q, prefix=rng.choice([0, _log(rng, 1, 8192)]),
                     kv_new=q + _log(rng, 1, 130000), ragged=rng.random() < 0.6)
            most = _cost(dict(op=op, heads="235b", seqs=64, q=5, prefix=8192, kv_new=640))
        if all(x <= y for x, y in zip(_cost(c), most)):
            return c


# ---- lengths: from the case alone ------------------------------------------------------------------

def _prompts(c):
    """The prompts' lengths; ragged batches hold empty ones and one of a single token."""
    n = [c["longest"] if not c["ragged"] or b == 0 else (7919 * b + 13) % (c["longest"] + 1) for b in range(c["seqs"])]
    if c["ragged"]:
        n[3:5] = [0, 1][:len(n[3:5])]
    return n


def _lengths(c):
    """Per sequence: new tokens and positions in the cache with them. A ragged batch of several tokens has idle sequences."""
    qs, kv, prefix = [], [], c.get("prefix", 0)
    for b in range(c["seqs"]):
        n = c["q"] if not c["ragged"] or b == 0 or c["q"] == 1 else (5 * b + 2) % (c["q"] + 1)
        qs.append(n)
        kv.append(prefix + (c["kv_new"] if not c["ragged"] or b == 0 else n + (7919 * b + 13) % (c["kv_new"] - n + 1)))
    return qs, kv


def work(case):
    c = case
    if c["op"] == "logprobs":
        return {"bytes": c["rows"] * (4 * c["vocab"] + 8 * c["ids"] + 8 * c["top"] + 4), "flops": 6 * c["rows"] * c["vocab"]}
    H, Hk, D = HEADS[c["heads"]]
    if c["op"] == "prompt":
        n = _prompts(c)
        return {"bytes": 4 * sum(n) * (H + Hk) * D, "flops": 4 * sum(x * (x + 1) // 2 for x in n) * H * D}
    qs, kv = _lengths(c)
    row = D * 9 // 16                               # a K or V row in the cache
    if c["op"] == "append":
        out = 2 * (H + 2 * Hk) * D if c["rows"] else 4 * H * D
        pool = sum(-(-n // c["page"]) for n in kv) * c["page"]
        # the tokens' rows in and out; then the pool, read back as the values it stands for
        return {"bytes": sum(qs) * (4 * (H + 2 * Hk) * D + out + 2 * Hk * row + 4 * D) + pool * Hk * 2 * (row + 4 * D),
                "flops": 12 * sum(qs) * (H + 2 * Hk) * D + 2 * pool * Hk * D}
    rows = c["prefix"] + sum(n - c["prefix"] for n, t in zip(kv, qs) if t)
    pairs = sum(t * (n - t) + t * (t + 1) // 2 for n, t in zip(kv, qs))
    return {"bytes": 2 * rows * Hk * row + 8 * sum(qs) * H * D, "flops": 4 * pairs * H * D}


# ---- the cache in 4 bits ------------------------------------------------------------------------------

def _scales(x):
    """x [..., groups, 32] -> their scales, 8 significant bits, float64 [..., groups, 1]."""
    a = x.abs()
    at = (a == a.amax(-1, keepdim=True)).int().argmax(-1, keepdim=True)         # the first of equals
    m, e = torch.frexp(x.gather(-1, at).double() / -8.0)
    return torch.ldexp(torch.round(m * 256.0) / 256.0, e).clamp(-8160.0, 8160.0).half().double()


def _pack(x):
    """Values [..., D] as (words int32 [..., D / 8], scales fp16 [..., D / 32])."""
    x = x.unflatten(-1, (-1, 32))
    d = _scales(x)
    n = torch.where(d == 0, 8.0, torch.floor(x.double() / d + 8.5)).clamp(0, 15).to(torch.int64)
    shifts = torch.tensor(SHIFTS, device=x.device)
    w = (n.unflatten(-1, (4, 8)) << shifts).sum(-1)                             # below 2^32
    return torch.where(w >= 1 << 31, w - (1 << 32), w).int().flatten(-2), d[..., 0].half()


def _planes(pool, page, D):
    """The words [n_pages][Hk][page][D / 8] and scales [n_pages][Hk][page][D / 32] of a pool, as views."""
    n = page * D // 2
    words, scales = pool[..., :n].view(torch.int32), pool[..., n:].view(torch.float16)
    return words.unflatten(-1, (page, D // 8)), scales.unflatten(-1, (page, D // 32))


def _unpack(words, scales):
    """float32 [..., D]"""
    shifts = torch.tensor(SHIFTS, dtype=torch.int32, device=words.device)
    n = (words[..., None] >> shifts) & 15
    return ((n.flatten(-2).unflatten(-1, (-1, 32)) - 8).float() * scales[..., None].float()).flatten(-2)


# ---- inputs -----------------------------------------------------------------------------------------

def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _paged(c, seed, g):
    """A pool in 4 bits and a batch: the prompt's full pages are shared, every sequence has its own pages after them."""
    H, Hk, D = HEADS[c["heads"]]
    P, prefix = c["page"], c.get("prefix", 0)
    qs, kv = _lengths(c)
    B, shared = c["seqs"], prefix // P
    need = [max(0, -(-n // P) - shared) for n in kv]
    order = np.random.default_rng(seed).permutation(shared + sum(need)).astype(np.int32)
    table = np.zeros((B, max(1, shared + max(need))), np.int32)
    table[:, :shared] = order[:shared]
    at = shared
    for b in range(B):
        table[b, shared:shared + need[b]] = order[at:at + need[b]]
        at += need[b]
    table = torch.from_numpy(table).cuda()
    pools = []
    for _ in range(2):
        pool = torch.empty((len(order), Hk, P * (D // 2 + D // 16)), dtype=torch.uint8, device="cuda")
        words, scales = _planes(pool, P, D)
        step = max(1, (1 << 24) // (Hk * P * D))
        for i in range(0, len(order), step):
            x = torch.randn((min(step, len(order) - i), Hk, P, D), generator=g, device="cuda")
            words[i:i + step], scales[i:i + step] = _pack(x)
        tail = prefix - shared * P
        if tail:                                    # the prompt ends inside a page: each sequence has a copy of its end
            own_pages, first = table[:, shared].long(), table[0, shared].long()
            for z in (words, scales):
                z[own_pages, :, :tail] = z[first, :, :tail].clone()
        pools.append(pool)
    start = _ints([0] + np.cumsum(qs).tolist())
    return dict(case=c, k=pools[0], v=pools[1], table=table, q_start=start, kv_len=_ints(kv), n_tok=sum(qs), max_q=max(qs), max_kv=max(kv))


def _rope(n, D):
    ang = np.arange(n)[:, None] * ROPE_BASE ** (-2.0 * np.arange(D // 2) / D)[None, :]
    return torch.from_numpy(np.cos(ang).astype(np.float32)).cuda(), torch.from_numpy(np.sin(ang).astype(np.float32)).cuda()


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    if c["op"] == "logprobs":
        R, V = c["rows"], c["vocab"]
        x = 2.5 * torch.randn((R, V), generator=g, device="cuda")
        # tokens of a text: drawn from the rows themselves; and others that could have stood there
        drawn = (x - torch.empty_like(x).exponential_(generator=g).log_()).argmax(-1, keepdim=True)
        ids = torch.cat([drawn, torch.randint(0, V, (R, c["ids"] - 1), generator=g, device="cuda")], 1).int()
        out = (torch.zeros((R, c["ids"]), device="cuda"), torch.zeros((R,), device="cuda"),
               torch.zeros((R, c["top"]), dtype=torch.int32, device="cuda"), torch.zeros((R, c["top"]), device="cuda"))
        return dict(case=c, logits=x, ids=ids, out=out)
    H, Hk, D = HEADS[c["heads"]]
    if c["op"] == "prompt":
        n = _prompts(c)
        T = sum(n) + c["pad"]
        # q | k | v rows as they leave the norm and the rotation; those behind the last prompt belong to nobody
        rows = torch.randn((T, H + 2 * Hk, D), generator=g, device="cuda")
        rows[:, :H] *= 1.2
        rows = rows.to(DTYPES[c["type"]])
        return dict(case=c, rows=rows, q_start=_ints([0] + np.cumsum(n).tolist()), n=n, n_tok=T,
                    out=torch.zeros((T, H, D), dtype=rows.dtype, device="cuda"))
    s = _paged(c, seed, g)
    if c["op"] == "append":
        s["qkv"] = torch.randn((s["n_tok"], (H + 2 * Hk) * D), generator=g, device="cuda")
        s["q_norm"] = 1 + 0.2 * torch.randn((D,), generator=g, device="cuda")
        s["k_norm"] = 1 + 0.2 * torch.randn((D,), generator=g, device="cuda")
        s["cos"], s["sin"] = _rope(s["max_kv"], D)
        s["out"] = (torch.zeros((s["n_tok"], (H + 2 * Hk) * D), dtype=DTYPES[c["rows"]], device="cuda") if c["rows"] else
                    torch.zeros((s["n_tok"], H * D), device="cuda"))
        s["values"] = tuple(torch.zeros((s["k"].shape[0], c["page"], Hk, D), device="cuda") for _ in range(2))
    else:                                           # q as it leaves the norm: rows of length about sqrt(D)
        s["q"] = 1.2 * torch.randn((s["n_tok"], H * D), generator=g, device="cuda")
        s["out"] = torch.zeros((s["n_tok"], H * D), device="cuda")
    return s


# ---- plain forms ------------------------------------------------------------------------------------

def _where(s):
    """Per new token: its sequence, its index there and its position."""
    t = torch.arange(s["n_tok"], device="cuda")
    b = (t[:, None] >= s["q_start"][None, 1:]).sum(1)
    i = t - s["q_start"][b]
    n = s["q_start"][b + 1] - s["q_start"][b]
    return b, i, s["kv_len"][b] - n + i


def _softmax_rows(q, k, v, first):
    """q [Hk, G, n, D], k, v [Hk, L, D], row i sees the positions up to first + i; a kv head and some rows at a time."""
    Hk, G, n, D = q.shape
    out = torch.empty_like(q)
    at = torch.arange(k.shape[1], device="cuda")
    step = max(1, (1 << 28) // max(1, G * k.shape[1]))
    for h in range(Hk):
        for i in range(0, n, step):
            pos = first + torch.arange(i, min(n, i + step), device="cuda")
            L = first + min(n, i + step)
            x = q[h, :, i:i + step] @ k[h, :L].T * (1 / math.sqrt(D))
            x = torch.where(at[:L] <= pos[:, None], x, -math.inf)
            e = torch.exp(x - x.amax(-1, keepdim=True))
            out[h, :, i:i + step] = e @ v[h, :L] / e.sum(-1, keepdim=True)
    return out


def _prompt_plain(s):
    H, Hk, D = HEADS[s["case"]["heads"]]
    out, t = torch.zeros_like(s["out"]), 0
    for n in s["n"]:
        if n:
            x = s["rows"][t:t + n].float()
            q = x[:, :H].unflatten(1, (Hk, H // Hk)).permute(1, 2, 0, 3)
            o = _softmax_rows(q, x[:, H:H + Hk].transpose(0, 1), x[:, H + Hk:].transpose(0, 1), 0)
            out[t:t + n] = o.permute(2, 0, 1, 3).flatten(1, 2).to(out.dtype)
        t += n
    return out


def _append_plain(s):
    c = s["case"]
    H, Hk, D = HEADS[c["heads"]]
    b, _, pos = _where(s)
    x = s["qkv"].view(-1, H + 2 * Hk, D)
    # in 64 bits: a value of K next to a border between two of the 16 steps
    qk = x[:, :H + Hk].double()
    qk = qk / torch.sqrt((qk * qk).mean(-1, keepdim=True) + EPS)
    qk = qk * torch.cat([s["q_norm"].expand(H, D), s["k_norm"].expand(Hk, D)])
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    lo, hi = qk[..., :D // 2], qk[..., D // 2:]
    qk = torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1)
    page, off = s["table"][b, pos // c["page"]].long(), pos % c["page"]
    values = []
    for pool, z in ((s["k"], qk[:, H:]), (s["v"], x[:, H + Hk:])):
        words, scales = _planes(pool, c["page"], D)
        words[page, :, off], scales[page, :, off] = _pack(z)
        values.append(_unpack(words, scales).transpose(1, 2).contiguous())
    if c["rows"]:
        out = torch.cat([qk.float(), x[:, H + Hk:]], 1).to(s["out"].dtype)
    else:
        out = qk[:, :H].float()
    return (out.reshape(s["out"].shape), *values)


def _attend_plain(s):
    c = s["case"]
    H, Hk, D = HEADS[c["heads"]]
    B, Q, G = c["seqs"], s["max_q"], H // Hk
    k, v = (_unpack(*(z[s["table"].long()].transpose(2, 3).flatten(1, 2) for z in _planes(s[x], c["page"], D))).transpose(1, 2) for x in "kv")
    at = torch.arange(k.shape[2], device="cuda")                                # k, v [B, Hk, L, D]
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


def _logprobs_plain(s):
    c = s["case"]
    x = s["logits"]
    y = (x - x.amax(-1, keepdim=True)) / c["temp"]
    e = torch.exp(y)
    # the sum without the row's largest: 1 + z rounds away what a sure token leaves to the others
    at = x.argmax(-1, keepdim=True)
    z = e.scatter(1, at, 0.0).sum(-1, keepdim=True)
    lz = torch.log1p(z)
    entropy = lz - (e * y).sum(-1, keepdim=True) / (1 + z)
    logp = y.gather(1, s["ids"].long()) - lz
    # the likeliest tokens, the lowest index first among equals
    _, top = torch.sort(x, dim=-1, descending=True, stable=True)
    top = top[:, :c["top"]]
    return logp, entropy[:, 0], top.int(), y.gather(1, top) - lz


_PLAIN = {"prompt": _prompt_plain, "append": _append_plain, "attend": _attend_plain, "logprobs": _logprobs_plain}


# ---- the framework's calls ----------------------------------------------------------------------------

def _handles(s):
    """The cache's and the batch's descriptors, which a program keeps beside its buffers."""
    import large_model_b200 as m
    if "batch" not in s:
        if "k" in s:
            s["pages"] = m.KvPages.packed(s["k"], s["v"], HEADS[s["case"]["heads"]][2])
            s["batch"] = m.PagedBatch(s["q_start"], s["kv_len"], s["table"], s["n_tok"], s["max_q"], s["max_kv"], s["case"].get("prefix", 0))
        else:
            s["batch"] = m.PagedBatch.prompts(s["q_start"], s["n_tok"], max(s["n"]))
    return m, s.get("pages"), s["batch"], HEADS[s["case"]["heads"]]


def _prompt_own(s):
    m, _, batch, (H, Hk, D) = _handles(s)
    return m.prompt_attention(batch, s["rows"][:, :H], s["rows"][:, H:H + Hk], s["rows"][:, H + Hk:], out=s["out"])


def _append_own(s):
    m, pages, batch, (H, Hk, D) = _handles(s)
    call = m.prompt_append if s["case"]["rows"] else m.paged_append
    out = call(pages, batch, s["qkv"], H, s["q_norm"], s["k_norm"], EPS, (s["cos"], s["sin"]), s["out"])
    return (out, *pages.values(*s["values"]))


def _attend_own(s):
    m, pages, batch, (H, Hk, D) = _handles(s)
    return m.paged_attention(pages, batch, s["q"], H, out=s["out"])


def _logprobs_own(s):
    import large_model_b200 as m
    return m.logprobs(s["logits"], s["ids"], top=s["case"]["top"], temp=s["case"]["temp"], out=s["out"])


_OWN = {"prompt": _prompt_own, "append": _append_own, "attend": _attend_own, "logprobs": _logprobs_own}


def run(state):
    return (_OWN if own else _PLAIN)[state["case"]["op"]](state)


# ---- from the definitions, in 64 bits -----------------------------------------------------------------

def _exact_attention(q, k, v):
    """q [n, G, D], k, v [L, D] in float64: row i sees the first L - n + i + 1 positions."""
    n, L = q.shape[0], k.shape[0]
    out = torch.empty_like(q)
    step = max(1, (1 << 26) // max(1, L))
    for g in range(q.shape[1]):
        for i in range(0, n, step):
            x = torch.einsum("id,jd->ij", q[i:i + step, g], k) / math.sqrt(q.shape[2])
            late = torch.arange(L, device="cuda") > torch.arange(L - n + i, L - n + i + x.shape[0], device="cuda")[:, None]
            out[i:i + step, g] = torch.softmax(x.masked_fill_(late, -math.inf), -1) @ v
    return out


def _exact_values(pool, c):
    """float64 [n_pages][page][Hk][D], a nibble plane at a time."""
    H, Hk, D = HEADS[c["heads"]]
    P = c["page"]
    raw = pool[..., :P * D // 2].reshape(-1, Hk, P, D // 8, 4).long()
    d = pool[..., P * D // 2:].contiguous().view(torch.float16).reshape(-1, Hk, P, D // 32).double()
    n = torch.empty(raw.shape[:-1] + (8,), dtype=torch.float64, device="cuda")
    for i in range(8):                              # value i: bits 4 (i / 2) + 16 (i % 2) on
        bit = 4 * (i // 2) + 16 * (i % 2)
        n[..., i] = (raw[..., bit // 8] // (1 << bit % 8) % 16).double()
    return ((n.flatten(-2) - 8.0) * d.repeat_interleave(32, -1)).transpose(1, 2)


def _exact_stored(x):
    """What the cache gives back for x [..., 32] float64."""
    big = x.abs().max(-1, keepdim=True).values
    first = (x.abs() >= big).cumsum(-1).cumsum(-1) == 1
    d = (x * first).sum(-1, keepdim=True) / -8.0
    unit = torch.exp2(torch.floor(torch.log2(d.abs().clamp(min=1e-30))) - 7)
    d = (torch.round(d / unit) * unit).half().double()
    n = torch.floor(x / torch.where(d == 0, 1.0, d) + 8.5).clamp(0.0, 15.0)
    return torch.where(d == 0, 0.0, (n - 8.0) * d)


def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["op"] == "logprobs":
        logp, entropy, top = (torch.empty(x.shape, dtype=torch.float64, device="cuda") for x in (s["out"][0], s["out"][1], s["out"][3]))
        for r in range(c["rows"]):
            x = s["logits"][r].double() / c["temp"]
            lp = x - torch.logsumexp(x, 0)
            logp[r] = lp[s["ids"][r].long()]
            entropy[r] = -(lp.exp() * lp).sum()
            top[r] = lp.topk(c["top"]).values
        return logp, entropy, None, top
    H, Hk, D = HEADS[c["heads"]]
    G = H // Hk
    if c["op"] == "prompt":
        out, t = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda"), 0
        for n in s["n"]:
            for h in range(Hk if n else 0):
                x = s["rows"][t:t + n]
                out[t:t + n, h * G:(h + 1) * G] = _exact_attention(x[:, h * G:(h + 1) * G].double(), x[:, H + h].double(), x[:, H + Hk + h].double())
            t += n
        return out
    qs, kv = _lengths(c)
    ends = np.cumsum(qs)
    if c["op"] == "attend":
        out = torch.zeros((s["n_tok"], H, D), dtype=torch.float64, device="cuda")
        for b, (n, end, t1) in enumerate(zip(qs, kv, ends)):
            if n == 0:
                continue
            pages = s["table"][b, :-(-end // c["page"])].long()
            k, v = (_exact_values(s[x][pages], c).flatten(0, 1)[:end] for x in "kv")
            for h in range(Hk):
                out[t1 - n:t1, h * G:(h + 1) * G] = _exact_attention(s["q"][t1 - n:t1].double().view(n, H, D)[:, h * G:(h + 1) * G], k[:, h], v[:, h])
        return out.view(s["n_tok"], H * D)
    k, v = (_exact_values(s[x], c).contiguous() for x in "kv")
    rows = torch.empty((s["n_tok"], H + 2 * Hk, D), dtype=torch.float64, device="cuda")
    cos, sin = s["cos"].double(), s["sin"].double()
    for b, (n, end, t1) in enumerate(zip(qs, kv, ends)):
        x = s["qkv"][t1 - n:t1].double().view(n, H + 2 * Hk, D)
        at = torch.arange(end - n, end, device="cuda")
        z = torch.complex(cos[at], sin[at])[:, None]

        def turned(y, w):
            y = y * (y.pow(2).sum(-1, keepdim=True) / D + EPS).pow(-0.5) * w.double()
            r = torch.complex(y[..., :D // 2].contiguous(), y[..., D // 2:].contiguous()) * z
            return torch.cat([r.real, r.imag], -1)
        y = torch.cat([turned(x[:, :H], s["q_norm"]), turned(x[:, H:H + Hk], s["k_norm"]), x[:, H + Hk:]], 1)
        rows[t1 - n:t1] = y
        page = s["table"][b, at // c["page"]].long()
        for pool, first in ((k, H), (v, H + Hk)):
            pool[page, at % c["page"]] = _exact_stored(y[:, first:first + Hk].unflatten(-1, (-1, 32))).flatten(-2)
    return (rows if c["rows"] else rows[:, :H]).reshape(s["out"].shape), k, v
