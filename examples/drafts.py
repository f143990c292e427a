"""Several sequences on one prompt, generated with drafted tokens: the paged cache, the attention that reads it and the
verification of drafts, around the library's projections and MoE layers.

    python examples/drafts.py [--seqs 4] [--new 48] [--draft 4] [--temp 0.8] [--fp16-cache]

One forward step takes any number of token rows of any number of sequences (src/model.c:1252-1296 one sequence at a time).
The shared prompt is run once and its pages stand in every sequence's table; each sequence then adds its own
prompt. From there a step takes, for each sequence, its last token and up to --draft guesses at what follows (here: what followed the
last time that its last two tokens came up), and the verification says how many guesses stand and which token comes
after them. Cache positions of guesses that fell are written again by the next step. The weights are the seeded
synthetic ones of large_model_b200.synth, so the text means nothing; what is guessed still stands now and then."""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import numpy as np
import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))
import large_model_b200 as m
from large_model_b200 import synth


def q4_0_values(blocks: np.ndarray, cols: int) -> np.ndarray:
    """ggml Q4_0 blocks {f16 d; u8 qs[16]} as float32 rows: d * (nibble - 8), low nibbles first."""
    b = blocks.reshape(-1, 18)
    d = b[:, :2].copy().view(np.float16).astype(np.float32)
    q = np.concatenate([b[:, 2:] & 15, b[:, 2:] >> 4], 1).astype(np.float32) - 8.0
    return (d * q).reshape(-1, cols)


class PagedModel:
    """A synthetic model's layers over a pool of cache pages (one KvPages per layer, one table for all)."""

    def __init__(self, cfg, seed: int, n_pages: int, page: int, ctx: int, kv_type: int = m.T_F32):
        t = {name: synth.tensor_data(cfg, seed, i) for i, (name, _, _) in enumerate(synth.model_tensors(cfg))}
        dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()
        self.cfg, self.page, self.ctx = cfg, page, ctx
        self.embd = dev(q4_0_values(t["token_embd.weight"], cfg.n_embd))
        self.out_norm, self.out = dev(t["output_norm.weight"]), dev(t["output.weight"])
        self.rope = m.rope_tables(ctx, cfg.head_dim, cfg.rope_base)
        self.layers = []
        for l in range(cfg.n_layer):
            w = {k.split(".")[2]: v for k, v in t.items() if k.startswith(f"blk.{l}.")}
            moe = m.MoeLayer(cfg.n_embd, cfg.n_expert, cfg.n_used, cfg.n_ff, w["ffn_gate_inp"], w["ffn_gate_exps"], w["ffn_up_exps"],
                             w["ffn_down_exps"])
            qkv = dev(np.concatenate([w[f"attn_{x}"].reshape(-1) for x in "qkv"]))       # q | k | v rows, one product
            self.layers.append((*(dev(w[x]) for x in ("attn_norm", "attn_q_norm", "attn_k_norm", "ffn_norm")), qkv, dev(w["attn_output"]), moe,
                                m.KvPages.empty(n_pages, page, cfg.n_head_kv, cfg.head_dim, kv_type)))

    def norm(self, x, w):
        return x * torch.rsqrt(x.double().pow(2).mean(-1, keepdim=True) + self.cfg.eps).float() * w

    def step(self, ids, batch):
        """Logits [T][vocab] of token rows ids (CUDA int [T]), which join the cache where `batch` says."""
        c = self.cfg
        E, W = c.n_embd, c.n_head * c.head_dim
        x, T = self.embd[ids.long()], len(ids)
        for attn_norm, q_norm, k_norm, ffn_norm, wqkv, wo, moe, pages in self.layers:
            qkv = m.matvec_q8(m.T_Q4_0, wqkv, W + 2 * c.n_head_kv * c.head_dim, E, m.quantize_q8(self.norm(x, attn_norm)), T)
            q = m.paged_append(pages, batch, qkv, c.n_head, q_norm, k_norm, c.eps, self.rope)
            a = m.paged_attention(pages, batch, q, c.n_head)
            x = x + m.matvec_q8(m.T_Q4_0, wo, E, W, m.quantize_q8(a), T)
            x = moe.forward(self.norm(x, ffn_norm), resid=x)
        return m.matvec_q8(c.output_type, self.out, c.vocab, E, m.quantize_q8(self.norm(x, self.out_norm)), T)


def guess(known: list[int], n: int) -> list[int]:
    """What followed the last two tokens the time before, up to n tokens."""
    for i in range(len(known) - 3, 0, -1):
        if known[i - 1:i + 1] == known[-2:]:
            return known[i + 1:i + 1 + n]
    return []


def generate(model: PagedModel, prompt: list[int], tails: list[list[int]], new: int, temp: float = 0.0, max_draft: int = 4, draft=None,
             seed: int = 0):
    """`new` tokens for each sequence prompt + tails[b] (no tail is empty). draft(b, known, n) -> at most n guesses. Returns
    (the sequences' tokens, steps, guesses made, guesses that stood)."""
    draft = draft or (lambda b, known, n: guess(known, n))
    B, page = len(tails), model.page
    known = [prompt + t for t in tails]
    goal = [len(k) + new for k in known]
    # whole pages of the prompt are shared; each sequence has pages of its own behind them
    shared = len(prompt) // page
    each = -(-(max(goal) + max_draft) // page) - shared
    if shared + B * each > model.layers[0][-1].desc.n_pages or max(goal) + max_draft > model.ctx:
        raise ValueError("generate: the pool or the context is too small")
    table = np.empty((B, shared + each), np.int32)
    table[:, :shared] = np.arange(shared)
    table[:, shared:] = shared + np.arange(B * each).reshape(B, each)
    dev = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")
    table = dev(table)
    if shared:                                                       # the shared pages, once
        n = shared * page
        batch = m.PagedBatch(dev([0, n]), dev([n]), table[:1].contiguous(), n, n, n)
        model.step(dev(prompt[:n]), batch)
        batch.status()
    gen = torch.Generator(device="cuda").manual_seed(seed)
    cached, steps, made, stood = [shared * page] * B, 0, 0, 0
    while any(len(k) < g for k, g in zip(known, goal)):
        # the tokens that are not in the cache yet and the guesses after them (none for sequences that are done)
        todo = [k[c:] if len(k) < g else [] for k, c, g in zip(known, cached, goal)]
        drafts = [draft(b, known[b], min(max_draft, goal[b] - len(known[b]) - 1))[:max_draft] if todo[b] else [] for b in range(B)]
        rows = [t + d for t, d in zip(todo, drafts)]
        start = np.concatenate([[0], np.cumsum([len(r) for r in rows])])
        kv = [c + len(r) for c, r in zip(cached, rows)]
        batch = m.PagedBatch(dev(start), dev(kv), table, int(start[-1]), max(map(len, rows)), max(kv), shared * page)
        logits = model.step(dev([t for r in rows for t in r]), batch)
        p = m.probs(logits, temp)
        # each sequence's rows of p: the one after its last known token, then one per guess (a sequence that is done
        # gets some row, and its result is not looked at)
        first = [min(int(start[b]) + max(0, len(todo[b]) - 1), int(start[-1]) - 1) for b in range(B)]
        ids = np.zeros((B, max_draft), np.int32)
        for b, d in enumerate(drafts):
            ids[b, :len(d)] = d
        u = torch.rand((B, max_draft + 1), generator=gen, device="cuda")
        n_accept, tokens = m.verify(p, dev(ids), u, n_draft=dev([len(d) for d in drafts]), row_start=dev(first), err=batch.err)
        batch.status()
        n_accept, tokens = n_accept.tolist(), tokens.tolist()
        steps += 1
        for b in range(B):
            if not todo[b]:
                continue
            known[b] = known[b] + tokens[b][:n_accept[b] + 1]
            cached[b] = len(known[b]) - 1                            # all but the new last token
            made += len(drafts[b])
            stood += n_accept[b]
    return known, steps, made, stood


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--seqs", type=int, default=4)
    ap.add_argument("--new", type=int, default=48)
    ap.add_argument("--draft", type=int, default=4)
    ap.add_argument("--temp", type=float, default=0.0)
    ap.add_argument("--fp16-cache", action="store_true")
    a = ap.parse_args()
    cfg = synth.MODEL_CONFIGS["tiny"]
    m.init()
    model = PagedModel(cfg, 1, 256, 16, 1024, m.T_F16 if a.fp16_cache else m.T_F32)
    prompt = synth.random_ids(cfg.vocab, 40, 5)
    tails = [synth.random_ids(cfg.vocab, 3 + b, 6 + b) for b in range(a.seqs)]
    known, steps, made, stood = generate(model, prompt, tails, a.new, a.temp, a.draft)
    for b, k in enumerate(known):
        print(f"sequence {b}: {k[len(prompt) + len(tails[b]):]}")
    print(f"{a.seqs * a.new} tokens in {steps} steps; {stood} of {made} guesses stood")


if __name__ == "__main__":
    main()
