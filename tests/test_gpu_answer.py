"""Answering prompts on a B200 with the operators together: whole prompts into pages of 4 bits with their rows in 16 bits, attention within the
prompts, log probabilities of what the prompts say, then tokens one at a time over the pages, eager and as one captured graph.

Bounds: those of the two attentions (the 64-bit formulas on the rows and the pages as they are stored); through the head, in 64 bits and rounded
to fp32, |W| times that and e |logit|, e = 2^-24; a log probability is off by at most twice the row's largest error of a logit, and by (64 + 4 |logp|) e: the
subtraction of the maximum, the exponentials and their sum at 44 e, the logarithm and the last subtraction."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
E = 2.0 ** -24
H, HK, PAGE, VOCAB, STEPS = 16, 2, 32, 1003, 5


class Chain:
    """Tables in place of layers: a token's q | k | v, and the head."""

    def __init__(self, lens, D, seed):
        import torch
        import large_model_b200 as m
        g = torch.Generator(device="cuda").manual_seed(seed)
        rand = lambda *s: torch.randn(s, generator=g, device="cuda")
        self.D, self.lens = D, lens
        self.qkv, self.head = rand(VOCAB, (H + 2 * HK) * D), 0.05 * rand(VOCAB, H * D).double()
        self.qn, self.kn = 1 + 0.1 * rand(D), 1 + 0.1 * rand(D)
        most = max(lens) + STEPS
        self.rope = m.rope_tables(most, D)
        self.ids = torch.randint(0, VOCAB, (sum(lens),), generator=g, device="cuda")
        need = -(-most // PAGE)
        perm = np.random.default_rng(seed).permutation(need * len(lens)).astype(np.int32)
        ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
        self.start, self.table = ints([0] + np.cumsum(lens).tolist()), ints(perm.reshape(len(lens), need))
        self.ones, self.kv, self.most = ints(list(range(len(lens) + 1))), ints(lens), most
        self.pages = m.KvPages.empty(len(perm), PAGE, HK, D, m.T_Q4_0)

    def logits(self, o):
        return (o.flatten(1).double() @ self.head.T).float()

    def prompts(self, dtype):
        import torch
        import large_model_b200 as m
        T, n = sum(self.lens), max(self.lens)
        batch = m.PagedBatch(self.start, self.kv, self.table, T, n, self.most)
        rows = m.prompt_append(self.pages, batch, self.qkv[self.ids], H, self.qn, self.kn, 1e-6, self.rope, dtype=dtype)
        o = m.prompt_attention(batch, rows[:, :H], rows[:, H:H + HK], rows[:, H + HK:], out_dtype=torch.float32)
        x = self.logits(o)
        said = torch.roll(self.ids, -1).int()
        got = m.logprobs(x, said, top=4)
        batch.status()
        return rows, x, said, got

    def stepper(self, tokens):
        """A batch of one token per sequence, and the step that takes its tokens to the likeliest next ones, in place."""
        import large_model_b200 as m
        B = len(self.lens)
        batch = m.PagedBatch(self.ones, self.kv, self.table, B, 1, self.most)

        def step():
            self.kv.add_(1)
            q = m.paged_append(self.pages, batch, self.qkv[tokens], H, self.qn, self.kn, 1e-6, self.rope)
            x = self.logits(m.paged_attention(self.pages, batch, q, H))
            got = m.logprobs(x, tokens.int(), top=4)
            tokens.copy_(got[2][:, 0])
            return q, x, got
        return batch, step


def held_to(x, want, tol, ids, got):
    """Logits and log probabilities against the attention's 64-bit result and its bound, through the head."""
    import torch
    logits, tol = want, tol + E * want.abs()
    assert ((x.double() - logits).abs() <= tol).all()
    exact = torch.log_softmax(logits, -1)
    room = 2 * tol.amax(-1, keepdim=True)
    lp, ent, top, top_lp = got
    for i, v in ((ids.long()[:, None], lp), (top.long(), top_lp)):
        y = exact.gather(1, i)
        assert ((v.double() - y).abs() <= room + (64 + 4 * y.abs()) * E).all()
    best = torch.topk(x, 4, dim=-1).values
    assert torch.equal(x.gather(1, top.long()), best)
    # the entropy's derivative by a logit is -p (logp + entropy)
    p = exact.exp()
    y = -(p * exact).sum(-1)
    slope = (p * (exact + y[:, None]).abs()).sum(-1) * tol.amax(-1)
    assert ((ent.double() - y).abs() <= 2 * slope + (64 + 8 * np.log(VOCAB)) * E).all()


@pytest.mark.parametrize("lens", [[1], [75, 1, 200], [33, 130, 64, 5]])
@pytest.mark.parametrize("D,dtype", [(64, "float16"), (128, "bfloat16")])
def test_prompts_then_tokens(cuda, lens, D, dtype):
    import torch
    import test_gpu_attention_prompt as prompt
    import test_gpu_cache4 as cache
    chain = Chain(lens, D, sum(lens))
    rows, x, said, got = chain.prompts(getattr(torch, dtype))
    want, tol = prompt.reference(lens, rows[:, :H], rows[:, H:H + HK], rows[:, H + HK:], D ** -0.5, True)
    W = chain.head.T
    held_to(x, want.flatten(1) @ W, tol.expand_as(want).flatten(1) @ W.abs(), said, got)

    last = chain.start[1:].long() - 1
    tokens = got[2][last, 0].long()
    batch, step = chain.stepper(tokens)
    at = list(lens)
    for _ in range(STEPS):
        asked = tokens.clone()
        q, x, got = step()
        batch.status()
        at = [n + 1 for n in at]
        K, V = ([pool[chain.table[b].long()].flatten(0, 1)[:n].double() for b, n in enumerate(at)] for pool in chain.pages.values())
        want, tol = cache.reference([1] * len(at), at, q, K, V, H // HK, D ** -0.5)
        held_to(x, want @ W, tol @ W.abs(), asked, got)


def test_a_captured_step_says_the_same(cuda):
    import torch
    lens = [75, 1, 200]
    a, b = Chain(lens, 128, 3), Chain(lens, 128, 3)
    first = None
    for c in (a, b):
        _, _, _, got = c.prompts(torch.float16)
        c.tokens = got[2][c.start[1:].long() - 1, 0].long()
        first = first if first is not None else got[2]
        assert torch.equal(first, got[2])
    batch, step = a.stepper(a.tokens)
    eager = []
    for _ in range(STEPS):
        _, x, got = step()
        eager.append([t.clone() for t in (x, *got, a.tokens)])
    batch.status()

    batch, step = b.stepper(b.tokens)
    kv, tokens, pools = b.kv.clone(), b.tokens.clone(), [b.pages.k.clone(), b.pages.v.clone()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()                                   # (what is made on first use; undone below)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        _, x, got = step()
    torch.cuda.synchronize()
    b.kv.copy_(kv), b.tokens.copy_(tokens), b.pages.k.copy_(pools[0]), b.pages.v.copy_(pools[1])
    for want in eager:
        graph.replay()
        for g, w in zip((x, *got, b.tokens), want):
            assert torch.equal(g, w)
    batch.status()
    assert torch.equal(a.pages.k, b.pages.k) and torch.equal(a.pages.v, b.pages.v)
