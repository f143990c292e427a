"""Probabilities of logits rows and the verification of drafted tokens on a B200 (qms_cuda_probs, qms_cuda_verify).

Verification is checked for equality with whole-number arithmetic on the host. Probabilities: exp's argument
(l - max) / temp is off by 2^-23 of itself, exp and the sum of V terms by a few roundings, the sum's being at
most V 2^-24 and in practice far less: the bound is (2^-22 |x| + 2^-20) p, plus the smallest normal number."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def host_verify(p, q, draft, n_draft, row_start, u, V):
    """The definition, with Python's integers."""
    f32 = np.float32
    B, N = draft.shape
    acc, toks, err = [], [], 0
    for b in range(B):
        nd = N if n_draft is None else int(n_draft[b])
        r0 = b * (N + 1) if row_start is None else int(row_start[b])
        if nd < 0 or nd > N or r0 < 0 or r0 + nd >= len(p):
            acc.append(0)
            toks.append([-1] * (N + 1))
            err |= 1
            continue
        n = 0
        while n < nd:
            x = int(draft[b, n])
            if not 0 <= x < V:
                err |= 4
                break
            qx = f32(1) if q is None else q[b * N + n, x]
            if not f32(u[b, n] * qx) < p[r0 + n, x]:
                break
            n += 1
        row = p[r0 + n]
        rest = row.copy()
        if n < nd and 0 <= int(draft[b, n]) < V:
            if q is None:
                rest[int(draft[b, n])] = 0
            else:
                rest = (row - q[b * N + n]).astype(f32)

        def whole(r):
            with np.errstate(invalid="ignore"):
                r = np.where(r > 0, np.minimum(r, f32(1)), f32(0)).astype(np.float64) * 2.0 ** 40
            return [int(w) for w in np.rint(r)]
        w = whole(rest)
        if sum(w) == 0:
            w = whole(row)
        pick = -1
        if sum(w):
            want = sum(w) * int(np.floor(float(u[b, N]) * 2 ** 24)) >> 24
            c = 0
            for pick, x in enumerate(w):
                c += x
                if c > want:
                    break
        else:
            err |= 8
        acc.append(n)
        toks.append([int(x) for x in draft[b, :n]] + [pick] + [-1] * (N - n))
    return acc, toks, err


def run(p, q, draft, n_draft, row_start, u, pad=0):
    import torch
    import large_model_b200 as m

    def rows(x):
        if x is None:
            return None
        w = torch.full((x.shape[0], x.shape[1] + pad), 3.0, device="cuda")
        w[:, :x.shape[1]] = torch.from_numpy(x).cuda()
        return w[:, :x.shape[1]]
    ints = lambda x: None if x is None else torch.from_numpy(np.ascontiguousarray(x, np.int32)).cuda()
    err = torch.zeros((1,), dtype=torch.int32, device="cuda")
    n, t = m.verify(rows(p), ints(draft), torch.from_numpy(u).cuda(), q=rows(q), n_draft=ints(n_draft), row_start=ints(row_start), err=err)
    return n.tolist(), t.tolist(), int(err.item())


def softmax(x):
    e = np.exp(x - x.max(-1, keepdims=True))
    return (e / e.sum(-1, keepdims=True)).astype(np.float32)


def case(B, N, V, with_q, seed, spread=2.0):
    r = np.random.default_rng(seed)
    x = r.standard_normal((B, N + 1, V)) * spread
    p = softmax(x).reshape(B * (N + 1), V)
    q = softmax(x[:, :N] + 0.5 * r.standard_normal((B, N, V))).reshape(B * N, V)
    draft = np.array([[r.choice(V, p=(lambda w: w / w.sum())(q[b * N + i].astype(np.float64))) for i in range(N)] for b in range(B)],
                     np.int32).reshape(B, N)
    u = r.random((B, N + 1), np.float32)
    return p, q if with_q else None, draft, u


@pytest.mark.parametrize("with_q", [False, True])
@pytest.mark.parametrize("pad", [0, 1, 4])
@pytest.mark.parametrize("B,N,V", [(1, 1, 1), (1, 4, 2), (3, 2, 31), (5, 3, 1000), (2, 5, 1025), (70, 3, 4096), (2, 2, 32003), (3, 4, 151936),
                                   (2, 1, 300001)])
def test_verify_equals_the_definition(cuda, with_q, pad, B, N, V):
    p, q, draft, u = case(B, N, V, with_q, B * 1000 + V)
    assert run(p, q, draft, None, None, u, pad) == host_verify(p, q, draft, None, None, u, V)
    nd = np.arange(B) % (N + 1)
    assert run(p, q, draft, nd, None, u, pad) == host_verify(p, q, draft, nd, None, u, V)


@pytest.mark.parametrize("with_q", [False, True])
def test_verify_rows_elsewhere_and_no_drafts(cuda, with_q):
    p, q, draft, u = case(6, 3, 517, with_q, 3)
    start = np.array([20, 0, 9, 4, 4, 13])
    nd = np.array([3, 0, 2, 1, 3, 3])
    assert run(p, q, draft, nd, start, u) == host_verify(p, q, draft, nd, start, u, 517)
    none = np.zeros((6, 0), np.int32)
    assert run(p, None, none, None, None, u[:, :1].copy()) == host_verify(p, None, none, None, None, u[:, :1], 517)


def test_verify_picks_every_index_at_its_boundary(cuda):
    """u at, just below and just above each step of a row whose steps are multiples of 2^-24."""
    V = 9
    r = np.random.default_rng(0)
    cuts = np.sort(r.integers(1, 2 ** 24, V - 1))
    w = np.diff(np.concatenate([[0], cuts, [2 ** 24]]))
    w[4] += w[5]
    w[5] = 0                                         # a token of no weight is never drawn
    row = (w / 2.0 ** 24).astype(np.float32)
    at = np.cumsum(w)[:-1]
    u = np.concatenate([[0, 2 ** 24 - 1], at, at - 1, at + 1]).clip(0, 2 ** 24 - 1)
    u = (u / 2.0 ** 24).astype(np.float32)[:, None]
    p = np.tile(row, (len(u), 1))
    none = np.zeros((len(u), 0), np.int32)
    got = run(p, None, none, None, None, u)
    assert got == host_verify(p, None, none, None, None, u, V)
    assert all(t[0] != 5 for t in got[1])


def test_verify_greedy(cuda):
    """With probabilities of 0 and 1 a draft stands exactly where it is the argmax."""
    import torch
    import large_model_b200 as m
    B, N, V = 4, 3, 3001
    r = np.random.default_rng(1)
    x = r.standard_normal((B * (N + 1), V)).astype(np.float32)
    best = x.argmax(1).reshape(B, N + 1)
    draft = best[:, :N].copy()
    draft[1, 0] += 1
    draft[2, 2] = 7
    p = m.probs(torch.from_numpy(x).cuda(), 0.0).cpu().numpy()
    n, t, e = run(p, None, draft, None, None, r.random((B, N + 1), np.float32))
    assert n == [3, 0, 2, 3] and e == 0
    assert t == [[*best[0]], [best[1, 0], -1, -1, -1], [best[2, 0], best[2, 1], best[2, 2], -1], [*best[3]]]


@pytest.mark.parametrize("with_q", [False, True])
def test_verify_faulty_inputs(cuda, with_q):
    p, q, draft, u = case(5, 2, 100, with_q, 9)
    draft[0, 0] = -1
    draft[1, 1] = 100
    nd = np.array([2, 2, 3, -1, 2])
    assert run(p, q, draft, nd, None, u) == host_verify(p, q, draft, nd, None, u, 100)
    p, q, draft, u = case(4, 2, 100, with_q, 10)
    p[0:3] = 0                                       # no mass
    p[3:6, 5] = np.nan                               # NaN is no probability
    p[6:9] *= -1
    p[9:12] = np.inf                                 # counts as 1
    assert run(p, q, draft, None, None, u) == host_verify(p, q, draft, None, None, u, 100)
    start = np.array([0, -1, 10, 9])
    assert run(p, q, draft, None, start, u) == host_verify(p, q, draft, None, start, u, 100)


def test_verify_falls_back_to_p(cuda):
    """A rejected draft whose p nowhere exceeds q (both rounded): the next token is drawn from p."""
    p = np.full((2, 4), 0.25, np.float32)
    q = np.full((1, 4), 0.2500001, np.float32)
    u = np.array([[0.9999999, 0.6]], np.float32)
    draft = np.array([[2]], np.int32)
    got = run(p, q, draft, None, None, u)
    assert got == host_verify(p, q, draft, None, None, u, 4)
    assert got[0] == [0] and got[1] == [[2, -1]]


def test_verify_keeps_the_targets_distribution(cuda):
    """The first token of 60000 sequences is distributed as the target's p: each count within 5 standard
    deviations."""
    r = np.random.default_rng(4)
    B, V = 60000, 7
    p1 = softmax(r.standard_normal(V) * 1.5)
    q1 = softmax(r.standard_normal(V) * 1.5)
    draft = r.choice(V, size=(B, 1), p=q1.astype(np.float64) / q1.astype(np.float64).sum()).astype(np.int32)
    p = np.tile(p1, (2 * B, 1))
    for q in (np.tile(q1, (B, 1)), None):
        d = draft if q is not None else np.full((B, 1), 3, np.int32)
        n, t, e = run(p, q, d, None, None, r.random((B, 2), np.float32))
        count = np.bincount([x[0] for x in t], minlength=V)
        assert e == 0 and (np.abs(count - B * p1) <= 5 * np.sqrt(B * p1 * (1 - p1))).all()


# ---- probabilities -----------------------------------------------------------------------------------

@pytest.mark.parametrize("temp", [0.3, 1.0, 2.5])
@pytest.mark.parametrize("rows,V,pad", [(1, 1, 0), (3, 2, 0), (2, 1023, 1), (7, 1025, 3), (200, 4096, 0), (3, 32003, 4), (2, 151936, 0), (2, 300001, 2),
                                        (1, 1000003, 0)])
def test_probs(cuda, temp, rows, V, pad):
    import torch
    import large_model_b200 as m
    g = torch.Generator(device="cuda").manual_seed(V)
    wide = 4 * torch.randn((rows, V + pad), generator=g, device="cuda")
    l = wide[:, :V]
    l[0, V // 2] = -float("inf")
    if V > 1:
        l[-1, V // 3] = 40.0                         # one token takes nearly everything
    out = torch.full((rows, V + pad + 1), 5.0, device="cuda")
    m.probs(l, temp, out=out[:, :V])
    assert (out[:, V:] == 5).all()
    if V == 1:
        assert (out[:, 0] == 0).all()                # its only logit is -inf
        return
    x = l.double() / temp
    want = torch.softmax(x, -1)
    far = (x - x.amax(-1, keepdim=True)).abs().clamp(max=200)
    assert ((out[:, :V].double() - want).abs() <= (2.0 ** -22 * far + 2.0 ** -20) * want + 2.0 ** -126).all()
    again = l.clone()
    m.probs(again, temp, out=again)                  # in place
    assert torch.equal(again, out[:, :V])


def test_probs_rows_with_special_values(cuda):
    import torch
    import large_model_b200 as m
    inf = float("inf")
    l = torch.randn((5, 3000), device="cuda")
    l[0] = -inf
    l[1, 7] = float("nan")
    l[2, 9] = inf
    l[3, 10:] = -inf
    p = m.probs(l, 1.0)
    assert (p[0] == 0).all() and p[1].isnan().all() and p[2].isnan().all() and (p[3, 10:] == 0).all()
    assert torch.isfinite(p[3:]).all()
    l[4] = 2.0
    l[1, 0] = 50.0
    p = m.probs(l, 0.0)                              # greedy: the first maximum, never NaN
    assert p.sum(1).tolist() == [0, 1, 1, 1, 1]
    assert p.argmax(1).tolist()[1:] == [0, 9, int(l[3].argmax()), 0]
    assert torch.equal(m.probs(l, -1.0), p)


def test_probs_of_a_row_that_is_mostly_masked(cuda):
    """All values far below 0, and so few of them that most threads see none."""
    import torch
    import large_model_b200 as m
    l = torch.full((2, 151936), -float("inf"), device="cuda")
    l[0, 77:80] = torch.tensor([-20000.0, -20001.0, -20000.0])
    l[1, 151935] = 3e38
    p = m.probs(l, 1.0)
    want = torch.softmax(l.double(), -1)
    assert ((p.double() - want).abs() <= 2.0 ** -19 * want).all() and torch.isfinite(p).all()


def test_probs_small_and_large_temperatures(cuda):
    import torch
    import large_model_b200 as m
    l = torch.randn((3, 5001), device="cuda")
    assert ((m.probs(l, 1e-6) - m.probs(l, 0.0)).abs() <= 2.0 ** -20).all()
    assert ((m.probs(l, 1e6).double() - 1 / 5001).abs() <= 1e-4 / 5001).all()
