"""Log probabilities of logits rows on a B200 through the C ABI (qms_cuda_logprobs), against their definition in 64 bits.

Bounds, with e = 2^-24, x = (l - max) / temp <= 0, p the probabilities, A = sum p |x|, Q = sum p x^2. A weight 2^(x log2 e) is off by the
exponent's two roundings, 2 e |x| relatively, and by the exponential's own 4 e; a sum has at most 48 roundings on its way. So Z is off by
(52 + 2 A) e relatively, log Z by as much, log p by that, three roundings of x, the logarithm's two and the difference's: e (52 + 2 A + 3 |x|
+ 2 log Z + |log p|). sum p x: every term's weight as above and two roundings more, and Z: e (54 A + 2 Q + (52 + 2 A) A); the logarithms are taken under a base up to 2^4 below
the largest value so far, which adds up to 4 ln 2 < 3 to each of them: 54 * 3 e more."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
E = 2.0 ** -24


def _want(l, ids, temp):
    import torch
    x = l.double() / temp
    x = x - x.amax(-1, keepdim=True)
    lz = torch.logsumexp(x, -1, keepdim=True)
    p = torch.exp(x - lz)
    px = torch.where(p > 0, p * x, 0.0)
    A, Q = -px.sum(-1, keepdim=True), torch.where(p > 0, px * x, 0.0).sum(-1, keepdim=True)
    lp = x - lz
    tol = E * (52 + 2 * A + 3 * x.abs() + 2 * lz + lp.abs())
    ent, tol_ent = (lz + A)[:, 0], (E * (52 + 2 * A + 2 * lz + 54 * (A + 3) + 2 * Q + (52 + 2 * A) * A + 2 * (lz + A)))[:, 0]
    return lp, tol, ent, tol_ent


def _top(l, n):
    """The n largest, the lowest index first among equals; -1 where only -inf and NaN are left."""
    out = np.full((l.shape[0], n), -1, np.int64)
    for r, row in enumerate(l):
        at = np.flatnonzero(row > -np.inf)
        at = at[np.argsort(-row[at], kind="stable")][:n]
        out[r, :len(at)] = at
    return out


def check(l, ids, top, temp=1.0, **kw):
    import torch
    import large_model_b200 as m
    lp, ent, ti, tl = m.logprobs(l, ids, top=top, temp=temp, **kw)
    want, tol, went, tent = _want(l, ids, temp)
    if ids is not None:
        at = ids.long().view(l.shape[0], -1)
        err = torch.where(lp.double() == want.gather(1, at), -1.0, (lp.double() - want.gather(1, at)).abs() - tol.gather(1, at))
        assert err.max().item() <= 0, f"logp: {err.max().item()} over the bound"
    assert ((ent.double() - went).abs() - tent).max().item() <= 0, "entropy"
    wi = _top(l.cpu().numpy(), top)
    assert np.array_equal(ti.cpu().numpy(), wi)
    if top:
        i = torch.from_numpy(wi).cuda().clamp(min=0)
        err = torch.where(torch.from_numpy(wi).cuda() >= 0, (tl.double() - want.gather(1, i)).abs() - tol.gather(1, i), -1.0)
        assert err.max().item() <= 0, f"likeliest: {err.max().item()} over the bound"
        assert (tl[torch.from_numpy(wi).cuda() < 0] == -float("inf")).all()
    return lp, ent, ti, tl


@pytest.mark.parametrize("V", [1, 2, 3, 31, 100, 128, 1000, 2047, 2049, 4096, 19457, 32003])
@pytest.mark.parametrize("top", [0, 1, 10, 32])
def test_sizes(cuda, V, top):
    import torch
    g = torch.Generator(device="cuda").manual_seed(V + top)
    l = 3 * torch.randn((5, V), generator=g, device="cuda")
    ids = torch.randint(0, V, (5, 3), generator=g, device="cuda").int()
    check(l, ids, top)


@pytest.mark.parametrize("rows,V", [(1, 151936), (3, 155648), (2, 155649), (1, 300007), (40, 151936)])
def test_long_rows(cuda, rows, V):
    import torch
    g = torch.Generator(device="cuda").manual_seed(V + rows)
    l = 2.5 * torch.randn((rows, V), generator=g, device="cuda")
    check(l, torch.randint(0, V, (rows,), generator=g, device="cuda").int(), 20, temp=0.7)


@pytest.mark.parametrize("ld,off", [(1001, 0), (1003, 1), (1008, 2), (1004, 0)])
def test_strides(cuda, ld, off):
    import torch
    g = torch.Generator(device="cuda").manual_seed(ld)
    base = torch.full((7 * ld + 8,), float("nan"), device="cuda")
    l = base[off:off + 7 * ld].view(7, ld)[:, :1000]
    l.copy_(4 * torch.randn((7, 1000), generator=g, device="cuda"))
    check(l, torch.arange(7, device="cuda").int(), 5, temp=1.3)


@pytest.mark.parametrize("V", [40, 3001, 32003, 151936])
def test_equal_values_go_to_the_lowest_id(cuda, V):
    import torch
    g = torch.Generator(device="cuda").manual_seed(V)
    l = torch.randint(-3, 3, (6, V), generator=g, device="cuda").float()
    l[1] = 2.0                                               # nothing but equals
    l[2] = -0.0
    l[2, ::2] = 0.0                                          # 0 and -0 are equal
    l[3, V // 2:] = 7.0
    l[4] = torch.arange(V, device="cuda").float()            # ascending, descending
    l[5] = -l[4]
    check(l, torch.zeros(6, dtype=torch.int32, device="cuda"), 32)


@pytest.mark.parametrize("low", [-float("inf"), -3.4028234663852886e38])
@pytest.mark.parametrize("V", [50, 32003, 151936])
def test_masked_rows(cuda, low, V):
    """All but a few tokens masked away, down to one, in one slice of the row or in several."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(V)
    l = torch.full((5, V), low, device="cuda")
    for r, n in enumerate((1, 2, 9, 12, 40)):
        at = torch.randperm(V, generator=g, device="cuda")[:n]
        l[r, at] = torch.randn((n,), generator=g, device="cuda")
    first = l.argmax(-1).int()
    lp, ent, ti, _ = check(l, torch.stack([first, (first + 1) % V], 1).contiguous(), 10)
    assert lp[0, 0].item() == 0.0 and ent[0].item() == 0.0
    if low == -float("inf"):
        assert lp[0, 1].item() == low and ti[0, 1:].tolist() == [-1] * 9


def test_rows_without_a_value(cuda):
    import torch
    import large_model_b200 as m
    inf = float("inf")
    l = torch.randn((5, 30000), device="cuda")
    l[0] = -inf
    l[1, 77] = float("nan")
    l[2, 20001] = inf
    l[3] = float("nan")
    ids = torch.tensor([[0, 77], [0, 77], [0, 20001], [0, 1], [0, 1]], dtype=torch.int32, device="cuda")
    lp, ent, ti, tl = m.logprobs(l, ids, top=3)
    assert (lp[0] == -inf).all() and ent[0] == 0 and (ti[0] == -1).all() and (tl[0] == -inf).all()
    for r in (1, 2, 3):
        assert lp[r].isnan().all() and ent[r].isnan() and tl[r].isnan().all(), r
    assert ti[2, 0].item() == 20001 and (ti[3] == -1).all()
    assert ti[1].tolist() == _top(l[1:2].cpu().numpy(), 3)[0].tolist()
    assert lp[4].isfinite().all() and ent[4].isfinite()


def test_a_sure_token_keeps_its_digits(cuda):
    """log p near 0 is the others' share: it does not vanish beside 1."""
    import torch
    import large_model_b200 as m
    l = torch.full((3, 32000), -12.0, device="cuda")
    l[0, 5], l[1, 31999], l[2, 16000] = 12.0, 25.0, 40.0
    lp, ent, _, _ = m.logprobs(l, l.argmax(-1).int(), top=1)
    z = 31999 * torch.exp(torch.tensor([-24.0, -37.0, -52.0], dtype=torch.float64, device="cuda"))
    want = -torch.log1p(z)
    assert ((lp[:, 0].double() / want - 1).abs() <= E * (52 + 2 * 52 + 4)).all()
    went = torch.log1p(z) + z / (1 + z) * torch.tensor([24.0, 37.0, 52.0], device="cuda")
    assert ((ent.double() / went - 1).abs() <= E * 4 * (52 + 2 * 52 + 4)).all()


def test_bad_ids(cuda):
    import torch
    import large_model_b200 as m
    l = torch.randn((2, 100), device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    ids = torch.tensor([[0, -1, 99], [100, 1 << 30, 5]], dtype=torch.int32, device="cuda")
    lp = m.logprobs(l, ids, err=err)[0]
    assert err.item() == 4
    assert lp.isnan().tolist() == [[False, True, False], [True, True, False]]


def test_streams_graphs_and_repeats(cuda):
    import torch
    import large_model_b200 as m
    l = torch.randn((9, 151936), device="cuda")
    ids = torch.arange(9, device="cuda").int()
    want = m.logprobs(l, ids, top=10)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = m.logprobs(l, ids, top=10, stream=s)
    s.synchronize()
    out = tuple(torch.empty_like(x) for x in want)
    m.logprobs(l, ids, top=10, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        m.logprobs(l, ids, top=10, out=out)
    for x in out:
        x.zero_()
    graph.replay()
    torch.cuda.synchronize()
    for a, b, c in zip(want, got, out):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_refusals(cuda):
    import torch
    import large_model_b200 as m
    l = torch.randn((2, 100), device="cuda")
    ids = torch.zeros(2, dtype=torch.int32, device="cuda")
    for bad in (lambda: m.logprobs(l.half(), ids), lambda: m.logprobs(l, ids.long()), lambda: m.logprobs(l, ids[:1]),
                lambda: m.logprobs(l.cpu(), ids), lambda: m.logprobs(l.T, ids)):
        with pytest.raises(ValueError):
            bad()
    for kw in (dict(temp=0.0), dict(top=33), dict(top=-1)):
        with pytest.raises((m.QmsCudaError, RuntimeError)):
            m.logprobs(l, ids, **kw)
    lp = m.logprobs(l[:0], ids[:0], top=3)
    assert lp[0].shape == (0, 1) and lp[2].shape == (0, 3)
