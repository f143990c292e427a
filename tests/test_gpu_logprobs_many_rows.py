"""Log probabilities of many rows on a B200 through the C ABI (qms_cuda_logprobs): rows that are read once, through two buffers per warp,
with the likeliest kept on the way, by one, two, four or eight CTAs each; against their definition in 64 bits. Few different rows are
repeated: every copy that starts as far from a 16-byte boundary has the same bits, whatever its neighbours and the order in which its
warps meet.

Bounds as in test_gpu_logprobs.py, with the roundings of a sum counted: a lane adds every 512 nc-th value to one of two sums, nc CTAs per
row, and brings the sum under another base at most once in each of its V / (4096 nc) chunks: one rounding, 2 e |d| for the exponent d (all d together are
at most |x| and 4, as counted there) and the exponential's 4 e, so up to 6 e; the lanes, warps and CTAs join in less than 30 more. So N = V / (512 nc) + 7
V / (4096 nc) + 30 in place of 52."""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_logprobs import E, _top

pytestmark = pytest.mark.gpu
INF = float("inf")


def ctas(rows, V):
    nc = 1
    while nc < 8 and V > 4096 * nc and rows * nc < 500:
        nc *= 2
    return nc


def want(l, temp, rows):
    import torch
    V = l.shape[1]
    nc = ctas(rows, V)
    N = -(-V // (512 * nc)) + 7 * -(-V // (4096 * nc)) + 30
    x = l.double() / temp
    x = x - x.amax(-1, keepdim=True)
    lz = torch.logsumexp(x, -1, keepdim=True)
    p = torch.exp(x - lz)
    px = torch.where(p > 0, p * x, 0.0)
    A, Q = -px.sum(-1, keepdim=True), torch.where(p > 0, px * x, 0.0).sum(-1, keepdim=True)
    lp = x - lz
    tol = E * (N + 2 * A + 3 * x.abs() + 2 * lz + lp.abs())
    return lp, tol, (lz + A)[:, 0], (E * (N + 2 * A + 2 * lz + (N + 2) * (A + 3) + 2 * Q + (N + 2 * A) * A + 2 * (lz + A)))[:, 0]


def strided(l, rows, ld, off):
    """l's rows in turn, at distance ld from `off` values behind a 16-byte boundary, NaN between them."""
    import torch
    V = l.shape[1]
    base = torch.full((rows * ld + 8,), float("nan"), device="cuda")
    out = base[off:off + rows * ld].view(rows, ld)[:, :V]
    out.copy_(l.repeat(-(-rows // l.shape[0]), 1)[:rows])
    return out


def call(l, ids, top, rows, temp=1.0, ld=None, off=0, **kw):
    """The results for l's rows at each of 4 distances from a 16-byte boundary, [4 n]; those of the copies are the same."""
    import torch
    import large_model_b200 as m
    n, V = l.shape
    many = ids.repeat(-(-rows // n), 1)[:rows].contiguous()
    got = m.logprobs(strided(l, rows, ld or V, off), many, top=top, temp=temp, **kw)
    copies = torch.arange(rows, device="cuda") % (4 * n)
    for t in got:
        assert torch.equal(t.view(torch.int32), t.view(torch.int32)[copies]), "copies of a row differ"
    return tuple(t[:4 * n] for t in got)


def check(l, ids, top, rows, temp=1.0, **kw):
    import torch
    lp, ent, ti, tl = call(l, ids, top, rows, temp, **kw)
    wlp, tol, went, tent = (x.repeat(4, *[1] * (x.dim() - 1)) for x in want(l, temp, rows))
    ids = ids.repeat(4, 1)
    w = wlp.gather(1, ids.long())
    assert torch.where(lp.double() == w, True, (lp.double() - w).abs() <= tol.gather(1, ids.long())).all()
    assert ((ent.double() - went).abs() <= tent).all()
    wi = torch.from_numpy(_top(l.cpu().numpy(), top)).cuda().repeat(4, 1)
    assert torch.equal(ti.long(), wi)
    w = wlp.gather(1, wi.clamp(min=0))
    assert torch.where(wi < 0, tl == -INF, (tl.double() - w).abs() <= tol.gather(1, wi.clamp(min=0))).all()
    return lp, ent, ti, tl


SHAPES = [(512, 32003), (300, 32003), (150, 32003), (80, 32003), (512, 151936), (80, 151936)]


def randn(n, V, seed, scale=3.0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    return scale * torch.randn((n, V), generator=g, device="cuda"), torch.randint(0, V, (n, 2), generator=g, device="cuda").int()


@pytest.mark.parametrize("rows,V", SHAPES + [(512, 300007)])
@pytest.mark.parametrize("top", [0, 1, 10, 32])
def test_random_rows(cuda, rows, V, top):
    check(*randn(7, V, V + top), top, rows, temp=0.7)


@pytest.mark.parametrize("V", [1, 2, 3, 31, 127, 513, 1000, 2047, 2049, 4095, 4097, 4603, 8192, 12289])
@pytest.mark.parametrize("rows", [75, 600])
def test_sizes(cuda, V, rows):
    for top in (1, 10, 32):
        check(*randn(7, V, V), top, rows)


@pytest.mark.parametrize("rows,V", SHAPES)
@pytest.mark.parametrize("over,off", [(1, 0), (2, 1), (5, 2), (8, 3)])
def test_strides(cuda, rows, V, over, off):
    check(*randn(5, V, off), 10, rows, ld=V + over, off=off)


@pytest.mark.parametrize("rows,V", SHAPES + [(600, 40), (75, 3001), (600, 4097)])
def test_equal_values_go_to_the_lowest_id(cuda, rows, V):
    import torch
    g = torch.Generator(device="cuda").manual_seed(V)
    l = torch.randint(-3, 3, (7, V), generator=g, device="cuda").float()
    l[1] = 2.0                                               # nothing but equals
    l[2] = -0.0
    l[2, ::2] = 0.0                                          # 0 and -0 are equal
    l[3, V // 2:] = 7.0
    l[4] = torch.arange(V, device="cuda").float()            # ascending, descending: every chunk is past the bound, or none is
    l[5] = -l[4]
    l[6] = torch.arange(V, device="cuda").div(100, rounding_mode="floor").float()
    check(l, torch.zeros((7, 1), dtype=torch.int32, device="cuda"), 32, rows)
    check(l, torch.zeros((7, 1), dtype=torch.int32, device="cuda"), 7, rows, ld=V + 3, off=1)


@pytest.mark.parametrize("low", [-INF, -3.4028234663852886e38])
@pytest.mark.parametrize("rows,V", SHAPES + [(600, 50)])
def test_masked_rows(cuda, low, rows, V):
    import torch
    g = torch.Generator(device="cuda").manual_seed(V)
    l = torch.full((6, V), low, device="cuda")
    for r, n in enumerate((1, 2, 9, 12, 40)):
        at = torch.randperm(V, generator=g, device="cuda")[:n]
        l[r, at] = torch.randn((n,), generator=g, device="cuda")
    l[5, V - 2] = 1.5                                        # behind the last group of 4, or before the first
    l[5, 1] = 0.5
    first = l.argmax(-1).int()
    lp, ent, ti, _ = check(l, torch.stack([first, (first + 1) % V], 1).contiguous(), 10, rows, ld=V + 1, off=3)
    assert lp[0, 0].item() == 0.0 and ent[0].item() == 0.0
    if low == -INF:
        assert lp[0, 1].item() == low and ti[0, 1:].tolist() == [-1] * 9


@pytest.mark.parametrize("rows,V", SHAPES)
def test_rows_without_a_value(cuda, rows, V):
    import torch
    l, _ = randn(6, V, 1, 1.0)
    l[0] = -INF
    l[1, 77] = float("nan")
    l[2, V - 1] = INF
    l[3] = float("nan")
    l[5, [0, 9000]] = INF
    ids = torch.tensor([[0, 77], [0, 77], [0, V - 1], [0, 1], [0, 1], [0, 9000]], dtype=torch.int32, device="cuda")
    for lp, ent, ti, tl in zip(*(t.view(4, 6, *t.shape[1:]) for t in call(l, ids, 3, rows))):
        assert (lp[0] == -INF).all() and ent[0] == 0 and (ti[0] == -1).all() and (tl[0] == -INF).all()
        for r in (1, 2, 3, 5):
            assert lp[r].isnan().all() and ent[r].isnan() and tl[r].isnan().all(), r
        assert ti[2, 0].item() == V - 1 and (ti[3] == -1).all() and ti[5, :2].tolist() == [0, 9000]
        assert ti[1].tolist() == _top(l[1:2].cpu().numpy(), 3)[0].tolist()
        assert lp[4].isfinite().all() and ent[4].isfinite()


@pytest.mark.parametrize("rows", [512, 300, 150, 80])
def test_a_sure_token_keeps_its_digits(cuda, rows):
    """32,000 values: N is at most 63 + 56 + 30 < 150."""
    import torch
    l = torch.full((3, 32000), -12.0, device="cuda")
    l[0, 5], l[1, 31999], l[2, 16000] = 12.0, 25.0, 40.0
    lp, ent, _, _ = call(l, l.argmax(-1, keepdim=True).int(), 1, rows)
    x = torch.tensor([24.0, 37.0, 52.0], dtype=torch.float64, device="cuda").repeat(4)
    z = 31999 * torch.exp(-x)
    assert ((lp[:, 0].double() / -torch.log1p(z) - 1).abs() <= E * (150 + 2 * 52 + 4)).all()
    went = torch.log1p(z) + z / (1 + z) * x
    assert ((ent.double() / went - 1).abs() <= E * 4 * (150 + 2 * 52 + 4)).all()


@pytest.mark.parametrize("rows,V", [(300, 32003), (600, 1000)])
def test_more_ids_than_threads_and_bad_ones(cuda, rows, V):
    import torch
    l, _ = randn(3, V, 8)
    ids = torch.arange(700, device="cuda").int().repeat(3, 1) % V
    check(l, ids, 2, rows)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    ids[1, 5], ids[1, 600], ids[2, 299] = -1, V, 1 << 30
    lp = call(l, ids, 2, rows, err=err)[0]
    assert err.item() == 4
    assert lp.isnan().nonzero().tolist() == [[3 * c + r, i] for c in range(4) for r, i in ((1, 5), (1, 600), (2, 299))]


@pytest.mark.parametrize("rows,V", [(512, 32003), (150, 32003)])
def test_streams_and_graphs(cuda, rows, V):
    import torch
    import large_model_b200 as m
    l, ids = randn(rows, V, 5)
    want = m.logprobs(l, ids, top=10)
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    a = m.logprobs(l, ids, top=10, stream=other)             # two at once
    b = m.logprobs(l, ids, top=10)
    torch.cuda.synchronize()
    out = tuple(torch.empty_like(x) for x in want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        m.logprobs(l, ids, top=10, out=out)
        m.logprobs(l, ids, top=10, out=out)
    for _ in range(3):
        for x in out:
            x.zero_()
        graph.replay()
    torch.cuda.synchronize()
    for w, x, y, z in zip(want, a, b, out):
        assert torch.equal(w, x) and torch.equal(w, y) and torch.equal(w, z)
