"""Paged attention on a B200 at inputs that few callers meet: values that are not finite beside positions that nobody sees,
scores that jump, sums that are exact, orders of magnitude that differ. Formula and bounds as in test_gpu_paged.py,
unless a test says otherwise."""
from __future__ import annotations

import pytest

from test_gpu_paged import make, reference

pytestmark = pytest.mark.gpu


def put(pages, batch, b, p, h, d, value, what="v"):
    """One value of K or V of position p of sequence b."""
    page = pages.k.shape[1]
    getattr(pages, what)[batch.table[b, p // page].long(), p % page, h, d] = value


# ---- values that are not finite -----------------------------------------------------------------------

@pytest.mark.parametrize("typ", ["f16", "f32"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("G,n,prefix,kv,p,page", [(8, 3, 40, 60, 59, 64), (16, 1, 24, 30, 26, 64), (16, 2, 24, 31, 30, 64), (16, 1, 50, 60, 55, 64),
                                                  (8, 4, 50, 62, 59, 64), (16, 1, 20, 27, 25, 32), (16, 2, 100, 127, 126, 128)])
def test_value_behind_a_prompt_that_ends_inside_a_page(cuda, typ, bad, G, n, prefix, kv, p, page):
    """A tile of own positions that begins with shared ones, which its rows do not see: what they see in it still shows."""
    import torch
    import large_model_b200 as m
    pages, batch, q, K, V = make([n], [kv], typ=typ, G=G, Hk=1, page=page, prefix=prefix)
    put(pages, batch, 0, p, 0, 7, bad)
    V[0][p, 0, 7] = 0
    out = m.paged_attention(pages, batch, q, G).view(n, G, 128)
    batch.status()
    want, tol = (x.view(n, G, 128) for x in reference([n], [kv], q, K, V, G, 128 ** -0.5))
    for i in range(n):
        if kv - n + i >= p:
            assert not torch.isfinite(out[i, :, 7]).any()
            out[i, :, 7] = want[i, :, 7].float()
    assert ((out.double() - want).abs() <= tol + want.abs() * 2.0 ** -24).all()


@pytest.mark.parametrize("typ", ["f16", "f32"])
@pytest.mark.parametrize("G,n,kv", [(16, 1, 30), (16, 2, 30), (8, 2, 28), (16, 1, 62)])
def test_value_behind_a_bad_page(cuda, typ, G, n, kv):
    """The first page does not exist: the value behind it still shows."""
    import torch
    import large_model_b200 as m
    pages, batch, q, K, V = make([n], [kv], typ=typ, G=G, Hk=1)
    p = kv - 3
    put(pages, batch, 0, p, 0, 7, float("inf"))
    V[0][p, 0, 7] = 0
    batch.table[0, 0] = -1
    out = m.paged_attention(pages, batch, q, G).view(n, G, 128)
    with pytest.raises(m.QmsCudaError, match="0x2"):
        batch.status()
    want, tol = (x.view(n, G, 128) for x in reference([n], [kv - 16], q, [K[0][16:]], [V[0][16:]], G, 128 ** -0.5))
    assert not torch.isfinite(out[..., 7]).any()
    out[..., 7] = want[..., 7].float()
    assert ((out.double() - want).abs() <= tol + want.abs() * 2.0 ** -24).all()


@pytest.mark.parametrize("G,n,kv,p", [(16, 1, 40, 35), (16, 2, 40, 34), (16, 4, 50, 33), (8, 1, 5, 2), (16, 8, 40, 30)])
def test_value_beside_what_nobody_sees(cuda, G, n, kv, p):
    """fp32 cache: V of a seen position is inf in a tile whose other rows, past the sequence, hold large numbers."""
    import torch
    import large_model_b200 as m
    pages, batch, q, K, V = make([n], [kv], typ="f32", G=G, Hk=1, page=64, garbage=1e30)
    put(pages, batch, 0, p, 0, 7, float("inf"))
    V[0][p, 0, 7] = 0
    out = m.paged_attention(pages, batch, q, G).view(n, G, 128)
    batch.status()
    want, tol = (x.view(n, G, 128) for x in reference([n], [kv], q, K, V, G, 128 ** -0.5))
    assert not torch.isfinite(out[..., 7]).any()
    out[..., 7] = want[..., 7].float()
    assert ((out.double() - want).abs() <= tol + want.abs() * 2.0 ** -24).all()


# ---- the same in every kernel ---------------------------------------------------------------------------
# (own positions: rows of a tile x positions x sequences; idle sequences count, and make one unit of a sequence's positions)

KERNELS = [("f16", 1), ("f32", 1), ("f16", 2), ("f32", 2), ("f16", 4), ("f32", 4), ("f16", 8), ("f32", 8), ("f16", 16)]
# tokens of 16 q heads each: 16, 32 or 64 rows over mma.sync; 128 rows over tcgen05, two streams of tiles; 256 rows, one stream per 128


def one_unit(n, kv, **kw):
    """One sequence of n tokens, and so many idle ones that all its positions are one unit of work."""
    return make([n] + [0] * 69, [kv] + [0] * 69, G=16, Hk=2, page=64, **kw)


def scores(pages, batch, q, K, s):
    """q and K such that the scores of every row, in powers of two at scale ln 2, are s[position] (fp16 values)."""
    import torch
    q.zero_()
    q[:, ::pages.head_dim] = 1.0
    kv = len(s)
    K[0].zero_()
    K[0][:, :, 0] = s[:, None].to(K[0].dtype)
    j = torch.arange(kv, device="cuda")
    pages.k[batch.table[0].long()[j // 64], j % 64] = K[0]


@pytest.mark.parametrize("typ,n,jump", [("f16", 16, 45), ("f16", 16, 90), ("f16", 8, 140), ("f32", 8, 140), ("f16", 2, 140), ("f32", 2, 140)])
def test_value_before_scores_rise_by_far(cuda, typ, n, jump):
    """V of an early position is inf and seen by all rows, and a later score takes all the weight: inf times any weight is not
    finite, whatever became of the early sums meanwhile."""
    import math
    import torch
    import large_model_b200 as m
    kv, D = 2300, 128
    pages, batch, q, K, V = one_unit(n, kv, typ=typ)
    for late in (70, 130, 1100, 2000):
        s = torch.zeros(kv, device="cuda")
        s[late] = jump
        scores(pages, batch, q, K, s)
        put(pages, batch, 0, 10, 1, 7, float("inf"))
        out = m.paged_attention(pages, batch, q, 32, scale=math.log(2)).view(n, 2, 16, D)
        batch.status()
        assert not torch.isfinite(out[:, 1, :, 7]).any(), late
        assert torch.isfinite(out[:, 0]).all() and torch.isfinite(out[:, 1, :, 8:]).all(), late


@pytest.mark.parametrize("typ,n", [k for k in KERNELS if k[1] >= 8])
@pytest.mark.parametrize("up", [20, 25, 30])
def test_scores_that_jump_inside_a_tile(cuda, typ, n, up):
    """A tile of scores 6 above those before it, and at its end one far above: the 6s keep their share, 2^(6 - up) each of the
    row. Scores are exact, so a weight is off by its own roundings, some 25 * 2^-24 for the exponent: 4e-6 of max |V|."""
    import math
    import torch
    import large_model_b200 as m
    kv, TP = 1152, 128 if typ == "f16" else 64
    pages, batch, q, K, V = one_unit(n, kv, typ=typ)
    for tile in (2, 3, 8):
        s = torch.zeros(kv, device="cuda")
        s[tile * TP:(tile + 1) * TP - 32] = 6
        s[(tile + 1) * TP - 5] = up
        scores(pages, batch, q, K, s)
        out = m.paged_attention(pages, batch, q, 32, scale=math.log(2))
        batch.status()
        want, _ = reference([n], [kv], q, K, V, 16, math.log(2))
        assert (out.double() - want).abs().max() <= 4e-6 * V[0].abs().max(), tile


# ---- sums that are exact -------------------------------------------------------------------------------

@pytest.mark.parametrize("typ,n", KERNELS)
@pytest.mark.parametrize("kv", [1000, 2300, 5000, 9000])
def test_equal_scores_over_equal_values(cuda, typ, n, kv):
    """The mean of the same number: the sums are exact, and some four roundings of 2^-24 are left."""
    import torch
    import large_model_b200 as m
    for prefix in (0, kv - kv // 4):
        pages, batch, q, K, V = one_unit(n, kv, typ=typ)
        batch.desc.prefix_len = prefix
        j = torch.arange(kv, device="cuda")
        pages.v[batch.table[0].long()[j // 64], j % 64] = 1.0
        out = m.paged_attention(pages, batch, q, 32, scale=0.0)
        batch.status()
        assert (out - 1).abs().max() <= 1e-6, prefix


@pytest.mark.parametrize("typ,n", KERNELS)
@pytest.mark.parametrize("top", [30, 40, 60])
def test_one_position_far_above_the_others(cuda, typ, n, top):
    """The first position's weight is 2^top of another's, over 1000 to 9000 positions."""
    import math
    import torch
    import large_model_b200 as m
    for kv in (1000, 9000):
        pages, batch, q, K, V = one_unit(n, kv, typ=typ)
        s = torch.zeros(kv, device="cuda")
        s[0] = top
        scores(pages, batch, q, K, s)
        out = m.paged_attention(pages, batch, q, 32, scale=math.log(2))
        batch.status()
        want, _ = reference([n], [kv], q, K, V, 16, math.log(2))
        assert (out.double() - want).abs().max() <= 1e-6 * V[0].abs().max(), kv


@pytest.mark.parametrize("typ,n", KERNELS)
@pytest.mark.parametrize("kv", [2300, 9000])
def test_values_of_one_sign(cuda, typ, n, kv):
    """All products of a sum have its sign, so that what the tensor cores cut off each adds up: 16 products of an addition at some 2^-27
    of the sum each, 64 additions of hi terms while it grows from 0, is 64 * 16 * 2^-27 / 2 = 4e-6 of an output; 8e-6 with the
    additions themselves and the scores' share."""
    import torch
    import large_model_b200 as m
    for kind in range(2):
        pages, batch, q, K, V = one_unit(n, kv, typ=typ)
        if kind:
            V[0].abs_()
        else:
            V[0].mul_(0.1).add_(1)
        j = torch.arange(kv, device="cuda")
        pages.v[batch.table[0].long()[j // 64], j % 64] = V[0]
        out = m.paged_attention(pages, batch, q, 32)
        batch.status()
        want, _ = reference([n], [kv], q, K, V, 16, 128 ** -0.5)
        assert (out.double() - want).norm() <= 8e-6 * want.norm(), kind


# ---- orders of magnitude -------------------------------------------------------------------------------

@pytest.mark.parametrize("n", [1, 2, 4, 8])
def test_small_q_and_large_k(cuda, n):
    """fp32: q near the smallest normal numbers, K so large that the scores are ordinary."""
    import torch
    import large_model_b200 as m
    kv = 700
    pages, batch, q, K, V = one_unit(n, kv, typ="f32")
    q *= 2.0 ** -120
    K[0] *= 2.0 ** 120
    j = torch.arange(kv, device="cuda")
    pages.k[batch.table[0].long()[j // 64], j % 64] = K[0]
    out = m.paged_attention(pages, batch, q, 32)
    batch.status()
    want, tol = reference([n], [kv], q, K, V, 16, 128 ** -0.5)
    assert ((out.double() - want).abs() <= tol).all()


# ---- K that is not finite ------------------------------------------------------------------------------

@pytest.mark.parametrize("typ,n", KERNELS)
def test_infinite_scores(cuda, typ, n):
    """K of one seen position is infinite in one value. A row whose q there makes the score -inf gives the position no weight; where it
    makes +inf, or q is 0 there, nothing finite is left (inf - inf, 0 * inf)."""
    import torch
    import large_model_b200 as m
    kv, p = 700, 321
    for bad in (float("inf"), -float("inf")):
        pages, batch, q, K, V = one_unit(n, kv, typ=typ)
        x = q.view(n, 2, 16, 128)
        x[0, 0, 3, 5] = 0.0
        x[0, 0, 4, 5] = 1e-30
        x[0, 0, 5, 5] = -1e-30
        put(pages, batch, 0, p, 0, 5, bad, "k")
        out = m.paged_attention(pages, batch, q, 32).view(n, 2, 16, 128)
        batch.status()
        keep = torch.arange(kv, device="cuda") != p
        # (the reference: head 1 as it is; head 0 without the position, whose weight is 0)
        full, tol1 = reference([n], [kv], q, K, V, 16, 128 ** -0.5)
        less = torch.zeros_like(full).view(n, 2, 16, 128)
        tol = torch.zeros_like(less)
        for i in range(n):
            last = kv - n + i + 1
            a, b = reference([1], [last - 1], q[i:i + 1], [K[0][:last][keep[:last]]], [V[0][:last][keep[:last]]], 16, 128 ** -0.5)
            less[i], tol[i] = a.view(2, 16, 128), b.view(2, 16, 128)
        less[:, 1], tol[:, 1] = full.view(n, 2, 16, 128)[:, 1], tol1.view(n, 2, 16, 128)[:, 1]
        none = x[:, 0, :, 5] * bad < 0               # [n, 16]: score -inf
        ok = torch.ones((n, 2, 16), dtype=torch.bool, device="cuda")
        ok[:, 0] = none
        assert not torch.isfinite(out[~ok]).any()
        assert ((out.double() - less).abs() <= tol)[ok].all()


# ---- lengths -------------------------------------------------------------------------------------------

@pytest.mark.parametrize("typ,n", KERNELS)
def test_lengths_of_idle_sequences_are_checked(cuda, typ, n):
    """A sequence without rows whose length is past max_kv, or negative: reported, whichever kernel runs."""
    import torch
    import large_model_b200 as m
    pages, batch, q, K, V = one_unit(n, 700, typ=typ)
    good = m.paged_attention(pages, batch, q, 32)
    batch.status()
    for value in (701, -1):
        batch.kv_len[69] = value
        out = m.paged_attention(pages, batch, q, 32)
        with pytest.raises(m.QmsCudaError, match="0x1"):
            batch.status()
        assert torch.equal(out, good)
