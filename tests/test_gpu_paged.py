"""The paged KV cache on a B200 through the C ABI: qms_cuda_paged_append and qms_cuda_paged_attention against
their formulas in 64 bits, at the sizes, masks and layouts where they can go wrong.

Bounds. Attention: with e the unit roundoff 2^-24, a score (a dot of head_dim fp32 products, scaled) is off by
at most head_dim e times A = scale * sum |q k|, in practice by a few e A, and a weight exp(s - max) by as much
relatively; the output is a weighted mean of V, so it is off by at most that times max |V|, plus a
few roundings. The tests allow (16 e A + 16 e) max |V|, A and max |V| over what the row sees. Append: three
roundings of the normalised value and three of the rotation, 8 e (|x1| + |x2|), then half an ulp of the
cache type."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
E24 = 2.0 ** -24


def make(qs, kv, *, G=2, Hk=2, D=128, page=16, typ="f16", prefix=0, seed=0, order="nhd", garbage=float("nan"),
         pad=0, qscale=1.0):
    """A batch over a pool whose every value is `garbage` except at positions that some sequence owns."""
    import torch
    import large_model_b200 as m
    g = torch.Generator(device="cuda").manual_seed(seed)
    B, T = len(qs), sum(qs) + pad
    dt = torch.float16 if typ == "f16" else torch.float32
    shared = prefix // page
    need = [max(0, -(-n // page) - shared) for n in kv]
    perm = np.random.default_rng(seed).permutation(shared + sum(need) + 2).astype(np.int32)
    table = np.full((B, max(1, shared + max(need, default=0))), perm[-1], np.int32)
    table[:, :shared] = perm[:shared]
    at = shared
    for b in range(B):
        table[b, shared:shared + need[b]] = perm[at:at + need[b]]
        at += need[b]
    shape = (len(perm), page, Hk, D)
    if order == "nhd":
        k, v = (torch.full(shape, garbage, dtype=dt, device="cuda") for _ in range(2))
    else:                                            # heads before positions, and a gap between pages
        k, v = (torch.full((len(perm), Hk + 1, page, D), garbage, dtype=dt, device="cuda")[:, :Hk].transpose(1, 2)
                for _ in range(2))
    K, V = [], []
    for b in range(B):
        kb, vb = (torch.randn((kv[b], Hk, D), generator=g, device="cuda").to(dt) for _ in range(2))
        n = min(prefix, kv[b])
        if b:
            kb[:n], vb[:n] = K[0][:n], V[0][:n]
        j = torch.arange(kv[b], device="cuda")
        pg = torch.from_numpy(table[b]).cuda().long()[j // page]
        k[pg, j % page], v[pg, j % page] = kb, vb
        K.append(kb)
        V.append(vb)
    start = torch.tensor([0] + np.cumsum(qs).tolist(), dtype=torch.int32, device="cuda")
    q = qscale * torch.randn((T, Hk * G * D), generator=g, device="cuda")
    batch = m.PagedBatch(start, torch.tensor(kv, dtype=torch.int32, device="cuda"), torch.from_numpy(table).cuda(), T,
                         max(qs, default=0), max(kv, default=0), prefix)
    return m.KvPages(k, v), batch, q, K, V


def reference(qs, kv, q, K, V, G, scale):
    """Row by row in 64 bits, and the bound on each row."""
    import torch
    Hk, D = K[0].shape[1:]
    out = torch.zeros((q.shape[0], Hk, G, D), dtype=torch.float64, device="cuda")
    tol = torch.zeros((q.shape[0], Hk, G, 1), dtype=torch.float64, device="cuda")
    t = 0
    for b, n in enumerate(qs):
        for i in range(n):
            p = kv[b] - n + i
            if p >= 0:
                x, k, v = q[t].double().view(Hk, G, D), K[b][:p + 1].double(), V[b][:p + 1].double()
                s = torch.einsum("hgd,jhd->hgj", x, k) * scale
                out[t] = torch.einsum("hgj,jhd->hgd", torch.softmax(s, -1), v)
                A = (torch.einsum("hgd,jhd->hgj", x.abs(), k.abs()) * abs(scale)).amax(-1)
                tol[t, ..., 0] = (16 * A + 16) * E24 * v.abs().amax((0, 2))[:, None]
            t += 1
    return out.flatten(1), tol.expand_as(out).flatten(1)


def check(qs, kv, scale=None, **kw):
    import torch
    import large_model_b200 as m
    pages, batch, q, K, V = make(qs, kv, **kw)
    G, D = kw.get("G", 2), kw.get("D", 128)
    sc = D ** -0.5 if scale is None else scale
    H = G * kw.get("Hk", 2)
    out = m.paged_attention(pages, batch, q, H, scale=scale)
    batch.status()
    want, tol = reference(qs, kv, q, K, V, G, sc)
    assert torch.isfinite(out).all()
    over = ((out.double() - want).abs() - tol).max().item()
    assert over <= 0, f"{over} over the bound (worst error {(out.double() - want).abs().max().item()})"
    again = m.paged_attention(pages, batch, q, H, scale=scale)
    assert torch.equal(out.view(torch.int32), again.view(torch.int32)), "two runs differ"
    return out


@pytest.mark.parametrize("typ", ["f16", "f32"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("G", [1, 3, 8, 16])
def test_attention_one_token(cuda, typ, D, G):
    check([1, 1, 1, 1], [1, 2, 63, 333], typ=typ, D=D, G=G, seed=G)


@pytest.mark.parametrize("typ", ["f16", "f32"])
@pytest.mark.parametrize("page", [1, 4, 16, 128, 512])
def test_attention_page_sizes(cuda, typ, page):
    check([1, 3, 0, 2], [200, 129, 0, 17], typ=typ, page=page, seed=page)


@pytest.mark.parametrize("typ", ["f16", "f32"])
@pytest.mark.parametrize("prefix", [0, 1, 16, 100, 127, 128, 129, 300])
def test_attention_shared_prompt(cuda, typ, prefix):
    qs, new = [1, 4, 0, 2, 1], [5, 4, 0, 130, 1]
    check(qs, [prefix + n for n in new], typ=typ, prefix=prefix, G=8, seed=prefix)


@pytest.mark.parametrize("typ", ["f16", "f32"])
@pytest.mark.parametrize("D", [64, 128])
def test_attention_many_rows_one_prompt(cuda, typ, D):
    """More rows than a tile holds, a number that divides nothing, over several tiles of positions."""
    B = 37
    qs = [(5 * b + 2) % 4 for b in range(B)]
    check(qs, [700 + n + (91 * b) % 57 for b, n in enumerate(qs)], typ=typ, prefix=700, G=16, Hk=2, D=D, seed=D)


@pytest.mark.parametrize("typ", ["f16", "f32"])
@pytest.mark.parametrize("n,kv", [(70, 70), (65, 300), (129, 129), (200, 1111)])
def test_attention_prompt_chunks(cuda, typ, n, kv):
    check([n], [kv], typ=typ, G=4, Hk=1, seed=n)
    check([n, 1, 31], [kv, 40, 31], typ=typ, G=5, Hk=2, page=64, seed=n)


@pytest.mark.parametrize("typ", ["f16", "f32"])
def test_attention_prompt_inside_the_shared_part(cuda, typ):
    """The shared positions are themselves the rows of the first sequence: the mask crosses them."""
    check([90, 1], [90, 91], typ=typ, prefix=90, G=4)
    check([150], [200], typ=typ, prefix=130, G=2)


@pytest.mark.parametrize("typ", ["f16", "f32"])
def test_attention_layouts(cuda, typ):
    check([1, 5, 40], [77, 130, 90], typ=typ, order="hnd", prefix=33, G=16, Hk=2)
    check([1, 5, 40], [77, 130, 90], typ=typ, order="hnd", garbage=float("inf"), D=64, G=6, Hk=3)


@pytest.mark.parametrize("typ", ["f16", "f32"])
def test_attention_long(cuda, typ):
    check([1, 2], [16001, 9000], typ=typ, G=16, Hk=1, page=64)


@pytest.mark.parametrize("typ", ["f16", "f32"])
def test_attention_scores(cuda, typ):
    """One position takes all the weight; equal scores; q beyond the range of 16-bit types."""
    check([1, 3], [300, 64], typ=typ, G=16, qscale=200.0)
    check([1, 3], [300, 64], typ=typ, G=16, scale=0.0)
    check([70, 3], [300, 64], typ=typ, G=2, scale=0.0)
    check([1, 70], [300, 90], typ=typ, G=2, qscale=1e30, scale=1e-31)
    check([1, 70], [300, 90], typ=typ, G=2, qscale=1e-30, scale=1e29)
    check([1, 3], [300, 64], typ=typ, G=4, scale=-0.1)


@pytest.mark.parametrize("typ", ["f16", "f32"])
@pytest.mark.parametrize("n", [3, 40, 130])
def test_attention_rows_that_see_nothing(cuda, typ, n):
    """Idle sequences, padding rows and rows before position 0 are zero; the others are not disturbed."""
    import torch
    import large_model_b200 as m
    qs, kv = [0, n, 2, 0], [0, n - 2, 50, 7]
    pages, batch, q, K, V = make(qs, kv, typ=typ, G=4, pad=3)
    out = torch.full((sum(qs) + 3, 8 * 128), float("nan"), device="cuda")
    m.paged_attention(pages, batch, q, 8, out=out)
    batch.status()
    want, tol = reference(qs, kv, q, K, V, 4, 128 ** -0.5)
    assert (out[:2] == 0).all() and (out[-3:] == 0).all()
    assert ((out.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("typ", ["f16", "f32"])
@pytest.mark.parametrize("n,prefix", [(2, 0), (5, 40), (64, 0), (140, 0), (9, 50)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_attention_masked_values_have_no_effect(cuda, typ, n, prefix, bad):
    """K and V of the newest token are not finite: only its own row may show it."""
    import torch
    import large_model_b200 as m
    kv = 45 + n
    pages, batch, q, K, V = make([n, 1], [kv, prefix + 3], typ=typ, G=16, Hk=1, prefix=prefix)
    last = batch.table[0, (kv - 1) // 16].long()
    pages.k[last, (kv - 1) % 16, 0, 5] = bad
    pages.v[last, (kv - 1) % 16, 0, 7] = bad
    K[0][-1, 0, 5] = 0                               # the other rows must not see the difference
    V[0][-1, 0, 7] = 0
    out = m.paged_attention(pages, batch, q, 16)
    batch.status()
    want, tol = reference([n, 1], [kv, prefix + 3], q, K, V, 16, 128 ** -0.5)
    keep = [i for i in range(n + 1) if i != n - 1]
    assert ((out.double() - want).abs() <= tol)[keep].all()
    assert not torch.isfinite(out[n - 1].view(16, 128)[:, 7]).any()
    # a value that a row does see: not finite where V is not, and nowhere else
    pages.k[last, (kv - 1) % 16, 0, 5] = 0
    out = m.paged_attention(pages, batch, q, 16)
    row = out[n - 1].view(16, 128)
    assert not torch.isfinite(row[:, 7]).any() and torch.isfinite(row[:, [d for d in range(128) if d != 7]]).all()
    assert ((out.double() - want).abs() <= tol)[keep].all()


@pytest.mark.parametrize("typ", ["f16", "f32"])
@pytest.mark.parametrize("prefix", [0, 4900])
def test_attention_long_units(cuda, typ, prefix):
    """So many rows that the positions are hardly cut: results of thousands of additions into one fp32 sum. Where each cuts at
    most 2^-23, on average 0.72 * 2^-24, of the sum off, 288 of them leave the outputs' 2-norm off by 288 * 0.72 * 2^-24 / 2 =
    6.2e-6 of itself; 1e-5 with the scores' share."""
    import torch
    import large_model_b200 as m
    B, n, G, Hk, D = 20, 17, 8, 8, 64
    qs, kv = [n] * B, [5300 - 13 * b for b in range(B)]
    pages, batch, q, K, V = make(qs, kv, typ=typ, G=G, Hk=Hk, D=D, prefix=prefix, seed=2)
    out = m.paged_attention(pages, batch, q, G * Hk)
    batch.status()
    want, tol = reference(qs, kv, q, K, V, G, D ** -0.5)
    assert ((out.double() - want).abs() <= tol).all()
    assert (out.double() - want).norm() <= 1e-5 * want.norm()
    for _ in range(30):                              # many units, waits in every order
        assert torch.equal(m.paged_attention(pages, batch, q, G * Hk), out)
    batch.status()


@pytest.mark.parametrize("typ", ["f16", "f32"])
@pytest.mark.parametrize("n,G,kv", [(5, 16, 700), (17, 8, 5000), (40, 1, 2100), (2, 4, 900)])
def test_attention_values_that_are_not_finite(cuda, typ, n, G, kv):
    """V of two positions of every sequence, one that only the last row sees and one that every row sees."""
    import torch
    import large_model_b200 as m
    B, Hk, D = 40, 4, 64
    qs, kvs = [n] * B, [kv - 3 * b for b in range(B)]
    pages, batch, q, K, V = make(qs, kvs, typ=typ, G=G, Hk=Hk, D=D)
    for b, x in enumerate(kvs):
        for p, d, value in ((x - 1, 7, float("nan")), (x * 2 // 3, 9, float("inf"))):
            pages.v[batch.table[b, p // 16].long(), p % 16, b % Hk, d] = value
            V[b][p, b % Hk, d] = 0
    out = m.paged_attention(pages, batch, q, G * Hk).view(B, n, Hk, G, D)
    batch.status()
    want, tol = (x.reshape(B, n, Hk, G, D) for x in reference(qs, kvs, q, K, V, G, D ** -0.5))
    for b in range(B):
        assert not torch.isfinite(out[b, -1, b % Hk, :, 7]).any() and not torch.isfinite(out[b, :, b % Hk, :, 9]).any()
        out[b, -1, b % Hk, :, 7] = want[b, -1, b % Hk, :, 7].float()
        out[b, :, b % Hk, :, 9] = want[b, :, b % Hk, :, 9].float()
    assert ((out.double() - want).abs() <= tol + want.abs() * E24).all()


@pytest.mark.parametrize("typ", ["f16", "f32"])
def test_attention_bad_arrays_are_reported(cuda, typ):
    import torch
    import large_model_b200 as m
    pages, batch, q, K, V = make([1, 40, 1], [50, 60, 33], typ=typ, G=16, Hk=1)
    good = m.paged_attention(pages, batch, q, 16)
    batch.status()
    keep = batch.table.clone()
    for bad in (-1, 10 ** 6, pages.k.shape[0]):      # a page that does not exist: not seen, and reported
        batch.table[2, 1] = bad
        out = m.paged_attention(pages, batch, q, 16)
        with pytest.raises(m.QmsCudaError, match="0x2"):
            batch.status()
        batch.table.copy_(keep)
        assert torch.equal(out[:41], good[:41])
        k, v = (x[2][torch.arange(33, device="cuda") // 16 != 1] for x in (K, V))
        want, tol = reference([1], [17], q[41:], [k], [v], 16, 128 ** -0.5)
        assert ((out[41:].double() - want).abs() <= tol).all()
    for what, value in (("kv_len", 61), ("kv_len", -5), ("q_start", -1), ("q_start", 100)):
        t = getattr(batch, what)
        was = t.clone()
        t[1 if what == "kv_len" else 2] = value
        m.paged_attention(pages, batch, q, 16)
        with pytest.raises(m.QmsCudaError, match="0x1"):
            batch.status()
        t.copy_(was)
    assert torch.equal(m.paged_attention(pages, batch, q, 16), good)
    batch.status()


# ---- the same where many rows meet many positions: the bounds of a call say so, so idle sequences (own positions) and padding
# rows (a shared prompt) make a small batch count as a large one

def crowd(qs, kv, G, Hk, prefix=0):
    """(qs, kv) with so many idle sequences that the own positions count as 3 million rows x positions."""
    rows = -(-max(qs) * G // 64) * 64
    assert max(qs) * G > 64
    n = max(0, -(-3000000 // (rows * max(1, max(kv) - prefix) * Hk)) - len(qs))
    return list(qs) + [0] * n, list(kv) + [prefix] * n


def padding(qs, G, Hk, prefix):
    """Padding rows with which the shared positions count as 3 million rows x positions."""
    return max(0, -(-3000000 // (prefix * Hk * G)) - sum(qs))


@pytest.mark.parametrize("typ", ["f16", "f32"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n,kv,G,page", [(70, 70, 1, 16), (33, 300, 2, 8), (129, 129, 1, 64), (200, 1111, 4, 16), (9, 1030, 8, 128), (17, 640, 16, 512)])
def test_attention_crowded_chunks(cuda, typ, D, n, kv, G, page):
    qs, kvs = crowd([n, 1, 31], [kv, 40, 31], G, 2)
    check(qs, kvs, typ=typ, D=D, G=G, Hk=2, page=page, seed=n)


@pytest.mark.parametrize("typ", ["f16", "f32"])
@pytest.mark.parametrize("page", [1, 2, 4, 32, 1024])
def test_attention_crowded_page_sizes(cuda, typ, page):
    qs, kvs = crowd([9, 3, 0, 2], [400, 129, 0, 17], 8, 1)
    check(qs, kvs, typ=typ, page=page, G=8, Hk=1, D=64, seed=page)


@pytest.mark.parametrize("typ", ["f16", "f32"])
@pytest.mark.parametrize("prefix", [1, 16, 100, 127, 128, 129, 300, 2100])
def test_attention_crowded_shared_prompt(cuda, typ, prefix):
    qs, new = [1, 4, 0, 2, 1], [5, 4, 0, 130, 1]
    check(qs, [prefix + n for n in new], typ=typ, prefix=prefix, G=8, D=64, seed=prefix, pad=min(12000, padding(qs, 8, 2, prefix)))


@pytest.mark.parametrize("typ", ["f16", "f32"])
def test_attention_crowded_prompt_inside_the_shared_part(cuda, typ):
    check([90, 1], [90, 91], typ=typ, prefix=90, G=4, pad=padding([91], 4, 2, 90))
    check([150], [200], typ=typ, prefix=130, G=2, pad=padding([150], 2, 2, 130))


@pytest.mark.parametrize("typ", ["f16", "f32"])
def test_attention_crowded_layouts(cuda, typ):
    qs, kv = crowd([1, 5, 40], [77, 130, 90], 16, 2, 33)
    check(qs, kv, typ=typ, order="hnd", prefix=33, G=16, Hk=2, pad=padding(qs, 16, 2, 33))
    qs, kv = crowd([1, 5, 40], [77, 130, 90], 6, 3)
    check(qs, kv, typ=typ, order="hnd", garbage=float("inf"), D=64, G=6, Hk=3)


@pytest.mark.parametrize("typ", ["f16", "f32"])
def test_attention_crowded_scores(cuda, typ):
    """One position takes all the weight; equal scores; q beyond the range of 16-bit types; scores that rise by far over the tiles."""
    import torch
    import large_model_b200 as m
    qs, kv = crowd([70, 3], [1300, 64], 2, 2)
    for kw in (dict(qscale=200.0), dict(scale=0.0), dict(qscale=1e30, scale=1e-31), dict(qscale=1e-30, scale=1e29), dict(scale=-0.1)):
        check(qs, kv, typ=typ, G=2, **kw)
    qs, kv = crowd([70, 130], [1300, 1290], 2, 2)
    pages, batch, q, K, V = make(qs, kv, typ=typ, G=2)
    for b in range(2):                               # K grows with the position, so that the maximum moves in every tile
        K[b] *= (torch.arange(kv[b], device="cuda").to(K[b].dtype) / 100)[:, None, None]
        j = torch.arange(kv[b], device="cuda")
        pages.k[batch.table[b].long()[j // 16], j % 16] = K[b]
    for scale in (0.05, 1.0):
        out = m.paged_attention(pages, batch, q, 4, scale=scale)
        batch.status()
        want, tol = reference(qs, kv, q, K, V, 2, scale)
        assert ((out.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("typ", ["f16", "f32"])
@pytest.mark.parametrize("n", [40, 130])
def test_attention_crowded_rows_that_see_nothing(cuda, typ, n):
    import torch
    import large_model_b200 as m
    qs, kv = crowd([0, n, 2, 0], [0, n - 2, 50, 7], 4, 2)
    pages, batch, q, K, V = make(qs, kv, typ=typ, G=4, pad=3)
    out = torch.full((sum(qs) + 3, 8 * 128), float("nan"), device="cuda")
    m.paged_attention(pages, batch, q, 8, out=out)
    batch.status()
    want, tol = reference(qs, kv, q, K, V, 4, 128 ** -0.5)
    assert (out[:2] == 0).all() and (out[-3:] == 0).all()
    assert ((out.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("typ", ["f16", "f32"])
@pytest.mark.parametrize("n,prefix", [(5, 40), (64, 0), (140, 0), (9, 50)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_attention_crowded_masked_values_have_no_effect(cuda, typ, n, prefix, bad):
    """K and V of the newest token are not finite: only its own row may show it."""
    import large_model_b200 as m
    kv = 45 + n
    qs, kvs = crowd([n, 1], [kv, prefix + 3], 16, 1, prefix)
    pages, batch, q, K, V = make(qs, kvs, typ=typ, G=16, Hk=1, prefix=prefix, pad=padding(qs, 16, 1, prefix) if prefix else 0)
    last = batch.table[0, (kv - 1) // 16].long()
    pages.k[last, (kv - 1) % 16, 0, 5] = bad
    pages.v[last, (kv - 1) % 16, 0, 7] = bad
    K[0][-1, 0, 5] = 0
    V[0][-1, 0, 7] = 0
    out = m.paged_attention(pages, batch, q, 16)
    batch.status()
    want, tol = reference(qs, kvs, q, K, V, 16, 128 ** -0.5)
    keep = [i for i in range(n + 1) if i != n - 1]
    assert ((out.double() - want).abs() <= tol)[keep].all()
    import torch
    assert not torch.isfinite(out[n - 1].view(16, 128)[:, 7]).any()


@pytest.mark.parametrize("typ", ["f16", "f32"])
def test_attention_crowded_bad_arrays_are_reported(cuda, typ):
    import torch
    import large_model_b200 as m
    qs, kv = crowd([1, 40, 1], [50, 60, 33], 16, 1)
    pages, batch, q, K, V = make(qs, kv, typ=typ, G=16, Hk=1)
    good = m.paged_attention(pages, batch, q, 16)
    batch.status()
    keep = batch.table.clone()
    for bad in (-1, 10 ** 6, pages.k.shape[0]):      # a page that does not exist: not seen, and reported
        batch.table[2, 1] = bad
        out = m.paged_attention(pages, batch, q, 16)
        with pytest.raises(m.QmsCudaError, match="0x2"):
            batch.status()
        batch.table.copy_(keep)
        assert torch.equal(out[:41], good[:41])
        k, v = (x[2][torch.arange(33, device="cuda") // 16 != 1] for x in (K, V))
        want, tol = reference([1], [17], q[41:], [k], [v], 16, 128 ** -0.5)
        assert ((out[41:].double() - want).abs() <= tol).all()
    for what, value in (("kv_len", 61), ("kv_len", -5), ("q_start", -1), ("q_start", 100)):
        t = getattr(batch, what)
        was = t.clone()
        t[1 if what == "kv_len" else 2] = value
        m.paged_attention(pages, batch, q, 16)
        with pytest.raises(m.QmsCudaError, match="0x1"):
            batch.status()
        t.copy_(was)
    assert torch.equal(m.paged_attention(pages, batch, q, 16), good)
    batch.status()


@pytest.mark.parametrize("typ", ["f16", "f32"])
def test_attention_offsets_past_32_bits(cuda, typ):
    """Two pages more than 2^32 bytes apart."""
    import torch
    import large_model_b200 as m
    dt, es = (torch.float16, 2) if typ == "f16" else (torch.float32, 4)
    stride = (2 ** 32 + 2 ** 20) // es
    pool = torch.empty((stride + 2 * 64 * 128,), dtype=dt, device="cuda")
    k = pool.as_strided((2, 64, 1, 128), (stride, 128, 128, 1))
    v = pool.as_strided((2, 64, 1, 128), (stride, 128, 128, 1), 64 * 128)
    g = torch.Generator(device="cuda").manual_seed(1)
    for x in (k, v):
        x.copy_(torch.randn((2, 64, 1, 128), generator=g, device="cuda"))
    for qs, prefix in (([2], 0), ([40], 0), ([2], 100)):
        kv = [120]
        q = torch.randn((qs[0], 16 * 128), generator=g, device="cuda")
        batch = m.PagedBatch(torch.tensor([0, qs[0]], dtype=torch.int32, device="cuda"), torch.tensor(kv, dtype=torch.int32, device="cuda"),
                             torch.tensor([[1, 0]], dtype=torch.int32, device="cuda"), qs[0], qs[0], 120, prefix)
        out = m.paged_attention(m.KvPages(k, v), batch, q, 16)
        batch.status()
        K, V = (x[[1, 0]].reshape(128, 1, 128)[:120] for x in (k, v))
        want, tol = reference(qs, kv, q, [K], [V], 16, 128 ** -0.5)
        assert ((out.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("typ", ["f16", "f32"])
def test_attention_crowded_offsets_past_32_bits(cuda, typ):
    import torch
    import large_model_b200 as m
    dt, es = (torch.float16, 2) if typ == "f16" else (torch.float32, 4)
    stride = (2 ** 32 + 2 ** 20) // es
    pool = torch.empty((stride + 2 * 64 * 128,), dtype=dt, device="cuda")
    k = pool.as_strided((2, 64, 1, 128), (stride, 128, 128, 1))
    v = pool.as_strided((2, 64, 1, 128), (stride, 128, 128, 1), 64 * 128)
    g = torch.Generator(device="cuda").manual_seed(1)
    for x in (k, v):
        x.copy_(torch.randn((2, 64, 1, 128), generator=g, device="cuda"))
    for n, prefix in ((40, 0), (7, 100)):
        qs, kv = crowd([n], [120], 16, 1, prefix)
        q = torch.randn((n + 2000, 16 * 128), generator=g, device="cuda")
        start = torch.tensor([0] + [n] * len(qs), dtype=torch.int32, device="cuda")
        table = torch.tensor([[1, 0]] * len(qs), dtype=torch.int32, device="cuda")
        batch = m.PagedBatch(start, torch.tensor(kv, dtype=torch.int32, device="cuda"), table, n + 2000, n, 120, prefix)
        out = m.paged_attention(m.KvPages(k, v), batch, q, 16)
        batch.status()
        K, V = (x[[1, 0]].reshape(128, 1, 128)[:120] for x in (k, v))
        want, tol = reference([n], [120], q, [K], [V], 16, 128 ** -0.5)
        assert ((out.double() - want).abs() <= tol).all()


def test_attention_strided_rows_and_streams(cuda):
    """q inside the projections' rows, out inside wider rows, on a stream of its own."""
    import torch
    import large_model_b200 as m
    qs, kv = [1, 4, 30], [90, 64, 200]
    pages, batch, q, K, V = make(qs, kv, G=8, prefix=20)
    wide, res = torch.zeros((35, 3000), device="cuda"), torch.full((35, 2100), 7.0, device="cuda")
    wide[:, 100:2148] = q
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    m.paged_attention(pages, batch, wide[:, 100:2148], 16, out=res[:, 4:2052], stream=s)
    s.synchronize()
    want, tol = reference(qs, kv, q, K, V, 8, 128 ** -0.5)
    assert ((res[:, 4:2052].double() - want).abs() <= tol).all()
    assert (res[:, :4] == 7).all() and (res[:, 2052:] == 7).all()


@pytest.mark.parametrize("typ", ["f16", "f32"])
def test_decode_in_a_captured_graph(cuda, typ):
    """Append and attention captured once, replayed as the sequences grow."""
    import torch
    import large_model_b200 as m
    pages, batch, q, K, V = make([1, 1, 1], [40, 60, 33], typ=typ, G=4, Hk=2, prefix=20, garbage=0.0)
    B, H, Hk, D = 3, 8, 2, 128
    ctx = batch.table.shape[1] * 16
    batch.desc.max_kv = ctx                          # a bound for the whole run
    rope = m.rope_tables(ctx, D)
    one = torch.ones((D,), device="cuda")
    qkv = torch.zeros((B, (H + 2 * Hk) * D), device="cuda")
    qr, out = torch.empty((B, H * D), device="cuda"), torch.empty((B, H * D), device="cuda")

    def step():
        m.paged_append(pages, batch, qkv, H, one, one, 1e-6, rope, q=qr)
        m.paged_attention(pages, batch, qr, H, out=out)
    step()
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        step()
    g = torch.Generator(device="cuda").manual_seed(3)
    for _ in range(4):
        batch.kv_len += 1
        qkv.copy_(torch.randn(qkv.shape, generator=g, device="cuda"))
        gr.replay()
        batch.status()
        kv = batch.kv_len.tolist()
        Ks, Vs = [], []
        for b in range(B):
            j = torch.arange(kv[b], device="cuda")
            pg = batch.table[b].long()[j // 16]
            Ks.append(pages.k[pg, j % 16])
            Vs.append(pages.v[pg, j % 16])
        want, tol = reference([1] * B, kv, qr, Ks, Vs, 4, D ** -0.5)
        assert ((out.double() - want).abs() <= tol).all()


# ---- append ----------------------------------------------------------------------------------------

@pytest.mark.parametrize("typ", ["f16", "f32"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("order", ["nhd", "hnd"])
def test_append(cuda, typ, D, order):
    import torch
    import large_model_b200 as m
    qs, kv, H, Hk = [1, 0, 5, 33], [9, 0, 5, 100], 6, 3
    pages, batch, _, _, _ = make(qs, kv, typ=typ, D=D, Hk=Hk, G=2, order=order, garbage=0.0, pad=2)
    before = pages.k.clone(), pages.v.clone()
    T = sum(qs)
    g = torch.Generator(device="cuda").manual_seed(5)
    qkv = 3 * torch.randn((T + 2, (H + 2 * Hk) * D), generator=g, device="cuda")
    qkv[0] = 0                                       # a row of zeros stays zero
    qn, kn = (torch.randn((D,), generator=g, device="cuda") for _ in range(2))
    rope = m.rope_tables(100, D, 1e4)
    q = m.paged_append(pages, batch, qkv, H, qn, kn, 1e-6, rope, q=torch.full((T + 2, H * D), 7.0, device="cuda"))
    batch.status()
    assert (q[T:] == 7).all()
    es = 2.0 ** -11 if typ == "f16" else E24
    touched = torch.zeros(pages.k.shape[:2], dtype=torch.bool, device="cuda")
    t = 0
    for b, n in enumerate(qs):
        for i in range(n):
            p = kv[b] - n + i
            x = qkv[t].double().view(H + 2 * Hk, D)
            ang = p * 1e4 ** (-2.0 * torch.arange(D // 2, dtype=torch.float64, device="cuda") / D)
            c, s = ang.cos(), ang.sin()

            def turned(y, w):
                y = y / torch.sqrt(y.pow(2).mean(-1, keepdim=True) + 1e-6) * w.double()
                a, z = y[:, :D // 2], y[:, D // 2:]
                mag = torch.cat([a.abs() + z.abs()] * 2, -1)
                return torch.cat([a * c - z * s, z * c + a * s], -1), mag
            want, mag = turned(x[:H], qn)
            assert ((q[t].double().view(H, D) - want).abs() <= 8 * E24 * mag).all()
            want, mag = turned(x[H:H + Hk], kn)
            pg = batch.table[b, p // 16].long()
            tol = (8 * E24 + es) * mag + 2.0 ** -25
            assert ((pages.k[pg, p % 16].double() - want).abs() <= tol).all()
            assert torch.equal(pages.v[pg, p % 16], qkv[t].view(H + 2 * Hk, D)[H + Hk:].to(pages.v.dtype))
            touched[pg, p % 16] = True
            t += 1
    assert torch.equal(pages.k[~touched], before[0][~touched]) and torch.equal(pages.v[~touched], before[1][~touched])
    # in place: the q heads over their own rows
    own = qkv.clone()
    m.paged_append(pages, batch, own, H, qn, kn, 1e-6, rope, q=own[:, :H * D])
    assert torch.equal(own[:T, :H * D], q[:T]) and torch.equal(own[:, H * D:], qkv[:, H * D:])


@pytest.mark.parametrize("typ", ["f16", "f32"])
@pytest.mark.parametrize("D,H,Hk", [(64, 6, 3), (128, 8, 4), (128, 5, 1)])
def test_append_many_rows(cuda, typ, D, H, Hk):
    """As many rows as several per warp are used for: the same bits as a few tokens at a time; groups of rows that cross
    from q to k to v, and a last one that is not full."""
    import torch
    import large_model_b200 as m
    n, B = 90, 12
    qs, kv = [n - b for b in range(B)], [n + 3 * b for b in range(B)]
    pages, batch, _, _, _ = make(qs, kv, typ=typ, D=D, Hk=Hk, G=2, garbage=0.0, pad=5)
    T = sum(qs)
    assert (T + 5) * (H + 2 * Hk) >= 148 * 48
    g = torch.Generator(device="cuda").manual_seed(7)
    qkv = 3 * torch.randn((T + 5, (H + 2 * Hk) * D), generator=g, device="cuda")
    qkv[100] = 0
    qn, kn = (torch.randn((D,), generator=g, device="cuda") for _ in range(2))
    rope = m.rope_tables(max(kv), D)
    q = m.paged_append(pages, batch, qkv, H, qn, kn, 1e-6, rope, q=torch.full((T + 5, H * D), 7.0, device="cuda"))
    batch.status()
    assert (q[T:] == 7).all() and (q[100] == 0).all()
    other = m.KvPages(torch.zeros_like(pages.k), torch.zeros_like(pages.v))
    t = 0
    for b in range(B):
        one = m.PagedBatch(torch.tensor([0, qs[b]], dtype=torch.int32, device="cuda"), batch.kv_len[b:b + 1].clone(), batch.table[b:b + 1].clone(),
                           qs[b], qs[b], kv[b])
        assert torch.equal(m.paged_append(other, one, qkv[t:t + qs[b]], H, qn, kn, 1e-6, rope), q[t:t + qs[b]])
        one.status()
        for j in range(kv[b] - qs[b], kv[b]):
            pg = batch.table[b, j // 16].long()
            assert torch.equal(other.k[pg, j % 16], pages.k[pg, j % 16]) and torch.equal(other.v[pg, j % 16], pages.v[pg, j % 16])
        t += qs[b]


def test_append_refuses_on_the_device(cuda):
    import torch
    import large_model_b200 as m
    qs, kv = [2, 1], [20, 40]
    pages, batch, _, _, _ = make(qs, kv, garbage=0.0, D=64)
    one, qkv = torch.ones((64,), device="cuda"), torch.randn((3, 8 * 64), device="cuda")

    def attempt(rope_len=40):
        k, v = pages.k.clone(), pages.v.clone()
        q = m.paged_append(pages, batch, qkv, 4, one, one, 1e-6, m.rope_tables(rope_len, 64), q=torch.zeros((3, 256), device="cuda"))
        return q, (pages.k != k).any((1, 2, 3)), (pages.v != v).any((1, 2, 3))
    q, k, v = attempt(39)                            # a position past the rotation tables
    with pytest.raises(m.QmsCudaError, match="0x1"):
        batch.status()
    assert (q[2] == 0).all() and (q[:2] != 0).any() and k.sum() == 1
    page = int(batch.table[1, 2])
    batch.table[1, 2] = pages.k.shape[0]             # a page that does not exist
    q, k, v = attempt()
    with pytest.raises(m.QmsCudaError, match="0x2"):
        batch.status()
    assert (q[2] == 0).all()
    batch.table[1, 2] = page
    batch.kv_len[0] = 1                              # two rows, one position
    q, k, v = attempt()
    with pytest.raises(m.QmsCudaError, match="0x1"):
        batch.status()
    assert (q[0] == 0).all() and (q[1] != 0).any()


def test_nothing_to_do(cuda):
    import torch
    import large_model_b200 as m
    pages, batch, q, _, _ = make([0, 0], [0, 5], G=2)
    assert m.paged_attention(pages, batch, q, 4).shape == (0, 512)
    pages, batch, q, _, _ = make([0, 0], [0, 5], G=2, pad=2)
    assert (m.paged_attention(pages, batch, q, 4) == 0).all()
    batch.status()
