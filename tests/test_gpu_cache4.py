"""The paged KV cache in 4 bits on a B200 through the C ABI: the append (with rows in 16 bits for whole prompts), what the pool
holds, and the attention over it, against their formulas in 64 bits.

Bounds. What is stored is exact: the append goes in double to the end, and the test's 64 bits meet it but for values within 1e-12 of a
border, which the seeds do not hold. Attention: K and V as the cache gives them are exact in fp16; a score, a weight and the output are
off as over an fp16 cache: (16 e A + 16 e) max |V| with e = 2^-24 and A = scale * sum |q k|, the largest over what the row sees. Rows:
three roundings of the normalised value and three of the rotation, 8 e (|x1| + |x2|), then half a step of the 16-bit type."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
E24 = 2.0 ** -24
NAN = float("nan")


# ---- the format, apart from the library ------------------------------------------------------------

def held(x):
    """What the cache gives back for x (numpy float64 [..., D]), and the (nibbles, scales) it holds."""
    g = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    bad = ~np.isfinite(g).all(-1)
    y = np.where(bad[..., None], 0.0, g)
    first = np.abs(y).argmax(-1)
    m, e = np.frexp(np.take_along_axis(y, first[..., None], -1)[..., 0] / -8.0)
    d = np.clip(np.ldexp(np.rint(m * 256) / 256, e), -2720.0, 2720.0).astype(np.float16)
    with np.errstate(divide="ignore", invalid="ignore"):
        n = np.floor(y / d[..., None].astype(np.float64) + 8.5)
    n = np.where(d[..., None] == 0, 8.0, np.clip(n, 0, 15)).astype(np.int64)
    v = (n - 8) * d[..., None].astype(np.float64)
    v = np.where(bad[..., None], np.nan, v)
    return v.reshape(x.shape), n.reshape(x.shape), np.where(bad, np.float16(NAN), d)


def pack(n, d):
    """Nibbles [..., page, D] and scales [..., page, D / 32] as the bytes of (page, head) blocks."""
    w = np.zeros(n.shape[:-1] + (n.shape[-1] // 8,), np.uint32)
    for i in range(8):
        w |= n[..., i::8].astype(np.uint32) << np.uint32(4 * (i // 2) + 16 * (i % 2))
    lead = n.shape[:-2]
    return np.concatenate([np.ascontiguousarray(w).view(np.uint8).reshape(*lead, -1),
                           np.ascontiguousarray(d.astype(np.float16)).view(np.uint8).reshape(*lead, -1)], -1)


def make(qs, kv, *, G=2, Hk=2, D=128, page=16, prefix=0, seed=0, pad=0, qscale=1.0, gap=0, edit=None):
    """A batch over a pool whose nibbles are 15 and whose scales are NaN except at positions that some sequence owns."""
    import torch
    import large_model_b200 as m
    rng = np.random.default_rng(seed)
    B, T = len(qs), sum(qs) + pad
    shared = prefix // page
    need = [max(0, -(-n // page) - shared) for n in kv]
    perm = rng.permutation(shared + sum(need) + 2).astype(np.int32)
    table = np.full((B, max(1, shared + max(need, default=0))), perm[-1], np.int32)
    table[:, :shared] = perm[:shared]
    at = shared
    for b in range(B):
        table[b, shared:shared + need[b]] = perm[at:at + need[b]]
        at += need[b]
    N = len(perm)
    nib = [np.full((N, Hk, page, D), 15, np.int64) for _ in range(2)]
    sc = [np.full((N, Hk, page, D // 32), NAN, np.float16) for _ in range(2)]
    vals = [[], []]
    for b in range(B):
        for z in range(2):
            x = rng.standard_normal((kv[b], Hk, D))
            if edit:
                edit(z, b, x)
            v, n, d = held(x)
            k = min(prefix, kv[b])
            if b:
                v[:k] = vals[z][0][:k]
            else:
                k = 0
            vals[z].append(v)
            j = np.arange(kv[b])
            pg, off = table[b][j // page], j % page
            own = j >= k                             # the shared prompt's values are the first sequence's, its tail page's copies too
            nib[z][pg[own], :, off[own]], sc[z][pg[own], :, off[own]] = n[own], d[own]
            if k:
                t0 = table[0][j[:k] // page]
                nib[z][pg[:k], :, off[:k]], sc[z][pg[:k], :, off[:k]] = nib[z][t0, :, off[:k]], sc[z][t0, :, off[:k]]
    size = page * D * 9 // 16
    pools = []
    for z in range(2):
        p = torch.full((N, Hk + gap, size + 16 * gap), 255, dtype=torch.uint8, device="cuda")[:, :Hk, :size]
        p.copy_(torch.from_numpy(pack(nib[z], sc[z])))
        pools.append(p)
    ints = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")
    q = qscale * torch.from_numpy(rng.standard_normal((T, Hk * G * D)).astype(np.float32)).cuda()
    batch = m.PagedBatch(ints([0] + np.cumsum(qs).tolist()), ints(kv), ints(table), T, max(qs, default=0), max(kv, default=0), prefix)
    K, V = ([torch.from_numpy(x).cuda() for x in z] for z in vals)
    return m.KvPages.packed(*pools, D), batch, q, K, V


def reference(qs, kv, q, K, V, G, scale):
    import torch
    Hk, D = K[0].shape[1:]
    out = torch.zeros((q.shape[0], Hk, G, D), dtype=torch.float64, device="cuda")
    tol = torch.zeros((q.shape[0], Hk, G, 1), dtype=torch.float64, device="cuda")
    t = 0
    for b, n in enumerate(qs):
        for i in range(n):
            p = kv[b] - n + i
            if p >= 0:
                x, k, v = q[t].double().view(Hk, G, D), K[b][:p + 1], V[b][:p + 1]
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
    H = G * kw.get("Hk", 2)
    out = m.paged_attention(pages, batch, q, H, scale=scale)
    batch.status()
    want, tol = reference(qs, kv, q, K, V, G, D ** -0.5 if scale is None else scale)
    assert torch.isfinite(out).all()
    over = ((out.double() - want).abs() - tol).max().item()
    assert over <= 0, f"{over} over the bound (worst error {(out.double() - want).abs().max().item()})"
    again = m.paged_attention(pages, batch, q, H, scale=scale)
    assert torch.equal(out.view(torch.int32), again.view(torch.int32)), "two runs differ"
    return out


# ---- append ------------------------------------------------------------------------------------------

def append_case(qs, kv, *, G=2, Hk=2, D=128, page=16, rows=None, typ=None, seed=0, edit=None, pad=0):
    """Appends through the library, and what the formula gives: ((got, want, bound) of the rows, of K and of V at the new positions)."""
    import torch
    import large_model_b200 as m
    typ = m.T_Q4_0 if typ is None else typ
    rng = np.random.default_rng(seed)
    H, T = G * Hk, sum(qs) + pad
    need = [-(-n // page) for n in kv]
    table = np.zeros((len(qs), max(1, max(need))), np.int32)
    perm = rng.permutation(sum(need) + 1).astype(np.int32)
    for b, at in enumerate(np.cumsum([0] + need[:-1])):
        table[b, :need[b]] = perm[at:at + need[b]]
    pages = m.KvPages.empty(len(perm), page, Hk, D, typ)
    ints = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")
    batch = m.PagedBatch(ints([0] + np.cumsum(qs).tolist()), ints(kv), ints(table), T, max(qs), max(kv))
    x = rng.standard_normal((T, H + 2 * Hk, D)).astype(np.float32)
    if edit:
        edit(x)
    qn, kn = ((1 + 0.2 * rng.standard_normal(D)).astype(np.float32) for _ in range(2))
    cos, sin = m.rope_tables(max(kv) + 1, D)
    dev = lambda a: torch.from_numpy(a).cuda()
    args = (pages, batch, dev(x.reshape(T, -1)), H, dev(qn), dev(kn), 1e-6, (cos, sin))
    if rows is None:
        got = m.paged_append(*args, q=torch.full((T, H * D), 7.0, device="cuda")).view(T, H, D)
    else:
        got = m.prompt_append(*args, rows=torch.full((T, H + 2 * Hk, D), 7.0, dtype=rows, device="cuda"))
    batch.status()
    k, v = pages.values()
    # the formula
    b_of = np.repeat(np.arange(len(qs)), qs)
    pos = np.concatenate([np.arange(n - t, n) for t, n in zip(qs, kv)]) if sum(qs) else np.zeros(0, int)
    y = x[:len(pos)].astype(np.float64)
    with np.errstate(invalid="ignore"):
        y[:, :H + Hk] /= np.sqrt((y[:, :H + Hk] ** 2).mean(-1, keepdims=True) + float(np.float32(1e-6)))
        y[:, :H] *= qn
        y[:, H:H + Hk] *= kn
        c, s = (z.cpu().numpy().astype(np.float64)[pos][:, None] for z in (cos, sin))
        lo, hi = y[:, :H + Hk, :D // 2].copy(), y[:, :H + Hk, D // 2:].copy()
        y[:, :H + Hk, :D // 2], y[:, :H + Hk, D // 2:] = lo * c - hi * s, hi * c + lo * s
    size = np.zeros_like(y)
    size[:, :H + Hk] = np.concatenate([np.abs(lo) + np.abs(hi)] * 2, -1)
    at = (table[b_of, pos // page], pos % page)
    stored = [z.cpu().numpy()[at] for z in (k, v)]
    return got.float().cpu().numpy(), y, size, stored, (k, v), pages


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("qs,kv,G,Hk,page", [
    ([1], [1], 16, 4, 16), ([1, 1, 1], [1, 17, 300], 1, 1, 16), ([3, 0, 5], [3, 9, 70], 3, 2, 32), ([200, 1, 129], [200, 5, 400], 8, 4, 128)])
def test_append(cuda, D, qs, kv, G, Hk, page):
    got, y, size, stored, _, _ = append_case(qs, kv, G=G, Hk=Hk, D=D, page=page, seed=D + G, pad=2)
    H = G * Hk
    assert (np.abs(got[:len(y)] - y[:, :H]) <= 8 * E24 * size[:, :H]).all()
    assert (got[len(y):] == 7.0).all(), "rows behind the last sequence"
    for z, first in zip(stored, (H, H + Hk)):
        assert np.array_equal(z.astype(np.float64), held(y[:, first:first + Hk])[0])


@pytest.mark.parametrize("typ", ["f32", "f16", "q4"])
@pytest.mark.parametrize("rows", ["float16", "bfloat16"])
@pytest.mark.parametrize("qs", [[1], [37, 0, 1, 260]])
def test_prompt_append(cuda, typ, rows, qs):
    """Rows in 16 bits; the pages hold what paged_append stores."""
    import torch
    import large_model_b200 as m
    dt, G, Hk, D = getattr(torch, rows), 8, 2, 128
    T_ = {"f32": m.T_F32, "f16": m.T_F16, "q4": m.T_Q4_0}[typ]
    got, y, size, stored, _, pages = append_case(qs, qs, G=G, Hk=Hk, D=D, rows=dt, typ=T_, seed=len(qs), pad=3)
    n, half = len(y), torch.finfo(dt).eps / 2
    assert (np.abs(got[:n] - y) <= 8 * E24 * size + half * (np.abs(y) + 8 * E24 * size) + 2.0 ** -25).all()      # (2^-25: fp16's smallest step)
    assert (got[n:] == 7.0).all()
    _, _, _, other, _, pages2 = append_case(qs, qs, G=G, Hk=Hk, D=D, typ=T_, seed=len(qs), pad=3)
    assert torch.equal(pages.k, pages2.k) and torch.equal(pages.v, pages2.v)


def test_prompt_append_without_a_cache(cuda):
    import torch
    import large_model_b200 as m
    g = torch.Generator(device="cuda").manual_seed(1)
    qs, H, Hk, D = [5, 0, 40], 4, 2, 64
    qkv = torch.randn((45, (H + 2 * Hk) * D), generator=g, device="cuda")
    w = torch.randn((2, D), generator=g, device="cuda")
    start = torch.tensor([0, 5, 5, 45], dtype=torch.int32, device="cuda")
    kv = torch.tensor(qs, dtype=torch.int32, device="cuda")
    table = torch.arange(9, dtype=torch.int32, device="cuda").view(3, 3)
    pages = m.KvPages.empty(9, 16, Hk, D, m.T_F16)
    rope = m.rope_tables(64, D)
    want = m.prompt_append(pages, m.PagedBatch(start, kv, table, 45, 40, 40), qkv, H, w[0], w[1], 1e-6, rope)
    batch = m.PagedBatch.prompts(start, 45, 40)
    got = m.prompt_append(None, batch, qkv, H, w[0], w[1], 1e-6, rope, n_head_kv=Hk)
    batch.status()
    assert got.dtype == torch.bfloat16 and torch.equal(got, want)
    short = m.PagedBatch.prompts(start, 45, 39)                      # a prompt above its bound
    m.prompt_append(None, short, qkv, H, w[0], w[1], 1e-6, rope, n_head_kv=Hk)
    with pytest.raises(m.QmsCudaError):
        short.status()


@pytest.mark.parametrize("D", [64, 128])
def test_append_special_values(cuda, D):
    """V rows of zeros, ties, equal magnitudes of either sign, coarse values, huge, tiny and not finite ones, -8 .. 8 times the step."""
    H, Hk = 4, 2
    pick = np.random.default_rng(5)

    def edit(x):
        v = x[:, H + Hk:]
        v[0] = 0.0
        v[1] = -0.0
        v[2] = (np.arange(D) % 33 - 16) * 0.25                        # ties between steps
        v[3, :, ::2], v[3, :, 1::2] = 1.5, -1.5
        v[4, :, ::2], v[4, :, 1::2] = -1.5, 1.5
        v[5] = pick.integers(-20, 20, (Hk, D)) / 16.0
        v[6] *= 3e4
        v[7] *= 1e30
        v[8] *= 1e-7
        v[9] *= 1e-30
        v[10, 0, 5] = np.inf
        v[11, 1, D - 1] = np.nan
        v[12] = (np.arange(D) % 17 - 8) * 0.171875
        v[13, :, 1:] = 0.0
        v[14] = np.round(v[14] * 8) / 8
        v[15, 0, 3] = -np.inf
    got, y, size, stored, _, _ = append_case([16], [16], G=2, Hk=Hk, D=D, seed=9, edit=edit)
    want = held(y[:, H + Hk:])[0]
    assert np.array_equal(stored[1].astype(np.float64), want, equal_nan=True)
    assert np.isnan(want[10, 0, :32]).all() and np.isfinite(want[10, 1]).all() and np.abs(want[7]).max() == 8 * 2720.0
    assert np.array_equal(stored[0].astype(np.float64), held(y[:, H:H + Hk])[0])


def test_append_bad_pages_and_positions(cuda):
    import torch
    import large_model_b200 as m
    H, Hk, D = 2, 1, 64
    qkv = torch.randn((3, (H + 2 * Hk) * D), device="cuda")
    w = torch.ones(D, device="cuda")
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    for kv, page, n_rope, bit in ((3, 5, 8, "2"), (3, -1, 8, "2"), (3, 0, 2, "1"), (2, 0, 8, "1"), (40, 0, 8, "1")):
        pages = m.KvPages.empty(2, 16, Hk, D, m.T_Q4_0)
        batch = m.PagedBatch(ints(0, 3), ints(kv), ints([page]), 3, 3, 16)
        cos, sin = m.rope_tables(n_rope, D)
        m.paged_append(pages, batch, qkv, H, w, w, 1e-6, (cos, sin))
        with pytest.raises(m.QmsCudaError, match=f"0x{bit}"):
            batch.status()
        if bit == "2" or kv == 40:
            assert not pages.k.any() and not pages.v.any()


@pytest.mark.parametrize("typ,order", [("f32", 0), ("f16", 1), ("q4", 0)])
@pytest.mark.parametrize("D,page,Hk", [(64, 16, 3), (128, 32, 4), (128, 16, 1)])
def test_values(cuda, typ, order, D, page, Hk):
    import torch
    import large_model_b200 as m
    g = torch.Generator(device="cuda").manual_seed(D + Hk)
    if typ == "q4":
        rng = np.random.default_rng(3)
        v, n, d = held(rng.standard_normal((5, Hk, page, D)))
        base = torch.zeros((5, Hk + 1, page * D * 9 // 16 + 32), dtype=torch.uint8, device="cuda")
        k = base[:, :Hk, :page * D * 9 // 16]
        k.copy_(torch.from_numpy(pack(n, d)))
        pages = m.KvPages.packed(k, k, D)
        want = torch.from_numpy(v).cuda().transpose(1, 2)
    else:
        dt = torch.float32 if typ == "f32" else torch.float16
        k = torch.randn((5, page, Hk, D), generator=g, device="cuda").to(dt)
        if order:
            k = torch.randn((5, Hk, page, D), generator=g, device="cuda").to(dt).transpose(1, 2)
        pages = m.KvPages(k, k)
        want = k.double()
    for x in pages.values():
        assert torch.equal(x.double(), want)


# ---- attention ---------------------------------------------------------------------------------------

@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("G", [1, 3, 8, 16])
def test_attention_one_token(cuda, D, G):
    check([1, 1, 1, 1], [1, 2, 63, 333], D=D, G=G, seed=G)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 512])
def test_attention_page_sizes(cuda, page):
    check([1, 3, 0, 2], [200, 129, 0, 17], page=page, seed=page, gap=1)


@pytest.mark.parametrize("prefix", [1, 16, 100, 127, 128, 129, 300])
def test_attention_shared_prompt(cuda, prefix):
    qs, new = [1, 4, 0, 2, 1], [5, 4, 0, 130, 1]
    check(qs, [prefix + n for n in new], prefix=prefix, G=8, seed=prefix)


@pytest.mark.parametrize("D", [64, 128])
def test_attention_many_rows_one_prompt(cuda, D):
    qs = [(5 * b + 2) % 4 for b in range(37)]
    for prefix in (700, 2100):                       # mma.sync, tcgen05
        check(qs, [prefix + n + (91 * b) % 57 for b, n in enumerate(qs)], prefix=prefix, G=16, Hk=2, D=D, seed=D)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n,kv", [(70, 70), (65, 300), (129, 129), (200, 1111), (300, 5000)])
def test_attention_prompt_chunks(cuda, n, kv, D):
    check([n], [kv], G=8, Hk=2, D=D, seed=n, page=32)


def test_attention_wide_sequences(cuda):
    """The kernel for many rows over several sequences' own positions, idle ones among them, and pages larger than a tile."""
    check([40, 0, 33, 1, 50], [900, 20, 1500, 1, 50], G=16, Hk=2, page=256, seed=3)
    check([40, 0, 33, 1, 50], [900, 20, 1500, 1, 50], G=16, Hk=2, page=16, seed=4, prefix=0)


@pytest.mark.parametrize("qscale,scale", [(30.0, None), (1.0, -0.05), (1e-20, 1e20), (1.0, 0.0)])
def test_attention_scales(cuda, qscale, scale):
    check([2, 70], [100, 1200], G=8, qscale=qscale, scale=scale, seed=2)


def test_padding_is_zero_and_nothing_seen_is_zero(cuda):
    import large_model_b200 as m
    pages, batch, q, K, V = make([2, 0, 3], [2, 0, 40], pad=3)
    out = m.paged_attention(pages, batch, q, 4)
    batch.status()
    assert (out[5:] == 0).all()
    batch.kv_len[0] = 1                              # its first row's position is -1
    out = m.paged_attention(pages, batch, q, 4)
    batch.status()
    assert (out[0] == 0).all() and out[1].isfinite().all() and out[1].any()


@pytest.mark.parametrize("n,G", [(4, 2), (4, 16), (80, 16)])
def test_values_behind_the_mask_do_not_count(cuda, n, G):
    """K and V that are NaN at the last new token's position: the rows before it do not see them, it does."""
    import torch
    import large_model_b200 as m
    kv, D = 600 if n < 80 else 1300, 128
    clean = make([n], [kv], G=G, seed=1)
    want = m.paged_attention(clean[0], clean[1], clean[2], 2 * G)

    def edit(z, b, x):
        x[kv - 1, :, 40] = np.nan if z else np.inf
    pages, batch, q, _, _ = make([n], [kv], G=G, seed=1, edit=edit)
    out = m.paged_attention(pages, batch, q, 2 * G)
    batch.status()
    assert torch.isfinite(out[:-1]).all()
    assert (out[:-1] - want[:-1]).abs().max().item() <= 32 * E24 * 16
    assert out[-1].isnan().any()

    def only_v(z, b, x):
        if z:
            x[kv - 2, :, 40] = np.nan
    pages, batch, q, _, _ = make([n], [kv], G=G, seed=1, edit=only_v)
    out = m.paged_attention(pages, batch, q, 2 * G).view(n, 2, G, D)
    assert torch.isfinite(out[:-2]).all()
    assert out[-2:, ..., 32:64].isnan().all() and torch.isfinite(out[-2:, ..., :32]).all() and torch.isfinite(out[-2:, ..., 64:]).all()


@pytest.mark.parametrize("n", [1, 80])
def test_attention_bad_pages(cuda, n):
    """Positions on a page that is not there count as not seen, and are reported."""
    import torch
    import large_model_b200 as m
    kv, G = 700 if n == 1 else 1500, 16
    pages, batch, q, K, V = make([n], [kv], G=G, seed=7, page=32)
    batch.table[0, 3] = 1 << 20
    out = m.paged_attention(pages, batch, q, 2 * G)
    with pytest.raises(m.QmsCudaError, match="0x2"):
        batch.status()
    keep = [j for j in range(kv) if j // 32 != 3]
    want, tol = reference([n], [kv - 32], q, [K[0][keep]], [V[0][keep]], G, 128 ** -0.5)
    assert ((out.double() - want).abs() <= tol).all()


def test_bad_lengths(cuda):
    import large_model_b200 as m
    pages, batch, q, K, V = make([1, 2], [30, 40])
    batch.kv_len[1] = 41
    out = m.paged_attention(pages, batch, q, 4)
    with pytest.raises(m.QmsCudaError, match="0x1"):
        batch.status()
    assert (out[1:] == 0).all() and out[0].any()


def test_long_cache(cuda):
    """A page pool above 4 GB of bytes: offsets pass 32 bits."""
    import torch
    import large_model_b200 as m
    D, page, Hk = 128, 1024, 4
    size = page * D * 9 // 16
    N = (5 << 30) // (Hk * size)
    pool = torch.zeros((N, Hk, size), dtype=torch.uint8, device="cuda")
    small = make([1], [page], page=page, Hk=Hk, G=2, seed=1)
    used = small[1].table[0, 0].item()
    pool[N - 1].copy_(small[0].k[used])
    pages = m.KvPages.packed(pool, pool, D)
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    batch = m.PagedBatch(ints(0, 1), ints(page), ints([N - 1]), 1, 1, page)
    out = m.paged_attention(pages, batch, small[2], 2 * Hk)
    batch.status()
    k = small[3][0]
    want, tol = reference([1], [page], small[2], [k], [k], 2, D ** -0.5)
    assert ((out.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("n", [1, 80])
def test_graphs_and_streams(cuda, n):
    import torch
    import large_model_b200 as m
    pages, batch, q, K, V = make([n], [1200], G=16, seed=3)
    want = m.paged_attention(pages, batch, q, 32)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = m.paged_attention(pages, batch, q, 32, stream=s)
    s.synchronize()
    out = torch.zeros_like(want)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        m.paged_attention(pages, batch, q, 32, out=out)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(want, got) and torch.equal(want, out)


def test_append_then_attend(cuda):
    """A prompt in one call, then tokens one at a time: what the last row sees is what was stored."""
    import torch
    import large_model_b200 as m
    H, Hk, D, page, n = 8, 2, 64, 16, 75
    g = torch.Generator(device="cuda").manual_seed(2)
    qkv = torch.randn((n, (H + 2 * Hk) * D), generator=g, device="cuda")
    w = 1 + 0.1 * torch.randn((2, D), generator=g, device="cuda")
    rope = m.rope_tables(n, D)
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    table = ints([4, 2, 0, 3, 1])
    whole, steps = (m.KvPages.empty(5, page, Hk, D, m.T_Q4_0) for _ in range(2))
    b = m.PagedBatch(ints(0, n), ints(n), table, n, n, n)
    q = m.paged_append(whole, b, qkv, H, w[0], w[1], 1e-6, rope)
    out = m.paged_attention(whole, b, q, H)
    rows = []
    for t in range(n):
        b1 = m.PagedBatch(ints(0, 1), ints(t + 1), table, 1, 1, n)
        q1 = m.paged_append(steps, b1, qkv[t:t + 1], H, w[0], w[1], 1e-6, rope)
        rows.append(m.paged_attention(steps, b1, q1, H))
        b1.status()
    b.status()
    assert torch.equal(whole.k, steps.k) and torch.equal(whole.v, steps.v)
    k, v = (x[table[0].long()].flatten(0, 1)[:n].double() for x in whole.values())
    want, tol = reference([n], [n], q, [k], [v], H // Hk, D ** -0.5)
    assert ((out.double() - want).abs() <= tol).all()
    assert ((torch.cat(rows).double() - want).abs() <= tol).all()


def test_refusals(cuda):
    import torch
    import large_model_b200 as m
    u8 = lambda *s: torch.zeros(s, dtype=torch.uint8, device="cuda")
    for bad in (lambda: m.KvPages.packed(u8(2, 2, 1000), u8(2, 2, 1000), 128), lambda: m.KvPages.packed(u8(2, 2, 1152), u8(2, 3, 1152), 128),
                lambda: m.KvPages.packed(u8(2, 2, 1152).float(), u8(2, 2, 1152).float(), 128), lambda: m.KvPages.packed(u8(2, 1152), u8(2, 1152), 128)):
        with pytest.raises(ValueError):
            bad()
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    batch = m.PagedBatch(ints(0, 1), ints(1), ints([0]), 1, 1, 8)
    for pages in (m.KvPages.packed(u8(2, 2, 576), u8(2, 2, 576), 128),                            # 8 positions a page
                  m.KvPages.packed(u8(2, 2, 96 * 18), u8(2, 2, 96 * 18), 32),                     # heads of 32
                  m.KvPages.packed(u8(2, 2, 1160)[..., :1152], u8(2, 2, 1160)[..., :1152], 128)):  # strides of 8 bytes
        with pytest.raises(m.QmsCudaError):
            m.paged_attention(pages, batch, torch.zeros((1, 2 * pages.head_dim), device="cuda"), 2)
        with pytest.raises(m.QmsCudaError):
            pages.values()


def test_prompt_append_takes_weights_and_tables_of_any_alignment(cuda):
    import torch
    import large_model_b200 as m
    g = torch.Generator(device="cuda").manual_seed(1)
    T, H, Hk, D = 40, 8, 2, 128
    qkv = torch.randn((T, (H + 2 * Hk) * D), generator=g, device="cuda")
    w = torch.randn((D,), generator=g, device="cuda")
    cos, sin = m.rope_tables(64, D)
    off = lambda x: torch.cat([x.new_zeros(1), x.flatten()])[1:].view(x.shape)
    batch = m.PagedBatch.prompts(torch.tensor([0, T], dtype=torch.int32, device="cuda"), T, T)
    want = m.prompt_append(None, batch, qkv, H, w, w, 1e-6, (cos, sin), n_head_kv=Hk)
    got = m.prompt_append(None, batch, qkv, H, off(w), off(w), 1e-6, (off(cos), off(sin)), n_head_kv=Hk)
    assert off(w).data_ptr() % 8 == 4 and torch.equal(got, want)


@pytest.mark.parametrize("qs,kv,G,Hk,D,page,prefix", [
    ([70], [1400], 16, 2, 128, 32, 0),                            # one sequence's own positions
    ([130], [6001], 4, 1, 128, 512, 0),                           # a page larger than a tile
    ([40], [6500], 8, 2, 64, 16, 0),
    ([20, 0, 41, 1, 20], [1400, 1310, 1361, 20, 1302], 16, 2, 128, 16, 1301),     # a shared prompt, and a sequence shorter than it
    ([70], [3000], 16, 2, 128, 64, 1500),                         # a prompt and own positions, both
    ([16], [6100], 16, 2, 128, 64, 0),                            # 256 rows: 4 bits to the kernel
    ([3, 2, 3], [6500, 6500, 6410], 16, 2, 64, 64, 6400),
])
def test_attention_many_rows_by_fp16(cuda, qs, kv, G, Hk, D, page, prefix):
    check(qs, kv, G=G, Hk=Hk, D=D, page=page, prefix=prefix, pad=2, seed=sum(kv))


def test_many_rows_of_a_sequence_shorter_than_the_batch_allows(cuda):
    """Table entries past the sequence's length lead nowhere, and count for nothing; the same batch object grows afterwards."""
    import torch
    import large_model_b200 as m
    n, kv, G = 70, 1400, 16
    pages, small, q, K, V = make([n], [kv], G=G, page=32, seed=9)
    table = torch.full((1, 64), 1 << 20, dtype=torch.int32, device="cuda")
    table[:, :small.table.shape[1]] = small.table
    batch = m.PagedBatch(small.q_start, torch.tensor([kv], dtype=torch.int32, device="cuda"), table, n, n, 2048)
    for now in (kv, 801, n, kv):
        batch.kv_len.fill_(now)
        out = m.paged_attention(pages, batch, q, 2 * G)
        batch.status()
        want, tol = reference([n], [now], q, [K[0][:now]], [V[0][:now]], G, 128 ** -0.5)
        assert ((out.double() - want).abs() <= tol).all()


def test_masked_values_and_bad_pages_of_many_rows_in_two_sequences(cuda):
    """What holds for one sequence's many rows, for the kernel that reads 4 bits."""
    import torch
    import large_model_b200 as m
    n, kv, G, D = 80, 1300, 16, 128
    clean = make([n, 1], [kv, 5], G=G, seed=1)
    want = m.paged_attention(clean[0], clean[1], clean[2], 2 * G)

    def edit(z, b, x):
        if b == 0:
            x[kv - 1, :, 40] = np.nan if z else np.inf
    pages, batch, q, _, _ = make([n, 1], [kv, 5], G=G, seed=1, edit=edit)
    out = m.paged_attention(pages, batch, q, 2 * G)
    batch.status()
    assert torch.isfinite(out[:n - 1]).all() and torch.isfinite(out[n]).all()
    assert (out[:n - 1] - want[:n - 1]).abs().max().item() <= 32 * E24 * 16
    assert out[n - 1].isnan().any()

    pages, batch, q, K, V = make([n, 1], [kv, 5], G=G, seed=7, page=32)
    batch.table[0, 3] = -5
    out = m.paged_attention(pages, batch, q, 2 * G)
    with pytest.raises(m.QmsCudaError, match="0x2"):
        batch.status()
    keep = [j for j in range(kv) if j // 32 != 3]
    want, tol = reference([n, 1], [kv - 32, 5], q, [K[0][keep], K[1]], [V[0][keep], V[1]], G, 128 ** -0.5)
    assert ((out.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("q", [2, 3, 4, 5])
def test_attention_many_tiles_of_rows(cuda, D, q):
    """Two to five tokens of 40 sequences, short ones and idle ones among them: tiles of 32 and 64 rows; and one of their pages missing."""
    import torch
    import large_model_b200 as m
    qs = [0 if b % 13 == 5 else min(q, 1 + b % (q + 2)) for b in range(40)]
    qs[0] = q
    kv = [n + (17 * b) % 90 for b, n in enumerate(qs)]
    check(qs, kv, G=16, D=D, page=32, seed=q, pad=1)
    check(qs, [n + 70 for n in kv], G=16, D=D, page=16, prefix=70, seed=q)
    pages, batch, rows, K, V = make(qs, kv, G=16, D=D, page=16, seed=7)
    b = max(range(40), key=lambda b: kv[b])
    batch.table[b, 1] = -1
    out = m.paged_attention(pages, batch, rows, 32)
    with pytest.raises(m.QmsCudaError, match="0x2"):
        batch.status()
    keep = [j for j in range(kv[b]) if j // 16 != 1]
    K, V = ([x[keep] if i == b else x for i, x in enumerate(z)] for z in (K, V))
    lens = [len(keep) if i == b else n for i, n in enumerate(kv)]
    want, tol = reference(qs, lens, rows, K, V, 16, D ** -0.5)
    assert ((out.double() - want).abs() <= tol).all()
