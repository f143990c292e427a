"""The paged cache in 4 bits at the lengths it is for, on a B200 through the C ABI: sequences of 131,072 positions and more, on both
sides of what goes to fp16 in the workspace, and offsets past 32 bits. Bounds as in test_gpu_cache4.py. Pools are drawn on the device:
any nibbles, scales of 8 bits."""
from __future__ import annotations

import pytest

from test_gpu_cache4 import E24

pytestmark = pytest.mark.gpu


def ints(x):
    import torch
    return torch.as_tensor(x, dtype=torch.int32, device="cuda")


def pool(n_pages, Hk, page, D, g):
    """(the pool's bytes, its values float32 [n_pages][page][Hk][D])"""
    import torch
    raw = torch.empty((n_pages, Hk, page * D * 9 // 16), dtype=torch.uint8, device="cuda")
    nib, sc = raw[..., :page * D // 2], raw[..., page * D // 2:]
    nib.copy_(torch.randint(0, 256, nib.shape, generator=g, device="cuda", dtype=torch.uint8))
    d = torch.randint(128, 256, (n_pages, Hk, page, D // 32), generator=g, device="cuda") / 1024.0 * (1 - 2 * torch.randint(0, 2, (n_pages, Hk, page, D // 32), generator=g, device="cuda"))
    sc.copy_(d.half().view(torch.uint8).flatten(2))
    w = nib.contiguous().view(torch.int32).view(n_pages, Hk, page, D // 8, 1)
    n = w >> torch.tensor([4 * (i // 2) + 16 * (i % 2) for i in range(8)], device="cuda", dtype=torch.int32) & 15
    v = (n.flatten(-2) - 8).float() * d.float().repeat_interleave(32, -1)
    return raw, v.transpose(1, 2)


def case(qs, kv, G, Hk, D, page, prefix=0, seed=0):
    import torch
    import large_model_b200 as m
    g = torch.Generator(device="cuda").manual_seed(seed)
    shared = prefix // page
    need = [max(0, -(-n // page) - shared) for n in kv]
    order = torch.randperm(shared + sum(need) + 1, generator=g, device="cuda").int()
    table = torch.full((len(qs), shared + max(need)), 1 << 20, dtype=torch.int32, device="cuda")
    table[:, :shared] = order[:shared]
    at = shared
    for b, n in enumerate(need):
        table[b, shared:shared + n] = order[at:at + n]
        at += n
    (k, kx), (v, vx) = (pool(len(order), Hk, page, D, g) for _ in range(2))
    T = sum(qs)
    q = torch.randn((T, Hk * G * D), generator=g, device="cuda")
    starts = [sum(qs[:b]) for b in range(len(qs) + 1)]
    batch = m.PagedBatch(ints(starts), ints(kv), table, T, max(qs), max(kv), prefix)
    out = m.paged_attention(m.KvPages.packed(k, v, D), batch, q, Hk * G)
    batch.status()
    for b, n in enumerate(qs):
        pages = table[b, :-(-kv[b] // page)].long()
        K, V = (x[pages].flatten(0, 1)[:kv[b]].transpose(0, 1).double() for x in (kx, vx))       # [Hk][positions][D]
        for i in range(n):
            end = kv[b] - n + i + 1
            x = q[starts[b] + i].double().view(Hk, G, D) * D ** -0.5
            want = torch.softmax(x @ K[:, :end].transpose(1, 2), -1) @ V[:, :end]
            A = (x.abs() @ K[:, :end].abs().transpose(1, 2)).amax(-1, keepdim=True)
            tol = (16 * A + 16) * E24 * V[:, :end].abs().amax((1, 2), keepdim=True)
            got = out[starts[b] + i].double().view(Hk, G, D)
            assert ((got - want).abs() <= tol).all(), f"sequence {b}, token {i}: {((got - want).abs() / tol).max().item()} of the bound"
    again = m.paged_attention(m.KvPages.packed(k, v, D), batch, q, Hk * G)
    assert torch.equal(out.view(torch.int32), again.view(torch.int32))


@pytest.mark.parametrize("qs,kv,G,Hk,D,page,prefix", [
    ([1], [131072], 8, 4, 128, 64, 0),
    ([1], [131071], 16, 4, 128, 16, 0),
    ([2], [200003], 4, 1, 64, 1024, 0),
    ([1, 3, 1], [131072, 7, 99999], 8, 2, 128, 64, 0),
    ([1, 2], [131200, 131105], 4, 2, 128, 64, 131072),                 # few rows on a long shared prompt
])
def test_few_rows(cuda, qs, kv, G, Hk, D, page, prefix):
    case(qs, kv, G, Hk, D, page, prefix, seed=sum(kv))


@pytest.mark.parametrize("qs,kv,G,Hk,D,page,prefix", [
    ([20], [131072], 16, 4, 128, 64, 0),                               # 128 MiB of K in fp16, and of V: the most that goes to the workspace
    ([20], [131073], 16, 4, 128, 64, 0),                               # past it: a tile at a time
    ([40], [150001], 8, 4, 128, 16, 0),
    ([9, 8], [131072 + 70, 131072 + 40], 16, 4, 128, 128, 131072),     # a prompt of that length, and one past it
    ([9, 8], [131200 + 70, 131200 + 40], 16, 4, 128, 128, 131200),
    ([5], [131072], 14, 4, 128, 32, 0),                                # 70 rows
])
def test_many_rows_on_both_sides_of_the_workspace(cuda, qs, kv, G, Hk, D, page, prefix):
    case(qs, kv, G, Hk, D, page, prefix, seed=sum(kv))


def test_the_workspace_is_bounded(cuda):
    """Past 128 MiB there are the slots alone: one per unit of at most 2304 positions, and of more than 512 here (320 rows in 3 tiles on 4 kv
    heads are 12 units per slot, so 256 slots would be some 3000 units for 148 CTAs), 520 bytes per row and slot."""
    import large_model_b200 as m
    import torch
    Hk, D, page, H = 4, 128, 64, 64
    pages = m.KvPages.empty(4, page, Hk, D, m.T_Q4_0)
    sizes = []
    for kv in (131072, 131073):
        table = torch.zeros((1, -(-kv // page)), dtype=torch.int32, device="cuda")
        sizes.append(m.PagedBatch(ints([0, 20]), ints([kv]), table, 20, 20, kv).workspace(pages, H)[1])
    assert sizes[0] > 256 << 20
    assert 57 * 20 * H * 520 <= sizes[1] <= 256 * 20 * H * 520 + 512


@pytest.mark.parametrize("D", [64, 128])
def test_append_past_4_gb(cuda, D):
    """The last page of a pool of 5 GB, and a small one: the same bytes; what lies around them stays."""
    import torch
    import large_model_b200 as m
    H, Hk, page = 4, 2, 64
    size = page * D * 9 // 16
    N = (5 << 30) // (Hk * size)
    g = torch.Generator(device="cuda").manual_seed(D)
    qkv = torch.randn((40, (H + 2 * Hk) * D), generator=g, device="cuda")
    w = torch.rand((2, D), generator=g, device="cuda") + 0.5
    rope = m.rope_tables(64, D)
    results = []
    for n_pages in (2, N):
        k, v = (torch.full((n_pages, Hk, size), 77, dtype=torch.uint8, device="cuda") for _ in range(2))
        batch = m.PagedBatch(ints([0, 40]), ints([60]), ints([[n_pages - 1]]), 40, 40, 64)
        pages = m.KvPages.packed(k, v, D)
        q = m.paged_append(pages, batch, qkv, H, w[0], w[1], 1e-6, rope)
        one = (k[n_pages - 1].clone(), v[n_pages - 1].clone())
        k.fill_(77), v.fill_(77)
        rows = m.prompt_append(pages, batch, qkv, H, w[0], w[1], 1e-6, rope)
        batch.status()
        assert torch.equal(k[n_pages - 1], one[0]) and torch.equal(v[n_pages - 1], one[1])
        assert (k[n_pages - 2] == 77).all() and (v[0] == 77).all()
        results.append((q, rows.view(torch.int16), *one))
    for a, b in zip(*results):
        assert torch.equal(a, b)
