"""Pages in 4 bits with scales that the append does not make, on a B200 through the C ABI: all kernels over a pool read them alike.

A value is d (16 + n) - 24 d, 24 d rounded to fp16 and the difference too: finite up to |d| = 2728 (24 d = 65472; of 2730 it is 65520,
which rounds to infinity). Bounds: K is as the append leaves it, V is exact in fp16 as it is read, so the attention's is that of any pool."""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_cache4 import E24, make, reference

pytestmark = pytest.mark.gpu


def read(n, d):
    """Nibbles and a scale as the kernels read them."""
    d = np.float16(d)
    with np.errstate(over="ignore", invalid="ignore"):
        m24 = np.float16(24.0 * np.float64(d)).astype(np.float64)
        return (np.float64(d) * (16 + n) - m24).astype(np.float16).astype(np.float64)


def rescale(pages, batch, V, at, d, D, page):
    """V's scales at position `at` of the first sequence to d, in the pool and in the values V; the first 32 values of each head."""
    import torch
    P, off = batch.table[0, at // page].item(), at % page
    nib = pages.v[P, :, :page * D // 2].reshape(-1, page, D // 2)[:, off, :16].cpu().numpy().copy().view(np.uint32)
    n = np.stack([nib >> np.uint32(4 * (i // 2) + 16 * (i % 2)) & np.uint32(15) for i in range(8)], -1).reshape(len(nib), 32)
    scales = pages.v[P, :, page * D // 2:]
    scales[:, off * (D // 16):off * (D // 16) + 2] = torch.from_numpy(np.array([d], np.float16).view(np.uint8)).cuda()
    V[0][at, :, :32] = torch.from_numpy(read(n.astype(np.float64), d)).cuda()


@pytest.mark.parametrize("d", [2724.0, 2722.0, -2726.0, 2728.0, -2728.0])
@pytest.mark.parametrize("n,G,D", [(1, 8, 128), (4, 2, 128), (4, 16, 64), (5, 4, 128), (80, 16, 128), (40, 16, 64)])
def test_scales_up_to_where_the_step_overflows(cuda, d, n, G, D):
    """At positions that all new tokens see, that some do, that only the last does."""
    import torch
    import large_model_b200 as m
    kv, page = 600 if n < 40 else 1300, 16
    pages, batch, q, K, V = make([n], [kv], G=G, D=D, page=page, seed=n + G)
    for at in {7, kv - 1, kv - max(1, n // 2)}:
        rescale(pages, batch, V, at, d, D, page)
    k, v = pages.values()
    table = batch.table[0].long()
    assert torch.equal(v[table].flatten(0, 1)[:kv].double(), V[0])
    out = m.paged_attention(pages, batch, q, 2 * G)
    batch.status()
    want, tol = reference([n], [kv], q, K, V, G, D ** -0.5)
    assert ((out.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("d", [2730.0, -2736.0, 8160.0, 65504.0])
@pytest.mark.parametrize("n,G,D", [(4, 2, 128), (4, 16, 64), (80, 16, 128)])
def test_scales_beyond(cuda, d, n, G, D):
    """They are not finite for who sees them, and nothing for who does not."""
    import torch
    import large_model_b200 as m
    kv, page = 600 if n < 40 else 1300, 16
    pages, batch, q, K, V = make([n], [kv], G=G, D=D, page=page, seed=3)
    want, tol = reference([n], [kv], q, K, V, G, D ** -0.5)
    rescale(pages, batch, V, kv - 2, d, D, page)
    assert not V[0][kv - 2, :, :32].isfinite().any()
    out = m.paged_attention(pages, batch, q, 2 * G)
    batch.status()
    assert ((out[:-2].double() - want[:-2]).abs() <= tol[:-2]).all()
    out, want, tol = (x[-2:].reshape(2, 2 * G, D) for x in (out.double(), want, tol))
    assert not out[..., :32].isfinite().any()
    assert ((out[..., 32:] - want[..., 32:]).abs() <= tol[..., 32:]).all()
