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
