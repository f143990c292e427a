"""Rows far apart, so that offsets pass 32 bits, on a B200 through the C ABI: the same bits as for rows that lie together."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu


def apart(t, step):
    """t's first dimension at distance `step`, in a buffer of its own."""
    import torch
    out = torch.empty((t.shape[0] * step,), dtype=t.dtype, device="cuda").as_strided(t.shape, (step, *t.stride()[1:]))
    out.copy_(t)
    return out


@pytest.mark.parametrize("rows", [3, 700])
def test_logprobs(cuda, rows):
    import torch
    import large_model_b200 as m
    l = torch.randn((rows, 1000), device="cuda")
    ids = torch.arange(rows, device="cuda").int()
    far = apart(l, (5 << 30) // rows // 4 * 4)
    for a, b in zip(m.logprobs(l, ids, top=5), m.logprobs(far, ids, top=5)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("D", [64, 128])
def test_prompt_attention(cuda, dtype, D):
    """With V that is not finite behind the mask, which is fetched again from there."""
    import torch
    import large_model_b200 as m
    n, H, Hk = 200, 4, 2
    q, k, v = (torch.randn((n, h, D), device="cuda").to(getattr(torch, dtype)) for h in (H, Hk, Hk))
    v[150, 1, 3] = float("inf")
    batch = m.PagedBatch.prompts(torch.tensor([0, 60, n], dtype=torch.int32, device="cuda"), n, 140)
    step = (5 << 30) // n // 64 * 64
    want = m.prompt_attention(batch, q, k, v)
    out = apart(torch.zeros_like(want), step)
    got = m.prompt_attention(batch, apart(q, step), apart(k, step), apart(v, step), out=out)
    batch.status()
    assert torch.equal(got.contiguous().view(torch.int16), want.view(torch.int16))


def test_prompt_append(cuda):
    import torch
    import large_model_b200 as m
    n, H, Hk, D = 50, 4, 2, 128
    qkv = torch.randn((n, (H + 2 * Hk) * D), device="cuda")
    w = torch.ones(D, device="cuda")
    rope = m.rope_tables(n, D)
    batch = m.PagedBatch.prompts(torch.tensor([0, n], dtype=torch.int32, device="cuda"), n, n)
    step = (5 << 30) // n // 64 * 64
    want = m.prompt_append(None, batch, qkv, H, w, w, 1e-6, rope, n_head_kv=Hk)
    rows = apart(torch.zeros((n, (H + 2 * Hk) * D), dtype=torch.bfloat16, device="cuda"), step)
    m.prompt_append(None, batch, apart(qkv, step), H, w, w, 1e-6, rope, rows=rows, n_head_kv=Hk)
    batch.status()
    assert torch.equal(rows.contiguous().view(torch.int16), want.flatten(1).view(torch.int16))
