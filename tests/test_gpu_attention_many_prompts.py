"""Many prompts in one call of the prompt attention on a B200: what the search for their rows and the check of their lengths have to
cope with. A prompt of one token has its own value as its output, whatever the scores are: a weight of 1 and a sum of 1."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu


def rows(n_tok, H, Hk, D, seed=0, dtype=None):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = dtype or torch.bfloat16
    return tuple(torch.randn((n_tok, h, D), generator=g, device="cuda").to(dtype) for h in (H, Hk, Hk))


@pytest.mark.parametrize("n_seq,H,Hk", [(5, 4, 2), (700, 4, 1), (700, 16, 4)])
@pytest.mark.parametrize("empty", [False, True])
def test_a_prompt_that_makes_no_sense_is_reported_wherever_it_stands(cuda, n_seq, H, Hk, empty):
    """One token each, or all empty but two: then there are fewer units of work than prompts."""
    import torch
    import large_model_b200 as m
    n_tok = 2 if empty else n_seq
    q, k, v = rows(n_tok, H, Hk, 64)
    start = torch.arange(n_seq + 1, device="cuda").clamp(max=n_tok).int()
    batch = m.PagedBatch.prompts(start.clone(), n_tok, 1)
    want = m.prompt_attention(batch, q, k, v)
    batch.status()
    assert torch.equal(want, v.repeat_interleave(H // Hk, 1))
    for at in sorted({1, n_seq // 2, n_seq - 1, min(n_seq - 1, 31), min(n_seq - 1, 32), min(n_seq - 1, 33)}):
        for bad in (-1, n_tok + 1, 1 << 30):
            batch.q_start.copy_(start)
            batch.q_start[at] = bad
            out = m.prompt_attention(batch, q, k, v)
            with pytest.raises(m.QmsCudaError, match="0x1"):
                batch.status()
            rest = [t for t in range(n_tok) if t not in (at - 1, at)]
            assert torch.equal(out[rest], want[rest])
    batch.q_start.copy_(start)
    batch.q_start[n_seq] = n_tok + 1
    m.prompt_attention(batch, q, k, v)
    with pytest.raises(m.QmsCudaError, match="0x1"):
        batch.status()
