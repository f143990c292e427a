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


@pytest.mark.parametrize("n_seq,H,Hk", [(65536, 2, 1), (33000, 4, 4)])
def test_thousands_of_prompts_take_a_time_that_grows_with_them(cuda, n_seq, H, Hk):
    """A token each, then none each but for the last. A search from the first prompt on for every unit would take some n_seq^2 / 64 round trips
    to memory, 160 ms; the work itself is 1 to 5."""
    import torch
    import large_model_b200 as m
    q, k, v = rows(n_seq, H, Hk, 64)
    batch = m.PagedBatch.prompts(torch.arange(n_seq + 1, device="cuda").int(), n_seq, 1)
    out = m.prompt_attention(batch, q, k, v)
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    a.record()
    m.prompt_attention(batch, q, k, v, out=out)
    b.record()
    batch.status()
    assert torch.equal(out, v.repeat_interleave(H // Hk, 1))
    assert a.elapsed_time(b) < 60.0
    batch.q_start.zero_()
    batch.q_start[n_seq] = 1
    out.fill_(7.0)
    m.prompt_attention(batch, q, k, v, out=out)
    batch.status()
    assert torch.equal(out[0], v[0].repeat_interleave(H // Hk, 0)) and (out[1:] == 7.0).all()


def test_lengths_in_an_order_that_jumps(cuda):
    """Long prompts between thousands of short and empty ones: units of a prompt from its end, many per block of the search, or none."""
    import torch
    import large_model_b200 as m
    g = torch.Generator().manual_seed(5)
    n = torch.randint(0, 3, (3000,), generator=g)
    n[[0, 700, 701, 1999, 2999]] = torch.tensor([900, 0, 1300, 257, 400])
    n[100:400] = 0
    start = torch.cat([torch.zeros(1, dtype=torch.long), n.cumsum(0)])
    T = int(start[-1])
    q, k, v = rows(T, 8, 2, 64, dtype=torch.float16)
    batch = m.PagedBatch.prompts(start.int().cuda(), T, 1300)
    out = m.prompt_attention(batch, q, k, v)
    batch.status()
    for i in (0, 1, 50, 399, 400, 699, 701, 702, 1500, 1999, 2000, 2998, 2999):     # each by itself says the same
        t0, t1 = int(start[i]), int(start[i + 1])
        if t1 == t0:
            continue
        alone = m.PagedBatch.prompts(torch.tensor([0, t1 - t0], dtype=torch.int32, device="cuda"), t1 - t0, t1 - t0)
        assert torch.equal(out[t0:t1], m.prompt_attention(alone, q[t0:t1], k[t0:t1], v[t0:t1])), i
