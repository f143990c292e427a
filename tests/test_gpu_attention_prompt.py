"""Attention within whole prompts on a B200 through the C ABI (qms_cuda_prompt_attention), against its formula in 64 bits.

Bounds, with e = 2^-24 and h the type's half step (bf16 2^-8, fp16 2^-11). q, k, v are exact. A score is off by at most head_dim additions
that cut at e, times A = scale * sum |q k|; a weight by that relatively, by the exponential's 2.6e-6 < 44 e (a polynomial of that error, or 4 e)
and by its rounding, h; an fp16 weight also by half of fp16's smallest step, 2^-25, where the row's largest weight is 2^7 at least.
The sum that divides is that of the rounded weights: with relative errors d_i of the weights p_i the output is off by sum p_i d_i (v_i - o)
/ (1 + sum p_i d_i), at most max |d| (1 + 2 h) (M + |o|) with M = sum p |v|. So by ((D + 8) e A + 48 e + h) (1 + 2 h) (M + |o|), by 2^-31 L
max |v| (fp16; L the positions that the row sees) and by the sums' own cuts, (L / 16 + 8) 2 e M; then by its own rounding, h of
itself (fp32 out: none)."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
E = 2.0 ** -24


def make(lens, *, G=2, Hk=2, D=128, dtype="float16", pad=0, seed=0, qscale=1.0, layout="rows", start0=0):
    """q, k, v as views of one buffer of rows (or heads first), a batch, and the rows behind the last prompt NaN."""
    import torch
    import large_model_b200 as m
    g = torch.Generator(device="cuda").manual_seed(seed)
    H, T = G * Hk, start0 + sum(lens) + pad
    x = torch.randn((T, H + 2 * Hk, D), generator=g, device="cuda")
    x[:, :H] *= qscale
    x = x.to(getattr(torch, dtype))
    x[:start0] = float("nan")
    x[T - pad:] = float("nan")
    if layout == "heads":
        x = x.transpose(0, 1).contiguous().transpose(0, 1)
    elif layout == "wide":
        y = torch.full((T, H + 2 * Hk + 1, D + 8), float("nan"), dtype=x.dtype, device="cuda")
        y[:, :H + 2 * Hk, :D] = x
        x = y[:, :H + 2 * Hk, :D]
    start = torch.tensor((start0 + np.concatenate([[0], np.cumsum(lens)])).tolist(), dtype=torch.int32, device="cuda")
    batch = m.PagedBatch.prompts(start, T, max(lens))
    return batch, x[:, :H], x[:, H:H + Hk], x[:, H + Hk:H + 2 * Hk]


def reference(lens, q, k, v, scale, out32=False, start0=0):
    import torch
    H, D = q.shape[1:]
    Hk = k.shape[1]
    G = H // Hk
    h = torch.finfo(q.dtype).eps / 2
    want = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(want)
    t = start0
    for n in lens:
        for hk in range(Hk):
            for i in range(0, n, 512):
                e = min(n, i + 512)
                x, kk, vv = q[t + i:t + e, hk * G:(hk + 1) * G].double(), k[t:t + e, hk].double(), v[t:t + e, hk].double()
                late = torch.arange(e, device="cuda") > torch.arange(i, e, device="cuda")[:, None]
                s = torch.einsum("igd,jd->gij", x, kk) * scale
                A = (torch.einsum("igd,jd->gij", x.abs(), kk.abs()) * abs(scale)).masked_fill(late, 0.0).amax(-1)
                p = torch.softmax(s.masked_fill(late, -float("inf")), -1)
                want[t + i:t + e, hk * G:(hk + 1) * G] = (p @ vv).transpose(0, 1)
                M, L = p @ vv.abs(), torch.arange(i + 1, e + 1, device="cuda").double()[:, None]
                b = ((D + 8) * E * A + 48 * E + h)[..., None] * (1 + 2 * h) * (M + (p @ vv).abs()) + (L / 16 + 8) * 2 * E * M
                if q.dtype == torch.float16:
                    b = b + 2.0 ** -31 * L * vv.abs().amax()
                tol[t + i:t + e, hk * G:(hk + 1) * G] = b.transpose(0, 1)
        t += n
    if not out32:
        tol = tol + h * (want.abs() + tol) + (2.0 ** -25 if q.dtype == torch.float16 else 0.0)
    return want, tol


def check(lens, scale=None, out32=False, **kw):
    import torch
    import large_model_b200 as m
    batch, q, k, v = make(lens, **kw)
    D = q.shape[2]
    T, t0, t1 = q.shape[0], kw.get("start0", 0), kw.get("start0", 0) + sum(lens)
    out = torch.full(q.shape, 7.0, dtype=torch.float32 if out32 else q.dtype, device="cuda")
    m.prompt_attention(batch, q, k, v, scale=scale, out=out)
    batch.status()
    want, tol = reference(lens, q, k, v, D ** -0.5 if scale is None else scale, out32, t0)
    assert torch.isfinite(out).all()
    over = ((out.double() - want).abs() - tol)[t0:t1]
    assert not sum(lens) or over.max().item() <= 0, f"{over.max().item()} over the bound (worst {(out.double() - want)[t0:t1].abs().max().item()})"
    assert (out[:t0] == 7.0).all() and (out[t1:] == 7.0).all(), "rows of no prompt"
    again = m.prompt_attention(batch, q, k, v, scale=scale, out=torch.full_like(out, 7.0))
    assert torch.equal(out, again), "two runs differ"
    return out


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n", [1, 2, 15, 17, 100, 128, 129, 257])
def test_one_prompt(cuda, dtype, D, n):
    check([n], dtype=dtype, D=D, seed=n, G=4)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("G", [1, 2, 3, 5, 8, 12, 16, 24, 64, 100, 128])
def test_heads_per_group(cuda, D, G):
    check([70, 1, 0, 131, 9], dtype="bfloat16", D=D, G=G, Hk=1 if G > 16 else 3, seed=G, pad=2)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("lens", [[0], [0, 0, 5], [1] * 40, [3, 0, 700, 1, 0, 64, 333, 128, 127, 256, 2], [1500, 40, 900]])
def test_packed(cuda, dtype, lens):
    check(lens, dtype=dtype, G=8, Hk=2, seed=sum(lens), pad=5)
    check(lens, dtype=dtype, G=1, Hk=2, D=64, seed=sum(lens) + 1, start0=3)


@pytest.mark.parametrize("layout", ["heads", "wide"])
@pytest.mark.parametrize("D", [64, 128])
def test_strides(cuda, layout, D):
    check([200, 33], layout=layout, D=D, G=4, Hk=3, seed=1, pad=1)


def test_long(cuda):
    check([5000], G=2, Hk=1, dtype="float16", seed=1)
    check([4097, 100], G=4, Hk=1, D=64, dtype="bfloat16", seed=2)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_rows_out_in_fp32(cuda, dtype):
    check([300, 5], dtype=dtype, out32=True, G=4, seed=4)
    check([300, 5], dtype=dtype, out32=True, G=3, D=64, seed=5)


@pytest.mark.parametrize("qscale,scale", [(30.0, None), (1.0, 1e-6), (1.0, 3.0), (0.0, None)])
def test_scores_large_and_small(cuda, qscale, scale):
    check([700], scale=scale, qscale=qscale, dtype="bfloat16", G=8, Hk=1, seed=3)
    check([700], scale=scale, qscale=qscale, dtype="float16", G=2, Hk=1, seed=3)


@pytest.mark.parametrize("G", [1, 16])
def test_the_base_moves(cuda, G):
    """Scores that rise along the positions, by far more than the weights' range: every tile moves the base."""
    import torch
    import large_model_b200 as m
    n, D = 600, 64
    batch, q, k, v = make([n], G=G, Hk=1, D=D, dtype="bfloat16", seed=1)
    q.fill_(0.25)
    k.copy_((torch.arange(n, device="cuda") * 0.5)[:, None, None].expand(n, 1, D).to(k.dtype))
    out = m.prompt_attention(batch, q, k, v, scale=1.0)
    want, tol = reference([n], q, k, v, 1.0)
    assert ((out.double() - want).abs() <= tol).all()
    k.copy_(-k)                                      # and fall: the first position keeps all the weight
    out = m.prompt_attention(batch, q, k, v, scale=1.0)
    want, tol = reference([n], q, k, v, 1.0)
    assert ((out.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("G,D", [(1, 128), (3, 64), (16, 128)])
def test_what_a_row_does_not_see(cuda, dtype, G, D):
    """NaN and infinities at later tokens and in other prompts change nothing; where they are seen they show."""
    import torch
    import large_model_b200 as m
    lens = [300, 40, 200]
    batch, q, k, v = make(lens, G=G, Hk=2, D=D, dtype=dtype, seed=6)
    want = m.prompt_attention(batch, q, k, v)
    k[290, 1] = float("nan")
    v[297, 0, 5] = float("inf")
    v[340:, :, 3] = float("nan")
    q[339] = float("nan")
    out = m.prompt_attention(batch, q, k, v)
    same = torch.ones(q.shape, dtype=torch.bool, device="cuda")
    same[290:300, G:] = False
    same[297:300, :G, 5] = False
    same[339] = False
    same[340:, :, 3] = False
    assert torch.equal(out[same], want[same])
    assert out[290:300, G:].isnan().all() and not out[297:300, :G, 5].isfinite().any() and out[339].isnan().all() and out[340:, :, 3].isnan().all()


def test_infinite_scores(cuda):
    """A key of score -inf has no weight; one of +inf makes the row NaN, as the formula does."""
    import torch
    import large_model_b200 as m
    batch, q, k, v = make([50], G=2, Hk=1, D=64, dtype="bfloat16", seed=2)
    q.copy_(q.abs() + 0.125)
    k[7] = -float("inf")
    k[45] = float("inf")
    out = m.prompt_attention(batch, q, k, v)
    keep = torch.arange(50, device="cuda") != 7
    want, tol = reference([49], q[keep], k[keep], v[keep], 64 ** -0.5)
    rows = torch.arange(50, device="cuda")[keep] < 45
    assert ((out[keep].double() - want).abs() <= tol)[rows].all()
    assert out[45:].isnan().all()


def test_in_place(cuda):
    import torch
    import large_model_b200 as m
    batch, q, k, v = make([300, 77], G=8, Hk=2, seed=1, pad=1)
    want = m.prompt_attention(batch, q, k, v)
    got = m.prompt_attention(batch, q, k, v, out=q)
    assert got.data_ptr() == q.data_ptr() and torch.equal(got[:377], want[:377])


def test_prompts_that_make_no_sense(cuda):
    import torch
    import large_model_b200 as m
    batch, q, k, v = make([30, 40, 50], G=4, seed=1)
    want = m.prompt_attention(batch, q, k, v)
    for bad, ok in (([0, 30, 25, 120], slice(0, 30)), ([0, 30, 70, 121], slice(0, 70)), ([-1, 30, 70, 120], slice(30, 120)), ([0, 30, 70, 1 << 30], slice(0, 70))):
        batch.q_start.copy_(torch.tensor(bad, dtype=torch.int32))
        out = m.prompt_attention(batch, q, k, v, out=torch.full_like(want, 7.0))
        with pytest.raises(m.QmsCudaError, match="0x1"):
            batch.status()
        if bad[2] > bad[1]:
            assert torch.equal(out[ok], want[ok])
        else:
            assert torch.equal(out[ok][:25], want[ok][:25])


def test_graphs_and_streams(cuda):
    import torch
    import large_model_b200 as m
    batch, q, k, v = make([700, 33, 128], G=8, seed=3)
    want = m.prompt_attention(batch, q, k, v)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = m.prompt_attention(batch, q, k, v, stream=s)
    s.synchronize()
    out = torch.zeros_like(want)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        m.prompt_attention(batch, q, k, v, out=out)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(want, got) and torch.equal(want, out)
    batch.q_start.copy_(torch.tensor([0, 100, 100, 861], dtype=torch.int32))         # replayed as the prompts change
    batch.desc.max_q = 861
    graph.replay()
    with pytest.raises(m.QmsCudaError):                                             # (the graph's bound is 700)
        batch.status()
    batch.q_start.copy_(torch.tensor([0, 161, 161, 861], dtype=torch.int32))
    out.zero_()
    graph.replay()
    batch.status()
    assert torch.equal(out, m.prompt_attention(batch, q, k, v))


def test_refusals(cuda):
    import torch
    import large_model_b200 as m
    batch, q, k, v = make([30], G=4, seed=1)
    for bad in (lambda: m.prompt_attention(batch, q.float(), k.float(), v.float()), lambda: m.prompt_attention(batch, q, k.bfloat16(), v),
                lambda: m.prompt_attention(batch, q[:20], k, v), lambda: m.prompt_attention(batch, q, k[:, :1], v),
                lambda: m.prompt_attention(batch, q, k, v, out=torch.empty_like(q, dtype=torch.bfloat16)), lambda: m.prompt_attention(batch, q.cpu(), k, v)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: m.prompt_attention(batch, q[:, :7], k, v), lambda: m.prompt_attention(batch, q, k, v, scale=0.0),
                lambda: m.prompt_attention(batch, q, k, v, scale=-1.0), lambda: m.prompt_attention(batch, q[..., :96], k[..., :96], v[..., :96])):
        with pytest.raises(m.QmsCudaError):
            bad()


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_scores_beyond_two_to_the_27(cuda, dtype):
    """Scores whose own rounding in fp32 is whole powers of 2 of a weight: the rows say so. (What a row does not see is no reason to.)"""
    import torch
    import large_model_b200 as m
    n, D = 200, 64
    g = torch.Generator(device="cuda").manual_seed(3)
    step = torch.randperm(n, generator=g, device="cuda") // 2 + 100          # two positions each
    typ = getattr(torch, dtype)
    q = torch.full((n, 2, D), 4096.0, device="cuda", dtype=typ)
    k = (step * 256.0)[:, None, None].expand(n, 1, D).to(typ).contiguous()
    v = torch.randn((n, 1, D), generator=g, device="cuda").to(typ)
    batch = m.PagedBatch.prompts(torch.tensor([0, n], dtype=torch.int32, device="cuda"), n, n)
    out = m.prompt_attention(batch, q, k, v, out_dtype=torch.float32)
    batch.status()
    assert out.isnan().all()
    q[:150] = 0
    out = m.prompt_attention(batch, q, k, v, out_dtype=torch.float32)
    want = v[:, 0].double().cumsum(0)[:150] / torch.arange(1, 151, device="cuda")[:, None]
    assert ((out[:150].double() - want[:, None]).abs() <= 32 * E * v.abs().max()).all() and out[150:].isnan().all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype,out", [("float16", "float16"), ("bfloat16", "bfloat16"), ("float16", "float32")])
def test_rows_out_on_16_byte_boundaries(cuda, D, dtype, out):
    """Rows that begin between two sectors of 32 bytes hold the same bits, and what lies between them stays."""
    import torch
    import large_model_b200 as m
    lens, H, Hk = [37, 1, 150], 6, 2
    n = sum(lens)
    g = torch.Generator(device="cuda").manual_seed(D)
    x = torch.randn((n, H + 2 * Hk, D), generator=g, device="cuda").to(getattr(torch, dtype))
    q, k, v = x[:, :H], x[:, H:H + Hk], x[:, H + Hk:]
    batch = m.PagedBatch.prompts(torch.tensor([0] + np.cumsum(lens).tolist(), dtype=torch.int32, device="cuda"), n, max(lens))
    typ = getattr(torch, out)
    step = 16 // typ.itemsize                        # values in 16 bytes
    want = m.prompt_attention(batch, q, k, v, out_dtype=typ)
    for first, gap in ((step, 0), (0, step), (step, step)):
        flat = torch.full((first + n * (H * D + gap),), float("nan"), dtype=typ, device="cuda")
        rows = flat[first:].view(n, H * D + gap)
        m.prompt_attention(batch, q, k, v, out=rows[:, :H * D].unflatten(1, (H, D)))
        assert torch.equal(rows[:, :H * D], want.flatten(1))
        assert flat[:first].isnan().all() and rows[:, H * D:].isnan().all()
    heads = torch.full((H, n * D + step), float("nan"), dtype=typ, device="cuda")             # heads before tokens
    m.prompt_attention(batch, q, k, v, out=heads[:, step:].unflatten(1, (n, D)).transpose(0, 1))
    assert torch.equal(heads[:, step:].unflatten(1, (n, D)).transpose(0, 1), want) and heads[:, :step].isnan().all()
    batch.status()
