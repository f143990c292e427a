"""The paged operators on streams other than the one that their tensors come from: what a PagedBatch keeps for itself (its error
word, its workspaces) and the results that a call allocates are ordered with the call."""
from __future__ import annotations

import pytest

from test_gpu_paged import make, reference

pytestmark = pytest.mark.gpu
LONG = 100_000_000                                   # cycles, some 50 ms


def test_status_waits_for_every_stream(cuda):
    import torch
    import large_model_b200 as m
    pages, batch, q, K, V = make([1, 2], [50, 33], G=4)
    batch.table[1, 1] = -1
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(LONG)
    out = m.paged_attention(pages, batch, q, 8, stream=side)
    with pytest.raises(m.QmsCudaError, match="0x2"):
        batch.status()
    torch.cuda.synchronize()
    del out


def test_error_word_is_zero_before_a_call_on_another_stream(cuda):
    """The batch is made behind work of the current stream; a call on another stream waits for its error word."""
    import torch
    import large_model_b200 as m
    pages, old, q, K, V = make([1, 2], [50, 33], G=4)
    old.table[1, 1] = -1
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    torch.cuda._sleep(LONG)
    batch = m.PagedBatch(old.q_start, old.kv_len, old.table, 3, 2, 50)
    m.paged_attention(pages, batch, q, 8, stream=side)
    with pytest.raises(m.QmsCudaError, match="0x2"):
        batch.status()
    torch.cuda._sleep(LONG)                          # the same after an error was cleared
    batch.err.fill_(0)
    batch._cleared()
    with torch.cuda.stream(side):
        m.paged_attention(pages, batch, q, 8)
    with pytest.raises(m.QmsCudaError, match="0x2"):
        batch.status()
    old.table[1, 1] = old.table[0, 0]
    m.paged_attention(pages, batch, q, 8)
    batch.status()


def test_workspace_and_results_live_as_long_as_the_call(cuda):
    """A batch object that goes while its call is queued on another stream: its workspace is not handed out meanwhile, nor is
    the memory of a result that the call allocates still in use on the current stream."""
    import torch
    import large_model_b200 as m
    qs, kv = [3, 1, 5], [300, 90, 170]
    pages, batch, q, K, V = make(qs, kv, G=8)
    want, tol = reference(qs, kv, q, K, V, 8, 128 ** -0.5)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(LONG)
    out = m.paged_attention(pages, batch, q, 16, stream=side)
    n = batch.workspace(pages, 16, side.cuda_stream)[1] + 256
    del batch
    fill = [torch.full((n,), 7, dtype=torch.uint8, device="cuda") for _ in range(3)]
    torch.cuda.synchronize()
    assert all((x == 7).all() for x in fill)
    assert ((out.double() - want).abs() <= tol).all()


def test_two_streams_share_a_batch(cuda):
    import torch
    import large_model_b200 as m
    qs, kv = [1, 4, 30], [900, 640, 2000]
    pages, batch, q, K, V = make(qs, kv, G=8)
    want, tol = reference(qs, kv, q, K, V, 8, 128 ** -0.5)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [m.paged_attention(pages, batch, q, 16, stream=streams[i % 2]) for i in range(40)]
    batch.status()
    for out in outs:
        assert ((out.double() - want).abs() <= tol).all()


def test_results_of_probs_and_verify_on_another_stream(cuda):
    import torch
    import large_model_b200 as m
    g = torch.Generator(device="cuda").manual_seed(1)
    logits = torch.randn((15, 4096), generator=g, device="cuda")
    draft = torch.randint(0, 4096, (3, 4), generator=g, device="cuda", dtype=torch.int32)
    u = torch.rand((3, 5), generator=g, device="cuda")
    p = m.probs(logits, 0.7)
    n, t = m.verify(p, draft, u)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(LONG)
    p2 = m.probs(logits, 0.7, stream=side)
    n2, t2 = m.verify(p2, draft, u, stream=side)
    torch.cuda.synchronize()
    assert torch.equal(p, p2) and torch.equal(n, n2) and torch.equal(t, t2)


FIRST_CALLS = """
import threading, torch
import large_model_b200 as m
m.init(0)
g = torch.Generator(device="cuda").manual_seed(1)
P, Hk, D, H, n = 16, 2, 128, 32, 5
k, v = (torch.randn((12, P, Hk, D), generator=g, device="cuda") for _ in range(2))
q = torch.randn((2 * n, H * D), generator=g, device="cuda")
logits = torch.randn((4, 32003), generator=g, device="cuda")
ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
start, kv, table = ints([0, n, 2 * n]), ints([90, 50]), ints([list(range(6)), list(range(6, 12))])
torch.cuda.synchronize()
res, go = [None] * 8, threading.Barrier(8)

def work(i):
    torch.cuda.set_device(0)
    with torch.cuda.stream(torch.cuda.Stream()):
        batch = m.PagedBatch(start, kv, table, 2 * n, n, 96)
        pages = m.KvPages(k, v) if i % 2 else m.KvPages(k.half(), v.half())
        torch.cuda.current_stream().synchronize()
        go.wait()
        out = [m.paged_attention(pages, batch, q, H), m.probs(logits, 0.8 * (i % 4 > 1))]
        batch.status()
        res[i] = out

t = [threading.Thread(target=work, args=(i,)) for i in range(8)]
[x.start() for x in t]
[x.join() for x in t]
for i in range(4, 8):
    assert torch.equal(res[i][0], res[i - 4][0]) and torch.equal(res[i][1], res[i - 4][1])
print("same")
"""


def test_first_calls_from_several_threads(cuda):
    import subprocess
    import sys
    from conftest import ROOT
    r = subprocess.run([sys.executable, "-c", FIRST_CALLS], cwd=ROOT, capture_output=True, text=True, timeout=240)
    assert r.returncode == 0 and "same" in r.stdout, r.stderr[-2000:]
