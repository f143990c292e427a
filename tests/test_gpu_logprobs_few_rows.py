"""Log probabilities of few rows on a B200 through the C ABI (qms_cuda_logprobs), where the likeliest come from a list: rows in which a
warp has hardly any values, or none that is not masked away. Bounds as in test_gpu_logprobs.py."""
from __future__ import annotations

import pytest

from test_gpu_logprobs import check

pytestmark = pytest.mark.gpu
INF = float("inf")


def ids_of(l):
    return l.argmax(-1).int()


@pytest.mark.parametrize("V", [513, 516, 1025, 1028, 1540, 1541, 2052, 3588, 4092, 8196, 151936])
@pytest.mark.parametrize("top", [1, 7, 8, 9, 10, 31, 32])
def test_warps_with_hardly_any_values(cuda, V, top):
    import torch
    g = torch.Generator(device="cuda").manual_seed(V + top)
    l = 3 * torch.randn((2, V), generator=g, device="cuda")
    check(l, ids_of(l), top)
    l[1] = -1.0
    l[1, V // 3] = 2.0
    check(l, ids_of(l), top)


@pytest.mark.parametrize("low", [-INF, -3.4028234663852886e38, -1e9])
@pytest.mark.parametrize("V", [1540, 4096, 32003, 151936])
def test_masks_that_leave_warps_with_nothing(cuda, low, V):
    """Ranges of values that some warps, or some CTAs, have no part in; down to fewer values than are asked for."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(V)
    for a, b in ((0, V // 2), (V // 2, V), (V // 3, V // 3 + 700), (0, 5), (V - 5, V), (V // 2, V // 2 + 40)):
        l = torch.full((2, V), low, device="cuda")
        l[0, a:b] = 3 * torch.randn((l[0, a:b].numel(),), generator=g, device="cuda")
        l[1, a:b] = torch.randint(-2, 3, (l[1, a:b].numel(),), generator=g, device="cuda").float()      # with equals
        for top in (10, 32):
            check(l, ids_of(l), top)


@pytest.mark.parametrize("V,every,some", [(151936, 128, 4), (32003, 128, 16), (4096, 512, 40)])
def test_values_that_few_lanes_have(cuda, V, every, some):
    """All but `some` of `every` ids masked away: those that are left are in fewer lanes than are asked for, or hardly more."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(V)
    l = torch.randn((2, V), generator=g, device="cuda")
    l[1] = torch.randint(-2, 3, (V,), generator=g, device="cuda").float()
    for first in (0, 64):
        x = l.clone()
        x[:, (torch.arange(V, device="cuda") + first) % every >= some] = -INF
        for top in (1, 10, 32):
            check(x, ids_of(x), top)


def us(f):
    """The least time of a call among 20 in a graph, of 10 replays."""
    import torch
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        f()
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            for _ in range(20):
                f()
        times = []
        for _ in range(10):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            graph.replay()
            b.record()
            s.synchronize()
            times.append(a.elapsed_time(b) * 1000 / 20)
    return min(times)


def test_no_size_or_mask_takes_many_times_as_long(cuda):
    """A list of all values, each ranked against each, takes 100 us for a row of 1540, and one pass per value 50 for a long one. Ordinary rows: 6
    and 10 us."""
    import torch
    import large_model_b200 as m
    l = torch.randn((1, 4096), device="cuda")
    usual = us(lambda: m.logprobs(l, top=10))
    for V in (1028, 1540, 2052, 4092):
        x = l[:, :V]
        assert us(lambda: m.logprobs(x, top=10)) < 3 * usual, V
    l = torch.randn((1, 151936), device="cuda")
    usual = us(lambda: m.logprobs(l, top=10))
    for low in (-INF, -1e9):
        x = l.clone()
        x[0, 40000:100000] = low
        assert us(lambda: m.logprobs(x, top=10)) < 3 * usual, low
        x[0, 1000:] = low
        assert us(lambda: m.logprobs(x, top=10)) < 3 * usual, low
