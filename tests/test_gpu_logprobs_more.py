"""More of the log probabilities on a B200 through the C ABI (qms_cuda_logprobs), against their definition in 64 bits; the bounds are
those of test_gpu_logprobs.py unless a test says otherwise."""
from __future__ import annotations

import pytest

from test_gpu_logprobs import _top, _want, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("V,rows", [(1000, 2), (32003, 2), (32003, 90)])
@pytest.mark.parametrize("temp", [2.0 ** -126, 2e-38, 1.3e-37, 1.5e37, 1.1e38])
def test_temperatures_at_the_ends_of_the_range(cuda, V, rows, temp):
    """log2(e) / temp is a normal number for all of these: the bounds are as for any other. (Logits of temp's size: x is an ordinary number.)"""
    import torch
    g = torch.Generator(device="cuda").manual_seed(V)
    l = torch.randn((rows, V), generator=g, device="cuda").clamp(-2.9, 2.9) * temp
    check(l, torch.randint(0, V, (rows, 2), generator=g, device="cuda").int(), 5, temp=torch.tensor(temp).item())


def test_the_largest_temperature(cuda):
    """log2(e) / temp is below 2^-126: its spacing of 2^-149 is off by up to 2^-150 / 2^-127.47 < 3 * 2^-24 of it, so that a weight is off by 5 e |x|
    where the bounds have 2 e |x|, and each of their terms by at most 2.5 times as much."""
    import torch
    import large_model_b200 as m
    temp = 3.4028234663852886e38
    g = torch.Generator(device="cuda").manual_seed(1)
    l = torch.randn((3, 5000), generator=g, device="cuda").clamp(-2.9, 2.9) * 1e38
    ids = torch.randint(0, 5000, (3, 2), generator=g, device="cuda").int()
    lp, ent, ti, tl = m.logprobs(l, ids, top=4, temp=temp)
    want, tol, went, tent = _want(l, ids, temp)
    assert ((lp.double() - want.gather(1, ids.long())).abs() <= 2.5 * tol.gather(1, ids.long())).all()
    assert ((ent.double() - went).abs() <= 2.5 * tent).all()
    assert ti.tolist() == _top(l.cpu().numpy(), 4).tolist()
    assert ((tl.double() - want.gather(1, ti.long())).abs() <= 2.5 * tol.gather(1, ti.long())).all()


@pytest.mark.parametrize("rows", [2, 90])
@pytest.mark.parametrize("temp", [0.5, 1.0, 3.0, 2.0 ** 100, 2.0 ** 126])
def test_logits_over_the_whole_range(cuda, rows, temp):
    """Two of fp32's extremes differ by more than fp32 holds; x may be an ordinary number all the same. What x is past fp32 is -inf."""
    import torch
    import large_model_b200 as m
    big, V = 3.4028234663852886e38, 20011
    g = torch.Generator(device="cuda").manual_seed(int(temp % 97))
    l = (2 * torch.rand((rows, V), generator=g, device="cuda") - 1) * big
    l[0, 5], l[0, V - 1] = big, -big
    l[1] = -big
    l[1, V // 2] = big
    ids = torch.tensor([5, V - 1, V // 2], device="cuda").int().repeat(rows, 1)
    lp, ent, ti, tl = m.logprobs(l, ids, top=3, temp=temp)
    want, tol, went, tent = _want(l, ids, temp)
    at = want.gather(1, ids.long())
    ok = torch.where(at < -big, lp == -float("inf"), (lp.double() - at).abs() <= tol.gather(1, ids.long()))
    assert ok.all()
    assert ((ent.double() - went).abs() <= tent).all()
    assert ti.tolist() == _top(l.cpu().numpy(), 3).tolist() and ti[1].tolist() == [V // 2, 0, 1]
    at = want.gather(1, ti.long())
    assert torch.where(at < -big, tl == -float("inf"), (tl.double() - at).abs() <= tol.gather(1, ti.long())).all()
