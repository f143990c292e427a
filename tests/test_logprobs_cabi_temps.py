"""qms_cuda_logprobs refuses temperatures whose reciprocal fp32 does not hold, on the host. CPU only."""
from __future__ import annotations

import pytest

import large_model_b200 as q
from test_logprobs_cabi import _call


@pytest.mark.parametrize("temp", [1e-45, 1e-39, 1.1754942e-38])
def test_temperatures_below_the_normal_numbers(temp):
    assert _call(temp=temp) == q.EINVAL and b"temp" in q.lib().qms_cuda_last_error()


@pytest.mark.parametrize("temp", [2.0 ** -126, 3.4028234663852886e38])
def test_temperatures_at_the_ends(temp):
    assert _call(temp=temp, rows=0) == q.OK
