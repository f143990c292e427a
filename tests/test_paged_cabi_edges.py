"""More of what the paged-cache entries refuse on the host, before any device call. CPU only."""
from __future__ import annotations

import large_model_b200 as q
from test_paged_cabi import P, _append, _batch, _pages


def test_append_in_place_needs_equal_strides():
    """q over the front of qkv at another stride: a token's q rows would land on rows that others still read."""
    for ldx, ldy in ((1024, 512), (1024, 1028), (1028, 1024)):
        assert _append(_pages(), _batch(), ldx=ldx, ldy=ldy) == q.EINVAL
        assert b"in place" in q.lib().qms_cuda_last_error()
