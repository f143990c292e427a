"""A paged cache in 4 bits, rows of whole prompts and what a pool holds: bad arguments are refused on the host, before any device
call. CPU only."""
from __future__ import annotations

import ctypes as C

import pytest

import large_model_b200 as q

P = C.c_void_p(4096)


def _pages(**kw):
    d = dict(type=q.T_Q4_0, n_pages=4, page_size=16, n_head_kv=2, head_dim=128, page_stride=2304, pos_stride=0, head_stride=1152, k=4096, v=4096)
    d.update(kw)
    return q.PagesDesc(**d)


def _batch(**kw):
    d = dict(n_seq=2, n_tok=3, q_start=4096, kv_len=4096, table=4096, table_stride=2, max_q=2, max_kv=32, prefix_len=16)
    d.update(kw)
    return q.PagedBatchDesc(**d)


def _rows(pg, bt, x=P, ldx=1024, H=4, n=P, cos=P, n_rope=32, typ=q.T_BF16, y=P, ldy=1024):
    return q.lib().qms_cuda_prompt_append(C.byref(pg), C.byref(bt), x, ldx, H, n, n, 1e-6, cos, cos, n_rope, typ, y, ldy, None, None)


@pytest.mark.parametrize("kw,rc", [
    (dict(page_size=8), q.EINVAL), (dict(page_size=24), q.EINVAL), (dict(page_size=1 << 21), q.EINVAL), (dict(pos_stride=64), q.EINVAL),
    (dict(head_stride=1160), q.EINVAL), (dict(page_stride=-16), q.EINVAL), (dict(head_dim=32), q.EUNSUPPORTED), (dict(k=4104), q.EINVAL),
    (dict(type=q.T_Q4_1), q.EUNSUPPORTED), (dict(v=None), q.EINVAL), (dict(n_pages=0), q.EINVAL)])
def test_pages_are_checked(kw, rc):
    pg, L = _pages(**kw), q.lib()
    assert _rows(pg, _batch()) == rc and L.qms_cuda_last_error()
    assert L.qms_cuda_paged_append(C.byref(pg), C.byref(_batch()), P, 1024, 4, P, P, 1e-6, P, P, 32, P, 512, None, None) == rc
    assert L.qms_cuda_paged_attention(C.byref(pg), C.byref(_batch()), P, 512, 4, 1.0, P, 512, P, 1 << 40, None, None) == rc
    assert L.qms_cuda_paged_attention_ws(C.byref(pg), C.byref(_batch()), 4) == rc
    assert L.qms_cuda_paged_values(C.byref(pg), P, P, None) == rc


def test_prompt_rows_are_checked():
    pg, bt = _pages(), _batch()
    for kw in (dict(x=None), dict(x=C.c_void_p(4100)), dict(ldx=1020), dict(y=None), dict(y=C.c_void_p(4104)), dict(ldy=1020), dict(ldy=1028),
               dict(n=None), dict(cos=None), dict(n_rope=0), dict(H=3), dict(H=0)):
        assert _rows(pg, bt, **kw) == q.EINVAL, kw
    assert _rows(pg, bt, typ=q.T_F32) == q.EUNSUPPORTED
    assert _rows(pg, _batch(max_kv=33)) == q.EINVAL and _rows(pg, _batch(kv_len=None)) == q.EINVAL
    none = _pages(n_pages=0, k=None, v=None, page_size=0)
    assert _rows(none, _batch(q_start=None)) == q.EINVAL and _rows(none, _batch(), ldx=1000) == q.EINVAL
    assert _rows(none, _batch(), H=5) == q.EINVAL
    assert _rows(none, _batch(n_tok=0, kv_len=None, table=None)) == q.OK


def test_values_need_room():
    L = q.lib()
    for k, v in ((None, P), (P, None), (C.c_void_p(4104), P)):
        assert L.qms_cuda_paged_values(C.byref(_pages()), k, v, None) == q.EINVAL
    assert L.qms_cuda_paged_values(None, P, P, None) == q.EINVAL
