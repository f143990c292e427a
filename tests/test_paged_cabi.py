"""The paged-cache, probabilities and verification entries refuse bad arguments on the host, before any
device call. CPU only."""
from __future__ import annotations

import ctypes as C

import pytest

import large_model_b200 as q

P = C.c_void_p(4096)
INF = float("inf")


def _pages(**kw):
    d = dict(type=q.T_F16, n_pages=4, page_size=16, n_head_kv=2, head_dim=128, page_stride=4096, pos_stride=256,
             head_stride=128, k=4096, v=4096)
    d.update(kw)
    return q.PagesDesc(**d)


def _batch(**kw):
    d = dict(n_seq=2, n_tok=3, q_start=4096, kv_len=4096, table=4096, table_stride=2, max_q=2, max_kv=32, prefix_len=16)
    d.update(kw)
    return q.PagedBatchDesc(**d)


def _append(pg, bt, x=P, ldx=1024, H=4, n=P, cos=P, n_rope=32, y=P, ldy=512):
    return q.lib().qms_cuda_paged_append(C.byref(pg), C.byref(bt), x, ldx, H, n, n, 1e-6, cos, cos, n_rope, y, ldy, None, None)


def _attend(pg, bt, x=P, ldx=512, H=4, y=P, ldy=512, ws=P, nb=1 << 40):
    return q.lib().qms_cuda_paged_attention(C.byref(pg), C.byref(bt), x, ldx, H, 1.0, y, ldy, ws, nb, None, None)


@pytest.mark.parametrize("kw,rc", [
    (dict(type=q.T_Q8_0), q.EUNSUPPORTED), (dict(head_dim=96), q.EUNSUPPORTED), (dict(n_pages=0), q.EINVAL),
    (dict(page_size=24), q.EINVAL), (dict(page_size=0), q.EINVAL), (dict(n_head_kv=3), q.EINVAL), (dict(n_head_kv=0), q.EINVAL),
    (dict(k=None), q.EINVAL), (dict(v=4104), q.EINVAL), (dict(pos_stride=100), q.EINVAL), (dict(head_stride=-8), q.EINVAL)])
def test_pages_are_checked(kw, rc):
    assert _append(_pages(**kw), _batch()) == rc and q.lib().qms_cuda_last_error()
    assert _attend(_pages(**kw), _batch()) == rc
    assert q.lib().qms_cuda_paged_attention_ws(C.byref(_pages(**kw)), C.byref(_batch()), 4) == rc


@pytest.mark.parametrize("kw", [
    dict(n_seq=-1), dict(n_tok=-1), dict(n_tok=1 << 21), dict(q_start=None), dict(kv_len=None), dict(table=None), dict(max_q=-1),
    dict(max_kv=33), dict(prefix_len=33), dict(prefix_len=-1), dict(table_stride=-1), dict(table=4098)])
def test_batches_are_checked(kw):
    assert _append(_pages(), _batch(**kw)) == q.EINVAL and q.lib().qms_cuda_last_error()
    assert _attend(_pages(), _batch(**kw)) == q.EINVAL


def test_rows_and_workspace_are_checked():
    pg, bt = _pages(), _batch()
    for kw in (dict(x=None), dict(x=C.c_void_p(4100)), dict(ldx=500), dict(ldx=1026), dict(y=None), dict(ldy=510), dict(n=None),
               dict(cos=None), dict(n_rope=0), dict(H=3), dict(H=0)):
        assert _append(pg, bt, **kw) == q.EINVAL, kw
    for kw in (dict(x=None), dict(x=C.c_void_p(4100)), dict(ldx=500), dict(y=None), dict(ldy=513), dict(H=3), dict(H=-4)):
        assert _attend(pg, bt, **kw) == q.EINVAL, kw
    need = q.lib().qms_cuda_paged_attention_ws(C.byref(pg), C.byref(_batch(max_kv=32, n_seq=2)), 4)
    assert need >= 0
    if need:
        assert _attend(pg, bt, ws=None) == q.EINVAL and _attend(pg, bt, nb=need - 1) == q.EINVAL
        assert _attend(pg, bt, ws=C.c_void_p(4096 + 16)) == q.EINVAL
    assert q.lib().qms_cuda_paged_append(None, C.byref(bt), P, 1024, 4, P, P, 0.0, P, P, 1, P, 512, None, None) == q.EINVAL
    assert q.lib().qms_cuda_paged_attention(C.byref(pg), None, P, 512, 4, 1.0, P, 512, P, 1, None, None) == q.EINVAL


def test_nothing_to_do_needs_no_device():
    assert _append(_pages(), _batch(n_tok=0)) == q.OK
    assert _attend(_pages(), _batch(n_tok=0)) == q.OK
    assert _append(_pages(), _batch(n_seq=0, q_start=None, kv_len=None, table=None)) == q.OK


def test_probs_and_verify_check_arguments():
    L = q.lib()
    assert L.qms_cuda_probs(None, 8, 1, 8, 1.0, P, 8, None) == q.EINVAL
    assert L.qms_cuda_probs(P, 7, 1, 8, 1.0, P, 8, None) == q.EINVAL
    assert L.qms_cuda_probs(P, 9, 1, 8, 1.0, P, 8, None) == q.EINVAL          # in place with another stride
    assert L.qms_cuda_probs(P, 8, 1, 0, 1.0, P, 8, None) == q.EINVAL
    assert L.qms_cuda_probs(P, 8, -1, 8, 1.0, P, 8, None) == q.EINVAL
    assert L.qms_cuda_probs(P, 8, 1, 8, float("nan"), P, 8, None) == q.EINVAL
    assert L.qms_cuda_probs(P, 8, 0, 8, 1.0, P, 8, None) == q.OK
    ok = dict(p=P, ldp=8, rows=4, start=None, dq=None, ldq=0, draft=P, nd=None, B=2, N=1, V=8, u=P, n=P, t=P)

    def verify(**kw):
        a = {**ok, **kw}
        return L.qms_cuda_verify(a["p"], a["ldp"], a["rows"], a["start"], a["dq"], a["ldq"], a["draft"], a["nd"], a["B"], a["N"], a["V"],
                                 a["u"], a["n"], a["t"], None, None)
    for kw in (dict(p=None), dict(draft=None), dict(u=None), dict(n=None), dict(t=None), dict(ldp=7), dict(dq=P, ldq=7), dict(B=-1), dict(N=-1),
               dict(N=1025), dict(V=0), dict(V=(1 << 22) + 1), dict(rows=-1)):
        assert verify(**kw) == q.EINVAL, kw
    assert verify(B=0) == q.OK
