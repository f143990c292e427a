"""qms_cuda_logprobs refuses bad arguments on the host, before any device call. CPU only."""
from __future__ import annotations

import ctypes as C

import pytest

import large_model_b200 as q

P = C.c_void_p(4096)
OK = dict(l=P, ldl=8, rows=2, V=8, temp=1.0, ids=P, n=1, lp=P, ent=P, top=2, ti=P, tl=P)


def _call(**kw):
    a = {**OK, **kw}
    return q.lib().qms_cuda_logprobs(a["l"], a["ldl"], a["rows"], a["V"], a["temp"], a["ids"], a["n"], a["lp"], a["ent"], a["top"], a["ti"],
                                     a["tl"], None, None)


@pytest.mark.parametrize("kw", [
    dict(l=None), dict(l=C.c_void_p(4098)), dict(ldl=7), dict(rows=-1), dict(V=0), dict(V=(1 << 22) + 1, ldl=1 << 23), dict(temp=0.0),
    dict(temp=-1.0), dict(temp=float("nan")), dict(temp=float("inf")), dict(ids=None), dict(lp=None), dict(n=-1), dict(ti=None), dict(tl=None),
    dict(top=-1), dict(ent=C.c_void_p(4097))])
def test_bad_arguments(kw):
    assert _call(**kw) == q.EINVAL and q.lib().qms_cuda_last_error()


def test_too_many_alternatives():
    assert _call(top=33) == q.EUNSUPPORTED


def test_nothing_to_do_needs_no_device():
    assert _call(rows=0) == q.OK
    assert _call(rows=0, n=0, ids=None, lp=None, top=0, ti=None, tl=None, ent=None) == q.OK
