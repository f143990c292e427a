"""qms_cuda_prompt_attention refuses bad arguments on the host, before any device call. CPU only."""
from __future__ import annotations

import ctypes as C

import pytest

import large_model_b200 as q


def _heads(data=4096, tok=512, head=128):
    return q.HeadsDesc(data, tok, head)


def _call(bt=None, typ=q.T_F16, qh=None, kh=None, vh=None, H=4, Hk=2, D=128, scale=1.0, otyp=q.T_F16, oh=None, **batch):
    d = dict(n_seq=2, n_tok=3, q_start=4096, kv_len=None, table=None, table_stride=0, max_q=2, max_kv=0, prefix_len=0)
    d.update(batch)
    h = lambda x: C.byref(_heads() if x is None else x)
    return q.lib().qms_cuda_prompt_attention(C.byref(q.PagedBatchDesc(**d)), typ, h(qh), h(kh), h(vh), H, Hk, D, scale, otyp, h(oh), None, None)


@pytest.mark.parametrize("kw,rc", [
    (dict(typ=q.T_F32), q.EUNSUPPORTED), (dict(otyp=q.T_BF16), q.EUNSUPPORTED), (dict(D=96), q.EUNSUPPORTED), (dict(H=5), q.EINVAL),
    (dict(H=0), q.EINVAL), (dict(Hk=0), q.EINVAL), (dict(H=258, Hk=2), q.EUNSUPPORTED), (dict(H=2048, Hk=1024), q.EINVAL),
    (dict(scale=0.0), q.EINVAL), (dict(scale=float("nan")), q.EINVAL), (dict(scale=float("inf")), q.EINVAL), (dict(n_seq=-1), q.EINVAL),
    (dict(n_tok=1 << 21), q.EINVAL), (dict(q_start=None), q.EINVAL), (dict(q_start=4097), q.EINVAL), (dict(max_q=-1), q.EINVAL),
    (dict(qh=_heads(data=None)), q.EINVAL), (dict(kh=_heads(data=4104)), q.EINVAL), (dict(vh=_heads(tok=100)), q.EINVAL),
    (dict(qh=_heads(head=64)), q.EINVAL), (dict(oh=_heads(tok=516)), q.EINVAL), (dict(kh=_heads(head=-128)), q.EINVAL)])
def test_bad_arguments(kw, rc):
    assert _call(**kw) == rc and q.lib().qms_cuda_last_error()


def test_nothing_to_do_needs_no_device():
    assert _call(n_tok=0) == q.OK and _call(n_seq=0, q_start=None) == q.OK
