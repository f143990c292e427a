"""The paged operators' Python calls refuse tensors that lie on several devices, before any library call: a kernel would read the
other device's address. Stand-ins for CUDA tensors; CPU only."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

import large_model_b200 as m


class On:
    """What the calls look at of a contiguous CUDA tensor on device `d`."""

    def __init__(self, shape, d=0, dtype=torch.float32):
        self.shape, self.dtype, self.d, self.is_cuda = torch.Size(shape), dtype, d, True
        self.device = torch.device("cuda", d)

    def dim(self):
        return len(self.shape)

    def numel(self):
        return self.shape.numel()

    def stride(self):
        st, n = [], 1
        for x in reversed(self.shape):
            st.insert(0, n)
            n *= x
        return tuple(st)

    def is_contiguous(self):
        return True

    def flatten(self, first):
        return On((*self.shape[:first], self.shape[first:].numel()), self.d, self.dtype)

    def data_ptr(self):
        return 4096

    def get_device(self):
        return self.d


class Library:
    """Every entry records its name and says OK."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        return lambda *a: self.calls.append(name) or 0


@pytest.fixture
def library(monkeypatch):
    L = Library()
    monkeypatch.setattr(m, "lib", lambda: L)
    monkeypatch.setattr(m, "_raw_stream", lambda stream, t: 0)
    monkeypatch.setattr(m, "_on_device", lambda d, call, *a: call(*a))
    return L


def pool(d=0, head_dim=128):
    p = m.KvPages.__new__(m.KvPages)
    p.k = p.v = On((4, 16, 2, head_dim), d)
    p.n_head_kv, p.head_dim, p._dev, p._key = 2, head_dim, d, ("pool", head_dim)
    p.desc = m.PagesDesc(m.T_F32, 4, 16, 2, head_dim, 16 * 2 * head_dim, 2 * head_dim, head_dim, 4096, 4096)
    p._ref = C.byref(p.desc)
    return p


def batch(d=0, n_tok=3):
    b = m.PagedBatch.__new__(m.PagedBatch)
    b.n_tok, b.err, b._err, b._dev, b._ready, b._ws = n_tok, On((1,), d, torch.int32), 4096, d, {0}, {}
    b.desc = m.PagedBatchDesc(2, n_tok, 4096, 4096, 4096, 2, 2, 32, 0)
    b._ref = C.byref(b.desc)
    return b


APPEND = dict(qkv=(3, 8 * 128), q=(3, 512), q_norm=(128,), k_norm=(128,), cos=(32, 64), sin=(32, 64))


def append(other=None):
    t = {k: On(s, int(k == other)) for k, s in APPEND.items()}
    return m.paged_append(pool(int(other == "pages")), batch(int(other == "batch")), t["qkv"], 4, t["q_norm"], t["k_norm"], 1e-6,
                          (t["cos"], t["sin"]), q=t["q"])


@pytest.mark.parametrize("other", [*APPEND, "pages", "batch"])
def test_append_on_two_devices(library, other):
    with pytest.raises(ValueError, match="paged_append: tensors on"):
        append(other)
    assert library.calls == []


def test_append_on_one_device(library):
    append()
    assert library.calls == ["qms_cuda_paged_append"]


I32 = torch.int32
PROBS = dict(logits=(3, 50), out=(3, 50))
VERIFY = dict(p=(6, 50), draft=(2, 2), u=(2, 3), q=(2, 2, 50), n_draft=(2,), row_start=(2,), n_accept=(2,), tokens=(2, 3), err=(1,))


def verify(other=None):
    t = {k: On(s, int(k == other), torch.float32 if k in ("p", "u", "q") else I32) for k, s in VERIFY.items()}
    t["q"].view = lambda *shape: On((4, 50), t["q"].d)
    return m.verify(**t)


@pytest.mark.parametrize("other", PROBS)
def test_probs_on_two_devices(library, other):
    with pytest.raises(ValueError, match="probs: tensors on"):
        m.probs(On(PROBS["logits"], int(other == "logits")), 1.0, out=On(PROBS["out"], int(other == "out")))
    assert library.calls == []


@pytest.mark.parametrize("other", VERIFY)
def test_verify_on_two_devices(library, other):
    with pytest.raises(ValueError, match="verify: tensors on"):
        verify(other)
    assert library.calls == []


def test_probs_and_verify_on_one_device(library, monkeypatch):
    """The call is made with the tensors' device as the current one."""
    devices = []
    monkeypatch.setattr(m, "_on_device", lambda d, call, *a: devices.append(d) or call(*a))
    m.probs(On((3, 50), 1), 1.0, out=On((3, 50), 1))
    verify()
    assert library.calls == ["qms_cuda_probs", "qms_cuda_verify"] and devices == [1, 0]


def test_a_batch_on_two_devices(monkeypatch):
    monkeypatch.setattr(torch, "zeros", lambda shape, dtype, device: On(shape, device.index, dtype))
    monkeypatch.setattr(m.PagedBatch, "_cleared", lambda self: None)
    for other in (None, "q_start", "kv_len", "table"):
        t = {k: On(s, int(k == other), I32) for k, s in dict(q_start=(3,), kv_len=(2,), table=(2, 2)).items()}
        make = lambda: m.PagedBatch(t["q_start"], t["kv_len"], t["table"], 3, 2, 32)
        if other is None:
            assert make()._dev == 0
            continue
        with pytest.raises(ValueError, match="PagedBatch: tensors on"):
            make()
