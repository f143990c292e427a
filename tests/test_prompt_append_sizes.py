"""prompt_append takes the heads' sizes from the pages, and refuses weights, tables and rows of others before any library call: the
kernel would read past the weights' ends, or cut the rows into other heads. Stand-ins for CUDA tensors; CPU only."""
from __future__ import annotations

import pytest
import torch

import large_model_b200 as m
from test_paged_devices import On, batch, library, pool  # noqa: F401 (a fixture among them)


class Wide(On):
    """Rows further apart than they are long."""

    def stride(self):
        return (8 * 128, 1)


def call(page_dim, weight_dim, kind=On, n_head_kv=None, with_pages=True):
    W = 8 * weight_dim
    return m.prompt_append(pool(0, page_dim) if with_pages else None, batch(), kind((3, W)), 4, On((weight_dim,)), On((weight_dim,)), 1e-6,
                           (On((32, weight_dim // 2)), On((32, weight_dim // 2))), rows=kind((3, W), dtype=torch.bfloat16), n_head_kv=n_head_kv)


@pytest.mark.parametrize("page_dim,weight_dim,kind", [(64, 128, On), (128, 64, On), (128, 64, Wide), (64, 128, Wide)])
def test_weights_of_another_head_dim(library, page_dim, weight_dim, kind):
    with pytest.raises(ValueError):
        call(page_dim, weight_dim, kind)
    assert library.calls == []


@pytest.mark.parametrize("page_dim,weight_dim", [(64, 128), (128, 64)])
def test_rows_of_the_pages_and_weights_of_another_head_dim(library, page_dim, weight_dim):
    with pytest.raises(ValueError, match="q_norm"):
        m.prompt_append(pool(0, page_dim), batch(), On((3, 8 * page_dim)), 4, On((weight_dim,)), On((page_dim,)), 1e-6,
                        (On((32, page_dim // 2)), On((32, page_dim // 2))), rows=On((3, 8 * page_dim), dtype=torch.bfloat16))
    assert library.calls == []


def test_n_head_kv_other_than_the_pages(library):
    with pytest.raises(ValueError, match="n_head_kv"):
        call(128, 128, n_head_kv=4)
    assert library.calls == []


def test_what_fits(library):
    call(128, 128)
    call(64, 64, n_head_kv=2)
    call(64, 64, n_head_kv=2, with_pages=False)
    assert library.calls == ["qms_cuda_prompt_append"] * 3
