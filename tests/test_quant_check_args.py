"""The refusals of blocks that one call would write in two places, as far as the CPU tells."""

from __future__ import annotations

import ctypes as C

import pytest
import torch

import deltakv_b200 as dkv
from deltakv_b200 import _lib as L
from tests.test_quant_args import P, _cache, _pages, _scales


def test_a_table_that_names_a_block_twice_is_refused():
    with pytest.raises(ValueError, match="twice"):
        dkv.scatter_into_paged(torch.zeros(9, 2, 8), _pages(), [1, 2, 1], 4, page_scales=_scales())
    with pytest.raises(ValueError, match="twice"):
        dkv.scatter_into_paged(torch.zeros(5, 2, 8), _pages(), [3, -1], 4, page_scales=_scales())
    with pytest.raises(ValueError, match="CUDA"):
        dkv.scatter_into_paged(torch.zeros(5, 2, 8), _pages(), [3, 1, 1], 4, page_scales=_scales())


def test_the_checks_entries_look_before_touching_the_device():
    lib = L.lib()

    def rows(**c):
        a = dict(n_rows=3, slots=P, k_pages=_cache(), v_pages=_cache())
        a.update(c)
        return lib.dkv_append_paged_quant_check(C.byref(L.AppendArgs(**a)), None)

    assert lib.dkv_append_paged_quant_check(None, None) == rows(slots=None) == rows(n_rows=-1) == L.DKV_ERR_INVALID_ARGUMENT
    assert rows(k_pages=_cache(dtype=L.DKV_F16)) == L.DKV_ERR_UNSUPPORTED
    assert rows(k_pages=_cache(block_size=0)) == rows(v_pages=_cache(num_blocks=-1)) == L.DKV_ERR_LAYOUT
    assert rows(n_rows=0) == L.DKV_OK

    def blocks(n=3, cache=None, **c):
        a = dict(cu_seqlens=P, block_tables=P, table_stride=4, n_seqs=2, max_seq_len=9)
        a.update(c)
        return lib.dkv_scatter_paged_quant_check(n, C.byref(cache or _cache()), C.byref(L.SeqBatch(**a)), None, None)

    assert blocks(-1) == blocks(n_seqs=-1) == blocks(cu_seqlens=None) == L.DKV_ERR_INVALID_ARGUMENT
    assert blocks(n_seqs=65536) == blocks(cache=_cache(dtype=L.DKV_F16)) == L.DKV_ERR_UNSUPPORTED
    assert blocks(cache=_cache(block_size=0)) == L.DKV_ERR_LAYOUT
    assert blocks(0) == blocks(n_seqs=0) == L.DKV_OK
    assert "two places" in lib.dkv_status_string(L.DKV_ERR_BLOCK_TWICE).decode()
