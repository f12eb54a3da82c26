"""Refusals of the paged step operators: argument checks that need no GPU."""

from __future__ import annotations

import ctypes as C

import pytest
import torch

import deltakv_b200 as dkv
from deltakv_b200 import _lib as L

I32, I64, BF, F16, F32 = torch.int32, torch.int64, torch.bfloat16, torch.float16, torch.float32
P = 1 << 20  # a stand-in address, never dereferenced on these paths


def _plan(**change):
    a = dict(lengths=torch.tensor([3, 4], dtype=I32), block_tables=torch.zeros(2, 4, dtype=I32), block_size=4, rows=2,
             max_seq_len=8)
    a.update(change)
    return dkv.plan_paged_step(a.pop("lengths"), a.pop("block_tables"), a.pop("block_size"), **a)


@pytest.mark.parametrize("change,error,text", [
    (dict(), ValueError, "CUDA"),
    (dict(lengths=torch.tensor([3, 4])), TypeError, "lengths must be int32"),
    (dict(lengths=torch.zeros(4, dtype=I32)[::2]), ValueError, "contiguous"),
    (dict(new_lengths=torch.ones(3, dtype=I32)), ValueError, "new_lengths"),
    (dict(table_lens=torch.ones(2, dtype=I64)), TypeError, "table_lens"),
    (dict(free_blocks=torch.zeros(2, 2, dtype=I32)), ValueError, "free_blocks"),
    (dict(block_tables=torch.zeros(2, 4, dtype=I64)), TypeError, "int32"),
    (dict(block_tables=torch.zeros(3, 4, dtype=I32)), ValueError, "n_seqs, max_blocks"),
    (dict(block_tables=torch.zeros(4, 2, dtype=I32).T), ValueError, "row-major"),
    (dict(block_tables=torch.zeros(1, 4, dtype=I32).expand(2, 4)), ValueError, "overlap"),
    (dict(block_size=0), ValueError, "positive"),
    (dict(rows=-1), ValueError, "negative"),
    (dict(rows=1 << 31), ValueError, "below"),
    (dict(max_seq_len=1 << 31), ValueError, "below"),
])
def test_plan_refuses(change, error, text):
    with pytest.raises(error, match=text):
        _plan(**change)


@pytest.mark.parametrize("name", ["lengths", "new_lengths", "table_lens", "free_blocks"])
def test_plan_refuses_a_table_over_its_inputs(name):
    """The table is written while other CTAs read them."""
    whole = torch.zeros(10, dtype=I32)
    with pytest.raises(ValueError, match=f"block_tables and {name} share memory"):
        _plan(block_tables=whole[:8].view(2, 4), **{name: whole[7:9]})
    with pytest.raises(ValueError, match="CUDA"):  # beside it: on to the next check
        _plan(block_tables=whole[:8].view(2, 4), **{name: whole[8:10]})


def _append(**change):
    a = dict(k=torch.zeros(3, 2, 8, dtype=BF), v=torch.zeros(3, 2, 8, dtype=BF),
             k_pages=torch.zeros(4, 4, 2, 8, dtype=BF), v_pages=torch.zeros(4, 4, 2, 8, dtype=BF),
             slots=torch.arange(3))
    a.update(change)
    return dkv.append_into_paged(a.pop("k"), a.pop("v"), a.pop("k_pages"), a.pop("v_pages"), a.pop("slots"), **a)


_ACROSS = torch.zeros(128, dtype=BF)
_ROPE = dict(rope=(torch.zeros(9, 4), torch.zeros(9, 4)), positions=torch.zeros(3, dtype=I32))


@pytest.mark.parametrize("change,error,text", [
    (dict(), ValueError, "CUDA"),
    (dict(k_pages=torch.zeros(2, 4, 4, 2, 8, dtype=BF)), ValueError, "unsupported paged KV layout"),
    (dict(v_pages=torch.zeros(4, 4, 2, 16, dtype=BF)), ValueError, "must share"),
    (dict(v_pages=torch.zeros(4, 4, 2, 8, dtype=F16)), ValueError, "must share"),
    (dict(slots=torch.arange(3, dtype=I32)), TypeError, "int64"),
    (dict(slots=torch.arange(4)), ValueError, r"k \(3, 2, 8\)"),
    (dict(k=torch.zeros(3, 1, 8, dtype=BF)), ValueError, "k "),
    (dict(v=torch.zeros(3, 2, 4, dtype=BF)), ValueError, "v "),
    (dict(v=torch.zeros(3, 2, 8)), TypeError, "share a dtype"),
    (dict(k=torch.zeros(3, 2, 8, dtype=F16), v=torch.zeros(3, 2, 8, dtype=F16)), TypeError, "pages"),
    (dict(k=torch.zeros(3, 2, 16, dtype=BF)[..., ::2]), ValueError, "contiguous head_dim"),
    (dict(rope=_ROPE["rope"]), ValueError, "positions"),
    (dict(rope=_ROPE["rope"], positions=torch.zeros(3)), TypeError, "positions"),
    (dict(q=torch.zeros(3, 4, 8, dtype=BF)), ValueError, "rope"),
    (dict(q=torch.zeros(2, 4, 8, dtype=BF), **_ROPE), ValueError, "q "),
    (dict(q=torch.zeros(3, 4, 8), **_ROPE), TypeError, "share a dtype"),
    (dict(q=torch.zeros(3, 4, 8, dtype=BF), q_out=torch.zeros(3, 4, 8), **_ROPE), TypeError, "q_out"),
    (dict(q_out=torch.zeros(3, 4, 8, dtype=BF)), ValueError, "q_out without q"),
    (dict(q=torch.zeros(3, 4, 8, dtype=BF), q_out=torch.zeros(1, 4, 8, dtype=BF).expand(3, 4, 8), **_ROPE), ValueError,
     "share memory"),
    (dict(q=_ACROSS[:96].view(3, 4, 8), q_out=_ACROSS[32:].view(3, 4, 8), **_ROPE), ValueError, "overlaps q"),
    (dict(v_pages=torch.zeros(1, 4, 2, 8, dtype=BF).expand(4, 4, 2, 8)), ValueError, "v_pages has elements"),
    (dict(k=None), TypeError, "k must be a tensor"),
])
def test_append_refuses(change, error, text):
    with pytest.raises(error, match=text):
        _append(**change)


@pytest.mark.parametrize("change,text", [
    (lambda p, x: dict(k_pages=p, v_pages=p), "k_pages and v_pages share memory"),
    (lambda p, x: dict(k_pages=p[:4], v_pages=p[2:6]), "k_pages and v_pages share memory"),
    (lambda p, x: dict(q=torch.zeros(3, 2, 8, dtype=BF), k=x[:3], q_out=x[:3], **_ROPE), "q_out and k share memory"),
    (lambda p, x: dict(q=torch.zeros(3, 2, 8, dtype=BF), v=x[:3], q_out=x[1:4], **_ROPE), "q_out and v share memory"),
    (lambda p, x: dict(k_pages=p[:4], v_pages=p[4:]), "CUDA"),  # side by side: on to the next check
])
def test_append_refuses_shared_memory(change, text):
    pages, rows = torch.zeros(8, 4, 2, 8, dtype=BF), torch.zeros(4, 2, 8, dtype=BF)
    with pytest.raises(ValueError, match=text):
        _append(**change(pages, rows))


def _attend(**change):
    a = dict(q=torch.zeros(2, 4, 8, dtype=BF), k_pages=torch.zeros(4, 4, 2, 8, dtype=BF),
             v_pages=torch.zeros(4, 4, 2, 8, dtype=BF))
    seqs = dkv.SeqBatchTensors(cu_seqlens=torch.tensor([0, 3, 5], dtype=I32),
                               block_tables=change.pop("tables", torch.zeros(2, 1, dtype=I32)), max_seq_len=3)
    a.update(change)
    return dkv.paged_decode_attention(a.pop("q"), a.pop("k_pages"), a.pop("v_pages"), seqs, **a)


@pytest.mark.parametrize("change,error,text", [
    (dict(), ValueError, "CUDA"),
    (dict(q=torch.zeros(3, 4, 8, dtype=BF)), ValueError, "q "),
    (dict(q=torch.zeros(2, 4, 16, dtype=BF)), ValueError, "q "),
    (dict(q=torch.zeros(2, 4, 8)), TypeError, "the pages are"),
    (dict(q=torch.zeros(2, 3, 8, dtype=BF)), ValueError, "evenly"),
    (dict(q=torch.zeros(2, 0, 8, dtype=BF)), ValueError, "evenly"),
    (dict(tables=torch.zeros(1, 1, dtype=I32)), ValueError, "block_tables has 1 rows"),
    (dict(out=torch.zeros(2, 4, 8)), TypeError, "out"),
    (dict(out=torch.zeros(2, 2, 8, dtype=BF)), ValueError, "out"),
    (dict(out=torch.zeros(2, 1, 8, dtype=BF).expand(2, 4, 8)), ValueError, "share memory"),
    (dict(q=_ACROSS[:64].view(2, 4, 8), out=_ACROSS[32:96].view(2, 4, 8)), ValueError, "overlaps q"),
    (dict(q=[1.0]), TypeError, "q must be a tensor"),
    (dict(scale="half"), TypeError, "real number"),
    (dict(q=torch.zeros(2, 4, 264, dtype=BF), k_pages=torch.zeros(4, 4, 2, 264, dtype=BF),
          v_pages=torch.zeros(4, 4, 2, 264, dtype=BF)), ValueError, "256"),
])
def test_attention_refuses(change, error, text):
    with pytest.raises(error, match=text):
        _attend(**change)


def test_append_refuses_rope_tables_without_positions():
    """No address stands for them: the C entry would take them for no rotation at all."""
    for tables in ((torch.zeros(0, 4), torch.zeros(0, 4)), dkv.RotaryEmbedding(8, 0)):
        with pytest.raises(ValueError, match="without positions"):
            _append(rope=tables, positions=_ROPE["positions"])


@pytest.mark.parametrize("tables", [torch.zeros(2, 9, dtype=I32)[:, 3:], torch.zeros(1, 4, dtype=I32).expand(2, 4)])
def test_attention_refuses_tables_put_into_a_batch_without_lengths(tables):
    """SeqBatchTensors copies such tables when it is made; one put into it later would be read past its rows."""
    seqs = dkv.SeqBatchTensors(cu_seqlens=torch.tensor([0, 3, 5], dtype=I32), block_tables=tables, max_seq_len=3)
    x = torch.zeros(2, 4, 8, dtype=BF), torch.zeros(4, 4, 2, 8, dtype=BF), torch.zeros(4, 4, 2, 8, dtype=BF)
    with pytest.raises(ValueError, match="CUDA"):  # as it was made: on to the next check
        dkv.paged_decode_attention(*x, seqs)
    seqs.block_tables = tables
    with pytest.raises(ValueError, match="follow one another"):
        dkv.paged_decode_attention(*x, seqs)
    seqs.table_lens = torch.ones(2, dtype=I32)
    with pytest.raises(ValueError, match="CUDA"):
        dkv.paged_decode_attention(*x, seqs)


def test_attention_passes_on_a_truth_that_raises():
    with pytest.raises(RuntimeError, match="ambiguous"):
        _attend(return_lse=torch.zeros(2))  # used to go on, with the error pending


def _cache(**change):
    a = dict(base=P, dtype=L.DKV_BF16, block_size=16, n_heads=2, head_dim=64, num_blocks=4, stride_block=2048,
             stride_slot=128, stride_head=64)
    a.update(change)
    return L.PagedCache(**a)


def test_struct_sizes_match_the_header():
    # under the x86-64 SysV layout of include/dkv_b200.h
    assert (C.sizeof(L.StepPlanArgs), C.sizeof(L.AppendArgs), C.sizeof(L.PagedDecodeArgs)) == (128, 272, 248)


def test_c_entries_check_before_touching_the_device():
    lib = L.lib()
    assert lib.dkv_plan_paged_step(None, None) == L.DKV_ERR_INVALID_ARGUMENT
    assert lib.dkv_append_paged(None, None) == L.DKV_ERR_INVALID_ARGUMENT
    assert lib.dkv_paged_decode_attention(None, None) == L.DKV_ERR_INVALID_ARGUMENT
    assert lib.dkv_paged_decode_workspace_bytes(None, None) == L.DKV_ERR_INVALID_ARGUMENT

    def plan(**c):
        a = dict(lengths=P, block_tables=P, table_stride=4, table_width=4, n_seqs=2, block_size=16, n_rows=2,
                 cu_seqlens=P, cu_new=P, table_lens_out=P + 64, blocks_used=P, positions=P, slots=P)
        a.update(c)
        return lib.dkv_plan_paged_step(C.byref(L.StepPlanArgs(**a)), None)

    assert plan(n_seqs=-1) == plan(block_size=0) == plan(n_rows=-1) == plan(lengths=None) == L.DKV_ERR_INVALID_ARGUMENT
    assert plan(slots=None) == plan(block_tables=None) == plan(cu_new=None) == L.DKV_ERR_INVALID_ARGUMENT
    assert plan(n_free=3) == L.DKV_ERR_INVALID_ARGUMENT                       # a count without a list
    assert plan(table_lens=P + 64) == L.DKV_ERR_INVALID_ARGUMENT              # output over input
    assert plan(n_seqs=16385) == L.DKV_ERR_UNSUPPORTED

    def append(**c):
        a = dict(k=P, v=P, in_dtype=L.DKV_BF16, n_rows=3, slots=P, k_pages=_cache(), v_pages=_cache())
        a.update(c)
        return lib.dkv_append_paged(C.byref(L.AppendArgs(**a)), None)

    assert append(k=None) == append(slots=None) == append(n_rows=-1) == L.DKV_ERR_INVALID_ARGUMENT
    assert append(q=P, n_q_heads=4) == append(rope_cos=P) == L.DKV_ERR_INVALID_ARGUMENT
    assert append(rope_cos=P, rope_sin=P) == L.DKV_ERR_INVALID_ARGUMENT       # no positions
    assert append(in_dtype=L.DKV_F16) == append(in_dtype=L.DKV_E4M3) == L.DKV_ERR_UNSUPPORTED
    assert append(v_pages=_cache(head_dim=32)) == append(k_pages=_cache(block_size=0)) == L.DKV_ERR_LAYOUT
    assert append(n_rows=0) == L.DKV_OK

    def attend(**c):
        seqs = L.SeqBatch(cu_seqlens=P, block_tables=P, table_stride=4, n_seqs=c.pop("n_seqs", 2), max_seq_len=9)
        a = dict(q=P, n_q_heads=4, scale=1.0, seqs=seqs, k_pages=_cache(), v_pages=_cache(), out=P)
        a.update(c)
        return lib.dkv_paged_decode_attention(C.byref(L.PagedDecodeArgs(**a)), None)

    assert attend(n_q_heads=3) == attend(n_q_heads=0) == attend(n_seqs=65536) == L.DKV_ERR_UNSUPPORTED
    big = _cache(head_dim=264)
    assert attend(k_pages=big, v_pages=big) == L.DKV_ERR_UNSUPPORTED
    assert attend(v_pages=_cache(dtype=L.DKV_F16)) == attend(v_pages=_cache(n_heads=4)) == L.DKV_ERR_LAYOUT
    assert attend(q=None) == attend(out=None) == attend(n_seqs=-1) == L.DKV_ERR_INVALID_ARGUMENT
    assert attend(n_seqs=0) == L.DKV_OK
    assert lib.dkv_status_string(L.DKV_ERR_NO_BLOCKS).decode() == "free block list exhausted"
