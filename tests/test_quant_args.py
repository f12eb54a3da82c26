"""8-bit pages and rotary forms: refusals and table arithmetic that need no GPU."""

from __future__ import annotations

import ctypes as C
import math

import pytest
import torch

import deltakv_b200 as dkv
from deltakv_b200 import _lib as L
from deltakv_b200.rope import RotaryEmbedding, half_tables, scaled_frequencies

I32, BF, F16, F32 = torch.int32, torch.bfloat16, torch.float16, torch.float32
E4M3, I8 = torch.float8_e4m3fn, torch.int8
P = 1 << 20  # a stand-in address, never dereferenced on these paths


def _pages(dtype=E4M3, blocks=4, block=4, heads=2, hd=8):
    return torch.zeros(blocks, block, heads, hd, dtype=torch.uint8).view(dtype)


def _scales(blocks=4, heads=2):
    return torch.ones(blocks, heads)


def _append(**change):
    a = dict(k=torch.zeros(3, 2, 8, dtype=BF), v=torch.zeros(3, 2, 8, dtype=BF), k_pages=_pages(), v_pages=_pages(),
             slots=torch.arange(3), kv_scales=(_scales(), _scales()))
    a.update(change)
    return dkv.append_into_paged(a.pop("k"), a.pop("v"), a.pop("k_pages"), a.pop("v_pages"), a.pop("slots"), **a)


_ONE = _scales()
_POS = torch.zeros(3, dtype=I32)
_BF = torch.zeros(4, 4, 2, 8, dtype=BF), torch.zeros(4, 4, 2, 8, dtype=BF)


@pytest.mark.parametrize("change,error,text", [
    (dict(), ValueError, "CUDA"),
    (dict(k_pages=_pages(I8), v_pages=_pages(I8)), ValueError, "CUDA"),
    (dict(k=torch.zeros(3, 2, 8), v=torch.zeros(3, 2, 8)), ValueError, "CUDA"),
    (dict(kv_scales=None), TypeError, "need kv_scales"),
    (dict(k_pages=_BF[0], v_pages=_BF[1]), TypeError, "8-bit pages"),
    (dict(k_pages=_pages(I8)), ValueError, "must share"),
    (dict(kv_scales=_scales()), TypeError, "tuple"),
    (dict(kv_scales=(_scales(),)), TypeError, "tuple"),
    (dict(kv_scales=(_scales(), None)), TypeError, "v_scales must be a tensor"),
    (dict(kv_scales=(_scales(5), _scales())), ValueError, r"k_scales \(5, 2\)"),
    (dict(kv_scales=(_scales(), _scales().T)), ValueError, r"v_scales"),
    (dict(kv_scales=(_scales().half(), _scales())), TypeError, "k_scales must be float32"),
    (dict(kv_scales=(torch.ones(1, 2).expand(4, 2), _scales())), ValueError, "k_scales has elements that share memory"),
    (dict(kv_scales=(_ONE, _ONE)), ValueError, "k_scales and v_scales share memory"),
    (dict(v_pages=torch.zeros(1, 4, 2, 8, dtype=torch.uint8).view(E4M3).expand(4, 4, 2, 8)), ValueError, "v_pages has elements"),
    (dict(k_pages=_pages(block=1025), v_pages=_pages(block=1025)), ValueError, "1024"),
    (dict(k=torch.zeros(3, 2, 8, dtype=torch.float64), v=torch.zeros(3, 2, 8, dtype=torch.float64)), TypeError, "float64|Double"),
    (dict(rotary_dim=4), ValueError, "pass rope"),
    (dict(interleaved=True), ValueError, "pass rope"),
    (dict(rope=(torch.zeros(9, 2),) * 2, positions=_POS, rotary_dim=3), ValueError, "rotary_dim 3"),
    (dict(rope=(torch.zeros(9, 2),) * 2, positions=_POS, rotary_dim=0), ValueError, "rotary_dim 0"),
    (dict(rope=(torch.zeros(9, 2),) * 2, positions=_POS, rotary_dim=10), ValueError, "rotary_dim 10"),
    (dict(rope=RotaryEmbedding(8, 9, rotary_dim=4), positions=_POS, rotary_dim=2), ValueError, "may not say otherwise"),
    (dict(rope=RotaryEmbedding(8, 9, interleaved=True), positions=_POS, interleaved=False), ValueError, "may not say otherwise"),
    (dict(rope=RotaryEmbedding(16, 9, rotary_dim=4), positions=_POS), ValueError, "heads of 16"),
])
def test_append_refuses(change, error, text):
    with pytest.raises(error, match=text):
        _append(**change)


def _attend(**change):
    a = dict(q=torch.zeros(2, 4, 8, dtype=BF), k_pages=_pages(), v_pages=_pages(), kv_scales=(_scales(), _scales()))
    seqs = dkv.SeqBatchTensors(cu_seqlens=torch.tensor([0, 3, 5], dtype=I32), block_tables=torch.zeros(2, 1, dtype=I32),
                               max_seq_len=3)
    a.update(change)
    return dkv.paged_decode_attention(a.pop("q"), a.pop("k_pages"), a.pop("v_pages"), seqs, **a)


@pytest.mark.parametrize("change,error,text", [
    (dict(), ValueError, "CUDA"),
    (dict(q=torch.zeros(2, 4, 8)), ValueError, "CUDA"),
    (dict(kv_scales=None), TypeError, "need kv_scales"),
    (dict(k_pages=_BF[0], v_pages=_BF[1]), TypeError, "8-bit pages"),
    (dict(v_pages=_pages(I8)), ValueError, "must share"),
    (dict(kv_scales=(_scales(), _scales(3))), ValueError, r"v_scales \(3, 2\)"),
    (dict(q=torch.zeros(2, 4, 8, dtype=torch.uint8).view(E4M3)), TypeError, "not supported"),
    (dict(q=torch.zeros(2, 4, 264, dtype=BF), k_pages=_pages(hd=264), v_pages=_pages(hd=264)), ValueError, "256"),
])
def test_attention_refuses(change, error, text):
    with pytest.raises(error, match=text):
        _attend(**change)


def _seqs(**change):
    a = dict(cu_seqlens=torch.tensor([0, 3, 5], dtype=I32), block_tables=torch.zeros(2, 1, dtype=I32), max_seq_len=3)
    a.update(change)
    return dkv.SeqBatchTensors(**a)


@pytest.mark.parametrize("change,error,text", [
    (dict(), ValueError, "CUDA"),
    (dict(pages=_BF[0]), TypeError, "8-bit pages"),
    (dict(pages=_pages()[0]), ValueError, "unsupported paged KV layout"),
    (dict(pages=_pages(hd=16)[..., ::2]), ValueError, "contiguous"),
    (dict(pages=_pages(block=2048)), ValueError, "1024"),
    (dict(scales=_scales(heads=3)), ValueError, "page_scales"),
    (dict(scales=_scales().double()), TypeError, "page_scales must be float32"),
    (dict(seqs=_seqs(block_tables=torch.zeros(1, 1, dtype=I32))), ValueError, "block_tables has 1 rows"),
    (dict(seqs=_seqs(max_seq_len=-1)), ValueError, "max_seq_len"),
])
@pytest.mark.parametrize("op", ["gather", "scatter"])
def test_gather_and_scatter_refuse(op, change, error, text):
    a = dict(pages=_pages(), scales=_scales(), seqs=_seqs())
    a.update(change)
    with pytest.raises(error, match=text):
        if op == "gather":
            dkv.gather_from_paged_batched(a["pages"], a["seqs"], 5, page_scales=a["scales"])
        else:
            dkv.scatter_into_paged_batched(torch.zeros(5, 2, 8), a["pages"], a["seqs"], page_scales=a["scales"])


def test_gather_refuses_its_own():
    ok = _pages(), _seqs()
    for error, text, change in [(ValueError, "rows", dict(rows=-1)), (ValueError, r"out \(4, 2, 8\)", dict(out=torch.zeros(4, 2, 8))),
                                (TypeError, "not supported", dict(dtype=I8)), (TypeError, "out has its own", dict(
                                    out=torch.zeros(5, 2, 8), dtype=BF)),
                                (ValueError, "share memory", dict(out=torch.zeros(1, 2, 8).expand(5, 2, 8)))]:
        a = dict(rows=5)
        a.update(change)
        with pytest.raises(error, match=text):
            dkv.gather_from_paged_batched(*ok, a.pop("rows"), page_scales=_scales(), **a)


def test_scatter_refuses_its_own():
    for error, text, change in [(ValueError, r"delta \(5, 3, 8\)", dict(delta=torch.zeros(5, 3, 8))),
                                (ValueError, "delta", dict(delta=torch.zeros(5, 16))),
                                (TypeError, "not supported", dict(delta=torch.zeros(5, 2, 8, dtype=I8))),
                                (ValueError, "share memory", dict(scales=torch.ones(1, 2).expand(4, 2)))]:
        a = dict(delta=torch.zeros(5, 2, 8), scales=_scales())
        a.update(change)
        with pytest.raises(error, match=text):
            dkv.scatter_into_paged_batched(a["delta"], _pages(), _seqs(), page_scales=a["scales"])


def test_single_sequence_forms_refuse():
    with pytest.raises(ValueError, match="a block has one scale"):
        dkv.scatter_into_paged(torch.zeros(3, 2, 8), _pages(), [0, 1], 2, page_scales=_scales())
    with pytest.raises(ValueError, match="a block has one scale"):
        dkv.gather_from_paged(_pages(), [0, 1], 3, 2, page_scales=_scales())
    with pytest.raises(TypeError, match="8-bit pages"):
        dkv.gather_from_paged(_BF[0], [0], 3, 4, dtype=F32)
    with pytest.raises(ValueError, match="shorter than prefix"):
        dkv.scatter_into_paged(torch.zeros(5, 2, 8), _pages(), [0], 4, page_scales=_scales())


# ---------------------------------------------------------------------------------------
# the C entries
# ---------------------------------------------------------------------------------------
def _cache(**change):
    a = dict(base=P, dtype=L.DKV_E4M3, block_size=16, n_heads=2, head_dim=64, num_blocks=4, stride_block=2048,
             stride_slot=128, stride_head=64)
    a.update(change)
    return L.PagedCache(**a)


def test_struct_sizes_match_the_header():
    assert (C.sizeof(L.Rotary), C.sizeof(L.PageScales)) == (8, 24)


def test_c_entries_check_before_touching_the_device():
    lib, ok = L.lib(), L.PageScales(base=P, stride_block=2, stride_head=1)
    none = L.PageScales(base=None, stride_block=2, stride_head=1)

    def append(scales=ok, rotary=None, **c):
        a = dict(k=P, v=P, in_dtype=L.DKV_BF16, n_rows=3, slots=P, k_pages=_cache(), v_pages=_cache())
        a.update(c)
        return lib.dkv_append_paged_quant(C.byref(L.AppendArgs(**a)), rotary, C.byref(scales), C.byref(ok), None)

    assert lib.dkv_append_paged_quant(None, None, C.byref(ok), C.byref(ok), None) == L.DKV_ERR_INVALID_ARGUMENT
    assert append(k=None) == append(slots=None) == append(n_rows=-1) == append(scales=none) == L.DKV_ERR_INVALID_ARGUMENT
    assert append(q=P, n_q_heads=4) == append(rope_cos=P) == append(rope_cos=P, rope_sin=P) == L.DKV_ERR_INVALID_ARGUMENT
    assert append(k_pages=_cache(dtype=L.DKV_BF16)) == append(in_dtype=L.DKV_E4M3) == L.DKV_ERR_UNSUPPORTED
    big = _cache(block_size=1025)
    assert append(k_pages=big, v_pages=big) == L.DKV_ERR_UNSUPPORTED
    assert append(v_pages=_cache(dtype=L.DKV_I8)) == append(v_pages=_cache(n_heads=4)) == L.DKV_ERR_LAYOUT
    turns = dict(rope_cos=P, rope_sin=P, positions=P)
    for dim in (0, 3, 66, -2):
        assert append(rotary=C.byref(L.Rotary(dim=dim)), **turns) == L.DKV_ERR_UNSUPPORTED
        args = L.AppendArgs(k=P, v=P, in_dtype=L.DKV_BF16, n_rows=3, slots=P, k_pages=_cache(dtype=L.DKV_BF16),
                            v_pages=_cache(dtype=L.DKV_BF16), **turns)
        assert lib.dkv_append_paged_rotary(C.byref(args), C.byref(L.Rotary(dim=dim)), None) == L.DKV_ERR_UNSUPPORTED
    assert append(n_rows=0) == L.DKV_OK

    def batch(**c):
        a = dict(cu_seqlens=P, block_tables=P, table_stride=4, n_seqs=2, max_seq_len=9)
        a.update(c)
        return C.byref(L.SeqBatch(**a))

    def scatter(rows=3, delta=P, dtype=L.DKV_F32, cache=None, scales=ok, seqs=None):
        return lib.dkv_scatter_paged_quant(delta, dtype, rows, 128, 64, C.byref(cache or _cache()), C.byref(scales),
                                           seqs or batch(), None, None)

    def gather(rows=3, out=P, dtype=L.DKV_F32, cache=None, scales=ok, seqs=None):
        return lib.dkv_gather_paged_quant(C.byref(cache or _cache()), C.byref(scales), seqs or batch(), out, dtype, rows, 128, 64,
                                          1, None, None)

    for f in (scatter, gather):
        assert f(-1) == f(3, None) == f(scales=none) == f(seqs=batch(n_seqs=-1)) == L.DKV_ERR_INVALID_ARGUMENT
        assert f(seqs=batch(cu_seqlens=None)) == L.DKV_ERR_INVALID_ARGUMENT
        assert f(dtype=L.DKV_E4M3) == f(cache=_cache(dtype=L.DKV_F16)) == f(seqs=batch(n_seqs=65536)) == L.DKV_ERR_UNSUPPORTED
        assert f(cache=_cache(block_size=0)) == f(cache=_cache(num_blocks=-1)) == L.DKV_ERR_LAYOUT
        assert f(0) == L.DKV_OK

    def attend(q_dtype=L.DKV_BF16, n_seqs=2, scales=ok, **c):
        seqs = L.SeqBatch(cu_seqlens=P, block_tables=P, table_stride=4, n_seqs=n_seqs, max_seq_len=9)
        a = dict(q=P, n_q_heads=4, scale=1.0, seqs=seqs, k_pages=_cache(), v_pages=_cache(), out=P)
        a.update(c)
        return lib.dkv_paged_decode_attention_quant(C.byref(L.PagedDecodeArgs(**a)), q_dtype, C.byref(scales), C.byref(ok), None)

    assert attend(n_q_heads=3) == attend(q_dtype=L.DKV_I8) == attend(n_seqs=65536) == L.DKV_ERR_UNSUPPORTED
    f16 = _cache(dtype=L.DKV_F16)
    assert attend(k_pages=f16, v_pages=f16) == L.DKV_ERR_UNSUPPORTED
    assert attend(v_pages=_cache(dtype=L.DKV_I8)) == L.DKV_ERR_LAYOUT
    assert attend(q=None) == attend(out=None) == attend(n_seqs=-1) == attend(scales=none) == L.DKV_ERR_INVALID_ARGUMENT
    assert attend(n_seqs=0) == L.DKV_OK
    size = C.c_int64()
    assert lib.dkv_paged_decode_quant_workspace_bytes(None, L.DKV_BF16, C.byref(size)) == L.DKV_ERR_INVALID_ARGUMENT


# ---------------------------------------------------------------------------------------
# rotary forms
# ---------------------------------------------------------------------------------------
def test_default_tables_are_unchanged():
    """The reference's operations, in its order (src/deltakv/rope.py:35-45)."""
    inv = 1.0 / (10000.0 ** (torch.arange(0, 64, 2, dtype=torch.float32) / 64))
    emb = torch.cat((torch.outer(torch.arange(50, dtype=torch.float32), inv),) * 2, dim=-1)
    rope = RotaryEmbedding(64, 50)
    assert torch.equal(rope.cos_cached, emb.cos()) and torch.equal(rope.sin_cached, emb.sin())


@pytest.mark.parametrize("scaling", [
    {"type": "linear", "factor": 4.0},
    {"type": "ntk", "factor": 8.0},
    {"type": "llama3", "factor": 8.0, "original_max_seq": 8192},
    {"type": "yarn", "factor": 16.0, "original_max_seq": 4096},
    {"type": "yarn", "factor": 2.0, "original_max_seq": 4096, "attention_factor": 1.5, "beta_fast": 16.0},
])
@pytest.mark.parametrize("dim,base", [(64, 10000.0), (128, 500000.0)])
def test_scaled_frequencies(scaling, dim, base):
    """Each pair against the definition, one by one in Python's fp64; the tables at far positions."""
    s, kind = scaling["factor"], scaling["type"]
    want, amplitude = [], 1.0
    for i in range(dim // 2):
        theta = base ** (-2 * i / dim)
        if kind == "linear":
            want.append(theta / s)
        elif kind == "ntk":
            want.append((base * s ** (dim / (dim - 2))) ** (-2 * i / dim))
        elif kind == "llama3":
            wave, length = 2 * math.pi / theta, 8192
            if wave < length / 4:
                want.append(theta)
            elif wave > length / 1:
                want.append(theta / s)
            else:
                a = (length / wave - 1) / (4 - 1)
                want.append(theta * (a + (1 - a) / s))
        else:
            at = lambda turns: dim * math.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
            lo, hi = math.floor(at(scaling.get("beta_fast", 32.0))), math.ceil(at(1.0))
            a = 1 - min(max((i - lo) / (hi - lo), 0.0), 1.0)
            want.append(theta * (a + (1 - a) / s))
            amplitude = scaling.get("attention_factor", 0.1 * math.log(s) + 1)
    got, amp = scaled_frequencies(dim, base, scaling)
    assert got.dtype == torch.float64 and amp == pytest.approx(amplitude, rel=1e-15)
    assert torch.allclose(got, torch.tensor(want, dtype=torch.float64), rtol=1e-12, atol=0)
    rope = RotaryEmbedding(dim, 300000, base, scaling=scaling)
    for pos in (0, 1, 777, 299999):
        for i in (0, 1, dim // 4, dim // 2 - 1):
            # the angle's relative error is a few 2^-53, so up to 3e5 * 2^-51 of the value; then one rounding to fp32
            tol = 2.0 ** -24 * amplitude + pos * 2.0 ** -48
            assert abs(float(rope.cos_cached[pos, i]) - amplitude * math.cos(pos * want[i])) <= tol
            assert abs(float(rope.sin_cached[pos, dim // 2 + i]) - amplitude * math.sin(pos * want[i])) <= tol


@pytest.mark.parametrize("scaling,text", [
    ({"type": "dynamic", "factor": 2.0}, "none of"),
    ({"factor": 2.0}, "none of"),
    ({"type": "linear"}, "needs factor"),
    ({"type": "linear", "factor": 0.0}, "positive"),
    ({"type": "linear", "factor": 2.0, "beta_fast": 1.0}, "does not take beta_fast"),
    ({"type": "llama3", "factor": 2.0}, "original_max_seq"),
    ({"type": "llama3", "factor": 2.0, "original_max_seq": 64, "high_freq_factor": 1.0}, "above low_freq_factor"),
])
def test_scaling_refuses(scaling, text):
    with pytest.raises(ValueError, match=text):
        RotaryEmbedding(64, 9, scaling=scaling)


def test_forms_are_refused_where_whole_heads_turn_in_halves():
    cpu = torch.device("cpu")
    for rope in (RotaryEmbedding(64, 9, rotary_dim=32), RotaryEmbedding(64, 9, interleaved=True)):
        with pytest.raises(ValueError, match="whole heads in halves"):
            half_tables(rope, cpu)
        assert half_tables(rope, cpu, forms=True)[0].shape == (9, rope.rotary_dim // 2)
    scaled = RotaryEmbedding(64, 9, scaling={"type": "linear", "factor": 2.0})
    assert half_tables(scaled, cpu)[0].shape == (9, 32)  # the tables are all that differs
    for bad in (dict(rotary_dim=3), dict(rotary_dim=0), dict(rotary_dim=66)):
        with pytest.raises(ValueError, match="rotary_dim"):
            RotaryEmbedding(64, 9, **bad)


@pytest.mark.parametrize("width", [16, 64])
def test_patch_routes_refuse_tables_of_another_width(width):
    """The kernels read head_dim / 2 angles a position, whatever the table's width."""
    from deltakv_b200 import ops

    tables = torch.zeros(9, width)
    with pytest.raises(ValueError, match="do not cover head_dim"):
        ops._check_rope(tables, tables, 64)
    ops._check_rope(torch.zeros(9, 32), torch.zeros(9, 32), 64)
    ops._check_rope(None, None, 64)
