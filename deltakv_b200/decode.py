"""One decode step of a paged cache: plan, append, attend.

The patch routes of this package change the K/V of tokens that are already cached; these three
operators are what a serving loop does between two patches, on the same pages, block tables
and :class:`~deltakv_b200.ops.SeqBatchTensors`:

* :func:`plan_paged_step`        block tables, slots and positions from lengths on the GPU
* :func:`append_into_paged`      rotate-half RoPE of the new q and k, K and V into their slots
* :func:`paged_decode_attention` attention of one new token per sequence over its pages

The first two take any number of new tokens a sequence, so they also serve prompt chunks; the
attention of a chunk's rows, several a sequence, is not here.

None of them reads anything back to the host (``check=True`` does, to raise what the kernels
recorded), so a step can be captured into a CUDA graph and replayed with other lengths, up to the
capacities of its capture.  The first call may be inside the capture, but for a rope that is not on
the GPU: its tables are made by a call before (see :func:`deltakv_b200.rope.half_tables`).  They
run on the current stream of the tensors' device, which need not be the current device.  They are
forms for serving: their outputs carry no gradient.  The cache layouts are the ones of
:func:`~deltakv_b200.paged.scatter_into_paged`; for its 5-D forms pass the K and V views
(``ops.page_view(cache, 0)``, ``ops.page_view(cache, 1)``).  The rotation is the reference's
(src/deltakv/rope.py:9-63), the page arithmetic that of src/deltakv/paged.py:39-43.
"""

from __future__ import annotations

import ctypes as C
import importlib
from dataclasses import dataclass

import torch
from torch import Tensor

from deltakv_b200 import _lib as L
from deltakv_b200 import ops
from deltakv_b200.rope import RotaryEmbedding, half_tables

_native_module = None


def _raise_error(status: int, where: str) -> None:
    raise L.DkvError(status, where)


def _status_address(device_index: int) -> int:
    return ops.status_word(torch.device("cuda", device_index)).ptr


def _native():
    """The extension module with these operators' host side (csrc/step_binding.cpp), on the library's entries.

    A decode step calls them once a layer and their kernels take a few microseconds: checked and
    described in Python, a call took 10 us of host time beside the launch, in C++ 2.
    """
    global _native_module
    if _native_module is None:
        try:
            module = importlib.import_module("deltakv_b200._step")
        except ModuleNotFoundError as e:
            raise ImportError("_step.so is not built; run `python -m deltakv_b200.build` "
                              "(the CUDA path has no fallback)") from e
        lib = L.lib()
        entries = (lib.dkv_plan_paged_step, lib.dkv_append_paged_rotary, lib.dkv_paged_decode_workspace_bytes,
                   lib.dkv_paged_decode_attention, lib.dkv_append_paged_quant, lib.dkv_scatter_paged_quant,
                   lib.dkv_gather_paged_quant, lib.dkv_paged_decode_quant_workspace_bytes,
                   lib.dkv_paged_decode_attention_quant, lib.dkv_append_paged_quant_check, lib.dkv_scatter_paged_quant_check)
        module.bind(*(C.cast(f, C.c_void_p).value for f in entries), _raise_error, _status_address)
        _native_module = module
    return _native_module


@dataclass
class PagedStep:
    """What one step needs: all of it on the GPU."""

    seqs: ops.SeqBatchTensors  # cu_seqlens / tables / lengths after the step: what the attention reads
    cu_new: Tensor             # int32 [n_seqs + 1]: rows of sequence b are [cu_new[b], cu_new[b + 1])
    positions: Tensor          # int32 [rows]
    slots: Tensor              # int64 [rows], block * block_size + offset; -1: store nothing
    blocks_used: Tensor        # int32 [1]: entries taken from the front of free_blocks


def plan_paged_step(lengths: Tensor, block_tables: Tensor, block_size: int, *, rows: int, max_seq_len: int,
                    new_lengths: Tensor | None = None, table_lens: Tensor | None = None,
                    free_blocks: Tensor | None = None, check: bool = False) -> PagedStep:
    """Block tables, slots and positions of one step, from lengths that live on the GPU.

    ``lengths`` int32 ``[n_seqs]`` counts each sequence's tokens after the step, the last
    ``new_lengths`` of them new (``None``: all, a prefill).  ``block_tables`` int32
    ``[n_seqs, width]`` holds ``table_lens`` valid blocks a row (``None``: ``width``) and is
    extended in place from the front of ``free_blocks``, sequence by sequence; it shares no memory
    with the other inputs.  ``rows`` is the
    capacity of the row outputs (the sum of the new lengths, or more in a padded batch: rows
    past the last sequence get slot -1 and position 0); ``max_seq_len`` bounds the lengths and
    goes into the returned ``seqs``.

    With ``check=True`` what the kernel recorded (lengths out of range, a full table, no free
    blocks left) is raised after a synchronisation; otherwise the affected tokens only have
    slot -1.  At most 16384 sequences.
    """
    cu, cu_new, lens, used, positions, slots = (_native_module or _native()).plan(
        lengths, block_tables, block_size, rows, max_seq_len, new_lengths, table_lens, free_blocks)
    if check:
        ops.status_word(lengths.device).raise_if_set("plan_paged_step")
    seqs = ops.SeqBatchTensors(cu_seqlens=cu, block_tables=block_tables, max_seq_len=max_seq_len, table_lens=lens)
    return PagedStep(seqs, cu_new, positions, slots, used)


def append_into_paged(k: Tensor, v: Tensor, k_pages: Tensor, v_pages: Tensor, slots: Tensor, *,
                      q: Tensor | None = None, positions: Tensor | None = None, rope=None,
                      q_out: Tensor | None = None, check: bool = False, rotary_dim: int | None = None,
                      interleaved: bool | None = None, kv_scales: tuple[Tensor, Tensor] | None = None) -> Tensor | None:
    """Store this step's ``k`` and ``v [rows, n_kv, head_dim]`` in their ``slots``, rotated.

    ``slots`` (int64) and ``positions`` (int32) are a :class:`PagedStep`'s; a negative slot
    stores nothing.  With ``rope`` (a ``RotaryEmbedding`` or a half-width ``(cos, sin)`` pair)
    K gets the rotate-half RoPE of its position, and so do the rows of ``q [rows, n_q, head_dim]``
    — padding rows too — into ``q_out`` (default: a new tensor; ``q`` itself is allowed), which
    is returned.  The inputs may be strided views (heads of one fused projection); their dtype
    is the pages' or fp32, rounded once on the way into the pages.

    The stored values replace what the slots held (``scatter_into_paged`` adds).  Slots must be
    distinct, and the K pages, the V pages, ``q_out`` and the inputs other than ``q`` apart in memory.
    ``check=True`` raises recorded range errors (a slot beyond the pages, a position
    beyond the tables: those rows store nothing).

    ``rotary_dim`` turns only the first columns of each head (tables of half that width), and
    ``interleaved`` the pairs ``(2i, 2i + 1)`` instead of ``(i, i + rotary_dim / 2)``.  A
    :class:`~deltakv_b200.rope.RotaryEmbedding` made with them brings its own; they are for pairs of tables.

    **8-bit pages** (``torch.float8_e4m3fn`` or ``torch.int8``, at most 1024 slots a block) come with
    ``kv_scales = (k_scales, v_scales)``, fp32 ``[num_blocks, n_kv]``: a slot's value is its code times its block's and
    head's scale.  The operator keeps them: storing a block's slot 0 begins the block with the scale that this call's
    values need (e4m3: the least power of two; int8: the largest magnitude times 1/127 in fp32), and nothing the block held
    is kept; later values that do not fit make the scale grow by powers of two, and what the block holds is rounded to the
    new one (int8: by less than one step in all; e4m3: not at all above its subnormals).  So codes and scales may start as any memory.
    Rows may be fp32, fp16 or bf16, and the rows of one block follow one another, with no row
    of a negative slot between them (as :func:`plan_paged_step` lays them out): ``check=True`` refuses a call in which they do not
    before it stores anything; without it such a call is recorded, and the block holds anything.  A value that is not finite makes
    the block's head read as NaN until the block is begun anew.
    """
    native = _native_module or _native()
    cos = sin = None
    if rope is not None:
        if type(rope) is tuple and native.rope_ready(*rope, k):
            cos, sin = rope
        else:
            cos, sin = half_tables(rope, k.device, forms=True)
            if isinstance(rope, RotaryEmbedding):
                rotary_dim, interleaved = rope.form(k.shape[-1], rotary_dim, interleaved)
    q_out = native.append(k, v, k_pages, v_pages, slots, q, positions, cos, sin, q_out, rotary_dim,
                          interleaved or False, kv_scales, check)
    if check:
        ops.status_word(k.device).raise_if_set("append_into_paged")
    return q_out


def paged_decode_attention(q: Tensor, k_pages: Tensor, v_pages: Tensor, seqs: ops.SeqBatchTensors, *,
                           scale: float | None = None, out: Tensor | None = None, return_lse: bool = False,
                           check: bool = False,
                           kv_scales: tuple[Tensor, Tensor] | None = None) -> Tensor | tuple[Tensor, Tensor]:
    """``softmax(scale * q K^T) V`` of one query token per sequence over its cached tokens.

    ``q [n_seqs, n_q, head_dim]`` in the pages' dtype; query head ``h`` reads KV head
    ``h // (n_q // n_kv)``.  ``seqs`` counts the cached tokens, the new one included (its
    ``cu_seqlens`` are the lengths' prefix sums, as :func:`plan_paged_step` writes them).
    ``scale`` defaults to ``head_dim ** -0.5``.  Returns ``out [n_seqs, n_q, head_dim]`` and with
    ``return_lse`` also ``ln sum exp`` of the scores (fp32 ``[n_seqs, n_q]``), with which parts
    of a cache attended separately (a shared prefix) can be joined.  A sequence without tokens
    gives zeros and ``-inf``.  The form of the launch goes by the batch and by ``seqs.max_seq_len``,
    which may be any bound: with one of a few hundred tokens short sequences take one launch, about
    half the time of the form that cuts long ones.  A captured step keeps the form of its
    capture, so a serving loop is faster with a graph for each class of lengths.  Any head_dim up to
    256 and any strides; rows that start on 16 bytes and are a multiple of 16 bytes long are read
    fastest.

    Slots behind a sequence's length are not read into the result, whatever they hold.  An infinite
    V element of a token that counts makes its column infinite (NaN where both signs meet; perhaps
    also where the token's weight is below 2^-126 of the largest and so 0 in fp32).  Tokens
    in blocks outside the cache or beyond the table are left out and recorded (``check=True``
    raises).

    **8-bit pages** (``torch.float8_e4m3fn`` or ``torch.int8``) come with ``kv_scales = (k_scales, v_scales)``, fp32
    ``[num_blocks, n_kv]``, one factor for each block and KV head — those that :func:`append_into_paged` keeps, or any.  ``q``
    then is bf16, fp16 or fp32 and ``out`` has its type; products are fp16 with fp32 sums, in which the codes and a 16-bit ``q``
    are exact (bf16: elements down to 2^-27 of the head's largest, those below in steps of 2^-38 of it); fp32 ``q`` and the weights
    enter as two terms each (2^-22).  A weight enters times its token's V scale, in steps of 2^-33 of the largest such product: beside
    a token whose V scale is 2^33 times theirs, others vanish even from the columns in which that token's codes are 0.  Weights below
    2^-122 of the largest are 0, whatever their V scale.
    A NaN code or scale of a token that counts gives NaN.
    """
    got = (_native_module or _native()).attend(q, k_pages, v_pages, seqs.cu_seqlens, seqs.block_tables, seqs.table_lens,
                                               seqs.max_seq_len, scale, out, return_lse, kv_scales)
    if check:
        ops.status_word(q.device).raise_if_set("paged_decode_attention")
    return got
