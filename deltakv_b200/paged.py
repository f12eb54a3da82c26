"""Drop-ins for ``deltakv.paged`` (src/deltakv/paged.py:8-70) on the B200 kernels, and their forms for batches and
8-bit pages.

Same signatures, layouts, in-place additive semantics and error messages as the
reference; the per-block Python loop becomes one kernel launch.  Results are
bit-identical: each element is ``round(fp32(page) + fp32(delta))`` in the page dtype.
"""

from __future__ import annotations

from typing import Sequence

import torch
from torch import Tensor

from deltakv_b200 import ops


def _normalise_table(block_table: Sequence[int], num_blocks: int) -> list[int]:
    # torch indexing accepts negative block ids (pages[-1] is the last block)
    out = []
    for bid in block_table:
        b = int(bid)
        if b < -num_blocks or b >= num_blocks:
            raise IndexError(f"index {b} is out of bounds for dimension 0 with size {num_blocks}")
        out.append(b % num_blocks)
    return out


def scatter_into_paged(delta: Tensor, cache: Tensor, block_table: list[int], block_size: int, *,
                       kv_dim: int = 0, page_scales: Tensor | None = None) -> None:
    """Add ``delta [seq, n_kv_heads, head_dim]`` into a paged cache, in place.

    Layouts: ``[num_blocks, block_size, h, d]``, ``[2, num_blocks, block_size, h, d]``
    (``kv_dim`` picks K=0 / V=1) and ``[num_blocks, 2, block_size, h, d]``.  ``page_scales``: of 8-bit
    pages, see :func:`scatter_into_paged_batched`; ``block_size`` is the cache's then.
    """
    seq = delta.shape[0]
    n_blocks_needed = (seq + block_size - 1) // block_size
    if len(block_table) < n_blocks_needed:
        raise ValueError("block_table shorter than prefix")
    pages = ops.page_view(cache, kv_dim)
    if seq == 0:
        return
    if block_size > pages.shape[1]:
        raise ValueError(f"block_size {block_size} exceeds the cache's {pages.shape[1]} slots per block")
    table = _normalise_table(list(block_table)[:n_blocks_needed], pages.shape[0])
    seqs = ops.SeqBatchTensors.single(seq, table, pages.device)
    if page_scales is not None:
        _whole_blocks(pages, block_size)
        if len(set(table)) != len(table):
            raise ValueError("block_table names a block of 8-bit pages twice")
        return scatter_into_paged_batched(delta, pages, seqs, page_scales=page_scales)
    # the kernel reads slot i % block_size of block i // block_size, as the reference does
    view = pages if block_size == pages.shape[1] else pages[:, :block_size]
    ops.scatter_paged(delta, view, seqs)


def gather_from_paged(cache: Tensor, block_table: list[int], seq_len: int, block_size: int, *,
                      kv_dim: int = 0, page_scales: Tensor | None = None,
                      dtype: torch.dtype | None = None) -> Tensor:
    """Inverse of :func:`scatter_into_paged`: ``[seq_len, n_kv_heads, head_dim]``.

    Rows past the end of a short block table stay zero, as in the reference.  ``page_scales`` and
    ``dtype``: of 8-bit pages, see :func:`gather_from_paged_batched`; ``block_size`` is the cache's then.
    """
    pages = ops.page_view(cache, kv_dim)
    n_kv, hd = pages.shape[-2], pages.shape[-1]
    if page_scales is None and (dtype or pages.dtype) != pages.dtype:
        raise TypeError("dtype goes with 8-bit pages: values of other pages come in their own type")
    n_blocks_needed = (seq_len + block_size - 1) // block_size
    table = _normalise_table(list(block_table)[:n_blocks_needed], pages.shape[0])
    if page_scales is not None:
        _whole_blocks(pages, block_size)
        seqs = ops.SeqBatchTensors.single(min(seq_len, len(table) * block_size), table, pages.device)
        return gather_from_paged_batched(pages, seqs, seq_len, page_scales=page_scales, dtype=dtype)
    out = pages.new_zeros(seq_len, n_kv, hd)
    covered = min(seq_len, len(table) * block_size)
    if covered == 0:
        return out
    view = pages if block_size == pages.shape[1] else pages[:, :block_size]
    seqs = ops.SeqBatchTensors.single(covered, table, pages.device)
    ops.gather_paged(view, seqs, out)
    return out


def _whole_blocks(pages: Tensor, block_size: int) -> None:
    if block_size != pages.shape[1]:
        raise ValueError(f"8-bit pages of {pages.shape[1]} slots a block cannot be used as blocks of {block_size}: "
                         "a block has one scale")


def scatter_into_paged_batched(delta: Tensor, pages: Tensor, seqs: ops.SeqBatchTensors,
                               check: bool = False, *, page_scales: Tensor | None = None) -> None:
    """Many sequences in one launch: ``delta`` rows follow ``seqs.cu_seqlens``.

    With ``check=True`` device-side range errors (short table, block id out of range) are
    raised after a synchronisation; otherwise they are recorded in the status word only.

    8-bit pages (``torch.float8_e4m3fn`` or ``torch.int8``, at most 1024 slots a block) come with their ``page_scales``, fp32
    ``[num_blocks, heads]`` (:func:`~deltakv_b200.append_into_paged` keeps such): value + delta is formed in fp32 and
    the block quantised again.  A block that a sequence covers whole gets the scale that its new values need; in
    a sequence's last block the slots behind its end are kept, and the scale only grows.  Pages of one sequence
    must not be another's (a shared prefix is patched by one of them): ``check=True`` refuses such a call before it stores anything, without it
    it is recorded, and the pages hold anything.  ``delta`` may be fp32, fp16 or bf16; the launch runs on the current stream of the pages' device.
    """
    st = ops.status_word(pages.device) if pages.is_cuda else None
    if page_scales is not None:
        _native().scatter(delta, pages, page_scales, seqs.cu_seqlens, seqs.block_tables, seqs.table_lens, seqs.max_seq_len, check)
    else:
        ops.scatter_paged(delta, pages, seqs, st)
    if check:
        st.raise_if_set("scatter_into_paged_batched")


def gather_from_paged_batched(pages: Tensor, seqs: ops.SeqBatchTensors, rows: int, *, page_scales: Tensor,
                              dtype: torch.dtype | None = None, out: Tensor | None = None, check: bool = False) -> Tensor:
    """The values of many sequences' tokens in 8-bit pages, in one launch: ``[rows, heads, head_dim]``, rows as
    ``seqs.cu_seqlens`` lays them out.

    ``page_scales``: as for :func:`scatter_into_paged_batched`.  ``rows`` is the capacity (the lengths live on the GPU); rows behind the last
    sequence are zero in a new tensor and left as they are in ``out``.  ``dtype`` (fp32, the default, fp16 or bf16) is
    the new tensor's: values are rounded to fp32 and then to it (an e4m3 code times a power of two is exact in all but fp16's range).  Tokens without a block
    are zero, recorded and raised with ``check=True``.
    """
    if out is not None and dtype not in (None, out.dtype):
        raise TypeError("dtype is that of a new tensor: out has its own")
    like = _LIKE.get(torch.float32 if dtype is None else dtype)
    if like is None:
        raise TypeError(f"dtype {dtype} is not supported by the B200 kernels")
    out = _native().gather(pages, page_scales, seqs.cu_seqlens, seqs.block_tables, seqs.table_lens, seqs.max_seq_len, rows, like,
                           out)
    if check:
        ops.status_word(pages.device).raise_if_set("gather_from_paged_batched")
    return out


_LIKE = {t: torch.empty(0, dtype=t) for t in (torch.float32, torch.float16, torch.bfloat16)}  # what names a type to C++


def _native():
    from deltakv_b200 import decode  # the extension module's loader; decode's operators need nothing of this file

    return decode._native_module or decode._native()
