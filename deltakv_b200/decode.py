"""One prefill or decode step of a paged cache: plan, append, attend.

The patch routes of this package change the K/V of tokens that are already cached; these three
operators are what a serving loop does between two patches, on the same pages, block tables
and :class:`~deltakv_b200.ops.SeqBatchTensors`:

* :func:`plan_paged_step`        block tables, slots and positions from lengths on the GPU
* :func:`append_into_paged`      rotate-half RoPE of the new q and k, K and V into their slots
* :func:`paged_decode_attention` attention of one new token per sequence over its pages

None of them reads anything back to the host (``check=True`` does, to raise what the kernels
recorded), so a step can be captured into a CUDA graph and replayed with other lengths.  They
are forms for serving: their outputs carry no gradient.  They run on the current stream of the tensors' device.  The cache layouts are the ones of
:func:`~deltakv_b200.paged.scatter_into_paged`; for its 5-D forms pass the K and V views
(``ops.page_view(cache, 0)``, ``ops.page_view(cache, 1)``).  The rotation is the reference's
(src/deltakv/rope.py:9-63), the page arithmetic that of src/deltakv/paged.py:39-43.
"""

from __future__ import annotations

import ctypes as C
from dataclasses import dataclass

import torch
from torch import Tensor

from deltakv_b200 import _lib as L
from deltakv_b200 import ops
from deltakv_b200.rope import half_tables


_I32 = torch.int32
_empty, _empty_like, _raw_stream = torch.empty, torch.empty_like, torch._C._cuda_getCurrentRawStream
# A decode step calls these operators once a layer, with kernels of a few microseconds: the checks
# read each attribute once and take strides as tuples, and the stream is taken as its raw handle
# (current_stream() builds an object: 3 us).


def _same_device(where: str, first: Tensor, *rest: Tensor | None) -> torch.device:
    dev = first.device
    if dev.type != "cuda":
        ops._require_cuda(first)
    for t in rest:
        if t is not None and t.device != dev:
            ops._require_cuda(t)
            raise ValueError(f"{where}: tensors on {dev} and {t.device}")
    return dev


def _call(fn, args, dev: torch.device, where: str) -> None:
    """Launch on the current stream of ``dev``, which need not be the current device."""
    index = dev.index
    if index == torch.cuda.current_device():
        rc = fn(C.byref(args), _raw_stream(index))
    else:
        with torch.cuda.device(dev):
            rc = fn(C.byref(args), _raw_stream(index))
    if rc:
        raise L.DkvError(rc, where)


def _int32_vector(t: Tensor, name: str, n: int | None) -> None:
    if t.dtype is not _I32:
        raise TypeError(f"{name} must be int32")
    if t.dim() != 1 or not t.is_contiguous() or (n is not None and t.numel() != n):
        raise ValueError(f"{name} must be a contiguous vector" + ("" if n is None else f" of {n}"))


def _rows(t: Tensor, name: str, rows: int, heads: int | None, hd: int) -> tuple[int, ...]:
    """The strides of a ``[rows, heads, hd]`` tensor."""
    shape = t.shape
    if len(shape) != 3 or shape[0] != rows or shape[2] != hd or (heads is not None and shape[1] != heads):
        raise ValueError(f"{name} {tuple(shape)} must be [{rows}, {'heads' if heads is None else heads}, {hd}]")
    strides = t.stride()
    if strides[2] != 1 and hd > 1:
        raise ValueError(f"{name} must have contiguous head_dim")
    return strides


def _page_pair(k_pages: Tensor, v_pages: Tensor) -> tuple[L.PagedCache, L.PagedCache]:
    shape, v_shape, dtype = k_pages.shape, v_pages.shape, k_pages.dtype
    if len(shape) != 4 or len(v_shape) != 4:
        raise ValueError(f"unsupported paged KV layout {tuple(shape)}, {tuple(v_shape)}")
    nb, bs, h, d = shape
    if dtype is not v_pages.dtype or bs != v_shape[1] or h != v_shape[2] or d != v_shape[3]:
        raise ValueError("k_pages and v_pages must share dtype, block size, heads and head_dim")
    code = ops.dkv_dtype(dtype)
    ks, vs = k_pages.stride(), v_pages.stride()
    if (ks[3] != 1 or vs[3] != 1) and d > 1:
        raise ValueError("paged cache head_dim must be contiguous")
    return (L.PagedCache(k_pages.data_ptr(), code, bs, h, d, nb, ks[0], ks[1], ks[2]),
            L.PagedCache(v_pages.data_ptr(), code, bs, h, d, v_shape[0], vs[0], vs[1], vs[2]))


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
    extended in place from the front of ``free_blocks``, sequence by sequence.  ``rows`` is the
    capacity of the row outputs (the sum of the new lengths, or more in a padded batch: rows
    past the last sequence get slot -1 and position 0); ``max_seq_len`` bounds the lengths and
    goes into the returned ``seqs``.

    With ``check=True`` what the kernel recorded (lengths out of range, a full table, no free
    blocks left) is raised after a synchronisation; otherwise the affected tokens only have
    slot -1.  At most 16384 sequences.
    """
    n = lengths.numel()
    _int32_vector(lengths, "lengths", n)
    if new_lengths is not None:
        _int32_vector(new_lengths, "new_lengths", n)
    if table_lens is not None:
        _int32_vector(table_lens, "table_lens", n)
    n_free = 0
    if free_blocks is not None:
        _int32_vector(free_blocks, "free_blocks", None)
        n_free = free_blocks.numel()
    if block_tables.dtype is not _I32:
        raise TypeError("block_tables must be int32")
    shape, strides = block_tables.shape, block_tables.stride()
    if len(shape) != 2 or shape[0] != n or (strides[1] != 1 and shape[1] > 1):
        raise ValueError("block_tables must be a row-major [n_seqs, max_blocks] int32 tensor")
    width = shape[1]
    if n > 1 and strides[0] < width:
        raise ValueError("block_tables rows overlap: the plan writes them")
    if not 0 < block_size < 1 << 31 or not 0 <= rows < 1 << 31 or not 0 <= max_seq_len < 1 << 31:
        raise ValueError("block_size must be positive, rows and max_seq_len not negative, all below 2**31")
    dev = _same_device("plan_paged_step", lengths, block_tables, new_lengths, table_lens, free_blocks)
    out = _empty(3 * n + 3 + rows, dtype=_I32, device=dev)
    cu, cu_new, lens, used, positions = torch.unsafe_split_with_sizes(out, (n + 1, n + 1, n, 1, rows))
    slots = _empty(rows, dtype=torch.int64, device=dev)
    st = ops.status_word(dev)
    base = out.data_ptr()
    args = L.StepPlanArgs(
        lengths.data_ptr(), ops.ptr(new_lengths), ops.ptr(table_lens), ops.ptr(free_blocks), n_free,
        block_tables.data_ptr(), strides[0], width, n, block_size, rows, base, base + 4 * (n + 1), base + 8 * (n + 1),
        base + 4 * (3 * n + 2), base + 4 * (3 * n + 3), slots.data_ptr(), st.ptr)
    _call(L.lib().dkv_plan_paged_step, args, dev, "dkv_plan_paged_step")
    if check:
        st.raise_if_set("plan_paged_step")
    seqs = ops.SeqBatchTensors(cu_seqlens=cu, block_tables=block_tables, max_seq_len=max_seq_len, table_lens=lens)
    return PagedStep(seqs, cu_new, positions, slots, used)


def append_into_paged(k: Tensor, v: Tensor, k_pages: Tensor, v_pages: Tensor, slots: Tensor, *,
                      q: Tensor | None = None, positions: Tensor | None = None, rope=None,
                      q_out: Tensor | None = None, check: bool = False) -> Tensor | None:
    """Store this step's ``k`` and ``v [rows, n_kv, head_dim]`` in their ``slots``, rotated.

    ``slots`` (int64) and ``positions`` (int32) are a :class:`PagedStep`'s; a negative slot
    stores nothing.  With ``rope`` (a ``RotaryEmbedding`` or a half-width ``(cos, sin)`` pair)
    K gets the rotate-half RoPE of its position, and so do the rows of ``q [rows, n_q, head_dim]``
    — padding rows too — into ``q_out`` (default: a new tensor; ``q`` itself is allowed), which
    is returned.  The inputs may be strided views (heads of one fused projection); their dtype
    is the pages' or fp32, rounded once on the way into the pages.

    The stored values replace what the slots held (``scatter_into_paged`` adds).  Slots must be
    distinct.  ``check=True`` raises recorded range errors (a slot beyond the pages, a position
    beyond the tables: those rows store nothing).
    """
    kd, vd = _page_pair(k_pages, v_pages)
    rows, n_kv, hd, dtype = slots.numel(), kd.n_heads, kd.head_dim, k.dtype
    if slots.dtype is not torch.int64:
        raise TypeError("slots must be int64")
    if slots.dim() != 1 or not slots.is_contiguous():
        raise ValueError("slots must be a contiguous vector")
    ks, vs = _rows(k, "k", rows, n_kv, hd), _rows(v, "v", rows, n_kv, hd)
    if v.dtype is not dtype or (q is not None and q.dtype is not dtype):
        raise TypeError("q, k and v must share a dtype")
    if dtype is not k_pages.dtype and dtype is not torch.float32:
        raise TypeError(f"{dtype} rows do not go into {k_pages.dtype} pages (pass the pages' dtype or fp32)")
    if rope is not None:
        if positions is None:
            raise ValueError("rope needs positions")
        _int32_vector(positions, "positions", rows)
    n_q, qs, os = 0, (0, 0), (0, 0)
    if q is None:
        if q_out is not None:
            raise ValueError("q_out without q")
    else:
        if rope is None:
            raise ValueError("q is only rotated: pass rope and positions with it")
        qs, n_q = _rows(q, "q", rows, None, hd), q.shape[1]
        if q_out is not None:
            os = _rows(q_out, "q_out", rows, n_q, hd)
            if q_out.dtype is not dtype:
                raise TypeError("q_out must have q's dtype")
    dev = _same_device("append_into_paged", k, v, k_pages, v_pages, slots, q, positions, q_out)
    cos = sin = None
    max_pos = 0
    if rope is not None:
        cos, sin = half_tables(rope, dev)
        shape = cos.shape
        if len(shape) != 2 or shape != sin.shape or 2 * shape[1] != hd:
            raise ValueError(f"rope tables {tuple(shape)} do not cover head_dim {hd}")
        max_pos = shape[0]
    if q is not None and q_out is None:
        q_out = _empty_like(q)
        os = q_out.stride()
    st = ops.status_word(dev)
    args = L.AppendArgs(
        k.data_ptr(), v.data_ptr(), ops.ptr(q), ops.dkv_dtype(dtype), n_q, rows, ks[0], ks[1], vs[0], vs[1], qs[0], qs[1],
        ops.ptr(q_out), os[0], os[1], slots.data_ptr(), ops.ptr(positions) if max_pos else None, ops.ptr(cos),
        ops.ptr(sin), max_pos, kd, vd, st.ptr)
    _call(L.lib().dkv_append_paged, args, dev, "dkv_append_paged")
    if check:
        st.raise_if_set("append_into_paged")
    return q_out


_workspace_bytes: dict[tuple, int] = {}  # a function of the shape and the device alone


def paged_decode_attention(q: Tensor, k_pages: Tensor, v_pages: Tensor, seqs: ops.SeqBatchTensors, *,
                           scale: float | None = None, out: Tensor | None = None, return_lse: bool = False,
                           check: bool = False) -> Tensor | tuple[Tensor, Tensor]:
    """``softmax(scale * q K^T) V`` of one query token per sequence over its cached tokens.

    ``q [n_seqs, n_q, head_dim]`` in the pages' dtype; query head ``h`` reads KV head
    ``h // (n_q // n_kv)``.  ``seqs`` counts the cached tokens, the new one included (its
    ``cu_seqlens`` are the lengths' prefix sums, as :func:`plan_paged_step` writes them).
    ``scale`` defaults to ``head_dim ** -0.5``.  Returns ``out [n_seqs, n_q, head_dim]`` and with
    ``return_lse`` also ``ln sum exp`` of the scores (fp32 ``[n_seqs, n_q]``), with which parts
    of a cache attended separately (a shared prefix) can be joined.  A sequence without tokens
    gives zeros and ``-inf``.  Any head_dim up to 256 and any strides; rows that start on 16
    bytes and are a multiple of 16 bytes long are read fastest.

    Slots behind a sequence's length are not read into the result, whatever they hold.  Tokens
    in blocks outside the cache or beyond the table are left out and recorded (``check=True``
    raises).
    """
    kd, vd = _page_pair(k_pages, v_pages)
    n_kv, hd, dtype = kd.n_heads, kd.head_dim, q.dtype
    cu, tables, lens = seqs.cu_seqlens, seqs.block_tables, seqs.table_lens
    n = cu.numel() - 1
    qs = _rows(q, "q", n, None, hd)
    heads = q.shape[1]
    if dtype is not k_pages.dtype:
        raise TypeError(f"q is {dtype}, the pages are {k_pages.dtype}")
    if hd > 256:
        raise ValueError(f"head_dim {hd} is above 256")
    if heads == 0 or n_kv == 0 or heads % n_kv:
        raise ValueError(f"{heads} query heads do not share {n_kv} KV heads evenly")
    if tables.dim() == 2 and tables.shape[0] < n:
        raise ValueError(f"block_tables has {tables.shape[0]} rows for {n} sequences")
    if lens is not None and (lens.numel() < n or not lens.is_contiguous()):
        raise ValueError(f"table_lens must be a contiguous vector of {n}")
    if out is not None:
        os = _rows(out, "out", n, heads, hd)
        if out.dtype is not dtype:
            raise TypeError("out must have q's dtype")
    dev = _same_device("paged_decode_attention", q, k_pages, v_pages, cu, tables, lens, out)
    sb = seqs.struct()
    if out is None:
        out = _empty_like(q)
        os = out.stride()
    lse = _empty((n, heads), dtype=torch.float32, device=dev) if return_lse else None
    st = ops.status_word(dev)
    args = L.PagedDecodeArgs(
        q.data_ptr(), qs[0], qs[1], heads, hd ** -0.5 if scale is None else scale, sb, kd, vd,
        out.data_ptr(), os[0], os[1], ops.ptr(lse), None, 0, st.ptr)
    key = (dev.index, heads, n_kv, hd, kd.dtype, n, sb.max_seq_len)
    nbytes = _workspace_bytes.get(key)
    if nbytes is None:
        got = C.c_int64()
        with torch.cuda.device(dev):
            L.check(L.lib().dkv_paged_decode_workspace_bytes(C.byref(args), C.byref(got)),
                    "dkv_paged_decode_workspace_bytes")
        if len(_workspace_bytes) > 4096:
            _workspace_bytes.clear()
        nbytes = _workspace_bytes[key] = got.value
    if nbytes:
        ws = _empty(nbytes, dtype=torch.uint8, device=dev)
        args.workspace, args.workspace_bytes = ws.data_ptr(), nbytes
    _call(L.lib().dkv_paged_decode_attention, args, dev, "dkv_paged_decode_attention")
    if check:
        st.raise_if_set("paged_decode_attention")
    return (out, lse) if return_lse else out
