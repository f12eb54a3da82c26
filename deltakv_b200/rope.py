"""RoPE tables for the fused patch kernel.

The kernel reads ``cos/sin[position, i]`` for ``i < head_dim/2`` (the reference builds
``emb = cat(freqs, freqs)``, so the second half repeats the first; src/deltakv/rope.py:35-45).
Tables are built on the CPU with the same torch operations as the reference, so the angles
and their cos/sin are bit-identical to ``RotaryEmbedding.cos_cached/sin_cached``.
"""

from __future__ import annotations

from weakref import WeakKeyDictionary

import torch
from torch import Tensor


class RotaryEmbedding:
    """Llama rotate-half RoPE tables (src/deltakv/rope.py:28-63), without the module."""

    def __init__(self, head_dim: int, max_seq: int = 8192, base: float = 10000.0):
        if head_dim % 2 != 0:
            raise ValueError("RoPE head_dim must be even")
        self.head_dim = head_dim
        self.max_seq = max_seq
        self.base = base
        with torch.inference_mode(False):  # ordinary tensors, whose changes half_tables can see
            inv_freq = 1.0 / (base ** (torch.arange(0, head_dim, 2, dtype=torch.float32) / head_dim))
            t = torch.arange(max_seq, dtype=torch.float32)
            freqs = torch.outer(t, inv_freq)
            emb = torch.cat((freqs, freqs), dim=-1)
            self.inv_freq = inv_freq
            self.cos_cached = emb.cos()
            self.sin_cached = emb.sin()


class _Kept:
    """Half-width tables, and the tensors (with their versions) they were made from: holding those keeps
    "is" meaningful, neither an object nor a tensor whose address was reused can match.

    They are read on any stream.  So they are finished when they are kept, and each stream that reads
    them is told to the allocator, which then does not hand out their memory before its work is done."""

    __slots__ = ("cos_full", "sin_full", "versions", "tables", "captured", "streams")

    def __init__(self, cos_full: Tensor, sin_full: Tensor, versions: tuple[int, int], tables: tuple[Tensor, Tensor]):
        self.cos_full, self.sin_full, self.versions, self.tables = cos_full, sin_full, versions, tables
        self.captured = False
        device = tables[0].device
        if device.type == "cuda":
            torch.cuda.current_stream(device).synchronize()
            self.streams = {_raw_stream(device.index)}

    def match(self, cos_full: Tensor, sin_full: Tensor) -> bool:
        return (self.cos_full is cos_full and self.sin_full is sin_full
                and self.versions == (cos_full._version, sin_full._version))

    def read(self, capturing: bool) -> tuple[Tensor, Tensor]:
        """The tables, for a launch on the current stream of their device."""
        tables = self.tables
        if capturing:
            if not self.captured:
                self.captured = True
                _captured_tables.append(tables)
        elif tables[0].is_cuda and (raw := _raw_stream(tables[0].device.index)) not in self.streams:
            self.streams.add(raw)
            stream = torch.cuda.current_stream(tables[0].device)
            tables[0].record_stream(stream), tables[1].record_stream(stream)
        return tables


_table_cache: WeakKeyDictionary = WeakKeyDictionary()  # per rope object, while it lives: {device: _Kept}
_captured_tables: list[tuple[Tensor, Tensor]] = []     # what captured launches read: replays have only addresses


def _raw_stream(index: int) -> int:
    return torch._C._cuda_getCurrentRawStream(index)


def _capturing(device: torch.device) -> bool:
    if device.type != "cuda":
        return False
    if device.index is None or device.index == torch._C._cuda_getDevice():
        return torch._C._cuda_isCurrentStreamCapturing()
    with torch.cuda.device(device):
        return torch.cuda.is_current_stream_capturing()


def _on_device(cos: Tensor, sin: Tensor, device: torch.device, capturing: bool) -> tuple[Tensor, Tensor]:
    if capturing and (cos.device != device or sin.device != device):
        raise RuntimeError(f"RoPE tables on {cos.device} cannot be copied to {device} inside a graph capture: "
                           "call the operator (or half_tables) with this rope once before it")
    return cos.to(device=device, dtype=torch.float32).contiguous(), sin.to(device=device, dtype=torch.float32).contiguous()


def half_tables(rope, device: torch.device) -> tuple[Tensor, Tensor]:
    """``(cos, sin)`` as contiguous fp32 ``[max_seq, head_dim/2]`` on ``device``.

    ``rope`` is a reference ``RotaryEmbedding`` module, one of this package, or a
    ``(cos, sin)`` pair that is already half-width.  A rope's tables are made once and again when
    its tensors change; tensors made in inference mode do not tell, so theirs are made anew
    each call (pass the pair to have none made).

    Inside a graph capture, kept tables are used as they are and stay for the life of the process
    (a replay knows their address alone, and goes on with the tables of its capture).  What is
    not there yet is made by the graph itself, at every replay, and not kept; for that the rope's
    tensors have to be on ``device``.
    """
    if isinstance(rope, tuple):
        c, s = rope
        if (c.dtype is torch.float32 and s.dtype is torch.float32 and c.device == device and s.device == device
                and c.is_contiguous() and s.is_contiguous()):
            return c, s
        return _on_device(c, s, device, _capturing(device))
    cos_full, sin_full = rope.cos_cached, rope.sin_cached
    half = cos_full.shape[-1] // 2
    capturing = _capturing(device)
    if cos_full.is_inference() or sin_full.is_inference():
        return _on_device(cos_full[:, :half], sin_full[:, :half], device, capturing)
    try:
        kept = _table_cache.setdefault(rope, {})
    except TypeError:  # an object without hash or weak references: made anew each call
        return _on_device(cos_full[:, :half], sin_full[:, :half], device, capturing)
    hit = kept.get(device)
    if hit is None or not hit.match(cos_full, sin_full):
        versions = (cos_full._version, sin_full._version)
        tables = _on_device(cos_full[:, :half], sin_full[:, :half], device, capturing)
        if capturing:
            return tables
        hit = kept[device] = _Kept(cos_full, sin_full, versions, tables)
    return hit.read(capturing)


def max_positions(rope) -> int:
    if isinstance(rope, tuple):
        return int(rope[0].shape[0])
    return int(getattr(rope, "max_seq", rope.cos_cached.shape[0]))
