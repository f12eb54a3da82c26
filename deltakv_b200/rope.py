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


# per rope object (while it lives) and device: the tensors the tables were made from, their
# versions, and the tables.  Holding the source tensors keeps "is" meaningful: neither an object
# nor a tensor whose address was reused can match.
_table_cache: WeakKeyDictionary = WeakKeyDictionary()


def half_tables(rope, device: torch.device) -> tuple[Tensor, Tensor]:
    """``(cos, sin)`` as contiguous fp32 ``[max_seq, head_dim/2]`` on ``device``.

    ``rope`` is a reference ``RotaryEmbedding`` module, one of this package, or a
    ``(cos, sin)`` pair that is already half-width.  A rope's tables are made once and again when
    its tensors change; tensors made in inference mode do not tell, so theirs are made anew
    each call (pass the pair to have none made).
    """
    if isinstance(rope, tuple):
        c, s = rope
        if (c.dtype is torch.float32 and s.dtype is torch.float32 and c.device == device and s.device == device
                and c.is_contiguous() and s.is_contiguous()):
            return c, s
        return c.to(device=device, dtype=torch.float32).contiguous(), s.to(device=device, dtype=torch.float32).contiguous()
    cos_full, sin_full = rope.cos_cached, rope.sin_cached
    hd = cos_full.shape[-1]

    def make() -> tuple[Tensor, Tensor]:
        return (cos_full[:, : hd // 2].to(device=device, dtype=torch.float32).contiguous(),
                sin_full[:, : hd // 2].to(device=device, dtype=torch.float32).contiguous())

    if cos_full.is_inference() or sin_full.is_inference():
        return make()
    try:
        made = _table_cache.setdefault(rope, {})
    except TypeError:  # an object without hash or weak references: made anew each call
        made = {}
    source = (cos_full, sin_full, cos_full._version, sin_full._version)
    hit = made.get(str(device))
    if hit is not None and all(x is y for x, y in zip(hit[0][:2], source[:2])) and hit[0][2:] == source[2:]:
        return hit[1]
    out = make()
    made[str(device)] = (source, out)
    return out


def max_positions(rope) -> int:
    if isinstance(rope, tuple):
        return int(rope[0].shape[0])
    return int(getattr(rope, "max_seq", rope.cos_cached.shape[0]))
