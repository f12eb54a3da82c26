"""RoPE tables for the fused patch kernel and the append.

The kernel reads ``cos/sin[position, i]`` for ``i < head_dim/2`` (the reference builds
``emb = cat(freqs, freqs)``, so the second half repeats the first; src/deltakv/rope.py:35-45).
Tables are built on the CPU with the same torch operations as the reference, so the angles
and their cos/sin are bit-identical to ``RotaryEmbedding.cos_cached/sin_cached``.
"""

from __future__ import annotations

import math
from weakref import WeakKeyDictionary

import torch
from torch import Tensor


_SCALINGS = {  # type -> the keys it takes, with their defaults (... : none)
    "linear": {"factor": ...},
    "ntk": {"factor": ...},
    "llama3": {"factor": ..., "original_max_seq": ..., "low_freq_factor": 1.0, "high_freq_factor": 4.0},
    "yarn": {"factor": ..., "original_max_seq": ..., "beta_fast": 32.0, "beta_slow": 1.0, "attention_factor": None},
}


def scaled_frequencies(dim: int, base: float, scaling: dict) -> tuple[Tensor, float]:
    """``(inv_freq, amplitude)``: the fp64 frequencies of ``dim / 2`` column pairs, changed for a long context, and the
    factor that cos and sin get (1 except for ``yarn``).  With theta_i = base^(-2i/dim) and s = ``factor``:

    * ``linear``  theta_i / s: positions are squeezed into the trained range;
    * ``ntk``     base' = base * s^(dim / (dim - 2)): the fastest pair stays, the slowest is divided by s;
    * ``llama3``  by the wavelength w_i = 2 pi / theta_i against L = ``original_max_seq``: pairs with w_i < L / ``high_freq_factor``
      stay, those with w_i > L / ``low_freq_factor`` are divided by s, between them
      theta_i (a + (1 - a) / s) with a = (L / w_i - low) / (high - low);
    * ``yarn``    theta_i (a_i + (1 - a_i) / s), where a_i falls from 1 to 0 between the pairs that make ``beta_fast`` and
      ``beta_slow`` turns within L; the amplitude is ``attention_factor``, by default 0.1 ln s + 1 (1 for s <= 1).
    """
    kind = scaling.get("type")
    if kind not in _SCALINGS:
        raise ValueError(f"rope scaling type {kind!r} is none of {', '.join(_SCALINGS)}")
    known = _SCALINGS[kind]
    if odd := set(scaling) - set(known) - {"type"}:
        raise ValueError(f"rope scaling {kind!r} does not take {', '.join(sorted(odd))}")
    if missing := [k for k, v in known.items() if v is ... and k not in scaling]:
        raise ValueError(f"rope scaling {kind!r} needs {', '.join(missing)}")
    given = {k: scaling.get(k, v) for k, v in known.items()}
    if any(v is not None and not v > 0 for v in given.values()):
        raise ValueError(f"rope scaling {kind!r}: its numbers must be positive")
    factor = float(given["factor"])
    i = torch.arange(0, dim, 2, dtype=torch.float64)
    if kind == "ntk":
        if dim <= 2:
            raise ValueError("rope scaling 'ntk' needs more than one pair of columns")
        return (base * factor ** (dim / (dim - 2))) ** (-i / dim), 1.0
    inv = float(base) ** (-i / dim)
    if kind == "linear":
        return inv / factor, 1.0
    length = float(given["original_max_seq"])
    if kind == "llama3":
        low, high = float(given["low_freq_factor"]), float(given["high_freq_factor"])
        if not high > low:
            raise ValueError("rope scaling 'llama3': high_freq_factor must be above low_freq_factor")
        a = ((length * inv / (2 * math.pi) - low) / (high - low)).clamp(0.0, 1.0)
        return inv * (a + (1.0 - a) / factor), 1.0

    def pair_of(turns):  # the (fractional) pair that makes so many turns within the length
        return dim * math.log(length / (turns * 2 * math.pi)) / (2 * math.log(base))

    first = max(math.floor(pair_of(given["beta_fast"])), 0)
    last = min(math.ceil(pair_of(given["beta_slow"])), dim - 1)
    a = 1.0 - ((i / 2 - first) / max(last - first, 0.001)).clamp(0.0, 1.0)
    amplitude = given["attention_factor"]
    if amplitude is None:
        amplitude = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    return inv * (a + (1.0 - a) / factor), float(amplitude)


class RotaryEmbedding:
    """Llama rotate-half RoPE tables (src/deltakv/rope.py:28-63), without the module.

    Beyond the reference's form, which the defaults are: ``rotary_dim`` turns only the first columns of each head,
    ``interleaved`` the pairs ``(2i, 2i + 1)`` instead of ``(i, i + rotary_dim / 2)``, and ``scaling`` stretches the
    frequencies for long contexts (a dict with ``type`` and its numbers, see :func:`scaled_frequencies`; its tables come from
    angles in fp64, so that positions of a million keep their accuracy).  :func:`~deltakv_b200.append_into_paged` takes
    every form; the patch routes rotate whole heads in halves (scaled or not) and refuse the other two.
    """

    def __init__(self, head_dim: int, max_seq: int = 8192, base: float = 10000.0, *, rotary_dim: int | None = None,
                 interleaved: bool = False, scaling: dict | None = None):
        if head_dim % 2 != 0 and rotary_dim is None:
            raise ValueError("RoPE head_dim must be even")
        dim = head_dim if rotary_dim is None else rotary_dim
        if not 0 < dim <= head_dim or dim % 2:
            raise ValueError(f"rotary_dim {dim} must be even and in (0, head_dim]")
        self.head_dim = head_dim
        self.rotary_dim = dim
        self.interleaved = bool(interleaved)
        self.max_seq = max_seq
        self.base = base
        with torch.inference_mode(False):  # ordinary tensors, whose changes half_tables can see
            if scaling is None:
                inv_freq = 1.0 / (base ** (torch.arange(0, dim, 2, dtype=torch.float32) / dim))
                t = torch.arange(max_seq, dtype=torch.float32)
                freqs = torch.outer(t, inv_freq)
                emb = torch.cat((freqs, freqs), dim=-1)
                self.inv_freq = inv_freq
                self.cos_cached = emb.cos()
                self.sin_cached = emb.sin()
            else:
                inv_freq, amplitude = scaled_frequencies(dim, base, scaling)
                freqs = torch.outer(torch.arange(max_seq, dtype=torch.float64), inv_freq)
                self.inv_freq = inv_freq.float()
                self.cos_cached = (freqs.cos() * amplitude).float().repeat(1, 2)
                self.sin_cached = (freqs.sin() * amplitude).float().repeat(1, 2)

    def form(self, head_dim: int, rotary_dim: int | None = None, interleaved: bool | None = None) -> tuple[int | None, bool]:
        """``(rotary_dim, interleaved)`` of this rope for heads of ``head_dim`` (``None``: the whole head), which what a
        caller asked for may not contradict."""
        if rotary_dim not in (None, self.rotary_dim) or interleaved not in (None, self.interleaved):
            raise ValueError(f"rope turns {self.rotary_dim} columns{' interleaved' if self.interleaved else ''}: "
                             "rotary_dim and interleaved may not say otherwise")
        if self.rotary_dim != self.head_dim and self.head_dim != head_dim:
            raise ValueError(f"rope for heads of {self.head_dim} columns does not go with head_dim {head_dim}")
        return (self.rotary_dim if self.rotary_dim != self.head_dim else None), self.interleaved


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


def half_tables(rope, device: torch.device, *, forms: bool = False) -> tuple[Tensor, Tensor]:
    """``(cos, sin)`` as contiguous fp32 ``[max_seq, head_dim/2]`` on ``device``.

    ``rope`` is a reference ``RotaryEmbedding`` module, one of this package, or a
    ``(cos, sin)`` pair that is already half-width.  A rope's tables are made once and again when
    its tensors change; tensors made in inference mode do not tell, so theirs are made anew
    each call (pass the pair to have none made).

    Inside a graph capture, kept tables are used as they are and stay for the life of the process
    (a replay knows their address alone, and goes on with the tables of its capture).  What is
    not there yet is made by the graph itself, at every replay, and not kept; for that the rope's
    tensors have to be on ``device``.

    ``forms``: the caller turns parts of heads and interleaved pairs too; without it such a rope is refused.
    """
    if not forms and isinstance(rope, RotaryEmbedding) and (rope.interleaved or rope.rotary_dim != rope.head_dim):
        raise ValueError("this operator rotates whole heads in halves: a rope with rotary_dim or interleaved is for "
                         "append_into_paged")
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
