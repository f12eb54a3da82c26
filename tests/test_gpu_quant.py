"""The 8-bit paged cache and the rotary forms of the append, against plain implementations in 64 bits.

Tolerances, derived.  A stored value is off by half a step of its scale: for int8 s/2, for e4m3 half a unit of its last place,
2^-4 of the value or 2^-10 s where that is more (subnormals).  Before that come a few fp32 roundings: the rotation's two
products and their sum (3 * 2^-24 of |x| + |y| each), the factor 1/s and the product with it (2 * 2^-24); next to a tie
they may choose the other neighbour, so they add to the half step.  What a growing scale rounds again is off by half a
step of each scale that it had, and a scale that grows doubles at least: less than one step of the last in all (e4m3: only what
becomes subnormal is rounded again: 2^-10 s for each growth, so 2^-9 s).

The attention: a score is a product sum of head_dim terms times two scales, off by (head_dim + 12) 2^-23 sum |q_d k_d| scale
=: ds (tensor cores may truncate, hence 2^-23; fp32 q as two f16 terms adds 2^-21), which moves every weight by a relative
2 ds.  Weights enter to 2^-21 as two f16 terms and to 2^-11 as one (bf16); exp and the running sums add 2^-20 and n 2^-24.
All relative to A = sum p |v| / sum p; out is rounded once.  And a floor: a weight W = p (V's scale) enters as an f16 number in
units of 2^-8 of a power of two that is at most the largest W (headroom for larger scores and scales of V's to come).  f16 steps
are never below 2^-24, so a weight is off by up to 2^-25 2^-8 = 2^-33 of the largest W, whatever its size (a column where the
heavy tokens' codes are 0 shows it): n tokens with codes of up to c add n c 2^-33 max W.
"""

from __future__ import annotations

import math
import random

import pytest
import torch

import deltakv_b200 as dkv
from deltakv_b200 import ops

pytestmark = pytest.mark.gpu

BF, F16, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64
E4M3, I8 = torch.float8_e4m3fn, torch.int8
KINDS, TYPES = [E4M3, I8], [BF, F16, F32]


def bits(t):
    return t.view(torch.uint8) if t.element_size() == 1 else t


def first_scale(top, kind):
    """Of a block that holds nothing, in fp64 from the fp32 quotient that the kernel forms."""
    x = (top.float() / (448.0 if kind == E4M3 else 127.0)).double()
    if kind == E4M3:
        m, e = torch.frexp(x)
        x = torch.ldexp(torch.ones_like(x), e - (m == 0.5).int())
    return torch.where(top > 0, x.clamp(min=2.0 ** -126), 0.0)


def most(kind):
    return 448.0 if kind == E4M3 else 127.0


def power_of_two(x):
    return torch.frexp(x)[0] == 0.5


def half_step(values, scale, kind):
    if kind == I8:
        return scale / 2 + 0 * values
    return torch.maximum(values.abs() * 2.0 ** -4, scale * 2.0 ** -10)


class Cache8:
    """K and V pages of 8 bits in a layout, with scales; tables with shuffled blocks over lens."""

    def __init__(self, lens, n_kv, hd, block, kind, dev, layout="kv_first", seed=0, spare=3, garbage=True, spread=(-9, -5)):
        g = torch.Generator().manual_seed(seed)
        need = [-(-n // block) for n in lens]
        nb = sum(need) + spare
        self.lens, self.block, self.kind = lens, block, kind
        shape = (block, n_kv, hd)
        # any codes but NaN (int8: but -128), then scales that differ from block to block
        def codes(*lead):
            c = torch.randint(0, 256, (*lead, *shape), generator=g, dtype=torch.uint8)
            if kind == E4M3:
                c[(c & 0x7F) == 0x7F] = 0x31
            else:
                c[c == 0x80] = 0x05
            return c
        if layout == "kv_first":
            full = codes(2, nb)
            pick = lambda f: (f[0], f[1])  # noqa: E731
        elif layout == "block_first":
            full = codes(nb, 2)
            pick = lambda f: (f[:, 0], f[:, 1])  # noqa: E731
        elif layout == "odd":  # every stride padded, nothing aligned
            full = torch.zeros(2, nb, block + 1, n_kv + 1, hd + 3, dtype=torch.uint8)
            full[:, :, 1:, 1:, 1:hd + 1] = codes(2, nb)
            pick = lambda f: (f[0, :, 1:, 1:, 1:hd + 1], f[1, :, 1:, 1:, 1:hd + 1])  # noqa: E731
        else:  # heads before slots
            full = codes(2, nb).transpose(2, 3).contiguous()
            pick = lambda f: (f[0].transpose(1, 2), f[1].transpose(1, 2))  # noqa: E731
        scales = torch.exp2(torch.randint(*spread, (nb, 2, n_kv), generator=g).float())
        if kind == I8:
            scales *= 1 + torch.rand(scales.shape, generator=g)
        order = torch.randperm(nb, generator=g)
        tables = torch.zeros(max(len(lens), 1), max(max(need, default=0), 1), dtype=torch.int32)
        used = torch.zeros(nb, block, dtype=torch.bool)
        at = 0
        for b, n in enumerate(need):
            tables[b, :n] = order[at:at + n]
            for i in range(n):
                used[order[at + i], : min(block, lens[b] - i * block)] = True
            at += n
        if garbage:  # what no token owns: NaN codes, and NaN scales where no token of the block counts
            for x in pick(full):
                x[~used] = 0x7F if kind == E4M3 else 0x80
            scales[~used.any(1)] = math.nan
        full = full.to(dev)
        self.k, self.v = (x.view(kind) for x in pick(full))
        scales = scales.to(dev)
        self.scales = (scales[:, 0], scales[:, 1])  # strided views of one tensor
        self.tables, self.used = tables.to(dev), used
        cu = [0]
        for n in lens:
            cu.append(cu[-1] + n)
        self.cu = torch.tensor(cu, dtype=torch.int32, device=dev)

    def seqs(self, longest=None, **kw):
        return dkv.SeqBatchTensors(cu_seqlens=self.cu, block_tables=self.tables,
                                   max_seq_len=max(self.lens, default=0) if longest is None else longest, **kw)

    def values(self, dtype=F64):
        return tuple(bits(x).contiguous().view(self.kind).to(dtype) * s.to(dtype)[:, None, :, None]
                     for x, s in zip((self.k, self.v), self.scales))

    def tokens(self, b):
        """K, V (fp64) and V's scales times the largest code, of each token."""
        n = self.lens[b]
        ids = self.tables[b, : -(-n // self.block)].long()
        k, v = ((bits(x)[ids].contiguous().view(self.kind).double() * s[ids].double()[:, None, :, None])
                .reshape(-1, x.shape[2], x.shape[3])[:n] for x, s in zip((self.k, self.v), self.scales))
        return k, v, most(self.kind) * self.scales[1][ids].double().repeat_interleave(self.block, 0)[:n]


# ---------------------------------------------------------------------------------------
# rotary forms
# ---------------------------------------------------------------------------------------
def turned(x, cos, sin, pos, rot, interleaved):
    """In x's type, one operation at a time."""
    c, s = cos[pos.long()][:, None].to(x.dtype), sin[pos.long()][:, None].to(x.dtype)
    y = x.clone()
    one, two = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    lo, hi = x[..., one], x[..., two]
    y[..., one], y[..., two] = lo * c - hi * s, hi * c + lo * s
    return y


FORMS = [(128, 64, True), (128, 128, True), (128, 32, False), (64, 48, False), (64, 2, True), (80, 40, True), (96, 24, False),
         (50, 20, True), (33, 10, False), (256, 64, True), (48, 16, False)]


@pytest.mark.parametrize("hd,rot,interleaved", FORMS)
def test_rotary_forms_into_fp32_pages_bit_for_bit(cuda, hd, rot, interleaved):
    g = torch.Generator(device=cuda).manual_seed(hd + rot)
    rows, heads, n_kv = 37, 5, 3
    qkv = torch.randn(rows, heads + 2 * n_kv, hd, device=cuda, generator=g)
    q, k, v = qkv.split([heads, n_kv, n_kv], dim=1)
    pos = torch.randint(0, 300, (rows,), device=cuda, dtype=torch.int32, generator=g)
    slots = torch.randperm(64, device=cuda, generator=g)[:rows]
    pages = torch.zeros(2, 4, 16, n_kv, hd, device=cuda)
    rope = dkv.RotaryEmbedding(hd, 300, rotary_dim=rot, interleaved=interleaved, scaling={"type": "linear", "factor": 2.0})
    cos, sin = (t[:, :rot // 2].to(cuda) for t in (rope.cos_cached, rope.sin_cached))
    got = dkv.append_into_paged(k, v, pages[0], pages[1], slots, q=q, positions=pos, rope=rope, check=True)
    want = pages[0].clone()
    want[slots // 16, slots % 16] = turned(k, cos, sin, pos, rot, interleaved)
    assert torch.equal(got, turned(q, cos, sin, pos, rot, interleaved))
    assert torch.equal(pages[0], want) and torch.equal(pages[1][slots // 16, slots % 16], v)
    # the same as a pair of tables, in place
    again = torch.zeros_like(pages)
    inplace = dkv.append_into_paged(k, v, again[0], again[1], slots, q=q, q_out=q, positions=pos, rope=(cos, sin), rotary_dim=rot,
                                    interleaved=interleaved)
    assert inplace is q and torch.equal(q, got) and torch.equal(again, pages)


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("hd,rot,interleaved", FORMS)
def test_rotary_forms_into_16_bit_pages(cuda, dtype, hd, rot, interleaved):
    g = torch.Generator(device=cuda).manual_seed(hd + rot)
    rows, heads, n_kv = 70, 6, 2
    q, k, v = (torch.randn(rows, h, hd, device=cuda, generator=g).to(dtype) for h in (heads, n_kv, n_kv))
    pos = torch.randint(0, 300, (rows,), device=cuda, dtype=torch.int32, generator=g)
    slots = torch.randperm(96, device=cuda, generator=g)[:rows]
    slots[5] = -1
    pages = torch.zeros(2, 6, 16, n_kv, hd, device=cuda, dtype=dtype)
    rope = dkv.RotaryEmbedding(hd, 300, rotary_dim=rot, interleaved=interleaved)
    cos, sin = (t[:, :rot // 2].to(cuda) for t in (rope.cos_cached, rope.sin_cached))
    got = dkv.append_into_paged(k, v, pages[0], pages[1], slots, q=q, positions=pos, rope=rope, check=True)
    kept = slots >= 0
    for out, x in ((got, q), (pages[0][slots[kept] // 16, slots[kept] % 16], k[kept])):
        want = turned(x.double(), cos, sin, pos if x is q else pos[kept], rot, interleaved)
        # two products and a sum in fp32, one rounding
        tol = torch.finfo(dtype).eps / 2 * want.abs() + 2.0 ** -22 * x.double().abs().amax(-1, keepdim=True) + 1e-7
        assert torch.all((out.double() - want).abs() <= tol)
    assert torch.equal(pages[1][slots[kept] // 16, slots[kept] % 16], v[kept])


# ---------------------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------------------
def check_stored(c, side, x, slots, slack):
    """x (fp64, [rows, heads, hd]) as they lie in the slots: off by half a step, plus slack (fp32 roundings before)."""
    pages, scales = (c.k, c.scales[0]) if side == 0 else (c.v, c.scales[1])
    block, at = slots // c.block, slots % c.block
    s = scales[block].double()[..., None]
    got = bits(pages)[block, at].view(c.kind).double() * s
    off = (got - x).abs()
    tol = half_step(x, s, c.kind) + slack + 2.0 ** -22 * x.abs()
    assert torch.all(off <= tol), float((off / tol).max())


def append_case(cuda, kind, dtype, hd, rot, interleaved, block, layout, n_kv, heads, chunks, seed=0, use_q=True):
    """chunks: (first slot in its block, tokens) of each sequence.  Every block's first slots hold tokens already where a
    chunk does not begin it."""
    g = torch.Generator().manual_seed(seed)
    total = [at + n for at, n in chunks]
    c = Cache8(total, n_kv, hd, block, kind, cuda, layout=layout, seed=seed, garbage=False)
    slots, pos, rows = [], [], sum(n for _, n in chunks)
    for b, (at, n) in enumerate(chunks):
        for i in range(at, at + n):
            slots.append(int(c.tables[b, i // block]) * block + i % block)
            pos.append(i)
    slots, pos = torch.tensor(slots, device=cuda), torch.tensor(pos, dtype=torch.int32, device=cuda)
    amp = torch.exp2(torch.randint(-2, 3, (rows, 1, 1), generator=g).float())
    qkv = (torch.randn(rows, heads + 2 * n_kv, hd, generator=g) * amp).to(dtype).to(cuda)
    q, k, v = qkv.split([heads, n_kv, n_kv], dim=1)
    before, scales_before = c.values(), [s.clone() for s in c.scales]
    raw = [bits(x).clone() for x in (c.k, c.v)]
    rope = dkv.RotaryEmbedding(hd, max(total) + 1, rotary_dim=rot, interleaved=interleaved) if rot else None
    got = dkv.append_into_paged(k, v, c.k, c.v, slots, q=q if rope and use_q else None, positions=pos if rope else None, rope=rope,
                                kv_scales=c.scales, check=True)
    want_k, want_q = k.double(), q.double()
    if rope:
        cos, sin = (t[:, :rot // 2].to(cuda).double() for t in (rope.cos_cached, rope.sin_cached))
        want_k, want_q = (turned(t, cos, sin, pos, rot, interleaved) for t in (want_k, want_q))
        if use_q:
            tol = torch.finfo(dtype).eps / 2 * want_q.abs() + 2.0 ** -22 * q.double().abs().amax(-1, keepdim=True) + 1e-7
            assert torch.all((got.double() - want_q).abs() <= tol)
        else:
            assert got is None
    slack = 2.0 ** -22 * k.double().abs().amax(-1, keepdim=True)
    check_stored(c, 0, want_k, slots, slack if rope else 0)
    check_stored(c, 1, v.double(), slots, 0)
    # scales and what else the blocks hold
    written = torch.zeros(c.k.shape[0], block, dtype=torch.bool, device=cuda)
    written[slots // block, slots % block] = True
    touched, begun = written.any(1), written[:, 0]
    for side, x in ((0, want_k), (1, v.double())):
        scale, old = c.scales[side].double(), scales_before[side].double()
        top = torch.zeros_like(scale).index_reduce_(0, slots // block, x.abs().amax(-1), "amax")
        assert torch.equal(scale[~touched], old[~touched])
        fresh = first_scale(top, kind)
        rel = (scale / torch.where(fresh > 0, fresh, 1.0) - 1).abs()
        if kind == I8 or side == 1:  # a rotated e4m3 maximum may lie across a power of two by its rounding
            assert torch.all(rel[begun] <= 2.0 ** -20)
        else:
            assert torch.all((rel[begun] <= 2.0 ** -20) | (rel[begun] == 1.0) | (rel[begun] == 0.5)) and (rel[begun] > 0.1).sum() < 2
        grown = touched & ~begun
        ratio = scale[grown] / old[grown]
        fits = 448.0 if kind == E4M3 else 127.5
        assert torch.all(power_of_two(ratio)) and torch.all(ratio >= 1)
        assert torch.all(top[grown] <= fits * scale[grown] * (1 + 2.0 ** -20))
        assert torch.all((ratio == 1) | (top[grown] > fits * scale[grown] / 2 * (1 - 2.0 ** -20)))
        now, was, pages = c.values()[side], before[side], bits((c.k, c.v)[side])
        kept = ~written & grown[:, None]
        step = scale[:, None, :, None] * torch.ones_like(now)
        off = (now - was).abs()
        again = half_step(was, step, kind) if kind == I8 else 2.0 ** -10 * step
        same = (scale == old)[:, None, :, None] & torch.ones_like(now, dtype=torch.bool)
        assert torch.all((off <= again * (1 + 2.0 ** -20))[kept]) and torch.all((off == 0)[kept & same.all(-1).all(-1)])
        alone = ~written & ~grown[:, None]
        assert torch.equal(pages[alone], raw[side][alone])


APPENDS = [
    dict(hd=128, rot=128, interleaved=False, block=16, layout="kv_first", n_kv=8, heads=32, chunks=[(5, 1), (0, 1), (15, 1), (3, 50)]),
    dict(hd=64, rot=32, interleaved=True, block=16, layout="block_first", n_kv=3, heads=9, chunks=[(0, 100), (7, 1), (9, 23), (16, 1)]),
    dict(hd=256, rot=64, interleaved=False, block=8, layout="kv_first", n_kv=2, heads=4, chunks=[(0, 9), (3, 3), (7, 2)]),
    dict(hd=96, rot=96, interleaved=True, block=24, layout="heads", n_kv=5, heads=5, chunks=[(0, 24), (1, 47), (23, 1)]),
    dict(hd=80, rot=40, interleaved=False, block=128, layout="kv_first", n_kv=1, heads=7, chunks=[(0, 300), (100, 5), (64, 64)]),
    dict(hd=50, rot=20, interleaved=True, block=16, layout="odd", n_kv=2, heads=6, chunks=[(0, 16), (2, 40), (5, 1)]),
    dict(hd=33, rot=0, interleaved=False, block=1, layout="odd", n_kv=3, heads=3, chunks=[(0, 5), (3, 1)]),
    dict(hd=128, rot=0, interleaved=False, block=1024, layout="kv_first", n_kv=1, heads=1, chunks=[(0, 1500), (1000, 30), (5, 700)]),
    dict(hd=32, rot=32, interleaved=False, block=7, layout="kv_first", n_kv=4, heads=4, chunks=[(i % 9, 1 + i % 5) for i in range(60)]),
    dict(hd=16, rot=16, interleaved=False, block=16, layout="kv_first", n_kv=2, heads=2, chunks=[(i % 16, 1) for i in range(3000)]),
]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", range(len(APPENDS)))
def test_append(cuda, kind, dtype, case):
    append_case(cuda, kind, dtype, seed=case, use_q=case % 3 != 1, **APPENDS[case])


@pytest.mark.parametrize("kind", KINDS)
def test_append_token_by_token(cuda, kind):
    """One token a call, growing and shrinking by turns, zeros first: everything held stays within the rounding it had."""
    n_kv, hd, block = 3, 64, 16
    pages = torch.full((2, 3, block, n_kv, hd), 0x7F, dtype=torch.uint8, device=cuda).view(kind)  # garbage
    scales = torch.full((2, 3, n_kv), math.nan, device=cuda)
    g = torch.Generator(device=cuda).manual_seed(3)
    held, worst = [], torch.zeros(n_kv, dtype=F64, device=cuda)
    for i in range(40):
        amp = [0.0, 0.0, 1e-3, 1.0, 0.5, 3.0, 100.0, 1e-5, 1.0, 1e4, 2.0, 0.0, 1e-30, 7e4, 1.0, 1.0][i % block]
        x = amp * torch.randn(1, n_kv, hd, device=cuda, generator=g)
        held.append(x.double())
        slot = torch.tensor([i // block * 16 + i % block + block], device=cuda)
        slot = torch.where(slot >= 3 * block, slot - 3 * block, slot)
        dkv.append_into_paged(x, 2 * x, pages[0], pages[1], slot, kv_scales=(scales[0], scales[1]), check=True)
        block_id, first = int(slot) // block, i - i % block
        for side, by in ((0, 1.0), (1, 2.0)):
            s = scales[side, block_id].double()
            got = bits(pages)[side, block_id, : i % block + 1].view(kind).double() * s[None, :, None]
            want = by * torch.cat(held[first:])
            step = s[None, :, None]
            tol = step * (1 + 2.0 ** -20) if kind == I8 else half_step(want, step, kind) * (1 + 2.0 ** -18) + step * 2.0 ** -9
            assert torch.all((got - want).abs() <= tol), (i, side)
            top = want.abs().amax((0, 2))
            assert torch.all(s * (448 if kind == E4M3 else 127.5) * (1 + 2.0 ** -20) >= top)
            assert torch.all(s <= 2 * first_scale(top, kind) * (1 + 2.0 ** -20))


@pytest.mark.parametrize("kind", KINDS)
def test_append_of_what_is_not_finite(cuda, kind):
    c = Cache8([40, 40], 2, 64, 16, kind, cuda)
    before = [s.clone() for s in c.scales]
    raw = bits(c.v).clone()
    slots = torch.tensor([int(c.tables[0, 0]) * 16 + 3, -1, int(c.tables[1, 2]) * 16 + 7], device=cuda)
    k = torch.randn(3, 2, 64, device=cuda)
    k[1], v = math.nan, k.clone()  # a padding row holds anything
    k[2, 1, 5], v[0, 0, 63] = math.inf, math.nan
    dkv.append_into_paged(k, v, c.k, c.v, slots, kv_scales=c.scales, check=True)
    b0, b2 = int(c.tables[0, 0]), int(c.tables[1, 2])
    assert torch.isnan(c.scales[0][b2, 1]) and torch.isnan(c.scales[1][b0, 0])
    for side, b, h in ((0, b0, 0), (0, b0, 1), (0, b2, 0), (1, b0, 1), (1, b2, 0), (1, b2, 1)):
        assert c.scales[side][b, h] >= before[side][b, h]
    others = [i for i in range(c.k.shape[0]) if i not in (b0, b2)]
    assert torch.equal(bits(c.v)[others], raw[others])
    # it stays so for later tokens, until the block begins anew
    one = torch.randn(1, 2, 64, device=cuda)
    dkv.append_into_paged(one, one, c.k, c.v, slots[2:] + 1, kv_scales=c.scales)
    assert torch.isnan(c.scales[0][b2, 1])
    dkv.append_into_paged(one, one, c.k, c.v, torch.tensor([b2 * 16], device=cuda), kv_scales=c.scales)
    check_stored(c, 0, one.double(), torch.tensor([b2 * 16], device=cuda), 0)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [BF, F32])
def test_append_ranges(cuda, kind, dtype):
    """Slots beyond the cache and positions beyond the tables store nothing and are recorded; scales stay."""
    c = Cache8([100], 2, 64, 16, kind, cuda, garbage=False)
    cos, sin = torch.randn(50, 32, device=cuda), torch.randn(50, 32, device=cuda)
    k = torch.randn(5, 2, 64, device=cuda).to(dtype)
    q, out = torch.randn(5, 4, 64, device=cuda).to(dtype), torch.full((5, 4, 64), 3.0, dtype=dtype, device=cuda)
    n = c.k.shape[0] * 16
    slots = torch.tensor([n, 1 << 40, (1 << 32) + 5, 5, 6], device=cuda)
    pos = torch.tensor([1, 2, 3, 50, -1], dtype=torch.int32, device=cuda)
    before = [x.clone() for x in (bits(c.k), bits(c.v), *c.scales)]
    with pytest.raises(dkv.DkvError):
        dkv.append_into_paged(k, k, c.k, c.v, slots, q=q, q_out=out, positions=pos, rope=(cos, sin), kv_scales=c.scales, check=True)
    for x, y in zip(before, (bits(c.k), bits(c.v), *c.scales)):
        assert torch.equal(x, y)
    assert torch.all(out[3:] == 3.0) and not torch.any(torch.all(out[:3] == 3.0, -1))
    empty = dkv.append_into_paged(k[:0], k[:0], c.k, c.v, slots[:0], kv_scales=c.scales)
    assert empty is None
    with pytest.raises(ValueError, match="do not cover rotary_dim 32"):
        dkv.append_into_paged(k, k, c.k, c.v, slots, positions=pos, rope=(cos, sin), rotary_dim=32, kv_scales=c.scales)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd", [64, 50])
def test_append_keeps_the_slot_of_a_row_that_stores_nothing(cuda, kind, hd):
    """A row among others of its block whose position lies beyond the tables: its slot's value stays where the scale grows."""
    c = Cache8([20], 2, hd, 16, kind, cuda, garbage=False, layout="kv_first" if hd == 64 else "odd")
    block = int(c.tables[0, 0])
    slots = block * 16 + torch.tensor([6, 7, 8, 9], device=cuda)
    pos = torch.tensor([6, 50, 8, -1], dtype=torch.int32, device=cuda)
    angle = torch.outer(torch.arange(50.0), torch.rand(hd // 2)).to(cuda)
    before, scales_before = c.values(), [x.clone() for x in c.scales]
    k = 1000.0 * torch.randn(4, 2, hd, device=cuda)
    with pytest.raises(dkv.DkvError):
        dkv.append_into_paged(k, k, c.k, c.v, slots, positions=pos, rope=(angle.cos(), angle.sin()), kv_scales=c.scales, check=True)
    kept = [i for i in range(16) if i not in (6, 8)]
    for now, was, scale, old in zip(c.values(), before, c.scales, scales_before):
        assert torch.all(scale[block] > old[block])
        step = scale[block].double()[None, :, None] * torch.ones_like(was[block, kept])
        again = half_step(was[block, kept], step, kind) if kind == I8 else 2.0 ** -10 * step  # (kept codes are rounded once more)
        assert torch.all((now[block, kept] - was[block, kept]).abs() <= again * (1 + 2.0 ** -20))


# ---------------------------------------------------------------------------------------
# reading back and patching
# ---------------------------------------------------------------------------------------
READS = [
    dict(lens=[333], n_kv=3, hd=64, block=16, layout="block_first"),
    dict(lens=[1, 0, 17, 0, 0, 16, 200, 0], n_kv=8, hd=128, block=16, layout="kv_first"),
    dict(lens=[5, 40, 1], n_kv=2, hd=50, block=7, layout="odd"),
    dict(lens=[0, 0], n_kv=2, hd=32, block=8, layout="kv_first"),
    dict(lens=[2500, 1, 90], n_kv=4, hd=96, block=128, layout="heads"),
    dict(lens=[7000, 5000, 300], n_kv=1, hd=256, block=24, layout="kv_first"),
    dict(lens=[(i * 37) % 50 for i in range(300)], n_kv=2, hd=16, block=1, layout="kv_first"),
]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", range(len(READS)))
def test_gather(cuda, kind, dtype, case):
    """Code times scale in fp32, rounded once: bit for bit."""
    c = Cache8(kind=kind, dev=cuda, seed=case, **READS[case])
    rows = sum(c.lens)
    want = torch.cat([c.tokens(b)[0] for b in range(len(c.lens))]).float().to(dtype)
    # (a product of an 8-bit and a 24-bit number is exact in fp64 and rounded once to fp32, as the kernel's)
    got = dkv.gather_from_paged_batched(c.k, c.seqs(), rows, page_scales=c.scales[0], dtype=dtype, check=True)
    assert got.dtype == dtype and torch.equal(got, want)
    more = dkv.gather_from_paged_batched(c.v, c.seqs(), rows + 37, page_scales=c.scales[1], dtype=dtype)
    want = torch.cat([c.tokens(b)[1] for b in range(len(c.lens))]).float().to(dtype)
    assert torch.equal(more[:rows], want) and torch.all(more[rows:] == 0)
    n_kv, hd = c.k.shape[2:]
    out = torch.full((rows + 5, n_kv + 1, hd + 1), 9.0, dtype=dtype, device=cuda)
    view = out[:, 1:, 1:] if case % 2 else out[:, :n_kv, :hd]
    assert dkv.gather_from_paged_batched(c.v, c.seqs(), rows + 5, page_scales=c.scales[1], out=view) is view
    assert torch.equal(view[:rows], want) and torch.all(view[rows:] == 9.0)
    edge = out.clone()
    (edge[:, 1:, 1:] if case % 2 else edge[:, :n_kv, :hd])[:rows] = 9.0
    assert torch.all(edge == 9.0)


@pytest.mark.parametrize("kind", KINDS)
def test_gather_and_scatter_ranges(cuda, kind):
    c = Cache8([40, 20, 33], 2, 64, 16, kind, cuda)
    scale = c.scales[0]
    lens = torch.tensor([3, 1, 3], dtype=torch.int32, device=cuda)  # the second table is a block short
    seqs = c.seqs(table_lens=lens)
    want = torch.cat([c.tokens(b)[0] for b in range(3)]).float()
    want[56:60] = 0
    with pytest.raises(dkv.DkvError, match="block_table shorter"):
        dkv.gather_from_paged_batched(c.k, seqs, 93, page_scales=scale, check=True)
    assert torch.equal(dkv.gather_from_paged_batched(c.k, seqs, 93, page_scales=scale), want)
    ops.status_word(cuda).t.zero_()
    c.tables[2, 1], c.tables[0, 0] = 1000, -7
    want[0:16], want[76:92] = 0, 0
    with pytest.raises(dkv.DkvError):
        dkv.gather_from_paged_batched(c.k, seqs, 93, page_scales=scale, check=True)
    got = dkv.gather_from_paged_batched(c.k, seqs, 93, page_scales=scale)
    assert torch.equal(got, want)
    ops.status_word(cuda).t.zero_()
    # fewer rows than the lengths say: those there are, and a record
    with pytest.raises(dkv.DkvError):
        dkv.gather_from_paged_batched(c.k, seqs, 50, page_scales=scale, check=True)
    assert torch.equal(dkv.gather_from_paged_batched(c.k, seqs, 50, page_scales=scale), want[:50])
    ops.status_word(cuda).t.zero_()
    raw, before = bits(c.k).clone(), scale.clone()
    delta = torch.randn(50, 2, 64, device=cuda)
    with pytest.raises(dkv.DkvError):
        dkv.scatter_into_paged_batched(delta, c.k, seqs, page_scales=scale, check=True)
    ops.status_word(cuda).t.zero_()
    touched = [int(c.tables[0, 1]), int(c.tables[0, 2]), int(c.tables[1, 0])]
    others = [i for i in range(c.k.shape[0]) if i not in touched]
    assert torch.equal(bits(c.k)[others], raw[others]) and torch.equal(scale[others].nan_to_num(7), before[others].nan_to_num(7))
    assert not torch.equal(bits(c.k)[touched], raw[touched])
    # and nothing at all
    none = dkv.SeqBatchTensors(cu_seqlens=torch.zeros(1, dtype=torch.int32, device=cuda),
                               block_tables=torch.zeros(0, 1, dtype=torch.int32, device=cuda), max_seq_len=0)
    assert dkv.gather_from_paged_batched(c.k, none, 0, page_scales=scale).shape == (0, 2, 64)
    assert torch.all(dkv.gather_from_paged_batched(c.k, none, 3, page_scales=scale, check=True) == 0)
    dkv.scatter_into_paged_batched(delta[:0], c.k, none, page_scales=scale, check=True)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", range(len(READS)))
def test_scatter(cuda, kind, dtype, case):
    c = Cache8(kind=kind, dev=cuda, seed=case, garbage=False, **READS[case])
    if not sum(c.lens):
        return
    g = torch.Generator(device=cuda).manual_seed(case)
    n_kv, hd = c.k.shape[2:]
    delta = torch.randn(sum(c.lens), n_kv, hd, device=cuda, generator=g).to(dtype)
    was, old, raw = c.values()[0], c.scales[0].clone().double(), bits(c.k).clone()
    dkv.scatter_into_paged_batched(delta, c.k, c.seqs(), page_scales=c.scales[0], check=True)
    now, scale = c.values()[0], c.scales[0].double()
    want, count = was.clone(), torch.zeros(c.k.shape[0], dtype=torch.long, device=cuda)
    at = 0
    for b, n in enumerate(c.lens):
        for i in range(0, n, c.block):
            m, blk = min(c.block, n - i), int(c.tables[b, i // c.block])
            want[blk, :m] += delta[at + i: at + i + m].double()
            count[blk] = m
        at += n
    slot = torch.arange(c.block, device=cuda)
    stored = slot[None] < count[:, None]
    full, part = count == c.block, (count > 0) & (count < c.block)
    top = (want.abs() * stored[..., None, None]).amax((1, 3))
    rel = (scale / first_scale(top, kind) - 1).abs()
    near = rel <= 2.0 ** -20
    if kind == E4M3:  # the maximum may lie across a power of two by its rounding
        near = near | (rel == 1.0) | (rel == 0.5)
        assert (rel[full] > 0.1).sum() < 2
    assert torch.all(near[full])
    ratio, fits = scale[part] / old[part], 448.0 if kind == E4M3 else 127.5
    assert torch.all(power_of_two(ratio)) and torch.all(ratio >= 1)
    assert torch.all(top[part] <= fits * scale[part] * (1 + 2.0 ** -20))
    assert torch.all((ratio == 1) | (top[part] > fits * scale[part] / 2 * (1 - 2.0 ** -20)))
    step = scale[:, None, :, None] * torch.ones_like(now)
    # the product and the sum are rounded to fp32
    tol = half_step(want, step, kind) * (1 + 2.0 ** -20) + 2.0 ** -22 * (was.abs() + want.abs())
    assert torch.all(((now - want).abs() <= tol)[stored])
    again = (half_step(was, step, kind) if kind == I8 else 2.0 ** -10 * step) * (1 + 2.0 ** -20)
    rest = ~stored & part[:, None]
    assert torch.all(((now - was).abs() <= again)[rest])
    assert torch.equal(bits(c.k)[count == 0], raw[count == 0]) and torch.equal(scale[count == 0], old[count == 0])


@pytest.mark.parametrize("kind", KINDS)
def test_single_sequence_forms(cuda, kind):
    """The drop-ins with a Python block table, on the five-dimensional layouts."""
    g = torch.Generator(device=cuda).manual_seed(0)
    for lead, scales_of in (((2, 6), lambda s, i: s[i]), ((6, 2), lambda s, i: s[:, i])):
        cache = torch.zeros(*lead, 16, 2, 64, dtype=torch.uint8, device=cuda).view(kind)
        scales = torch.zeros(*lead, 2, device=cuda)
        delta = torch.randn(50, 2, 64, device=cuda, generator=g)
        table = [4, 0, -1, 2]
        dkv.scatter_into_paged(delta, cache, table, 16, kv_dim=1, page_scales=scales_of(scales, 1))
        got = dkv.gather_from_paged(cache, table, 50, 16, kv_dim=1, page_scales=scales_of(scales, 1))
        step = torch.cat([scales_of(scales, 1)[b][None].expand(16, 2) for b in table])[:50, :, None].double()
        assert got.dtype == F32
        assert torch.all((got.double() - delta.double()).abs() <= half_step(delta.double(), step, kind) * (1 + 2.0 ** -18))
        short = dkv.gather_from_paged(cache, table[:2], 50, 16, kv_dim=1, page_scales=scales_of(scales, 1), dtype=BF)
        assert torch.equal(short[:32], got[:32].to(BF)) and torch.all(short[32:] == 0)
        other = dkv.gather_from_paged(cache, table, 50, 16, kv_dim=0, page_scales=scales_of(scales, 0))
        assert torch.all(other == 0)
        assert dkv.gather_from_paged(cache, [], 3, 16, kv_dim=1, page_scales=scales_of(scales, 1)).abs().sum() == 0


# ---------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------
def check_attention(got, lse, q, tokens_of, scale):
    n, heads, hd = q.shape
    for b in range(n):
        k, v, big = tokens_of(b)
        if k.shape[0] == 0:
            assert torch.all(got[b] == 0), b
            assert lse is None or torch.all(lse[b] == -math.inf)
            continue
        kv = k.shape[1]
        qb = q[b].double().view(kv, heads // kv, hd)
        s = torch.einsum("ugd,nud->ugn", qb, k) * scale
        ds = (torch.einsum("ugd,nud->ugn", qb.abs(), k.abs()) * abs(scale)).amax(-1)
        ds = ds * ((hd + 12) * 2.0 ** -23 + (2.0 ** -21 if q.dtype == F32 else 0))
        ref_lse = torch.logsumexp(s, -1)
        p = torch.exp(s - ref_lse[..., None])
        ref = torch.einsum("ugn,nud->ugd", p, v)
        spread = torch.einsum("ugn,nud->ugd", p, v.abs())
        tol = torch.finfo(q.dtype).eps / 2 * ref.abs() + torch.finfo(q.dtype).smallest_normal * torch.finfo(q.dtype).eps
        tol = tol + spread * (2 * ds[..., None] + 2.0 ** -19 + k.shape[0] * 2.0 ** -24 + (2.0 ** -11 if q.dtype == BF else 2.0 ** -21))
        tol = tol + k.shape[0] * 2.0 ** -33 * (p * big.T[:, None]).amax(-1)[..., None]
        off = (got[b].double().view(kv, heads // kv, hd) - ref).abs()
        assert torch.all(off <= tol), (b, k.shape[0], float((off / tol).max()))
        if lse is not None:
            off = (lse[b].double().view(kv, heads // kv) - ref_lse).abs()
            tol = 2 * ds + k.shape[0] * 2.0 ** -24 + 2.0 ** -20 + 2.0 ** -22 * ref_lse.abs()
            assert torch.all(off <= tol), (b, float((off / tol).max()))


def run_attention(c, heads, dtype, dev, seed=1, scale=None, amp=1.5, bounds=None):
    g = torch.Generator().manual_seed(seed)
    hd = c.k.shape[3]
    q = (amp * torch.randn(len(c.lens), heads, hd, generator=g)).to(dtype).to(dev)
    for bound in bounds or (max(c.lens), 5000):  # short batches are joined within a CTA unless the bound is long
        out, lse = dkv.paged_decode_attention(q, c.k, c.v, c.seqs(bound), scale=scale, return_lse=True, check=True,
                                              kv_scales=c.scales)
        check_attention(out, lse, q, c.tokens, hd ** -0.5 if scale is None else scale)
    return q, out, lse


ATTENDS = [
    dict(lens=[333], n_kv=3, heads=9, hd=64, block=16, layout="block_first"),
    dict(lens=[1], n_kv=1, heads=1, hd=128, block=16, layout="kv_first"),
    dict(lens=[1, 0, 17, 0, 16, 15, 700, 2], n_kv=8, heads=32, hd=128, block=16, layout="kv_first"),
    dict(lens=[2000, 100, 1, 0], n_kv=2, heads=10, hd=128, block=32, layout="heads"),
    dict(lens=[50, 7, 300], n_kv=2, heads=16, hd=256, block=8, layout="kv_first"),
    dict(lens=[100, 9], n_kv=1, heads=12, hd=32, block=1, layout="kv_first"),
    dict(lens=[31, 333, 64], n_kv=4, heads=4, hd=96, block=24, layout="kv_first"),
    dict(lens=[31, 200, 5], n_kv=2, heads=6, hd=80, block=40, layout="block_first"),
    dict(lens=[31, 90, 5], n_kv=2, heads=4, hd=50, block=16, layout="odd"),
    dict(lens=[63, 20], n_kv=3, heads=3, hd=100, block=16, layout="kv_first"),
    dict(lens=[40, 18, 1], n_kv=1, heads=40, hd=33, block=7, layout="odd"),
    dict(lens=[9000, 1, 3000], n_kv=2, heads=4, hd=128, block=16, layout="kv_first"),
    dict(lens=[20, 20], n_kv=2, heads=4, hd=1, block=16, layout="kv_first"),
]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", range(len(ATTENDS)))
def test_attention(cuda, kind, dtype, case):
    a = dict(ATTENDS[case])
    heads = a.pop("heads")
    run_attention(Cache8(kind=kind, dev=cuda, seed=case, **a), heads, dtype, cuda)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n_seq", [40, 220, 900])
def test_attention_of_many_short(cuda, kind, dtype, n_seq):
    rng = random.Random(n_seq)
    c = Cache8([rng.choice([0, 1, 16, rng.randrange(70)]) for _ in range(n_seq)], 4, 64, 16, kind, cuda)
    g = torch.Generator().manual_seed(7)
    q = torch.randn(n_seq, 12, 64, generator=g).to(dtype).to(cuda)
    for bound in (70, 5000):
        out, lse = dkv.paged_decode_attention(q, c.k, c.v, c.seqs(bound), return_lse=True, check=True, kv_scales=c.scales)
        for b in rng.sample(range(n_seq), 16):
            check_attention(out[b:b + 1], lse[b:b + 1], q[b:b + 1], lambda _, b=b: c.tokens(b), 64 ** -0.5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", KINDS)
def test_attention_scales_that_differ_widely(cuda, kind, dtype):
    """V's scales from 2^-30 to 2^30 within a head (a zero one among them): neither the weights' range nor l may suffer.  K's
    scales are equal, so that scores stay ordinary."""
    c = Cache8([200, 30, 3000], 2, 64, 16, kind, cuda)
    g = torch.Generator().manual_seed(5)
    c.scales = (torch.full_like(c.scales[0], 2.0 ** -8),
                torch.exp2(torch.randint(-30, 31, c.scales[1].shape, generator=g).float()).to(cuda))
    c.scales[1][c.tables[0, 3].long(), 0] = 0.0
    c.scales[1][c.tables[1, 0].long()] = 0.0
    if dtype == F16:
        c.scales[1].mul_(2.0 ** -24)  # within the type
    run_attention(c, 8, dtype, cuda)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", TYPES)
def test_attention_small_weights_alone_meet_values(cuda, kind, dtype):
    """The heaviest tokens' values are zero (as is their scale), tokens of weight e^-80 give the result, and the weight of a
    token with large values is 0 in fp32.  Scores are exact products; the weight's exponent, 116 in base 2, is off by
    four roundings of 2^-24 of it (2^-15.5 of the weight), the f16 weight by 2^-11 for bf16 out (else 2^-22)."""
    c = Cache8([24], 2, 64, 8, kind, cuda, garbage=False)
    blocks = c.tables[0].long()
    codes = torch.zeros(c.k.shape, device=cuda)
    codes[blocks[1:], :, :, 0] = -1.0
    c.k = codes.to(kind)
    c.v = torch.randint(-9, 10, c.v.shape, device=cuda).float().to(kind)
    c.scales = tuple(torch.zeros_like(x) for x in c.scales)
    c.scales[0][blocks] = torch.tensor([1.0, 80.0, 200.0], device=cuda)[:, None]
    c.scales[1][blocks] = torch.tensor([0.0, 1.0, 1024.0], device=cuda)[:, None]
    q = torch.ones(1, 8, 64, device=cuda).to(dtype)
    k, v, _ = c.tokens(0)
    want = torch.einsum("tu,tud->ud", torch.softmax(k.sum(-1), 0), v).repeat_interleave(4, 0)
    tol = want.abs() * (torch.finfo(dtype).eps / 2 + 2.0 ** -15.5 + (2.0 ** -11 if dtype == BF else 2.0 ** -22))
    # the sum of a column may cancel: the weights' roundings count against the sum of magnitudes
    sizes = torch.einsum("tu,tud->ud", torch.softmax(k.sum(-1), 0), v.abs()).repeat_interleave(4, 0)
    tol = tol + sizes * (2.0 ** -15.5 + (2.0 ** -11 if dtype == BF else 2.0 ** -22)) + (2.0 ** -25 if dtype == F16 else 0)
    for bound in (24, 5000):
        out = dkv.paged_decode_attention(q, c.k, c.v, c.seqs(bound), scale=1.0, kv_scales=c.scales)
        assert torch.all((out[0].double() - want).abs() <= tol)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("amp", [1e-30, 1e-3, 40.0, 1e20])
def test_attention_q_of_any_size(cuda, dtype, amp):
    """q is scaled into f16's range by a power of two of each head; scale brings the scores back to ordinary ones."""
    if dtype == F16 and amp not in (1e-3, 40.0):
        return
    c = Cache8([100, 40], 2, 128, 16, E4M3, cuda)
    run_attention(c, 4, dtype, cuda, amp=amp, scale=0.05 / amp)


@pytest.mark.parametrize("kind", KINDS)
def test_attention_nan(cuda, kind):
    """A NaN code or scale of a token that counts: NaN where it enters, and nowhere else."""
    for dtype in TYPES:
        c = Cache8([100, 40, 60], 2, 64, 16, kind, cuda)
        q = torch.randn(3, 4, 64, device=cuda).to(dtype)
        clean = dkv.paged_decode_attention(q, c.k, c.v, c.seqs(), kv_scales=c.scales)
        assert not torch.any(torch.isnan(clean))
        c.scales[1][c.tables[1, 1].long(), 1] = math.nan
        c.scales[0][c.tables[2, 0].long(), 0] = math.nan
        expect = torch.zeros(3, 4, 64, dtype=torch.bool, device=cuda)
        expect[1, 2:], expect[2, :2] = True, True
        if kind == E4M3:
            bits(c.v)[c.tables[0, 2].long(), 3, 0, 17] = 0x7F
            expect[0, :2, 17] = True
        for bound in (100, 5000):
            got = dkv.paged_decode_attention(q, c.k, c.v, c.seqs(bound), kv_scales=c.scales)
            assert torch.equal(torch.isnan(got), expect)
            if bound == 100:
                assert torch.equal(got[~expect], clean[~expect])


@pytest.mark.parametrize("kind", KINDS)
def test_attention_bad_tables(cuda, kind):
    """Tokens of blocks outside the cache or beyond the table are left out and recorded."""
    c = Cache8([100, 50, 5], 2, 64, 16, kind, cuda)
    q = torch.randn(3, 4, 64, device=cuda).to(BF)
    c.tables[0, 2], c.tables[2, 0] = 1 << 20, -1
    lens = torch.tensor([7, 2, 1], dtype=torch.int32, device=cuda)

    def tokens(b):
        n, ok = c.lens[b], []
        for i in range(n):
            blk = i // 16
            if not (b == 0 and blk == 2) and not (b == 1 and blk >= 2) and b != 2:
                ok.append((int(c.tables[b, blk]), i % 16))
        ids, at = torch.tensor([x[0] for x in ok], dtype=torch.long), torch.tensor([x[1] for x in ok], dtype=torch.long)
        big = most(kind) * c.scales[1].cpu()[ids].double().to(cuda)
        return *(x.cpu()[ids, at].to(cuda) for x in c.values()), big

    for bound in (100, 5000):
        with pytest.raises(dkv.DkvError):
            dkv.paged_decode_attention(q, c.k, c.v, c.seqs(bound, table_lens=lens), kv_scales=c.scales, check=True)
        out, lse = dkv.paged_decode_attention(q, c.k, c.v, c.seqs(bound, table_lens=lens), kv_scales=c.scales, return_lse=True)
        ops.status_word(cuda).t.zero_()
        check_attention(out, lse, q, tokens, 64 ** -0.5)
    # a cache without blocks
    none = torch.zeros(0, 16, 2, 64, dtype=torch.uint8, device=cuda).view(kind)
    empty = torch.zeros(0, 2, device=cuda)
    out = dkv.paged_decode_attention(q, none, none.clone(), c.seqs(), kv_scales=(empty, empty.clone()))
    ops.status_word(cuda).t.zero_()
    assert torch.all(out == 0)


def test_attention_equals_that_over_the_values(cuda):
    """e4m3 codes times powers of two are exact in bf16: the 16-bit attention over the values read back says the same,
    within the weights' roundings; and parts attended apart join by lse."""
    c = Cache8([500, 77, 1300], 4, 128, 16, E4M3, cuda)
    q = torch.randn(3, 16, 128, device=cuda).to(BF)
    values = [(bits(x).contiguous().view(E4M3).float() * s.nan_to_num(1.0)[:, None, :, None]).nan_to_num(0.0).to(BF)
              for x, s in zip((c.k, c.v), c.scales)]
    a, la = dkv.paged_decode_attention(q, c.k, c.v, c.seqs(), kv_scales=c.scales, return_lse=True)
    b, lb = dkv.paged_decode_attention(q, *values, c.seqs(), return_lse=True)
    spread = max(float(v.float().abs().max()) for v in values)
    assert (a.float() - b.float()).abs().max() <= spread * (2 * 2.0 ** -8 + 2.0 ** -11) and (la - lb).abs().max() < 1e-4
    cut = torch.tensor([0, 256, 320, 576], dtype=torch.int32, device=cuda)  # the first 256, 64 and 256 tokens
    first = dkv.SeqBatchTensors(cu_seqlens=cut, block_tables=c.tables, max_seq_len=256)
    x, lx = dkv.paged_decode_attention(q, c.k, c.v, first, kv_scales=c.scales, return_lse=True)
    tails = [torch.cat([row[n // 16:], row[:n // 16]]) for row, n in zip(c.tables, (256, 64, 256))]
    rest = dkv.SeqBatchTensors(cu_seqlens=c.cu - cut, block_tables=torch.stack(tails), max_seq_len=1100)
    y, ly = dkv.paged_decode_attention(q, c.k, c.v, rest, kv_scales=c.scales, return_lse=True)
    both = torch.logaddexp(lx, ly)
    joined = x.float() * (lx - both).exp()[..., None] + y.float() * (ly - both).exp()[..., None]
    assert (both - la).abs().max() < 1e-4
    assert (joined - a.float()).abs().max() <= spread * (3 * 2.0 ** -8 + 2.0 ** -10)


def test_outputs_of_any_order_and_scale(cuda):
    c = Cache8([100, 40], 2, 64, 16, I8, cuda)
    for dtype in TYPES:
        whole = torch.randn(8, 2, 65, device=cuda).to(dtype)
        q = whole.transpose(0, 1)[:, :, 1:]  # heads before sequences, odd rows
        want = dkv.paged_decode_attention(q.contiguous(), c.k, c.v, c.seqs(), kv_scales=c.scales, scale=0.3)
        out = torch.zeros(8, 2, 67, dtype=dtype, device=cuda).transpose(0, 1)[:, :, 2:66]
        assert dkv.paged_decode_attention(q, c.k, c.v, c.seqs(), kv_scales=c.scales, scale=0.3, out=out) is out
        assert torch.equal(out, want)
        same = q.contiguous()
        assert dkv.paged_decode_attention(same, c.k, c.v, c.seqs(), kv_scales=c.scales, scale=0.3, out=same) is same
        assert torch.equal(same, want)


# ---------------------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------------------
class Server8:
    """A small serving loop on an 8-bit cache; keeps every token's K and V beside it."""

    def __init__(self, dev, kind, dtype=BF, n_req=5, heads=8, n_kv=2, hd=64, block=16, width=20, rows=64):
        self.dev, self.kind, self.dtype, self.heads, self.n_kv, self.hd, self.block = dev, kind, dtype, heads, n_kv, hd, block
        nb = n_req * width
        self.pages = torch.full((2, nb, block, n_kv, hd), 0x7F, dtype=torch.uint8, device=dev).view(kind)
        self.scales = torch.full((nb, 2, n_kv), math.nan, device=dev)
        self.kv_scales = (self.scales[:, 0], self.scales[:, 1])
        self.rope = dkv.RotaryEmbedding(hd, width * block, rotary_dim=hd // 2, interleaved=True)
        ints = lambda *s: torch.zeros(*s, dtype=torch.int32, device=dev)  # noqa: E731
        self.lengths, self.new, self.held, self.tables = ints(n_req), ints(n_req), ints(n_req), ints(n_req, width)
        self.free = torch.randperm(nb, generator=torch.Generator().manual_seed(0)).to(torch.int32).to(dev)
        self.rows, self.width = rows, width
        self.qkv = torch.zeros(rows, heads + 2 * n_kv, hd, dtype=dtype, device=dev)
        self.history = [[] for _ in range(n_req)]

    def step(self):
        q, k, v = self.qkv.split([self.heads, self.n_kv, self.n_kv], dim=1)
        p = dkv.plan_paged_step(self.lengths, self.tables, self.block, rows=self.rows, max_seq_len=self.width * self.block,
                                new_lengths=self.new, table_lens=self.held, free_blocks=self.free)
        turned_q = dkv.append_into_paged(k, v, self.pages[0], self.pages[1], p.slots, q=q, positions=p.positions, rope=self.rope,
                                         kv_scales=self.kv_scales)
        last = (p.cu_new[1:] - 1).clamp(min=0).long()
        out = dkv.paged_decode_attention(turned_q[last], self.pages[0], self.pages[1], p.seqs, kv_scales=self.kv_scales)
        return p, turned_q, last, out

    def fill(self, new, seed):
        g = torch.Generator().manual_seed(seed)
        amp = torch.exp2(torch.randint(-3, 4, (self.rows, 1, 1), generator=g).float())
        self.qkv.copy_((torch.randn(self.qkv.shape, generator=g) * amp).to(self.dtype))
        self.new.copy_(torch.tensor(new, dtype=torch.int32))
        self.lengths.add_(self.new)

    def check(self, p, turned_q, last, out, new):
        k, v = self.qkv[:, self.heads:self.heads + self.n_kv], self.qkv[:, self.heads + self.n_kv:]
        cos, sin = (t[:, : self.hd // 4].to(self.dev).double() for t in (self.rope.cos_cached, self.rope.sin_cached))
        k = turned(k.double(), cos, sin, p.positions, self.hd // 2, True)
        at = 0
        for b, n in enumerate(new):
            self.history[b] += [(k[at + i], v[at + i].double()) for i in range(n)]
            at += n
        for side in (0, 1):
            for b, held in enumerate(self.history):
                if not held:
                    continue
                want = torch.stack([x[side] for x in held])
                ids = p.seqs.block_tables[b, : -(-len(held) // self.block)].long()
                s = self.kv_scales[side][ids].double().repeat_interleave(self.block, 0)[: len(held), :, None]
                got = bits(self.pages)[side, ids].view(self.kind).double().reshape(-1, self.n_kv, self.hd)[: len(held)] * s
                tol = s * (1 + 2.0 ** -18) if self.kind == I8 else half_step(want, s, E4M3) * (1 + 2.0 ** -16) + s * 2.0 ** -9
                assert torch.all((got - want).abs() <= tol + 2.0 ** -22 * want.abs().amax(-1, keepdim=True)), (b, side)

        def tokens(b):
            n = len(self.history[b])
            ids = p.seqs.block_tables[b, : -(-n // self.block)].long()
            k, v = ((bits(self.pages)[i, ids].view(self.kind).double() * self.kv_scales[i][ids].double()[:, None, :, None])
                    .reshape(-1, self.n_kv, self.hd)[:n] for i in (0, 1))
            return k, v, most(self.kind) * self.kv_scales[1][ids].double().repeat_interleave(self.block, 0)[:n]

        check_attention(out, None, turned_q[last], tokens, self.hd ** -0.5)
        self.held.copy_(p.seqs.table_lens)
        self.free = self.free[int(p.blocks_used):]


STEPS = [[20, 1, 0, 33, 7], [1, 1, 1, 1, 1], [1, 0, 30, 1, 9], [1, 1, 1, 1, 1], [1, 1, 1, 1, 1], [16, 15, 2, 1, 17]]


@pytest.mark.parametrize("kind", KINDS)
def test_serving_loop(cuda, kind):
    s = Server8(cuda, kind)
    for i, new in enumerate(STEPS):
        s.fill(new, i)
        s.check(*s.step(), new)
    # a patch of every token, and what is read back after it
    seqs = dkv.SeqBatchTensors(cu_seqlens=torch.nn.functional.pad(s.lengths.cumsum(0), (1, 0)).int(), block_tables=s.tables,
                               max_seq_len=320)
    rows = int(s.lengths.sum())
    delta = 0.1 * torch.randn(rows, s.n_kv, s.hd, device=cuda)
    for side in (0, 1):
        was = dkv.gather_from_paged_batched(s.pages[side], seqs, rows, page_scales=s.kv_scales[side], check=True)
        dkv.scatter_into_paged_batched(delta, s.pages[side], seqs, page_scales=s.kv_scales[side], check=True)
        now = dkv.gather_from_paged_batched(s.pages[side], seqs, rows, page_scales=s.kv_scales[side], check=True)
        want = was.double() + delta.double()
        top = s.kv_scales[side][s.tables[s.tables >= 0].long()].nan_to_num(0).max().double()
        assert torch.all((now.double() - want).abs() <= half_step(want, top, kind) + 2.0 ** -20 * want.abs())


@pytest.mark.parametrize("kind", KINDS)
def test_captured_step(cuda, kind):
    """A step captured once, replayed with other lengths, values and a growing cache, beside eager steps of a twin."""
    s, twin = Server8(cuda, kind), Server8(cuda, kind)
    for x in (s, twin):
        x.fill(STEPS[0], 0)
        x.check(*x.step(), STEPS[0])
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    free = torch.full((s.free.numel(),), -1, dtype=torch.int32, device=cuda)  # of the captured call
    free.copy_(s.free)
    s.free = free
    lengths = s.lengths.clone()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        got = s.step()
    s.lengths.copy_(lengths)
    for i, new in enumerate(STEPS[1:], 1):
        s.fill(new, i), twin.fill(new, i)
        graph.replay()
        want = twin.step()
        torch.cuda.synchronize()
        assert torch.equal(got[3], want[3])
        twin.check(*want, new)
        s.held.copy_(got[0].seqs.table_lens)
        used = int(got[0].blocks_used)
        free.copy_(torch.cat([free[used:], free[:used]]))
    assert torch.equal(bits(s.pages), bits(twin.pages))
    assert torch.equal(s.scales.nan_to_num(-1), twin.scales.nan_to_num(-1))


def test_other_streams(cuda):
    """Operators on a stream of their own, their inputs made on it, while the default stream works."""
    c = Cache8([300, 50], 2, 64, 16, E4M3, cuda)
    q = torch.randn(2, 4, 64, device=cuda).to(BF)
    want = dkv.paged_decode_attention(q, c.k, c.v, c.seqs(), kv_scales=c.scales)
    back = dkv.gather_from_paged_batched(c.k, c.seqs(), 350, page_scales=c.scales[0])
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    busy = torch.randn(4096, 4096, device=cuda)
    for _ in range(5):
        busy = busy @ busy * 1e-3
        with torch.cuda.stream(side):
            got = dkv.paged_decode_attention(q + 0, c.k, c.v, c.seqs(), kv_scales=c.scales)
            read = dkv.gather_from_paged_batched(c.k, c.seqs(), 350, page_scales=c.scales[0])
        side.synchronize()
        assert torch.equal(got, want) and torch.equal(read, back)


def test_offsets_beyond_32_bits(cuda):
    """Blocks more than 2^32 bytes from the base, in a pool of 4.4 GB."""
    nb, block, n_kv, hd = 17000, 16, 64, 256
    pages = torch.zeros(nb, block, n_kv, hd, dtype=torch.uint8, device=cuda).view(E4M3)
    scales = torch.zeros(nb, n_kv, device=cuda)
    assert pages.numel() > 2 ** 32
    last = nb - 1
    x = torch.randn(20, n_kv, hd, device=cuda)
    seqs = dkv.SeqBatchTensors(cu_seqlens=torch.tensor([0, 20], dtype=torch.int32, device=cuda),
                               block_tables=torch.tensor([[last, 1]], dtype=torch.int32, device=cuda), max_seq_len=20)
    dkv.scatter_into_paged_batched(x, pages, seqs, page_scales=scales, check=True)
    got = dkv.gather_from_paged_batched(pages, seqs, 20, page_scales=scales, check=True)
    top = scales[[last, 1]].max()
    assert torch.all((got - x).abs() <= half_step(x, top, E4M3) * (1 + 2.0 ** -18))
    other = torch.zeros(nb, block, n_kv, hd, dtype=torch.uint8, device=cuda).view(E4M3)
    slots = torch.cat([torch.arange(16, device=cuda) + last * 16, torch.arange(4, device=cuda) + 16])
    dkv.append_into_paged(x, x, other, pages, slots, kv_scales=(torch.zeros_like(scales), scales), check=True)
    assert torch.equal(bits(other)[last], bits(pages)[last]) and torch.equal(bits(other)[1, :4], bits(pages)[1, :4])
    q = torch.randn(1, n_kv, hd, device=cuda).to(BF)
    near = dkv.SeqBatchTensors(cu_seqlens=seqs.cu_seqlens, block_tables=torch.tensor([[0, 1]], dtype=torch.int32, device=cuda),
                               max_seq_len=20)
    small, small_s = bits(pages)[[last, 1]].view(E4M3), scales[[last, 1]]
    want = dkv.paged_decode_attention(q, small, small.clone(), near, kv_scales=(small_s, small_s.clone()))
    far = dkv.paged_decode_attention(q, pages, other, seqs, kv_scales=(scales, scales.clone()), check=True)
    assert torch.equal(want, far)
