"""The scales that the stores into 8-bit pages choose, and steps of single rows in long blocks."""

from __future__ import annotations

import pytest
import torch

import deltakv_b200 as dkv
from tests.test_gpu_quant import BF, E4M3, F16, F32, KINDS, append_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", KINDS)
def test_first_scales_bit_for_bit(cuda, kind):
    """Of a block of which nothing is kept: amax times 1/127, each rounded to fp32, or the least power of two that amax / 448 does not
    pass; not below 2^-126, 0 for zeros."""
    blocks, block, n_kv, hd = 500, 4, 8, 16
    g = torch.Generator(device=cuda).manual_seed(0)
    x = torch.randn(blocks * block, n_kv, hd, device=cuda, generator=g)
    x *= torch.exp2(torch.randint(-40, 40, (x.shape[0], 1, 1), device=cuda, generator=g).float())
    top = x.view(blocks, block, n_kv, hd).abs().amax((1, 3))
    # next to the borders of e4m3's scales, and the smallest scale
    edge = 448.0 * torch.exp2(torch.arange(-8, 8, device=cuda).float())
    for i, e in enumerate(torch.stack([edge, torch.nextafter(edge, edge + 1), torch.nextafter(edge, edge - 1)]).flatten()):
        x[block * i: block * (i + 1), 0] = x[block * i: block * (i + 1), 0].clamp(-e / 2, e / 2)
        x[block * i, 0, 0] = top[i, 0] = e
    x[-block:, 1], top[-1, 1] = 1e-38, 1e-38
    x[-block:, 2], top[-1, 2] = 0.0, 0.0
    if kind == E4M3:
        m, e = torch.frexp(top)  # 448 is 0.875 2^9 (no division, whose rounding would matter at 448 2^n)
        want = torch.ldexp(torch.ones_like(top, dtype=torch.float64), e - 9 + (m > 0.875).int())
    else:
        want = (top.double() * (torch.tensor(1.0) / torch.tensor(127.0)).double().item()).float().double()  # (an exact product, rounded)
    want = torch.where(top > 0, want.clamp(min=2.0 ** -126), 0.0).float()
    pages = torch.zeros(2, blocks, block, n_kv, hd, dtype=torch.uint8, device=cuda).view(kind)
    scales = torch.full((2, blocks, n_kv), 3.0, device=cuda)
    dkv.append_into_paged(x, x, pages[0], pages[1], torch.arange(blocks * block, device=cuda), kv_scales=(scales[0], scales[1]),
                          check=True)
    assert torch.equal(scales[0], want) and torch.equal(scales[1], want)
    pages.view(torch.uint8).zero_(), scales.fill_(3.0)
    seqs = dkv.SeqBatchTensors(cu_seqlens=torch.tensor([0, blocks * block], dtype=torch.int32, device=cuda),
                               block_tables=torch.arange(blocks, dtype=torch.int32, device=cuda)[None], max_seq_len=blocks * block)
    dkv.scatter_into_paged_batched(x, pages[0], seqs, page_scales=scales[0], check=True)
    assert torch.equal(scales[0], want)


@pytest.mark.parametrize("dtype", [BF, F16])
def test_values_are_rounded_to_fp32_first(cuda, dtype):
    """Where code times scale lies so near a tie of the 16-bit type that fp32 makes it one, the value is the fp32 number's rounding."""
    g = torch.Generator().manual_seed(0)
    places = 8 if dtype == BF else 11
    code = torch.randint(-127, 128, (4_000_000,), generator=g)
    scale = 1e-2 * (1 + torch.rand(code.shape, generator=g))
    exact = code.double() * scale.double()
    m, e = torch.frexp(exact)
    once = torch.ldexp(torch.round(m * 2 ** places), e - places)  # (ties to even)
    want = (code.float() * scale).to(dtype)
    twice = torch.nonzero(want.double() != once)[:, 0][:64]
    assert len(twice) > 8
    pages = code[twice].to(torch.int8)[:, None, None, None].expand(-1, 8, 1, 32).contiguous().to(cuda)
    seqs = dkv.SeqBatchTensors(cu_seqlens=torch.tensor([0, 8 * len(twice)], dtype=torch.int32, device=cuda),
                               block_tables=torch.arange(len(twice), dtype=torch.int32, device=cuda)[None], max_seq_len=8 * len(twice))
    got = dkv.gather_from_paged_batched(pages, seqs, 8 * len(twice), page_scales=scale[twice][:, None].to(cuda), dtype=dtype, check=True)
    assert torch.equal(got.view(len(twice), 8, 32), want[twice][:, None, None].expand(-1, 8, 32).to(cuda))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("block,hd,layout", [(64, 128, "kv_first"), (1024, 64, "block_first"), (100, 50, "odd")])
def test_single_rows_in_long_blocks(cuda, kind, dtype, block, hd, layout):
    """A decode step whose rows, one a block, lie behind a block's 32nd slot, and whose scales grow: the slots of all 32-slot words
    keep their values."""
    chunks = [(at % block, 1) for at in (32, 33, 40, 63, 64, 95, 96, 31, 500, 992, 1023, 991, 99, 65, 5, 60)]
    append_case(cuda, kind, dtype, hd=hd, rot=0, interleaved=False, block=block, layout=layout, n_kv=3, heads=3, chunks=chunks, seed=block)
