"""The weights of the attention over 8-bit pages, against plain implementations in 64 bits: values that cancel, and V's scales that
are zero for whole tiles."""

from __future__ import annotations

import pytest
import torch

import deltakv_b200 as dkv
from tests.test_gpu_quant import E4M3, F16, KINDS, TYPES, Cache8, run_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", TYPES)
def test_weights_of_values_that_cancel(cuda, kind, dtype):
    """Two tokens of nearly equal weight and opposite values: out is tanh of half the scores' difference, far below the
    values, and the weights' rounding shows whole.

    Scores are one exact product each (at most 2.1, so 3.1 in base 2): four roundings of 2^-24 of that are 2^-20.4 of a weight, exp 2^-22,
    the weight as two f16 terms 2^-22, sums and quotient 2^-22: together below 2^-19 of the sum of magnitudes, 1."""
    n = 64
    lo, hi, most = (96.0, 104.0, 0.02) if kind == E4M3 else (100.0, 101.0, 0.02)
    c = Cache8([2] * n, 2, 64, 16, kind, cuda, garbage=False)
    first = c.tables[:, 0].long()
    k, v = torch.zeros(c.k.shape, device=cuda), torch.ones(c.v.shape, device=cuda)
    k[first, 0, :, 0], k[first, 1, :, 0] = lo, hi
    v[first, 0] = -1.0
    c.k, c.v = k.to(kind), v.to(kind)
    g = torch.Generator().manual_seed(2)
    difference = 0.004 + (most - 0.004) * torch.rand(c.scales[0].shape, generator=g)
    c.scales = ((difference / (hi - lo)).to(cuda), torch.ones_like(c.scales[1]))
    q = torch.ones(n, 8, 64, device=cuda).to(dtype)
    want = torch.tanh(c.scales[0][first].double() * (hi - lo) / 2).repeat_interleave(4, 1)[..., None]
    tol = torch.finfo(dtype).eps / 2 * want.abs() + 2.0 ** -19
    for bound in (2, 5000):
        out = dkv.paged_decode_attention(q, c.k, c.v, c.seqs(bound), scale=1.0, kv_scales=c.scales, check=True)
        off = (out.double() - want).abs()
        assert torch.all(off <= tol), float((off / tol).max())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("span", [32, 512])
@pytest.mark.parametrize("later", [-6, -12, -20])
def test_tiles_whose_v_scales_are_zero(cuda, kind, dtype, span, later):
    """Spans of tokens with V scales of 0 (as append stores zero rows) come first, and their scores are the larger ones; what
    counts are the small V scales behind them.  Spans of 512 tokens: the first tile of each of up to 16 warps of a CTA."""
    c = Cache8([1000, 1100, 96, 40], 2, 64, 32, kind, cuda, seed=span)
    k_scales, v_scales = (torch.full_like(s, x) for s, x in zip(c.scales, (2.0 ** -9, 2.0 ** later)))
    for b, n in enumerate(c.lens):
        for i in range(0, n, 32):
            if i // span % 2 == 0:
                block = int(c.tables[b, i // 32])
                v_scales[block] = 0.0
                k_scales[block] = 2.0 ** -8
    c.scales = (k_scales, v_scales)
    _, out, _ = run_attention(c, 8, dtype, cuda, amp=3.0)
    assert torch.all(out[0].abs().amax(-1) > 0)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", TYPES)
def test_small_weights_behind_a_tile_of_zero_values(cuda, kind, dtype):
    """The heaviest 32 tokens' values are zero (as is their scale), the 32 behind them, of weight e^-80, give the result; the last
    32 have large values and a weight of 0 in fp32.  Scores are exact products; the weight's exponent, 116 in base 2, is off by
    four roundings of 2^-24 of it (2^-15.5 of the weight), the weight as two f16 terms by 2^-22."""
    c = Cache8([96], 2, 64, 32, kind, cuda, garbage=False)
    blocks = c.tables[0].long()
    codes = torch.zeros(c.k.shape, device=cuda)
    codes[blocks, :, :, 0] = -1.0
    c.k = codes.to(kind)
    c.v = torch.randint(-9, 10, c.v.shape, device=cuda).float().to(kind)
    c.scales = tuple(torch.zeros_like(x) for x in c.scales)
    c.scales[0][blocks] = torch.tensor([0.0, 80.0, 200.0], device=cuda)[:, None]
    c.scales[1][blocks] = torch.tensor([0.0, 1.0, 1024.0], device=cuda)[:, None]
    q = torch.ones(1, 8, 64, device=cuda).to(dtype)
    k, v, _ = c.tokens(0)
    p = torch.softmax(k.sum(-1), 0)
    want = torch.einsum("tu,tud->ud", p, v).repeat_interleave(4, 0)
    sizes = torch.einsum("tu,tud->ud", p, v.abs()).repeat_interleave(4, 0)
    tol = want.abs() * torch.finfo(dtype).eps / 2 + sizes * (2.0 ** -15.5 + 2.0 ** -22) + (2.0 ** -25 if dtype == F16 else 0)
    for bound in (96, 5000):
        out = dkv.paged_decode_attention(q, c.k, c.v, c.seqs(bound), scale=1.0, kv_scales=c.scales)
        assert torch.all((out[0].double() - want).abs() <= tol), float(((out[0].double() - want).abs() / tol).max())
