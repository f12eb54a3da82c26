"""The weights of the attention over 8-bit pages, against plain implementations in 64 bits: values that cancel."""

from __future__ import annotations

import pytest
import torch

import deltakv_b200 as dkv
from tests.test_gpu_quant import E4M3, KINDS, TYPES, Cache8

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
