"""One step of a paged cache (plan, append, attend) against plain implementations in 64 bits.

Tolerances, derived: an output is rounded once to its type, at most eps/2 of the value.  Before
that, fp32 arithmetic: a score is a product sum of head_dim terms, off by at most
(head_dim + 8) 2^-23 sum |q_d k_d| scale =: ds (a tensor core may truncate, hence 2^-23); an
error ds of the scores moves every weight by a relative 2 ds (it enters the numerator and the
sum).  Weights enter the output product to 2^-16 (as two 16-bit terms in 16-bit types), exp and
the running sums add 2^-20 and n 2^-24 for n tokens.  All of that is relative to
A = sum p |v| / sum p, the output without cancellation.
"""

from __future__ import annotations

import math
import random
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import deltakv_b200 as dkv
from deltakv_b200 import ops

pytestmark = pytest.mark.gpu

BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
TYPES = [BF, F16, F32]


class Cache:
    """Random pages of a layout, tables with shuffled blocks, and the tokens they hold."""

    def __init__(self, lens, n_kv, hd, block, dtype, dev, layout="kv_first", seed=0, fill=None, spare=3):
        g = torch.Generator().manual_seed(seed)
        need = [-(-n // block) for n in lens]
        nb = sum(need) + spare
        width = max(max(need, default=0), 1)
        self.lens, self.block = lens, block
        shape = (block, n_kv, hd)
        if layout == "kv_first":
            full = torch.randn(2, nb, *shape, generator=g).to(dtype)
            k, v = full[0], full[1]
        elif layout == "block_first":
            full = torch.randn(nb, 2, *shape, generator=g).to(dtype)
            k, v = full[:, 0], full[:, 1]
        elif layout == "odd":  # every stride padded, nothing aligned
            full = torch.randn(2, nb, block + 1, n_kv + 1, hd + 3, generator=g).to(dtype)
            k, v = full[0, :, 1:, 1:, 1:hd + 1], full[1, :, 1:, 1:, 1:hd + 1]
        else:  # heads before slots
            full = torch.randn(2, nb, n_kv, block, hd, generator=g).to(dtype)
            k, v = full[0].transpose(1, 2), full[1].transpose(1, 2)
        order = torch.randperm(nb, generator=g)
        tables = torch.zeros(max(len(lens), 1), width, dtype=torch.int32)
        used = torch.zeros(nb, block, dtype=torch.bool)
        at = 0
        for b, n in enumerate(need):
            tables[b, :n] = order[at:at + n]
            for i in range(n):
                used[order[at + i], : min(block, lens[b] - i * block)] = True
            at += n
        if fill is not None:  # what no token owns holds garbage
            k[~used], v[~used] = fill, fill
        self.used = used
        full = full.to(dev)
        if layout == "kv_first":
            self.k, self.v = full[0], full[1]
        elif layout == "block_first":
            self.k, self.v = full[:, 0], full[:, 1]
        elif layout == "odd":
            self.k, self.v = full[0, :, 1:, 1:, 1:hd + 1], full[1, :, 1:, 1:, 1:hd + 1]
        else:
            self.k, self.v = full[0].transpose(1, 2), full[1].transpose(1, 2)
        self.tables = tables.to(dev)
        cu = [0]
        for n in lens:
            cu.append(cu[-1] + n)
        self.cu = torch.tensor(cu, dtype=torch.int32, device=dev)

    def seqs(self, **kw):
        return dkv.SeqBatchTensors(cu_seqlens=self.cu, block_tables=self.tables, max_seq_len=max(self.lens, default=0), **kw)

    def tokens(self, b):
        n = self.lens[b]
        ids = self.tables[b, : -(-n // self.block)].long()
        take = lambda t: t[ids].reshape(-1, t.shape[2], t.shape[3])[:n]  # noqa: E731
        return take(self.k), take(self.v)


def check_attention(got, lse, q, tokens_of, scale):
    """Every sequence's output (and lse) against the definition in fp64."""
    n, heads, hd = q.shape
    for b in range(n):
        k, v = (t.double() for t in tokens_of(b))
        if k.shape[0] == 0:
            assert torch.all(got[b] == 0), b
            assert lse is None or torch.all(lse[b] == -math.inf)
            continue
        kv = k.shape[1]
        qb = q[b].double().view(kv, heads // kv, hd)
        s = torch.einsum("ugd,nud->ugn", qb, k) * scale
        ds = (hd + 8) * 2.0 ** -23 * (torch.einsum("ugd,nud->ugn", qb.abs(), k.abs()) * abs(scale)).amax(-1)
        ref_lse = torch.logsumexp(s, -1)
        p = torch.exp(s - ref_lse[..., None])
        ref = torch.einsum("ugn,nud->ugd", p, v)
        spread = torch.einsum("ugn,nud->ugd", p, v.abs())
        tol = torch.finfo(q.dtype).eps / 2 * ref.abs() + torch.finfo(q.dtype).smallest_normal * torch.finfo(q.dtype).eps
        tol = tol + spread * (2 * ds[..., None] + 2.0 ** -20 + k.shape[0] * 2.0 ** -24
                              + (2.0 ** -16 if q.dtype != F32 else 0))
        off = (got[b].double().view(kv, heads // kv, hd) - ref).abs()
        assert torch.all(off <= tol), (b, k.shape[0], float((off / tol).max()))
        if lse is not None:
            off = (lse[b].double().view(kv, heads // kv) - ref_lse).abs()
            tol = 2 * ds + k.shape[0] * 2.0 ** -24 + 2.0 ** -20 + 2.0 ** -22 * ref_lse.abs()
            assert torch.all(off <= tol), (b, float((off / tol).max()))


def run_attention(c, heads, hd, dtype, dev, seed=1, scale=None, amp=1.5):
    g = torch.Generator().manual_seed(seed)
    q = (amp * torch.randn(len(c.lens), heads, hd, generator=g)).to(dtype).to(dev)
    for bound in (max(c.lens), 5000):  # short batches are joined within a CTA unless the bound is long
        seqs = dkv.SeqBatchTensors(cu_seqlens=c.cu, block_tables=c.tables, max_seq_len=bound)
        out, lse = dkv.paged_decode_attention(q, c.k, c.v, seqs, scale=scale, return_lse=True, check=True)
        check_attention(out, lse, q, c.tokens, hd ** -0.5 if scale is None else scale)
    return q, out, lse


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n_seq", [16, 40, 100, 220, 600, 900])
def test_attention_one_launch_of_fewer_warps(cuda, dtype, n_seq):
    """More pairs of sequence and KV head than SMs: CTAs of 6, 4, 3, 2 or 1 warps, up to one a CTA."""
    rng = random.Random(n_seq)
    c = Cache([rng.choice([0, 1, 16, rng.randrange(70)]) for _ in range(n_seq)], 4, 64, 16, dtype, cuda)
    g = torch.Generator().manual_seed(7)
    q = torch.randn(n_seq, 12, 64, generator=g).to(dtype).to(cuda)
    out, lse = dkv.paged_decode_attention(q, c.k, c.v, c.seqs(), return_lse=True, check=True)
    for b in rng.sample(range(n_seq), 16):
        check_attention(out[b:b + 1], lse[b:b + 1], q[b:b + 1], lambda _, b=b: c.tokens(b), 64 ** -0.5)
    split = dkv.SeqBatchTensors(cu_seqlens=c.cu, block_tables=c.tables, max_seq_len=9000)
    other = dkv.paged_decode_attention(q, c.k, c.v, split)
    # both are within the derived tolerance of the exact result, here taken at its largest
    assert float((out.double() - other.double()).abs().max()) <= 2 * (torch.finfo(dtype).eps + 2.0 ** -15) * float(c.v.double().abs().max())


def test_attention_one_launch_of_every_number_of_warps(cuda):
    """As many pairs of sequence and KV head as leave each number of warps a CTA, down to one, and one more pair than
    has a warp each (that batch is split).  The sizes follow from the number of SMs."""
    sms = torch.cuda.get_device_properties(cuda).multi_processor_count
    g = torch.Generator().manual_seed(11)
    for dtype, warps in ((BF, 12), (F16, 12), (F32, 8)):  # head_dim 64; fp32: up to 4 heads a KV head
        seen = []
        for per_sm in (1, 2, 3, 4, warps // 2, warps, warps + 1):
            n = sms * per_sm - 3  # one KV head: a pair a sequence
            seen.append(warps // per_sm)
            rng = random.Random(per_sm)
            c = Cache([rng.choice([0, 1, 16, 17, rng.randrange(40)]) for _ in range(n)], 1, 64, 16, dtype, cuda)
            q = torch.randn(n, 3, 64, generator=g).to(dtype).to(cuda)
            out, lse = dkv.paged_decode_attention(q, c.k, c.v, c.seqs(), return_lse=True, check=True)
            for b in [n - 1, 0] + rng.sample(range(n), 12):
                check_attention(out[b:b + 1], lse[b:b + 1], q[b:b + 1], lambda _, b=b: c.tokens(b), 64 ** -0.5)
        assert {warps, warps // 2, 3 if warps == 12 else 4, 1, 0} <= set(seen)


LENS = [0, 1, 2, 15, 16, 17, 33, 100, 0, 333, 64]


# ---------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n_kv,group,hd", [(3, 3, 64), (8, 4, 128), (1, 1, 32), (2, 8, 128), (1, 16, 256), (2, 7, 80),
                                           (1, 9, 96), (1, 33, 64), (5, 5, 64), (2, 2, 256), (3, 1, 48)])
def test_attention_heads_and_types(cuda, dtype, n_kv, group, hd):
    run_attention(Cache(LENS, n_kv, hd, 16, dtype, cuda), n_kv * group, hd, dtype, cuda)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [1, 2, 7, 20, 33, 72, 100, 130, 200, 255])
def test_attention_odd_head_dims(cuda, dtype, hd):
    run_attention(Cache([5, 0, 70], 2, hd, 16, dtype, cuda), 6, hd, dtype, cuda)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("block", [1, 3, 8, 24, 64, 256, 1000])
def test_attention_block_sizes(cuda, dtype, block):
    run_attention(Cache([1, 40, 0, 257, 1000], 2, 64, block, dtype, cuda), 8, 64, dtype, cuda)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["block_first", "odd", "heads_first"])
def test_attention_layouts_and_strides(cuda, dtype, layout):
    c = Cache([31, 0, 500, 16], 3, 64, 16, dtype, cuda, layout=layout)
    q, out, lse = run_attention(c, 9, 64, dtype, cuda)
    # q and out as strided views
    wide = torch.zeros(4, 11, 70, dtype=dtype, device=cuda)
    qs = wide[:, 1:10, 3:67]
    qs.copy_(q)
    out = dkv.paged_decode_attention(q, c.k, c.v, c.seqs())
    into = torch.full((4, 10, 65), 7.0, dtype=dtype, device=cuda)
    got = dkv.paged_decode_attention(qs, c.k, c.v, c.seqs(), out=into[:, 1:, 1:])
    assert got.data_ptr() == into[:, 1:, 1:].data_ptr() and torch.equal(got, out)
    assert torch.all(into[:, 0] == 7.0) and torch.all(into[:, :, 0] == 7.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("strides", [(1, 0, 1), (0, 0, 1), (7, 1, 1), (64, 2, 1), (0, 64, 1)])
def test_queries_that_lie_over_each_other(cuda, dtype, strides):
    """Broadcast and sliding-window q: the new output is an ordinary tensor."""
    c = Cache([40, 3], 2, 64, 16, dtype, cuda)
    rope, _, _ = rope_tables(64, 50, cuda)
    slots = torch.tensor([3, 4], device=cuda)
    pos = torch.tensor([7, 30], dtype=torch.int32, device=cuda)
    k = torch.randn(2, 2, 64, device=cuda).to(dtype)
    for n in (1, 2):
        q = torch.randn(500, device=cuda).to(dtype).as_strided((n, 4, 64), strides)
        seqs = dkv.SeqBatchTensors(cu_seqlens=c.cu[:n + 1], block_tables=c.tables[:n], max_seq_len=40)
        got = dkv.paged_decode_attention(q, c.k, c.v, seqs, check=True)
        assert torch.equal(got, dkv.paged_decode_attention(q.contiguous(), c.k, c.v, seqs)) and got.stride(2) == 1
        turned = [dkv.append_into_paged(k[:n], k[:n], c.k, c.v, slots[:n], q=x, positions=pos[:n], rope=rope, check=True)
                  for x in (q, q.contiguous())]
        assert torch.equal(*turned) and turned[0].stride(2) == 1


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("fill", [math.nan, math.inf, -math.inf])
def test_attention_never_reads_what_no_token_owns(cuda, dtype, fill):
    run_attention(Cache([1, 17, 0, 300, 15], 2, 64, 32, dtype, cuda, fill=fill), 8, 64, dtype, cuda)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [32, 50, 64, 128, 256])
@pytest.mark.parametrize("lens,bound", [([1, 40, 300, 0, 17, 75], 300), ([1, 40, 300, 0, 17, 75], 9000), ([9000, 20], 9000)])
@pytest.mark.parametrize("scale", [0.1, 0.4])
def test_attention_infinite_values(cuda, dtype, hd, lens, bound, scale):
    """Infinite and NaN V elements in tokens that count: +-inf or NaN in their columns as by the definition in 64
    bits, every other column as without them.  Scores spread by 40 at most, so no weight is 0 in fp32."""
    c = Cache(lens, 2, hd, 16, dtype, cuda)
    g = torch.Generator().manual_seed(hd)
    q = (8 * torch.randn(len(lens), 8, hd, generator=g) / hd ** 0.5).to(dtype).to(cuda)
    seqs = dkv.SeqBatchTensors(cu_seqlens=c.cu, block_tables=c.tables, max_seq_len=bound)
    plain = dkv.paged_decode_attention(q, c.k, c.v, seqs, scale=scale, check=True)
    for b, n in enumerate(lens):
        for j in range(0 if n == 0 else hd // 4):  # about a quarter of the columns, one to three elements each
            for _ in range(1 + j % 3):
                t, x = int(torch.randint(n, (1,), generator=g)), (math.inf, -math.inf, math.inf, math.nan)[j % 4]
                x = -x if j % 7 == 0 and _ else x
                c.v[int(c.tables[b, t // 16]), t % 16, j % 2, int(torch.randint(hd, (1,), generator=g))] = x
    got, lse = dkv.paged_decode_attention(q, c.k, c.v, seqs, scale=scale, return_lse=True, check=True)
    ref = torch.zeros(got.shape, dtype=torch.float64, device=cuda)
    for b, n in enumerate(lens):
        if n:
            k, v = (t.double() for t in c.tokens(b))
            s = torch.einsum("ugd,nud->ugn", q[b].double().view(2, 4, hd), k) * scale
            assert float(s.amax() - s.amin()) < 40
            p = torch.softmax(s, -1)  # [2, 4, n] against [n, 2, hd]
            ref[b] = (p[..., None] * v.permute(1, 0, 2)[:, None]).sum(2).reshape(8, hd)
    odd = ~torch.isfinite(ref)
    assert odd.any() and torch.equal(got[odd].double().nan_to_num(nan=7.0, posinf=math.inf, neginf=-math.inf),
                                     ref[odd].nan_to_num(nan=7.0, posinf=math.inf, neginf=-math.inf))
    clean = lambda b: tuple(t.nan_to_num(nan=0.0, posinf=0.0, neginf=0.0) for t in c.tokens(b))  # noqa: E731
    assert torch.equal(got[~odd], plain[~odd])
    check_attention(torch.where(odd, 0, got), lse, q, lambda b: (clean(b)[0], torch.where(
        torch.isfinite(c.tokens(b)[1]).all(0), clean(b)[1], 0)), scale)


@pytest.mark.parametrize("dtype", [BF, F16])
def test_attention_infinite_value_at_the_end_of_the_longest_sequence(cuda, dtype):
    """2^31 - 1 tokens, the last of them infinite in one column: one block of equal tokens, over and over."""
    n, block = (1 << 31) - 1, 1 << 20
    last = (n - 1) // block
    k = torch.zeros(2, block, 1, 32, dtype=dtype, device=cuda)
    v = torch.ones_like(k)
    v[1, (n - 1) % block, 0, 5] = -math.inf
    tables = torch.zeros(1, last + 1, dtype=torch.int32, device=cuda)
    tables[0, last] = 1
    seqs = dkv.SeqBatchTensors(cu_seqlens=torch.tensor([0, n], dtype=torch.int32, device=cuda), block_tables=tables,
                               max_seq_len=n)
    got = dkv.paged_decode_attention(torch.ones(1, 2, 32, dtype=dtype, device=cuda), k, v, seqs, check=True)
    assert torch.all(got[..., 5] == -math.inf)
    got[..., 5] = 1
    # sums of up to 2^31 equal fp32 terms stop growing at 2^24 of them, alike in numerator and denominator
    assert torch.all((got.float() - 1).abs() <= torch.finfo(dtype).eps + 2.0 ** -16)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens", [[20011], [9000, 1, 0, 7000], [1] * 300, [0] * 40, [3, 2049] * 20, list(range(130))])
def test_attention_long_and_ragged(cuda, dtype, lens):
    run_attention(Cache(lens, 2, 64, 16, dtype, cuda), 8, 64, dtype, cuda)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens,n_kv,heads,hd", [
    ([30001], 1, 2, 128), ([30001], 1, 2, 50), ([7000, 9000, 4], 1, 3, 32),  # hundreds of parts of few heads
    ([5000] * 8, 2, 24, 80), ([3001] * 9, 1, 20, 33), ([20000, 30], 1, 140, 64),  # of more heads, each CTA with one
    ([2500] * 12, 2, 64, 96), ([4000] * 30, 4, 40, 64), ([900] * 3, 3, 3, 256),  # parts of many heads; few parts
])
def test_attention_joins_of_every_kind(cuda, dtype, lens, n_kv, heads, hd):
    run_attention(Cache(lens, n_kv, hd, 16, dtype, cuda), heads, hd, dtype, cuda)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_many_sequences(cuda, dtype):
    rng = random.Random(5)
    lens = [rng.choice([0, 1, 5, rng.randrange(60)]) for _ in range(3000)]
    c = Cache(lens, 1, 32, 8, dtype, cuda)
    g = torch.Generator().manual_seed(2)
    q = torch.randn(len(lens), 2, 32, generator=g).to(dtype).to(cuda)
    out = dkv.paged_decode_attention(q, c.k, c.v, c.seqs(), check=True)
    for b in range(0, 3000, 37):  # one sequence alone gives the same tokens' answer
        check_attention(out[b:b + 1], None, q[b:b + 1], lambda _, b=b: c.tokens(b), 32 ** -0.5)
    empty = torch.tensor([n == 0 for n in lens], device=cuda)
    assert torch.all(out[empty] == 0) and torch.all(torch.isfinite(out))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_attention_largest_batch_and_dense_cache(cuda, dtype):
    """65535 sequences, the most there can be; and a dense cache as one block of odd length."""
    n = 65535
    c = Cache([3], 1, 32, 16, dtype, cuda)
    lens = torch.arange(n, device=cuda) % 4
    cu = torch.cat([torch.zeros(1, device=cuda), lens.cumsum(0)]).to(torch.int32)
    q = torch.randn(n, 1, 32, device=cuda).to(dtype)
    seqs = dkv.SeqBatchTensors(cu_seqlens=cu, block_tables=c.tables.repeat(n, 1), max_seq_len=3)
    out = dkv.paged_decode_attention(q, c.k, c.v, seqs, check=True)
    k, v = c.tokens(0)
    check_attention(out[-9:], None, q[-9:], lambda b: (k[: int(lens[n - 9 + b])], v[: int(lens[n - 9 + b])]), 32 ** -0.5)
    check_attention(out[:9], None, q[:9], lambda b: (k[: int(lens[b])], v[: int(lens[b])]), 32 ** -0.5)
    with pytest.raises(dkv.DkvError, match="unsupported"):
        seqs = dkv.SeqBatchTensors(cu_seqlens=torch.zeros(n + 2, dtype=torch.int32, device=cuda),
                                   block_tables=torch.zeros(n + 1, 1, dtype=torch.int32, device=cuda), max_seq_len=0)
        dkv.paged_decode_attention(torch.zeros(n + 1, 1, 32, dtype=dtype, device=cuda), c.k, c.v, seqs)
    length = 777
    kd, vd = (torch.randn(length, 2, 64, device=cuda).to(dtype) for _ in range(2))
    qd = torch.randn(1, 8, 64, device=cuda).to(dtype)
    seqs = dkv.SeqBatchTensors(cu_seqlens=torch.tensor([0, length], dtype=torch.int32, device=cuda),
                               block_tables=torch.zeros(1, 1, dtype=torch.int32, device=cuda), max_seq_len=length)
    got = dkv.paged_decode_attention(qd, kd[None], vd[None], seqs, check=True)
    check_attention(got, None, qd, lambda _: (kd, vd), 64 ** -0.5)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_caches_of_unequal_size_and_a_slice_of_the_batch(cuda, dtype):
    c = Cache([100, 50, 900, 30], 2, 64, 16, dtype, cuda)
    q = torch.randn(4, 4, 64, device=cuda).to(dtype)
    want = dkv.paged_decode_attention(q, c.k, c.v, c.seqs())
    more = torch.cat([c.k, torch.full_like(c.k[:2], math.nan)])  # blocks that V does not have
    assert torch.equal(dkv.paged_decode_attention(q, more, c.v, c.seqs(), check=True), want)
    part = dkv.SeqBatchTensors(cu_seqlens=c.cu[1:4], block_tables=c.tables[1:3], max_seq_len=900)  # cu starts at 100
    got = dkv.paged_decode_attention(q[1:3], c.k, c.v, part, check=True)
    check_attention(got, None, q[1:3], lambda b: c.tokens(b + 1), 64 ** -0.5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("amp,scale", [(1.5, 30.0), (60.0, None), (0.0, None), (1.5, -0.2)])
def test_attention_extreme_scores(cuda, dtype, amp, scale):
    """One token takes all the weight, equal scores, a negative scale."""
    run_attention(Cache([700, 1, 90], 2, 64, 16, dtype, cuda), 4, 64, dtype, cuda, amp=amp, scale=scale)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_tokens_of_no_weight(cuda, dtype):
    """K rows that score -inf weigh nothing; a sequence of only such rows has no weight at all."""
    c = Cache([40, 20], 1, 32, 16, dtype, cuda)
    g = torch.Generator().manual_seed(3)
    q = torch.randn(2, 2, 32, generator=g).abs().add(0.1).to(dtype).to(cuda)
    ids0, ids1 = c.tables[0].long(), c.tables[1].long()
    c.k[ids0[1], 3:9] = -math.inf   # tokens 19..24 of sequence 0
    c.k[ids1[:2]] = -math.inf       # all of sequence 1
    out, lse = dkv.paged_decode_attention(q, c.k, c.v, c.seqs(), return_lse=True)
    k, v = c.tokens(0)
    keep = torch.tensor([not 19 <= i < 25 for i in range(40)], device=cuda)
    check_attention(out[:1], lse[:1], q[:1], lambda _: (k[keep], v[keep]), 32 ** -0.5)
    assert torch.all(out[1] == 0) and torch.all(lse[1] == -math.inf)


def test_attention_offsets_beyond_32_bits(cuda):
    """Blocks whose element offset passes 2^31 (and byte offset 2^32)."""
    block, n_kv, hd = 256, 8, 128
    nb = (1 << 31) // (block * n_kv * hd) + 6
    pages = torch.zeros(nb, block, n_kv, hd, dtype=BF, device=cuda)
    lens = [700, 300]
    c = Cache(lens, n_kv, hd, block, BF, cuda)
    moved = c.tables.clone()
    for i, (b, j) in enumerate([(0, 0), (0, 1), (0, 2), (1, 0), (1, 1)]):
        moved[b, j] = nb - 1 - i
        pages[nb - 1 - i] = c.k[c.tables[b, j].long()]
    vp = pages.clone()
    for i, (b, j) in enumerate([(0, 0), (0, 1), (0, 2), (1, 0), (1, 1)]):
        vp[nb - 1 - i] = c.v[c.tables[b, j].long()]
    q = torch.randn(2, 32, hd, device=cuda).to(BF)
    want = dkv.paged_decode_attention(q, c.k, c.v, c.seqs())
    seqs = dkv.SeqBatchTensors(cu_seqlens=c.cu, block_tables=moved, max_seq_len=700)
    assert torch.equal(dkv.paged_decode_attention(q, pages, vp, seqs, check=True), want)
    check_attention(want, None, q, c.tokens, hd ** -0.5)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_bad_blocks_are_left_out(cuda, dtype):
    c = Cache([100, 50], 2, 64, 16, dtype, cuda)
    q = torch.randn(2, 4, 64, device=cuda).to(dtype)
    c.tables[0, 2] = c.k.shape[0]  # one past the cache
    c.tables[1, 0] = -1
    with pytest.raises(dkv.DkvError, match="block id outside"):
        dkv.paged_decode_attention(q, c.k, c.v, c.seqs(), check=True)
    out, lse = dkv.paged_decode_attention(q, c.k, c.v, c.seqs(), return_lse=True)
    ops.status_word(cuda).t.zero_()

    def good(b):
        ids = c.tables[b].long()
        ids = ids[(ids >= 0) & (ids < c.k.shape[0])]
        n = c.lens[b] - 16
        return tuple(t[ids].reshape(-1, 2, 64)[:n] for t in (c.k, c.v))

    check_attention(out, lse, q, good, 64 ** -0.5)


def test_attention_short_table(cuda):
    c = Cache([100, 50], 2, 64, 16, BF, cuda)
    q = torch.randn(2, 4, 64, device=cuda).to(BF)
    seqs = c.seqs(table_lens=torch.tensor([3, 4], dtype=torch.int32, device=cuda))
    with pytest.raises(dkv.DkvError, match="block_table shorter"):
        dkv.paged_decode_attention(q, c.k, c.v, seqs, check=True)
    out = dkv.paged_decode_attention(q, c.k, c.v, seqs)
    ops.status_word(cuda).t.zero_()
    check_attention(out, None, q, lambda b: tuple(t[: (48, 50)[b]] for t in c.tokens(b)), 64 ** -0.5)
    # a table without columns: no token has a block
    seqs = dkv.SeqBatchTensors(cu_seqlens=c.cu, block_tables=c.tables[:, :0], max_seq_len=100)
    assert torch.all(dkv.paged_decode_attention(q, c.k, c.v, seqs) == 0)
    ops.status_word(cuda).t.zero_()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cu", [[0, 700, 100], [0, 2000000, 40], [900, 100, 500], [0, 5, 5]])
def test_attention_of_lengths_that_are_no_prefix_sums(cuda, dtype, cu):
    """No answer is promised for them, but every access stays in bounds and the call after is right."""
    c = Cache([3000, 900], 2, 64, 16, dtype, cuda)
    q = torch.randn(2, 8, 64, device=cuda).to(dtype)
    want = dkv.paged_decode_attention(q, c.k, c.v, c.seqs())
    for bound in (40, 3000):
        seqs = dkv.SeqBatchTensors(cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=cuda), block_tables=c.tables,
                                   max_seq_len=bound)
        dkv.paged_decode_attention(q, c.k, c.v, seqs)
        torch.cuda.synchronize()
    ops.status_word(cuda).t.zero_()
    assert torch.equal(dkv.paged_decode_attention(q, c.k, c.v, c.seqs(), check=True), want)


def test_attention_empty_batch_and_understated_bound(cuda):
    c = Cache([900, 20], 2, 64, 16, BF, cuda)
    q = torch.randn(2, 4, 64, device=cuda).to(BF)
    none = dkv.SeqBatchTensors(cu_seqlens=c.cu[:1], block_tables=c.tables[:0], max_seq_len=0)
    assert dkv.paged_decode_attention(q[:0], c.k, c.v, none).shape == (0, 4, 64)
    for bound in (0, 7, 1 << 20):  # a wrong bound costs speed, not the answer
        seqs = dkv.SeqBatchTensors(cu_seqlens=c.cu, block_tables=c.tables, max_seq_len=bound)
        check_attention(dkv.paged_decode_attention(q, c.k, c.v, seqs, check=True), None, q, c.tokens, 64 ** -0.5)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_parts_join_by_lse(cuda, dtype):
    c = Cache([600], 2, 64, 16, dtype, cuda)
    q, _, lse = run_attention(c, 8, 64, dtype, cuda)
    got = []
    for lo, hi in ((0, 25), (25, 38)):  # blocks
        n = min(600, hi * 16) - lo * 16
        seqs = dkv.SeqBatchTensors(cu_seqlens=torch.tensor([0, n], dtype=torch.int32, device=cuda),
                                   block_tables=c.tables[:, lo:hi].contiguous(), max_seq_len=n)
        got.append(dkv.paged_decode_attention(q, c.k, c.v, seqs, return_lse=True))
    joined = torch.logaddexp(got[0][1].double(), got[1][1].double())
    assert float((joined - lse.double()).abs().max()) < 1e-5


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens,cut", [([600], 25), ([5000, 40, 16], 1), ([333, 9000], 7)])
def test_attention_outputs_of_parts_join_by_lse(cuda, dtype, lens, cut):
    """A prefix of `cut` blocks and the rest attended apart: out = sum_i exp(lse_i - lse) out_i is the whole's.

    Each part is off by its own tolerance of check_attention, which is what the weights scale; the join in 64 bits adds
    the parts' lse errors, again below the 2^-20 and n 2^-24 of that bound, hence twice the bound of a whole."""
    c = Cache(lens, 2, 64, 16, dtype, cuda)
    q, whole, lse = run_attention(c, 8, 64, dtype, cuda)
    outs, lses = [], []
    for part in (0, 1):
        n = [min(x, cut * 16) if part == 0 else max(x - cut * 16, 0) for x in lens]
        cu = torch.tensor([0] + n, dtype=torch.int32, device=cuda).cumsum(0).to(torch.int32)
        table = c.tables[:, :cut] if part == 0 else c.tables[:, cut:]
        if table.shape[1] == 0:
            table = c.tables[:, :1]
        seqs = dkv.SeqBatchTensors(cu_seqlens=cu, block_tables=table.contiguous(), max_seq_len=max(n))
        out, part_lse = dkv.paged_decode_attention(q, c.k, c.v, seqs, return_lse=True, check=True)
        outs.append(out.double()), lses.append(part_lse.double())
    total = torch.logaddexp(*lses)
    joined = sum(torch.exp(x - total)[..., None] * o for x, o in zip(lses, outs))
    for b in range(len(lens)):
        k, v = (t.double() for t in c.tokens(b))
        s = torch.einsum("ugd,nud->ugn", q[b].double().view(2, 4, 64), k) * 64 ** -0.5
        ds = (64 + 8) * 2.0 ** -23 * (torch.einsum("ugd,nud->ugn", q[b].double().abs().view(2, 4, 64), k.abs()) * 64 ** -0.5).amax(-1)
        p = torch.softmax(s, -1)
        ref, spread = torch.einsum("ugn,nud->ugd", p, v), torch.einsum("ugn,nud->ugd", p, v.abs())
        # each part's rounding to its type is relative to its own output: at most spread after weighting
        bound = spread * (torch.finfo(dtype).eps / 2 + 2 * (2 * ds[..., None] + 2.0 ** -20 + len(k) * 2.0 ** -24
                                                            + (2.0 ** -16 if dtype != F32 else 0)))
        bound = bound + 2 * torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
        assert torch.all((joined[b].view(2, 4, 64) - ref).abs() <= bound), b


def test_attention_is_deterministic_and_reads_the_right_stream(cuda):
    c = Cache([5000, 300, 0, 17], 2, 128, 16, BF, cuda)
    q = torch.randn(4, 8, 128, device=cuda).to(BF)
    want = dkv.paged_decode_attention(q, c.k, c.v, c.seqs())
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        late = torch.zeros_like(q)
        torch.cuda._sleep(20_000_000)
        late.copy_(q)  # only ordered before the call on this stream
        got = dkv.paged_decode_attention(late, c.k, c.v, c.seqs())
    other = dkv.paged_decode_attention(q, c.k, c.v, c.seqs())  # at the same time on another
    torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.equal(other, want)


def test_attention_is_done_when_the_stream_is(cuda):
    """As many equal sequences as ranges: none is cut, the joining launch has nothing to do, and still a
    copy queued behind the call reads the finished output."""
    sms = torch.cuda.get_device_properties(cuda).multi_processor_count
    n = sms * 12 // 8  # twelve warps an SM over eight KV heads
    c = Cache([16] * n, 8, 128, 16, BF, cuda)
    q = torch.randn(n, 32, 128, device=cuda).to(BF)
    length = 1024
    tables = torch.randint(0, n, (n, length // 16), dtype=torch.int32, device=cuda)
    seqs = dkv.SeqBatchTensors(cu_seqlens=torch.arange(n + 1, dtype=torch.int32, device=cuda) * length,
                               block_tables=tables, max_seq_len=length)
    out = torch.zeros_like(q)
    copies = []
    for _ in range(5):
        out.zero_()
        dkv.paged_decode_attention(q, c.k, c.v, seqs, out=out)
        copies.append(out.clone())
    torch.cuda.synchronize()
    assert all(torch.equal(x, out) for x in copies) and bool(out.abs().amax(-1).min() > 0)


@pytest.mark.parametrize("lens", [[40, 0, 300], [6000, 3]])
def test_attention_into_its_query(cuda, lens):
    c = Cache(lens, 2, 64, 16, BF, cuda)
    q = torch.randn(len(lens), 8, 64, device=cuda).to(BF)
    want = dkv.paged_decode_attention(q, c.k, c.v, c.seqs())
    assert dkv.paged_decode_attention(q, c.k, c.v, c.seqs(), out=q) is q and torch.equal(q, want)


def test_attention_workspace_of_the_c_entry(cuda):
    """A missing, short or misaligned workspace is refused before anything is launched."""
    import ctypes as C

    from deltakv_b200 import _lib as L

    c = Cache([9000], 2, 64, 16, BF, cuda)
    q = torch.randn(1, 8, 64, device=cuda).to(BF)
    out = torch.full_like(q, 7.0)
    a = L.PagedDecodeArgs(q.data_ptr(), 512, 64, 8, 0.125, c.seqs().struct(), ops.paged_desc(c.k), ops.paged_desc(c.v),
                          out.data_ptr(), 512, 64, None, None, 0, None)
    need = C.c_int64()
    lib = L.lib()
    assert lib.dkv_paged_decode_workspace_bytes(C.byref(a), C.byref(need)) == L.DKV_OK and need.value > 0
    stream = torch.cuda.current_stream().cuda_stream
    ws = torch.empty(need.value + 16, dtype=torch.uint8, device=cuda)
    assert lib.dkv_paged_decode_attention(C.byref(a), stream) == L.DKV_ERR_WORKSPACE
    a.workspace, a.workspace_bytes = ws.data_ptr(), need.value - 1
    assert lib.dkv_paged_decode_attention(C.byref(a), stream) == L.DKV_ERR_WORKSPACE
    a.workspace, a.workspace_bytes = ws.data_ptr() + 4, need.value
    assert lib.dkv_paged_decode_attention(C.byref(a), stream) == L.DKV_ERR_ALIGNMENT
    torch.cuda.synchronize()
    assert torch.all(out == 7.0)
    a.workspace = ws.data_ptr()
    assert lib.dkv_paged_decode_attention(C.byref(a), stream) == L.DKV_OK
    assert torch.equal(out, dkv.paged_decode_attention(q, c.k, c.v, c.seqs(), scale=0.125))


def test_attention_without_blocks(cuda):
    pages = torch.zeros(0, 16, 2, 64, dtype=BF, device=cuda)
    q = torch.randn(2, 4, 64, device=cuda).to(BF)
    seqs = dkv.SeqBatchTensors(cu_seqlens=torch.tensor([0, 0, 5], dtype=torch.int32, device=cuda),
                               block_tables=torch.zeros(2, 1, dtype=torch.int32, device=cuda), max_seq_len=5)
    assert torch.all(dkv.paged_decode_attention(q, pages, pages, seqs) == 0)
    with pytest.raises(dkv.DkvError, match="block id outside"):
        ops.status_word(cuda).raise_if_set("attention")


# ---------------------------------------------------------------------------------------
# plan
# ---------------------------------------------------------------------------------------
def plan_oracle(lens, new, held, tables, free, block, rows):
    """The definition, one sequence at a time, on Python lists."""
    tables = [list(t) for t in tables]
    width = len(tables[0]) if tables else 0
    cu, cu_new, out_lens, pos, slot, used = [0], [0], [], [], [], 0
    for b, n in enumerate(lens):
        n = max(n, 0)
        k = min(max(new[b], 0), n)
        h = min(max(held[b], 0), width)
        extra = max(min(-(-n // block), width) - h, 0)
        got = max(min(extra, len(free) - used), 0)
        for j in range(got):
            tables[b][h + j] = free[used + j]
        used += extra
        cu.append(cu[-1] + n)
        cu_new.append(cu_new[-1] + k)
        out_lens.append(h + got)
        for i in range(n - k, n):
            pos.append(i)
            ok = i // block < h + got and tables[b][i // block] >= 0
            slot.append(tables[b][i // block] * block + i % block if ok else -1)
    pos, slot, cu_new = pos[:rows], slot[:rows], [min(x, rows) for x in cu_new]
    return cu, cu_new, out_lens, pos + [0] * (rows - len(pos)), slot + [-1] * (rows - len(slot)), min(used, len(free)), tables


def run_plan(dev, lens, new, held, tables, free, block, rows, check=True, view=False):
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    n, width = len(lens), len(tables[0]) if tables else 0
    t = ints(tables).view(n, width)
    if view:  # a column slice of a wider table
        wide = torch.full((n, width + 5), -9, dtype=torch.int32, device=dev)
        wide[:, 2:2 + width] = t
        t = wide[:, 2:2 + width]
    step = dkv.plan_paged_step(ints(lens), t, block, rows=rows, max_seq_len=max(lens, default=0),
                               new_lengths=None if new is None else ints(new),
                               table_lens=None if held is None else ints(held),
                               free_blocks=None if free is None else ints(free), check=check)
    want = plan_oracle(lens, lens if new is None else new, [width] * n if held is None else held, tables, free or [],
                       block, rows)
    got = (step.seqs.cu_seqlens, step.cu_new, step.seqs.table_lens, step.positions, step.slots, step.blocks_used, t)
    names = ("cu_seqlens", "cu_new", "table_lens", "positions", "slots", "used", "tables")
    for name, g, w in zip(names, got, want):
        assert g.reshape(-1).tolist() == torch.tensor(w).reshape(-1).tolist(), name
    assert step.seqs.block_tables.data_ptr() == t.data_ptr()
    if view:
        assert torch.all(wide[:, :2] == -9) and torch.all(wide[:, 2 + width:] == -9)
    return step


def random_plan(rng, n, longest, most_new, block):
    lens = [rng.choice([0, 1, rng.randrange(longest + 1)]) for _ in range(n)]
    new = [rng.randint(0, min(x, most_new)) for x in lens]
    held = [-(-(x - k) // block) for x, k in zip(lens, new)]
    width = max(-(-x // block) for x in lens) + 1
    ids = rng.sample(range(10 * n * width), n * width)
    tables = [[ids.pop() if j < held[b] else 0 for j in range(width)] for b in range(n)]
    free = [rng.randrange(10 ** 6) for _ in range(sum(-(-x // block) - h for x, h in zip(lens, held)) + 3)]
    return lens, new, held, tables, free


@pytest.mark.parametrize("n,longest,most_new,block,view", [(1, 5, 5, 16, False), (7, 100, 1, 16, True),
                                                           (40, 300, 300, 5, False), (513, 200, 3, 8, True),
                                                           (1100, 60, 60, 1, False), (100, 2000, 700, 64, False)])
def test_plan_random(cuda, n, longest, most_new, block, view):
    rng = random.Random(n)
    lens, new, held, tables, free = random_plan(rng, n, longest, most_new, block)
    total = sum(new)
    for rows in (total, total + 333):
        run_plan(cuda, lens, new, held, tables, free, block, rows, view=view)


def test_plan_forms_and_edges(cuda):
    run_plan(cuda, [], [], [], [], [], 16, 0)
    run_plan(cuda, [], [], [], [], [], 16, 5)                                  # only padding rows
    run_plan(cuda, [0, 0], None, None, [[4], [5]], None, 16, 0)
    run_plan(cuda, [3, 20], None, None, [[4, 1], [5, 2]], None, 16, 23)        # full tables, all tokens new
    run_plan(cuda, [3, 20], [1, 1], [1, 2], [[4, 1], [5, 2]], None, 16, 2)     # blocks held beyond the need
    run_plan(cuda, [33], None, [0], [[0, 0, 0]], [7, 8, 9], 16, 33)            # a fresh prefill
    run_plan(cuda, [0, 0], [0, 0], [0, 0], [[], []], [], 16, 0)                # a table without columns


def test_plan_largest_batch(cuda):
    n = 16384
    lens = [1 + (i * 7) % 40 for i in range(n)]
    held = [-(-(x - 1) // 16) for x in lens]
    tables = [[3 * i + j for j in range(3)] for i in range(n)]
    free = list(range(10 ** 6, 10 ** 6 + n))
    run_plan(cuda, lens, [1] * n, held, tables, free, 16, n)
    with pytest.raises(dkv.DkvError, match="unsupported"):
        z = torch.zeros(n + 1, dtype=torch.int32, device=cuda)
        dkv.plan_paged_step(z, z[:, None].clone(), 16, rows=0, max_seq_len=0)


def test_plan_without_memory_for_its_outputs(cuda):
    """torch's own error, which a serving loop catches; the limit is this process's, nothing is filled up."""
    z = torch.ones(1, dtype=torch.int32, device=cuda)
    torch.cuda.empty_cache()
    total = torch.cuda.get_device_properties(cuda).total_memory
    torch.cuda.set_per_process_memory_fraction((torch.cuda.memory_reserved(cuda) + (64 << 20)) / total, cuda)
    try:
        with pytest.raises(torch.OutOfMemoryError):
            dkv.plan_paged_step(z, z[:, None].clone(), 16, rows=1 << 28, max_seq_len=1)
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0, cuda)
    dkv.plan_paged_step(z, z[:, None].clone(), 16, rows=1, max_seq_len=1, check=True)


_BATCHES_ALONE = """
import torch, deltakv_b200 as dkv
for n in (5119, 5120, 6095, 6096, 6100, 6143, 6144):
    lens = torch.arange(1, n + 1, dtype=torch.int32, device="cuda") % 32 + 1
    tables = torch.arange(2 * n, dtype=torch.int32, device="cuda").view(n, 2)
    step = dkv.plan_paged_step(lens, tables, 16, rows=n, max_seq_len=32, new_lengths=torch.ones_like(lens), check=True)
    pos = lens.long() - 1
    assert torch.equal(step.slots, tables.gather(1, (pos // 16)[:, None])[:, 0].long() * 16 + pos % 16), n
    assert torch.equal(step.positions.long(), pos) and int(step.seqs.cu_seqlens[-1]) == int(lens.sum()), n
print("planned")
"""


def test_plan_batches_at_the_default_shared_memory_limit(cuda):
    """Around 48 KB of shared memory, in a process that has planned no larger batch before."""
    root = Path(__file__).resolve().parent.parent
    got = subprocess.run([sys.executable, "-c", _BATCHES_ALONE], cwd=root, capture_output=True, text=True, timeout=300)
    assert got.returncode == 0 and got.stdout.split()[-1] == "planned", got.stderr[-2000:]


@pytest.mark.parametrize("text,lens,new,held,tables,free,rows", [
    ("free block list", [40, 40], [40, 40], [0, 0], [[0] * 3, [0] * 3], [5, 6, 7, 8], 80),
    ("block_table shorter", [40, 20], [2, 1], [2, 2], [[4, 5], [6, 7]], [9], 3),
    ("invalid argument", [-3, 20], [1, 1], [1, 2], [[4, 5], [6, 7]], [], 2),
    ("invalid argument", [3, 20], [5, -1], [1, 2], [[4, 5], [6, 7]], [], 3),
    ("invalid argument", [3, 20], [1, 1], [-1, 9], [[4, 5], [6, 7]], [8], 2),
    ("invalid argument", [3, 20], [3, 4], [1, 2], [[4, 5], [6, 7]], [], 5),
])
def test_plan_records_what_does_not_fit(cuda, text, lens, new, held, tables, free, rows):
    with pytest.raises(dkv.DkvError, match=text):
        run_plan(cuda, lens, new, held, tables, free, 16, rows)
    run_plan(cuda, lens, new, held, tables, free, 16, rows, check=False)  # the rest is as documented
    ops.status_word(cuda).t.zero_()


# ---------------------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------------------
def rope_tables(hd, n, dev):
    rope = dkv.RotaryEmbedding(hd, n)
    return rope, rope.cos_cached[:, : hd // 2].to(dev), rope.sin_cached[:, : hd // 2].to(dev)


def check_append(dev, c, dtype, heads, n_kv, hd, rows, seed=0, rope=True, with_q=True, fused=False, in_place=False):
    g = torch.Generator().manual_seed(seed)
    n_slots = c.k.shape[0] * c.block
    slots = torch.randperm(n_slots, generator=g)[:rows]
    slots[torch.rand(rows, generator=g) < 0.1] = -1
    pos = torch.randint(0, 500, (rows,), generator=g, dtype=torch.int32)
    qkv = torch.randn(rows, heads + 2 * n_kv, hd, generator=g).to(dtype).to(dev)
    q, k, v = qkv.split([heads, n_kv, n_kv], 1)
    if not fused:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    table, cos, sin = rope_tables(hd, 500, dev) if rope else (None, None, None)
    want_k, want_v, q_in = c.k.clone(), c.v.clone(), q.clone()

    def turn(x):
        """In fp64, rounded once: off by the two fp32 products and their sum at most."""
        if not rope:
            return x.double()
        cs, sn = cos[pos.to(dev).long()].double()[:, None], sin[pos.to(dev).long()].double()[:, None]
        lo, hi = x.double().chunk(2, -1)
        return torch.cat([lo * cs - hi * sn, hi * cs + lo * sn], -1)

    got = dkv.append_into_paged(k, v, c.k, c.v, slots.to(dev), q=q if with_q else None,
                                positions=pos.to(dev) if rope else None, rope=table,
                                q_out=q if in_place else None, check=True)
    at = slots >= 0
    where = (slots[at].to(dev) // c.block, slots[at].to(dev) % c.block)

    def close(a, ref, big):
        eps = torch.finfo(a.dtype).eps / 2
        tol = eps * ref.abs() + 2.0 ** -22 * big + torch.finfo(a.dtype).smallest_normal * torch.finfo(a.dtype).eps
        assert torch.all((a.double() - ref).abs() <= tol)

    biggest = lambda x: x.double().abs().amax(-1, keepdim=True)  # noqa: E731
    close(c.k[where], turn(k if not in_place else k)[at.to(dev)], biggest(k)[at.to(dev)])
    close(c.v[where], v.double()[at.to(dev)], biggest(v)[at.to(dev)])
    if dtype == c.v.dtype:
        assert torch.equal(c.v[where], v[at.to(dev)])
    want_k[where], want_v[where] = c.k[where], c.v[where]
    assert torch.equal(want_k, c.k) and torch.equal(want_v, c.v)  # nothing else was touched
    if with_q:
        close(got, turn(q_in), biggest(q_in))
        assert (got.data_ptr() == q.data_ptr()) == in_place
    else:
        assert got is None


@pytest.mark.parametrize("dtype,pages", [(BF, BF), (F16, F16), (F32, F32), (F32, BF), (F32, F16)])
@pytest.mark.parametrize("heads,n_kv,hd,rows", [(32, 8, 128, 64), (9, 3, 64, 111), (1, 1, 2, 5), (4, 4, 80, 33),
                                                (6, 2, 36, 17), (16, 1, 256, 3), (8, 8, 16, 1), (5, 5, 32, 500)])
def test_append_shapes(cuda, dtype, pages, heads, n_kv, hd, rows):
    c = Cache([600], n_kv, hd, 16, pages, cuda)
    check_append(cuda, c, dtype, heads, n_kv, hd, rows)
    check_append(cuda, c, dtype, heads, n_kv, hd, rows, seed=1, fused=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["block_first", "odd", "heads_first"])
def test_append_layouts(cuda, dtype, layout):
    c = Cache([600], 3, 64, 24, dtype, cuda, layout=layout)
    check_append(cuda, c, dtype, 9, 3, 64, 100, in_place=True)
    check_append(cuda, c, dtype, 9, 3, 64, 100, fused=True, in_place=True)
    check_append(cuda, c, dtype, 9, 3, 64, 100, with_q=False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [1, 7, 64, 100])
def test_append_without_rope(cuda, dtype, hd):
    check_append(cuda, Cache([300], 2, hd, 16, dtype, cuda), dtype, 2, 2, hd, 90, rope=False, with_q=False)


@pytest.mark.parametrize("hd", [2, 64, 100, 128])
def test_append_in_fp32_equals_tensor_operations(cuda, hd):
    """Products and sums rounded one by one, so every bit is that of the reference's rotate-half in fp32."""
    c = Cache([300], 2, hd, 16, F32, cuda)
    rows, slots = 200, torch.randperm(300, generator=torch.Generator().manual_seed(1))[:200].to(cuda)
    q, k = torch.randn(rows, 4, hd, device=cuda), torch.randn(rows, 2, hd, device=cuda)
    pos = torch.randint(0, 500, (rows,), device=cuda, dtype=torch.int32)
    rope, cos, sin = rope_tables(hd, 500, cuda)

    def turn(x):
        cs, sn = (torch.cat([t, t], -1)[pos.long()][:, None] for t in (cos, sin))
        lo, hi = x.chunk(2, -1)
        return x * cs + torch.cat([-hi, lo], -1) * sn

    got = dkv.append_into_paged(k, k, c.k, c.v, slots, q=q, positions=pos, rope=rope, check=True)
    assert torch.equal(got, turn(q))
    assert torch.equal(c.k[slots // 16, slots % 16], turn(k)) and torch.equal(c.v[slots // 16, slots % 16], k)


def test_append_ranges(cuda):
    """A slot beyond the pages and a position beyond the tables: recorded, nothing written."""
    c = Cache([100], 2, 64, 16, BF, cuda)
    rope, _, _ = rope_tables(64, 50, cuda)
    k = torch.randn(4, 2, 64, device=cuda).to(BF)
    q, out = torch.randn(4, 4, 64, device=cuda).to(BF), torch.full((4, 4, 64), 3.0, dtype=BF, device=cuda)
    before = c.k.clone(), c.v.clone()
    n_slots = c.k.shape[0] * 16
    slots = torch.tensor([n_slots, 1 << 40, 5, 6], device=cuda)
    pos = torch.tensor([1, 2, 50, -1], dtype=torch.int32, device=cuda)
    with pytest.raises(dkv.DkvError):
        dkv.append_into_paged(k, k, c.k, c.v, slots, q=q, positions=pos, rope=rope, q_out=out, check=True)
    assert torch.equal(c.k, before[0]) and torch.equal(c.v, before[1])
    assert torch.all(out[2:] == 3.0) and not torch.any(torch.all(out[:2] == 3.0, -1))
    assert dkv.append_into_paged(k[:0], k[:0], c.k, c.v, slots[:0]) is None
    with pytest.raises(ValueError, match="do not cover head_dim"):
        dkv.append_into_paged(k, k, c.k, c.v, slots, positions=pos, rope=rope_tables(32, 50, cuda)[0])


# ---------------------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------------------
class Server:
    """A small serving loop on the three operators; keeps every token's K and V beside the pages."""

    def __init__(self, dev, dtype, n_req=5, heads=8, n_kv=2, hd=64, block=16, width=20, rows=64, layout="kv_first"):
        self.dev, self.dtype, self.heads, self.n_kv, self.hd, self.block = dev, dtype, heads, n_kv, hd, block
        nb = n_req * width
        cache = torch.full((2, nb, block, n_kv, hd), math.nan, dtype=dtype, device=dev)
        self.k, self.v = ops.page_view(cache, 0), ops.page_view(cache, 1)
        ints = lambda *s: torch.zeros(*s, dtype=torch.int32, device=dev)  # noqa: E731
        self.tables, self.held, self.lens, self.new = ints(n_req, width), ints(n_req), ints(n_req), ints(n_req)
        self.free = torch.randperm(nb, generator=torch.Generator().manual_seed(9)).to(torch.int32).to(dev)
        self.rope, self.cos, self.sin = rope_tables(hd, width * block, dev)
        self.qkv = torch.zeros(rows, heads + 2 * n_kv, hd, dtype=dtype, device=dev)
        self.rows = rows
        self.n_req = n_req
        self.max_len = width * block
        self.stored = [[] for _ in range(n_req)]
        self.q_of = None

    def launch(self):
        """The calls of one step, free of any host round trip."""
        step = dkv.plan_paged_step(self.lens, self.tables, self.block, rows=self.rows, max_seq_len=self.max_len,
                                   new_lengths=self.new, table_lens=self.held, free_blocks=self.free)
        q, k, v = self.qkv.split([self.heads, self.n_kv, self.n_kv], 1)
        q = dkv.append_into_paged(k, v, self.k, self.v, step.slots, q=q, positions=step.positions, rope=self.rope)
        last = (step.cu_new[1:].long() - 1).clamp(min=0)
        out = dkv.paged_decode_attention(q[last], self.k, self.v, step.seqs)
        return step, out

    def feed(self, new, seed):
        """This step's inputs, in the buffers a captured step reads."""
        g = torch.Generator().manual_seed(seed)
        assert sum(new) <= self.rows
        self.new.copy_(torch.tensor(new, dtype=torch.int32))
        self.lens += self.new
        self.qkv.copy_(torch.randn(self.qkv.shape, generator=g).to(self.dtype))

    def verify(self, new, step, out):
        cu = step.cu_new.tolist()
        pos = step.positions[: cu[-1]].long()
        cs, sn = self.cos[pos].double()[:, None], self.sin[pos].double()[:, None]

        def turn(x):
            lo, hi = x[: cu[-1]].double().chunk(2, -1)
            return torch.cat([lo * cs - hi * sn, hi * cs + lo * sn], -1).to(self.dtype)

        q, k, v = self.qkv.split([self.heads, self.n_kv, self.n_kv], 1)
        q, k = turn(q), turn(k)
        for b in range(self.n_req):
            self.stored[b] += [(k[r], v[r].clone()) for r in range(cu[b], cu[b + 1])]
        rows = [cu[b + 1] - 1 for b in range(self.n_req)]

        def tokens(b):
            if not self.stored[b]:
                return (torch.zeros(0, self.n_kv, self.hd, device=self.dev),) * 2
            return tuple(torch.stack([t[i] for t in self.stored[b]]) for i in (0, 1))

        # a rotation in fp32 may round to the neighbour of the fp64 one: compare through what is stored
        for b in range(self.n_req):
            k_ref, v_ref = tokens(b)
            n = k_ref.shape[0]
            ids = step.seqs.block_tables[b, : -(-n // self.block)].long()
            kk, vv = (t[ids].reshape(-1, self.n_kv, self.hd)[:n] for t in (self.k, self.v))
            assert torch.equal(vv, v_ref)
            assert torch.all((kk.double() - k_ref.double()).abs() <= 2.0 ** -20 * 8 + torch.finfo(self.dtype).eps * k_ref.double().abs())
        have = [b for b in range(self.n_req) if new[b]]
        for b in have:
            n = len(self.stored[b])
            ids = step.seqs.block_tables[b, : -(-n // self.block)].long()
            pages = tuple(t[ids].reshape(-1, self.n_kv, self.hd)[:n] for t in (self.k, self.v))
            qd = q[rows[b]].double()
            s = torch.einsum("ugd,nud->ugn", qd.view(self.n_kv, -1, self.hd), pages[0].double()) * self.hd ** -0.5
            ref = torch.einsum("ugn,nud->ugd", torch.softmax(s, -1), pages[1].double()).reshape(self.heads, self.hd)
            # q's rotation may round to its neighbour (eps of q): the scores move by eps sum |q k| scale at most
            ds = torch.finfo(self.dtype).eps * float((torch.einsum(
                "ugd,nud->ugn", qd.abs().view(self.n_kv, -1, self.hd), pages[0].double().abs()) * self.hd ** -0.5).max())
            spread = float(pages[1].double().abs().max())
            assert float((out[b].double() - ref).abs().max()) <= (torch.finfo(self.dtype).eps + 2 * ds) * spread
        self.held.copy_(step.seqs.table_lens)
        used = int(step.blocks_used)
        self.free.copy_(torch.cat([self.free[used:], self.free[:used]]))  # taken entries to the end


@pytest.mark.parametrize("dtype", TYPES)
def test_steps_of_a_serving_loop(cuda, dtype):
    """A ragged prefill, then decode steps that cross block borders, one request idle for a while."""
    s = Server(cuda, dtype)
    for i, new in enumerate([[13, 0, 30, 5, 16], [1, 1, 1, 1, 1], [1, 20, 1, 0, 1], [1, 1, 1, 1, 1], [1, 0, 1, 1, 17]]):
        s.feed(new, i)
        step, out = s.launch()
        s.verify(new, step, out)
    ops.status_word(cuda).raise_if_set("steps")


@pytest.mark.parametrize("dtype", [BF, F32])
def test_captured_steps(cuda, dtype):
    """The whole step in one graph, replayed with other lengths; a second captured step shares the allocator."""
    a, b = Server(cuda, dtype), Server(cuda, dtype, n_req=3, heads=6, n_kv=3, hd=32, block=8, rows=40)
    for i, (s, new) in enumerate([(a, [13, 2, 30, 5, 3]), (b, [9, 1, 20])]):
        s.feed(new, i)
        s.verify(new, *s.launch())  # eager first: everything is loaded
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        for s in (a, b):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                made = s.launch()
            graphs.append((graph, made))
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for i in range(4):
        news = ([1, 1, 3, 0, 1], [1, 7, 1])
        a.feed(news[0], 10 + i)
        b.feed(news[1], 20 + i)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):  # both at once
            graphs[0][0].replay()
        graphs[1][0].replay()
        torch.cuda.synchronize()
        a.verify(news[0], *graphs[0][1])
        b.verify(news[1], *graphs[1][1])
    ops.status_word(cuda).raise_if_set("captured steps")


def test_steps_without_autograd_or_with_it(cuda):
    """Inference mode, no_grad and inputs that require gradients: the same values, and no graph behind them."""
    c = Cache([40, 5], 2, 64, 16, BF, cuda)
    rope, _, _ = rope_tables(64, 50, cuda)
    lens = torch.tensor([40, 5], dtype=torch.int32, device=cuda)
    qkv = torch.randn(2, 12, 64, device=cuda).to(BF)
    ones = torch.ones(2, dtype=torch.int32, device=cuda)

    def step(x):
        plan = dkv.plan_paged_step(lens, c.tables, 16, rows=2, max_seq_len=40, new_lengths=ones)
        q = dkv.append_into_paged(x[:, 8:10], x[:, 10:], c.k, c.v, plan.slots, q=x[:, :8], positions=plan.positions,
                                  rope=rope)
        return plan.slots, q, *dkv.paged_decode_attention(q, c.k, c.v, plan.seqs, return_lse=True)

    want = step(qkv)
    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in zip(step(qkv), want))
    with torch.inference_mode():
        got = step(qkv)
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and all(a.is_inference() for a in got)
    got = step(qkv.clone().requires_grad_())
    assert all(torch.equal(a, b) and not a.requires_grad for a, b in zip(got, want))
    got[1].zero_(), got[2].mul_(2)  # ordinary tensors


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("width,bound", [(3, 48), (3, 5000), (40, 640)])
def test_attention_right_behind_its_plan(cuda, dtype, width, bound):
    """The plan fills the tables that the next launch reads: new blocks every time, and nothing in between."""
    n = 6
    c = Cache([16 * n * width], 2, 64, 16, dtype, cuda)  # pages of normal values, all owned
    lens = torch.tensor([16 * width - b for b in range(n)], dtype=torch.int32, device=cuda)
    q = torch.randn(n, 4, 64, device=cuda).to(dtype)
    held = torch.zeros(n, dtype=torch.int32, device=cuda)
    tables = torch.zeros(n, width, dtype=torch.int32, device=cuda)
    free = [torch.randperm(n * width, device=cuda).to(torch.int32) for _ in range(12)]

    def run(wait):
        outs = []
        for f in free:
            step = dkv.plan_paged_step(lens, tables, 16, rows=0, max_seq_len=bound, table_lens=held, free_blocks=f,
                                       new_lengths=held)
            wait()
            outs.append(dkv.paged_decode_attention(q, c.k, c.v, step.seqs))
            wait()
        return torch.stack(outs)

    want = run(torch.cuda.synchronize)
    assert float((want[0] - want[1]).abs().max()) > 0.01  # the tables do differ
    for _ in range(10):
        assert torch.equal(run(lambda: None), want)


@pytest.mark.parametrize("n", [4, 300])
def test_joins_of_lengths_that_the_plan_just_wrote(cuda, n):
    """Other lengths every step, in memory that the steps before held theirs in; long sequences cut into parts."""
    rng = random.Random(n)
    longest = 12000 // n ** 0.5
    c = Cache([4000], 1, 64, 16, BF, cuda)
    q = torch.randn(n, 8, 64, device=cuda).to(BF)
    width = -(-12000 // 16)
    tables = torch.randint(0, c.k.shape[0] - 3, (n, width), dtype=torch.int32, device=cuda)
    steps = [torch.tensor([rng.randrange(int(longest)) for _ in range(n)], dtype=torch.int32, device=cuda) for _ in range(12)]

    def run(wait):
        outs = []
        for lens in steps:
            step = dkv.plan_paged_step(lens, tables, 16, rows=0, max_seq_len=12000, new_lengths=torch.zeros_like(lens))
            wait()
            outs.append(dkv.paged_decode_attention(q, c.k, c.v, step.seqs))
            wait()
            del step
        return torch.stack(outs)

    want = run(torch.cuda.synchronize)
    for _ in range(10):
        assert torch.equal(run(lambda: None), want)


@pytest.mark.parametrize("lens", [[300, 40], [9000, 40]])
def test_calls_behind_one_another(cuda, lens):
    """Each call reads what the one before it wrote; nothing waits in between."""
    c = Cache(lens, 2, 64, 16, BF, cuda)
    rope, _, _ = rope_tables(64, 50, cuda)
    k = torch.randn(2, 2, 64, device=cuda).to(BF)
    pos = torch.tensor([3, 4], dtype=torch.int32, device=cuda)
    slots = torch.tensor([int(c.tables[b, 0]) * 16 for b in range(2)], device=cuda)  # the sequences' first tokens
    first = torch.randn(2, 8, 64, device=cuda).to(BF)

    def chain(wait):
        c.k.copy_(keep[0]), c.v.copy_(keep[1])
        x = first
        for _ in range(12):
            x = dkv.append_into_paged(x[:, :2], x[:, 2:4], c.k, c.v, slots, q=x, positions=pos, rope=rope)
            wait()
            x = dkv.paged_decode_attention(x, c.k, c.v, c.seqs())
            wait()
        return x

    keep = c.k.clone(), c.v.clone()
    want = chain(torch.cuda.synchronize)
    for _ in range(5):
        assert torch.equal(chain(lambda: None), want)


def test_captured_between_copies_and_memsets(cuda):
    """The operators in a graph whose other nodes are copies and memsets, on two branches."""
    c = Cache([500, 40], 2, 64, 16, BF, cuda)
    lens = torch.tensor([500, 40], dtype=torch.int32, device=cuda)
    q = torch.randn(2, 8, 64, device=cuda).to(BF)
    want = dkv.paged_decode_attention(q, c.k, c.v, c.seqs())
    src, q_in, out = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(q)
    host = torch.zeros(2, 8, 64, dtype=BF).pin_memory()
    free = torch.arange(c.k.shape[0], dtype=torch.int32, device=cuda)
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        q_in.copy_(src)
        out.zero_()
        other.wait_stream(side)
        with torch.cuda.stream(other):
            held = torch.zeros(2, dtype=torch.int32, device=cuda)
            tables = torch.zeros(2, 32, dtype=torch.int32, device=cuda)
            step = dkv.plan_paged_step(lens, tables, 16, rows=540, max_seq_len=500, table_lens=held, free_blocks=free)
        dkv.paged_decode_attention(q_in, c.k, c.v, c.seqs(), out=out)
        side.wait_stream(other)
        again = dkv.paged_decode_attention(out, c.k, c.v, step.seqs)
        host.copy_(out, non_blocking=True)
    for _ in range(3):
        src.copy_(q)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(host.to(cuda), want)
        assert int(step.blocks_used) == 35 and step.positions[:3].tolist() == [0, 1, 2]
        assert torch.equal(again, dkv.paged_decode_attention(want, c.k, c.v, step.seqs))


class DeviceRope:
    """A rope whose tables live on the GPU, as a module's buffers do; angles of the rows differ by `by`."""

    def __init__(self, dev, hd=64, n=4096, by=1.0):
        rope = dkv.RotaryEmbedding(hd, n, base=10000.0 * by)
        self.cos_cached, self.sin_cached = rope.cos_cached.to(dev), rope.sin_cached.to(dev)

    def turn(self, x, pos):
        """fp32 in fp64, to be compared within two roundings."""
        c, s = (t[pos.long(), : x.shape[2] // 2].double()[:, None] for t in (self.cos_cached, self.sin_cached))
        lo, hi = x.double().chunk(2, -1)
        return torch.cat([lo * c - hi * s, hi * c + lo * s], -1)


class Turner:
    """append_into_paged on fp32 rows of its own, for the q it returns."""

    def __init__(self, dev, rows=3):
        self.c = Cache([100], 2, 64, 16, F32, dev)
        self.q, self.k = torch.randn(rows, 4, 64, device=dev), torch.randn(rows, 2, 64, device=dev)
        self.pos = torch.arange(rows, dtype=torch.int32, device=dev) * 17 + 5
        self.slots = torch.arange(rows, device=dev)

    def __call__(self, rope):
        return dkv.append_into_paged(self.k, self.k, self.c.k, self.c.v, self.slots, q=self.q, positions=self.pos, rope=rope)

    def check(self, got, rope):
        big = self.q.double().abs().amax(-1, keepdim=True)
        assert torch.all((got.double() - rope.turn(self.q, self.pos)).abs() <= 2.0 ** -22 * big)


def test_rope_first_used_inside_a_capture(cuda):
    """The graph makes its tables itself; eager calls, also before any replay, have their own."""
    turner, rope = Turner(cuda), DeviceRope(cuda)
    turner(DeviceRope(cuda))  # the kernels are loaded
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        captured = turner(rope)
    turner.check(turner(rope), rope)
    graph.replay()
    turner.check(captured, rope)
    rope.cos_cached.mul_(0.5)
    graph.replay()  # reads the rope's tensors
    turner.check(captured, rope)
    turner.check(turner(rope), rope)


def test_rope_changed_and_dropped_after_a_capture(cuda):
    """A replay goes on with the tables of its capture, whatever took their rope's place."""
    turner, rope = Turner(cuda), DeviceRope(cuda)
    turner(rope)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        captured = turner(rope)
    graph.replay()
    want = captured.clone()
    turner.check(want, rope)
    rope.sin_cached.mul_(3.0)
    turner.check(turner(rope), rope)
    del rope
    junk = [torch.full((4096, 32), math.nan, device=cuda) for _ in range(20)]
    captured.zero_()
    graph.replay()
    assert torch.equal(captured, want)
    del junk


def test_rope_on_the_host_cannot_be_copied_inside_a_capture(cuda):
    turner, rope = Turner(cuda), dkv.RotaryEmbedding(64, 200)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="once before it"):
        with torch.cuda.graph(graph):
            turner.q.mul_(1.0)
            turner(rope)
    turner(rope)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = turner(rope)
    graph.replay()
    assert torch.equal(captured, turner(rope))


def test_rope_tables_made_on_another_stream(cuda):
    """The first use is behind other work of its stream; the second, elsewhere, does not wait for that stream."""
    turner, side = Turner(cuda), torch.cuda.Stream()
    turner(DeviceRope(cuda))
    for _ in range(3):
        rope = DeviceRope(cuda)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(20_000_000)
            first = turner(rope)
        turner.check(turner(rope), rope)
        torch.cuda.synchronize()
        turner.check(first, rope)


@pytest.mark.parametrize("how", ["dropped", "changed"])
def test_rope_tables_outlive_the_streams_that_read_them(cuda, how):
    turner, side = Turner(cuda), torch.cuda.Stream()
    want = turner(DeviceRope(cuda))
    for _ in range(3):
        rope = DeviceRope(cuda)
        turner(rope)  # the tables are made on this stream
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(20_000_000)
            got = turner(rope)
        if how == "changed":
            rope.cos_cached.zero_(), rope.sin_cached.zero_()
            turner(rope)
        else:
            del rope
        junk = [torch.full((4096, 32), math.nan, device=cuda) for _ in range(8)]
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        del junk


_CAPTURE_FIRST = """
import torch, deltakv_b200 as dkv
from deltakv_b200 import ops
dev = torch.device("cuda", 0)
q = torch.ones(1, 4, 64, device=dev, dtype=torch.bfloat16)
k = torch.ones(4, 16, 2, 64, device=dev, dtype=torch.bfloat16)
v = torch.ones_like(k)
ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
class Rope: cos_cached, sin_cached = torch.zeros(2, 50, 64, device=dev)  # a quarter turn
Rope.sin_cached += 1
step_graph, rope, lens, table = torch.cuda.CUDAGraph(), Rope(), ints([20]), ints([[1, 0]])
x = torch.randn(1, 2, 64, device=dev, dtype=torch.bfloat16)
held, free, new = ints([1]), ints([3]), ints([1])
torch.cuda.synchronize()
with torch.cuda.graph(step_graph):
    step = dkv.plan_paged_step(lens, table, 16, rows=1, max_seq_len=20, new_lengths=new, table_lens=held, free_blocks=free)
    turned = dkv.append_into_paged(x, x, k, v, step.slots, q=x, positions=step.positions, rope=rope)
step_graph.replay()
quarter = torch.cat([-x[..., 32:], x[..., :32]], -1)
assert table.tolist() == [[1, 3]] and step.slots.tolist() == [3 * 16 + 3] and torch.equal(turned, quarter)
assert torch.equal(k[3, 3], quarter[0]) and torch.equal(v[3, 3], x[0])
assert torch.equal(dkv.append_into_paged(x, x, k, v, step.slots, q=x, positions=step.positions, rope=rope), quarter)
k.fill_(1), v.fill_(1)
seqs = dkv.SeqBatchTensors(cu_seqlens=ints([0, 20]), block_tables=ints([[1, 9]]), max_seq_len=20)  # no block 9
graph = torch.cuda.CUDAGraph()
torch.cuda.synchronize()
with torch.cuda.graph(graph):
    out = dkv.paged_decode_attention(q, k, v, seqs)
word = ops.status_word(dev)
word.raise_if_set("nothing has run")
good = dkv.SeqBatchTensors(cu_seqlens=ints([0, 20]), block_tables=ints([[1, 3]]), max_seq_len=20)
assert torch.equal(dkv.paged_decode_attention(q, k, v, good, check=True), torch.ones_like(q))
graph.replay()
try:
    word.raise_if_set("replay")
except dkv.DkvError as e:
    assert "block id outside" in str(e)
else:
    raise AssertionError("the replay recorded nothing")
assert torch.equal(out, torch.ones_like(q))
dkv.paged_decode_attention(q, k, v, seqs)  # recorded by an eager call
seqs.block_tables.copy_(ints([[1, 3]]))
graph.replay()                             # a good replay leaves it
assert int(word.t) != 0
del graph, out
torch.cuda.empty_cache()
word.t.zero_()
dkv.paged_decode_attention(q, k, v, good, check=True)
print("captured first")
"""


def test_first_use_inside_a_capture(cuda):
    """A process whose first calls are captured; eager calls and replays share a status word that is valid."""
    root = Path(__file__).resolve().parent.parent
    got = subprocess.run([sys.executable, "-c", _CAPTURE_FIRST], cwd=root, capture_output=True, text=True, timeout=300)
    assert got.returncode == 0 and got.stdout.strip() == "captured first", got.stderr[-2000:]


def test_step_beside_a_patch(cuda):
    """The pages the step writes are the ones the patch operators change: attend, patch, attend."""
    s = Server(cuda, BF)
    new = [13, 4, 26, 5, 16]
    s.feed(new, 0)
    step, out = s.launch()
    s.verify(new, step, out)
    g = torch.Generator().manual_seed(4)
    total = sum(new)
    delta = (0.5 * torch.randn(total, 2, 64, generator=g)).to(cuda)
    q = torch.randn(5, 8, 64, generator=g).to(BF).to(cuda)
    dkv.scatter_into_paged_batched(delta, s.v, step.seqs, check=True)
    got = dkv.paged_decode_attention(q, s.k, s.v, step.seqs)

    def tokens(b):
        ids = step.seqs.block_tables[b, : -(-new[b] // 16)].long()
        return tuple(t[ids].reshape(-1, 2, 64)[: new[b]] for t in (s.k, s.v))

    check_attention(got, None, q, tokens, 64 ** -0.5)
    lo = sum(new[:2])
    patched = torch.stack([v for _, v in s.stored[2]]).float() + delta[lo:lo + 26]
    assert torch.equal(tokens(2)[1], patched.to(BF))
