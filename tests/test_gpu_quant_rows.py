"""Blocks of 8-bit pages that one call would write in two places: refused where it is asked to check, recorded otherwise."""

from __future__ import annotations

import pytest
import torch

import deltakv_b200 as dkv
from deltakv_b200 import _lib as L
from deltakv_b200 import ops
from tests.test_gpu_quant import KINDS, bits

pytestmark = pytest.mark.gpu


def cache(cuda, kind, blocks, block, n_kv=2, hd=32):
    pages = torch.zeros(2, blocks, block, n_kv, hd, dtype=torch.uint8, device=cuda).view(kind)
    return pages, torch.ones(2, blocks, n_kv, device=cuda)


def append(pages, scales, slots, check=True):
    rows = slots.numel()
    x = torch.randn(rows, *pages.shape[3:], device=slots.device)
    dkv.append_into_paged(x, x, pages[0], pages[1], slots, kv_scales=(scales[0], scales[1]), check=check)


# slots of blocks of 16, by block and slot
APART = {
    "a row between": [(3, 0), (5, 0), (3, 1)],
    "a row of none between": [(3, 0), (-1, 0), (3, 1)],
    "a row beyond the pages between": [(3, 2), (1 << 30, 0), (3, 3)],
    "the last rows": [(0, i) for i in range(16)] + [(1, 0), (0, 3)],
    "neighbouring windows": [(i, 0) for i in range(40)] + [(7, 1)],
}


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("case", APART)
@pytest.mark.parametrize("hd", [32, 17])
def test_append_refuses_rows_apart(cuda, kind, case, hd):
    slots = torch.tensor([b * 16 + i if b >= 0 else -1 for b, i in APART[case]], device=cuda)
    pages, scales = cache(cuda, kind, 64, 16, hd=hd)
    with pytest.raises(dkv.DkvError, match="two places") as e:
        append(pages, scales, slots)
    assert e.value.status == L.DKV_ERR_BLOCK_TWICE
    assert torch.all(bits(pages) == 0) and torch.all(scales == 1)
    assert int(ops.status_word(cuda).t) == 0  # (the refusal has a word of its own)


@pytest.mark.parametrize("rows", [300, 5000, 20000])
def test_append_of_many_blocks(cuda, rows):
    """Single rows of distinct blocks in any order pass; one block twice anywhere among them does not (several watchers' worth)."""
    g = torch.Generator().manual_seed(rows)
    pages, scales = cache(cuda, KINDS[0], rows + 9, 2)
    order = torch.randperm(rows + 9, generator=g)[:rows]
    slots = (order * 2 + torch.randint(0, 2, (rows,), generator=g)).to(cuda)
    append(pages, scales, slots)
    pages, scales = cache(cuda, KINDS[0], rows + 9, 2)
    for first, second in ((0, rows - 1), (rows // 2, rows // 2 + 2), (17, rows // 3), (rows - 3, rows - 1)):
        twice = slots.clone()
        twice[second] = twice[first] ^ 1
        with pytest.raises(dkv.DkvError, match="two places"):
            append(pages, scales, twice)
    assert torch.all(bits(pages) == 0) and torch.all(scales == 1)


def test_append_of_runs_passes(cuda):
    """Runs of any length, over several windows, in blocks of any order; slots within a run in any order."""
    g = torch.Generator().manual_seed(1)
    block = 32
    pages, scales = cache(cuda, KINDS[0], 900, block)
    slots = []
    for b in torch.randperm(900, generator=g).tolist():
        n = int(torch.randint(1, block + 1, (1,), generator=g))
        slots += [b * block + i for i in torch.randperm(block, generator=g)[:n].tolist()]
        slots += [-1] * int(torch.randint(0, 2, (1,), generator=g))
    append(pages, scales, torch.tensor(slots, device=cuda))
    append(pages, scales, torch.tensor(slots[:1], device=cuda))


def test_append_records_rows_apart(cuda):
    """Without a check the launch itself records it.  One KV head and a window of 8 or 16 rows: the first and the third of its runs, of one
    block, are one warp's, one after the other."""
    rows, block = 16000, 4
    pages, scales = cache(cuda, KINDS[0], rows + 1, block, n_kv=1)
    slots = torch.arange(rows, device=cuda) * block
    slots[32:36] = torch.tensor([32 * block, 32 * block + 1, 33 * block, 32 * block + 2], device=cuda)
    append(pages, scales, slots, check=False)
    word = ops.status_word(cuda)
    assert int(word.t) == L.DKV_ERR_BLOCK_TWICE
    with pytest.raises(dkv.DkvError, match="two places"):
        word.raise_if_set("append_into_paged")
    slots[35] = 35 * block
    append(pages, scales, slots, check=False)
    assert int(word.t) == 0


def batch(cuda, lens, tables, width=None):
    cu = torch.tensor([0, *lens], dtype=torch.int32).cumsum(0).int()
    width = width or max(len(t) for t in tables)
    table = torch.full((len(lens), width), 2, dtype=torch.int32)  # entries behind a sequence's end say nothing
    for row, t in zip(table, tables):
        row[: len(t)] = torch.as_tensor(t, dtype=torch.int32)
    return dkv.SeqBatchTensors(cu_seqlens=cu.to(cuda), block_tables=table.to(cuda), max_seq_len=max(lens))


def patch(pages, scales, lens, seqs, check=True, rows=None):
    delta = torch.randn(sum(lens) if rows is None else rows, *pages.shape[2:], device=pages.device)
    dkv.scatter_into_paged_batched(delta, pages, seqs, page_scales=scales, check=check)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd", [32, 17])
@pytest.mark.parametrize("lens,tables", [
    ([40, 40], [[1, 5, 3], [1, 7, 9]]),                       # a shared prefix
    ([40], [[4, 5, 4]]),                                      # a block twice in one sequence
    ([16, 0, 1] + [0] * 100 + [5], [[1], [], [3]] + [[]] * 100 + [[1]]),
])
def test_patch_refuses_shared_blocks(cuda, kind, hd, lens, tables):
    pages, scales = (x[0] for x in cache(cuda, kind, 12, 16, hd=hd))
    with pytest.raises(dkv.DkvError, match="two places") as e:
        patch(pages, scales, lens, batch(cuda, lens, tables))
    assert e.value.status == L.DKV_ERR_BLOCK_TWICE
    assert torch.all(bits(pages) == 0) and torch.all(scales == 1)
    assert int(ops.status_word(cuda).t) == 0


def test_patch_of_what_is_not_shared_passes(cuda):
    """Rows that the call does not have, entries behind a sequence's end and blocks outside the cache count for nothing."""
    pages, scales = (x[0] for x in cache(cuda, KINDS[0], 12, 16))
    patch(pages, scales, [16, 7], batch(cuda, [16, 7], [[2], [5]], width=6))
    with pytest.raises(dkv.DkvError, match="invalid argument"):  # (fewer rows than the lengths say: the second sequence has none)
        patch(pages, scales, [16, 16], batch(cuda, [16, 16], [[3], [3]]), rows=16)
    with pytest.raises(dkv.DkvError, match="outside"):
        patch(pages, scales, [32], batch(cuda, [32], [[50, 50]]))


@pytest.mark.parametrize("n_seq", [1, 70, 4000])
def test_patch_of_many_blocks(cuda, n_seq):
    total, block = 24000, 2
    g = torch.Generator().manual_seed(n_seq)
    pages, scales = (x[0] for x in cache(cuda, KINDS[0], total, block))
    order = torch.randperm(total, generator=g).to(torch.int32)
    cut = torch.cat([torch.zeros(1, dtype=torch.long), torch.randint(0, 9000, (n_seq - 1,), generator=g).sort()[0], torch.tensor([9000])])
    tables = [order[a:b] for a, b in zip(cut[:-1].tolist(), cut[1:].tolist())]
    lens = [2 * len(t) - (1 if len(t) and i % 3 else 0) for i, t in enumerate(tables)]
    patch(pages, scales, lens, batch(cuda, lens, tables))
    pages, scales = (x[0] for x in cache(cuda, KINDS[0], total, block))
    for first, second in ((0, 8999), (4000, 4001), (123, 7000)):
        twice = order.clone()
        twice[second] = twice[first]
        with pytest.raises(dkv.DkvError, match="two places"):
            patch(pages, scales, lens, batch(cuda, lens, [twice[a:b] for a, b in zip(cut[:-1].tolist(), cut[1:].tolist())]))
    assert torch.all(bits(pages) == 0) and torch.all(scales == 1)


def test_patch_records_shared_blocks(cuda):
    """Without a check.  Blocks of one slot and one head, a window of 16 rows: its first and fifth runs are one warp's, one after the other."""
    rows = 20000
    pages, scales = (x[0] for x in cache(cuda, KINDS[0], rows, 1, n_kv=1))
    table = torch.arange(rows)
    table[36] = 32
    patch(pages, scales, [rows], batch(cuda, [rows], [table]), check=False)
    word = ops.status_word(cuda)
    assert int(word.t) == L.DKV_ERR_BLOCK_TWICE
    word.t.zero_()
    patch(pages, scales, [rows], batch(cuda, [rows], [torch.arange(rows)]), check=False)
    assert int(word.t) == 0
