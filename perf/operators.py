"""The paged-cache step operators as measured: planning a step (block tables, slots, positions), appending the new
tokens' K and V (with RoPE), and the attention of one new token over the pages.

Every case is plain data; lengths follow from the case, values and page order from the seed.
"""

import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # the step's bookkeeping for a handful of interactive requests: pure latency
        {"name": "plan decode 8", "op": "plan", "batch": 8, "longest": 4000, "new": 1, "block": 16, "pad": 0},
        # a full decode batch with very unequal contexts; a sixteenth of the requests need a new block
        {"name": "plan decode 512", "op": "plan", "batch": 512, "longest": 32768, "new": 1, "block": 16, "pad": 0},
        # chunked prefill of many requests, rows padded to a captured size
        {"name": "plan prefill 96", "op": "plan", "batch": 96, "longest": 6000, "new": 2048, "block": 16, "pad": 1001},
        # one decode step of a 64-request batch, Llama-3-8B heads
        {"name": "append decode 64", "op": "append", "rows": 64, "heads": 32, "kv_heads": 8, "dim": 128, "block": 16,
         "dtype": "bf16", "layout": "kv_first", "pad": 0},
        # a prefill chunk of the same shape
        {"name": "append prefill 16384", "op": "append", "rows": 16384, "heads": 32, "kv_heads": 8, "dim": 128,
         "block": 16, "dtype": "bf16", "layout": "kv_first", "pad": 0},
        # SmolLM2-135M heads, odd row count with padding rows, blocks before K/V
        {"name": "append ragged 1111", "op": "append", "rows": 1111, "heads": 9, "kv_heads": 3, "dim": 64, "block": 16,
         "dtype": "f16", "layout": "block_first", "pad": 57},
        # one short request on a small model: the smallest call
        {"name": "attend one short", "op": "attend", "batch": 1, "shortest": 333, "longest": 333, "heads": 9,
         "kv_heads": 3, "dim": 64, "block": 16, "dtype": "bf16", "layout": "kv_first", "lse": False},
        # one request with a very long context: the work has to be split over the cache's length
        {"name": "attend one long", "op": "attend", "batch": 1, "shortest": 131071, "longest": 131071, "heads": 32,
         "kv_heads": 8, "dim": 128, "block": 16, "dtype": "bf16", "layout": "kv_first", "lse": False},
        # an ordinary serving batch with unequal contexts, Llama-3-70B heads, lse for joining with a shared prefix
        {"name": "attend ragged 64", "op": "attend", "batch": 64, "shortest": 1, "longest": 8192, "heads": 64,
         "kv_heads": 8, "dim": 128, "block": 16, "dtype": "bf16", "layout": "kv_first", "lse": True},
        # many short requests in f16
        {"name": "attend short 256", "op": "attend", "batch": 256, "shortest": 1, "longest": 600, "heads": 32,
         "kv_heads": 8, "dim": 128, "block": 16, "dtype": "f16", "layout": "block_first", "lse": False},
        # an fp32 cache (the reference's own storage type), SmolLM2-135M heads
        {"name": "attend f32 24", "op": "attend", "batch": 24, "shortest": 1, "longest": 4096, "heads": 9,
         "kv_heads": 3, "dim": 64, "block": 16, "dtype": "f32", "layout": "split", "lse": True},
        # the largest: a long-context batch, Llama-3-8B heads
        {"name": "attend long 32", "op": "attend", "batch": 32, "shortest": 20000, "longest": 32768, "heads": 32,
         "kv_heads": 8, "dim": 128, "block": 16, "dtype": "bf16", "layout": "kv_first", "lse": False},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["plan", "append", "attend", "attend"])
    block = rng.choice([8, 16, 16, 32, 64, 128, 24])
    if op == "plan":
        new = rng.choice([1, 1, _log(rng, 2, 2048)])
        return {"op": op, "batch": _log(rng, 1, 96 if new > 1 else 1024), "longest": _log(rng, 16, 32768), "new": new,
                "block": block, "pad": rng.choice([0, _log(rng, 1, 1024)])}
    dim = rng.choice([32, 64, 64, 80, 96, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 3, 4, 5, 8, 8, 16])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 8, 16])
    common = {"heads": heads, "kv_heads": kv_heads, "dim": dim, "block": block,
              "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]),
              "layout": rng.choice(["kv_first", "block_first", "split"])}
    if op == "append":
        rows = _log(rng, 1, max(1, min(16384, (1 << 26) // (heads * dim))))
        return {"op": op, "rows": rows, "pad": rng.choice([0, 0, _log(rng, 1, 64)]), **common}
    batch = _log(rng, 1, 256)
    longest = _log(rng, 1, max(1, min(131072, (1 << 28) // (batch * kv_heads * dim))))
    return {"op": op, "batch": batch, "shortest": rng.choice([0, 1, longest]), "longest": longest,
            "lse": rng.random() < 0.5, **common}


# --------------------------------------------------------------------------------------------------------------
# lengths and sizes: functions of the case alone
# --------------------------------------------------------------------------------------------------------------
def _lengths(case):
    """Context lengths, spread over their logarithm between the shortest and the longest; one request is the longest."""
    lo, hi = case.get("shortest", 1), case["longest"]
    rng = random.Random(977 * case["batch"] + hi)
    lens = [_log(rng, max(lo, 1), hi) for _ in range(case["batch"])]
    if lo == 0 and len(lens) > 1:
        lens[rng.randrange(len(lens))] = 0  # an idle request of a padded batch
    lens[-1] = hi
    return lens


def _plan_sizes(case):
    """(lengths after the step, new tokens, blocks held before it, blocks needed, table width)."""
    lens = _lengths(case)
    rng = random.Random(31 * case["batch"] + case["longest"])
    new = [min(n, case["new"] if case["new"] == 1 else rng.randint(1, case["new"])) for n in lens]
    bs = case["block"]
    have = [-(-(n - k) // bs) for n, k in zip(lens, new)]
    need = [-(-n // bs) for n in lens]
    return lens, new, have, need, -(-case["longest"] // bs)


def _pages(gen, case, blocks, device):
    """K and V pages [blocks, block, kv_heads, dim] as views of the layout's storage."""
    shape = (case["block"], case["kv_heads"], case["dim"])
    dt = _DTYPES[case["dtype"]]
    if case["layout"] == "split":
        caches = [torch.empty(blocks, *shape, dtype=dt, device=device) for _ in range(2)]
    else:
        lead = (2, blocks) if case["layout"] == "kv_first" else (blocks, 2)
        caches = [torch.empty(*lead, *shape, dtype=dt, device=device)]
    for part in [p for c in caches for p in c.view(-1).split(1 << 28)]:  # in parts, each within 32-bit sizes
        part.normal_(generator=gen)
    if case["layout"] == "split":
        return caches[0], caches[1]
    return (caches[0][0], caches[0][1]) if case["layout"] == "kv_first" else (caches[0][:, 0], caches[0][:, 1])


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(1000003 * seed + 17)
    host = random.Random(seed)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    if case["op"] == "plan":
        lens, new, have, need, width = _plan_sizes(case)
        total = sum(need)
        order = torch.randperm(total + 64, device=dev, generator=gen).to(torch.int32)
        held = torch.arange(width, device=dev)[None, :] < ints(have)[:, None]
        tables = torch.zeros(len(lens), width, dtype=torch.int32, device=dev)
        n_held = sum(have)
        tables[held] = order[:n_held]
        free = order[n_held:].clone()
        return {"case": case, "lengths": ints(lens), "new": ints(new), "table_lens": ints(have), "tables": tables,
                "free": free, "rows": sum(new) + case["pad"], "longest": case["longest"]}
    if case["op"] == "append":
        rows, pad, bs, d = case["rows"], case["pad"], case["block"], case["dim"]
        blocks = rows // bs + 8
        k_pages, v_pages = _pages(gen, case, blocks, dev)
        slots = torch.randperm(blocks * bs, device=dev, generator=gen)[:rows].sort().values  # chunks of sequences
        slots = torch.cat([slots, torch.full((pad,), -1, dtype=torch.int64, device=dev)])
        positions = torch.randint(0, 8192, (rows + pad,), device=dev, generator=gen, dtype=torch.int32)
        positions[rows:] = 0
        dt = _DTYPES[case["dtype"]]
        qkv = torch.randn(rows + pad, case["heads"] + 2 * case["kv_heads"], d, device=dev, generator=gen).to(dt)
        q, k, v = qkv.split([case["heads"], case["kv_heads"], case["kv_heads"]], dim=1)  # views of one projection
        inv = 1.0 / (500000.0 ** (torch.arange(0, d, 2, dtype=torch.float32, device=dev) / d))
        ang = torch.arange(8192, dtype=torch.float32, device=dev)[:, None] * inv[None, :]
        return {"case": case, "q": q, "k": k, "v": v, "k_pages": k_pages, "v_pages": v_pages, "slots": slots,
                "positions": positions, "cos": ang.cos(), "sin": ang.sin()}
    lens = _lengths(case)
    bs = case["block"]
    need = [-(-n // bs) for n in lens]
    width, total = max(max(need), 1), sum(need)
    k_pages, v_pages = _pages(gen, case, total + 3, dev)
    order = torch.randperm(total + 3, device=dev, generator=gen).to(torch.int32)
    tables = torch.zeros(len(lens), width, dtype=torch.int32, device=dev)
    tables[torch.arange(width, device=dev)[None, :] < ints(need)[:, None]] = order[:total]
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    q = torch.randn(len(lens), case["heads"], case["dim"], device=dev, generator=gen)
    q = (q * host.uniform(1.0, 2.0)).to(_DTYPES[case["dtype"]])  # scores of a standard deviation of 1 to 2
    return {"case": case, "q": q, "k_pages": k_pages, "v_pages": v_pages, "tables": tables, "cu": ints(cu),
            "longest": max(lens)}


# --------------------------------------------------------------------------------------------------------------
# plain forms
# --------------------------------------------------------------------------------------------------------------
def _plain_plan(s):
    bs = s["case"]["block"]
    lens, new, have, tables, free = s["lengths"].long(), s["new"].long(), s["table_lens"].long(), s["tables"], s["free"]
    need = (lens + bs - 1) // bs
    extra = (need - have).clamp(min=0)
    off = extra.cumsum(0) - extra
    j = torch.arange(tables.shape[1], device=tables.device)[None, :]
    take = (j >= have[:, None]) & (j < need[:, None])
    at = (off[:, None] + j - have[:, None]).clamp(0, free.numel() - 1)
    tables.copy_(torch.where(take, free[at], tables))
    zero = torch.zeros(1, dtype=torch.int64, device=tables.device)
    cu, cu_new = torch.cat([zero, lens.cumsum(0)]), torch.cat([zero, new.cumsum(0)])
    row = torch.arange(s["rows"], device=tables.device)
    b = (row[:, None] >= cu_new[None, 1:]).sum(1)
    real = b < lens.numel()
    b = b.clamp(max=lens.numel() - 1)
    pos = torch.where(real, lens[b] - new[b] + row - cu_new[b], 0)
    slot = torch.where(real, tables[b, pos // bs].long() * bs + pos % bs, -1)
    return {"cu_seqlens": cu.int(), "cu_new": cu_new.int(), "table_lens": torch.maximum(have, need).int(),
            "tables": tables, "positions": pos.int(), "slots": slot, "used": extra.sum()[None].int()}


def _rotate(x, c, s):
    lo, hi = x.chunk(2, dim=-1)
    return torch.cat([lo * c - hi * s, hi * c + lo * s], dim=-1)


def _plain_append(s):
    bs, k_pages, v_pages = s["case"]["block"], s["k_pages"], s["v_pages"]
    c, sn = s["cos"][s["positions"].long()][:, None, :], s["sin"][s["positions"].long()][:, None, :]
    n = s["case"]["rows"]  # the padding rows are the last ones
    block, slot = s["slots"][:n] // bs, s["slots"][:n] % bs
    k_pages[block, slot] = _rotate(s["k"].float(), c, sn)[:n].to(k_pages.dtype)
    v_pages[block, slot] = s["v"][:n].to(v_pages.dtype)
    return {"q": _rotate(s["q"].float(), c, sn).to(s["q"].dtype), "k_pages": k_pages, "v_pages": v_pages}


def _plain_attend(s):
    q, tables = s["q"].float(), s["tables"].long()
    n, heads, d = q.shape
    kv = s["case"]["kv_heads"]
    lens = (s["cu"][1:] - s["cu"][:-1]).long()
    longest = max(s["longest"], 1)
    k = s["k_pages"][tables].flatten(1, 2)[:, :longest].float().transpose(1, 2)  # [n, kv, longest, d]
    dead = torch.arange(longest, device=q.device)[None, :] >= lens[:, None]
    score = (q.view(n, kv, heads // kv, d) / math.sqrt(d)) @ k.transpose(2, 3)
    del k
    score = score.masked_fill(dead[:, None, None, :], -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, 0.0)
    p = (score - top).exp()
    total = p.sum(-1, keepdim=True)
    v = s["v_pages"][tables].flatten(1, 2)[:, :longest].float().transpose(1, 2)
    v = v.masked_fill(dead[:, None, :, None], 0.0)
    out = (p @ v) / torch.where(total > 0, total, 1.0)
    out = out.reshape(n, heads, d).to(s["q"].dtype)
    if not s["case"]["lse"]:
        return {"out": out}
    return {"out": out, "lse": (top + total.log()).reshape(n, heads)}


def run(state):
    op = state["case"]["op"]
    if own:
        import deltakv_b200 as dkv

        if op == "plan":
            step = dkv.plan_paged_step(state["lengths"], state["tables"], state["case"]["block"], rows=state["rows"],
                                       max_seq_len=state["longest"], new_lengths=state["new"],
                                       table_lens=state["table_lens"], free_blocks=state["free"])
            return {"cu_seqlens": step.seqs.cu_seqlens, "cu_new": step.cu_new, "table_lens": step.seqs.table_lens,
                    "tables": step.seqs.block_tables, "positions": step.positions, "slots": step.slots,
                    "used": step.blocks_used}
        if op == "append":
            q = dkv.append_into_paged(state["k"], state["v"], state["k_pages"], state["v_pages"], state["slots"],
                                      q=state["q"], positions=state["positions"], rope=(state["cos"], state["sin"]))
            return {"q": q, "k_pages": state["k_pages"], "v_pages": state["v_pages"]}
        seqs = dkv.SeqBatchTensors(cu_seqlens=state["cu"], block_tables=state["tables"], max_seq_len=state["longest"])
        if state["case"]["lse"]:
            out, lse = dkv.paged_decode_attention(state["q"], state["k_pages"], state["v_pages"], seqs, return_lse=True)
            return {"out": out, "lse": lse}
        return {"out": dkv.paged_decode_attention(state["q"], state["k_pages"], state["v_pages"], seqs)}
    return {"plan": _plain_plan, "append": _plain_append, "attend": _plain_attend}[op](state)


def work(case):
    size = {"bf16": 2, "f16": 2, "f32": 4}.get(case.get("dtype"), 4)
    if case["op"] == "plan":
        lens, new, have, need, _ = _plan_sizes(case)
        b, bs = len(lens), case["block"]
        taken = sum(n - h for n, h in zip(need, have))
        touched = sum(-(-n // bs) - (n - k) // bs for n, k in zip(lens, new))
        rows = sum(new) + case["pad"]
        return {"bytes": 12 * b + 4 * touched + 4 * (3 * b + 3) + 4 * taken + 12 * rows, "flops": 0}
    if case["op"] == "append":
        rows, h, kv, d = case["rows"] + case["pad"], case["heads"], case["kv_heads"], case["dim"]
        return {"bytes": size * d * (2 * h * rows + 4 * kv * case["rows"]) + rows * (12 + 4 * d),
                "flops": 3 * d * (h + kv) * rows}
    tokens, d = sum(_lengths(case)), case["dim"]
    kv_bytes = 2 * tokens * case["kv_heads"] * d * size
    io = 2 * case["batch"] * case["heads"] * d * size
    blocks = sum(-(-n // case["block"]) for n in _lengths(case))
    return {"bytes": kv_bytes + io + 4 * blocks + 4 * case["batch"], "flops": 4 * tokens * case["heads"] * d}


# --------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# --------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] == "plan":
        return None  # whole numbers: equal or wrong
    s = prepare(case, seed)
    if case["op"] == "append":
        n, d, bs = case["rows"], case["dim"], case["block"]
        ang_c, ang_s = s["cos"].double(), s["sin"].double()
        turn = torch.complex(ang_c, ang_s)[s["positions"].long()].unsqueeze(1)  # cos + i sin, on lo + i hi

        def rot(x):
            x = x.double()
            z = torch.complex(x[..., : d // 2].contiguous(), x[..., d // 2:].contiguous()) * turn
            return torch.cat([z.real, z.imag], dim=-1)

        k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
        at = (s["slots"][:n].div(bs, rounding_mode="floor"), s["slots"][:n].remainder(bs))
        k_pages.index_put_(at, rot(s["k"])[:n])
        v_pages.index_put_(at, s["v"][:n].double())
        return {"q": rot(s["q"]), "k_pages": k_pages, "v_pages": v_pages}
    heads, kv, d, bs = case["heads"], case["kv_heads"], case["dim"], case["block"]
    outs, lses = [], []
    for b, n in enumerate(_lengths(case)):
        if n == 0:
            outs.append(torch.zeros(heads, d, dtype=torch.float64, device="cuda"))
            lses.append(torch.full((heads,), -math.inf, dtype=torch.float64, device="cuda"))
            continue
        ids = s["tables"][b, : -(-n // bs)].long()
        k = s["k_pages"].index_select(0, ids).reshape(-1, kv, d)[:n].double()
        v = s["v_pages"].index_select(0, ids).reshape(-1, kv, d)[:n].double()
        q = s["q"][b].double().view(kv, heads // kv, d)
        score = torch.einsum("hgd,nhd->hgn", q, k) * d ** -0.5
        lse = torch.logsumexp(score, -1)
        outs.append(torch.einsum("hgn,nhd->hgd", torch.exp(score - lse[..., None]), v).reshape(heads, d))
        lses.append(lse.reshape(heads))
    got = {"out": torch.stack(outs)}
    if case["lse"]:
        got["lse"] = torch.stack(lses)
    return got
