"""The 8-bit paged cache as measured: quantising K and V as they are appended (with RoPE), reading them back, adding a
patch to them, the attention of one new token over them; and the rotary forms (interleaved, part of the head, far
positions) of the append into 16-bit pages.

Pages hold e4m3 or int8 codes; a value is its code times the fp32 scale of its block and KV head.  The scale of a block
that holds nothing yet is the least power of two (e4m3) or amax / 127 (int8) that its values fit; one that is too
small for new values grows by powers of two, and what the block held is rounded once more.  Storing slot 0 begins a block.

Every case is plain data; lengths follow from the case, values and page order from the seed.
"""

import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32,
           "e4m3": torch.float8_e4m3fn, "int8": torch.int8}
_SIZES = {"bf16": 2, "f16": 2, "f32": 4, "e4m3": 1, "int8": 1}


def listed():
    llama = {"heads": 32, "kv_heads": 8, "dim": 128, "block": 16, "dtype": "bf16", "layout": "kv_first"}
    smol = {"heads": 9, "kv_heads": 3, "dim": 64, "block": 16, "dtype": "bf16", "layout": "block_first"}
    whole = {"rot": 128, "interleaved": False, "far": 8192}
    return [
        # one decode step of a 64-request batch, Llama-3-8B heads: each row ends a block that holds earlier tokens
        {"name": "append8 decode 64", "op": "append", "rows": 64, "new": 1, "pad": 0, "pages": "e4m3", **whole, **llama},
        # prefill chunks of the same shape
        {"name": "append8 prefill 16384", "op": "append", "rows": 16384, "new": 2048, "pad": 0, "pages": "e4m3", **whole,
         **llama},
        # SmolLM2-135M heads in int8, short chunks that begin and end inside blocks, padding rows
        {"name": "append8 ragged 1111", "op": "append", "rows": 1111, "new": 37, "pad": 57, "pages": "int8", "rot": 64,
         "interleaved": False, "far": 8192, **{**smol, "dtype": "f16"}},
        # rotary forms into 16-bit pages: a decode step, pairs side by side, half the head, positions of a long context
        {"name": "rotate decode 64", "op": "append", "rows": 64, "new": 1, "pad": 0, "pages": "bf16", "rot": 64,
         "interleaved": True, "far": 131072, **llama},
        # the same for prefill chunks, rotate-half on a part of the head
        {"name": "rotate prefill 16384", "op": "append", "rows": 16384, "new": 2048, "pad": 0, "pages": "bf16", "rot": 64,
         "interleaved": False, "far": 131072, **llama},
        # reading one short request's K back: the smallest call
        {"name": "read one 333", "op": "read", "batch": 1, "shortest": 333, "longest": 333, "pages": "e4m3", **smol},
        # reading the K of a whole batch back
        {"name": "read ragged 64", "op": "read", "batch": 64, "shortest": 1, "longest": 8192, "pages": "int8", **llama},
        # a changed adapter's delta on one short request
        {"name": "patch one 333", "op": "patch", "batch": 1, "shortest": 333, "longest": 333, "pages": "e4m3", **smol},
        # the same on a whole batch with unequal contexts
        {"name": "patch ragged 64", "op": "patch", "batch": 64, "shortest": 1, "longest": 8192, "pages": "e4m3", **llama},
        # attention of one short request on a small model: latency
        {"name": "attend8 one short", "op": "attend", "batch": 1, "shortest": 333, "longest": 333, "pages": "e4m3",
         "lse": False, **smol},
        # an ordinary serving batch with unequal contexts, Llama-3-70B heads, lse for joining with a shared prefix
        {"name": "attend8 ragged 64", "op": "attend", "batch": 64, "shortest": 1, "longest": 8192, "pages": "int8",
         "lse": True, **{**llama, "heads": 64, "dtype": "f16"}},
        # the largest: a long-context batch, Llama-3-8B heads
        {"name": "attend8 long 32", "op": "attend", "batch": 32, "shortest": 20000, "longest": 32768, "pages": "e4m3",
         "lse": False, **llama},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "append", "read", "patch", "attend", "attend", "attend"])
    dim = rng.choice([32, 64, 64, 80, 96, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 3, 4, 5, 8, 8, 16])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 8, 16])
    common = {"heads": heads, "kv_heads": kv_heads, "dim": dim, "block": rng.choice([8, 16, 16, 32, 64, 128, 24]),
              "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]), "pages": rng.choice(["e4m3", "e4m3", "int8"]),
              "layout": rng.choice(["kv_first", "block_first", "split"])}
    if op == "append":
        if rng.random() < 0.4:
            common["pages"] = common["dtype"]
        rows = _log(rng, 1, max(1, min(16384, (1 << 26) // (heads * dim))))
        return {"op": op, "rows": rows, "new": rng.choice([1, _log(rng, 2, 2048)]),
                "pad": rng.choice([0, 0, _log(rng, 1, 64)]), "rot": rng.choice([dim, dim, dim // 2, dim // 4]),
                "interleaved": rng.random() < 0.5, "far": rng.choice([8192, 131072]), **common}
    batch = _log(rng, 1, 256)
    longest = _log(rng, 1, max(1, min(131072, (1 << (28 if op == "attend" else 26)) // (batch * kv_heads * dim))))
    case = {"op": op, "batch": batch, "shortest": rng.choice([0, 1, longest]), "longest": longest, **common}
    return {**case, "lse": rng.random() < 0.5} if op == "attend" else case


# --------------------------------------------------------------------------------------------------------------
# lengths and sizes: functions of the case alone
# --------------------------------------------------------------------------------------------------------------
def _lengths(case):
    """Context lengths, spread over their logarithm between the shortest and the longest; one request is the longest."""
    lo, hi = case["shortest"], case["longest"]
    rng = random.Random(977 * case["batch"] + hi)
    lens = [_log(rng, max(lo, 1), hi) for _ in range(case["batch"])]
    if lo == 0 and len(lens) > 1:
        lens[rng.randrange(len(lens))] = 0  # an idle request of a padded batch
    lens[-1] = hi
    return lens


def _chunks(case):
    """(slot in its first block, new tokens) of each sequence of an append; a third of the chunks begin a block."""
    rng = random.Random(31 * case["rows"] + case["new"])
    got, left = [], case["rows"]
    while left:
        n = min(left, rng.randint(1, case["new"]))
        got.append((rng.choice([0, rng.randrange(case["block"]), rng.randrange(case["block"])]), n))
        left -= n
    return got


def _pages(gen, case, blocks, device):
    """K and V pages [blocks, block, kv_heads, dim] as views of the layout's storage, normal values; 8 bits with scales."""
    shape = (case["block"], case["kv_heads"], case["dim"])
    dt = _DTYPES[case["pages"]]
    if case["layout"] == "split":
        caches = [torch.empty(blocks, *shape, dtype=dt, device=device) for _ in range(2)]
    else:
        lead = (2, blocks) if case["layout"] == "kv_first" else (blocks, 2)
        caches = [torch.empty(*lead, *shape, dtype=dt, device=device)]
    spread = {"e4m3": 90.0, "int8": 28.0}.get(case["pages"], 1.0)  # the largest of a block's head near the end of its codes
    for part in [p for c in caches for p in c.view(-1).split(1 << 28)]:  # in parts, each within 32-bit sizes
        x = torch.empty(part.shape, dtype=torch.float32 if dt == torch.float32 else torch.float16, device=device)
        part.copy_(x.normal_(0.0, spread, generator=gen).clamp_(-4.5 * spread, 4.5 * spread))
    k, v = caches if case["layout"] == "split" else caches[0] if case["layout"] == "kv_first" else caches[0].unbind(1)
    if _SIZES[case["pages"]] > 1:
        return k, v, None, None
    scales = torch.randint(-1, 2, (2, blocks, case["kv_heads"]), generator=gen, device=device).float().exp2() / 128.0
    if case["pages"] == "int8":
        scales *= 1.0 + torch.rand(scales.shape, generator=gen, device=device)
    return k, v, scales[0], scales[1]


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(1000003 * seed + 17)
    host = random.Random(seed)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    dt, bs, d = _DTYPES[case["dtype"]], case["block"], case["dim"]
    if case["op"] == "append":
        rows, pad = case["rows"], case["pad"]
        chunks = _chunks(case)
        need = [(at + n + bs - 1) // bs for at, n in chunks]
        blocks = sum(need) + 8
        order = torch.randperm(blocks, device=dev, generator=gen)
        counts = torch.tensor([n for _, n in chunks], device=dev)
        first = torch.tensor([at for at, _ in chunks], device=dev)
        held = torch.tensor([0] + need[:-1], device=dev).cumsum(0)
        seq = torch.repeat_interleave(torch.arange(len(chunks), device=dev), counts)
        token = torch.arange(rows, device=dev) - (counts.cumsum(0) - counts)[seq] + first[seq]
        slots = order[held[seq] + token // bs] * bs + token % bs
        slots = torch.cat([slots, torch.full((pad,), -1, dtype=torch.int64, device=dev)])
        before = torch.randint(0, (case["far"] - 4096) // bs, (len(chunks),), device=dev, generator=gen) * bs
        positions = torch.cat([(before[seq] + token).int(), torch.zeros(pad, dtype=torch.int32, device=dev)])
        k_pages, v_pages, k_scales, v_scales = _pages(gen, case, blocks, dev)
        qkv = torch.randn(rows + pad, case["heads"] + 2 * case["kv_heads"], d, device=dev, generator=gen)
        qkv = qkv.mul_(torch.rand(rows + pad, 1, 1, device=dev, generator=gen) + 0.5).to(dt)  # tokens differ in size
        q, k, v = qkv.split([case["heads"], case["kv_heads"], case["kv_heads"]], dim=1)  # views of one projection
        rot = case["rot"]
        inv = 500000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=dev) / rot)
        if case["far"] > 8192:
            inv = inv * 8192 / case["far"]  # positions of a long context on the angles of a shorter one
        ang = torch.arange(case["far"], dtype=torch.float64, device=dev)[:, None] * inv[None, :]
        return {"case": case, "q": q, "k": k, "v": v, "k_pages": k_pages, "v_pages": v_pages, "k_scales": k_scales,
                "v_scales": v_scales, "slots": slots, "positions": positions, "cos": ang.cos().float(),
                "sin": ang.sin().float()}
    lens = _lengths(case)
    need = [-(-n // bs) for n in lens]
    width, total = max(max(need), 1), sum(need)
    k_pages, v_pages, k_scales, v_scales = _pages(gen, case, total + 3, dev)
    order = torch.randperm(total + 3, device=dev, generator=gen).to(torch.int32)
    tables = torch.zeros(len(lens), width, dtype=torch.int32, device=dev)
    tables[torch.arange(width, device=dev)[None, :] < ints(need)[:, None]] = order[:total]
    cu = torch.cat([torch.zeros(1, dtype=torch.int32, device=dev), ints(lens).cumsum(0).int()])
    s = {"case": case, "k_pages": k_pages, "v_pages": v_pages, "k_scales": k_scales, "v_scales": v_scales,
         "tables": tables, "cu": cu, "longest": max(lens), "rows": sum(lens)}
    if case["op"] == "patch":
        delta = torch.randn(sum(lens), case["kv_heads"], d, device=dev, generator=gen)
        s["delta"] = delta.mul_(0.05).to(dt)
    if case["op"] == "attend":
        q = torch.randn(len(lens), case["heads"], d, device=dev, generator=gen)
        s["q"] = (q * host.uniform(1.0, 2.0)).to(dt)  # scores of a standard deviation of 1 to 2
    return s


# --------------------------------------------------------------------------------------------------------------
# plain forms
# --------------------------------------------------------------------------------------------------------------
def _bytes(pages):
    return pages.view(torch.uint8) if pages.element_size() == 1 else pages


def _values(pages, scales, at):
    """The values of pages[at], in 32 bits."""
    return _bytes(pages)[at].view(pages.dtype).float() * scales[at][..., None, :, None]


def _coded(x, scale, dtype):
    y = x * torch.where(scale > 0, scale.reciprocal(), 0.0)
    return y.to(dtype) if dtype == torch.float8_e4m3fn else y.round().clamp(-127, 127).to(dtype)


def _scale_for(top, held, dtype):
    """The scale that `top` fits: that of a block that holds nothing (held 0), or the held one grown by powers of two."""
    if dtype == torch.float8_e4m3fn:
        m, e = torch.frexp(top / 448.0)
        new = torch.ldexp(torch.ones_like(top), e - (m == 0.5).int())
    else:
        new = top / 127.0
    new = torch.where(top > 0, new.clamp(min=2.0 ** -126), 0.0)
    m, e = torch.frexp(top / ((448.0 if dtype == torch.float8_e4m3fn else 127.5) * held))
    grown = torch.ldexp(held, (e - (m == 0.5).int()).clamp(min=0))
    return torch.where(held > 0, torch.where(top > 0, grown, held), new)


def _plain_store(pages, scales, x, block, slot):
    """x [rows, heads, dim] into pages[block, slot], whose blocks' scales grow where they have to."""
    touched = torch.zeros(pages.shape[0], dtype=torch.bool, device=x.device)
    touched[block] = True
    begun = torch.zeros_like(touched)
    begun[block[slot == 0]] = True
    top = torch.zeros_like(scales).index_reduce_(0, block, x.abs().amax(-1), "amax")
    held = torch.where(begun[:, None], 0.0, scales)
    scale = _scale_for(top, held, pages.dtype)
    again = touched[:, None] & (held != scale) & ~begun[:, None]
    old = _coded(pages.float() * held[:, None, :, None], scale[:, None, :, None], pages.dtype)
    _bytes(pages).copy_(torch.where(again[:, None, :, None], _bytes(old), _bytes(pages)))
    scales.copy_(torch.where(touched[:, None], scale, scales))
    _bytes(pages)[block, slot] = _bytes(_coded(x, scale[block][..., None], pages.dtype))


def _rotate(x, c, s, interleaved):
    rot = 2 * c.shape[-1]
    x, rest = x[..., :rot], x[..., rot:]
    lo, hi = (x[..., ::2], x[..., 1::2]) if interleaved else x.chunk(2, dim=-1)
    lo, hi = lo * c - hi * s, hi * c + lo * s
    y = torch.stack([lo, hi], dim=-1).flatten(-2) if interleaved else torch.cat([lo, hi], dim=-1)
    return torch.cat([y, rest], dim=-1)


def _plain_append(s):
    case = s["case"]
    c, sn = s["cos"][s["positions"].long()][:, None, :], s["sin"][s["positions"].long()][:, None, :]
    n = case["rows"]  # the padding rows are the last ones
    block, slot = s["slots"][:n] // case["block"], s["slots"][:n] % case["block"]
    k = _rotate(s["k"].float(), c, sn, case["interleaved"])[:n]
    q = _rotate(s["q"].float(), c, sn, case["interleaved"]).to(s["q"].dtype)
    if s["k_scales"] is None:
        s["k_pages"][block, slot] = k.to(s["k_pages"].dtype)
        s["v_pages"][block, slot] = s["v"][:n].to(s["v_pages"].dtype)
    else:
        _plain_store(s["k_pages"], s["k_scales"], k, block, slot)
        _plain_store(s["v_pages"], s["v_scales"], s["v"][:n].float(), block, slot)
    return q


def _where(s):
    """Sequence, block and slot of each row."""
    row = torch.arange(s["rows"], device=s["cu"].device)
    seq = torch.searchsorted(s["cu"][1:].long(), row, right=True)
    token = row - s["cu"][seq].long()
    return s["tables"][seq, token // s["case"]["block"]].long(), token % s["case"]["block"]


def _plain_read(s):
    block, slot = _where(s)
    codes = _bytes(s["k_pages"])[block, slot].view(s["k_pages"].dtype)
    return (codes.float() * s["k_scales"][block][..., None]).to(_DTYPES[s["case"]["dtype"]])


def _plain_patch(s):
    pages, scales, bs = s["k_pages"], s["k_scales"], s["case"]["block"]
    block, slot = _where(s)
    codes = _bytes(pages)[block, slot].view(pages.dtype)
    x = codes.float() * scales[block][..., None] + s["delta"].float()
    full = torch.zeros(pages.shape[0], dtype=torch.bool, device=x.device)
    full[block[slot == bs - 1]] = True  # all of it is stored anew; a block's rest keeps what it holds
    held = torch.where(full[:, None], 0.0, scales)
    top = torch.zeros_like(scales).index_reduce_(0, block, x.abs().amax(-1), "amax")
    touched = torch.zeros_like(full)
    touched[block] = True
    scale = torch.where(touched[:, None], _scale_for(top, held, pages.dtype), scales)
    again = touched[:, None] & (held != scale) & ~full[:, None]
    old = _coded(pages.float() * held[:, None, :, None], scale[:, None, :, None], pages.dtype)
    _bytes(pages).copy_(torch.where(again[:, None, :, None], _bytes(old), _bytes(pages)))
    scales.copy_(scale)
    _bytes(pages)[block, slot] = _bytes(_coded(x, scale[block][..., None], pages.dtype))


def _plain_attend(s):
    q, tables = s["q"].float(), s["tables"].long()
    n, heads, d = q.shape
    kv = s["case"]["kv_heads"]
    lens = (s["cu"][1:] - s["cu"][:-1]).long()
    longest = max(s["longest"], 1)
    k = _values(s["k_pages"], s["k_scales"], tables).flatten(1, 2)[:, :longest].transpose(1, 2)  # [n, kv, longest, d]
    dead = torch.arange(longest, device=q.device)[None, :] >= lens[:, None]
    score = (q.view(n, kv, heads // kv, d) / math.sqrt(d)) @ k.transpose(2, 3)
    del k
    score = score.masked_fill(dead[:, None, None, :], -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, 0.0)
    p = (score - top).exp()
    total = p.sum(-1, keepdim=True)
    v = _values(s["v_pages"], s["v_scales"], tables).flatten(1, 2)[:, :longest].transpose(1, 2)
    v = v.masked_fill(dead[:, None, :, None], 0.0)
    out = (p @ v) / torch.where(total > 0, total, 1.0)
    out = out.reshape(n, heads, d).to(s["q"].dtype)
    if not s["case"]["lse"]:
        return {"out": out}
    return {"out": out, "lse": (top + total.log()).reshape(n, heads)}


def _cache(pages, scales):
    """What a cache holds: values, or e4m3 numbers with their scales."""
    if scales is None:
        return {"values": pages}
    if pages.dtype == torch.float8_e4m3fn:
        return {"codes": pages, "scales": scales}
    return {"values": pages * scales[:, None, :, None], "scales": scales}


def run(state):
    case, k_scales, v_scales = state["case"], state["k_scales"], state["v_scales"]
    op, k_pages, v_pages = case["op"], state["k_pages"], state["v_pages"]
    if op == "append":
        if own:
            import deltakv_b200 as dkv

            q = dkv.append_into_paged(state["k"], state["v"], k_pages, v_pages, state["slots"], q=state["q"],
                                      positions=state["positions"], rope=(state["cos"], state["sin"]),
                                      rotary_dim=case["rot"], interleaved=case["interleaved"],
                                      kv_scales=None if k_scales is None else (k_scales, v_scales))
        else:
            q = _plain_append(state)
        return {"q": q, "k": _cache(k_pages, k_scales), "v": _cache(v_pages, v_scales)}
    if not own:
        if op == "patch":
            _plain_patch(state)
            return _cache(k_pages, k_scales)
        return {"values": _plain_read(state)} if op == "read" else _plain_attend(state)
    import deltakv_b200 as dkv

    seqs = dkv.SeqBatchTensors(cu_seqlens=state["cu"], block_tables=state["tables"], max_seq_len=state["longest"])
    if op == "read":
        return {"values": dkv.gather_from_paged_batched(k_pages, seqs, state["rows"], page_scales=k_scales,
                                                        dtype=_DTYPES[case["dtype"]])}
    if op == "patch":
        dkv.scatter_into_paged_batched(state["delta"], k_pages, seqs, page_scales=k_scales)
        return _cache(k_pages, k_scales)
    got = dkv.paged_decode_attention(state["q"], k_pages, v_pages, seqs, kv_scales=(k_scales, v_scales),
                                     return_lse=case["lse"])
    return {"out": got[0], "lse": got[1]} if case["lse"] else {"out": got}


def work(case):
    size, code, kv, d, bs = _SIZES[case["dtype"]], _SIZES[case["pages"]], case["kv_heads"], case["dim"], case["block"]
    if case["op"] == "append":
        rows, h = case["rows"] + case["pad"], case["heads"]
        blocks = sum((at + n + bs - 1) // bs for at, n in _chunks(case)) if code == 1 else 0
        return {"bytes": size * d * (2 * h * rows + 2 * kv * case["rows"]) + 2 * code * d * kv * case["rows"]
                + 8 * kv * blocks + rows * (12 + 4 * case["rot"]), "flops": 3 * case["rot"] * (h + kv) * rows}
    tokens = sum(_lengths(case))
    blocks = sum(-(-n // bs) for n in _lengths(case))
    head = 4 * blocks + 4 * case["batch"]
    if case["op"] == "read":
        return {"bytes": tokens * kv * d * (1 + size) + 4 * kv * blocks + head, "flops": tokens * kv * d}
    if case["op"] == "patch":
        return {"bytes": tokens * kv * d * (2 + size) + 8 * kv * blocks + head, "flops": 4 * tokens * kv * d}
    io = 2 * case["batch"] * case["heads"] * d * size
    return {"bytes": 2 * tokens * kv * d + 8 * kv * blocks + io + head, "flops": 4 * tokens * case["heads"] * d}


# --------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# --------------------------------------------------------------------------------------------------------------
def _round8(x, kind):
    """The nearest code, as a number; the one with an even last bit where two are as near."""
    if kind == "int8":
        return torch.round(x).clamp(-127, 127)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def _exact_store(pages, scales, x, block, slot, whole, kind):
    """Numbers and scales after x [rows, heads, dim] went into pages[block, slot]; `whole`: blocks of which nothing is kept."""
    numbers, scale = pages.double(), scales.double()
    ids, at = torch.unique(block, return_inverse=True)
    top = torch.zeros(len(ids), x.shape[1], dtype=torch.float64, device=x.device)
    top.scatter_reduce_(0, at[:, None].expand(-1, x.shape[1]), x.abs().amax(-1), "amax")
    old = torch.where(torch.isin(ids, whole)[:, None], 0.0, scale[ids])
    new = torch.where(top > 0, torch.exp2(torch.ceil(torch.log2(top / 448))) if kind == "e4m3" else top / 127, 0.0)
    more = torch.ceil(torch.log2(top / (old * (448 if kind == "e4m3" else 127.5)))).clamp(min=0)
    new = torch.where(old > 0, old * torch.exp2(more), new)
    kept = _round8(numbers[ids] * (old / torch.where(new > 0, new, 1.0))[:, None, :, None], kind)
    numbers[ids] = torch.where(((old != new) & (old > 0))[:, None, :, None], kept, numbers[ids])
    scale[ids] = new
    numbers[block, slot] = _round8(x / torch.where(new > 0, new, 1.0)[at][..., None], kind)
    return {"codes": numbers, "scales": scale} if kind == "e4m3" else {"values": None, "scales": scale}


def exact(case, seed):
    s = prepare(case, seed)
    kind, d, bs, kv = case["pages"], case["dim"], case["block"], case["kv_heads"]
    if case["op"] == "append":
        n, rot = case["rows"], case["rot"]
        turn = torch.complex(s["cos"].double(), s["sin"].double())[s["positions"].long()].unsqueeze(1)
        i = torch.arange(rot // 2, device="cuda")
        one, two = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + rot // 2)

        def turned(x):
            y = x.double()
            z = torch.complex(y[..., one], y[..., two]) * turn
            y[..., one], y[..., two] = z.real, z.imag
            return y

        block, slot = s["slots"][:n].div(bs, rounding_mode="floor"), s["slots"][:n].remainder(bs)
        got = {"q": turned(s["q"])}
        for name, x in (("k", turned(s["k"])[:n]), ("v", s["v"][:n].double())):
            pages, scales = s[name + "_pages"], s[name + "_scales"]
            if scales is None:
                pages = pages.double()
                pages[block, slot] = x
                got[name] = {"values": pages}
            else:
                got[name] = _exact_store(pages, scales, x, block, slot, block[slot == 0], kind)
        return got
    values = s["k_pages"].double() * s["k_scales"].double()[:, None, :, None]
    if case["op"] != "attend":
        blocks, slots = [], []
        for b, n in enumerate(_lengths(case)):
            token = torch.arange(n, device="cuda")
            blocks.append(s["tables"][b].long()[token // bs])
            slots.append(token % bs)
        block, slot = torch.cat(blocks), torch.cat(slots)
        if case["op"] == "read":
            return {"values": values[block, slot]}
        x = values[block, slot] + s["delta"].double()
        return _exact_store(s["k_pages"], s["k_scales"], x, block, slot, block[slot == bs - 1], kind)
    heads, outs, lses = case["heads"], [], []
    del values
    for b, n in enumerate(_lengths(case)):
        if n == 0:
            outs.append(torch.zeros(heads, d, dtype=torch.float64, device="cuda"))
            lses.append(torch.full((heads,), -math.inf, dtype=torch.float64, device="cuda"))
            continue
        ids = s["tables"][b, : -(-n // bs)].long()
        k, v = ((s[x + "_pages"].view(torch.uint8).index_select(0, ids).view(s["k_pages"].dtype).double()
                 * s[x + "_scales"].double()[ids][:, None, :, None]).reshape(-1, kv, d)[:n] for x in "kv")
        q = s["q"][b].double().view(kv, heads // kv, d)
        score = torch.einsum("hgd,nhd->hgn", q, k) * d ** -0.5
        lse = torch.logsumexp(score, -1)
        outs.append(torch.einsum("hgn,nhd->hgd", torch.exp(score - lse[..., None]), v).reshape(heads, d))
        lses.append(lse.reshape(heads))
    got = {"out": torch.stack(outs)}
    if case["lse"]:
        got["lse"] = torch.stack(lses)
    return got
