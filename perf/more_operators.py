"""The KV cache held in 8 bits, and its blocks shared and moved on the device, as cases to measure:

  decode8  attention of one new token per sequence over a cache in 8 bits (a scale per page and KV head), optionally
           quantising the token's own K/V row into the cache first
  pack     rows of a 16-bit or f32 cache into the 8-bit one, whole or behind rows that are there already
  unpack   rows of the 8-bit cache into a 16-bit or f32 one (what a further prefill reads)
  beam     sequences become copies of others by sharing their blocks (fork), then grow by a row: a last block that
           several hold is copied first, in the pools of every layer
  compact  the blocks in use moved to the front of the pools

The plain forms are elementary torch operations in 32 bits; with `own` true the same calls go through epsp.Context.
"""
import math
import os
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn,
         "i8": torch.int8}
BYTES = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1, "i8": 1}
TOP = {"e4m3": 448.0, "i8": 127.0}  # largest magnitude
LEAST = -100  # exponent of the smallest scale


# ------------------------------------------------------------------ the cases
def _decode8(name, n_seq, min_len, max_len, heads, dtype, q8, block_rows, append, out=None, page=64):
    n_head, n_head_kv, dim = heads
    return {"name": name, "op": "decode8", "n_seq": n_seq, "min_len": min_len, "max_len": max_len, "n_head": n_head,
            "n_head_kv": n_head_kv, "head_dim": dim, "dtype": dtype, "out": out or dtype, "q8": q8,
            "block_rows": block_rows, "page": page, "append": append}


def _pack(name, op, n_seq, min_len, max_len, rows, heads, dtype, q8, block_rows, block_rows8, page=64):
    n_head, n_head_kv, dim = heads
    return {"name": name, "op": op, "n_seq": n_seq, "min_len": min_len, "max_len": max_len, "rows": rows,
            "n_head": n_head, "n_head_kv": n_head_kv, "head_dim": dim, "dtype": dtype, "q8": q8,
            "block_rows": block_rows, "block_rows8": block_rows8, "page": page}


def _beam(name, prompts, beams, kv_len, tail, n_layer, heads, cache, block_rows, page=64):
    n_head, n_head_kv, dim = heads
    return {"name": name, "op": "beam", "prompts": prompts, "beams": beams, "kv_len": kv_len, "tail": tail,
            "n_layer": n_layer, "n_head": n_head, "n_head_kv": n_head_kv, "head_dim": dim, "cache": cache,
            "block_rows": block_rows, "page": page}


def _compact(name, n_seq, kv_len, pool_blocks, n_layer, heads, cache, block_rows, page=64):
    n_head, n_head_kv, dim = heads
    return {"name": name, "op": "compact", "n_seq": n_seq, "kv_len": kv_len, "pool_blocks": pool_blocks,
            "n_layer": n_layer, "n_head": n_head, "n_head_kv": n_head_kv, "head_dim": dim, "cache": cache,
            "block_rows": block_rows, "page": page}


# Head layouts (query heads, KV heads, head size): the benchmark's three, then generic ones (no sharing, many
# heads on one, an odd group).
SMALL, LARGE, SEVEN = (14, 2, 64), (32, 8, 128), (28, 4, 128)
LAYOUTS = [SMALL, LARGE, SEVEN, (8, 8, 64), (16, 1, 128), (9, 3, 128), (24, 2, 64)]


def listed():
    return [
        # the first tokens of an answer to a short prompt, one user: the call's latency
        _decode8("decode8 short", 1, 200, 200, SMALL, "f16", "e4m3", 0, False),
        # one user, a 64 K prompt in cache blocks of a page
        _decode8("decode8 64K", 1, 65536, 65536, LARGE, "bf16", "e4m3", 128, False, page=128),
        # a server's step: 64 sequences of any length up to 4 K, each token's row quantised by the call
        _decode8("decode8 batch", 64, 1, 4096, LARGE, "bf16", "e4m3", 128, True, page=128),
        # long conversations, 8-bit integers
        _decode8("decode8 32K i8", 8, 16384, 32768, SEVEN, "bf16", "i8", 64, True),
        # the small configuration's f32 model over an 8-bit cache, a few sequences
        _decode8("decode8 f32 i8", 4, 1000, 4096, SMALL, "f32", "i8", 64, True),
        # after the prefill of a 64 K prompt: its cache, layer by layer, into 8 bits
        _pack("pack 64K", "pack", 1, 65536, 65536, 0, LARGE, "bf16", "e4m3", 128, 128, page=128),
        # a 500-row ubatch of each of 8 sequences behind what is in 8 bits already (pages begun, odd rows)
        _pack("pack chunk i8", "pack", 8, 5000, 8191, 500, SMALL, "f16", "i8", 0, 64),
        # a conversation goes on: 32 K rows back in 16 bits for the next gated prefill
        _pack("unpack 32K", "unpack", 1, 32768, 32768, 0, SEVEN, "bf16", "e4m3", 0, 64),
        # beam search: 4 beams of a 1000-row prompt, 24 layers in 8 bits (a small copy: latency)
        _beam("beam 4 x 1000 e4m3", 1, 4, 1000, 40, 24, SMALL, "e4m3", 64),
        # 8 prompts with 8 candidates each, 28 layers
        _beam("beam 8 x 8 x 4000", 8, 8, 4001, 200, 28, SEVEN, "bf16", 64),
        # a pool a little more than half in use after sequences have come and gone, 24 layers in 8 bits
        _compact("compact small e4m3", 16, 900, 400, 24, SMALL, "e4m3", 64),
        # the same of a large pool in 16 bits
        _compact("compact 1 GB", 12, 1500, 256, 8, LARGE, "bf16", 128, page=128),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    heads = rng.choice(LAYOUTS)
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    q8 = rng.choice(["e4m3", "i8"])
    page = rng.choice([32, 64, 128])
    block = rng.choice([0, page, page, 2 * page])
    row = heads[1] * heads[2] * 2  # bytes of a row's K and V in 8 bits
    op = rng.choice(["decode8", "decode8", "pack", "unpack", "beam", "compact"])
    if op == "decode8":
        n_seq = _log(rng, 1, 128)
        hi = _log(rng, 8, max(16, min(65536, int(130e6 / row / n_seq))))
        lo = rng.choice([hi, max(1, hi // 2), 1, 0])
        c = _decode8("", n_seq, lo, hi, heads, dtype, q8, block, rng.random() < 0.5, rng.choice([None, None, "f32"]),
                     page)
    elif op in ("pack", "unpack"):
        n_seq = _log(rng, 1, 32)
        hi = _log(rng, 16, max(32, min(65536, int(60e6 / row / n_seq))))
        lo = rng.choice([hi, max(1, hi // 2), 0])
        rows = rng.choice([0, 0, 1, _log(rng, 1, hi)])
        c = _pack("", op, n_seq, lo, hi, rows, heads, dtype, q8, block, rng.choice([0, page, 4 * page]), page)
    else:
        cache = rng.choice(["bf16", "f32", "e4m3", "i8"])
        block = max(page, block)
        n_layer = _log(rng, 1, 28)
        each = block * row * BYTES[cache]  # bytes of a block in one layer's pools
        if op == "beam":
            prompts, beams, tail = _log(rng, 1, 8), _log(rng, 1, 8), _log(rng, 1, 300)
            kv_len = _log(rng, tail, 4200)
            n_layer = max(1, min(n_layer, int(1e8 / (prompts * beams * each))))
            c = _beam("", prompts, beams, kv_len, tail, n_layer, heads, cache, block, page)
        else:
            blocks = max(8, min(_log(rng, 8, 2000), int(6e8 / each)))
            n_layer = max(1, min(n_layer, int(6e8 / (blocks * each))))
            n_seq = _log(rng, 1, min(40, blocks // 2))
            per = blocks * rng.choice([4, 6, 8]) // 10 // n_seq
            c = _compact("", n_seq, max(1, per * block - rng.randrange(block)), blocks, n_layer, heads, cache, block,
                         page)
    del c["name"]
    return c


def _lens(c):
    """The sequences' lengths: spread over [min_len, max_len], the longest among them."""
    span = c["max_len"] - c["min_len"] + 1
    return [c["max_len"] - (i * 2654435761) % 4294967296 * span // 4294967296 for i in range(c["n_seq"])]


def _firsts(c):
    """First row of each sequence that is packed or unpacked: 0, or the last `rows` rows."""
    return [max(0, n - c["rows"]) if c["rows"] else 0 for n in _lens(c)]


def _up(a, b):
    return -(-a // b)


def _block_bytes(c):
    """Bytes of one block in all pools of all layers (K, V and their scales)."""
    K, d, B = c["n_head_kv"], c["head_dim"], c["block_rows"]
    scales = B // c["page"] * K * 4 if c["cache"] in TOP else 0
    return c["n_layer"] * 2 * (B * K * d * BYTES[c["cache"]] + scales)


def work(c):
    K, d = c["n_head_kv"], c["head_dim"]
    if c["op"] == "decode8":
        lens, H, es = _lens(c), c["n_head"], BYTES[c["dtype"]]
        rows = sum(lens)
        b = rows * K * d * 2 + sum(_up(n, c["page"]) for n in lens) * K * 8
        b += c["n_seq"] * H * d * (es + BYTES[c["out"]]) + 4 * c["n_seq"]
        if c["append"]:  # the token's rows come in in the model's type and go out in 8 bits
            b += c["n_seq"] * K * d * 2 * es
        if c["block_rows"]:
            b += sum(_up(n, c["block_rows"]) for n in lens) * 4
        return {"bytes": b, "flops": 4.0 * rows * c["n_head"] * d}
    if c["op"] in ("pack", "unpack"):
        lens, firsts = _lens(c), _firsts(c)
        rows = sum(n - f for n, f in zip(lens, firsts))
        pages = sum(_up(n, c["page"]) - f // c["page"] for n, f in zip(lens, firsts) if n > f)
        return {"bytes": rows * K * d * 2 * (BYTES[c["dtype"]] + 1) + pages * K * 8 + 8 * c["n_seq"], "flops": 0}
    if c["op"] == "beam":
        n = c["prompts"] * c["beams"]
        held = _up(c["kv_len"], c["block_rows"])
        # tables once in and once out, and a block in and out for all sequences but, of each block, its last holder
        copies = n - _parents_used(c) if c["kv_len"] % c["block_rows"] else 0
        return {"bytes": 2 * copies * _block_bytes(c) + 8 * n * held + 16 * n, "flops": 0}
    held = c["n_seq"] * _up(c["kv_len"], c["block_rows"])
    moved = held * (c["pool_blocks"] - held) / c["pool_blocks"]  # in use past the first `held`, by their share
    return {"bytes": 2 * moved * _block_bytes(c) + 4 * held + 8 * c["pool_blocks"], "flops": 0}


# ---------------------------------------------------------------- the inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(TYPES[dtype])


def _keys(g, rows, c):
    """K rows: normal, with the per-channel spread that trained keys show."""
    spread = torch.exp(torch.randn((1, c["n_head_kv"], c["head_dim"]), generator=g, device="cuda") * 0.5)
    k = torch.randn((rows, c["n_head_kv"], c["head_dim"]), generator=g, device="cuda")
    return k.mul_(spread).to(TYPES[c["dtype"]])


def _cache(g, n_seq, rows_each, block_rows, page):
    """(tables or None, rows of the pool, rows from one sequence to the next where there are no tables)."""
    if not block_rows:
        each = _up(max(1, rows_each), page) * page
        return None, n_seq * each, each
    each = max(1, _up(rows_each, block_rows))
    blocks = n_seq * each + 3
    tables = torch.randperm(blocks, generator=g, device="cuda")[: n_seq * each].to(torch.int32).view(n_seq, each)
    return tables.contiguous(), blocks * block_rows, 0


def _cache8(g, rows, c):
    """(bytes, scales) of K or V as a pack of normal rows leaves them: magnitudes up to the type's largest in each
    page and head, scales around a unit normal's."""
    K, d, page = c["n_head_kv"], c["head_dim"], c["page"]
    x = torch.randn((rows // page, page, K, d), generator=g, device="cuda")
    x *= TOP[c["q8"]] / x.abs().amax((1, 3), keepdim=True)
    x = x.round() if c["q8"] == "i8" else x
    e = torch.randint(-9, -6, (rows // page, K), generator=g, device="cuda") + (2 if c["q8"] == "i8" else 0)
    return x.view(rows, K, d).to(TYPES[c["q8"]]), torch.exp2(e.float())


def _binding():
    at = os.path.join(os.getcwd(), "edge-prefill_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import epsp
    return epsp


def _context(c, max_ctx, dtype, out):
    epsp = _binding()
    code = {"f32": epsp.F32, "f16": epsp.F16, "bf16": epsp.BF16}
    ctx = epsp.Context(n_layer=c.get("n_layer", 1), n_head=c["n_head"], n_head_kv=c["n_head_kv"],
                       head_dim=c["head_dim"], dtype=code[dtype], out_dtype=code[out], max_ctx=max_ctx,
                       page_size=c["page"], device=torch.cuda.current_device())
    ctx.check(ctx.reserve())
    return epsp, ctx


def _space(n):
    return torch.empty(max(16, n), dtype=torch.uint8, device="cuda")


def _prepare_decode8(c, g):
    n_seq, H, K, d = c["n_seq"], c["n_head"], c["n_head_kv"], c["head_dim"]
    s = {"case": c, "lens": torch.tensor(_lens(c), dtype=torch.int32, device="cuda")}
    s["tables"], rows, s["seq_rows"] = _cache(g, n_seq, c["max_len"], c["block_rows"], c["page"])
    s["k8"], s["ks"] = _cache8(g, rows, c)
    s["v8"], s["vs"] = _cache8(g, rows, c)
    s["q"] = _randn(g, (n_seq, H, d), c["dtype"])
    if c["append"]:
        s["k_new"] = _keys(g, n_seq, c)
        s["v_new"] = _randn(g, (n_seq, K, d), c["dtype"])
    s["out"] = torch.zeros((n_seq, H, d), dtype=TYPES[c["out"]], device="cuda")
    if own:
        epsp, ctx = _context(c, max(1, c["max_len"]), c["dtype"], c["out"])
        kv = epsp.KvBatch(s["lens"], c["max_len"], s["tables"], c["block_rows"], rows, s["seq_rows"])
        s["own"] = (ctx, kv, epsp.Kv8(s["k8"], s["v8"], s["ks"], s["vs"]), _space(ctx.decode8_bytes(n_seq, c["max_len"])))
    return s


def _prepare_pack(c, g):
    n_seq, K, d = c["n_seq"], c["n_head_kv"], c["head_dim"]
    s = {"case": c, "lens": torch.tensor(_lens(c), dtype=torch.int32, device="cuda")}
    s["first"] = torch.tensor(_firsts(c), dtype=torch.int32, device="cuda") if c["rows"] else None
    s["tables"], rows, s["seq_rows"] = _cache(g, n_seq, c["max_len"], c["block_rows"], c["page"])
    s["tables8"], rows8, s["seq_rows8"] = _cache(g, n_seq, c["max_len"], c["block_rows8"], c["page"])
    s["k"] = _keys(g, rows, c)
    s["v"] = _randn(g, (rows, K, d), c["dtype"], 1.0 / math.sqrt(d))
    s["k8"], s["ks"] = _cache8(g, rows8, c)
    s["v8"], s["vs"] = _cache8(g, rows8, c)
    if own:
        epsp, ctx = _context(c, max(1, c["max_len"]), c["dtype"], c["dtype"])
        kv = epsp.KvBatch(s["lens"], c["max_len"], s["tables"], c["block_rows"], rows, s["seq_rows"])
        kv8 = epsp.KvBatch(s["lens"], c["max_len"], s["tables8"], c["block_rows8"], rows8, s["seq_rows8"])
        s["own"] = (ctx, kv, kv8, epsp.Kv8(s["k8"], s["v8"], s["ks"], s["vs"]))
    return s


def _pools(g, c, blocks):
    """K, V (and scales) of every layer: [layers][blocks][bytes of a block or elements]."""
    K, d, B, L = c["n_head_kv"], c["head_dim"], c["block_rows"], c["n_layer"]
    if c["cache"] == "i8":
        rows = [torch.randint(-127, 128, (L, blocks, B, K, d), generator=g, device="cuda", dtype=torch.int8)
                for _ in "kv"]
    else:
        rows = [torch.randn((L, blocks, B, K, d), generator=g, device="cuda", dtype=torch.bfloat16)
                .to(TYPES[c["cache"]]) for _ in "kv"]
    if c["cache"] in TOP:
        rows += [torch.rand((L, blocks, B // c["page"], K), generator=g, device="cuda") for _ in "kv"]
    return rows


def _own_pages(c, s):
    epsp, ctx = _context(c, s["tables"].shape[1] * c["block_rows"], "f16", "f16")
    pages = epsp.Pages(s["lens"], s["tables"], s["refs"], c["block_rows"])
    layers = [p[i] for p in s["pools"] for i in range(c["n_layer"])]
    return ctx, pages, epsp.Pools(layers, s["refs"].numel())


def _parents(c):
    """Each group's candidates go on from its first half, the better ones more often (position i from i * i / n / 2)."""
    b = c["beams"]
    return [p * b + i * i // (2 * b) for p in range(c["prompts"]) for i in range(b)]


def _parents_used(c):
    return len(set(_parents(c)))


def _prepare_beam(c, g):
    n, B = c["prompts"] * c["beams"], c["block_rows"]
    # each prompt's whole blocks are held by all of its candidates; the rows behind them are each one's own
    shared = max(0, c["kv_len"] - c["tail"]) // B
    mine = _up(c["kv_len"], B) - shared
    wide = shared + mine + 2
    blocks = c["prompts"] * shared + n * (mine + 2) + 5
    order = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)
    tables = torch.zeros((c["prompts"], c["beams"], wide), dtype=torch.int32, device="cuda")
    tables[:, :, :shared] = order[: c["prompts"] * shared].view(c["prompts"], 1, shared)
    at = c["prompts"] * shared
    tables[:, :, shared:shared + mine] = order[at:at + n * mine].view(c["prompts"], c["beams"], mine)
    refs = torch.zeros(blocks, dtype=torch.int32, device="cuda")
    refs[order[:at].long()] = c["beams"]
    refs[order[at:at + n * mine].long()] = 1
    s = {"case": c, "tables": tables.view(n, wide), "refs": refs, "pools": _pools(g, c, blocks),
         "lens": torch.full((n,), c["kv_len"], dtype=torch.int32, device="cuda"),
         "parents": torch.tensor(_parents(c), dtype=torch.int32, device="cuda")}
    s["keep"] = s["lens"].clone()
    s["grown"] = s["lens"] + 1
    if own:
        ctx, pages, pools = _own_pages(c, s)
        s["own"] = (ctx, pages, pools, _space(max(ctx.fork_bytes(pages), ctx.resize_bytes(pages))))
    return s


def _prepare_compact(c, g):
    n, B, blocks = c["n_seq"], c["block_rows"], c["pool_blocks"]
    each = _up(c["kv_len"], B)
    order = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)
    s = {"case": c, "tables0": order[: n * each].view(n, each).contiguous(), "pools": _pools(g, c, blocks),
         "lens": torch.full((n,), c["kv_len"], dtype=torch.int32, device="cuda"),
         "used": torch.zeros(1, dtype=torch.int32, device="cuda")}
    s["refs0"] = torch.zeros(blocks, dtype=torch.int32, device="cuda")
    s["refs0"][order[: n * each].long()] = 1
    s["tables"], s["refs"] = s["tables0"].clone(), s["refs0"].clone()
    if own:
        ctx, pages, pools = _own_pages(c, s)
        s["own"] = (ctx, pages, pools, _space(ctx.compact_bytes(pages)))
    return s


def prepare(c, seed):
    g = _gen(seed)
    if c["op"] == "decode8":
        return _prepare_decode8(c, g)
    if c["op"] in ("pack", "unpack"):
        return _prepare_pack(c, g)
    return _prepare_beam(c, g) if c["op"] == "beam" else _prepare_compact(c, g)


# --------------------------------------------------------------- plain forms
def _rows_of(tables, block_rows, seq_rows, n_seq, n):
    """Pool rows of the first n rows of every sequence, [n_seq][n]."""
    r = torch.arange(n, device="cuda")
    if tables is None:
        return torch.arange(n_seq, device="cuda")[:, None] * seq_rows + r[None, :]
    return tables.long()[:, r // block_rows] * block_rows + r % block_rows


def _scale_of(amax, q8):
    """The least power of two s with amax <= TOP s."""
    m, e = torch.frexp(amax)  # amax = m 2^e, m in [0.5, 1)
    top_m, top_e = math.frexp(TOP[q8])
    e = e - top_e + (m > top_m).int()
    return torch.ldexp(torch.ones_like(amax), torch.where(amax > 0, e, LEAST).clamp(min=LEAST))


def _to8(x, q8):
    return (x.round() if q8 == "i8" else x).to(TYPES[q8])


def _write_pages(pool, scales, at, x, old, new, page, q8):
    """Quantises rows `new` of x [pages][page][heads][d] into the pool behind the rows `old` of the same pages, whose
    bytes follow where the scale grows.  at: pool rows [pages][page]."""
    p = at[:, 0] // page
    amax = x.abs().masked_fill(~new[:, :, None, None], 0.0).amax((1, 3))
    was = torch.where(old.any(1)[:, None], scales[p], 0.0)
    s = torch.maximum(was, _scale_of(amax, q8))
    held = pool[at]
    moved = _to8(held.float() * (was / s)[:, None, :, None], q8)
    q = _to8(torch.where(new[:, :, None, None], x, 0.0) / s[:, None, :, None], q8)
    w = torch.uint8
    q = torch.where(new[:, :, None, None], q.view(w), torch.where(old[:, :, None, None], moved.view(w), held.view(w)))
    some = new.any(1)
    pool.view(w)[at] = torch.where(some[:, None, None, None], q, held.view(w))
    scales[p] = torch.where(some[:, None], s, scales[p])


def _plain_decode8(s):
    c = s["case"]
    n_seq, H, K, d, page, q8 = c["n_seq"], c["n_head"], c["n_head_kv"], c["head_dim"], c["page"], c["q8"]
    n = _up(max(1, c["max_len"]), page) * page
    at = _rows_of(s["tables"], c["block_rows"], s["seq_rows"], n_seq, n)
    lens = s["lens"].long()
    if c["append"]:
        r = torch.arange(page, device="cuda")[None, :]
        last = (lens - 1).clamp(min=0)[:, None]
        rows = at.gather(1, last // page * page + r)
        new = (r == last % page) & (lens > 0)[:, None]
        for t in "kv":
            x = s[t + "_new"].float()[:, None].expand(-1, page, -1, -1)
            _write_pages(s[t + "8"], s[t + "s"], rows, x, r < last % page, new, page, q8)
    k = s["k8"][at].float() * s["ks"][at // page][..., None]
    v = s["v8"][at].float() * s["vs"][at // page][..., None]
    q = s["q"].float().view(n_seq, K, H // K, d)
    valid = (torch.arange(n, device="cuda")[None, :] < lens[:, None])[:, None, None, :]
    x = torch.einsum("shgd,slhd->shgl", q, k) * (1.0 / math.sqrt(d))
    x = x.masked_fill(~valid, -math.inf)
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - m.masked_fill(m == -math.inf, 0.0))
    p = p / p.sum(-1, keepdim=True).masked_fill(~valid[..., :1], 1.0)
    s["out"].copy_(torch.einsum("shgl,slhd->shgd", p, v).reshape(n_seq, H, d))


def _span(s):
    """(rows of both caches [n_seq][n], [n_seq][n] whether a row is to be written, whether it is before those)."""
    c = s["case"]
    n = _up(max(1, c["max_len"]), c["page"]) * c["page"]
    r = torch.arange(n, device="cuda")[None, :]
    first = torch.zeros_like(s["lens"]) if s["first"] is None else s["first"]
    at8 = _rows_of(s["tables8"], c["block_rows8"], s["seq_rows8"], c["n_seq"], n)
    at = _rows_of(s["tables"], c["block_rows"], s["seq_rows"], c["n_seq"], n)
    return at, at8, (r >= first[:, None]) & (r < s["lens"][:, None]), r < first[:, None]


def _plain_pack(s):
    c = s["case"]
    page = c["page"]
    at, at8, new, old = _span(s)
    for t in "kv":
        x = s[t][at].float().view(-1, page, c["n_head_kv"], c["head_dim"])
        _write_pages(s[t + "8"], s[t + "s"], at8.view(-1, page), x, old.view(-1, page), new.view(-1, page), page,
                     c["q8"])


def _plain_unpack(s):
    c = s["case"]
    at, at8, new, _ = _span(s)
    for t in "kv":
        x = (s[t + "8"][at8].float() * s[t + "s"][at8 // c["page"]][..., None]).to(TYPES[c["dtype"]])
        s[t][at] = torch.where(new[..., None, None], x, s[t][at])


def _held(lens, tables, B):
    return torch.arange(tables.shape[1], device="cuda")[None, :] < ((lens + B - 1) // B)[:, None]


def _count(refs, tables, held, sign):
    refs.scatter_add_(0, torch.where(held, tables, 0).long().view(-1), held.int().view(-1) * sign)


def _plain_fork(s, B):
    tables, lens, parents = s["tables"], s["lens"], s["parents"].long()
    _count(s["refs"], tables, _held(lens, tables, B), -1)
    held = _held(s["keep"], tables, B)
    tables.copy_(torch.where(held, tables[parents], tables))
    lens.copy_(s["keep"])
    _count(s["refs"], tables, held, 1)


def _copy_blocks(pools, src, dst):
    for p in pools:
        b = p.view(p.shape[0], p.shape[1], -1).view(torch.uint8)
        b[:, dst] = b[:, src]


def _plain_resize(s, B):
    tables, lens, refs, grown = s["tables"], s["lens"], s["refs"].clone(), s["grown"]
    n, blocks = lens.numel(), refs.numel()
    was, now = _held(lens, tables, B), _held(grown, tables, B)
    _count(refs, tables, was & ~now, -1)
    seq = torch.arange(n, device="cuda")
    at = ((lens - 1).clamp(min=0) // B).long()
    last = tables.gather(1, at[:, None])[:, 0].long()
    shared = (grown > lens) & (lens % B != 0) & (refs[last] > 1)
    count = torch.zeros_like(refs).scatter_add_(0, last, shared.int())
    keeper = torch.full_like(refs, -1).scatter_reduce_(0, last, torch.where(shared, seq, -1).int(), "amax")
    copy = shared & ~((count[last] == refs[last]) & (keeper[last] == seq))
    fresh = (now & ~was).sum(1)
    need = fresh + copy
    off = need.cumsum(0) - need
    free = torch.sort((refs != 0).int(), stable=True)[1]  # the free blocks first, in order
    ok = need.sum() <= (refs == 0).sum()
    i = torch.arange(tables.shape[1], device="cuda")[None, :]
    pick = (off + copy)[:, None] + i - ((lens + B - 1) // B)[:, None]
    new = torch.where(now & ~was, free[pick.clamp(0, blocks - 1)], tables.long())
    mine = free[off.clamp(max=blocks - 1)]
    new = torch.where((i == at[:, None]) & copy[:, None], mine[:, None], new).int()
    _count(refs, tables, (i == at[:, None]) & copy[:, None], -1)
    _count(refs, new, (now & ~was) | ((i == at[:, None]) & copy[:, None]), 1)
    _copy_blocks(s["pools"], last, torch.where(copy & ok, mine, last))
    tables.copy_(torch.where(ok, new, tables))
    lens.copy_(torch.where(ok, grown, lens))
    s["refs"].copy_(torch.where(ok, refs, s["refs"]))


def _plain_compact(s, B):
    tables, refs = s["tables"], s["refs"]
    live = refs > 0
    n_live = live.sum()
    i = torch.arange(refs.numel(), device="cuda")
    src, dst = (live & (i >= n_live)).nonzero()[:, 0], (~live & (i < n_live)).nonzero()[:, 0]
    to = i.clone()
    to[src] = dst
    _copy_blocks(s["pools"], src, dst)
    tables.copy_(torch.where(_held(s["lens"], tables, B), to[tables.long()].int(), tables))
    refs[dst] = refs[src]
    refs[src] = 0
    s["used"].copy_(n_live)


# ------------------------------------------------------------------- one pass
def _run_cache8(s):
    c = s["case"]
    if c["op"] == "decode8":
        if own:
            ctx, kv, kv8, space = s["own"]
            ctx.check(ctx.decode8_layer(0, kv, s["q"], kv8, s["out"], space, k_new=s.get("k_new"),
                                        v_new=s.get("v_new")))
        else:
            _plain_decode8(s)
        return {"out": s["out"]} | ({t: s[t] for t in ("k8", "v8", "ks", "vs")} if c["append"] else {})
    if own:
        ctx, kv, kv8, rows8 = s["own"]
        if c["op"] == "pack":
            ctx.check(ctx.pack_kv(0, kv, s["k"], s["v"], kv8, rows8, first=s["first"]))
        else:
            ctx.check(ctx.unpack_kv(0, kv8, rows8, kv, s["k"], s["v"], first=s["first"]))
    else:
        _plain_pack(s) if c["op"] == "pack" else _plain_unpack(s)
    return {t: s[t] for t in (("k8", "v8", "ks", "vs") if c["op"] == "pack" else ("k", "v"))}


def run(s):
    c = s["case"]
    if c["op"] not in ("beam", "compact"):
        return _run_cache8(s)
    B = c["block_rows"]
    if c["op"] == "beam":
        # the candidates of a pass before are given back by the fork: each pass does the same work
        if own:
            ctx, pages, pools, space = s["own"]
            ctx.check(ctx.fork_seqs(pages, s["parents"], space, lens=s["keep"]))
            ctx.check(ctx.resize_seqs(pages, s["grown"], pools, space))
        else:
            _plain_fork(s, B)
            _plain_resize(s, B)
        return {"pools": s["pools"], "tables": s["tables"], "lens": s["lens"], "refs": s["refs"]}
    # the tables as the comings and goings left them (the moved blocks are still where they were, too)
    s["tables"].copy_(s["tables0"])
    s["refs"].copy_(s["refs0"])
    if own:
        ctx, pages, pools, space = s["own"]
        ctx.check(ctx.compact_pool(pages, pools, space, n_used=s["used"]))
    else:
        _plain_compact(s, B)
    return {"pools": s["pools"], "tables": s["tables"], "refs": s["refs"], "used": s["used"]}


# ------------------------------------------------- the definition, in 64 bits
def _place(tables, block_rows, seq_rows, i, n):
    """Pool rows of rows [0, n) of sequence i."""
    if tables is None:
        return torch.arange(i * seq_rows, i * seq_rows + n, device="cuda")
    blocks = tables[i, : _up(n, block_rows)].tolist()
    parts = [torch.arange(b * block_rows, (b + 1) * block_rows, device="cuda") for b in blocks]
    return torch.cat(parts)[:n] if parts else torch.arange(0, device="cuda")


def _round8(x, q8):
    """Nearest value of the type, ties to even: the step is that of the value's power of two (2^-9 below 2^-6)."""
    if q8 == "i8":
        return torch.round(x)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def _exact_write(pool, scales, at, x, a, page, q8):
    """Rows [a, n) of x (n rows) behind rows [0, a) of one sequence whose rows lie at `at`; pool in 64 bits."""
    n = x.shape[0]
    for r0 in range(a // page * page, n, page):
        r1, p = min(n, r0 + page), int(at[r0]) // page
        for h in range(x.shape[1]):
            fresh = x[max(a, r0):r1, h].double()
            top = float(fresh.abs().max())
            e = LEAST
            if top > 0:
                e = max(LEAST, math.frexp(top / TOP[q8])[1] - 1)
                e += top > math.ldexp(TOP[q8], e)
            s = math.ldexp(1.0, e)
            if r0 < a:
                was = float(scales[p, h])
                if was < s:
                    pool[at[r0:a], h] = _round8(pool[at[r0:a], h] * was / s, q8)
                s = max(s, was)
            pool[at[max(a, r0):r1], h] = _round8(fresh / s, q8)
            scales[p, h] = s


def _exact_cache8(c, s):
    lens, page, q8, K, d = _lens(c), c["page"], c["q8"], c["n_head_kv"], c["head_dim"]
    pools = {t: s[t + "8"].float().double() for t in "kv"}
    scales = {t: s[t + "s"].double() for t in "kv"}
    if c["op"] == "unpack":
        got = {t: s[t].double() for t in "kv"}
        for i, (n, a) in enumerate(zip(lens, _firsts(c))):
            at8 = _place(s["tables8"], c["block_rows8"], s["seq_rows8"], i, n)[a:]
            at = _place(s["tables"], c["block_rows"], s["seq_rows"], i, n)[a:]
            for t in "kv":
                got[t][at] = pools[t][at8] * scales[t][at8 // page][..., None]
        return got
    if c["op"] == "pack":
        if sum(_up(n, page) for n in lens) * K > 20000:
            return None  # a page and head at a time: too long
        for i, (n, a) in enumerate(zip(lens, _firsts(c))):
            at8 = _place(s["tables8"], c["block_rows8"], s["seq_rows8"], i, n)
            at = _place(s["tables"], c["block_rows"], s["seq_rows"], i, n)
            for t in "kv":
                _exact_write(pools[t], scales[t], at8, s[t][at], a, page, q8)
        got = {}
    else:
        H, G = c["n_head"], c["n_head"] // K
        out = torch.zeros((c["n_seq"], H, d), dtype=torch.float64, device="cuda")
        for i, n in enumerate(lens):
            if n == 0:
                continue
            at = _place(s["tables"], c["block_rows"], s["seq_rows"], i, n)
            if c["append"]:
                for t in "kv":
                    x = s[t + "_new"][i].expand(n, K, d)
                    _exact_write(pools[t], scales[t], at, x, n - 1, page, q8)
            k, v = (pools[t][at] * scales[t][at // page][..., None] for t in "kv")
            for h in range(K):
                x = s["q"][i, h * G:(h + 1) * G].double() @ k[:, h].T / math.sqrt(d)
                p = torch.exp(x - x.max(-1, keepdim=True)[0])
                out[i, h * G:(h + 1) * G] = p / p.sum(-1, keepdim=True) @ v[:, h]
        got = {"out": out}
        if not c["append"]:
            return got
    whole = {t + "8": pools[t].to(torch.int8) if q8 == "i8" else pools[t] for t in "kv"}
    return got | whole | {t + "s": scales[t] for t in "kv"}


def exact(c, seed):
    s = prepare(c, seed)
    # (beam and compact move bytes and whole numbers: nothing is computed)
    return _exact_cache8(c, s) if c["op"] not in ("beam", "compact") else None
