"""The serving operators that read and shrink the KV cache a prefill leaves behind, as cases to measure:

  decode   attention of one new token per sequence over its (paged) KV cache, optionally writing the token's
           own K/V row first and adding its softmax weights to the cache rows' accumulated weights
  prompt   accumulated softmax weights of the last rows of a prompt over its cache (what an eviction after
           the prefill ranks the rows by)
  evict    per KV head, keep the sink rows, the recent rows and the rows of largest accumulated weight, and
           gather them in order into another cache

The plain forms are elementary torch operations in 32 bits; with `own` true the same calls go through epsp.Context.
"""
import math
import os
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


# ------------------------------------------------------------------ the cases
def _decode(name, n_seq, min_len, max_len, heads, dtype, block_rows, append, weights, out=None, page=64):
    n_head, n_head_kv, dim = heads
    return {"name": name, "op": "decode", "n_seq": n_seq, "min_len": min_len, "max_len": max_len, "n_head": n_head,
            "n_head_kv": n_head_kv, "head_dim": dim, "dtype": dtype, "out": out or dtype, "block_rows": block_rows,
            "page": page, "append": append, "weights": weights}


def _prompt(name, kv_len, n_tok, window, heads, dtype, block_rows, page=64):
    n_head, n_head_kv, dim = heads
    return {"name": name, "op": "prompt", "kv_len": kv_len, "n_tok": n_tok, "window": window, "n_head": n_head,
            "n_head_kv": n_head_kv, "head_dim": dim, "dtype": dtype, "block_rows": block_rows, "page": page}


def _evict(name, n_seq, min_len, max_len, n_keep, sink, recent, heads, dtype, block_rows, page=64):
    n_head, n_head_kv, dim = heads
    return {"name": name, "op": "evict", "n_seq": n_seq, "min_len": min_len, "max_len": max_len, "n_keep": n_keep,
            "sink": sink, "recent": recent, "n_head": n_head, "n_head_kv": n_head_kv, "head_dim": dim, "dtype": dtype,
            "block_rows": block_rows, "page": page}


# Head layouts (query heads, KV heads, head size): the benchmark's three, then generic ones (no sharing, many
# heads on one, an odd group).
SMALL, LARGE, SEVEN = (14, 2, 64), (32, 8, 128), (28, 4, 128)
LAYOUTS = [SMALL, LARGE, SEVEN, (8, 8, 64), (16, 1, 128), (9, 3, 128), (24, 2, 64)]


def listed():
    return [
        # the first tokens of an answer to a short prompt, one user: the call's latency
        _decode("decode short", 1, 200, 200, SMALL, "f16", 0, False, False),
        # one user, a 64 K prompt in cache blocks of a page
        _decode("decode 64K", 1, 65536, 65536, LARGE, "bf16", 128, False, False, page=128),
        # a server's step: 64 sequences of any length up to 4 K, each token's K/V row written by the call
        _decode("decode batch", 64, 1, 4096, LARGE, "bf16", 128, True, False, page=128),
        # the f32 cache of the small configuration, a few sequences
        _decode("decode f32", 4, 1000, 4096, SMALL, "f32", 64, True, False),
        # steps that also keep the rows' accumulated weights, for an eviction later on
        _decode("decode weights 32K", 8, 16384, 32768, SEVEN, "bf16", 64, True, True),
        _decode("decode weights short", 1, 1001, 1001, SMALL, "f16", 0, True, True),
        # after the last ubatch of a 64 K prompt: weights of its last 64 rows
        _prompt("prompt 64K last 64", 65536, 4096, 64, LARGE, "bf16", 128, page=128),
        # every row of a 512-row ubatch over an 8 K cache
        _prompt("prompt 8K ubatch", 8192, 512, 512, SMALL, "f16", 0),
        # the f32 configuration: last 32 rows of a 4 K prompt
        _prompt("prompt 4K f32", 4096, 4096, 32, SMALL, "f32", 0),
        # a 64 K prompt's cache shrunk to 4 K rows per head, blocks to blocks
        _evict("evict 64K to 4K", 1, 65536, 65536, 4096, 128, 1024, LARGE, "bf16", 128, page=128),
        # a batch of short sequences, some below the budget already
        _evict("evict batch", 32, 1, 2048, 512, 4, 64, SMALL, "f16", 64),
        # the smallest: one 4 K cache in f32
        _evict("evict 4K f32", 1, 4096, 4096, 1000, 1, 100, SMALL, "f32", 0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    heads = rng.choice(LAYOUTS)
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    page = rng.choice([32, 64, 128])
    block = rng.choice([0, page, page, 2 * page])
    row = heads[1] * heads[2] * BYTES[dtype] * 2
    op = rng.choice(["decode", "decode", "prompt", "evict"])
    if op == "decode":
        n_seq = _log(rng, 1, 128)
        top = max(16, min(65536, int(200e6 / row / n_seq)))
        hi = _log(rng, 8, top)
        lo = rng.choice([hi, max(1, hi // 2), 1, 0])
        c = _decode("", n_seq, lo, hi, heads, dtype, block, rng.random() < 0.5, rng.random() < 0.4,
                    rng.choice([None, None, "f32"]), page)
    elif op == "prompt":
        # query rows times keys stays under that of the listed 64 K case; f32 runs on the CUDA cores
        most = (65536 * 64 * 32 if dtype != "f32" else 4096 * 32 * 14) // heads[0]
        kv_len = _log(rng, 16, 65536 if dtype != "f32" else 8192)
        window = _log(rng, 1, max(1, min(kv_len, 700, most // kv_len)))
        c = _prompt("", kv_len, min(kv_len, window + rng.choice([0, 3, 100])), window, heads, dtype, block, page)
    else:
        n_seq = _log(rng, 1, 64)
        top = max(64, min(65536, int(200e6 / row / n_seq)))
        hi = _log(rng, 32, top)
        lo = rng.choice([hi, max(1, hi // 2), 0])
        # what is gathered counts most: keep it under the largest listed eviction
        keep = _log(rng, 2, max(2, min(hi, int(15e6 / row / n_seq))))
        sink = rng.choice([0, 1, 4])
        recent = rng.choice([0, 1, 33, keep // 2])
        if sink + recent > keep:
            sink, recent = 0, keep // 2
        c = _evict("", n_seq, lo, hi, keep, sink, recent, heads, dtype, block, page)
    del c["name"]
    return c


def _lens(c):
    """The sequences' lengths: spread over [min_len, max_len], the longest among them."""
    span = c["max_len"] - c["min_len"] + 1
    return [c["max_len"] - (i * 2654435761) % 4294967296 * span // 4294967296 for i in range(c["n_seq"])]


def work(c):
    H, K, d, es = c["n_head"], c["n_head_kv"], c["head_dim"], BYTES[c["dtype"]]
    if c["op"] == "decode":
        lens = _lens(c)
        rows = sum(lens)
        b = rows * K * d * 2 * es + c["n_seq"] * H * d * (es + BYTES[c["out"]]) + 4 * c["n_seq"]
        if c["append"]:  # the token's rows come in once and go out once (instead of being read from the cache)
            b += c["n_seq"] * K * d * 2 * es
        if c["weights"]:
            b += rows * K * 8
        if c["block_rows"]:
            b += sum(-(-n // c["block_rows"]) for n in lens) * 4
        return {"bytes": b, "flops": 4.0 * rows * H * d}
    if c["op"] == "prompt":
        n, w = c["kv_len"], c["window"]
        pairs = w * (n - w) + w * (w + 1) // 2
        return {"bytes": n * K * d * es + w * H * d * es + n * K * 4, "flops": 2.0 * pairs * H * d}
    lens = _lens(c)
    kept = sum(min(n, c["n_keep"]) for n in lens)
    # the weights of every row, then the kept rows' K, V and weights once in and once out
    return {"bytes": sum(lens) * K * 4 + kept * K * (4 * d * es + 4) + kept * K * 4 + 8 * c["n_seq"], "flops": 0}


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


def _pool(g, n_seq, rows_each, block_rows, spare):
    """Block tables of n_seq sequences with room for rows_each rows in a shuffled pool: (tables, pool rows)."""
    each = max(1, -(-rows_each // block_rows))
    blocks = n_seq * each + spare
    tables = torch.randperm(blocks, generator=g, device="cuda")[: n_seq * each].to(torch.int32).view(n_seq, each)
    return tables, blocks * block_rows


def _cache(g, c, n_seq, rows_each):
    """(tables or None, rows of the pool, rows from one sequence to the next where there are no tables)."""
    if c["block_rows"]:
        tables, rows = _pool(g, n_seq, rows_each, c["block_rows"], 3)
        return tables.contiguous(), rows, 0
    return None, n_seq * max(1, rows_each), max(1, rows_each)


def _weights(g, shape):
    """Accumulated weights: heavy-tailed, with a share of rows that no query has looked at yet (exact zeros)."""
    a = torch.exp(torch.randn(shape, generator=g, device="cuda") * 1.5)
    return torch.where(torch.rand(shape, generator=g, device="cuda") < 0.1, torch.zeros_like(a), a)


def _binding():
    at = os.path.join(os.getcwd(), "edge-prefill_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import epsp
    return epsp


def _context(c, max_ctx, out):
    epsp = _binding()
    code = {"f32": epsp.F32, "f16": epsp.F16, "bf16": epsp.BF16}
    ctx = epsp.Context(n_layer=1, n_head=c["n_head"], n_head_kv=c["n_head_kv"], head_dim=c["head_dim"],
                       dtype=code[c["dtype"]], out_dtype=code[out], max_ctx=max_ctx, page_size=c["page"],
                       device=torch.cuda.current_device())
    ctx.check(ctx.reserve())
    return epsp, ctx


def prepare(c, seed):
    g = _gen(seed)
    s = {"case": c}
    H, K, d = c["n_head"], c["n_head_kv"], c["head_dim"]
    if c["op"] == "prompt":
        tables, rows, _ = _cache(g, c, 1, c["kv_len"])
        s["table"] = None if tables is None else tables[0].contiguous()
        s["k"] = _keys(g, rows, c)
        s["q"] = _randn(g, (c["n_tok"], H, d), c["dtype"])
        s["acc"] = torch.zeros((K, c["kv_len"]), device="cuda")
        if own:
            _, ctx = _context(c, c["kv_len"], c["dtype"])
            if tables is not None:
                ctx.check(ctx.set_paged_kv(c["block_rows"], s["table"], s["table"].numel(), rows))
            need = ctx.prompt_weights_bytes(c["kv_len"], c["n_tok"], c["n_tok"] - c["window"])
            s["own"] = (ctx, torch.empty(max(1, need), dtype=torch.uint8, device="cuda"))
        return s
    n_seq = c["n_seq"]
    s["lens"] = torch.tensor(_lens(c), dtype=torch.int32, device="cuda")
    s["tables"], rows, s["seq_rows"] = _cache(g, c, n_seq, c["max_len"])
    s["k"] = _keys(g, rows, c)
    s["v"] = _randn(g, (rows, K, d), c["dtype"], 1.0 / math.sqrt(d))
    if c["op"] == "decode":
        s["q"] = _randn(g, (n_seq, H, d), c["dtype"])
        if c["append"]:
            s["k_new"] = _keys(g, n_seq, c)
            s["v_new"] = _randn(g, (n_seq, K, d), c["dtype"], 1.0 / math.sqrt(d))
        if c["weights"]:
            s["acc"] = _weights(g, (n_seq, K, c["max_len"]))
        s["out"] = torch.zeros((n_seq, H, d), dtype=TYPES[c["out"]], device="cuda")
        if own:
            epsp, ctx = _context(c, max(1, c["max_len"]), c["out"])
            kv = epsp.KvBatch(s["lens"], c["max_len"], s["tables"], c["block_rows"], rows, s["seq_rows"])
            need = ctx.decode_bytes(n_seq, c["max_len"], c["weights"])
            s["own"] = (ctx, kv, torch.empty(max(1, need), dtype=torch.uint8, device="cuda"))
        return s
    s["acc"] = _weights(g, (n_seq, K, c["max_len"]))
    keep = c["n_keep"]
    s["tables_dst"], rows_dst, s["seq_rows_dst"] = _cache(g, c, n_seq, keep)
    s["k_dst"] = _randn(g, (rows_dst, K, d), c["dtype"])
    s["v_dst"] = _randn(g, (rows_dst, K, d), c["dtype"])
    s["acc_dst"] = _weights(g, (n_seq, K, keep + 5))
    s["new_lens"] = torch.zeros_like(s["lens"])
    s["kept"] = torch.zeros((n_seq, K, keep), dtype=torch.int32, device="cuda")
    if own:
        epsp, ctx = _context(c, c["max_len"], c["dtype"])
        src = epsp.KvBatch(s["lens"], c["max_len"], s["tables"], c["block_rows"], rows, s["seq_rows"])
        dst = epsp.KvBatch(s["new_lens"], keep, s["tables_dst"], c["block_rows"], rows_dst, s["seq_rows_dst"])
        need = ctx.evict_bytes(n_seq, c["max_len"], keep)
        s["own"] = (ctx, src, dst, torch.empty(max(1, need), dtype=torch.uint8, device="cuda"))
    return s


# --------------------------------------------------------------- plain forms
def _rows_of(tables, block_rows, seq_rows, n_seq, n):
    """Pool rows of the first n rows of every sequence, [n_seq][n]."""
    r = torch.arange(n, device="cuda")
    if tables is None:
        return torch.arange(n_seq, device="cuda")[:, None] * seq_rows + r[None, :]
    return tables.long()[:, r // block_rows] * block_rows + r % block_rows


def _plain_decode(s):
    c = s["case"]
    n_seq, n, H, K, d = c["n_seq"], c["max_len"], c["n_head"], c["n_head_kv"], c["head_dim"]
    at = _rows_of(s["tables"], c["block_rows"], s["seq_rows"], n_seq, n)
    lens = s["lens"].long()
    if c["append"]:
        live = lens > 0
        last = at.gather(1, (lens - 1).clamp(min=0)[:, None])[:, 0]
        live_k = live[:, None, None]
        s["k"][last] = torch.where(live_k, s["k_new"], s["k"][last])
        s["v"][last] = torch.where(live_k, s["v_new"], s["v"][last])
    q = s["q"].float().view(n_seq, K, H // K, d)
    valid = (torch.arange(n, device="cuda")[None, :] < lens[:, None])[:, None, None, :]
    x = torch.einsum("shgd,slhd->shgl", q, s["k"][at].float()) * (1.0 / math.sqrt(d))
    x = x.masked_fill(~valid, -math.inf)
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - m.masked_fill(m == -math.inf, 0.0))
    p = p / p.sum(-1, keepdim=True).masked_fill(~valid[..., :1], 1.0)
    v = s["v"][at].float().masked_fill(~valid[:, 0, 0, :, None, None], 0.0)
    s["out"].copy_(torch.einsum("shgl,slhd->shgd", p, v).reshape(n_seq, H, d))
    if c["weights"]:
        s["acc"].add_(p.sum(2))


def _plain_prompt(s):
    c = s["case"]
    n, w, H, K, d = c["kv_len"], c["window"], c["n_head"], c["n_head_kv"], c["head_dim"]
    k = s["k"] if s["table"] is None else s["k"][_rows_of(s["table"][None], c["block_rows"], 0, 1, n)[0]]
    q = s["q"][c["n_tok"] - w:].float().view(w, K, H // K, d)
    x = torch.einsum("whgd,lhd->hwgl", q, k[:n].float()) * (1.0 / math.sqrt(d))
    seen = torch.arange(n, device="cuda")[None, :] <= torch.arange(n - w, n, device="cuda")[:, None]
    x = x.masked_fill_(~seen[None, :, None, :], -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True))
    s["acc"].copy_((x / x.sum(-1, keepdim=True)).sum((1, 2)))


def _plain_evict(s):
    c = s["case"]
    n_seq, n, keep, K = c["n_seq"], c["max_len"], c["n_keep"], c["n_head_kv"]
    lens = s["lens"].long()[:, None]
    r = torch.arange(n, device="cuda")[None, :]
    held = (r < c["sink"]) | (r >= lens - c["recent"])
    rank = torch.where(held[:, None, :], math.inf, torch.nan_to_num(s["acc"], nan=-math.inf, posinf=math.inf))
    rank = torch.where((r < lens)[:, None, :], rank, -math.inf)
    first = torch.sort(rank, dim=-1, descending=True, stable=True)[1][..., :keep]
    first = torch.sort(torch.where(first < lens[:, None, :], first, n), dim=-1)[0]  # ascending, absent ones last
    first = torch.nn.functional.pad(first, (0, keep - first.shape[-1]), value=n)
    there = first < n
    new_lens = lens[:, 0].clamp(max=keep)
    s["kept"].copy_(torch.where(there, first, -1))
    s["new_lens"].copy_(new_lens)
    src = _rows_of(s["tables"], c["block_rows"], s["seq_rows"], n_seq, n)
    dst = _rows_of(s["tables_dst"], c["block_rows"], s["seq_rows_dst"], n_seq, keep)
    row = first.clamp(max=n - 1)
    head = torch.arange(K, device="cuda")[None, :, None].expand_as(row)
    at = dst[:, None, :].expand_as(row)
    src_at = src[:, None, :].expand(-1, K, -1).gather(2, row)
    keep_old = there[..., None]
    s["k_dst"][at, head] = torch.where(keep_old, s["k"][src_at, head], s["k_dst"][at, head])
    s["v_dst"][at, head] = torch.where(keep_old, s["v"][src_at, head], s["v_dst"][at, head])
    s["acc_dst"].zero_()
    s["acc_dst"][..., :keep] = torch.where(there, s["acc"].gather(2, row), 0.0)


# ------------------------------------------------------------------- one pass
def run(s):
    c = s["case"]
    if c["op"] == "decode":
        if own:
            ctx, kv, space = s["own"]
            ctx.check(ctx.decode_layer(0, kv, s["q"], s["k"], s["v"], s["out"], space, k_new=s.get("k_new"),
                                       v_new=s.get("v_new"), acc=s.get("acc")))
        else:
            _plain_decode(s)
        got = {"out": s["out"]}
        if c["append"]:
            got |= {"k": s["k"], "v": s["v"]}
        if c["weights"]:
            got["acc"] = s["acc"]
        return got
    if c["op"] == "prompt":
        if own:
            ctx, space = s["own"]
            ctx.check(ctx.prompt_weights(0, s["q"], s["k"], c["kv_len"], c["n_tok"], c["n_tok"] - c["window"],
                                         s["acc"], space))
        else:
            _plain_prompt(s)
        return {"acc": s["acc"]}
    if own:
        ctx, src, dst, space = s["own"]
        ctx.check(ctx.evict_layer(0, src, s["k"], s["v"], s["acc"], c["n_keep"], c["sink"], c["recent"], dst,
                                  s["k_dst"], s["v_dst"], space, acc_dst=s["acc_dst"], new_lens=s["new_lens"],
                                  kept_rows=s["kept"]))
    else:
        _plain_evict(s)
    return {"k": s["k_dst"], "v": s["v_dst"], "acc": s["acc_dst"], "new_lens": s["new_lens"], "kept": s["kept"]}


# ------------------------------------------------- the definition, in 64 bits
def _logical(pool, tables, block_rows, seq_rows, i, n):
    """The first n rows of sequence i, put together block by block."""
    if tables is None:
        return pool[i * seq_rows:i * seq_rows + n]
    blocks = [int(b) for b in tables[i, : -(-n // block_rows)]]
    parts = [pool[b * block_rows:(b + 1) * block_rows] for b in blocks]
    return torch.cat(parts)[:n] if parts else pool[:0]


def _place(pool, tables, block_rows, seq_rows, i, j):
    return i * seq_rows + j if tables is None else int(tables[i, j // block_rows]) * block_rows + j % block_rows


def _softmax(x):
    x = x - x.max(-1, keepdim=True)[0]
    e = torch.exp(x)
    return e / e.sum(-1, keepdim=True)


def exact(c, seed):
    s = prepare(c, seed)
    H, K, d = c["n_head"], c["n_head_kv"], c["head_dim"]
    G = H // K
    if c["op"] == "prompt":
        n, w = c["kv_len"], c["window"]
        k = s["k"][:n] if s["table"] is None else _logical(s["k"], s["table"][None], c["block_rows"], 0, 0, n)
        acc = torch.zeros((K, n), dtype=torch.float64, device="cuda")
        late = torch.ones((w, n), dtype=torch.bool, device="cuda").triu(n - w + 1)
        for hq in range(H):
            x = s["q"][c["n_tok"] - w:, hq].double() @ k[:, hq // G].double().T / math.sqrt(d)
            x[late] = -math.inf
            acc[hq // G] += _softmax(x).sum(0)
        return {"acc": acc}
    lens, B = _lens(c), c["block_rows"]
    if c["op"] == "decode":
        out = torch.zeros((c["n_seq"], H, d), dtype=torch.float64, device="cuda")
        acc = s["acc"].double() if c["weights"] else None
        for i, n in enumerate(lens):
            if n == 0:
                continue
            if c["append"]:
                at = _place(s["k"], s["tables"], B, s["seq_rows"], i, n - 1)
                s["k"][at] = s["k_new"][i]
                s["v"][at] = s["v_new"][i]
            k = _logical(s["k"], s["tables"], B, s["seq_rows"], i, n).double()
            v = _logical(s["v"], s["tables"], B, s["seq_rows"], i, n).double()
            for h in range(K):
                p = _softmax(s["q"][i, h * G:(h + 1) * G].double() @ k[:, h].T / math.sqrt(d))
                out[i, h * G:(h + 1) * G] = p @ v[:, h]
                if acc is not None:
                    acc[i, h, :n] += p.sum(0)
        got = {"out": out}
        if c["append"]:
            got |= {"k": s["k"], "v": s["v"]}
        if acc is not None:
            got["acc"] = acc
        return got
    keep, acc_dst = c["n_keep"], torch.zeros_like(s["acc_dst"])
    for i, n in enumerate(lens):
        m = min(n, keep)
        k, v = (_logical(s[t], s["tables"], B, s["seq_rows"], i, n) for t in ("k", "v"))
        to = torch.tensor([_place(s["k_dst"], s["tables_dst"], B, s["seq_rows_dst"], i, j) for j in range(m)],
                          dtype=torch.long, device="cuda")
        a = s["acc"][i, :, :n].cpu().tolist()
        s["new_lens"][i] = m
        for h in range(K):
            fixed = set(range(min(c["sink"], n))) | set(range(max(0, n - c["recent"]), n)) if n > keep else set(range(n))
            rest = sorted((j for j in range(n) if j not in fixed), key=lambda j: (-a[h][j], j))
            rows = torch.tensor(sorted(fixed | set(rest[: m - len(fixed)])), dtype=torch.long, device="cuda")
            s["kept"][i, h] = -1
            s["kept"][i, h, :m] = rows.int()
            s["k_dst"][to, h] = k[rows, h]
            s["v_dst"][to, h] = v[rows, h]
            acc_dst[i, h, :m] = s["acc"][i, h, rows]
    return {"k": s["k_dst"], "v": s["v_dst"], "acc": acc_dst, "new_lens": s["new_lens"], "kept": s["kept"]}
