"""The operators as they are used together: a gated prefill through the paged cache, the prompt's weights, an eviction,
decode steps that keep the weights up to date, a second eviction in place, and a further prefill chunk on the shrunk
cache -- each step against the same steps in 64 bits on a plain cache."""
import math

import pytest
import torch

import epsp
import workloads as W
from serving_util import Cache, TORCH, context, decode64, kept64, prompt64, rounding, workspace

pytestmark = pytest.mark.gpu


class Plain:
    """One sequence's rows per head, as plain tensors (what a Cache offers to decode64)."""

    def __init__(self, k, v):
        self.k, self.v, self.lens, self.cap = k, v, [k.shape[0]], k.shape[0]

    def seq(self, i):
        return self.k, self.v


@pytest.mark.parametrize("dtype,heads,page", [(epsp.BF16, (32, 8, 128), 128), (epsp.F16, (14, 2, 64), 64),
                                              (epsp.F32, (8, 2, 64), 32)], ids=str)
def test_prefill_evict_decode_evict_prefill(dtype, heads, page):
    H, K, d = heads
    n, window, keep, steps, keep2 = 1500, 40, 400, 30, 300
    w = W.Workload("chain", n + 200, 1, H, K, d, dtype, 512, page, 2, 2 * page)
    q, k, v = (t.cuda() for t in W.gen_layer(w, 0))
    B = page
    ctx = context(H, K, d, dtype, epsp.F32, w.n_tokens, page)
    ctx.check(ctx.set_ext(1, 0, 0))
    ctx.check(ctx.set_qg_bound(1, 2, 2, 0))
    blocks = -(-w.n_tokens // B)
    g = torch.Generator().manual_seed(3)
    table = torch.randperm(2 * blocks, generator=g)[:blocks].to(torch.int32).cuda()
    rows = 2 * blocks * B
    kp = torch.full((rows, K, d), float("nan"), dtype=k.dtype, device="cuda")
    vp = kp.clone()
    ctx.check(ctx.set_paged_kv(B, table, blocks, rows))
    at = lambda m: table.long()[torch.arange(m, device="cuda") // B] * B + torch.arange(m, device="cuda") % B  # noqa: E731
    # prefill in chunks, gated
    ctx.set_prefill_mode(True)
    out = torch.zeros(n, H, d, device="cuda")
    for a in range(0, n, 512):
        b = min(n, a + 512)
        ctx.check(ctx.append_kv(0, k[a:b].contiguous(), v[a:b].contiguous(), b - a, kp, vp, a))
        ctx.check(ctx.attend_layer(0, q[a:b].contiguous(), kp, vp, b, b - a, out[a:b]))
    ctx.set_prefill_mode(False)
    last = n - (n - 1) // 512 * 512  # the last chunk's rows
    acc = torch.zeros(K, w.n_tokens, device="cuda")
    qq = q[n - last:n].contiguous()
    begin = last - window
    ctx.check(ctx.prompt_weights(0, qq, kp, n, last, begin, acc, workspace(ctx.prompt_weights_bytes(n, last, begin))))
    ref, tol = prompt64(qq, k, n, last, begin)
    assert ((acc[:, :n].double() - ref).abs() <= tol).all()
    # shrink in place
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    kv = epsp.KvBatch(lens, w.n_tokens, table[None], B, rows)
    acc3 = acc[None]
    kept = torch.zeros(1, K, keep, dtype=torch.int32, device="cuda")
    ws = workspace(max(ctx.evict_bytes(1, w.n_tokens, keep), ctx.decode_bytes(1, w.n_tokens, True)))
    a_host = acc.cpu().tolist()
    want = [kept64(a_host[h][:n], n, keep, 4, 64) for h in range(K)]
    ctx.check(ctx.evict_layer(0, kv, kp, vp, acc3, keep, 4, 64, kv, kp, vp, ws, acc_dst=acc3, new_lens=lens,
                              kept_rows=kept))
    assert kept[0].tolist() == want and int(lens) == keep
    idx = torch.tensor(want, device="cuda")
    pk = torch.stack([k[idx[h], h] for h in range(K)], 1)
    pv = torch.stack([v[idx[h], h] for h in range(K)], 1)
    assert torch.equal(kp[at(keep)], pk) and torch.equal(vp[at(keep)], pv)
    # decode steps; each writes its row and adds its weights
    run = acc3.double().clone()
    lim = torch.zeros_like(run)
    for i in range(steps):
        lens.add_(1)
        m = keep + i + 1
        kn, vn, qn = (t[n + i][None].contiguous() for t in (k, v, q))
        pk, pv = torch.cat([pk, kn]), torch.cat([pv, vn])
        o = torch.zeros(1, H, d, device="cuda")
        ctx.check(ctx.decode_layer(0, kv, qn, kp, vp, o, ws, k_new=kn, v_new=vn, acc=acc3))
        r, t, add, add_tol = decode64(Plain(pk, pv), qn)
        assert ((o.double() - r).abs() <= t + rounding(r, epsp.F32)).all(), i
        run[:, :, :m] += add
        lim[:, :, :m] += add_tol
        lim += run * 2.0 ** -24
        assert ((acc3.double() - run).abs() <= lim).all(), i
    # a second eviction, then a gated prefill chunk over the shrunk cache: the same as on a fresh context
    a_host = acc3[0].cpu().tolist()
    m = keep + steps
    want = torch.tensor([kept64(a_host[h][:m], m, keep2, 4, 64) for h in range(K)], device="cuda")
    ctx.check(ctx.evict_layer(0, kv, kp, vp, acc3, keep2, 4, 64, kv, kp, vp, ws, acc_dst=acc3, new_lens=lens))
    pk = torch.stack([pk[want[h], h] for h in range(K)], 1)
    pv = torch.stack([pv[want[h], h] for h in range(K)], 1)
    assert torch.equal(kp[at(keep2)], pk) and torch.equal(vp[at(keep2)], pv)
    t = 90
    more = slice(n + steps, n + steps + t)
    qn, kn, vn = (x[more].contiguous() for x in (q, k, v))
    fresh = context(H, K, d, dtype, epsp.F32, w.n_tokens, page)
    fresh.check(fresh.set_ext(1, 0, 0))
    outs = []
    for c, kk, vv in ((ctx, kp, vp), (fresh, torch.cat([pk, kn]).contiguous(), torch.cat([pv, vn]).contiguous())):
        c.check(c.set_qg_bound(1, 1, 1, 0))
        c.set_prefill_mode(True)
        if c is ctx:
            c.check(c.append_kv(0, kn, vn, t, kk, vv, keep2))
        o = torch.zeros(t, H, d, device="cuda")
        sel = torch.full((1, K, 64), -1, dtype=torch.int32, device="cuda")
        cnt = torch.zeros((1, K), dtype=torch.int32, device="cuda")
        c.check(c.attend_layer(0, qn, kk, vv, keep2 + t, t, o, sel, cnt, 64))
        torch.cuda.synchronize()
        c.check(c.sync_status())
        outs.append((o, sel, cnt))
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    assert math.isfinite(float(outs[0][0].sum()))


@pytest.mark.parametrize("dtype", [epsp.BF16, epsp.F32], ids=["bf16", "f32"])
def test_prefill_after_decoding_over_a_cut_back_sequence(dtype):
    """A sequence is cut back, continued by decode steps over rows whose pages were summed, then prefilled further:
    the selection sees the new rows."""
    H, K, d, P = 8, 2, 64, 32
    n, back, t = 600, 300, 130
    w = W.Workload("back", 1000, 1, H, K, d, dtype, 1000, P, 2, 2 * P)
    q, k, v = (x.cuda() for x in W.gen_layer(w, 0))
    outs = []
    for fresh in (False, True):
        ctx = context(H, K, d, dtype, epsp.F32, 1000, P)
        ctx.check(ctx.set_ext(1, 0, 0))
        ctx.check(ctx.set_qg_bound(1, 2, 2, 0))
        ctx.set_prefill_mode(True)
        kc, vc = torch.zeros_like(k), torch.zeros_like(v)
        o = torch.zeros(n, H, d, device="cuda")
        if fresh:
            kc[:n], vc[:n] = k[:n], v[:n]
        else:
            ctx.check(ctx.append_kv(0, k[:n].contiguous(), v[:n].contiguous(), n, kc, vc, 0))
            ctx.check(ctx.attend_layer(0, q[:n].contiguous(), kc, vc, n, n, o))
        rows = range(back, back + 70)
        if fresh:
            for i, r in enumerate(rows):
                kc[r], vc[r] = 3 * k[n + i], v[n + i]
        else:
            ws = workspace(ctx.decode_bytes(1, 1000, False))
            lens = torch.tensor([back], dtype=torch.int32, device="cuda")
            kv = epsp.KvBatch(lens, 1000, seq_rows=1000)
            out = torch.zeros(1, H, d, device="cuda")
            for i, r in enumerate(rows):
                lens.add_(1)
                ctx.check(ctx.decode_layer(0, kv, q[r][None].contiguous(), kc, vc, out, ws,
                                           k_new=(3 * k[n + i])[None].contiguous(), v_new=v[n + i][None].contiguous()))
        u0 = back + 70
        kc[u0:u0 + t], vc[u0:u0 + t] = k[800:800 + t], v[800:800 + t]
        o = torch.zeros(t, H, d, device="cuda")
        sel = torch.full((1, K, 64), -1, dtype=torch.int32, device="cuda")
        cnt = torch.zeros((1, K), dtype=torch.int32, device="cuda")
        ctx.check(ctx.attend_layer(0, q[800:800 + t].contiguous(), kc, vc, u0 + t, t, o, sel, cnt, 64))
        torch.cuda.synchronize()
        ctx.check(ctx.sync_status())
        outs.append((o, sel, cnt))
    assert int(outs[0][2].sum()) > 0
    for a, b in zip(*outs):
        assert torch.equal(a, b)


def test_blocks_past_32_bit_offsets():
    """Pools of 2.2 M rows of 8 heads x 128 bf16 (4.5 GB each): the sequence's blocks lie at the end, past 2^31 elements
    and 2^32 bytes."""
    H, K, d, P, n, keep = 32, 8, 128, 128, 700, 256
    rows = 17200 * P
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(n, K, d, generator=g).bfloat16().cuda() for _ in range(2))
    kp, vp = (torch.empty(rows, K, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    used = -(-n // P)
    table = torch.tensor([17199 - 3 * i for i in range(used)], dtype=torch.int32, device="cuda")
    far = torch.tensor([17198, 17195], dtype=torch.int32, device="cuda")
    at = table.long()[torch.arange(n, device="cuda") // P] * P + torch.arange(n, device="cuda") % P
    assert int(at.min()) * K * d > 2 ** 31
    kp[at], vp[at] = k, v
    ctx = context(H, K, d, epsp.BF16, epsp.F32, 1024, P)
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    kv = epsp.KvBatch(lens, n, table[None], P, rows)
    q = torch.randn(40, H, d, generator=g).bfloat16().cuda()
    out, acc = torch.zeros(1, H, d, device="cuda"), torch.zeros(1, K, n, device="cuda")
    new = torch.randn(2, 1, K, d, generator=g).bfloat16().cuda()
    ws = workspace(max(ctx.decode_bytes(1, n, True), ctx.prompt_weights_bytes(n, 40, 0), ctx.evict_bytes(1, n, keep)))
    ctx.check(ctx.decode_layer(0, kv, q[:1].contiguous(), kp, vp, out, ws, k_new=new[0], v_new=new[1], acc=acc))
    k[-1], v[-1] = new[0, 0], new[1, 0]
    ref, tol, add, add_tol = decode64(Plain(k, v), q[:1])
    assert ((out.double() - ref).abs() <= tol + rounding(ref, epsp.F32)).all()
    assert ((acc.double() - add).abs() <= add_tol).all()
    assert torch.equal(kp[at[-1]], new[0, 0]) and torch.equal(vp[at[-1]], new[1, 0])
    ctx.check(ctx.set_paged_kv(P, table, used, rows))
    acc2 = torch.zeros(K, n, device="cuda")
    ctx.check(ctx.prompt_weights(0, q, kp, n, 40, 0, acc2, ws))
    ref, tol = prompt64(q, k, n, 40, 0)
    assert ((acc2.double() - ref).abs() <= tol).all()
    dst = epsp.KvBatch(None, keep, far[None], P, rows, n_seq=1)
    ctx.check(ctx.evict_layer(0, kv, kp, vp, acc2[None], keep, 4, 30, dst, kp, vp, ws))
    ctx.check(ctx.sync_status())
    a_host = acc2.cpu().tolist()
    to = far.long()[torch.arange(keep, device="cuda") // P] * P + torch.arange(keep, device="cuda") % P
    for h in range(K):
        idx = torch.tensor(kept64(a_host[h], n, keep, 4, 30), device="cuda")
        assert torch.equal(kp[to, h], k[idx, h]) and torch.equal(vp[to, h], v[idx, h])


def test_calls_on_two_streams_at_once():
    """Two sequences' steps on two streams of one context, each with its own workspace and caches."""
    H, K, d, n = 8, 2, 64, 3000
    ctx = context(H, K, d, epsp.F16, epsp.F32, n, 32)
    sides = []
    for seed in (1, 2):
        g = torch.Generator().manual_seed(seed)
        c = Cache([n], K, d, epsp.F16, 32, seed)
        q = torch.randn(30, H, d, generator=g).half().cuda()
        small = Cache([500], K, d, epsp.F16, 32, seed + 9)
        need = max(ctx.decode_bytes(1, n, True), ctx.evict_bytes(1, n, 500), ctx.prompt_weights_bytes(n, 30, 0))
        sides.append(dict(c=c, q=q, q1=q[:1].contiguous(), out=torch.zeros(1, H, d, device="cuda"), small=small,
                          acc=torch.zeros(1, K, n, device="cuda"), ws=workspace(need), s=torch.cuda.Stream(),
                          wacc=torch.zeros(K, n, device="cuda"),
                          kept=torch.zeros(1, K, 500, dtype=torch.int32, device="cuda")))
    torch.cuda.synchronize()
    for _ in range(20):
        for x in sides:
            with torch.cuda.stream(x["s"]):
                x["acc"].zero_()
                c = x["c"]
                ctx.check(ctx.decode_layer(0, c.batch, x["q1"], c.k, c.v, x["out"], x["ws"], acc=x["acc"]))
                ctx.check(ctx.set_paged_kv(32, c.d_table[0], c.d_table.shape[1], c.rows))
                ctx.check(ctx.prompt_weights(0, x["q"], c.k, n, 30, 0, x["wacc"], x["ws"]))
                ctx.check(ctx.evict_layer(0, c.batch, c.k, c.v, x["acc"], 500, 4, 30, x["small"].batch, x["small"].k,
                                          x["small"].v, x["ws"], kept_rows=x["kept"]))
    torch.cuda.synchronize()
    ctx.check(ctx.sync_status())
    for x in sides:
        ref, tol, add, add_tol = decode64(x["c"], x["q1"])
        assert ((x["out"].double() - ref).abs() <= tol + rounding(ref, epsp.F32)).all()
        assert ((x["acc"].double() - add).abs() <= add_tol).all()
        ref, tol = prompt64(x["q"], x["c"].seq(0)[0], n, 30, 0)
        assert ((x["wacc"].double() - ref).abs() <= tol).all()
        a_host = x["acc"][0].cpu().tolist()
        assert x["kept"][0].tolist() == [kept64(a_host[h], n, 500, 4, 30) for h in range(K)]


@pytest.mark.parametrize("dtype", [epsp.BF16, epsp.F32], ids=["bf16", "f32"])
def test_calls_that_follow_each_other_without_a_wait(dtype):
    """Evictions in place that rewrite the lengths the next call reads, and decode steps on the rows they leave: back to
    back the same as with a wait after each call."""
    H, K, d, B = 8, 2, 64, 64
    lens0 = [1500, 900, 64, 0, 301]
    n_seq = len(lens0)

    def run(wait):
        cache = Cache(lens0, K, d, dtype, B, 9)
        ctx = context(H, K, d, dtype, dtype, 2048, B)
        g = torch.Generator().manual_seed(3)
        q = torch.randn(12, n_seq, H, d, generator=g).to(TORCH[dtype]).cuda()
        acc = torch.rand(n_seq, K, cache.cap, generator=g).cuda()
        ws = workspace(max(ctx.decode_bytes(n_seq, cache.cap, True), ctx.evict_bytes(n_seq, cache.cap, 1400)))
        out = torch.zeros(12, n_seq, H, d, dtype=TORCH[dtype], device="cuda")
        torch.cuda.synchronize()
        for i in range(12):
            keep = 1400 - 110 * i
            ctx.check(ctx.evict_layer(0, cache.batch, cache.k, cache.v, acc, keep, 3, 17, cache.batch, cache.k, cache.v,
                                      ws, acc_dst=acc, new_lens=cache.d_lens))
            if wait:
                torch.cuda.synchronize()
            ctx.check(ctx.decode_layer(0, cache.batch, q[i], cache.k, cache.v, out[i], ws, acc=acc))
            if wait:
                torch.cuda.synchronize()
        ctx.check(ctx.sync_status())
        assert cache.d_lens.tolist() == [min(n, 1400 - 110 * 11) for n in lens0]
        return out, acc

    for x, y in zip(run(False), run(True)):
        assert torch.equal(x, y)
