"""ep_sp_evict_layer against the definition, row for row: which rows each head keeps (ties, NaN, infinities, rows that
must stay), where they go, and that nothing else changes."""
import math

import pytest
import torch

import epsp
from serving_util import Cache, TORCH, context, kept64, workspace

pytestmark = pytest.mark.gpu

F32, F16, BF16 = epsp.F32, epsp.F16, epsp.BF16


def same(a, b):
    """Bit equality (NaN rows included)."""
    bits = {4: torch.int32, 2: torch.int16}[a.element_size()]
    return torch.equal(a.view(bits), b.view(bits))


def weights(kind, n_seq, K, stride, seed):
    g = torch.Generator().manual_seed(seed)
    a = torch.exp(torch.randn(n_seq, K, stride, generator=g) * 1.5)
    if kind == "ties":  # few values, many equal
        a = torch.randint(0, 4, a.shape, generator=g).float()
    elif kind == "equal":
        a = torch.full_like(a, 0.25)
    elif kind == "odd":  # NaN, infinities, signed zeros, negatives, subnormals
        pick = torch.randint(0, 10, a.shape, generator=g)
        for i, x in enumerate((math.nan, math.inf, -math.inf, 0.0, -0.0, -1.5, 1e-45, -1e-45)):
            a[pick == i] = x
    return a.cuda()


def expected(cache, acc, n_keep, sink, recent):
    a = acc.cpu().tolist()
    K = acc.shape[1]
    return [[kept64(a[i][h][:n], n, n_keep, sink, recent) for h in range(K)] for i, n in enumerate(cache.lens)]


def run_case(lens, n_keep, sink, recent, heads, dtype, page, block, kind="random", mode="gather", dst_block=None,
             seed=0, extras=True):
    H, K, d = heads
    src = Cache(lens, K, d, dtype, block, seed)
    n_seq, cap = len(lens), src.cap
    most = min(n_keep, cap)
    acc = weights(kind, n_seq, K, cap + 3, seed)
    acc0, k0, v0 = acc.clone(), src.k.clone(), src.v.clone()
    ctx = context(H, K, d, dtype, dtype, max(cap, n_keep), page)
    want = expected(src, acc, n_keep, sink, recent)
    if mode == "place":
        dst, kd, vd = src, src.k, src.v
        acc_dst = acc
        new_lens = src.d_lens  # written over the lengths the call reads
        dst_batch = src.batch
    else:
        dst = Cache([most] * n_seq, K, d, dtype, block if dst_block is None else dst_block, seed + 50)
        kd, vd, dst_batch = dst.k, dst.v, dst.batch
        acc_dst = torch.full((n_seq, K, most + 2), 9.0, device="cuda") if extras else None
        new_lens = torch.full((n_seq,), -7, dtype=torch.int32, device="cuda") if extras else None
    kd0, vd0 = kd.clone(), vd.clone()
    kept = torch.full((n_seq, K, n_keep), -9, dtype=torch.int32, device="cuda") if extras else None
    ws = workspace(ctx.evict_bytes(n_seq, cap, n_keep))
    ctx.check(ctx.evict_layer(0, src.batch, src.k, src.v, acc, n_keep, sink, recent, dst_batch, kd, vd, ws,
                              acc_dst=acc_dst, new_lens=new_lens, kept_rows=kept))
    torch.cuda.synchronize()
    ctx.check(ctx.sync_status())
    kw, vw = kd0.clone(), vd0.clone()
    for i, n in enumerate(lens):
        m = min(n, n_keep)
        frm, to = src.at(i, n).cuda(), dst.at(i, m).cuda()
        for h in range(K):
            rows = torch.tensor(want[i][h], dtype=torch.long, device="cuda")
            assert len(rows) == m
            if extras:
                assert kept[i, h, :m].tolist() == want[i][h], (i, h)
                assert (kept[i, h, m:] == -1).all()
            kw[to, h], vw[to, h] = k0[frm[rows], h], v0[frm[rows], h]
            if acc_dst is not None:
                assert same(acc_dst[i, h, :m].contiguous(), acc0[i, h, rows].contiguous())
                assert (acc_dst[i, h, m:] == 0).all()
        if new_lens is not None:
            assert int(new_lens[i]) == m
    assert same(kd, kw) and same(vd, vw)  # rows past the kept ones, and other blocks, as they were
    if mode == "gather":
        assert same(src.k, k0) and same(src.v, v0) and same(acc, acc0)


LENS = [0, 1, 5, 31, 32, 33, 64, 100, 101, 128, 500, 1023, 1024, 1025, 2100]
SHAPES = [(BF16, (32, 8, 128), 128, 128), (BF16, (28, 4, 128), 64, 64), (F16, (14, 2, 64), 64, 0),
          (F32, (9, 3, 128), 32, 96), (F32, (4, 4, 64), 32, 0)]


@pytest.mark.parametrize("mode", ["gather", "place"])
@pytest.mark.parametrize("kind", ["random", "ties", "equal", "odd"])
@pytest.mark.parametrize("dtype,heads,page,block", SHAPES, ids=str)
def test_ragged_batch(dtype, heads, page, block, kind, mode):
    run_case(LENS, 100, 4, 30, heads, dtype, page, block, kind, mode, seed=len(kind))


@pytest.mark.parametrize("mode", ["gather", "place"])
@pytest.mark.parametrize("n_keep,sink,recent", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (64, 64, 0), (64, 0, 64), (64, 30, 34),
                                                (33, 0, 0), (999, 3, 500), (1000, 0, 0), (5000, 4, 4)], ids=str)
def test_budgets(n_keep, sink, recent, mode):
    run_case([1000, 999, 50, 1], n_keep, sink, recent, (8, 2, 64), F16, 32, 32, "ties", mode, seed=n_keep)


@pytest.mark.parametrize("mode", ["gather", "place"])
@pytest.mark.parametrize("n,n_keep", [(20000, 3000), (70000, 5), (70001, 69999), (66000, 16500)])
def test_long_sequences(n, n_keep, mode):
    run_case([n], n_keep, min(4, n_keep // 2), min(300, n_keep // 2), (4, 2, 64), BF16, 64, 64, "random", mode, seed=n)
    run_case([n], n_keep, 0, 0, (4, 2, 64), BF16, 64, 64, "ties", mode, seed=n)


@pytest.mark.parametrize("mode", ["gather", "place"])
def test_weights_longer_than_a_cluster_keeps_on_chip(mode):
    run_case([300001, 5], 70000, 4, 1000, (1, 1, 64), F16, 32, 32, "ties", mode, seed=8)


def test_many_short_sequences():
    run_case([1 + 13 * i % 200 for i in range(200)], 40, 2, 10, (14, 2, 64), F16, 64, 64)


def test_between_layouts_and_without_the_extra_outputs():
    run_case([300, 7, 90], 64, 1, 8, (8, 2, 64), BF16, 32, 32, dst_block=0)
    run_case([300, 7, 90], 64, 1, 8, (8, 2, 64), BF16, 32, 0, dst_block=96)
    run_case([300, 7, 90], 64, 1, 8, (8, 2, 64), BF16, 32, 32, dst_block=64, extras=False)


def test_into_other_blocks_of_the_same_pool():
    """The usual paged use: the kept rows go to fresh blocks of the pool, after which the old ones are free."""
    K, d, B, n, keep = 2, 64, 32, 500, 100
    src = Cache([n], K, d, BF16, B, 1, capacity=n + 200)
    acc = weights("random", 1, K, src.cap, 1)
    used = -(-n // B)
    fresh = src.d_table[:, used:used + 4].contiguous()
    dst = epsp.KvBatch(None, keep, fresh, B, src.rows, n_seq=1)
    k0, v0 = src.k.clone(), src.v.clone()
    ctx = context(4, K, d, BF16, BF16, src.cap, 32)
    ctx.check(ctx.evict_layer(0, src.batch, src.k, src.v, acc, keep, 4, 10, dst, src.k, src.v,
                              workspace(ctx.evict_bytes(1, src.cap, keep))))
    torch.cuda.synchronize()
    want = expected(src, acc, keep, 4, 10)[0]
    to = (fresh[0].long()[torch.arange(keep, device="cuda") // B] * B + torch.arange(keep, device="cuda") % B)
    for h in range(K):
        rows = torch.tensor(want[h], device="cuda")
        k0[to, h], v0[to, h] = k0[src.at(0, n).cuda()[rows], h], v0[src.at(0, n).cuda()[rows], h]
    assert same(src.k, k0) and same(src.v, v0)


def test_bad_lengths_and_table_entries_are_reported():
    K, d, B = 2, 64, 32
    ctx = context(4, K, d, BF16, BF16, 512, 32)
    for where in ("len", "long", "src", "dst"):
        src, dst = Cache([100, 60], K, d, BF16, B, 9), Cache([40, 40], K, d, BF16, B, 10)
        acc = weights("random", 2, K, 100, 1)
        if where == "len":
            src.d_lens[0] = -3
        elif where == "long":
            src.d_lens[0] = 101
        elif where == "src":
            src.d_table[0] = 10 ** 7
        else:
            dst.d_table[0, 0] = -1
        new = torch.zeros(2, dtype=torch.int32, device="cuda")
        kept = torch.zeros(2, K, 40, dtype=torch.int32, device="cuda")
        ctx.check(ctx.evict_layer(0, src.batch, src.k, src.v, acc, 40, 0, 5, dst.batch, dst.k, dst.v,
                                  workspace(ctx.evict_bytes(2, 100, 40)), new_lens=new, kept_rows=kept))
        assert ctx.sync_status() == epsp.PREFILL and ctx.sync_status() == epsp.OK
        src.lens = [0, 60]
        want = expected(src, acc, 40, 0, 5)[1]
        assert kept[1].tolist() == want and int(new[1]) == 40  # the other sequence is served
        if where in ("len", "long"):
            assert int(new[0]) == 0 and (kept[0] == -1).all()


def test_captured_replay_and_another_stream():
    K, d, B, n, keep = 4, 128, 64, 3000, 512
    src, dst = Cache([n, 700], K, d, BF16, B, 3), Cache([keep, keep], K, d, BF16, B, 4)
    ctx = context(8, K, d, BF16, BF16, n, 64)
    acc = weights("random", 2, K, n, 5)
    kept = torch.zeros(2, K, keep, dtype=torch.int32, device="cuda")
    ws = workspace(ctx.evict_bytes(2, n, keep))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ctx.check(ctx.evict_layer(0, src.batch, src.k, src.v, acc, keep, 4, 64, dst.batch, dst.k, dst.v, ws,
                                  kept_rows=kept))
    side = torch.cuda.Stream()
    for seed in (5, 6):
        acc.copy_(weights("random", 2, K, n, seed))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        torch.cuda.synchronize()
        want = expected(src, acc, keep, 4, 64)
        assert [[kept[i, h, :len(want[i][h])].tolist() for h in range(K)] for i in range(2)] == want
    ctx.check(ctx.sync_status())
