"""ep_sp_decode_layer against a 64-bit softmax attention: types, head layouts, lengths from none to many, paged and
contiguous caches with NaN in every row that no sequence holds, the fused append and the accumulated weights."""
import pytest
import torch

import epsp
import workloads as W
from serving_util import Cache, TORCH, context, decode64, rounding, workspace

pytestmark = pytest.mark.gpu

F32, F16, BF16 = epsp.F32, epsp.F16, epsp.BF16


def run_case(lens, heads, dtype, out_dtype, page, block, append, weights, seed=0, cap=None, extra_stride=0):
    H, K, d = heads
    cache = Cache(lens, K, d, dtype, block, seed, capacity=cap)
    g = torch.Generator().manual_seed(seed + 100)
    n_seq = len(lens)
    rnd = lambda *s: torch.randn(*s, generator=g).to(TORCH[dtype]).cuda()  # noqa: E731
    q = rnd(n_seq, H, d)
    k_new, v_new = (rnd(n_seq, K, d), rnd(n_seq, K, d)) if append else (None, None)
    if append:  # the cache's own last row is stale
        for i, n in enumerate(lens):
            if n:
                cache.k[cache.at(i, n)[-1].item()] = float("nan")
                cache.v[cache.at(i, n)[-1].item()] = float("nan")
    acc = torch.rand(n_seq, K, cache.cap + extra_stride, generator=g).cuda() if weights else None
    acc0 = None if acc is None else acc.clone()
    k0, v0 = cache.k.clone(), cache.v.clone()
    ctx = context(H, K, d, dtype, out_dtype, max(cache.cap, 1), page)
    out = torch.full((n_seq, H, d), float("nan"), dtype=TORCH[out_dtype], device="cuda")
    ws = workspace(ctx.decode_bytes(n_seq, cache.cap, weights))
    ctx.check(ctx.decode_layer(0, cache.batch, q, cache.k, cache.v, out, ws, k_new=k_new, v_new=v_new, acc=acc))
    torch.cuda.synchronize()
    ctx.check(ctx.sync_status())
    # the caches hold exactly what they held, plus the new rows
    for i, n in enumerate(lens):
        if append and n:
            at = cache.at(i, n)[-1].item()
            k0[at], v0[at] = k_new[i], v_new[i]
    assert torch.equal(torch.nan_to_num(cache.k.float(), nan=7e4), torch.nan_to_num(k0.float(), nan=7e4))
    assert torch.equal(torch.nan_to_num(cache.v.float(), nan=7e4), torch.nan_to_num(v0.float(), nan=7e4))
    ref, tol, add, add_tol = decode64(cache, q, k_new=k_new, v_new=v_new)
    err = (out.double() - ref).abs()
    assert torch.isfinite(out).all()
    assert (err <= tol + rounding(ref, out_dtype)).all(), float((err - tol - rounding(ref, out_dtype)).max())
    if weights:
        want = acc0.double()
        want[..., :cache.cap] += add
        lim = want.abs() * 2.0 ** -24
        lim[..., :cache.cap] += add_tol
        bad = (acc.double() - want).abs() - lim
        assert (bad <= 0).all(), float(bad.max())
        for i, n in enumerate(lens):  # rows past a sequence's length are left alone
            assert torch.equal(acc[i, :, n:], acc0[i, :, n:])
    return out


LENS = [0, 1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 500, 1000, 1031]


@pytest.mark.parametrize("weights", [False, True], ids=["plain", "weights"])
@pytest.mark.parametrize("append", [False, True], ids=["kept", "append"])
@pytest.mark.parametrize("dtype,heads,page,block", [
    (BF16, (32, 8, 128), 128, 128), (BF16, (28, 4, 128), 64, 64), (F16, (14, 2, 64), 64, 0), (F16, (8, 8, 64), 32, 32),
    (F32, (14, 2, 64), 64, 64), (F32, (9, 3, 128), 32, 96), (BF16, (16, 1, 128), 32, 0)], ids=str)
def test_ragged_batch(dtype, heads, page, block, append, weights):
    run_case(LENS, heads, dtype, dtype, page, block, append, weights)


@pytest.mark.parametrize("n", [1, 7, 32, 300, 2049, 9000])
@pytest.mark.parametrize("dtype,heads", [(BF16, (32, 8, 128)), (F16, (14, 2, 64)), (F32, (4, 4, 128))], ids=str)
def test_one_sequence_f32_output(dtype, heads, n):
    run_case([n], heads, dtype, F32, 64, 64, True, True, seed=n)


@pytest.mark.parametrize("heads", [(1, 1, 64), (2, 1, 128), (3, 1, 64), (17, 1, 64), (33, 1, 128), (64, 1, 64),
                                   (65, 1, 64), (96, 1, 128), (128, 1, 64), (128, 1, 128), (40, 2, 128)], ids=str)
@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_query_heads_per_kv_head(heads, dtype):
    run_case([5, 0, 129, 700], heads, dtype, F32, 32, 32, True, True, seed=heads[0])


@pytest.mark.parametrize("heads", [(7, 1, 128), (17, 1, 64), (65, 1, 128), (128, 1, 64), (256, 2, 128)], ids=str)
@pytest.mark.parametrize("dtype,out", [(BF16, BF16), (BF16, F32), (F16, F16), (F32, F32)], ids=["bf16", "bf16_f32", "f16", "f32"])
def test_few_rows_without_a_split(heads, dtype, out):
    """Up to 512 rows and as many runs as SMs: a CTA per run, no second kernel unless weights are kept."""
    run_case([3, 0, 300, 512], heads, dtype, out, 32, 32, True, False, seed=heads[0])
    run_case([33], heads, dtype, out, 32, 0, False, True, seed=heads[0])


@pytest.mark.parametrize("weights", [False, True], ids=["plain", "weights"])
@pytest.mark.parametrize("dtype,heads,out", [
    (BF16, (8, 2, 128), BF16), (F16, (14, 2, 64), F16), (BF16, (28, 2, 64), F32), (F32, (7, 1, 64), F32),
    (F32, (4, 2, 128), F32), (BF16, (128, 1, 128), BF16), (F32, (40, 1, 64), F32)], ids=str)
@pytest.mark.parametrize("lens", [[513], [900, 0, 1, 33], [1024, 40, 0], [1500, 1], [2048, 1025, 31]], ids=str)
def test_short_runs_joined_in_a_cluster(lens, dtype, heads, out, weights):
    """Few runs of up to 2048 rows: a cluster of 2 to 8 CTAs each, some of them without rows."""
    run_case(lens, heads, dtype, out, 32, 32, True, weights, seed=lens[0])
    run_case(lens, heads, dtype, out, 32, 0, False, weights, seed=lens[0], extra_stride=3)


def test_empty_batch_and_capacity_above_the_lengths():
    run_case([0, 0, 0], (32, 8, 128), BF16, BF16, 128, 128, True, True, cap=5000)
    run_case([3, 0, 70], (32, 8, 128), BF16, BF16, 128, 128, True, True, cap=5000, extra_stride=13)
    run_case([0], (14, 2, 64), F32, F32, 64, 0, False, False, cap=1)


def test_many_sequences_of_one_long_and_the_rest_short():
    run_case([6000] + [1 + i % 40 for i in range(300)], (8, 2, 64), F16, F16, 32, 32, False, True)


def test_more_sequences_than_a_cta_keeps_the_lengths_of():
    run_case([(7 * i) % 45 for i in range(2500)], (4, 2, 64), F16, F16, 32, 32, True, True)


def test_long_cache_spread_over_the_device():
    run_case([40000, 25000], (28, 4, 128), BF16, BF16, 128, 256, True, True, seed=3)


def test_all_scores_equal_and_large_scores():
    """Equal scores: every weight is 1/n.  Scores of +-80: all weight on a few rows, nothing overflows."""
    d, H, K, n = 128, 8, 2, 777
    ctx = context(H, K, d, BF16, F32, 1024, 32)
    cache = Cache([n], K, d, BF16, 32, 0)
    q = torch.zeros(1, H, d, dtype=torch.bfloat16, device="cuda")
    out = torch.zeros(1, H, d, device="cuda")
    acc = torch.zeros(1, K, n, device="cuda")
    ws = workspace(ctx.decode_bytes(1, n, True))
    ctx.check(ctx.decode_layer(0, cache.batch, q, cache.k, cache.v, out, ws, acc=acc))
    ref, tol, add, add_tol = decode64(cache, q)
    assert ((out.double() - ref).abs() <= tol + rounding(ref, F32)).all()
    assert ((acc.double() - add).abs() <= add_tol).all()
    q = torch.where(torch.arange(d, device="cuda") < 64, 8.0, -8.0).to(torch.bfloat16).expand(1, H, d).contiguous()
    ctx.check(ctx.decode_layer(0, cache.batch, q, cache.k, cache.v, out, ws))
    ref, tol, _, _ = decode64(cache, q)
    assert ((out.double() - ref).abs() <= tol + rounding(ref, F32)).all()


def test_rows_of_minus_infinity_weigh_nothing():
    """Keys whose scores are -inf (an f16 infinity in the row) get weight 0 wherever they stand, the first rows of the
    cache included."""
    d, H, K, n = 64, 4, 2, 300
    ctx = context(H, K, d, F16, F32, 512, 32)
    cache = Cache([n], K, d, F16, 32, 1)
    q = torch.rand(1, H, d, generator=torch.Generator().manual_seed(1)).half().cuda() + 0.5
    dead = list(range(0, 96)) + [150, 299]
    at = cache.at(0, n).cuda()
    cache.k[at[dead], :, 5] = float("-inf")
    out, acc = torch.zeros(1, H, d, device="cuda"), torch.zeros(1, K, n, device="cuda")
    ws = workspace(ctx.decode_bytes(1, n, True))
    ctx.check(ctx.decode_layer(0, cache.batch, q, cache.k, cache.v, out, ws, acc=acc))
    alive = torch.tensor([j for j in range(n) if j not in dead], device="cuda")
    k, v = (t[at][alive] for t in (cache.k, cache.v))
    for hq in range(H):
        p = torch.softmax(q[0, hq].double() @ k[:, hq // 2].double().T / 8.0, -1)
        assert ((out[0, hq].double() - p @ v[:, hq // 2].double()).abs() <= 1e-3).all()
    assert (acc[0][:, dead] == 0).all() and torch.isfinite(acc).all()


def test_scale_and_slice_of_heads():
    """kq_scale is the context's; a context over a slice of the KV heads gives that slice's rows."""
    H, K, d = 8, 4, 64
    cache = Cache([200, 77], K, d, F16, 0, 5)
    q = torch.randn(2, H, d, generator=torch.Generator().manual_seed(2)).half().cuda()
    ctx = context(H, K, d, F16, F32, 256, 32, kq_scale=0.31)
    out = torch.zeros(2, H, d, device="cuda")
    ws = workspace(ctx.decode_bytes(2, cache.cap, False))
    ctx.check(ctx.decode_layer(0, cache.batch, q, cache.k, cache.v, out, ws))
    ref, tol, _, _ = decode64(cache, q, scale=0.31)
    assert ((out.double() - ref).abs() <= tol + rounding(ref, F32)).all()
    part = context(4, 2, d, F16, F32, 256, 32, kq_scale=0.31, kv_head_offset=2, n_head_kv_total=4)
    ks, vs = cache.k[:, 2:].contiguous(), cache.v[:, 2:].contiguous()
    sub = torch.zeros(2, 4, d, device="cuda")
    part.check(part.decode_layer(0, cache.batch, q[:, 4:].contiguous(), ks, vs, sub,
                                 workspace(part.decode_bytes(2, cache.cap, False))))
    assert ((sub.double() - ref[:, 4:]).abs() <= tol[:, 4:] + rounding(ref[:, 4:], F32)).all()


def test_sequences_sharing_blocks():
    """A common prefix held once: two sequences' tables name the same blocks."""
    H, K, d, B = 8, 2, 64, 32
    cache = Cache([96, 160], K, d, F16, B, 9)
    table = cache.d_table.clone()
    table[0, :2] = table[1, :2]
    cache.table = table.cpu()
    kv = epsp.KvBatch(cache.d_lens, cache.cap, table, B, cache.rows)
    q = torch.randn(2, H, d, generator=torch.Generator().manual_seed(2)).half().cuda()
    ctx = context(H, K, d, F16, F32, 256, 32)
    out = torch.zeros(2, H, d, device="cuda")
    ctx.check(ctx.decode_layer(0, kv, q, cache.k, cache.v, out, workspace(ctx.decode_bytes(2, cache.cap, False))))
    ref, tol, _, _ = decode64(cache, q)
    assert ((out.double() - ref).abs() <= tol + rounding(ref, F32)).all()


def test_bad_table_entries_and_lengths_are_reported():
    H, K, d, B = 8, 2, 64, 32
    ctx = context(H, K, d, BF16, BF16, 512, 32)
    for bad in (10 ** 6, -1, 2 ** 31 - 1):
        cache = Cache([100, 60], K, d, BF16, B, 9)
        cache.d_table[0, 1] = bad
        q, out = (torch.zeros(2, H, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        new = torch.ones(2, K, d, dtype=torch.bfloat16, device="cuda")
        ws = workspace(ctx.decode_bytes(2, cache.cap, True))
        acc = torch.zeros(2, K, cache.cap, device="cuda")
        ctx.check(ctx.decode_layer(0, cache.batch, q, cache.k, cache.v, out, ws, k_new=new, v_new=new, acc=acc))
        assert ctx.sync_status() == epsp.PREFILL
        assert ctx.sync_status() == epsp.OK
        # the other sequence is not touched by it
        cache.lens[0] = 0
        ref, tol, _, _ = decode64(cache, q, k_new=new, v_new=new)
        assert ((out[1].double() - ref[1]).abs() <= tol[1] + rounding(ref[1], BF16)).all()
    for bad in (-1, 101, 2 ** 31 - 1, -2 ** 31):
        cache = Cache([100, 60], K, d, BF16, B, 9)
        cache.d_lens[0] = bad
        ctx.check(ctx.decode_layer(0, cache.batch, q, cache.k, cache.v, out, ws, k_new=new, v_new=new, acc=acc))
        assert ctx.sync_status() == epsp.PREFILL
        assert (out[0] == 0).all()
        cache.lens[0] = 0
        ref, tol, _, _ = decode64(cache, q, k_new=new, v_new=new)
        assert ((out[1].double() - ref[1]).abs() <= tol[1] + rounding(ref[1], BF16)).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("shift", [16, 48, 112])
def test_any_16_byte_workspace_and_4_byte_weights(dtype, shift):
    """The workspace may start at any multiple of 16 bytes and the weights at any of 4; nothing around either of them
    changes, and the results are the same."""
    heads, lens = (20, 2, 64), [2300, 0, 129, 1025]
    ctx = context(*heads, dtype, dtype, 4096, 64)
    cache = Cache(lens, heads[1], heads[2], dtype, 0, 5)
    q = torch.randn(len(lens), heads[0], heads[2], generator=torch.Generator().manual_seed(1)).to(TORCH[dtype]).cuda()
    n = ctx.decode_bytes(len(lens), cache.cap, True)

    def run(before, first):
        raw = torch.full((before + n + 256,), 0xAB, dtype=torch.uint8, device="cuda")
        flat = torch.full((first + len(lens) * heads[1] * cache.cap + 8,), 3.0, device="cuda")
        acc = flat[first:-8].view(len(lens), heads[1], cache.cap)
        out = torch.empty_like(q)
        ctx.check(ctx.decode_layer(0, cache.batch, q, cache.k, cache.v, out, raw[before:before + n], acc=acc))
        torch.cuda.synchronize()
        assert (raw[:before] == 0xAB).all() and (raw[before + n:] == 0xAB).all()
        assert (flat[:first] == 3).all() and (flat[-8:] == 3).all()
        return out, acc.clone()

    for x, y in zip(run(0, 0), run(shift, shift // 16)):
        assert torch.equal(x, y)


def test_same_result_every_time_and_on_another_stream():
    H, K, d = 32, 8, 128
    cache = Cache([3000, 17, 900, 0, 2222], K, d, BF16, 128, 4)
    g = torch.Generator().manual_seed(1)
    q = torch.randn(5, H, d, generator=g).bfloat16().cuda()
    ctx = context(H, K, d, BF16, F32, 4096, 128)
    ws = workspace(ctx.decode_bytes(5, cache.cap, True))
    outs, accs = [], []
    side = torch.cuda.Stream()
    for i in range(4):
        out, acc = torch.zeros(5, H, d, device="cuda"), torch.zeros(5, K, cache.cap, device="cuda")
        torch.cuda.synchronize()
        with torch.cuda.stream(side if i % 2 else torch.cuda.default_stream()):
            ctx.check(ctx.decode_layer(0, cache.batch, q, cache.k, cache.v, out, ws, acc=acc))
        torch.cuda.synchronize()
        outs.append(out)
        accs.append(acc)
    assert all(torch.equal(o, outs[0]) for o in outs) and all(torch.equal(a, accs[0]) for a in accs)


def test_captured_steps_replay_as_the_lengths_grow():
    """Two graphs with a workspace each, replayed at the same time on two streams while the lengths, the tokens and
    their K/V rows change in place; a capture before ep_sp_reserve is refused."""
    H, K, d, B, cap = 8, 2, 64, 32, 256
    ctx = context(H, K, d, F16, F32, cap, 32)
    runs = []
    for seed, lens in ((1, [31, 100]), (2, [200, 1])):
        g = torch.Generator().manual_seed(seed)
        full = Cache([cap, cap], K, d, F16, B, seed)
        full.lens = list(lens)
        full.d_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        rnd = lambda *s: torch.randn(*s, generator=g).half().cuda()  # noqa: E731
        r = dict(cache=full, q=rnd(2, H, d), kn=rnd(2, K, d), vn=rnd(2, K, d), out=torch.zeros(2, H, d, device="cuda"),
                 acc=torch.zeros(2, K, cap, device="cuda"), ws=workspace(ctx.decode_bytes(2, cap, True)), gen=g,
                 stream=torch.cuda.Stream())
        r["graph"] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(r["graph"]):
            ctx.check(ctx.decode_layer(0, full.batch, r["q"], full.k, full.v, r["out"], r["ws"], k_new=r["kn"],
                                       v_new=r["vn"], acc=r["acc"]))
        r["acc"].zero_()
        r["want"] = torch.zeros(2, K, cap, dtype=torch.float64, device="cuda")
        r["lim"] = torch.zeros_like(r["want"])
        runs.append(r)
    for step in range(5):
        for r in runs:
            for name in ("q", "kn", "vn"):
                r[name].copy_(torch.randn(r[name].shape, generator=r["gen"]).half())
        torch.cuda.synchronize()
        for r in runs:
            with torch.cuda.stream(r["stream"]):
                r["graph"].replay()
        torch.cuda.synchronize()
        ctx.check(ctx.sync_status())
        for r in runs:
            ref, tol, add, add_tol = decode64(r["cache"], r["q"], k_new=r["kn"], v_new=r["vn"])
            assert ((r["out"].double() - ref).abs() <= tol + rounding(ref, F32)).all()
            r["want"] += add
            r["lim"] += add_tol + r["want"] * 2.0 ** -24
            assert ((r["acc"].double() - r["want"]).abs() <= r["lim"]).all()
            r["cache"].lens = [n + 7 for n in r["cache"].lens]
            r["cache"].d_lens.add_(7)
    fresh = epsp.Context(n_layer=1, n_head=H, n_head_kv=K, head_dim=d, dtype=F16, out_dtype=F32, max_ctx=cap,
                         page_size=32)
    r = runs[0]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        torch.zeros(1, device="cuda")
        rc = fresh.decode_layer(0, r["cache"].batch, r["q"], r["cache"].k, r["cache"].v, r["out"], r["ws"])
    assert rc == epsp.INVALID_ARGUMENT and "captured" in fresh.last_error()


def test_profile_counts_the_family():
    H, K, d = 8, 2, 64
    cache = Cache([100], K, d, F16, 32, 1)
    ctx = context(H, K, d, F16, F16, 256, 32)
    q, out = (torch.zeros(1, H, d, dtype=torch.float16, device="cuda") for _ in range(2))
    ws = workspace(ctx.decode_bytes(1, 100, False))
    epsp.lib.ep_sp_profile_enable(ctx.h, 1)
    for _ in range(3):
        ctx.check(ctx.decode_layer(0, cache.batch, q, cache.k, cache.v, out, ws))
    ms, n = ctx.profile_families()["k6_decode"]
    assert n == 3 and ms > 0
