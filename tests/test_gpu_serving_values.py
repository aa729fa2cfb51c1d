"""The cache-serving calls on values that are no ordinary numbers, and on weights and sizes far apart: infinities in the
rows of a cache, rows whose weight is nothing, one row that outweighs all others, millions of rows kept."""
import pytest
import torch

import epsp
from serving_util import Cache, TORCH, context, decode64, prompt64, rounding, score_error, workspace

pytestmark = pytest.mark.gpu

F32, F16, BF16 = epsp.F32, epsp.F16, epsp.BF16


def with_dead_keys(kv_len, n_tok, row_begin, heads, dtype, page, block, seed):
    """Sums over a cache in which some rows hold an infinity that makes all of their scores -inf (elements of q of one
    sign meet an infinity of the other), their 64-bit reference, its tolerance, and the dead rows."""
    H, K, d = heads
    g = torch.Generator().manual_seed(seed)
    k = torch.randn(1, kv_len, K, d, generator=g)
    dead = torch.rand(kv_len, generator=g) < 0.1
    dead[0] = False  # every query sees a key that counts
    dead[kv_len // 2] = dead[-1] = True
    minus = torch.rand(kv_len, generator=g) < 0.5
    k[0, dead & minus, :, 5] = float("-inf")
    k[0, dead & ~minus, :, 9] = float("inf")
    cache = Cache([kv_len], K, d, dtype, block, seed, k=k.to(TORCH[dtype]))
    q = torch.randn(n_tok, H, d, generator=g)
    q[..., 5] = q[..., 5].abs() + 0.1
    q[..., 9] = -q[..., 9].abs() - 0.1
    q = q.to(TORCH[dtype]).cuda()
    ctx = context(H, K, d, dtype, dtype, kv_len, page)
    if block:
        ctx.check(ctx.set_paged_kv(block, cache.d_table[0], cache.d_table.shape[1], cache.rows))
    acc = torch.full((K, kv_len), 5.0, device="cuda")
    ws = workspace(ctx.prompt_weights_bytes(kv_len, n_tok, row_begin))
    ctx.check(ctx.prompt_weights(0, q, cache.k, kv_len, n_tok, row_begin, acc, ws))
    torch.cuda.synchronize()
    ctx.check(ctx.sync_status())
    # the same with the dead rows taken out of each query's softmax
    dead = dead.cuda()
    alive = cache.seq(0)[0].clone()
    alive[dead] = 0
    ref, tol = torch.zeros((K, kv_len), dtype=torch.float64, device="cuda"), 0.0
    late = torch.arange(kv_len, device="cuda")[None, :] > torch.arange(kv_len - n_tok + row_begin, kv_len, device="cuda")[:, None]
    for hq in range(H):
        a, b = q[row_begin:, hq].double(), alive[:, hq // (H // K)].double()
        x = (a @ b.T / d ** 0.5).masked_fill(late | dead, float("-inf"))
        ref[hq // (H // K)] += torch.softmax(x, -1).sum(0)
        tol = max(tol, 2 * score_error(a.abs() @ b.abs().T / d ** 0.5, d))
    return acc, ref, ref * (tol + (n_tok - row_begin) * (H // K) * 2.0 ** -24), dead


# windows that fill their last query tile and that do not, groups that divide it and that do not, query tiles that stay
# on chip, are split into parts and stream; in f32, scores that are kept and that are computed twice
DEAD_KEYS = [(500, 64, 0, (14, 2, 64)), (300, 36, 0, (7, 1, 128)), (1000, 37, 5, (8, 1, 64)), (129, 1, 0, (4, 4, 128)),
             (700, 32, 0, (32, 8, 128)), (260, 30, 0, (65, 1, 64)), (5000, 600, 0, (14, 2, 64)),
             (4300, 900, 0, (8, 1, 128)), (2000, 2000, 0, (16, 1, 128)), (17200, 4100, 0, (100, 1, 128))]


@pytest.mark.parametrize("dtype", [F16, BF16, F32], ids=["f16", "bf16", "f32"])
@pytest.mark.parametrize("kv_len,n_tok,row_begin,heads", DEAD_KEYS, ids=str)
def test_prompt_weights_of_rows_of_infinities(kv_len, n_tok, row_begin, heads, dtype):
    """A cache row whose scores are all -inf has weight 0, whatever the columns that hold no query make of it."""
    if dtype == F32 and kv_len > 10000:
        kv_len, n_tok = 4500, 500
    for block in (0, 32):
        acc, ref, tol, dead = with_dead_keys(kv_len, n_tok, row_begin, heads, dtype, 32, block, kv_len + block)
        assert torch.isfinite(acc).all()
        assert (acc[:, dead].abs() <= 2.0 ** -100).all()
        over = (acc.double() - ref).abs() - tol - 2.0 ** -100
        assert (over <= 0).all(), float(over.max())


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("kv_len,n_tok,heads", [(65536, 36, (28, 4, 128)), (17200, 2050, (100, 1, 128))], ids=str)
def test_prompt_weights_of_a_query_that_is_none(kv_len, n_tok, heads, dtype):
    """A NaN query, or a NaN cache row, ends in NaN sums and in time: no wait runs out."""
    H, K, d = heads
    if dtype == F32:
        kv_len //= 8
    g = torch.Generator().manual_seed(1)
    cache = Cache([kv_len], K, d, dtype, 0, 2)
    ctx = context(H, K, d, dtype, dtype, kv_len, 32)
    ws = workspace(ctx.prompt_weights_bytes(kv_len, n_tok, 0))
    for what in ("query", "key"):
        q = torch.randn(n_tok, H, d, generator=g).to(TORCH[dtype]).cuda()
        k = cache.k.clone()
        if what == "query":
            q[-1, -1, 3] = float("nan")
        else:
            k[7, -1, 3] = float("nan")
        acc = torch.zeros(K, kv_len, device="cuda")
        ctx.check(ctx.prompt_weights(0, q, k, kv_len, n_tok, 0, acc, ws))
        ctx.check(ctx.sync_status())
        assert torch.isnan(acc[-1]).all() and torch.isfinite(acc[:-1]).all()


@pytest.mark.parametrize("dtype", [F16, BF16, F32], ids=["f16", "bf16", "f32"])
@pytest.mark.parametrize("kv_len,n_tok,row_begin,heads", DEAD_KEYS, ids=str)
def test_prompt_weights_of_nothing_are_zero(kv_len, n_tok, row_begin, heads, dtype):
    """A weight of nothing is 0 itself, so that an eviction ranks such rows by their place alone; so is one that
    underflows in every query (scores 200 and more below the others)."""
    if dtype == F32 and kv_len > 10000:
        kv_len, n_tok = 4500, 500
    acc, _, _, dead = with_dead_keys(kv_len, n_tok, row_begin, heads, dtype, 32, 0, kv_len)
    assert (acc[:, dead] == 0).all()
    H, K, d = heads
    q = torch.full((n_tok, H, d), 4.0).to(TORCH[dtype]).cuda()
    k = torch.zeros(kv_len, K, d, dtype=TORCH[dtype], device="cuda")
    k[dead] = -200.0 / (4 * d ** 0.5)
    ctx = context(H, K, d, dtype, dtype, kv_len, 32)
    ctx.check(ctx.prompt_weights(0, q, k, kv_len, n_tok, row_begin, acc,
                                 workspace(ctx.prompt_weights_bytes(kv_len, n_tok, row_begin))))
    torch.cuda.synchronize()
    ctx.check(ctx.sync_status())
    assert (acc[:, dead] == 0).all()


TYPES = [(F16, F16), (F16, F32), (BF16, BF16), (BF16, F32), (F32, F32)]
TYPE_IDS = ["f16", "f16_f32", "bf16", "bf16_f32", "f32"]


def decode_once(cache, q, dtype, out_dtype, page=32):
    n_seq, H, d = q.shape
    K = cache.k.shape[1]
    ctx = context(H, K, d, dtype, out_dtype, cache.cap, page)
    out = torch.full((n_seq, H, d), 7.0, dtype=TORCH[out_dtype], device="cuda")
    acc = torch.zeros(n_seq, K, cache.cap, device="cuda")
    ctx.check(ctx.decode_layer(0, cache.batch, q, cache.k, cache.v, out,
                               workspace(ctx.decode_bytes(n_seq, cache.cap, True)), acc=acc))
    plain = torch.full_like(out, 7.0)  # without weights the rows may be split over CTAs in another way
    ctx.check(ctx.decode_layer(0, cache.batch, q, cache.k, cache.v, plain,
                               workspace(ctx.decode_bytes(n_seq, cache.cap, False))))
    torch.cuda.synchronize()
    ctx.check(ctx.sync_status())
    return out, plain, acc


@pytest.mark.parametrize("dtype,out_dtype", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("heads", [(4, 2, 64), (20, 1, 128)], ids=str)
@pytest.mark.parametrize("n", [200, 1000, 5000])
def test_decode_of_one_row_that_outweighs_all(n, heads, dtype, out_dtype):
    """One row's weight is e^10 to e^18 times each other's and its V row is zero, so that the output comes from the light
    rows alone: their weights have to keep their bits."""
    H, K, d = heads
    g = torch.Generator().manual_seed(n)
    for gap in (10.0, 14.0, 16.0, 17.5, 18.0):
        for at in (5, n // 2, n - 1):
            for spread in (0.0, 0.3):
                k = torch.randn(1, n, K, d, generator=g) * spread
                k[..., 0] = 0
                k[0, at] = 0
                k[0, at, :, 0] = gap * d ** 0.5 / 8
                v = torch.ones(1, n, K, d) if spread == 0 else torch.rand(1, n, K, d, generator=g)
                v[0, at] = 0
                q = torch.randn(1, H, d, generator=g)
                q[..., 0] = 8
                cache = Cache([n], K, d, dtype, 32, 1, k=k.to(TORCH[dtype]), v=v.to(TORCH[dtype]))
                q = q.to(TORCH[dtype]).cuda()
                outs = decode_once(cache, q, dtype, out_dtype)
                ref, tol, add, add_tol = decode64(cache, q)
                if spread == 0:
                    # every score is one exact product, and its scaling in log2 units off by half a step of a value under
                    # 32, 2^-20, once above and once below: 2^-18 of the ratio with the exponentials' own; 2^-16 for the
                    # weights' parts; and 200 additions in f32 of a warp's, its CTA's and the joined sums
                    tol = ref.abs() * (2.0 ** -18 + 2.0 ** -16 + 200 * 2.0 ** -24)
                for out in outs[:2]:
                    over = (out.double() - ref).abs() - tol - rounding(ref, out_dtype)
                    assert (over <= 0).all(), (gap, at, spread, float(((out.double() - ref) / ref).abs().max()))
                assert ((outs[2].double() - add).abs() <= add_tol).all()


@pytest.mark.parametrize("dtype,out_dtype", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("heads", [(14, 2, 64), (20, 1, 128)], ids=str)
@pytest.mark.parametrize("n", [1, 33, 200, 1000, 5000])
def test_decode_of_infinite_values(n, heads, dtype, out_dtype):
    """An infinite element of V makes its column of the output infinite, infinities of both signs or a NaN make it NaN,
    and the other columns are as they were."""
    H, K, d = heads
    g = torch.Generator().manual_seed(n)
    inf = float("inf")
    for rows in ([0], [n // 2, n - 1], sorted({0, n // 3, n - 1})):
        k, v = torch.randn(1, n, K, d, generator=g), torch.randn(1, n, K, d, generator=g)
        for i, r in enumerate(rows):
            v[0, r, :, 3] = inf
            v[0, r, :, 7 + 2 * i] = -inf
            v[0, r, :, d - 1] = inf if i % 2 else -inf
        v[0, rows[-1], 0, 20] = float("nan")
        cache = Cache([n], K, d, dtype, 32, 1, k=k.to(TORCH[dtype]), v=v.to(TORCH[dtype]))
        q = torch.randn(1, H, d, generator=g).to(TORCH[dtype]).cuda()
        outs = decode_once(cache, q, dtype, out_dtype)
        vals = cache.seq(0)[1].float()
        up, down, nan = (x.any(0).repeat_interleave(H // K, 0)[None] for x in (vals == inf, vals == -inf, vals.isnan()))
        cache.v = torch.where(torch.isfinite(cache.v), cache.v, torch.zeros_like(cache.v))
        ref, tol, add, add_tol = decode64(cache, q)
        ref[up], ref[down] = inf, -inf
        ref[nan | (up & down)] = float("nan")
        plain = torch.isfinite(ref)
        for out in outs[:2]:
            assert torch.equal(torch.isnan(out), torch.isnan(ref))
            assert torch.equal(torch.isinf(out), torch.isinf(ref)) and torch.equal(out[torch.isinf(ref)] > 0, ref[torch.isinf(ref)] > 0)
            over = (out.double() - ref).abs() - tol - rounding(ref, out_dtype)
            assert (over[plain] <= 0).all(), float(over[plain].max())
        assert ((outs[2].double() - add).abs() <= add_tol).all()


def test_eviction_that_keeps_millions_of_rows():
    """More chunks of rows than a grid's y and z can count: 2,100,000 rows of 512 bytes are gathered."""
    K, d, n, keep = 1, 128, 2_200_003, 2_100_001
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randn(n, K, d, generator=g, device="cuda") for _ in range(2))
    acc = torch.randint(0, 1 << 20, (1, K, n), generator=g, device="cuda").float()
    kd, vd = (torch.full((keep + 5, K, d), 3.0, device="cuda") for _ in range(2))
    ctx = context(2, K, d, F32, F32, n, 128)
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    new, kept = torch.zeros_like(lens), torch.zeros(1, K, keep, dtype=torch.int32, device="cuda")
    src, dst = epsp.KvBatch(lens, n, seq_rows=n), epsp.KvBatch(None, keep, seq_rows=keep, n_seq=1)
    rc = ctx.evict_layer(0, src, k, v, acc, keep, 4, 1000, dst, kd, vd, workspace(ctx.evict_bytes(1, n, keep)),
                         new_lens=new, kept_rows=kept)
    assert rc == epsp.OK, ctx.last_error()
    torch.cuda.synchronize()
    ctx.check(ctx.sync_status())
    rank = acc[0, 0].clone()
    rank[:4] = rank[n - 1000:] = float("inf")
    rows = torch.sort(torch.sort(rank, descending=True, stable=True)[1][:keep])[0]
    assert int(new) == keep and torch.equal(kept[0, 0].long(), rows)
    assert torch.equal(kd[:keep], k[rows]) and torch.equal(vd[:keep], v[rows])
    assert (kd[keep:] == 3).all() and (vd[keep:] == 3).all()


@pytest.mark.parametrize("kv_len,window,heads", [(4096, 17, (1, 1, 64)), (3000, 1, (3, 1, 128)), (2048, 2048, (2, 2, 64))],
                         ids=str)
def test_prompt_weights_keep_only_scores_that_are_read(kv_len, window, heads):
    """f32: scores wait in the cache between the passes at its highest priority, so only those of rows that see a key of
    their 64 are written."""
    H, K, d = heads
    cache = Cache([kv_len], K, d, F32, 0, 1)
    q = torch.randn(window, H, d, generator=torch.Generator().manual_seed(2)).cuda()
    ctx = context(H, K, d, F32, F32, kv_len, 32)
    acc = torch.zeros(K, kv_len, device="cuda")
    ws = workspace(ctx.prompt_weights_bytes(kv_len, window, 0))
    ctx.check(ctx.prompt_weights(0, q, cache.k, kv_len, window, 0, acc, ws))
    torch.cuda.synchronize()
    written = int((ws[:ws.numel() // 4 * 4].view(torch.int32) != -0x54545455).sum())  # 0xABABABAB: as it was
    sees = torch.arange(kv_len - window, kv_len) // 64 + 1  # tiles of 64 keys that each query row sees
    tiles = -(-window * (H // K) // 64) * -(-kv_len // 64) * K  # a maximum and a sum of 64 rows each, at most
    assert written <= int(sees.sum()) * 64 * H + tiles * 64 * 2
    ref, tol = prompt64(q, cache.k, kv_len, window, 0)
    assert ((acc.double() - ref).abs() <= tol).all()
