"""ep_sp_prompt_weights against a 64-bit causal softmax: types, head layouts, windows of one row to a whole ubatch,
paged caches with NaN past the prompt, adding to and overwriting the sums."""
import pytest
import torch

import epsp
from serving_util import Cache, TORCH, context, prompt64, workspace

pytestmark = pytest.mark.gpu

F32, F16, BF16 = epsp.F32, epsp.F16, epsp.BF16


def run_case(kv_len, n_tok, row_begin, heads, dtype, page, block, accumulate=False, pad=0, seed=0):
    H, K, d = heads
    cache = Cache([kv_len], K, d, dtype, block, seed)
    g = torch.Generator().manual_seed(seed + 7)
    q = torch.randn(n_tok, H, d, generator=g).to(TORCH[dtype]).cuda()
    if row_begin:
        q[:row_begin] = float("nan")  # rows before the window are not read
    ctx = context(H, K, d, dtype, dtype, kv_len, page)
    if block:
        ctx.check(ctx.set_paged_kv(block, cache.d_table[0], cache.d_table.shape[1], cache.rows))
    acc = torch.rand(K, kv_len + pad, generator=g).cuda()
    acc0 = acc.clone()
    ws = workspace(ctx.prompt_weights_bytes(kv_len, n_tok, row_begin))
    ctx.check(ctx.prompt_weights(0, q, cache.k, kv_len, n_tok, row_begin, acc, ws, accumulate=accumulate))
    torch.cuda.synchronize()
    ctx.check(ctx.sync_status())
    ref, tol = prompt64(q, cache.seq(0)[0], kv_len, n_tok, row_begin)
    if accumulate:
        ref = ref + acc0[:, :kv_len].double()
        tol = tol + ref.abs() * 2.0 ** -24
    over = (acc[:, :kv_len].double() - ref).abs() - tol
    assert (over <= 0).all(), float(over.max())
    assert torch.equal(acc[:, kv_len:], acc0[:, kv_len:])
    total = (acc[:, :kv_len].double().sum() - (acc0[:, :kv_len].double().sum() if accumulate else 0)).item()
    assert abs(total / ((n_tok - row_begin) * H) - 1) < 1e-4  # every row's weights sum to 1
    return acc


@pytest.mark.parametrize("dtype,heads,page,block", [
    (BF16, (32, 8, 128), 128, 128), (BF16, (28, 4, 128), 64, 64), (F16, (14, 2, 64), 64, 0), (F16, (8, 8, 64), 32, 32),
    (F32, (14, 2, 64), 64, 64), (F32, (9, 3, 128), 32, 96), (BF16, (16, 1, 128), 32, 0)], ids=str)
@pytest.mark.parametrize("kv_len,n_tok,row_begin", [
    (1, 1, 0), (2, 1, 0), (33, 33, 0), (128, 5, 4), (129, 129, 100), (500, 64, 0), (777, 300, 269), (1500, 1, 0),
    (2100, 513, 449)], ids=str)
def test_windows(kv_len, n_tok, row_begin, dtype, heads, page, block):
    run_case(kv_len, n_tok, row_begin, heads, dtype, page, block, seed=kv_len)


@pytest.mark.parametrize("heads", [(1, 1, 64), (3, 1, 128), (24, 2, 64), (33, 1, 64), (65, 1, 128), (128, 1, 64),
                                   (100, 1, 128)], ids=str)
@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_query_heads_per_kv_head(heads, dtype):
    run_case(300, 40, 0, heads, dtype, 32, 32, accumulate=True, pad=9, seed=heads[0])


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_whole_prompt(dtype):
    run_case(1111, 1111, 0, (8, 2, 64), dtype, 32, 32, seed=1)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("kv_len,n_tok,row_begin,heads", [
    (257, 174, 100, (16, 1, 128)), (300, 290, 0, (48, 1, 64)), (130, 129, 0, (100, 1, 64)), (700, 700, 0, (64, 2, 128)),
    (1000, 600, 0, (7, 1, 64)), (2000, 2000, 0, (16, 1, 128)), (7680, 320, 0, (16, 1, 128))], ids=str)
def test_many_rows_over_few_keys(kv_len, n_tok, row_begin, heads, dtype):
    """The rows of the sums are split over the device, and their parts put together."""
    run_case(kv_len, n_tok, row_begin, heads, dtype, 32, 32, seed=kv_len)
    run_case(kv_len, n_tok, row_begin, heads, dtype, 32, 0, accumulate=True, pad=3, seed=kv_len + 1)


def test_more_rows_than_parts_are_kept_of():
    """So many rows and keys that the sums are not split over the rows: the query tiles stream past the keys."""
    run_case(8250, 8250, 0, (128, 1, 128), BF16, 64, 64, seed=4)
    run_case(19000, 1800, 0, (256, 2, 128), F16, 128, 0, accumulate=True, pad=5, seed=5)


@pytest.mark.parametrize("kv_len,n_tok,row_begin,heads", [
    (5000, 600, 0, (14, 2, 64)), (3000, 3000, 17, (7, 1, 64)), (4300, 900, 0, (8, 1, 128)), (9000, 260, 3, (32, 8, 128))],
    ids=str)
def test_rows_split_over_parts(kv_len, n_tok, row_begin, heads):
    """More query tiles than stay on chip: parts of the rows, of which the early ones do not see the last keys."""
    run_case(kv_len, n_tok, row_begin, heads, BF16, 64, 64, seed=kv_len)
    run_case(kv_len, n_tok, row_begin, heads, F16, 32, 0, accumulate=True, pad=3, seed=kv_len + 1)


def test_long_cache():
    run_case(30000, 64, 0, (32, 8, 128), BF16, 128, 128, accumulate=True, seed=2)
    run_case(20011, 700, 500, (28, 4, 128), F16, 64, 64, seed=3)


def test_windows_add_up():
    """Two halves of a window, the second added to the first, give the whole window's sums."""
    H, K, d, n, t = 8, 2, 64, 900, 200
    cache = Cache([n], K, d, BF16, 0, 3)
    q = torch.randn(t, H, d, generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
    ctx = context(H, K, d, BF16, BF16, n, 32)
    acc = torch.full((K, n), 5.0, device="cuda")
    ws = workspace(ctx.prompt_weights_bytes(n, t, 0))
    ctx.check(ctx.prompt_weights(0, q, cache.k, n, t, 110, acc, ws))
    first = q[:110].contiguous()
    ctx.check(ctx.prompt_weights(0, first, cache.k, n - 90, 110, 0, acc, ws, accumulate=True))
    ref, tol = prompt64(q, cache.k, n, t, 0)
    assert ((acc.double() - ref).abs() <= tol + ref * 2.0 ** -23).all()


def test_same_result_every_time_captured_and_on_another_stream():
    H, K, d, n, t = 32, 8, 128, 3000, 96
    cache = Cache([n], K, d, BF16, 128, 3)
    q = torch.randn(t, H, d, generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
    ctx = context(H, K, d, BF16, BF16, n, 128)
    ctx.check(ctx.set_paged_kv(128, cache.d_table[0], cache.d_table.shape[1], cache.rows))
    ws = workspace(ctx.prompt_weights_bytes(n, t, 32))
    accs = [torch.zeros(K, n, device="cuda") for _ in range(3)]
    ctx.check(ctx.prompt_weights(0, q, cache.k, n, t, 32, accs[0], ws))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ctx.check(ctx.prompt_weights(0, q, cache.k, n, t, 32, accs[1], ws))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ctx.check(ctx.prompt_weights(0, q, cache.k, n, t, 32, accs[2], ws))
    graph.replay()
    torch.cuda.synchronize()
    ctx.check(ctx.sync_status())
    assert torch.equal(accs[0], accs[1]) and torch.equal(accs[0], accs[2])


def test_bad_table_entry_is_reported():
    H, K, d, n = 8, 2, 64, 200
    for dtype in (BF16, F32):
        cache = Cache([n], K, d, dtype, 32, 3)
        cache.d_table[0, 3] = -5
        ctx = context(H, K, d, dtype, dtype, n, 32)
        ctx.check(ctx.set_paged_kv(32, cache.d_table[0], cache.d_table.shape[1], cache.rows))
        q = torch.zeros(10, H, d, dtype=TORCH[dtype], device="cuda")
        acc = torch.zeros(K, n, device="cuda")
        ctx.check(ctx.prompt_weights(0, q, cache.k, n, 10, 0, acc, workspace(ctx.prompt_weights_bytes(n, 10, 0))))
        assert ctx.sync_status() == epsp.PREFILL
