"""A resize that finds too few free blocks, and the calls behind it on the stream: none of them writes a row through block
tables until the status is read, so that whatever sequences hold stays whole."""
import pytest
import torch

import epsp
from cache8_util import Cache8, decode64, write64
from serving_util import Cache, context, rounding, workspace

pytestmark = pytest.mark.gpu


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def same(a, b):
    return all(torch.equal(x.nan_to_num(nan=-7.0), y.nan_to_num(nan=-7.0)) for x, y in zip(a, b))


def book_of(c, pools, lens, free):
    """Pages over the sequences of `c` as they are, with all but `free` of the blocks that nobody holds taken away."""
    B, blocks = c.B, c.rows // c.B
    refs = torch.zeros(blocks, dtype=torch.int32, device="cuda")
    for i, n in enumerate(lens):
        refs[c.table[i, :-(-n // B)].long().cuda()] += 1
    none = (refs == 0).nonzero()[:, 0]
    refs[none[free:]] = 1  # (held by somebody else)
    return epsp.Pages(c.d_lens, c.d_table, refs, B), epsp.Pools(pools, blocks)


@pytest.mark.parametrize("heads", [(8, 2, 64), (65, 1, 64)], ids=str)  # new rows inside the call, and by a kernel before
@pytest.mark.parametrize("q8", [epsp.E4M3, epsp.I8], ids=["e4m3", "i8"])
def test_captured_steps_over_an_exhausted_pool(q8, heads):
    H, K, d = heads
    page, n = 32, 70
    c = Cache8([n, 0, 0], K, d, q8, page, page, 1, capacity=96)
    ctx = context(H, K, d, epsp.BF16, epsp.F32, 96, page)
    pages, pools = book_of(c, [c.k8, c.v8, c.ks, c.vs], c.lens, 1)
    ws = workspace(max(ctx.fork_bytes(pages), ctx.resize_bytes(pages), ctx.decode8_bytes(3, 96)))
    ctx.check(ctx.fork_seqs(pages, ints([0, 0, 0]), ws))  # three answers share the last, begun block
    lens = ints([n + 1] * 3)
    g = torch.Generator().manual_seed(3)
    q, kn, vn = (torch.randn(3, h, d, generator=g).bfloat16().cuda() * 4 for h in (H, K, K))
    out = torch.zeros(3, H, d, device="cuda")
    s, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=s):
        ctx.check(ctx.resize_seqs(pages, lens, pools, ws, stream=s))
        ctx.check(ctx.decode8_layer(0, c.batch, q, c.kv8, out, ws, k_new=kn, v_new=vn, stream=s))
    everything = lambda: c.state() + [c.d_lens.clone(), c.d_table.clone(), pages.refs.clone()]  # noqa: E731
    was = everything()
    for _ in range(3):  # two copies are needed, one block is free
        graph.replay()
    torch.cuda.synchronize()
    assert same(everything(), was)
    assert ctx.sync_status() == epsp.OUT_OF_MEMORY and "needed 1 more" in ctx.last_error()
    assert same(everything(), was) and ctx.sync_status() == epsp.OK
    # one answer gives its blocks back: the step is made again
    ctx.check(ctx.fork_seqs(pages, ints([0, 1, -1]), ws))
    lens.copy_(ints([n + 1, n + 1, 0]))
    torch.cuda.synchronize()
    graph.replay()
    ctx.check(ctx.sync_status())
    c.lens, c.table = c.d_lens.tolist(), c.d_table.cpu()
    assert c.lens == [n + 1, n + 1, 0] and c.table[0, 2] != c.table[1, 2]
    after, want = c.state(), [x.clone() for x in was[:4]]
    for a, b in zip(want, after):  # the copied block
        to, frm = int(c.table[0, 2]), int(was[5][0, 2])
        each = page if a.dim() == 3 else 1
        a[to * each:(to + 1) * each] = a[frm * each:(frm + 1) * each]
    for i in range(2):
        for t, x in enumerate((kn, vn)):
            write64(c, want, i, x[i].expand(n + 1, K, d), n, t)
    for i in range(2):
        at = c.at(i, n + 1).cuda()
        for t in range(2):
            assert torch.equal(after[t][at], want[t][at]) and torch.equal(after[2 + t][at // page], want[2 + t][at // page])
    ref, tol = decode64(c, q)
    assert bool(((out.double() - ref).abs() <= tol + rounding(ref, epsp.F32)).all())


@pytest.mark.parametrize("dtype", [epsp.BF16, epsp.F32], ids=["bf16", "f32"])
def test_every_call_that_writes_rows_is_held_back(dtype):
    """After a refused resize, then after its report; sequences without block tables are not held back."""
    H, K, d, page, n = 8, 2, 64, 32, 60
    ctx = context(H, K, d, dtype, dtype, 96, page)
    mk = lambda seed, B=page: Cache([n, 40], K, d, dtype, B, seed, capacity=96)  # noqa: E731
    src, c, flat, new = mk(1, 0), mk(2), mk(3, 0), mk(4)
    c8 = Cache8([n, 40], K, d, epsp.E4M3, page, page, 5, capacity=96)
    q = torch.randn(2, H, d, generator=torch.Generator().manual_seed(1)).to(c.k.dtype).cuda()
    kn, vn = q[:, :K].contiguous(), q[:, K:2 * K].contiguous()
    pages, pools = book_of(c, [c.k, c.v], c.lens, 0)
    ws = workspace(max(ctx.resize_bytes(pages), ctx.decode_bytes(2, 96, False), ctx.evict_bytes(2, 96, 20)))
    out, acc, new_lens = torch.zeros_like(q), torch.rand(2, K, 96, device="cuda"), ints([5, 6])

    def writes():
        """(call, what it writes)"""
        yield lambda: ctx.decode_layer(0, c.batch, q, c.k, c.v, out, ws, k_new=kn, v_new=vn), [c.k, c.v]
        yield lambda: ctx.pack_kv(0, src.batch, src.k, src.v, c8.batch, c8.kv8), [c8.k8.view(torch.uint8), c8.ks]
        yield lambda: ctx.unpack_kv(0, c8.batch, c8.kv8, new.batch, new.k, new.v), [new.k, new.v]
        yield (lambda: ctx.evict_layer(0, src.batch, src.k, src.v, acc, 20, 2, 4, new.batch, new.k, new.v, ws,
                                       acc_dst=acc, new_lens=new_lens), [new.k, new.v, new_lens, acc])
        yield lambda: append(), [c.k, c.v]

    def append():
        ctx.check(ctx.set_paged_kv(page, c.d_table[0].contiguous(), 3, c.rows))
        rc = ctx.append_kv(0, src.k[:n].contiguous(), src.v[:n].contiguous(), n, c.k, c.v, 0)
        ctx.check(ctx.set_paged_kv(0))
        return rc

    for refused in (True, False):
        if refused:
            ctx.check(ctx.resize_seqs(pages, ints([n + 10, 40]), pools, ws))
        for i, (call, what) in enumerate(writes()):
            was = [x.clone() for x in what]
            ctx.check(call())
            torch.cuda.synchronize()
            assert all(same([x], [y]) == refused for x, y in zip(what, was)), i
        if refused:  # rows that need no tables
            was = flat.k.clone()
            ctx.check(ctx.decode_layer(0, flat.batch, q, flat.k, flat.v, out, ws, k_new=kn, v_new=vn))
            torch.cuda.synchronize()
            assert not same([flat.k], [was])
        assert ctx.sync_status() == (epsp.OUT_OF_MEMORY if refused else epsp.OK)


def test_a_refusal_behind_another_failure_is_told_too():
    c = Cache([60, 40], 2, 64, epsp.F16, 32, 1, capacity=96)
    ctx = context(2, 2, 64, epsp.F16, epsp.F16, 96, 32)
    pages, pools = book_of(c, [c.k, c.v], c.lens, 0)
    ws = workspace(max(ctx.resize_bytes(pages), ctx.fork_bytes(pages)))
    ctx.check(ctx.fork_seqs(pages, ints([0, 7]), ws))
    ctx.check(ctx.resize_seqs(pages, ints([70, 40]), pools, ws))
    assert ctx.sync_status() == epsp.PREFILL and "refused" in ctx.last_error()
    assert ctx.sync_status() == epsp.OK


def test_a_refused_length_holds_the_step_back():
    """One sequence's new length is more than its table holds, and its last row one that another sequence holds too."""
    H, K, d, page, n = 8, 2, 64, 32, 96
    c = Cache8([n, 0, 40], K, d, epsp.E4M3, page, page, 1, capacity=96)
    ctx = context(H, K, d, epsp.BF16, epsp.F32, 96, page)
    pages, pools = book_of(c, [c.k8, c.v8, c.ks, c.vs], c.lens, 2)
    ws = workspace(max(ctx.fork_bytes(pages), ctx.resize_bytes(pages), ctx.decode8_bytes(3, 96)))
    ctx.check(ctx.fork_seqs(pages, ints([0, 0, 2]), ws))
    q = torch.randn(3, H, d, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    was, out = c.state(), torch.zeros(3, H, d, device="cuda")
    ctx.check(ctx.resize_seqs(pages, ints([n + 1, n, 41]), pools, ws))
    ctx.check(ctx.decode8_layer(0, c.batch, q, c.kv8, out, ws, k_new=q[:, :K].contiguous(), v_new=q[:, :K].contiguous()))
    torch.cuda.synchronize()
    assert same(c.state(), was) and c.d_lens.tolist() == [n, n, 41]
    assert ctx.sync_status() == epsp.PREFILL and "refused" in ctx.last_error()
    assert ctx.sync_status() == epsp.OK
