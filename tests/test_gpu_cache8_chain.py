"""The 8-bit cache and the calls on its blocks as they are used together: a gated prefill, its cache packed, answers to
the prompt that fork from it and grow row by row in shared blocks, a compaction, and a further gated prefill on what
was unpacked -- each step against the same on plain caches."""
import pytest
import torch

import epsp
import workloads as W
from cache8_util import Book, Cache8, decode64, write64
from serving_util import Cache, context, rounding, workspace

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,q8,heads,page", [(epsp.BF16, epsp.E4M3, (32, 8, 128), 128),
                                                 (epsp.F16, epsp.I8, (14, 2, 64), 64),
                                                 (epsp.F32, epsp.E4M3, (8, 2, 64), 32)], ids=str)
def test_prefill_pack_fork_decode_compact_unpack_prefill(dtype, q8, heads, page):
    H, K, d = heads
    n, beams, steps, B = 700, 3, 70, page
    w = W.Workload("chain8", n + 200, 1, H, K, d, dtype, 1024, page, 2, 2 * page)
    q, k, v = (t.cuda() for t in W.gen_layer(w, 0))
    ctx = context(H, K, d, dtype, epsp.F32, n + 200, page)
    ctx.check(ctx.set_ext(1, 0, 0))
    ctx.check(ctx.set_qg_bound(1, 2, 2, 0))
    ctx.set_prefill_mode(True)
    kc, vc = torch.zeros_like(k), torch.zeros_like(v)
    out = torch.zeros(n, H, d, device="cuda")
    ctx.check(ctx.append_kv(0, k[:n].contiguous(), v[:n].contiguous(), n, kc, vc, 0))
    ctx.check(ctx.attend_layer(0, q[:n].contiguous(), kc, vc, n, n, out))
    ctx.set_prefill_mode(False)
    # the prompt's blocks are taken and its cache packed into them
    each = -(-(n + steps) // B)
    c = Cache8([0] * beams, K, d, q8, page, B, 1, capacity=each * B, fill=False)
    blocks = c.rows // B
    refs = torch.zeros(blocks, dtype=torch.int32, device="cuda")
    pages = epsp.Pages(c.d_lens, c.d_table, refs, B)
    pools = epsp.Pools([c.k8, c.v8, c.ks, c.vs], blocks)
    book = Book([0] * beams, c.table.tolist(), [0] * blocks, B, range(blocks))
    ws = workspace(max(ctx.fork_bytes(pages), ctx.resize_bytes(pages), ctx.compact_bytes(pages),
                       ctx.decode8_bytes(beams, c.cap)))
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    ctx.check(ctx.resize_seqs(pages, ints([n, 0, 0]), pools, ws))
    book.resize([n, 0, 0])

    def follow():
        torch.cuda.synchronize()
        assert c.d_lens.tolist() == book.lens and refs.tolist() == book.refs and c.d_table.tolist() == book.tables
        c.lens, c.table = list(book.lens), torch.tensor(book.tables, dtype=torch.int32)

    follow()
    src = epsp.KvBatch(ints([n]), min(c.cap, n + 200), seq_rows=n + 200)
    one = epsp.KvBatch(None, c.cap, c.d_table[:1].contiguous(), B, c.rows, n_seq=1)
    want = c.state()
    for t, x in enumerate((kc, vc)):
        write64(c, want, 0, x[:n], 0, t)
    ctx.check(ctx.pack_kv(0, src, kc, vc, one, c.kv8))
    ctx.check(ctx.sync_status())
    assert all(torch.equal(a.nan_to_num(), b.nan_to_num()) for a, b in zip(c.state(), want))
    # three answers go on from it, each writing its own rows
    ctx.check(ctx.fork_seqs(pages, ints([0, 0, 0]), ws))
    book.fork([0, 0, 0])
    rows = [[], [], []]  # what each answer has appended
    g = torch.Generator().manual_seed(5)
    for i in range(steps):
        if i == 30:  # the first answer is dropped for a copy of the last, cut back by a few rows
            ctx.check(ctx.fork_seqs(pages, ints([2, 1, 2]), ws, lens=ints([n + 25, n + 30, n + 30])))
            book.fork([2, 1, 2], [n + 25, n + 30, n + 30])
            rows[0] = rows[2][:25]
            follow()
        lens = [m + 1 for m in book.lens]
        ctx.check(ctx.resize_seqs(pages, ints(lens), pools, ws))
        assert book.resize(lens)
        follow()
        kn, vn = (torch.randn(beams, K, d, generator=g).to(k.dtype).cuda() for _ in "kv")
        qn = torch.randn(beams, H, d, generator=g).to(k.dtype).cuda()
        for s in range(beams):
            rows[s] = rows[s] + [(kn[s], vn[s])]
        want = c.state()
        for s, m in enumerate(c.lens):
            for t, x in enumerate((kn, vn)):
                write64(c, want, s, x[s].expand(m, K, d), m - 1, t)
        o = torch.zeros(beams, H, d, device="cuda")
        ctx.check(ctx.decode8_layer(0, c.batch, qn, c.kv8, o, ws, k_new=kn, v_new=vn))
        assert all(torch.equal(a.nan_to_num(), b.nan_to_num()) for a, b in zip(c.state(), want)), i
        r, tol = decode64(c, qn)
        assert ((o.double() - r).abs() <= tol + rounding(r, epsp.F32)).all(), i
        if i in (10, 50):
            before = [c.seq(s) for s in range(beams)]
            if i == 50:
                ctx.check(ctx.resize_seqs(pages, ints([book.lens[0], 0, book.lens[2]]), pools, ws))
                book.resize([book.lens[0], 0, book.lens[2]])
            ctx.check(ctx.compact_pool(pages, pools, ws))
            used = book.compact()
            follow()
            assert all(b < used for s, m in enumerate(book.lens) for b in book.tables[s][:-(-m // B)])
            for s in range(beams):
                if book.lens[s]:
                    assert all(torch.equal(x, y) for x, y in zip(c.seq(s), before[s]))
            if i == 50:  # the freed one starts over from the first answer
                ctx.check(ctx.fork_seqs(pages, ints([0, 0, 2]), ws))
                book.fork([0, 0, 2])
                rows[1] = rows[0]
                follow()
    # an error of half a step per value, at most one more where scales grew: each answer holds what it was given
    ctx.check(ctx.sync_status())
    part = 2.0 ** -4 if q8 == epsp.E4M3 else 0.0
    for s in range(beams):
        for t, got in enumerate(c.seq(s)):
            given = torch.cat([(kc, vc)[t][:n], torch.stack([x[t] for x in rows[s]])]).double()
            at = c.at(s, c.lens[s]).cuda()
            step = (c.ks, c.vs)[t][at // page][..., None].double() * (1.0 if q8 == epsp.I8 else 2.0 ** -9)
            assert ((got - given).abs() <= 2 * (given.abs() * part * 1.07 + step)).all()
    # a further gated prefill chunk on the second answer, unpacked: the same as on a fresh context over the same rows
    m, t = book.lens[1], 60
    back = Cache([m] , K, d, dtype, 0, 1, capacity=n + 200)
    lens1, table1 = ints([m]), c.d_table[1:2].contiguous()
    cap = min(c.cap, n + 200)
    ctx.check(ctx.unpack_kv(0, epsp.KvBatch(lens1, cap, table1, B, c.rows), c.kv8,
                            epsp.KvBatch(None, cap, seq_rows=n + 200, n_seq=1), back.k, back.v))
    pk, pv = (x.to(k.dtype) for x in c.seq(1))
    assert torch.equal(back.k[:m], pk) and torch.equal(back.v[:m], pv)
    qn, kn, vn = (x[n:n + t].contiguous() for x in (q, k, v))
    outs = []
    for x, kk, vv in ((ctx, back.k, back.v), (context(H, K, d, dtype, epsp.F32, n + 200, page),
                                              torch.cat([pk, kn]).contiguous(), torch.cat([pv, vn]).contiguous())):
        x.check(x.set_ext(1, 0, 0))
        x.check(x.set_qg_bound(1, 1, 1, 0))
        x.set_prefill_mode(True)
        if x is ctx:
            x.check(x.append_kv(0, kn, vn, t, kk, vv, m))
        o = torch.zeros(t, H, d, device="cuda")
        sel = torch.full((1, K, 64), -1, dtype=torch.int32, device="cuda")
        cnt = torch.zeros((1, K), dtype=torch.int32, device="cuda")
        x.check(x.attend_layer(0, qn, kk, vv, m + t, t, o, sel, cnt, 64))
        torch.cuda.synchronize()
        x.check(x.sync_status())
        outs.append((o, sel, cnt))
    assert all(torch.equal(a, b) for a, b in zip(*outs))
