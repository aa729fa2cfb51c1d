"""The cache in 8 bits against its definition in 64 bits: bytes and scales exactly (a power of two divides exactly, so
there is one rounding and one right answer), decode within the tolerances of its arithmetic."""
import math

import pytest
import torch

import epsp
from cache8_util import TOP, TORCH8, Cache8, bytes_of, decode64, round8, write64
from serving_util import TORCH, Cache, context, rounding, workspace

pytestmark = pytest.mark.gpu

E, Q = epsp.E4M3, epsp.I8
IDS = {epsp.F32: "f32", epsp.F16: "f16", epsp.BF16: "bf16", E: "e4m3", Q: "i8"}


def name(x):
    return IDS.get(x, str(x)) if isinstance(x, int) else str(x)


def same(a, b):
    return all(torch.equal(x.nan_to_num(nan=-7.0) if x.is_floating_point() else x,
                           y.nan_to_num(nan=-7.0) if y.is_floating_point() else y) for x, y in zip(a, b))


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------- pack, unpack
LENS = [0, 1, 31, 32, 33, 64, 127, 130, 200]


@pytest.mark.parametrize("first", [False, True], ids=["whole", "behind"])
@pytest.mark.parametrize("blocks", [(0, 0), (1, 2), (2, 0), (0, 1)], ids=str)
@pytest.mark.parametrize("heads,page", [((2, 64), 32), ((3, 128), 64), ((1, 128), 128), ((5, 64), 128)], ids=str)
@pytest.mark.parametrize("dtype", [epsp.BF16, epsp.F16, epsp.F32], ids=name)
@pytest.mark.parametrize("q8", [E, Q], ids=name)
def test_pack_and_unpack(q8, dtype, heads, page, blocks, first):
    K, d = heads
    src = Cache(LENS, K, d, dtype, blocks[0] * page, 1)
    dst = Cache8(LENS, K, d, q8, page, blocks[1] * page, 2, capacity=max(LENS))
    ctx = context(K, K, d, dtype, dtype, max(LENS), page)
    at = [min(n, x) for n, x in zip(LENS, [0, 0, 30, 32, 32, 1, 64, 65, 131])] if first else [0] * len(LENS)
    want = dst.state()
    for i, n in enumerate(LENS):
        for t, x in enumerate(src.seq(i)):
            write64(dst, want, i, x, at[i], t)
    f = ints(at) if first else None
    for _ in range(2):  # (the second time everything is there already)
        ctx.check(ctx.pack_kv(0, src.batch, src.k, src.v, dst.batch, dst.kv8, first=f))
        torch.cuda.synchronize()
        assert same(dst.state(), want)
    # and back, into another layout: rows outside [first, length) stay NaN
    out = Cache(LENS, K, d, dtype, blocks[1] * page, 3)
    out.k.fill_(float("nan")), out.v.fill_(float("nan"))
    refs = [out.k.clone(), out.v.clone()]
    for i, n in enumerate(LENS):
        rows = out.at(i, n)[at[i]:].cuda()
        for t, x in enumerate(dst.seq(i)):
            refs[t][rows] = x[at[i]:].to(TORCH[dtype])
    ctx.check(ctx.unpack_kv(0, dst.batch, dst.kv8, out.batch, out.k, out.v, first=f))
    ctx.check(ctx.sync_status())
    assert same([out.k, out.v], refs)


@pytest.mark.parametrize("q8", [E, Q], ids=name)
def test_every_code_is_read_and_written(q8):
    """All 256 bytes through unpack, and back through pack: the same bytes (the largest code fixes the scale)."""
    codes = torch.arange(256, dtype=torch.uint8)
    codes[(codes == 0x7F) | (codes == 0xFF)] = 0 if q8 == E else codes[1]  # e4m3's NaN
    if q8 == Q:
        codes = torch.arange(256, dtype=torch.uint8)
        codes[128] = 0  # -128 is never written
    b = codes.view(4, 1, 64).repeat(8, 1, 1).cuda()
    c = Cache8([32], 1, 64, q8, 32, 0, 1)
    c.k8.view(torch.uint8).copy_(b), c.v8.view(torch.uint8).copy_(b.flip(2))
    c.ks.fill_(2.0 ** -3), c.vs.fill_(2.0 ** 5)
    ctx = context(1, 1, 64, epsp.F32, epsp.F32, 32, 32)
    x = Cache([32], 1, 64, epsp.F32, 0, 1)
    ctx.check(ctx.unpack_kv(0, c.batch, c.kv8, x.batch, x.k, x.v))
    value = b.view(TORCH8[q8]).float() / 8
    assert torch.equal(x.k, value)
    out = Cache8([32], 1, 64, q8, 32, 0, 1, fill=False)
    ctx.check(ctx.pack_kv(0, x.batch, x.k, x.v, out.batch, out.kv8))
    ctx.check(ctx.sync_status())
    assert torch.equal(out.ks, c.ks) and torch.equal(out.vs, c.vs)
    zero = b & 0x7F if q8 == E else b  # (-0 keeps its sign or not)
    keep = zero != 0
    assert torch.equal(out.k8.view(torch.uint8)[keep], c.k8.view(torch.uint8)[keep])
    assert torch.equal(out.k8.float(), c.k8.float())


@pytest.mark.parametrize("q8", [E, Q], ids=name)
def test_e4m3_nan_codes_and_scales_that_are_no_power_of_two(q8):
    c = Cache8([40], 2, 64, q8, 32, 0, 3)
    c.ks.mul_(1.37), c.vs.mul_(0.77)
    if q8 == E:
        c.k8.view(torch.uint8)[3, 1, 5] = 0xFF
    x = Cache([40], 2, 64, epsp.F32, 0, 1)
    ctx = context(2, 2, 64, epsp.F32, epsp.F32, 64, 32)
    ctx.check(ctx.unpack_kv(0, c.batch, c.kv8, x.batch, x.k, x.v))
    at = c.at(0, 40).cuda()
    for got, b, s in ((x.k, c.k8, c.ks), (x.v, c.v8, c.vs)):
        want = b[at].float() * s[at // 32][..., None]
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(got.nan_to_num(), want.nan_to_num())
    assert torch.isnan(x.k[3, 1, 5]) if q8 == E else True


@pytest.mark.parametrize("dtype", [epsp.BF16, epsp.F16, epsp.F32], ids=name)
@pytest.mark.parametrize("q8", [E, Q], ids=name)
def test_magnitudes(q8, dtype):
    """Zeros, the smallest and the largest numbers of the type, pages whose scale grows by far, ties."""
    K, d, page = 2, 64, 32
    f = torch.finfo(TORCH[dtype])
    n = 6 * page
    src = Cache([n], K, d, dtype, 0, 1)
    x = torch.randn(n, K, d, dtype=torch.float64)
    x[:page] = 0
    x[page:2 * page] *= f.smallest_normal
    x[2 * page:3 * page] *= f.max / 8
    x[2 * page, 0, 0] = f.max
    x[3 * page:4 * page, :, :] = torch.arange(d) * 0.5 * (1 if q8 == Q else 2.0 ** -8)  # ties between bytes
    x[3 * page] = TOP[q8]
    x[4 * page:4 * page + 7] *= 2.0 ** -9
    x[4 * page + 7:5 * page] *= 2.0 ** 9
    x[5 * page, 1] = -f.max
    src.k.copy_(x.to(TORCH[dtype])), src.v.copy_(x.flip(2).to(TORCH[dtype]))
    dst = Cache8([n], K, d, q8, page, 0, 2, fill=False)
    ctx = context(K, K, d, dtype, dtype, n, page)
    want = dst.state()
    for lo, hi in ((0, 4 * page + 7), (4 * page + 7, n)):  # in two parts: the fifth page's scale grows
        for t, y in enumerate(src.seq(0)):
            write64(dst, want, 0, y[:hi], lo, t)
        src.d_lens.fill_(hi)
        ctx.check(ctx.pack_kv(0, src.batch, src.k, src.v, dst.batch, dst.kv8, first=ints([lo])))
        ctx.check(ctx.sync_status())
        assert same(dst.state(), want)
    assert float(dst.ks[0, 0]) == 2.0 ** -100


@pytest.mark.parametrize("q8", [E, Q], ids=name)
def test_what_is_not_finite_is_reported(q8):
    K, d, page = 2, 64, 32
    for how in ("pack", "append"):
        src = Cache([page], K, d, epsp.F32, 0, 1)
        src.k[5, 1, 3], src.v[7, 0, 2], src.v[7, 0, 9] = float("nan"), float("inf"), float("-inf")
        dst = Cache8([page], K, d, q8, page, 0, 2, fill=False)
        want = dst.state()
        ctx = context(K, K, d, epsp.F32, epsp.F32, page, page)
        if how == "pack":
            for t, y in enumerate(src.seq(0)):
                write64(dst, want, 0, y, 0, t)
            ctx.check(ctx.pack_kv(0, src.batch, src.k, src.v, dst.batch, dst.kv8))
        else:
            dst.d_lens.fill_(1)
            for t, y in enumerate((src.k[5:6], src.v[7:8])):
                write64(dst, want, 0, y, 0, t)
            out = torch.zeros(1, K, d, device="cuda")
            ctx.check(ctx.decode8_layer(0, dst.batch, torch.ones_like(out), dst.kv8, out,
                                        workspace(ctx.decode8_bytes(1, page)), k_new=src.k[5:6].contiguous(),
                                        v_new=src.v[7:8].contiguous()))
        assert ctx.sync_status() == epsp.UNSUPPORTED and "8-bit" in ctx.last_error()
        assert ctx.sync_status() == epsp.OK
        assert same(dst.state(), want)


def test_bad_lengths_tables_and_firsts_are_left_out():
    K, d, page = 2, 64, 32
    lens = [50, 60, 70, 40]
    src = Cache(lens, K, d, epsp.BF16, page, 1)
    dst = Cache8(lens, K, d, E, page, page, 2)
    ctx = context(K, K, d, epsp.BF16, epsp.BF16, 70, page)
    want = dst.state()
    for i in (0, 3):
        for t, y in enumerate(src.seq(i)):
            # sequence 3: the first page's table entry is none, so only its second page is written
            write64(dst, want, i, y, 32 if i == 3 else 0, t)
    src.d_lens[1] = 71
    dst.d_table[3, 0] = 10 ** 6
    f = ints([0, 0, 71, 0])
    ctx.check(ctx.pack_kv(0, src.batch, src.k, src.v, dst.batch, dst.kv8, first=f))
    assert ctx.sync_status() == epsp.PREFILL
    assert same(dst.state(), want)
    k, v = src.k.clone(), src.v.clone()
    src.d_lens[0], src.d_lens[3] = 0, -1
    ctx.check(ctx.unpack_kv(0, src.batch, dst.kv8, src.batch, src.k, src.v, first=f))
    assert ctx.sync_status() == epsp.PREFILL
    assert same([src.k, src.v], [k, v])


# ------------------------------------------------------------------- decode
def run(ctx, c, q, out_dtype=epsp.F32, ws=None, kn=None, vn=None, stream=None):
    out = torch.full(q.shape, float("nan"), dtype=TORCH[out_dtype], device="cuda")
    ws = workspace(ctx.decode8_bytes(len(c.lens), c.cap)) if ws is None else ws
    ctx.check(ctx.decode8_layer(0, c.batch, q, c.kv8, out, ws, k_new=kn, v_new=vn, stream=stream))
    return out


def held(out, c, q, out_dtype, scale=None):
    ref, tol = decode64(c, q, scale, out_dtype == epsp.BF16 and q.dtype != torch.float32)
    err = (out.double() - ref).abs()
    assert bool((err <= tol + rounding(ref, out_dtype)).all()), float((err - tol).max())


def randq(n, H, d, dtype, seed=5, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n, H, d, generator=g) * scale).to(TORCH[dtype]).cuda()


HEADS = [(14, 2, 64), (32, 8, 128), (28, 4, 128), (8, 8, 64), (9, 1, 128), (16, 1, 64), (17, 1, 128), (40, 1, 64),
         (128, 1, 128), (65, 1, 64)]


@pytest.mark.parametrize("q8", [E, Q], ids=name)
@pytest.mark.parametrize("dtype", [epsp.BF16, epsp.F16, epsp.F32], ids=name)
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("capacity", [1111, 13000])  # joined in clusters, and split over the device
def test_decode8_heads(capacity, heads, dtype, q8):
    """Every number of query heads per KV head that takes another path, ragged lengths, a row appended."""
    H, K, d = heads
    page = 64
    lens = [0, 1, 33, 64, 500, 1111]
    c = Cache8(lens, K, d, q8, page, page, 1, capacity=capacity)
    ctx = context(H, K, d, dtype, epsp.F32, capacity, page)
    q, kn, vn = randq(6, H, d, dtype), randq(6, K, d, dtype, 6, 3.0), randq(6, K, d, dtype, 7)
    want = c.state()
    for i, n in enumerate(lens):
        if n:
            for t, x in enumerate((kn, vn)):
                write64(c, want, i, x[i].expand(n, K, d), n - 1, t)
    out = run(ctx, c, q, kn=kn, vn=vn)
    ctx.check(ctx.sync_status())
    assert same(c.state(), want)
    held(out, c, q, epsp.F32)


@pytest.mark.parametrize("q8", [E, Q], ids=name)
@pytest.mark.parametrize("lens,blocks", [([1], 0), ([31], 1), ([32], 0), ([200], 0), ([1001], 1), ([3000], 2),
                                         ([40000], 1), ([7] * 300, 1), ([100, 0, 4000, 1, 2048] * 9, 1),
                                         ([5, 0, 40] * 400, 0), ([0, 0], 0), ([513] * 16, 0)],
                         ids=["1", "31", "32", "200", "1001", "3000", "40000", "300x7", "ragged", "1200 short", "none",
                              "16x513"])
@pytest.mark.parametrize("heads,page,dtype,out", [((8, 2, 128), 128, epsp.BF16, epsp.BF16),
                                                  ((14, 2, 64), 32, epsp.F16, epsp.F32),
                                                  ((6, 2, 64), 64, epsp.F32, epsp.F16)], ids=str)
def test_decode8_lengths(lens, blocks, heads, page, dtype, out, q8):
    H, K, d = heads
    c = Cache8(lens, K, d, q8, page, blocks * page, 1)
    ctx = context(H, K, d, dtype, out, max(1, max(lens)), page)
    q = randq(len(lens), H, d, dtype)
    o = run(ctx, c, q, out)
    o2 = run(ctx, c, q, out)
    ctx.check(ctx.sync_status())
    assert torch.equal(o, o2)
    held(o, c, q, out)


@pytest.mark.parametrize("q8", [E, Q], ids=name)
@pytest.mark.parametrize("dtype", [epsp.BF16, epsp.F32], ids=name)
def test_steps_of_decoding(dtype, q8):
    """Row after row into begun and new pages, with magnitudes that make scales grow."""
    H, K, d, page = 8, 2, 64, 32
    c = Cache8([0, 20, 63], K, d, q8, page, page, 1, capacity=200)
    ctx = context(H, K, d, dtype, epsp.F32, 200, page)
    ws = workspace(ctx.decode8_bytes(3, 200))
    for i in range(70):
        c.lens = [n + 1 for n in c.lens]
        c.d_lens += 1
        q = randq(3, H, d, dtype, i)
        kn, vn = (randq(3, K, d, dtype, s + i, 2.0 ** ((i * 7) % 11 - 5)) for s in (100, 200))
        want = c.state()
        for s, n in enumerate(c.lens):
            for t, x in enumerate((kn, vn)):
                write64(c, want, s, x[s].expand(n, K, d), n - 1, t)
        out = run(ctx, c, q, ws=ws, kn=kn, vn=vn)
        assert same(c.state(), want), i
        held(out, c, q, epsp.F32)
    ctx.check(ctx.sync_status())


@pytest.mark.parametrize("q8", [E, Q], ids=name)
@pytest.mark.parametrize("heads,page,dtype", [((8, 2, 128), 128, epsp.BF16), ((7, 1, 64), 32, epsp.F16),
                                              ((12, 4, 128), 64, epsp.F32), ((34, 2, 64), 128, epsp.BF16)], ids=str)
def test_new_rows_of_ragged_batches(heads, page, dtype, q8):
    """Batches that are split over the device anywhere but in the page that a new row goes into: lengths that end
    pages, begin them, lie in the first or fill several, and rows that make scales grow."""
    H, K, d = heads
    lens = [(i * 977) % 2300 for i in range(37)] + [page, page + 1, 1, 2299, 2 * page - 1]
    c = Cache8(lens, K, d, q8, page, page, 1)
    ctx = context(H, K, d, dtype, epsp.F32, max(lens), page)
    n = len(lens)
    q, kn, vn = randq(n, H, d, dtype), randq(n, K, d, dtype, 6), randq(n, K, d, dtype, 7)
    kn[::3] *= 8
    vn[1::3] *= 8
    want = c.state()
    for i, m in enumerate(lens):
        if m:
            for t, x in enumerate((kn, vn)):
                write64(c, want, i, x[i].expand(m, K, d), m - 1, t)
    out = run(ctx, c, q, kn=kn, vn=vn)
    ctx.check(ctx.sync_status())
    assert same(c.state(), want)
    held(out, c, q, epsp.F32)
    assert torch.equal(run(ctx, c, q, kn=kn, vn=vn), out)  # (the same rows again: the same bytes)


def test_captured_packs_and_unpacks():
    """Replayed as lengths and rows change; on another stream than the current one."""
    K, d, page = 2, 64, 32
    src = Cache([150, 90], K, d, epsp.F16, 0, 1)
    dst = Cache8([150, 90], K, d, E, page, page, 2, capacity=150)
    out = Cache([150, 90], K, d, epsp.F16, page, 3)
    ctx = context(K, K, d, epsp.F16, epsp.F16, 150, page)
    first, s, g = ints([0, 0]), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    batch8 = epsp.KvBatch(src.d_lens, 150, dst.d_table, page, dst.rows)
    was = dst.state()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
        ctx.check(ctx.pack_kv(0, src.batch, src.k, src.v, dst.batch, dst.kv8, first=first, stream=s))
        ctx.check(ctx.unpack_kv(0, batch8, dst.kv8, out.batch, out.k, out.v, first=first, stream=s))
    torch.cuda.synchronize()
    assert same(dst.state(), was)
    for lens, at in (([40, 90], [0, 0]), ([150, 64], [40, 3]), ([0, 1], [0, 1])):
        src.d_lens.copy_(ints(lens)), first.copy_(ints(at))
        want, refs = dst.state(), [out.k.clone(), out.v.clone()]
        for i, n in enumerate(lens):
            for t, x in enumerate((src.k, src.v)):
                write64(dst, want, i, x[i * 150:i * 150 + n], at[i], t)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert same(dst.state(), want)
        for i, n in enumerate(lens):
            dst.lens[i] = n
            for t, x in enumerate(dst.seq(i)):
                refs[t][out.at(i, n)[at[i]:].cuda()] = x[at[i]:].half()
        assert same([out.k, out.v], refs)
    ctx.check(ctx.sync_status())


@pytest.mark.parametrize("dtype", [epsp.BF16, epsp.F16, epsp.F32], ids=name)
def test_magnitudes_of_queries_scales_and_weights(dtype):
    """Scales of neighbouring pages far apart, a large and a tiny query, weights that underflow."""
    H, K, d, page = 4, 2, 64, 32
    c = Cache8([700, 90], K, d, E, page, 0, 1)
    p = torch.arange(c.ks.shape[0], device="cuda")
    c.ks[:] = torch.exp2(-8.0 - (p % 3) * 6.0)[:, None]
    c.vs[:] = torch.exp2((p * 5 % 23).float() - 18.0)[:, None] * 1.3
    ctx = context(H, K, d, dtype, epsp.F32, 700, page)
    big = {epsp.F16: 60.0}.get(dtype, 200.0)
    for s in (1.0, big, 2.0 ** -12):
        q = randq(2, H, d, dtype, 3, s)
        # (scores of hundreds: their error counts as such in the tolerance)
        held(run(ctx, c, q), c, q, epsp.F32)
    q = randq(2, H, d, dtype)
    q[0, 1] = 0
    q[1, 2] *= 2.0 ** -14
    held(run(ctx, c, q), c, q, epsp.F32)
    ctx.check(ctx.sync_status())


@pytest.mark.parametrize("dtype", [epsp.F16, epsp.F32], ids=name)
def test_pages_of_zeros_next_to_large_values(dtype):
    """A page of zeros has the smallest scale there is; its weights count all the same."""
    H, K, d, page = 4, 2, 64, 32
    c = Cache8([700, 90], K, d, E, page, 0, 1)
    p = torch.arange(c.ks.shape[0], device="cuda") % 3
    c.ks[:] = 2.0 ** -8
    c.vs[:] = torch.exp2(torch.tensor([-100.0, 40.0, -8.0], device="cuda")[p])[:, None]
    c.v8.view(torch.uint8).view(-1, page, K, d)[p == 0] = 0
    ctx = context(H, K, d, dtype, epsp.F32, 700, page)
    q = randq(2, H, d, dtype, 3)
    ref, tol = decode64(c, q)
    # scores carry log2 of V's scale, 64 and their own few at most: half a step of [64, 128) is 2^-18, times ln 2, in
    # numerator and denominator: under 2^-17 of the sum of magnitudes, 16 times what the tolerance has of them at least
    assert bool(((run(ctx, c, q).double() - ref).abs() <= 17 * tol).all())
    ctx.check(ctx.sync_status())


@pytest.mark.parametrize("q8", [E, Q], ids=name)
@pytest.mark.parametrize("dtype", [epsp.F16, epsp.F32], ids=name)
def test_tiny_values(dtype, q8):
    """V scales below 2^-64: what they are short of it goes into the weights when those are f16."""
    H, K, d, page = 4, 2, 128, 32
    lens = [700, 90]
    c = Cache8(lens, K, d, q8, page, 0, 1)
    p = torch.arange(c.vs.shape[0], device="cuda") % 3
    c.vs[:] = torch.exp2(torch.tensor([-70.0, -65.0, -71.0], device="cuda")[p])[:, None]
    ctx = context(H, K, d, dtype, epsp.F32, 700, page)
    q = randq(2, H, d, dtype, 3)
    ref, tol = decode64(c, q)
    # 17: as above.  The weights' absolute part, 2^-39 of the largest where that is 2^14, is 2^-39 of the largest weight
    # times 2^-64 here: in all at most rows * 2^-39 * 2^-64 * the largest byte
    floor = torch.tensor(lens, device="cuda").double().view(2, 1, 1) * 2.0 ** -103 * 448
    assert bool(((run(ctx, c, q).double() - ref).abs() <= 17 * tol + floor).all())
    ctx.check(ctx.sync_status())


def test_long_caches_of_zeros():
    """40,000 rows of zeros, all one block, before a page that is not: the sum of the weights stays finite."""
    page, d, n_seq, n = 32, 64, 160, 40000
    each = n // page
    table = torch.zeros(n_seq, each, dtype=torch.int32, device="cuda")
    table[:, -1] = torch.arange(1, n_seq + 1, device="cuda")
    k = torch.zeros((n_seq + 1) * page, 1, d, dtype=torch.float8_e4m3fn, device="cuda")
    v = torch.zeros_like(k)
    scale = torch.full((n_seq + 1, 1), 2.0 ** -100, device="cuda")
    g = torch.Generator().manual_seed(1)
    v[page:] = torch.randn(n_seq * page, 1, d, generator=g).cuda().to(v.dtype)
    v_scale = scale.clone()
    v_scale[1:] = 0.5
    ctx = context(1, 1, d, epsp.F16, epsp.F32, n, page)
    batch = epsp.KvBatch(torch.full((n_seq,), n, dtype=torch.int32, device="cuda"), n, table, page, k.shape[0], 0)
    out = torch.full((n_seq, 1, d), float("nan"), device="cuda")
    ctx.check(ctx.decode8_layer(0, batch, randq(n_seq, 1, d, epsp.F16), epsp.Kv8(k, v, scale, v_scale), out,
                                workspace(ctx.decode8_bytes(n_seq, n))))
    ctx.check(ctx.sync_status())
    x = v[page:].view(n_seq, page, d).double() * 0.5
    # equal weights, exact; the sums of units over units in f32 (half a step each, numerator and denominator), a weight
    # that is two f16 (2^-22), the exponent's error (2^-17 as above)
    tol = x.abs().sum(1) / n * (2.0 ** -16 + 2 * n / 32 * 2.0 ** -24)
    assert bool(((out[:, 0].double() - x.sum(1) / n).abs() <= tol).all())


def test_not_finite_queries_and_codes_stay_with_their_heads():
    H, K, d, page = 8, 2, 128, 32
    for dtype in (epsp.BF16, epsp.F32):
        c = Cache8([300, 40], K, d, E, page, page, 1)
        ctx = context(H, K, d, dtype, epsp.F32, 300, page)
        q = randq(2, H, d, dtype)
        clean = run(ctx, c, q)
        q[0, 1, 5], q[1, 6, 0] = float("inf"), float("nan")
        out = run(ctx, c, q)
        bad = torch.zeros(2, H, dtype=torch.bool, device="cuda")
        bad[0, 1] = bad[1, 6] = True
        assert torch.isnan(out[bad]).all() and torch.equal(out[~bad], clean[~bad])
        # a NaN code in K makes its KV head's rows NaN, one in V its column
        q = randq(2, H, d, dtype)
        at = c.at(0, 300)
        c.k8.view(torch.uint8)[at[17], 0, 3] = 0x7F
        c.v8.view(torch.uint8)[at[29], 1, 7] = 0xFF
        out = run(ctx, c, q)
        assert torch.isnan(out[0, :4]).all() and torch.equal(out[1], clean[1])
        assert torch.isnan(out[0, 4:, 7]).all()
        keep = torch.arange(d, device="cuda") != 7
        assert torch.equal(out[0, 4:][:, keep], clean[0, 4:][:, keep])


def test_table_entries_outside_the_pool_and_lengths_are_reported():
    H, K, d, page = 8, 2, 64, 32
    c = Cache8([100, 200, 50], K, d, Q, page, page, 1)
    ctx = context(H, K, d, epsp.BF16, epsp.F32, 200, page)
    q = randq(3, H, d, epsp.BF16)
    clean = run(ctx, c, q)
    kn = randq(3, K, d, epsp.BF16)
    c.d_table[0, 1] = -5
    c.d_lens[2] = 1000
    out = run(ctx, c, q)
    assert ctx.sync_status() == epsp.PREFILL
    assert torch.equal(out[1], clean[1]) and not out[2].any()
    c.d_table[0, 3] = 1 << 20
    was = c.state()
    c.d_lens[1] = 0
    run(ctx, c, q, kn=kn, vn=kn)  # the row has no place: it is not written
    assert ctx.sync_status() == epsp.PREFILL and same(c.state(), was)


@pytest.mark.parametrize("capacity", [3000, 40000])  # joined in a cluster, and by the second kernel
def test_captured_steps_streams_and_workspaces(capacity):
    """A captured step replayed as lengths, rows and queries change, next to another one on its own workspace."""
    H, K, d, page = 14, 2, 64, 64
    ctx = context(H, K, d, epsp.F16, epsp.F32, capacity, page)
    runs = []
    for seed in (1, 2):
        c = Cache8([700, 2500, 64], K, d, E, page, page, seed, capacity=capacity)
        x = dict(q=randq(3, H, d, epsp.F16, seed), kn=randq(3, K, d, epsp.F16, seed + 10),
                 vn=randq(3, K, d, epsp.F16, seed + 20), out=torch.zeros(3, H, d, device="cuda"),
                 ws=workspace(ctx.decode8_bytes(3, capacity)), s=torch.cuda.Stream())
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        was = c.state()
        with torch.cuda.graph(g, stream=x["s"]):
            ctx.check(ctx.decode8_layer(0, c.batch, x["q"], c.kv8, x["out"], x["ws"], k_new=x["kn"], v_new=x["vn"],
                                        stream=x["s"]))
        assert same(c.state(), was)
        runs.append((c, x, g))
    for step in range(4):
        wants = []
        for c, x, g in runs:
            c.lens = [n + 1 for n in c.lens]
            c.d_lens += 1
            x["q"].copy_(randq(3, H, d, epsp.F16, 50 + step))
            x["kn"].copy_(randq(3, K, d, epsp.F16, 60 + step, 4.0))
            want = c.state()
            for s, n in enumerate(c.lens):
                for t, y in enumerate((x["kn"], x["vn"])):
                    write64(c, want, s, y[s].expand(n, K, d), n - 1, t)
            wants.append(want)
        torch.cuda.synchronize()
        for c, x, g in runs:
            with torch.cuda.stream(x["s"]):
                g.replay()
        torch.cuda.synchronize()
        for (c, x, g), want in zip(runs, wants):
            assert same(c.state(), want)
            held(x["out"], c, x["q"], epsp.F32)
    ctx.check(ctx.sync_status())


@pytest.mark.parametrize("q8", [E, Q], ids=name)
def test_rows_past_four_gigabytes(q8):
    """A pool whose rows lie up to 4.3 GB from its start, of which a sequence holds a few far blocks."""
    H, K, d, page = 8, 8, 128, 128
    rows = 4224 * 1024
    k8, v8 = (torch.empty((rows, K, d), dtype=torch.uint8, device="cuda") for _ in "kv")
    ks, vs = (torch.empty((rows // page, K), device="cuda") for _ in "kv")
    small = Cache8([1000], K, d, q8, page, page, 1, capacity=1024)
    blocks = torch.tensor([rows // page - 1 - 3 * i for i in range(8)], dtype=torch.int32)
    for i, b in enumerate(blocks.tolist()):
        at = small.at(0, 1024)[i * page:(i + 1) * page].cuda()
        for big, x, s, y in ((k8, small.k8, ks, small.ks), (v8, small.v8, vs, small.vs)):
            big[b * page:(b + 1) * page] = x.view(torch.uint8)[at]
            s[b] = y[int(at[0]) // page]
    far = Cache8([1000], K, d, q8, page, page, 1, capacity=1024, fill=False)
    far.table, far.rows = blocks[None], rows
    far.d_table = far.table.cuda()
    far.k8, far.v8, far.ks, far.vs = k8.view(TORCH8[q8]), v8.view(TORCH8[q8]), ks, vs
    far.batch, far.kv8 = epsp.KvBatch(far.d_lens, 1024, far.d_table, page, rows), epsp.Kv8(far.k8, far.v8, ks, vs)
    ctx = context(H, K, d, epsp.BF16, epsp.F32, 1024, page)
    q, kn = randq(1, H, d, epsp.BF16), randq(1, K, d, epsp.BF16, 9)
    a, b = (run(ctx, c, q, kn=kn, vn=kn) for c in (small, far))
    assert torch.equal(a, b)
    held(b, far, q, epsp.F32)
    x = Cache([1000], K, d, epsp.BF16, 0, 1, capacity=1024)
    ctx.check(ctx.unpack_kv(0, far.batch, far.kv8, x.batch, x.k, x.v))
    assert torch.equal(x.k[:1000], far.seq(0)[0].to(torch.bfloat16))
    y = Cache8([1000], K, d, q8, page, 0, 1, capacity=1024, fill=False)
    ctx.check(ctx.pack_kv(0, x.batch, x.k, x.v, far.batch, far.kv8))
    ctx.check(ctx.pack_kv(0, x.batch, x.k, x.v, y.batch, y.kv8))
    ctx.check(ctx.sync_status())
    assert all(torch.equal(s, t) for s, t in zip(far.seq(0), y.seq(0)))


def test_a_scale_factor_of_the_model_and_a_large_capacity():
    H, K, d, page = 8, 2, 64, 32
    c = Cache8([300, 5], K, d, E, page, page, 1, capacity=65536)
    ctx = context(H, K, d, epsp.BF16, epsp.BF16, 65536, page, kq_scale=0.31)
    q = randq(2, H, d, epsp.BF16, 4, 0.5)
    held(run(ctx, c, q, epsp.BF16), c, q, epsp.BF16, float(torch.tensor(0.31)))
    assert math.isclose(ctx.cfg.kq_scale, 0.31, rel_tol=1e-6)
    assert round8(torch.tensor([0.3], dtype=torch.float64), E) == 0.3125 and bytes_of(torch.ones(1), Q) == 1
