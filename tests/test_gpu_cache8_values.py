"""Decode over the cache in 8 bits where its arithmetic has its limits: terms that cancel, scales and queries at the ends
of their ranges, every output type."""
import pytest
import torch

import epsp
from cache8_util import Cache8, decode64, write64
from serving_util import TORCH, context, rounding, workspace
from test_gpu_cache8 import E, HEADS, Q, held, name, randq, run, same

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("q8", [E, Q], ids=name)
@pytest.mark.parametrize("dtype", [epsp.BF16, epsp.F16, epsp.F32], ids=name)
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("capacity", [1111, 13000])  # joined in clusters, and split over the device
def test_outputs_of_every_type_are_one_result_rounded(capacity, heads, dtype, q8):
    """A row appended, every head layout: 16-bit outputs are right to a rounding of what is right for f32 outputs."""
    H, K, d = heads
    page, lens = 64, [0, 1, 33, 64, 500, 1111]
    c = Cache8(lens, K, d, q8, page, page, 1, capacity=capacity)
    q, kn, vn = randq(6, H, d, dtype), randq(6, K, d, dtype, 6, 3.0), randq(6, K, d, dtype, 7)
    want, outs = c.state(), {}
    for i, n in enumerate(lens):
        if n:
            for t, x in enumerate((kn, vn)):
                write64(c, want, i, x[i].expand(n, K, d), n - 1, t)
    for o in (epsp.F32, epsp.BF16, epsp.F16):
        ctx = context(H, K, d, dtype, o, capacity, page)
        outs[o] = run(ctx, c, q, o, kn=kn, vn=vn)  # (the same row again: the same bytes)
        ctx.check(ctx.sync_status())
        assert same(c.state(), want)
    held(outs[epsp.F32], c, q, epsp.F32)
    ref, tol = decode64(c, q)
    for o in (epsp.BF16, epsp.F16):
        if dtype == epsp.F32:
            assert torch.equal(outs[o], outs[epsp.F32].to(TORCH[o]))
        # (16-bit models add their units up in the tensor cores for 16-bit outputs: off by tol as the other, then rounded)
        half = torch.finfo(TORCH[o]).eps / 2
        assert bool(((outs[o].double() - ref).abs() <= tol * (1 + half) + rounding(ref, o)).all())


@pytest.mark.parametrize("q8", [E, Q], ids=name)
@pytest.mark.parametrize("dtype", [epsp.BF16, epsp.F16], ids=name)
@pytest.mark.parametrize("heads", [(8, 2, 128), (14, 2, 64), (16, 1, 128), (40, 1, 64)], ids=str)
def test_bf16_outputs_of_terms_that_cancel(heads, dtype, q8):
    """Rows in pairs with opposite V and weights that differ by a few 2^-10: a weight in 11 bits would show."""
    H, K, d = heads
    page, lens = 32, [2, 16, 40, 700]
    c = Cache8(lens, K, d, q8, page, 0, 1)
    b = c.v8.view(torch.uint8)
    for i, n in enumerate(lens):
        at = c.at(i, n).cuda()
        b[at[1::2]] = b[at[0::2]] ^ 0x80 if q8 == E else (-c.v8[at[0::2]]).view(torch.uint8)
    ctx = context(H, K, d, dtype, epsp.BF16, 700, page)
    q = randq(4, H, d, dtype, scale=2.0 ** -11)
    ref, tol = decode64(c, q)  # (as for f32 outputs)
    out = run(ctx, c, q, epsp.BF16)
    ctx.check(ctx.sync_status())
    # what is rounded to bf16 is off by tol at most
    assert bool(((out.double() - ref).abs() <= tol * (1 + 2.0 ** -8) + rounding(ref, epsp.BF16)).all())


@pytest.mark.parametrize("q8", [E, Q], ids=name)
@pytest.mark.parametrize("dtype", [epsp.BF16, epsp.F32], ids=name)
@pytest.mark.parametrize("capacity", [64, 13000])  # joined in a CTA, and split over the device
@pytest.mark.parametrize("v_scale", [2.0 ** -126, 2.0 ** -100, 2.0 ** -64, 1.0, 2.0 ** 126, 2.0 ** 127, 1.3 * 2.0 ** 126], ids=str)
def test_weights_do_not_depend_on_the_scale_of_v(v_scale, capacity, dtype, q8):
    """V the unit matrix, so that an output element is one weight times V's scale: the scale, wherever it lies, costs it
    nothing."""
    d, n = 64, 32
    c = Cache8([n], 1, d, q8, 32, 0, 1, capacity=capacity)
    at, one = c.at(0, n), 1 if q8 == Q else 0x38
    k = torch.randint(-127, 128, (n,), generator=torch.Generator().manual_seed(1))
    c.k8.view(torch.uint8).zero_(), c.v8.view(torch.uint8).zero_()
    c.k8[at.cuda(), 0, 0] = k.cuda().to(c.k8.dtype)
    c.v8.view(torch.uint8)[at.cuda(), 0, torch.arange(n)] = one
    c.ks.fill_(2.0 ** -5), c.vs.fill_(v_scale)
    ctx = context(1, 1, d, dtype, epsp.F32, capacity, 32)
    q = torch.zeros(1, 1, d, device="cuda").to(TORCH[dtype])
    q[0, 0, 0] = 3.0
    out = run(ctx, c, q)[0, 0].double()
    ctx.check(ctx.sync_status())
    x = c.k8[at.cuda(), 0, 0].float().double() * 2.0 ** -5 * 3 / 8
    want = torch.zeros(d, dtype=torch.float64, device="cuda")
    want[:n] = torch.softmax(x, 0) * float(torch.tensor(v_scale, dtype=torch.float32))
    # In units of 2^-24.  The score is one exact product, times the factor, log2 e in it and V's own: 4 roundings of
    # |x| <= 1.5, so 6 of a weight; the subtraction of a maximum that is 16 off at most, 2^-21 ln 2, 5.5; the exponential
    # 2^-22, 4: 16 of a weight, 32 with its sum's.  The weight as two f16 4, its products with the byte 4, a scale that is
    # no power of two 1; the sum of weights 7, the quotient 2, the joins' factors 2 (of 2^-22 each, in one part)
    tol = want * (32 + 4 + 4 + 1 + 7 + 2 + 8) * 2.0 ** -24
    # Below f32's normal numbers (scales near 2^-126) steps are 2^-149: half a one in the sum, which the quotient by a sum
    # of weights of 1/2 or more can double, and half a one in the quotient
    tiny = 1.5 * 2.0 ** -149
    assert bool(((out - want).abs() <= tol + tiny).all()), float(((out - want).abs() / (want + tiny)).max() * 2 ** 24)


@pytest.mark.parametrize("q8", [E, Q], ids=name)
@pytest.mark.parametrize("dtype", [epsp.F16, epsp.F32], ids=name)
@pytest.mark.parametrize("scales", [(-100, -100, -100), (-100, -90, -89), (-80, -60, -88), (-126, -120, -110),
                                    (-100, 40, -8), (-100, 110, 0), (126, 120, 100), (115, -126, 115)], ids=str)
def test_scales_of_v_from_end_to_end(scales, dtype, q8):
    """Pages of three scales in turn, far apart or all at one end, within the usual tolerance; pages of the smallest of
    far scales hold zeros, as pack makes them."""
    H, K, d, page, lens = 4, 2, 64, 32, [700, 90, 1, 33]
    c = Cache8(lens, K, d, q8, page, 0, 1)
    p = torch.arange(c.vs.shape[0], device="cuda") % 3
    c.vs[:] = torch.exp2(torch.tensor(scales, dtype=torch.float64, device="cuda")[p])[:, None].float()
    b = c.v8.view(-1, page, K, d)
    b.copy_(torch.sign(b.float()).to(b.dtype))  # (448 * 2^126 is no f32)
    if max(scales) - min(scales) > 100:
        b.view(torch.uint8)[p == scales.index(min(scales))] = 0
    ctx = context(H, K, d, dtype, epsp.F32, 700, page)
    q = randq(4, H, d, dtype, 3)
    ref, tol = decode64(c, q)
    out = run(ctx, c, q)
    ctx.check(ctx.sync_status())
    assert bool(((out.double() - ref).abs() <= tol + rounding(ref, epsp.F32)).all())
    assert torch.isfinite(out).all() and bool((out != 0).any(2).all())


@pytest.mark.parametrize("dtype", [epsp.BF16, epsp.F32], ids=name)
@pytest.mark.parametrize("lens", [[20, 7], [1500, 700], [40000, 9]], ids=["a CTA", "a cluster", "split"])
def test_a_head_does_not_depend_on_the_others(lens, dtype):
    """One head of a group asks with queries far larger than the others': their bits stay."""
    H, K, d, page = 8, 2, 64, 64
    c = Cache8(lens, K, d, E, page, page, 1)
    ctx = context(H, K, d, dtype, epsp.F32, max(lens), page)
    q = randq(2, H, d, dtype)
    clean = run(ctx, c, q)
    q[:, 2] *= 40
    out = run(ctx, c, q)
    ctx.check(ctx.sync_status())
    keep = torch.arange(H, device="cuda") != 2
    assert torch.equal(out[:, keep], clean[:, keep]) and not torch.equal(out, clean)


@pytest.mark.parametrize("q8", [E, Q], ids=name)
@pytest.mark.parametrize("dtype", [epsp.BF16, epsp.F16, epsp.F32], ids=name)
@pytest.mark.parametrize("lens", [[20, 7], [1500, 700], [40000, 9]], ids=["a CTA", "a cluster", "split"])
def test_a_query_of_minus_infinity_on_keys_of_one_sign(lens, dtype, q8):
    """Every score of the head is -inf: a row of NaN, however a run is finished; other heads as without it."""
    H, K, d, page = 8, 2, 64, 64
    c = Cache8(lens, K, d, q8, page, page, 1)
    b = c.k8.view(torch.uint8)
    for i, n in enumerate(lens):
        b[c.at(i, n).cuda(), :, 5] = 0x30  # positive in both types
    ctx = context(H, K, d, dtype, epsp.F32, max(lens), page)
    q = randq(2, H, d, dtype)
    clean = run(ctx, c, q)
    bad = torch.zeros(2, H, dtype=torch.bool, device="cuda")
    bad[0, 1] = bad[0, 6] = bad[1, 3] = True
    q[..., 5][bad] = -float("inf")
    out = run(ctx, c, q)
    ctx.check(ctx.sync_status())
    assert torch.isnan(out[bad]).all() and torch.equal(out[~bad], clean[~bad])


@pytest.mark.parametrize("q8", [E, Q], ids=name)
@pytest.mark.parametrize("dtype", [epsp.BF16, epsp.F16, epsp.F32], ids=name)
@pytest.mark.parametrize("lens", [[70, 1], [1500, 700], [40000, 9]], ids=["a CTA", "a cluster", "split"])
@pytest.mark.parametrize("v_scale", [2.0 ** -100, 2.0 ** -40, 1.0, 2.0 ** 100], ids=str)
def test_scores_beyond_whole_numbers(v_scale, lens, dtype, q8):
    """Scores of up to 2^37 and more, where f32 has no fractions: the row of the largest is all there is, whatever V's
    scale."""
    K, d, page = 1, 64, 32
    c = Cache8(lens, K, d, q8, page, page, 1)
    g = torch.Generator().manual_seed(2)
    c.k8.view(torch.uint8).zero_()
    want = torch.zeros(len(lens), 1, d, device="cuda")
    for i, n in enumerate(lens):
        at, top = c.at(i, n).cuda(), int(torch.randint(n, (1,), generator=g))
        k = torch.randint(-112, 97, (n,), generator=g).float()
        k[top] = 112.0
        c.k8[at, 0, 3] = k.cuda().to(c.k8.dtype)
        want[i, 0] = c.v8[at[top], 0].float() * v_scale
    c.ks.fill_(2.0 ** 12), c.vs.fill_(v_scale)
    ctx = context(1, K, d, dtype, epsp.F32, max(lens), page)
    q = torch.zeros(len(lens), 1, d, device="cuda").to(TORCH[dtype])
    q[:, :, 3] = 2.0 ** 15 if dtype == epsp.F16 else 2.0 ** 40
    out = run(ctx, c, q)
    ctx.check(ctx.sync_status())
    assert torch.equal(out, want)


@pytest.mark.parametrize("q8", [E, Q], ids=name)
@pytest.mark.parametrize("dtype", [epsp.F16, epsp.F32], ids=name)
def test_f32_outputs_of_long_runs_have_no_bias(dtype, q8):
    """65,536 rows a sequence, all of one block: hundreds of units a warp, whose sums must not be cut one by one."""
    page, d, n_seq, n = 32, 64, 160, 65536
    table = torch.arange(n_seq, dtype=torch.int32, device="cuda")[:, None].repeat(1, n // page).contiguous()
    g = torch.Generator().manual_seed(1)
    v = torch.randint(1, 113, (n_seq * page, 1, d), generator=g).float().cuda().to(torch.int8 if q8 == Q else torch.float8_e4m3fn)
    scale = torch.full((n_seq, 1), 1.3, device="cuda")
    ctx = context(1, 1, d, dtype, epsp.F32, n, page)
    batch = epsp.KvBatch(torch.full((n_seq,), n, dtype=torch.int32, device="cuda"), n, table, page, n_seq * page, 0)
    out = torch.full((n_seq, 1, d), float("nan"), device="cuda")
    q = torch.zeros(n_seq, 1, d, device="cuda").to(TORCH[dtype])
    cache = epsp.Kv8(v.clone(), v, scale.clone(), scale)
    ctx.check(ctx.decode8_layer(0, batch, q, cache, out, workspace(ctx.decode8_bytes(n_seq, n))))
    ctx.check(ctx.sync_status())
    ref = v.float().double().view(n_seq, page, d).mean(1) * float(scale[0, 0])
    off = ((out[:, 0].double() - ref) / ref) * 2.0 ** 24
    # In units of 2^-24.  All weights are 1, and so are their sums.  P, the scale, is two f16: 4; a unit's four products cut
    # 2 each: 8; the quotient 2, the joins' factors 4.  A warp adds up 256 units at most, each addition off by half a step,
    # one way or the other with the column: uniform, so 0.29 of a step a unit and column, less where the sum is small yet
    assert abs(float(off.mean())) <= 18 + 6 * 0.29 * 256 / off.numel() ** 0.5, float(off.mean())
    assert float(off.abs().max()) <= 18 + 256
