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
    """A row appended, every head layout: 16-bit outputs are the f32 output rounded once, and that is right."""
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
    for o in (epsp.BF16, epsp.F16):
        assert torch.equal(outs[o], outs[epsp.F32].to(TORCH[o]))


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
