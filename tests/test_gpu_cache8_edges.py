"""What goes through the cache in 8 bits and comes back, at the ends of the types."""
import pytest
import torch

import epsp
from cache8_util import Cache8
from serving_util import TORCH, Cache, context
from test_gpu_cache8 import E, Q, name

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [epsp.BF16, epsp.F16, epsp.F32], ids=name)
@pytest.mark.parametrize("q8", [E, Q], ids=name)
def test_the_largest_values_come_back_finite(q8, dtype):
    """Pages whose largest magnitude is the type's: what rounding to 8 bits takes past it comes back as the largest."""
    K, d, page = 2, 64, 32
    top = torch.finfo(TORCH[dtype]).max
    src = Cache([2 * page], K, d, dtype, 0, 1)
    x = torch.linspace(-1, 1, page * d, dtype=torch.float64).view(page, d) * top
    for t, sign in ((src.k, 1), (src.v, -1)):
        t[:page] = (sign * x)[:, None].to(t.dtype).cuda()
        t[0, 0, 0], t[1, 1, 5] = top, -top
    c, out = Cache8([2 * page], K, d, q8, page, 0, 2, fill=False), Cache([2 * page], K, d, dtype, 0, 3)
    ctx = context(K, K, d, dtype, dtype, 2 * page, page)
    ctx.check(ctx.pack_kv(0, src.batch, src.k, src.v, c.batch, c.kv8))
    ctx.check(ctx.unpack_kv(0, c.batch, c.kv8, out.batch, out.k, out.v))
    ctx.check(ctx.sync_status())
    past = 0
    for got, value in zip((out.k, out.v), c.seq(0)):  # (64 bits)
        assert torch.equal(got, value.clamp(-top, top).to(TORCH[dtype]))
        assert torch.isfinite(got).all()
        past += int((value.abs() > top).sum())
    assert past > 0
    if q8 == E:  # a NaN code stays one next to them
        c.k8.view(torch.uint8)[3, 1, 7] = 0xFF
        ctx.check(ctx.unpack_kv(0, c.batch, c.kv8, out.batch, out.k, out.v))
        ctx.check(ctx.sync_status())
        bad = torch.isnan(out.k)
        assert bool(bad[3, 1, 7]) and int(bad.sum()) == 1
