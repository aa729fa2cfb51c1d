"""What the binding sees of pools before a call reaches the library."""
import pytest
import torch

import epsp
from test_serving_host import make


def test_pools_of_other_blocks_are_refused():
    """8 blocks of 64 rows (2 KV heads of 64): a cache or scales of another number of rows is not theirs."""
    c = make()
    i32 = dict(dtype=torch.int32)
    pages = epsp.Pages(torch.zeros(3, **i32), torch.zeros((3, 4), **i32), torch.zeros(8, **i32), 64)
    f16 = dict(dtype=torch.float16)
    bad = [torch.zeros((256, 2, 64), **f16), torch.zeros((1024, 2, 64), dtype=torch.int8),
           torch.zeros((2, 8, 64, 2, 64), **f16), torch.zeros((8, 32, 2, 64)), torch.zeros((32, 2)), torch.zeros((24, 2))]
    good = [torch.zeros((512, 2, 64), **f16), torch.zeros((8, 64, 2, 64), dtype=torch.int8), torch.zeros((16, 2)),
            torch.zeros((8, 2, 64)), torch.zeros((8, 2)), torch.zeros((8, 100)), torch.zeros(64)]
    news = torch.zeros(3, **i32)
    for t in bad:
        pools = epsp.Pools([good[0], t], 8)
        for call in (lambda: c.resize_seqs(pages, news, pools, None), lambda: c.compact_pool(pages, pools, None)):
            with pytest.raises(ValueError, match="pool 1 .* 8 blocks of 64 rows"):
                call()
    with pytest.raises(ValueError, match="not on cuda"):  # (what is refused next)
        c.resize_seqs(pages, news, epsp.Pools(good, 8), None)
