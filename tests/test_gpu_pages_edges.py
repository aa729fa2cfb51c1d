"""Calls on blocks at their edges: entries that name no block, who keeps a shared block, sizes at which plans change
kind."""
import pytest
import torch

import epsp
from test_gpu_pages import Both

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n_seq,blocks", [(3, 20), (3, 9000)], ids=["one CTA", "a cluster"])
def test_growth_in_a_block_that_is_none_is_reported(n_seq, blocks):
    """A sequence grows within its last block, whose table entry lies outside the pool: the entry is not followed, the
    lengths grow as asked, and the call says so."""
    x = Both(n_seq, 4, 32, blocks, 1, sizes=[4, 64])
    x.resize([40, 33, 64])
    for bad in (blocks, -1, 2 ** 31 - 1, -2 ** 31):
        was, refs = int(x.tables[0, 1]), x.refs.clone()
        x.tables[0, 1] = bad
        n = int(x.lens[0]) + 1
        x.ctx.check(x.ctx.resize_seqs(x.pages, x.ints([n, 33, 64]), x.pools, x.ws))
        assert x.ctx.sync_status() == epsp.PREFILL and "where 0xc1" in x.ctx.last_error()
        assert x.lens.tolist() == [n, 33, 64] and torch.equal(x.refs, refs) and int(x.tables[0, 1]) == bad
        x.tables[0, 1] = was
        x.book.resize([n, 33, 64])
        x.check()
