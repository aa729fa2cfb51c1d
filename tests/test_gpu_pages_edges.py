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


@pytest.mark.parametrize("n_seq,blocks", [(3, 3060), (55, 3000), (3, 6120), (2, 6143), (3, 6144), (4096, 8192), (3, 8193)],
                         ids=str)
def test_sizes_around_what_a_plan_holds_on_chip(n_seq, blocks):
    """Plans of 48 KB, a little less and a little more, of all that one CTA holds, and one more."""
    x = Both(n_seq, 2, 32, blocks, 2, sizes=[4])
    assert x.resize([(40 if s % 3 else 20) if s < 3000 else 0 for s in range(n_seq)])
    x.fork([s if s % 4 else min(s + 1, n_seq - 1) for s in range(n_seq)])
    assert x.resize([min(n + 1, 64) if n else 0 for n in x.book.lens])
    assert x.resize([0 if s % 2 else n for s, n in enumerate(x.book.lens)])
    x.compact()


def test_the_last_holder_keeps_a_block_that_all_grow_in():
    x = Both(4, 4, 32, 20, 1)
    x.resize([40, 0, 0, 0])
    kept = x.book.tables[0][1]
    x.fork([0, 0, 0, 0])
    x.resize([41, 41, 41, 41])
    last = x.tables[:, 1].tolist()
    assert last[3] == kept and len(set(last)) == 4
