"""Blocks shared, taken, given back and moved, against the same steps on plain lists: lengths, tables (whole, with the
entries that nobody holds), counts and every pool's contents, exactly."""
import random

import pytest
import torch

import epsp
from cache8_util import Book
from serving_util import context, workspace

pytestmark = pytest.mark.gpu


class Both:
    """The same state on the device and as a Book; pools of several block sizes whose blocks begin with a number."""

    SIZES = [4, 8, 20, 4096, 10000, 65536 + 12]

    def __init__(self, n_seq, stride, B, blocks, seed, sizes=None, page=32):
        r = self.r = random.Random(seed)
        self.B, self.blocks, self.stride = B, blocks, stride
        tables = [[r.randrange(blocks) for _ in range(stride)] for _ in range(n_seq)]  # stale entries: any blocks
        self.book = Book([0] * n_seq, tables, [0] * blocks, B, range(blocks))
        self.lens = torch.zeros(n_seq, dtype=torch.int32, device="cuda")
        self.tables = torch.tensor(tables, dtype=torch.int32, device="cuda")
        self.refs = torch.zeros(blocks, dtype=torch.int32, device="cuda")
        self.pages = epsp.Pages(self.lens, self.tables, self.refs, B)
        self.data = []
        for i, size in enumerate(self.SIZES if sizes is None else sizes):
            x = torch.randint(0, 256, (blocks, size), dtype=torch.uint8, device="cuda")
            # each block begins with its number; every third pool starts 4 bytes off a 16-byte boundary
            x.view(torch.int32)[:, 0] = torch.arange(blocks, device="cuda", dtype=torch.int32)
            if i % 3 == 2:
                room = torch.zeros(blocks * size + 4, dtype=torch.uint8, device="cuda")
                room[4:] = x.view(-1)
                x = room[4:].view(blocks, size)
            self.data.append(x)
        self.first = [x.clone() for x in self.data]
        self.pools = epsp.Pools(self.data, blocks)
        self.ctx = context(2, 2, 64, epsp.F16, epsp.F16, 64, page)
        self.ws = workspace(max(self.ctx.fork_bytes(self.pages), self.ctx.resize_bytes(self.pages),
                                self.ctx.compact_bytes(self.pages)))

    def ints(self, x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    def fork(self, parents, lens=None, rc=epsp.OK):
        c = self.ctx
        c.check(c.fork_seqs(self.pages, self.ints(parents), self.ws, lens=None if lens is None else self.ints(lens)))
        self.book.fork(parents, lens)
        self.check(rc)

    def resize(self, lens, rc=epsp.OK):
        self.ctx.check(self.ctx.resize_seqs(self.pages, self.ints(lens), self.pools, self.ws))
        fits = self.book.resize(lens)
        self.check(rc if fits else epsp.OUT_OF_MEMORY)
        return fits

    def compact(self):
        used = self.ints([-1])
        self.ctx.check(self.ctx.compact_pool(self.pages, self.pools, self.ws, n_used=used))
        assert int(used) == self.book.compact()
        self.check()

    def check(self, rc=epsp.OK):
        assert self.ctx.sync_status() == rc, self.ctx.last_error()
        b = self.book
        assert b.check()
        assert self.lens.tolist() == b.lens and self.refs.tolist() == b.refs
        assert self.tables.tolist() == b.tables
        # what blocks in use hold, in every pool; free ones may hold anything
        live = torch.tensor([r > 0 for r in b.refs], device="cuda")
        at = torch.tensor(b.pool, device="cuda")[live]
        for x, first in zip(self.data, self.first):
            assert torch.equal(x[live], first[at])

    def room(self):
        return self.stride * self.B


@pytest.mark.parametrize("n_seq,stride,B,blocks", [(1, 1, 32, 1), (5, 4, 32, 17), (40, 6, 64, 150), (300, 3, 32, 700),
                                                   (70, 5, 32, 5000), (70, 5, 32, 9000),
                                                   (5000, 2, 32, 6000)], ids=str)
def test_a_server_s_life(n_seq, stride, B, blocks):
    """Sequences grow, fork, are cut back, freed and compacted in a random order."""
    x = Both(n_seq, stride, B, blocks, n_seq, sizes=None if blocks < 1000 else [4, 20, 4100])
    r, refused = x.r, 0
    for step in range(25 if n_seq < 1000 else 8):
        was = list(x.book.lens)
        what = r.random()
        if what < 0.25:
            x.fork([r.choice([s, r.randrange(n_seq), r.randrange(-1, n_seq)]) for s in range(n_seq)])
        elif what < 0.45:
            parents = [r.choice([s, r.randrange(n_seq)]) for s in range(n_seq)]
            x.fork(parents, [r.randint(0, was[p]) for p in parents])
        elif what < 0.6:
            x.compact()
        elif what < 0.7:
            refused += not x.resize([r.choice([n, 0, n // 2]) for n in was])
        else:
            refused += not x.resize([min(x.room(), max(0, n + r.choice([0, 1, 1, B - 1, B, -1, -n]))) for n in was])
    # freed as a whole, everything fits again
    assert x.resize([0] * n_seq) and sum(x.book.refs) == 0
    x.compact()


def test_all_holders_of_a_block_grow_or_some_do():
    x = Both(4, 4, 32, 20, 1)
    x.resize([40, 0, 0, 0])
    x.fork([0, 0, 0, 0])
    assert x.book.refs.count(4) == 2
    x.resize([41, 41, 41, 41])  # the last one keeps the block
    assert x.book.tables[3][1] == x.book.tables[3][1] and sum(x.book.refs) == 8 and x.book.refs.count(4) == 1
    x.fork([0, 0, 0, 0], [33, 34, 35, 33])  # other lengths in the same block
    x.resize([33, 64, 36, 33])  # two of four holders grow: both copy
    x.fork([0, 0, 2, 3], [32, 32, 36, 33])  # whole blocks: nothing to copy
    free = x.book.refs.count(0)
    x.resize([33, 33, 36, 33])
    assert x.book.refs.count(0) == free - 2
    # a sequence that is cut back into a block that others hold, then grows: a copy
    x.fork([2, 2, 2, 2])
    x.resize([20, 36, 36, 36])
    x.resize([21, 36, 36, 36])


def test_too_few_blocks_change_nothing():
    x = Both(3, 8, 32, 10, 2)
    assert x.resize([100, 100, 30])  # 4 + 4 + 1 of 10
    assert not x.resize([100, 130, 70])  # 1 + 2 more
    assert x.resize([0, 130, 70])  # what one gives back another takes, in one call
    assert x.resize([33, 130, 64])
    x.fork([0, 0, 2])
    assert not x.resize([256, 34, 64])
    assert x.resize([34, 34, 64])
    x.compact()


def test_bad_parents_lengths_and_tables_are_reported():
    x = Both(4, 3, 32, 12, 3)
    x.resize([50, 64, 10, 0])
    x.fork([1, 4, -2, 0], rc=epsp.PREFILL)
    x.fork([0, 1, 2, 2], [51, 65, -1, 10], rc=epsp.PREFILL)
    x.resize([97, -1, 20, 11], rc=epsp.PREFILL)
    # a length and an entry that the tables cannot hold: the sequence counts as empty, the entry is not followed
    lens, tables = x.lens.clone(), x.tables.clone()
    x.lens[0] = 97
    x.tables[1, 0] = 12
    c = x.ctx
    for call in (lambda: c.compact_pool(x.pages, x.pools, x.ws), lambda: c.count_refs(x.pages),
                 lambda: c.fork_seqs(x.pages, x.ints([0, 1, 2, 3]), x.ws),
                 lambda: c.resize_seqs(x.pages, x.ints([0, 0, 0, 0]), x.pools, x.ws)):
        c.check(call())
        assert c.sync_status() == epsp.PREFILL
        x.lens.copy_(lens), x.tables.copy_(tables)
        x.lens[0] = 97
        x.tables[1, 0] = 12


def test_counts_of_tables_made_elsewhere():
    x = Both(6, 4, 64, 40, 4)
    x.resize([100, 256, 1, 64, 0, 200])
    x.fork([1, 1, 2, 3, 1, 5])
    want = x.refs.clone()
    x.refs.fill_(77)
    x.ctx.check(x.ctx.count_refs(x.pages))
    x.ctx.check(x.ctx.sync_status())
    assert torch.equal(x.refs, want)


def test_many_pools_and_all_lengths_aliases():
    """More pools than one launch takes; new_lens and lens may be the lengths themselves."""
    x = Both(3, 4, 32, 12, 5, sizes=[4, 16, 8, 1024] * 70)
    x.resize([100, 20, 40])
    x.fork([0, 0, 0])
    x.resize([101, 100, 101])
    c = x.ctx
    c.check(c.resize_seqs(x.pages, x.lens, x.pools, x.ws))
    c.check(c.fork_seqs(x.pages, x.ints([0, 1, 2]), x.ws, lens=x.lens))
    x.check()
    x.resize([0, 100, 0])
    x.compact()


def test_captured_steps():
    """A captured fork, growth and compaction replayed as parents and lengths change."""
    x = Both(6, 6, 32, 64, 6)
    x.resize([40, 70, 33, 10, 90, 0])
    parents, lens = x.ints([0] * 6), x.ints([0] * 6)
    s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    c = x.ctx
    with torch.cuda.graph(g, stream=s):
        c.check(c.fork_seqs(x.pages, parents, x.ws, stream=s))
        c.check(c.resize_seqs(x.pages, lens, x.pools, x.ws, stream=s))
        c.check(c.compact_pool(x.pages, x.pools, x.ws, stream=s))
    for step in range(6):
        p = [x.r.randrange(6) for _ in range(6)]
        parents.copy_(x.ints(p))
        x.book.fork(p)
        n = [min(192, m + x.r.choice([0, 1, 30])) for m in x.book.lens]
        lens.copy_(x.ints(n))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert x.book.resize(n)
        x.book.compact()
        x.check()


def test_far_blocks():
    """Blocks past 4 GB of their pool."""
    size, blocks = 1 << 20, 4200
    x = Both(3, 4, 32, blocks, 7, sizes=[64])
    big = torch.empty((blocks, size), dtype=torch.uint8, device="cuda")
    for b in (0, 1, 2, 4197, 4198, 4199):
        big[b] = b % 251
    pools = epsp.Pools([big], blocks)
    x.lens.copy_(x.ints([50, 0, 0])), x.refs.zero_()
    x.tables[0, :2] = x.ints([4199, 4197])
    x.ctx.check(x.ctx.count_refs(x.pages))
    x.ctx.check(x.ctx.fork_seqs(x.pages, x.ints([0, 0, -1]), x.ws))
    x.ctx.check(x.ctx.resize_seqs(x.pages, x.ints([51, 50, 0]), pools, x.ws))
    x.ctx.check(x.ctx.sync_status())
    assert x.tables[0, :2].tolist() == [4199, 0] and x.tables[1, :2].tolist() == [4199, 4197]
    assert bool((big[0] == 4197 % 251).all())
    x.ctx.check(x.ctx.compact_pool(x.pages, pools, x.ws))
    x.ctx.check(x.ctx.sync_status())
    assert x.tables[0, :2].tolist() == [2, 0] and x.tables[1, :2].tolist() == [2, 1]
    assert bool((big[2] == 4199 % 251).all()) and bool((big[1] == 4197 % 251).all())
