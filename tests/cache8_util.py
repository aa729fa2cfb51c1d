"""Plain 64-bit forms of the 8-bit cache and of the calls that manage blocks, for their tests."""
from __future__ import annotations

import math

import torch

import epsp
from serving_util import TORCH, score_error, softmax64

TOP = {epsp.E4M3: 448.0, epsp.I8: 127.0}
TORCH8 = {epsp.E4M3: torch.float8_e4m3fn, epsp.I8: torch.int8}


def scale64(top, q8):
    """The least power of two s (2^-100 or more) with top <= M s, by trying."""
    e = -100
    while top > TOP[q8] * 2.0 ** e:
        e += 1
    return 2.0 ** e


def round8(x, q8):
    """Nearest value of the type (ties to even) of doubles within its range; infinities to the largest, NaN to 0."""
    x = torch.nan_to_num(x, nan=0.0, posinf=TOP[q8], neginf=-TOP[q8])
    if q8 == epsp.I8:
        return torch.round(x)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)  # 2^-9 below 2^-6
    return torch.round(x / step) * step


def bytes_of(x, q8):
    """The bytes that hold these values exactly."""
    return x.float().to(TORCH8[q8]).view(torch.uint8)


class Cache8:
    """Sequences' rows in 8 bits, contiguous or scattered over a shuffled pool.  Bytes that no sequence holds are NaN
    codes (-1 as integers), scales of pages without rows NaN."""

    def __init__(self, lens, n_head_kv, d, q8, page, block_rows, seed, capacity=None, fill=True):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.B, self.q8, self.page, self.K, self.d = list(lens), block_rows, q8, page, n_head_kv, d
        n_seq, cap = len(lens), max(1, capacity or max(lens))
        self.cap = cap
        if block_rows:
            each = -(-cap // block_rows)
            blocks = n_seq * each + 3
            self.table = torch.randperm(blocks, generator=g)[: n_seq * each].view(n_seq, each).to(torch.int32)
            self.rows, self.seq_rows = blocks * block_rows, 0
        else:
            self.seq_rows = -(-cap // page) * page
            self.table, self.rows = None, n_seq * self.seq_rows
        shape = (self.rows, n_head_kv, d)
        b = {t: torch.full(shape, 0xFF, dtype=torch.uint8) for t in "kv"}
        s = {t: torch.full((self.rows // page, n_head_kv), float("nan")) for t in "kv"}
        if fill:
            for i, n in enumerate(self.lens):
                at = self.at(i, n)
                for t in "kv":
                    if q8 == epsp.I8:
                        x = torch.randint(-127, 128, (n, n_head_kv, d), generator=g).double()
                    else:
                        x = round8(torch.randn(n, n_head_kv, d, generator=g).double().clamp(-4, 4) * 110, q8)
                    b[t][at] = bytes_of(x, q8)
                    p = torch.unique(at // page)
                    # magnitudes of about a unit normal's, another power of two each
                    s[t][p] = torch.exp2(torch.randint(-9, -5, (len(p), n_head_kv), generator=g).float())
        self.k8, self.v8 = (b[t].cuda().view(TORCH8[q8]) for t in "kv")
        self.ks, self.vs = (s[t].cuda() for t in "kv")
        self.d_table = None if self.table is None else self.table.cuda()
        self.d_lens = torch.tensor(self.lens, dtype=torch.int32).cuda()
        self.batch = epsp.KvBatch(self.d_lens, cap, self.d_table, block_rows, self.rows, self.seq_rows)
        self.kv8 = epsp.Kv8(self.k8, self.v8, self.ks, self.vs)

    def at(self, i, n):
        r = torch.arange(n)
        if self.table is None:
            return i * self.seq_rows + r
        return self.table[i].long()[r // self.B] * self.B + r % self.B

    def seq(self, i):
        """The values that the rows of sequence i hold, in 64 bits."""
        at = self.at(i, self.lens[i]).cuda()
        return tuple(b[at].float().double() * s[at // self.page][..., None].double()
                     for b, s in ((self.k8, self.ks), (self.v8, self.vs)))

    def state(self):
        return [x.clone() for x in (self.k8.view(torch.uint8), self.v8.view(torch.uint8), self.ks, self.vs)]


def write64(cache, state, i, x, a, t):
    """Rows [a, n) of x ([n][heads][d], doubles) into sequence i of `state` (cache.state()), K (t 0) or V (t 1)."""
    b, s = state[t], state[2 + t]
    n, q8, page = x.shape[0], cache.q8, cache.page
    at = cache.at(i, n).cuda()
    for r0 in range(a // page * page, n, page):
        if max(a, r0) >= min(n, r0 + page):
            continue
        fresh, p = x[max(a, r0):min(n, r0 + page)].double(), int(at[r0]) // page
        new, old = at[max(a, r0):min(n, r0 + page)], at[r0:max(a, r0)]
        for h in range(cache.K):
            y = fresh[:, h]
            top = float(torch.where(torch.isfinite(y), y.abs(), 0.0).max())
            sc = scale64(top, q8)
            if len(old):
                was = float(s[p, h])
                if was < sc:
                    v = b[old, h].view(TORCH8[q8]).float().double()
                    b[old, h] = bytes_of(round8(v * was / sc, q8), q8)
                sc = max(sc, was)
            b[new, h] = bytes_of(round8(y / sc, q8), q8)
            s[p, h] = sc


def decode64(cache, q, scale=None, bf16_out=False):
    """Per sequence: out and its tolerance before the output's rounding, over what the cache holds."""
    n_seq, H, d = q.shape
    G = H // cache.K
    scale = scale or 1.0 / math.sqrt(d)
    out = torch.zeros((n_seq, H, d), dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    # q's own rounding, relative to its head's largest element: f32 keeps 22 bits of it, 16-bit types lose what is
    # 2^-39 of it
    part = 2.0 ** -22 if q.dtype == torch.float32 else 2.0 ** -38
    for i, n in enumerate(cache.lens):
        if n == 0:
            continue
        k, v = cache.seq(i)
        for h in range(cache.K):
            qq = q[i, h * G:(h + 1) * G]
            p, mag = softmax64(qq, k[:, h], scale)
            lost = float((qq.double().abs().amax(1) * part).max() * k[:, h].abs().sum(1).max() * scale)
            # numerator and denominator each carry one score error; a unit's sum of 32 and the sums over units (in f32)
            # cut at most a step each.  Weights (times V's scale) are two f16: 2^-22 of themselves, and no finer than
            # half of f16's smallest step, 2^-25, where the largest is 2^14 at least: n times 2^-39 of the largest
            # meets bytes of at most TOP.  For bf16 outputs of 16-bit models they are one f16: half a step, 2^-11
            e = 2 * (score_error(mag, d) + lost)
            out[i, h * G:(h + 1) * G] = p @ v[:, h]
            vs = cache.vs[cache.at(i, n).cuda() // cache.page, h].double()
            tol[i, h * G:(h + 1) * G] = ((p @ v[:, h].abs()) * (e + (2.0 ** -11 if bf16_out else 2.0 ** -21) + (64 + n / 32) * 2.0 ** -23)
                                         + n * 2.0 ** -39 * TOP[cache.q8] * (p * vs).amax(1, keepdim=True))
    return out, tol


# --------------------------------------------------------------------- blocks
class Book:
    """Sequences, tables and counts as plain lists, and the contents of one pool."""

    def __init__(self, lens, tables, refs, block_rows, pool):
        self.lens, self.tables, self.refs = list(lens), [list(t) for t in tables], list(refs)
        self.B, self.pool = block_rows, list(pool)

    def held(self, n):
        return -(-n // self.B)

    def fork(self, parents, lens=None):
        was, tables = list(self.lens), [list(t) for t in self.tables]
        for s, p in enumerate(parents):
            if not -1 <= p < len(was):
                continue
            have = 0 if p < 0 else was[p]
            n = have if lens is None else lens[s]
            if not 0 <= n <= have:
                continue
            for i in range(self.held(was[s])):
                self.refs[tables[s][i]] -= 1
            for i in range(self.held(n)):
                self.tables[s][i] = tables[p][i]
                self.refs[tables[p][i]] += 1
            self.lens[s] = n

    def resize(self, lens):
        """False, and nothing changed, where the free blocks do not do."""
        refs, tables, pool = list(self.refs), [list(t) for t in self.tables], list(self.pool)
        room = len(self.tables[0]) * self.B
        lens = [n if 0 <= n <= room else was for n, was in zip(lens, self.lens)]
        for s, (was, n) in enumerate(zip(self.lens, lens)):
            for i in range(self.held(n), self.held(was)):
                refs[tables[s][i]] -= 1
        grow = {}
        for s, (was, n) in enumerate(zip(self.lens, lens)):
            if n > was and was % self.B and refs[tables[s][was // self.B]] > 1:
                grow.setdefault(tables[s][was // self.B], []).append(s)
        copies = set()
        for b, who in grow.items():
            copies |= set(who[:-1] if len(who) == refs[b] else who)
        free = [b for b, r in enumerate(refs) if r == 0]
        need = len(copies) + sum(max(0, self.held(n) - self.held(was)) for was, n in zip(self.lens, lens))
        if need > len(free):
            return False
        for s, (was, n) in enumerate(zip(self.lens, lens)):
            if s in copies:
                b, to = tables[s][was // self.B], free.pop(0)
                tables[s][was // self.B], refs[to], pool[to] = to, 1, self.pool[b]
                refs[b] -= 1
            for i in range(self.held(was), self.held(n)):
                tables[s][i] = free.pop(0)
                refs[tables[s][i]] = 1
        self.refs, self.tables, self.pool, self.lens = refs, tables, pool, lens
        return True

    def compact(self):
        used = sum(r > 0 for r in self.refs)
        src = [b for b, r in enumerate(self.refs) if r > 0 and b >= used]
        dst = [b for b, r in enumerate(self.refs) if r <= 0 and b < used]
        to = dict(zip(src, dst))
        for s, n in enumerate(self.lens):
            for i in range(self.held(n)):
                self.tables[s][i] = to.get(self.tables[s][i], self.tables[s][i])
        for a, b in to.items():
            self.refs[b], self.refs[a], self.pool[b] = self.refs[a], 0, self.pool[a]
        return used

    def check(self):
        """The counts are those of the tables."""
        refs = [0] * len(self.refs)
        for s, n in enumerate(self.lens):
            for i in range(self.held(n)):
                refs[self.tables[s][i]] += 1
        return refs == self.refs
