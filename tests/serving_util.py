"""Plain 64-bit forms of the cache-serving operators, and the caches their tests run on."""
from __future__ import annotations

import math

import torch

import epsp
import workloads as W

TORCH = W.TORCH_DTYPE


class Cache:
    """K/V rows of a batch of sequences, contiguous or scattered over a shuffled pool of blocks.  Every row that no
    sequence holds is NaN."""

    def __init__(self, lens, n_head_kv, d, dtype, block_rows, seed, capacity=None, k=None, v=None):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.B = list(lens), block_rows
        n_seq, cap = len(lens), max(1, capacity or max(lens))
        self.cap = cap
        if block_rows:
            each = -(-cap // block_rows)
            blocks = n_seq * each + 3
            self.table = torch.randperm(blocks, generator=g)[: n_seq * each].view(n_seq, each).to(torch.int32)
            self.rows, self.seq_rows = blocks * block_rows, 0
        else:
            self.table, self.rows, self.seq_rows = None, n_seq * cap, cap
        dt = TORCH[dtype]
        self.k = torch.full((self.rows, n_head_kv, d), float("nan"), dtype=dt)
        self.v = torch.full((self.rows, n_head_kv, d), float("nan"), dtype=dt)
        spread = torch.exp(torch.randn(1, n_head_kv, d, generator=g) * 0.5)
        for i, n in enumerate(lens):
            at = self.at(i, n)
            self.k[at] = (torch.randn(n, n_head_kv, d, generator=g) * spread).to(dt) if k is None else k[i]
            self.v[at] = (torch.randn(n, n_head_kv, d, generator=g) / math.sqrt(d)).to(dt) if v is None else v[i]
        self.k, self.v = self.k.cuda(), self.v.cuda()
        self.d_table = None if self.table is None else self.table.cuda()
        self.d_lens = torch.tensor(self.lens, dtype=torch.int32).cuda()
        self.batch = epsp.KvBatch(self.d_lens, cap, self.d_table, block_rows, self.rows, self.seq_rows)

    def at(self, i, n):
        """Pool rows of the first n rows of sequence i."""
        r = torch.arange(n)
        if self.table is None:
            return i * self.seq_rows + r
        return self.table[i].long()[r // self.B] * self.B + r % self.B

    def seq(self, i, n=None):
        at = self.at(i, self.lens[i] if n is None else n).cuda()
        return self.k[at], self.v[at]


def softmax64(q, k, scale):
    """(weights, sum |q_i k_i| scale) of rows q [m][d] over keys k [n][d], in 64 bits."""
    q, k = q.double(), k.double()
    x = q @ k.T * scale
    return torch.softmax(x, dim=-1), q.abs() @ k.abs().T * scale


def score_error(mag, d):
    """Bound on the error of one score and its exponential, relative to the weight.  A sum of d exact products in f32
    is off by at most d roundings of half a step, and a tensor core may cut instead of rounding (a whole step,
    2^-23) at each of its additions; the scale, the subtraction of the maximum and the exponential itself (2 units in
    the last place, and its argument's rounding) add at most 2^-20 for the |x| < 64 of these tests."""
    return d * 2.0 ** -23 * float(mag.max()) + 2.0 ** -20


def decode64(cache, q, acc=None, k_new=None, v_new=None, scale=None):
    """Per sequence: out, its tolerance before the output's rounding, the acc update and its tolerance."""
    n_seq, H, d = q.shape
    K = cache.k.shape[1]
    G = H // K
    scale = scale or 1.0 / math.sqrt(d)
    out = torch.zeros((n_seq, H, d), dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    add = torch.zeros((n_seq, K, cache.cap), dtype=torch.float64, device="cuda")
    add_tol = torch.zeros_like(add)
    for i, n in enumerate(cache.lens):
        if n == 0:
            continue
        k, v = cache.seq(i)
        if k_new is not None:
            k, v = k.clone(), v.clone()
            k[-1], v[-1] = k_new[i], v_new[i]
        for h in range(K):
            p, mag = softmax64(q[i, h * G:(h + 1) * G], k[:, h], scale)
            # numerator and denominator each carry one score error; weights in 16-bit parts keep 2^-16 of theirs
            e = 2 * score_error(mag, d)
            out[i, h * G:(h + 1) * G] = p @ v[:, h].double()
            tol[i, h * G:(h + 1) * G] = (p @ v[:, h].double().abs()) * (e + 2.0 ** -16)
            add[i, h, :n] = p.sum(0)
            add_tol[i, h, :n] = p.sum(0) * (e + 2.0 ** -20)
    return out, tol, add, add_tol


def rounding(ref, dtype):
    """Half a step of the output type (its smallest subnormal step included)."""
    f = torch.finfo(TORCH[dtype])
    return ref.abs() * (f.eps / 2) + f.smallest_normal * f.eps


def prompt64(q, k, kv_len, n_tok, row_begin, scale=None):
    """acc [n_head_kv][kv_len] and its tolerance of the rows [row_begin, n_tok)."""
    _, H, d = q.shape
    K = k.shape[1]
    G = H // K
    scale = scale or 1.0 / math.sqrt(d)
    acc = torch.zeros((K, kv_len), dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(acc)
    for hq in range(H):
        x = q[row_begin:, hq].double() @ k[:kv_len, hq // G].double().T * scale
        mag = q[row_begin:, hq].double().abs() @ k[:kv_len, hq // G].double().abs().T * scale
        t = torch.arange(kv_len - n_tok + row_begin, kv_len, device="cuda")
        x = x.masked_fill(torch.arange(kv_len, device="cuda")[None, :] > t[:, None], -math.inf)
        p = torch.softmax(x, -1).sum(0)
        acc[hq // G] += p
        # one addition in f32 for each of the rows and heads a key's weights come from
        tol[hq // G] += p * (2 * score_error(mag, d) + (n_tok - row_begin) * G * 2.0 ** -24)
    return acc, tol


def kept64(acc, n, n_keep, sink, recent):
    """Ascending rows one head keeps of n, straight from the definition."""
    if n <= n_keep:
        return list(range(n))
    fixed = set(range(sink)) | set(range(n - recent, n))
    rank = lambda j: -math.inf if math.isnan(acc[j]) else acc[j]  # noqa: E731
    rest = sorted((j for j in range(n) if j not in fixed), key=lambda j: (-rank(j), j))
    return sorted(fixed | set(rest[: n_keep - len(fixed)]))


def context(n_head, n_head_kv, d, dtype, out_dtype, max_ctx, page, n_layer=1, **kw):
    c = epsp.Context(n_layer=n_layer, n_head=n_head, n_head_kv=n_head_kv, head_dim=d, dtype=dtype, out_dtype=out_dtype,
                     max_ctx=max_ctx, page_size=page, device=0, **kw)
    c.check(c.reserve())
    return c


def workspace(n, fill=0xAB):
    """A workspace of exactly n bytes (16-byte aligned) that starts as garbage."""
    return torch.full((max(16, n),), fill, dtype=torch.uint8, device="cuda")
