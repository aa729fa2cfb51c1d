"""Argument checks of the cache-serving entry points (decode, prompt weights, eviction), on the host: every refused
call returns before anything reaches a device, so plain numbers stand in for the device pointers."""
import ctypes

import pytest
import torch

import epsp

I = epsp.INVALID_ARGUMENT
PTR = 1 << 20  # a 16-byte aligned number


def make(**kw):
    args = dict(n_layer=2, n_head=8, n_head_kv=2, head_dim=64, dtype=epsp.BF16, max_ctx=4096, page_size=32)
    args.update(kw)
    return epsp.Context(**args)


def desc(**kw):
    d = dict(n_seq=3, max_kv_len=1000, kv_lens=PTR, block_tables=PTR, table_stride=32, block_rows=32, pool_rows=3200,
             seq_rows=0)
    d.update(kw)
    return epsp.KvBatchDesc(**d)


BAD_BATCH = [dict(n_seq=0), dict(n_seq=-1), dict(n_seq=70000), dict(max_kv_len=0), dict(max_kv_len=4097),
             dict(kv_lens=None), dict(block_tables=None), dict(block_rows=48), dict(block_rows=-32),
             dict(table_stride=31), dict(table_stride=0), dict(pool_rows=0), dict(pool_rows=3201),
             dict(block_rows=0, seq_rows=999), dict(block_rows=0, seq_rows=-5),
             dict(block_rows=0, seq_rows=1 << 30)]


def decode(c, kv, need=None, **kw):
    a = dict(layer=0, q=PTR, k_new=None, v_new=None, k=PTR, v=PTR, out=PTR, acc=None, stride=0, ws=PTR,
             n=1 << 40)
    a.update(kw)
    return epsp.lib.ep_sp_decode_layer(c.h, a["layer"], ctypes.byref(kv) if kv else None, a["q"], a["k_new"],
                                       a["v_new"], a["k"], a["v"], a["out"], a["acc"], a["stride"], a["ws"], a["n"],
                                       None)


@pytest.mark.parametrize("bad", BAD_BATCH, ids=str)
def test_decode_refuses_bad_batches(bad):
    c = make()
    assert decode(c, desc(**bad)) == I
    assert c.last_error().startswith("decode: ")


@pytest.mark.parametrize("bad", [dict(layer=-1), dict(layer=2), dict(q=None), dict(k=None), dict(v=None),
                                 dict(out=None), dict(k_new=PTR), dict(v_new=PTR), dict(q=PTR + 8), dict(k=PTR + 4),
                                 dict(v=PTR + 2), dict(out=PTR + 8), dict(k_new=PTR + 8, v_new=PTR),
                                 dict(acc=PTR, stride=999), dict(acc=PTR + 2, stride=1000), dict(ws=PTR + 8)], ids=str)
def test_decode_refuses_bad_arguments(bad):
    c = make()
    assert decode(c, desc(), **bad) == I
    assert c.last_error()


def test_decode_refuses_a_missing_batch_context_or_workspace():
    c = make()
    assert decode(c, None) == I
    assert epsp.lib.ep_sp_decode_layer(None, 0, ctypes.byref(desc()), PTR, None, None, PTR, PTR, PTR, None, 0, PTR,
                                       1 << 30, None) == I
    need = c.decode_bytes(3, 1000, True)
    assert need >= 3 * 8 * 1000 * 4  # the scores of every query head and row
    assert decode(c, desc(), acc=PTR, stride=1000, n=need - 1) == I
    assert decode(c, desc(), acc=PTR, stride=1000, ws=None) == I
    n = ctypes.c_size_t()
    for bad in ((0, 10, 0), (3, 0, 0), (3, 4097, 0), (3, 10, 2), (70000, 10, 0)):
        assert epsp.lib.ep_sp_decode_bytes(c.h, *bad, ctypes.byref(n)) == I
    assert epsp.lib.ep_sp_decode_bytes(None, 1, 10, 0, ctypes.byref(n)) == I
    assert epsp.lib.ep_sp_decode_bytes(c.h, 1, 10, 0, None) == I


def prompt(c, **kw):
    a = dict(layer=0, q=PTR, k=PTR, kv_len=1000, n_tok=100, row_begin=40, accumulate=0, acc=PTR, stride=1000, ws=PTR,
             n=1 << 40)
    a.update(kw)
    return epsp.lib.ep_sp_prompt_weights(c.h, a["layer"], a["q"], a["k"], a["kv_len"], a["n_tok"], a["row_begin"],
                                         a["accumulate"], a["acc"], a["stride"], a["ws"], a["n"], None)


@pytest.mark.parametrize("bad", [dict(layer=2), dict(q=None), dict(k=None), dict(acc=None), dict(q=PTR + 8),
                                 dict(k=PTR + 8), dict(acc=PTR + 1), dict(kv_len=99), dict(kv_len=4097),
                                 dict(n_tok=0), dict(row_begin=-1), dict(row_begin=100), dict(accumulate=2),
                                 dict(stride=999), dict(n=0), dict(ws=None), dict(ws=PTR + 4)], ids=str)
def test_prompt_weights_refuses_bad_arguments(bad):
    c = make()
    assert prompt(c, **bad) == I
    assert c.last_error()


def test_prompt_weights_refuses_a_short_block_table():
    c = make()
    table = torch.zeros(10, dtype=torch.int32)
    c.check(c.set_paged_kv(32, table, 10, 3200))
    assert prompt(c) == I  # 10 blocks of 32 rows do not cover 1000
    n = ctypes.c_size_t()
    for bad in ((99, 100, 0), (4097, 1, 0), (10, 0, 0), (10, 5, 5), (10, 5, -1)):
        assert epsp.lib.ep_sp_prompt_weights_bytes(c.h, *bad, ctypes.byref(n)) == I


def evict(c, src, dst, **kw):
    a = dict(layer=0, k=PTR, v=2 * PTR, acc=PTR, stride=1000, n_keep=100, sink=4, recent=30, k_dst=3 * PTR,
             v_dst=4 * PTR, acc_dst=None, dst_stride=0, new_lens=None, kept=None, ws=PTR, n=1 << 40)
    a.update(kw)
    ref = lambda d: ctypes.byref(d) if d else None  # noqa: E731
    return epsp.lib.ep_sp_evict_layer(c.h, a["layer"], ref(src), a["k"], a["v"], a["acc"], a["stride"], a["n_keep"],
                                      a["sink"], a["recent"], ref(dst), a["k_dst"], a["v_dst"], a["acc_dst"],
                                      a["dst_stride"], a["new_lens"], a["kept"], a["ws"], a["n"], None)


def dst(**kw):
    return desc(**{**dict(max_kv_len=100, kv_lens=None, block_tables=2 * PTR, table_stride=4), **kw})


@pytest.mark.parametrize("bad", BAD_BATCH, ids=str)
def test_evict_refuses_bad_sources(bad):
    c = make()
    assert evict(c, desc(**bad), dst()) == I
    assert "source" in c.last_error()


@pytest.mark.parametrize("bad", [dict(n_seq=2), dict(max_kv_len=99), dict(table_stride=3), dict(block_tables=None),
                                 dict(block_rows=0, seq_rows=99), dict(block_rows=40)], ids=str)
def test_evict_refuses_bad_destinations(bad):
    c = make()
    assert evict(c, desc(), dst(**bad)) == I
    assert c.last_error()


@pytest.mark.parametrize("bad", [dict(layer=2), dict(n_keep=0), dict(n_keep=4097), dict(sink=-1), dict(recent=-1),
                                 dict(sink=71), dict(sink=1 << 30, recent=1 << 30), dict(k=None), dict(v=None),
                                 dict(acc=None), dict(k_dst=None), dict(v_dst=None), dict(k=PTR + 8),
                                 dict(v_dst=4 * PTR + 2), dict(stride=999), dict(acc_dst=PTR + 8, dst_stride=99),
                                 dict(acc_dst=PTR, dst_stride=500), dict(n=0), dict(ws=None), dict(ws=PTR + 2),
                                 dict(k_dst=PTR), dict(v_dst=2 * PTR), dict(k_dst=2 * PTR), dict(v_dst=PTR)], ids=str)
def test_evict_refuses_bad_arguments(bad):
    c = make()
    assert evict(c, desc(), dst(), **bad) == I
    assert c.last_error()


def test_evict_in_place_needs_the_same_layout():
    c = make()
    flat = dict(block_rows=0, seq_rows=1000, block_tables=None)
    # the same tensors under another contiguous stride, or as pool and as plain rows
    assert evict(c, desc(**flat), dst(**{**flat, "seq_rows": 500}), k_dst=PTR, v_dst=2 * PTR) == I
    assert evict(c, desc(), dst(**flat), k_dst=PTR, v_dst=2 * PTR) == I
    # the same table read with another stride
    assert evict(c, desc(), dst(block_tables=PTR, table_stride=4), k_dst=PTR, v_dst=2 * PTR) == I
    assert evict(c, None, dst()) == I and evict(c, desc(), None) == I


def test_families_bounds():
    c = make()
    ms, n = (ctypes.c_double * 9)(), (ctypes.c_int64 * 9)()
    assert epsp.lib.ep_sp_profile_read_families(c.h, 10, ms, n) == I
    assert epsp.lib.ep_sp_profile_read_families(c.h, 0, ms, n) == I
    assert epsp.lib.ep_sp_profile_read_families(c.h, 9, ms, n) == epsp.OK
    assert set(c.profile_families()) == set(epsp.FAMILY_NAMES)


def test_binding_refuses_what_a_pointer_cannot_show():
    c = make()
    lens = torch.zeros(3, dtype=torch.int64)
    with pytest.raises(ValueError):
        epsp.KvBatch(lens, 100, seq_rows=100)
    with pytest.raises(ValueError):
        epsp.KvBatch(None, 100, seq_rows=100)
    kv = epsp.KvBatch(None, 100, seq_rows=100, n_seq=3)
    q = torch.zeros((3, 8, 64), dtype=torch.bfloat16)
    k = torch.zeros((300, 2, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="is on cpu"):
        c.decode_layer(0, kv, q, k, k, q, None)
    with pytest.raises(ValueError, match="torch.float32"):
        c.decode_layer(0, kv, q, k.float(), k, q, None)
    with pytest.raises(ValueError, match="not contiguous"):
        c.decode_layer(0, kv, q, k.transpose(0, 1), k, q, None)
