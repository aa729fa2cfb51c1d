"""Argument checks of the 8-bit cache's entry points and of those that manage blocks, on the host: every refused call
returns before anything reaches a device, so plain numbers stand in for the device pointers."""
import ctypes

import pytest
import torch

import epsp
from test_serving_host import BAD_BATCH, I, PTR, desc, make

BIG = 1 << 40


def cache(**kw):
    d = dict(type=epsp.E4M3, k=5 * PTR, v=6 * PTR, k_scale=7 * PTR, v_scale=8 * PTR)
    d.update(kw)
    return epsp.Kv8Desc(**d)


def ref(d):
    return ctypes.byref(d) if d is not None else None


def decode8(c, kv, c8, **kw):
    a = dict(layer=0, q=PTR, k_new=None, v_new=None, out=PTR, ws=PTR, n=BIG)
    a.update(kw)
    return epsp.lib.ep_sp_decode8_layer(c.h, a["layer"], ref(kv), a["q"], a["k_new"], a["v_new"], ref(c8), a["out"],
                                        a["ws"], a["n"], None)


def pack(c, src, dst, c8, back=False, **kw):
    a = dict(layer=0, k=PTR, v=2 * PTR, first=None)
    a.update(kw)
    if back:
        return epsp.lib.ep_sp_unpack_kv(c.h, a["layer"], ref(src), ref(c8), a["first"], ref(dst), a["k"], a["v"], None)
    return epsp.lib.ep_sp_pack_kv(c.h, a["layer"], ref(src), a["k"], a["v"], a["first"], ref(dst), ref(c8), None)


BAD_CACHE = [dict(type=0), dict(type=5), dict(k=None), dict(v=None), dict(k_scale=None), dict(v_scale=None),
             dict(k=5 * PTR + 8), dict(v=6 * PTR + 4), dict(k_scale=7 * PTR + 2), dict(v_scale=8 * PTR + 1),
             dict(v=5 * PTR), dict(v_scale=7 * PTR)]


@pytest.mark.parametrize("bad", BAD_BATCH, ids=str)
def test_bad_batches(bad):
    c = make()
    assert decode8(c, desc(**bad), cache()) == I and c.last_error().startswith("decode8: ")
    assert pack(c, desc(**bad), desc(), cache()) == I and c.last_error().startswith("pack source: ")
    assert pack(c, desc(**bad), desc(), cache(), True) == I and c.last_error().startswith("unpack source: ")
    if "kv_lens" not in bad:  # (a destination's are not read)
        assert pack(c, desc(), desc(**bad), cache()) == I
        assert pack(c, desc(), desc(**bad), cache(), True) == I


@pytest.mark.parametrize("bad", BAD_CACHE, ids=str)
def test_bad_caches(bad):
    c = make()
    assert decode8(c, desc(), cache(**bad)) == I and c.last_error().startswith("decode8: ")
    assert pack(c, desc(), desc(), cache(**bad)) == I and pack(c, desc(), desc(), cache(**bad), True) == I


@pytest.mark.parametrize("bad", [dict(layer=-1), dict(layer=2), dict(q=None), dict(out=None), dict(k_new=PTR),
                                 dict(v_new=PTR), dict(q=PTR + 8), dict(out=PTR + 4), dict(k_new=PTR + 8, v_new=PTR),
                                 dict(ws=PTR + 8)], ids=str)
def test_decode8_refuses_bad_arguments(bad):
    c = make()
    assert decode8(c, desc(), cache(), **bad) == I and c.last_error()


def test_decode8_workspace_and_missing_parts():
    c = make()
    need = c.decode8_bytes(3, 1000)
    assert decode8(c, desc(), cache(), n=need - 1) == I or need <= 16
    assert decode8(c, None, cache()) == I and decode8(c, desc(), None) == I
    assert epsp.lib.ep_sp_decode8_layer(None, 0, ref(desc()), PTR, None, None, ref(cache()), PTR, PTR, BIG, None) == I
    n = ctypes.c_size_t()
    for bad in ((0, 10), (3, 0), (3, 4097), (70000, 10)):
        assert epsp.lib.ep_sp_decode8_bytes(c.h, *bad, ctypes.byref(n)) == I
    assert epsp.lib.ep_sp_decode8_bytes(c.h, 1, 10, None) == I
    long = make(max_ctx=2 ** 31 - 1, n_head=1, n_head_kv=1)
    assert epsp.lib.ep_sp_decode8_bytes(long.h, 65535, 1 << 30, ctypes.byref(n)) == I  # more units than 32 bits count


@pytest.mark.parametrize("back", [False, True], ids=["pack", "unpack"])
def test_pack_refuses(back):
    c = make()
    for bad in (dict(layer=-1), dict(layer=2), dict(k=None), dict(v=None), dict(k=PTR + 8), dict(v=2 * PTR + 2),
                dict(first=PTR + 2), dict(k=5 * PTR), dict(v=6 * PTR)):
        assert pack(c, desc(), desc(), cache(), back, **bad) == I, bad
    assert pack(c, desc(), desc(n_seq=2), cache(), back) == I and "differ" in c.last_error()
    assert pack(c, desc(), desc(table_stride=31), cache(), back) == I
    assert pack(c, None, desc(), cache(), back) == I and pack(c, desc(), None, cache(), back) == I
    assert pack(c, desc(), desc(), None, back) == I
    # a page has one scale: sequences without blocks begin at whole pages of the 8-bit cache, not of the other
    flat = dict(block_rows=0, block_tables=None)
    odd, even = desc(**flat, seq_rows=1001), desc(**flat, seq_rows=1024)
    assert pack(c, *((odd, even) if back else (even, odd)), cache(), back) == I and "page" in c.last_error()
    assert decode8(c, odd, cache()) == I and "page" in c.last_error()
    if back:
        assert pack(c, desc(), desc(), cache(), back, k=PTR, v=PTR) == I and "same rows" in c.last_error()


def pages(**kw):
    d = dict(n_seq=3, table_stride=8, block_rows=32, pool_blocks=20, kv_lens=PTR, block_tables=2 * PTR, refs=3 * PTR)
    d.update(kw)
    return epsp.PagesDesc(**d)


BAD_PAGES = [dict(n_seq=0), dict(n_seq=65536), dict(table_stride=0), dict(block_rows=0), dict(block_rows=48),
             dict(block_rows=-32), dict(pool_blocks=0), dict(pool_blocks=2 ** 31 - 1), dict(kv_lens=None),
             dict(block_tables=None), dict(refs=None), dict(kv_lens=PTR + 2), dict(block_tables=PTR + 1),
             dict(refs=PTR + 3), dict(table_stride=2 ** 27),
             dict(n_seq=65535, table_stride=32769)]  # the blocks wanted would not fit 32 bits


def calls(c, p, **kw):
    a = dict(parents=4 * PTR, lens=None, new=4 * PTR, pool=(epsp.PoolDesc * 1)(epsp.PoolDesc(PTR, 1024)), n_pools=1,
             used=None, ws=PTR, n=BIG)
    a.update(kw)
    r = ref(p)
    return [epsp.lib.ep_sp_fork_seqs(c.h, r, a["parents"], a["lens"], a["ws"], a["n"], None),
            epsp.lib.ep_sp_resize_seqs(c.h, r, a["new"], a["pool"], a["n_pools"], a["ws"], a["n"], None),
            epsp.lib.ep_sp_compact_pool(c.h, r, a["pool"], a["n_pools"], a["used"], a["ws"], a["n"], None)]


@pytest.mark.parametrize("bad", BAD_PAGES, ids=str)
def test_bad_pages(bad):
    c = make()
    p = pages(**bad)
    assert calls(c, p) == [I] * 3
    assert epsp.lib.ep_sp_count_refs(c.h, ref(p), None) == I and c.last_error().startswith("count: ")
    n = ctypes.c_size_t()
    for f in (epsp.lib.ep_sp_fork_bytes, epsp.lib.ep_sp_resize_bytes, epsp.lib.ep_sp_compact_bytes):
        assert f(c.h, ref(p), ctypes.byref(n)) == I


def test_page_calls_refuse_bad_arguments():
    c = make()
    p = pages()
    assert calls(c, None) == [I] * 3 and epsp.lib.ep_sp_count_refs(c.h, None, None) == I
    assert epsp.lib.ep_sp_count_refs(None, ref(p), None) == I
    assert calls(c, p, parents=None, new=None, pool=None) == [I] * 3
    assert calls(c, p, parents=PTR + 2, new=PTR + 1, used=PTR + 2) == [I] * 3
    assert calls(c, p, lens=PTR + 2, n_pools=0) == [I] * 3
    assert calls(c, p, lens=PTR + 2, n_pools=4097) == [I] * 3
    assert calls(c, p, ws=None) == [I] * 3 and calls(c, p, ws=PTR + 4) == [I] * 3 and calls(c, p, n=8) == [I] * 3
    for bad in ((None, 64), (PTR, 0), (PTR, 6), (PTR + 2, 64), (PTR, 1 << 62)):
        pool = (epsp.PoolDesc * 1)(epsp.PoolDesc(*bad))
        assert calls(c, p, pool=pool)[1:] == [I] * 2 and "pool 0" in c.last_error()
    n = ctypes.c_size_t()
    for f, lo in ((epsp.lib.ep_sp_fork_bytes, 3 * 8 * 4), (epsp.lib.ep_sp_resize_bytes, 20 * 4),
                  (epsp.lib.ep_sp_compact_bytes, 20 * 4)):
        assert f(c.h, ref(p), ctypes.byref(n)) == epsp.OK and n.value >= lo
        assert f(None, ref(p), ctypes.byref(n)) == I and f(c.h, ref(p), None) == I


def test_family_bounds():
    c = make()
    ms, n = ctypes.c_double(), ctypes.c_int64()
    for f in (-1, 11):
        assert epsp.lib.ep_sp_profile_read_family(c.h, f, ctypes.byref(ms), ctypes.byref(n)) == I
    assert c.profile_family(epsp.FAMILY_PACK) == (0.0, 0) and c.profile_family(epsp.FAMILY_PAGES) == (0.0, 0)


def test_binding_refuses_what_a_pointer_cannot_show():
    c = make()
    k = torch.zeros((320, 2, 64), dtype=torch.int8)
    s = torch.zeros((10, 2))
    with pytest.raises(ValueError, match="8-bit"):
        epsp.Kv8(k.to(torch.uint8), k.to(torch.uint8), s, s)
    with pytest.raises(ValueError):
        epsp.Kv8(k, k[:-1], s, s)
    with pytest.raises(ValueError):
        epsp.Kv8(k, k, s, s[:, :1])
    with pytest.raises(ValueError):
        epsp.Kv8(k, k, s.double(), s)
    kv = epsp.KvBatch(None, 100, seq_rows=96, n_seq=3)
    q = torch.zeros((3, 8, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="not on cuda"):
        c.decode8_layer(0, kv, q, epsp.Kv8(k, k, s, s), q, None)
    with pytest.raises(ValueError):
        epsp.Pages(torch.zeros(3, dtype=torch.int64), torch.zeros((3, 4), dtype=torch.int32),
                   torch.zeros(9, dtype=torch.int32), 32)
    with pytest.raises(ValueError, match="no pools"):
        epsp.Pools([], 10)
    with pytest.raises(ValueError, match="whole 4-byte"):
        epsp.Pools([torch.zeros(10, 3, dtype=torch.int8)], 10)
    with pytest.raises(ValueError, match="contiguous"):
        epsp.Pools([torch.zeros(10, 8).T], 8)
