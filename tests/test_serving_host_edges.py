"""Further refusals of the cache-serving entry points, on the host: pointers and sizes that a kernel could not follow."""
import ctypes

import pytest

import epsp
from test_serving_host import I, PTR, decode, desc, dst, evict, make, prompt


@pytest.mark.parametrize("bad", [dict(kv_lens=PTR + 2), dict(block_tables=PTR + 1)], ids=str)
def test_lengths_and_tables_off_their_alignment_are_refused(bad):
    c = make()
    assert decode(c, desc(**bad)) == I and "aligned" in c.last_error()
    assert evict(c, desc(**bad), dst()) == I and "aligned" in c.last_error()
    if "block_tables" in bad:
        assert evict(c, desc(), dst(**bad)) == I and "aligned" in c.last_error()


@pytest.mark.parametrize("bad", [dict(new_lens=PTR + 2), dict(kept=PTR + 3)], ids=str)
def test_outputs_of_an_eviction_off_their_alignment_are_refused(bad):
    c = make()
    assert evict(c, desc(), dst(), **bad) == I and "aligned" in c.last_error()


def test_k_and_v_into_the_same_rows_is_refused():
    c = make()
    assert evict(c, desc(), dst(), k_dst=3 * PTR, v_dst=3 * PTR) == I and "same rows" in c.last_error()


def test_lengths_that_32_bits_cannot_round_up_are_refused():
    """A block table may name a small pool's blocks again and again, so such a length needs no such cache."""
    top = 2 ** 31 - 1
    c = make(max_ctx=top, n_layer=1, n_head=1, n_head_kv=1)
    long = dict(n_seq=1, max_kv_len=top, table_stride=1 << 20, block_rows=2048, pool_rows=2048)
    assert decode(c, desc(**long)) == I and "32 bits" in c.last_error()
    assert evict(c, desc(**long), dst(n_seq=1), stride=top) == I and "32 bits" in c.last_error()
    assert prompt(c, kv_len=top, stride=top) == I
    n = ctypes.c_size_t()
    assert epsp.lib.ep_sp_decode_bytes(c.h, 1, top, 0, ctypes.byref(n)) == I
    assert epsp.lib.ep_sp_evict_bytes(c.h, 1, top, 100, ctypes.byref(n)) == I
    assert epsp.lib.ep_sp_prompt_weights_bytes(c.h, top, 1, 0, ctypes.byref(n)) == I
    # what stays under it has a workspace of a plausible size
    assert epsp.lib.ep_sp_decode_bytes(c.h, 1, 1 << 30, 1, ctypes.byref(n)) == epsp.OK and n.value > 4 << 30
    assert epsp.lib.ep_sp_prompt_weights_bytes(c.h, 1 << 30, 1, 0, ctypes.byref(n)) == epsp.OK and n.value > 0
