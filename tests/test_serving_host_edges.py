"""Further refusals of the cache-serving entry points, on the host: pointers and sizes that a kernel could not follow."""
import pytest

import epsp
from test_serving_host import I, PTR, decode, desc, dst, evict, make


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
