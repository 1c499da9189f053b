"""Host side of the tree-decoding parts at the edges: pages of the cache that no
sequence has, rotary scalings, sizes that the C entry points refuse."""
from __future__ import annotations

import ctypes

from spark_b200 import _lib
from spark_b200.tree_decode import PagedKVCache


def test_a_page_is_in_one_sequence_only():
    c = PagedKVCache(1, 3, 64, 1, 64, page_size=16, pages=6, device="cpu")
    assert (c.page_table == -1).all() and c.held.tolist() == [0, 0, 0]
    c.reserve(0, 33)
    c.reserve(1, 16)
    assert c.held.tolist() == [1, 1, 0]
    c.release(0)
    c.reserve(1, 30)
    c.reserve(2, 40)
    assert c.held.tolist() == [0, 1, 1]
    assert (c.page_table[0] == -1).all() and (c.page_table[1, 2:] == -1).all() and (c.page_table[2, 3:] == -1).all()
    named = c.page_table[c.page_table >= 0].tolist()
    assert len(named) == 5 == len(set(named)) and not set(named) & set(c._free)
    c.release(1)
    c.release(2)
    assert sorted(c._free) == list(range(6)) and (c.page_table == -1).all() and c.held.tolist() == [0, 0, 0]


def test_capture_mode_refuses_other_modes():
    for mode in (None, -1, 3):
        m = ctypes.c_int(mode or 0)
        assert _lib.lib().spark_capture_mode(None if mode is None else ctypes.byref(m)) == _lib.ERR_INVALID
        assert "spark_capture_mode" in _lib.last_error()
