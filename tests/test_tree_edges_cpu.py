"""Host side of the tree-decoding parts at the edges: pages of the cache that no
sequence has, rotary scalings, sizes that the C entry points refuse."""
from __future__ import annotations

import ctypes
import math
import os

import pytest
import torch

from spark_b200 import _lib, rotary
from spark_b200.tree_decode import PagedKVCache

from test_tree_decode_cpu import P, attention, cache


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


@pytest.mark.parametrize("rot,base,original", [(128, 10000.0, 65536), (128, 10000.0, 1 << 20), (64, 10000.0, 131072), (64, 500000.0, 4096)])
def test_yarn_blends_every_pair_between_its_limits(rot, base, original):
    """Also where even the last pair turns more than `slow` times: it is not divided by
    the whole factor then."""
    factor, fast, slow = 8.0, 32.0, 1.0
    f, _ = rotary.rope_frequencies(rot, base)
    yarn, _ = rotary.rope_frequencies(rot, base, scaling="yarn", factor=factor, original_positions=original, fast=fast, slow=slow)
    turns = f * original / (2 * math.pi)
    # the pair's index (a real number) where a frequency turns n times
    at = [rot / 2 * math.log(original / (2 * math.pi * n)) / math.log(base) for n in (fast, slow)]
    lo, hi = math.floor(at[0]), math.ceil(at[1])
    assert lo >= 0 and hi < rot
    blend = ((torch.arange(rot // 2, dtype=torch.float64) - lo) / (hi - lo)).clamp(0, 1)
    assert torch.allclose(yarn, f * (1 - blend) + f / factor * blend, rtol=1e-12)
    kept = yarn / f
    assert (kept[turns > slow * 1.5] > 1 / factor).all() and (kept[:-1] >= kept[1:]).all()


def test_append_refuses_rows_of_two_to_the_31_values():
    st = (ctypes.c_int64 * 3)(1, 1, 1)
    for heads, dim in ((65535, 65535), (65535, 32769)):
        c = cache(kv_heads=heads, head_dim=dim)
        rc = _lib.lib().spark_kv_append(ctypes.byref(c), 1, 1, P(256), st, P(256), st, None, 1, None, P(512), None, None)
        assert rc == _lib.ERR_INVALID
        assert "cache size" in _lib.last_error()


@pytest.mark.parametrize("scale", [0.0, -0.1, 1e-46, 9e-31, 2e30, math.inf, math.nan])
def test_attention_refuses_scales_that_fp32_does_not_hold(scale):
    """A scale that is 0 in fp32 would make a NaN of a masked score."""
    a = attention(scale=scale)
    assert _lib.lib().spark_tree_attention_workspace_size(ctypes.byref(a)) == 0
    assert _lib.lib().spark_tree_attention(ctypes.byref(a), P(1 << 20), 1 << 30, None) == _lib.ERR_INVALID
    assert "scale" in _lib.last_error()


def test_attention_refuses_strides_of_zero():
    """A tensor map takes none; the extents of 1 have no stride."""
    def run(**kw):
        a = attention(cache(**{n: v for n, v in kw.items() if n in ("k_stride", "v_stride")}), batch=2)
        for n, v in kw.items():
            if n in ("k_stride", "v_stride"):
                continue
            setattr(a, n, v)
        return _lib.lib().spark_tree_attention(ctypes.byref(a), P(1 << 20), 1 << 30, None)

    three = ctypes.c_int64 * 3
    for name in ("q_stride", "kn_stride", "vn_stride", "out_stride", "k_stride", "v_stride"):
        for at in range(3):
            st = [1024, 256, 64]
            st[at] = 0
            assert run(**{name: three(*st)}) == _lib.ERR_ALIGNMENT, (name, at)
            assert "strides" in _lib.last_error()


def test_outputs_that_share_their_rows_are_refused():
    def turn(x, y, ys=(512, 128, 64), heads=2, x2=None, y2=None):
        q, k = _lib.SparkRopeHeads(x=x, y=y, heads=heads), _lib.SparkRopeHeads(x=x2, y=y2, heads=heads)
        for h in (q, k):
            h.xs[:], h.ys[:] = (512, 128, 64), ys
        return _lib.lib().spark_rope(ctypes.byref(q), ctypes.byref(k) if x2 else None, 1, 2, 4, 64, 32, 0, 0, P(256), 8, P(256), 10,
                                     None, None)

    for ys in ((0, 128, 64), (512, 0, 64), (512, 128, 0)):
        assert turn(1 << 20, 1 << 21, ys) == _lib.ERR_INVALID and "spark_rope: output rows" in _lib.last_error()
    a, b, c = 1 << 20, 1 << 21, 1 << 22
    for x, y, x2, y2 in ((a, b, b, a), (a, b, b, c), (a, a, b, a), (a, c, b, c)):
        assert turn(x, y, x2=x2, y2=y2) == _lib.ERR_INVALID and "the other's" in _lib.last_error()
    st, three = (ctypes.c_int64 * 3)(256, 128, 64), ctypes.c_int64 * 3
    for name in ("k_stride", "v_stride"):
        for at in range(3):
            bad = [2048, 128, 64]
            bad[at] = 0
            rc = _lib.lib().spark_kv_append(ctypes.byref(cache(**{name: three(*bad)})), 1, 2, P(256), st, P(256), st, None, 2, None,
                                            P(512), None, None)
            assert rc == _lib.ERR_INVALID and "rows of the cache" in _lib.last_error()


def test_the_zeroed_part_of_a_workspace_is_the_header_s():
    header = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "spark_b200.h")).read()
    assert f"#define SPARK_TREE_ATTENTION_ZEROED {_lib.TREE_ATTENTION_ZEROED}\n" in header
    assert _lib.lib().spark_tree_attention_workspace_size(ctypes.byref(attention())) > _lib.TREE_ATTENTION_ZEROED
