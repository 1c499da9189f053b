"""Which outputs that share memory norms, sampling and adapters refuse (host side; no pointer
here is one), and the arithmetic behind it against sets of bytes."""
from __future__ import annotations

import ctypes
import os
import random
import subprocess

import pytest

from spark_b200 import _lib
from test_decode_operators_cpu import adapters, norm_rope, sampling

INVALID = _lib.ERR_INVALID
CSRC = os.path.join(os.path.dirname(_lib.LIB_PATH), "csrc")
P = ctypes.c_void_p


@pytest.fixture(scope="module")
def rows(tmp_path_factory):
    """(apart, meet) of rows (address, item, n, [(extent, stride), ...])."""
    where = tmp_path_factory.mktemp("overlap")
    (where / "o.cpp").write_text(f'''#include "{CSRC}/overlap.cuh"
extern "C" bool apart(const spark::Rows* a) {{ return spark::rows_apart(*a); }}
extern "C" bool meet(const spark::Rows* a, const spark::Rows* b) {{ return spark::rows_meet(*a, *b); }}
''')
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", str(where / "o.cpp"), "-o", str(where / "o.so")], check=True)
    lib = ctypes.CDLL(str(where / "o.so"))
    lib.apart.restype = lib.meet.restype = ctypes.c_bool

    class Rows(ctypes.Structure):
        _fields_ = [("at", P), ("item", ctypes.c_int64), ("n", ctypes.c_int64), ("dims", ctypes.c_int), ("extent", ctypes.c_int64 * 3),
                    ("stride", ctypes.c_int64 * 3)]

    def make(r):
        at, item, n, dims = r
        return Rows(at, item, n, len(dims), (ctypes.c_int64 * 3)(*[e for e, _ in dims]), (ctypes.c_int64 * 3)(*[s for _, s in dims]))

    return (lambda a: lib.apart(ctypes.byref(make(a)))), (lambda a, b: lib.meet(ctypes.byref(make(a)), ctypes.byref(make(b))))


def spots(r):
    at, item, n, dims = r
    out = [at]
    for extent, stride in dims:
        out = [p + i * stride * item for p in out for i in range(extent)]
    return [range(p, p + n * item) for p in out]


def test_rows_against_sets_of_bytes(rows):
    apart, meet = rows
    rng = random.Random(1)
    seen = {True: 0, False: 0}
    for _ in range(4000):
        item, n = rng.choice([1, 2, 4]), rng.randint(1, 6)
        dims = [(rng.randint(1, 4), rng.choice([0, 1, 2, 3, 5, 6, 8, 12, 24, -6, -8, 30])) for _ in range(rng.randint(1, 3))]
        a = (10000 + rng.randint(-40, 40) * item, item, n, dims)
        other = [(rng.randint(1, 4), s) for _, s in dims] if rng.random() < 0.7 else \
            [(rng.randint(1, 4), rng.choice([0, 1, 3, 6, 8, 12, -6, 24])) for _ in range(rng.randint(1, 3))]
        b = (10000 + rng.randint(-40, 40) * item, item, rng.randint(1, 6), other)
        bytes_a, bytes_b = ({p for r in spots(v) for p in r} for v in (a, b))
        assert meet(a, b) == bool(bytes_a & bytes_b), (a, b)
        assert meet(b, a) == meet(a, b)
        seen[meet(a, b)] += 1
        if apart(a):
            assert len(bytes_a) == sum(len(r) for r in spots(a)), a
    assert min(seen.values()) > 500


def test_rows_of_parts_of_tensors(rows):
    """What tensors and their views look like: parts of a merged projection, other orders of dimensions, rows with gaps, sizes past 2^32."""
    apart, meet = rows
    b, t, h, d, row = 3, 5, 4, 64, 12 * 64
    q = (1 << 20, 2, d, [(b, t * row), (t, row), (h, d)])
    k = ((1 << 20) + h * d * 2, 2, d, [(b, t * row), (t, row), (2, d)])
    assert apart(q) and apart(k) and not meet(q, k)
    assert meet(q, (q[0] + 2, 2, d, q[3])) and meet(q, (q[0] + row * 2, 2, d, q[3])) and meet(k, (k[0] - d * 2, 2, d, k[3]))
    assert not meet(k, (k[0] + 2 * d * 2, 2, d, k[3]))
    heads_first = (1 << 20, 2, d, [(b, t * h * d), (t, d), (h, t * d)])
    assert apart(heads_first) and meet(heads_first, (1 << 20, 2, d, [(b, t * h * d), (t, h * d), (h, d)]))
    assert apart((0, 4, 10, [(1, 0), (7, 11)])) and not apart((0, 4, 10, [(2, 0), (7, 11)])) and not apart((0, 4, 10, [(7, 9)]))
    far = (0, 4, 409600, [(1 << 23, 409600)])
    assert apart(far) and meet(far, (409600 * 4 * ((1 << 23) - 1), 4, 409600, [(1, 0)]))
    assert not meet(far, (409600 * 4 * (1 << 23), 4, 409600, [(1, 0)]))
    assert not meet((0, 4, 0, [(5, 5)]), (0, 4, 8, [(5, 8)])) and not meet((0, 4, 8, [(0, 5)]), (0, 4, 8, [(5, 8)]))


@pytest.mark.parametrize("part", [
    dict(ys=(512, 128, 63)), dict(ys=(512, 100, 64)), dict(ys=(300, 128, 64)), dict(ys=(64, 128, 64)),     # its own rows
    dict(y=4096 + 2 * 64), dict(y=4096 - 2), dict(y=4096 + 2 * 512), dict(y=4096 + 2000, ys=(640, 160, 80)),   # x's
])
def test_norm_rope_refuses_outputs_that_overlap(part):
    a = norm_rope(part=part)
    assert _lib.lib().spark_qk_norm_rope(ctypes.byref(a), None, None) == INVALID
    assert "output" in _lib.last_error()


def test_norm_rope_refuses_parts_that_overlap():
    """q and k of merged rows: k's output on q's input or output, backward on a gradient."""
    L = _lib.lib()
    two = dict(xs=(1536, 384, 64), ys=(1536, 384, 64), dys=(1536, 384, 64))
    for at in (4096 + 64 * 2, 4096 + 384 * 2 - 2, 16384 + 64 * 2, 16384 - 384 * 2):
        a = norm_rope(part=two)
        ctypes.memmove(ctypes.byref(a.part[1]), ctypes.byref(a.part[0]), ctypes.sizeof(a.part[0]))
        a.part[1].x, a.part[1].y = 1 << 20, at
        assert L.spark_qk_norm_rope(ctypes.byref(a), None, None) == INVALID, at
    for y in (8192 + 128 * 2, 8192 - 2, 4096 + 64):
        a = norm_rope(part=dict(y=y))
        assert L.spark_qk_norm_rope_backward(ctypes.byref(a), P(256), 1 << 30, None, None) == INVALID
    # parts side by side: the next thing that is wrong is found (no workspace; without a GPU no device)
    a = norm_rope(part=dict(two, dweight=64, dy=1 << 21))
    ctypes.memmove(ctypes.byref(a.part[1]), ctypes.byref(a.part[0]), ctypes.sizeof(a.part[0]))
    a.part[1].x, a.part[1].y, a.part[1].dy = 4096 + 128 * 2, 16384 + 128 * 2, (1 << 21) + 128 * 2
    assert L.spark_qk_norm_rope_backward(ctypes.byref(a), None, 0, None, None) not in (_lib.OK, INVALID)


@pytest.mark.parametrize("kw", [
    dict(out=1 << 20, out_stride=(99, 0)), dict(nodes=3, out=1 << 20, out_stride=(250, 100), logits_stride=(300, 100)),
    dict(out=4096 + 4), dict(out=4096 + 400), dict(out=4096 - 4, out_stride=(200, 0)), dict(nodes=3, out=4096 + 400, out_stride=(300, 100), logits_stride=(300, 100)),
])
def test_sample_refuses_outputs_that_overlap(kw):
    a = sampling(token=None, **kw)
    assert _lib.lib().spark_sample(ctypes.byref(a), None) == INVALID
    assert "output" in _lib.last_error()


def test_lora_refuses_outputs_that_overlap():
    """out on y or x at another address; beside them in rows of both it is not refused (what is found next is that there is no
    workspace, or no device)."""
    L = _lib.lib()
    for kw in (dict(out=32768 + 2), dict(out=32768 - 32 * 2), dict(out=32768 + 64, ldo=40, ldy=40), dict(out=4096 + 100), dict(out=4096 - 2),
               dict(out=4096 + 64 * 2 * 3), dict(out=4096 + 96, ldo=64)):
        assert L.spark_lora(ctypes.byref(adapters(**kw)), P(256), 1 << 30, None, None) == INVALID, kw
        assert "overlaps" in _lib.last_error()
    for kw in (dict(out=4096 + 64 * 2, ldx=96, ldo=96), dict(out=32768 + 32 * 2, ldy=64, ldo=64), dict(out=32768), dict(y=4096 + 128, out=4096 + 128, ldx=96, ldy=96, ldo=96)):
        assert L.spark_lora(ctypes.byref(adapters(**kw)), None, 0, None, None) not in (_lib.OK, INVALID), kw
