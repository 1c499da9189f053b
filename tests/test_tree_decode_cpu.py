"""Host side of the tree-decoding operators: argument checks of the C entry
points before anything is launched, and the rotary tables."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

from spark_b200 import _lib, rotary

P = ctypes.c_void_p


def cache(**kw):
    c = _lib.SparkPagedCache(k=256, v=256, pages=4, page_size=16, kv_heads=2, head_dim=64, page_table=256,
                             page_table_stride=4, max_pages=4, lens=256, dtype=_lib.DTYPE_BF16)
    for i, s in enumerate((16 * 2 * 64, 2 * 64, 64)):
        c.k_stride[i] = c.v_stride[i] = s
    for name, v in kw.items():
        setattr(c, name, v)
    return c


def test_rope_checks():
    h = _lib.SparkRopeHeads(x=256, y=512, heads=2)
    q = ctypes.byref(h)

    def run(q=q, k=None, dtype=1, batch=1, tokens=1, dim=64, rot=32, pos=P(256), pb=8, table=P(256), rows=10):
        return _lib.lib().spark_rope(q, k, dtype, batch, tokens, dim, rot, 0, 0, pos, pb, table, rows, None, None)

    assert run(tokens=0) == _lib.OK
    for kw in ({"q": None}, {"dtype": 3}, {"rot": 31}, {"rot": 66}, {"rot": 0}, {"pb": 2}, {"pos": None}, {"table": None},
               {"rows": 0}, {"batch": -1}):
        assert run(**kw) == _lib.ERR_INVALID, kw
        assert "spark_rope" in _lib.last_error()
    bad = _lib.SparkRopeHeads(x=256, y=256, heads=2)
    bad.xs[1], bad.ys[1] = 64, 128
    assert run(q=ctypes.byref(bad)) == _lib.ERR_INVALID and "in place" in _lib.last_error()
    assert run(k=ctypes.byref(_lib.SparkRopeHeads(x=256, heads=1))) == _lib.ERR_INVALID


def test_append_checks():
    strides = (ctypes.c_int64 * 3)(128, 128, 64)

    def run(c=None, batch=1, tokens=2, k=P(256), index=None, width=2, new=P(512), st=strides):
        c = cache() if c is None else c
        return _lib.lib().spark_kv_append(ctypes.byref(c), batch, tokens, k, st, k, st, index, width, None, new, None, None)

    assert run(batch=0) == _lib.OK
    for kw in ({"c": cache(pages=0)}, {"c": cache(page_size=0)}, {"c": cache(max_pages=1 << 28)}, {"c": cache(dtype=5)},
               {"c": cache(k=None)}, {"c": cache(lens=None)}, {"batch": 1 << 16}, {"width": 3}, {"new": None},
               {"new": P(256)}, {"k": None}, {"st": None}):
        assert run(**kw) == _lib.ERR_INVALID, kw
        assert "spark_kv_append" in _lib.last_error()
    assert _lib.lib().spark_kv_append(None, 1, 1, None, None, None, None, None, 1, None, None, None, None) == _lib.ERR_INVALID


def attention(c=None, **kw):
    a = _lib.SparkTreeAttention(cache=cache() if c is None else c, batch=1, nodes=4, q_heads=4, q=256, k=256, v=256,
                                out=256, parents=256, scale=0.1)
    for i in range(3):
        s = (4 * 4 * 64, 4 * 64, 64)[i]
        a.q_stride[i] = a.out_stride[i] = a.kn_stride[i] = a.vn_stride[i] = s
    for name, v in kw.items():
        setattr(a, name, v)
    return a


def test_attention_checks():
    L = _lib.lib()

    def run(a, ws=P(1 << 20), n=1 << 30):
        return L.spark_tree_attention(ctypes.byref(a), ws, n, None), L.spark_tree_attention_workspace_size(ctypes.byref(a))

    rc, size = run(attention(batch=0))
    assert rc == _lib.OK and size >= 256
    for want, a in ((_lib.ERR_INVALID, attention(nodes=0)), (_lib.ERR_INVALID, attention(nodes=65)),
                    (_lib.ERR_INVALID, attention(q_heads=3)), (_lib.ERR_INVALID, attention(batch=1 << 16)),
                    (_lib.ERR_INVALID, attention(cache(kv_heads=0))), (_lib.ERR_UNSUPPORTED, attention(cache(dtype=0))),
                    (_lib.ERR_UNSUPPORTED, attention(cache(head_dim=68))), (_lib.ERR_UNSUPPORTED, attention(cache(head_dim=264)))):
        assert run(a) == (want, 0)
        assert "spark_tree_attention" in _lib.last_error()
    for name in ("q", "k", "v", "out", "parents"):
        assert run(attention(**{name: None}))[0] == _lib.ERR_INVALID
    assert run(attention(cache(lens=None)))[0] == _lib.ERR_INVALID
    assert run(attention(), ws=None)[0] == _lib.ERR_WORKSPACE
    assert run(attention(), n=100)[0] == _lib.ERR_WORKSPACE
    assert L.spark_tree_attention(None, P(256), 256, None) == _lib.ERR_INVALID


def test_verify_checks():
    def run(**kw):
        a = _lib.SparkTreeVerify(batch=1, nodes=2, vocab=100, logits=256, tokens=256, parents=256, uniforms=256, noise=256,
                                 path=256, accepted=256, next=256)
        for name, v in kw.items():
            setattr(a, name, v)
        return _lib.lib().spark_tree_verify(ctypes.byref(a), None, None)

    assert run(batch=0) == _lib.OK
    for kw in ({"nodes": 0}, {"vocab": 0}, {"logits_dtype": 3}, {"draft": 256, "draft_dtype": -1}, {"batch": -1},
               *({name: None} for name in ("logits", "tokens", "parents", "uniforms", "noise", "path", "accepted", "next"))):
        assert run(**kw) == _lib.ERR_INVALID, kw
        assert "spark_tree_verify" in _lib.last_error()
    assert run(vocab=1 << 20) == _lib.ERR_UNSUPPORTED
    assert _lib.lib().spark_tree_verify(None, None, None) == _lib.ERR_INVALID


def test_the_torch_binding_loads_and_refuses_cpu_tensors():
    from spark_b200 import ops
    x = torch.zeros(2, 3, 64)
    i = torch.zeros(2, 2, dtype=torch.int32)
    for call in (lambda: ops.rope(x, None, i[0], torch.zeros(4, 8)),
                 lambda: ops.kv_append(x[None], x[None], x[None], x[None], i, i[0]),
                 lambda: ops.tree_attention(x[None], x[None], x[None], x[None], x[None], i, i[0], i),
                 lambda: ops.tree_verify(x, i, i, x[..., 0], x[:, 0])):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            call()
    n = ops._native()
    with pytest.raises(RuntimeError, match="q must be a CUDA tensor"):
        n.rope(x, None, i[0], torch.zeros(4, 8), False, False, None, None, 0, 0)
    # the checks before the device's, by their kinds
    with pytest.raises(ValueError, match="kv_append"):
        n.kv_append(x, x, x, x, i, i[0], None, None, 0, 0)
    with pytest.raises(TypeError, match="differ in type"):
        n.kv_append(x[None], x[None].half(), x[None], x[None], i, i[0], None, None, 0, 0)


def test_rope_frequencies():
    f, m = rotary.rope_frequencies(8, 10000.0)
    assert m == 1.0 and torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64))
    lin, _ = rotary.rope_frequencies(8, 10000.0, scaling="linear", factor=4.0)
    assert torch.allclose(lin, f / 4)
    ntk, _ = rotary.rope_frequencies(8, 10000.0, scaling="ntk", factor=4.0)
    assert ntk[0] == 1.0 and math.isclose(ntk[-1], f[-1] / 4, rel_tol=1e-12)
    f, _ = rotary.rope_frequencies(128, 10000.0)
    yarn, m = rotary.rope_frequencies(128, 10000.0, scaling="yarn", factor=8.0, original_positions=4096)
    turns = f * 4096 / (2 * math.pi)
    assert torch.equal(yarn[turns > 34], f[turns > 34]) and torch.allclose(yarn[turns < 0.9], f[turns < 0.9] / 8)
    assert (yarn <= f).all() and (yarn >= f / 8 * (1 - 1e-12)).all() and math.isclose(m, 0.1 * math.log(8.0) + 1)
    t = rotary.rope_table(50, 8, device="cpu", scaling="yarn", factor=2.0)
    assert t.shape == (50, 8) and t.dtype == torch.float32
    assert torch.allclose(t[:, :4] ** 2 + t[:, 4:] ** 2, torch.full((50, 4), (0.1 * math.log(2.0) + 1) ** 2))
    for kw in ({"rot_dim": 7}, {"rot_dim": 8, "scaling": "other"}, {"rot_dim": 8, "base": -1.0}, {"rot_dim": 8, "factor": 0.0}):
        with pytest.raises(ValueError):
            rotary.rope_frequencies(**kw)
