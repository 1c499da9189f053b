"""Host side of the decode step's operators: what the C entry points refuse before they
touch a device (every pointer here is made up), structure sizes, wrappers on CPU tensors."""
from __future__ import annotations

import ctypes

import pytest
import torch

from spark_b200 import _lib, ops

P = ctypes.c_void_p
INVALID, ALIGNMENT, UNSUPPORTED, WORKSPACE = _lib.ERR_INVALID, _lib.ERR_ALIGNMENT, _lib.ERR_UNSUPPORTED, _lib.ERR_WORKSPACE


def norm_rope(**kw):
    """Arguments of one part of 2 heads of 64 with its weight; kw changes them, those of `part` by a dictionary."""
    a = _lib.SparkNormRope()
    part = dict(x=4096, dy=8192, y=16384, weight=32768, dweight=None, weight_dtype=_lib.DTYPE_F32, heads=2, xs=(512, 128, 64),
                dys=(512, 128, 64), ys=(512, 128, 64))
    part.update(kw.pop("part", {}))
    for name, v in part.items():
        if isinstance(v, tuple):
            v = (ctypes.c_int64 * 3)(*v)
        setattr(a.part[0], name, v)
    both = dict(dtype=_lib.DTYPE_BF16, batch=2, tokens=4, head_dim=64, rot_dim=32, interleaved=0, position_bytes=8, table_rows=10,
                eps=1e-6, positions=65536, table=131072)
    both.update(kw)
    for name, v in both.items():
        setattr(a, name, v)
    return a


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=3), INVALID), (dict(position_bytes=2), INVALID), (dict(head_dim=63), UNSUPPORTED), (dict(head_dim=258), UNSUPPORTED),
    (dict(head_dim=0), UNSUPPORTED), (dict(rot_dim=66), INVALID), (dict(rot_dim=31), INVALID), (dict(rot_dim=0), INVALID),
    (dict(eps=-1.0), INVALID), (dict(eps=float("nan")), INVALID), (dict(eps=float("inf")), INVALID), (dict(batch=-1), INVALID),
    (dict(tokens=-1), INVALID), (dict(table_rows=0), INVALID), (dict(positions=None), INVALID), (dict(table=None), INVALID),
    (dict(part=dict(x=None)), INVALID), (dict(part=dict(y=None)), INVALID), (dict(part=dict(heads=-1)), INVALID),
    (dict(part=dict(weight_dtype=5)), INVALID), (dict(part=dict(ys=(512, 128, 0))), INVALID), (dict(part=dict(ys=(0, 128, 64))), INVALID),
    (dict(part=dict(y=4096, ys=(512, 128, 66))), INVALID), (dict(part=dict(dweight=64)), INVALID),
    (dict(interleaved=1, part=dict(x=4098)), ALIGNMENT), (dict(interleaved=1, part=dict(xs=(513, 128, 64))), ALIGNMENT),
    (dict(batch=1 << 31), UNSUPPORTED),
])
def test_norm_rope_refuses(kw, status):
    a = norm_rope(**kw)
    assert _lib.lib().spark_qk_norm_rope(ctypes.byref(a), None, None) == status
    assert "spark_qk_norm_rope" in _lib.last_error()


def test_norm_rope_refuses_shared_outputs_and_null():
    L = _lib.lib()
    assert L.spark_qk_norm_rope(None, None, None) == INVALID and L.spark_qk_norm_rope_backward(None, None, 0, None, None) == INVALID
    for y, x in ((16384, 1 << 20), (1 << 21, 16384), (4096, 1 << 20)):
        a = norm_rope()
        ctypes.memmove(ctypes.byref(a.part[1]), ctypes.byref(a.part[0]), ctypes.sizeof(a.part[0]))
        a.part[1].y, a.part[1].x = y, x
        assert L.spark_qk_norm_rope(ctypes.byref(a), None, None) == INVALID
    for part in (dict(dy=None), dict(y=4096), dict(weight=None, dweight=64)):
        a = norm_rope(part=part)
        assert L.spark_qk_norm_rope_backward(ctypes.byref(a), P(256), 1 << 30, None, None) == INVALID


def test_norm_rope_without_tokens_or_heads_launches_nothing():
    L = _lib.lib()
    for kw in (dict(batch=0), dict(tokens=0), dict(part=dict(heads=0))):
        a = norm_rope(**kw)
        assert L.spark_qk_norm_rope(ctypes.byref(a), None, None) == _lib.OK
        assert L.spark_qk_norm_rope_backward(ctypes.byref(a), None, 0, None, None) == _lib.OK


def test_cpu_tensors_are_refused():
    q = torch.zeros(1, 2, 2, 64)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.qk_norm_rope(q, None, None, None, torch.zeros(1, 2, dtype=torch.int64), torch.zeros(4, 64))


def sampling(**kw):
    a = _lib.SparkSample()
    both = dict(batch=2, nodes=1, vocab=100, logits=4096, dtype=_lib.DTYPE_F32, logits_stride=(100, 0), temperature_all=1.0,
                top_p_all=1.0, noise=8192, noise_stride=100, token=16384, out=None, out_stride=(100, 100))
    both.update(kw)
    for name, v in both.items():
        setattr(a, name, (ctypes.c_int64 * 2)(*v) if isinstance(v, tuple) else v)
    return a


@pytest.mark.parametrize("kw,status", [
    (dict(batch=-1), INVALID), (dict(nodes=-1), INVALID), (dict(vocab=0), INVALID), (dict(dtype=3), INVALID),
    (dict(vocab=409601), UNSUPPORTED), (dict(batch=1 << 24), UNSUPPORTED), (dict(batch=1 << 13, nodes=1 << 13), UNSUPPORTED),
    (dict(logits=None), INVALID), (dict(token=None), INVALID), (dict(noise=None), INVALID), (dict(nodes=2), INVALID),
    (dict(token=None, out=4096, logprob=256), INVALID), (dict(token=None, out=4096, out_stride=(101, 0)), INVALID),
    (dict(token=None, out=8192, out_stride=(0, 0)), INVALID), (dict(token=None, nodes=3, out=8192, out_stride=(300, 0)), INVALID),
])
def test_sample_refuses(kw, status):
    a = sampling(**kw)
    assert _lib.lib().spark_sample(ctypes.byref(a), None) == status
    assert "spark_sample" in _lib.last_error()


def test_sample_of_nothing():
    assert _lib.lib().spark_sample(None, None) == INVALID
    for kw in (dict(batch=0), dict(nodes=0)):
        assert _lib.lib().spark_sample(ctypes.byref(sampling(**kw)), None) == _lib.OK


def test_sampling_refuses_cpu_tensors():
    x = torch.zeros(2, 10)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.sample(x, torch.ones(2, 10))
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.filter_logits(x)


def adapters(**kw):
    a = _lib.SparkLora()
    both = dict(tokens=4, ic=64, oc=32, rank=8, adapters=2, repeat=1, dtype=_lib.DTYPE_BF16, y_dtype=_lib.DTYPE_BF16, x=4096, a=8192,
                b=16384, y=32768, out=65536, ldx=64, ldy=32, ldo=32, adapter=256, scale=512)
    both.update(kw)
    for name, v in both.items():
        setattr(a, name, v)
    return a


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=_lib.DTYPE_F32), INVALID), (dict(dtype=7), INVALID), (dict(y_dtype=_lib.DTYPE_F16), INVALID), (dict(tokens=-1), INVALID),
    (dict(ic=0), INVALID), (dict(oc=-1), INVALID), (dict(adapters=-1), INVALID), (dict(repeat=0), INVALID), (dict(rank=0), UNSUPPORTED),
    (dict(rank=257), UNSUPPORTED), (dict(tokens=1 << 26), UNSUPPORTED), (dict(x=None), INVALID), (dict(a=None), INVALID),
    (dict(b=None), INVALID), (dict(y=None), INVALID), (dict(out=None), INVALID), (dict(adapter=None), INVALID), (dict(ldo=31), INVALID),
    (dict(ldo=0), INVALID), (dict(out=32768, ldo=40), INVALID), (dict(out=4096), INVALID),
])
def test_lora_refuses(kw, status):
    assert _lib.lib().spark_lora(ctypes.byref(adapters(**kw)), P(256), 1 << 30, None, None) == status
    assert "spark_lora" in _lib.last_error()


def test_lora_of_nothing():
    L = _lib.lib()
    assert L.spark_lora(None, None, 0, None, None) == INVALID
    for kw in (dict(tokens=0), dict(oc=0)):
        assert L.spark_lora(ctypes.byref(adapters(**kw)), None, 0, None, None) == _lib.OK
    assert L.spark_lora_workspace_size(0, 64, 8) == 0 and L.spark_lora_workspace_size(4, 64, 0) == 0
    with pytest.raises(RuntimeError, match="CUDA"):
        x = torch.zeros(2, 8, dtype=torch.bfloat16)
        ops.lora_add(x, x, torch.zeros(1, 1, 8), torch.zeros(1, 8, 1), torch.zeros(2, dtype=torch.int32))
