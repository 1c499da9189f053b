"""Low-rank adapters of many requests (ops.lora_add) against 64 bits.

Tolerances, e = 2^-24, u the unit roundoff of y's type.  h = A x is a sum of n products in
fp32 on the tensor cores, which may cut instead of round: 2 e a term of a chain of n / (8 splits) + 8 + 16
at most, bounded here by 2 e (n / 8 + 24) of hh = sum |A| |x|.  Its two terms are good to 2^-17 of h (bf16; f16
better), three to 2^-23; B h adds r terms (2 or 3 times) in a chain: 2 e (3 r + 4) of |B| hh; the product with
scale and y: e (|y| + 2 |scale B h|), then u |out|.
"""
from __future__ import annotations

import pytest
import torch

from test_gpu_tree_decode import BF, FP, HF, U, gen, randn

pytestmark = pytest.mark.gpu

E = 2.0 ** -24


def ops():
    from spark_b200 import ops as _ops
    return _ops


def check(y, x, a, b, adapter, scale, out):
    assert out.shape == y.shape and out.dtype == y.dtype
    ic, oc, r = x.shape[-1], y.shape[-1], a.shape[1]
    X, Y, O = x.reshape(-1, ic).double(), y.reshape(-1, oc).double(), out.reshape(-1, oc).double()
    ids = adapter.flatten().long().repeat_interleave(X.shape[0] // max(adapter.numel(), 1))
    want, room = Y.clone(), E * Y.abs()
    for i in ids.unique().tolist():
        if i < 0 or i >= a.shape[0]:
            continue
        rows = (ids == i).nonzero()[:, 0]
        A, B = a[i].double(), b[i].double()
        s = abs(float(scale[i] if isinstance(scale, torch.Tensor) else scale))
        sign = 1 if float(scale[i] if isinstance(scale, torch.Tensor) else scale) >= 0 else -1
        h, hh = X[rows] @ A.T, X[rows].abs() @ A.T.abs()
        term = 2.0 ** -23 if y.dtype == FP else 2.0 ** -17
        off = (h.abs() * term + 2 * E * (ic / 8 + 24) * hh) @ B.T.abs() + 2 * E * (3 * r + 4) * (hh @ B.T.abs())
        delta = h @ B.T * s
        want[rows] += sign * delta
        room[rows] += s * off + 2 * E * delta.abs()
    bad = (O - want).abs() - (U[y.dtype] * want.abs() + room) * 1.001
    assert float(bad.max()) <= (2.0 ** -25 if y.dtype == HF else 0), float(bad.max())


def make(seed, tokens, ic, oc, r, pool, dtype, y_dtype=None, ids=None):
    g = gen(seed)
    x, y = randn(g, tokens, ic, dtype=dtype), randn(g, tokens, oc, dtype=y_dtype or dtype)
    a, b = (randn(g, pool, r, ic) * ic ** -0.5).to(dtype), randn(g, pool, oc, r, dtype=dtype)
    scale = torch.rand(pool, generator=g, device="cuda") * 2 - 0.5
    if ids is None:
        ids = torch.randint(-1, pool, (tokens,), generator=g, device="cuda")
    return y, x, a, b, ids.to(torch.int32), scale


SIZES = [  # tokens, ic, oc, r, pool
    (1, 1, 1, 1, 1), (1, 2560, 4096, 16, 8), (3, 64, 40, 8, 2), (16, 512, 256, 16, 40), (17, 1000, 136, 4, 3), (48, 2560, 1000, 16, 32),
    (64, 96, 264, 33, 70), (65, 200, 72, 64, 5), (100, 1001, 1030, 12, 5), (130, 4096, 96, 100, 7), (300, 264, 1024, 32, 9),
    (33, 72, 513, 256, 2), (200, 520, 264, 128, 20), (1000, 512, 520, 24, 3), (7, 31, 9, 7, 4), (2, 8192, 64, 65, 2),
]


@pytest.mark.parametrize("dtype,y_dtype", [(BF, BF), (HF, HF), (BF, FP), (HF, FP)])
@pytest.mark.parametrize("size", SIZES)
def test_mixed_adapters(size, dtype, y_dtype):
    y, x, a, b, ids, scale = make(sum(size), *size, dtype, y_dtype)
    out = ops().lora_add(y, x, a, b, ids, scale=scale)
    check(y, x, a, b, ids, scale, out)
    assert torch.equal(out, ops().lora_add(y, x, a, b, ids, scale=scale))
    copy = y.clone()
    assert ops().lora_add(copy, x, a, b, ids, scale=scale, out=copy).data_ptr() == copy.data_ptr()
    assert torch.equal(copy, out)
    ops().check_device_errors()


@pytest.mark.parametrize("tokens,per", [(1, 1), (64, 4), (96, 16), (4096, 512), (777, 7), (2048, 2048)])
def test_runs_of_tokens(tokens, per):
    """One adapter for each run, in any of the ways that tiles are worked on."""
    y, x, a, b, _, scale = make(tokens, tokens, 264, 272, 16, 5, BF)
    ids = (torch.arange(tokens // per, device="cuda") * 3 % 6 - 1).to(torch.int32)
    out = ops().lora_add(y, x, a, b, ids, scale=scale)
    check(y, x, a, b, ids, scale, out)
    if tokens % per == 0 and tokens > 1:
        y3, x3 = y.view(-1, per, 272), x.view(-1, per, 264)
        assert torch.equal(ops().lora_add(y3, x3, a, b, ids, scale=scale).view(-1, 272), out)
    mixed = ids.repeat_interleave(per)
    mixed[1::2] = (mixed[1::2] + 3) % 5
    check(y, x, a, b, mixed, scale, ops().lora_add(y, x, a, b, mixed, scale=scale))


@pytest.mark.parametrize("dtype,y_dtype", [(BF, BF), (HF, HF), (BF, FP), (HF, FP)])
@pytest.mark.parametrize("rank,ic,oc", [(1, 40, 130), (12, 72, 128), (16, 256, 513), (24, 96, 1000), (40, 64, 136), (64, 128, 392)])
def test_many_tokens(rank, ic, oc, dtype, y_dtype):
    """Tiles of 128 tokens with one adapter, two, four, none, some without, and more than four, in one call and its last tile short."""
    y, x, a, b, _, scale = make(rank, 900, ic, oc, rank, 12, dtype, y_dtype)
    ids = torch.zeros(900, dtype=torch.int32, device="cuda")
    ids[128:200], ids[200:256] = 3, 5
    ids[256:384] = torch.arange(128, device="cuda") // 32 + 6
    ids[384:512] = -1
    ids[512:600], ids[600:640] = 2, -1
    ids[640:768] = torch.arange(128, device="cuda") * 5 % 12
    ids[768:900] = torch.arange(132, device="cuda") % 3 - 1
    out = ops().lora_add(y, x, a, b, ids, scale=scale)
    check(y, x, a, b, ids, scale, out)
    assert torch.equal(out[384:512], y[384:512])
    assert torch.equal(out, ops().lora_add(y, x, a, b, ids, scale=scale))
    wide = torch.cat([y, y[:, :3]], 1)
    part = wide[:, 3:]
    before = part.clone()
    ops().lora_add(part, x, a, b, ids, scale=scale, out=part)
    check(before, x, a, b, ids, scale, part)
    assert torch.equal(wide[:, :3], y[:, :3])
    ops().check_device_errors()


def test_no_adapter_and_every_token_its_own():
    y, x, a, b, _, scale = make(1, 70, 128, 136, 8, 70, HF)
    none = torch.full((70,), -1, dtype=torch.int32, device="cuda")
    assert torch.equal(ops().lora_add(y, x, a, b, none, scale=scale), y)
    assert torch.equal(ops().lora_add(y, x, a, b, none * 7, scale=scale, out=y.clone()), y)
    own = torch.arange(70, dtype=torch.int32, device="cuda").flip(0)
    check(y, x, a, b, own, 0.75, ops().lora_add(y, x, a, b, own, scale=0.75))
    empty = ops().lora_add(y[:0], x[:0], a, b, own[:0])
    assert empty.shape == (0, 136)
    assert torch.equal(ops().lora_add(y, x, a[:0], b[:0], none, scale=scale[:0]), y)
    one = ops().lora_add(y[0], x[0], a, b, own[0])
    check(y[:1], x[:1], a, b, own[:1], 1.0, one[None])


def test_adapter_outside_the_pool():
    from spark_b200._lib import SparkError
    y, x, a, b, ids, scale = make(2, 40, 64, 64, 8, 3, BF)
    ids[5], ids[33] = 3, 2 ** 31 - 1
    out = ops().lora_add(y, x, a, b, ids, scale=scale)
    with pytest.raises(SparkError, match="adapter"):
        ops().check_device_errors()
    check(y, x, a, b, ids, scale, out)
    assert torch.equal(out[[5, 33]], y[[5, 33]])


@pytest.mark.parametrize("y_dtype", [BF, FP])
def test_layouts(y_dtype):
    """Parts of a merged projection's output in place, rows at odd addresses, expanded inputs, weights in another order."""
    g = gen(3)
    for lead in (0, 8, 3):
        y, x, a, b, ids, scale = make(4, 50, 128, 96, 16, 4, BF, y_dtype)
        wide = randn(g, 50, 96 + 24, dtype=y_dtype)
        before, part = wide.clone(), wide[:, lead:lead + 96]
        ops().lora_add(part, x, a, b, ids, scale=scale, out=part)
        check(before[:, lead:lead + 96], x, a, b, ids, scale, part)
        assert torch.equal(wide[:, :lead], before[:, :lead]) and torch.equal(wide[:, lead + 96:], before[:, lead + 96:])
        xx = randn(g, 50, 150, dtype=BF)[:, lead:lead + 128]
        check(y, xx, a, b, ids, scale, ops().lora_add(y, xx, a, b, ids, scale=scale))
    check(y[:1].expand(50, 96), x[:1].expand(50, 128), a, b, ids, scale, ops().lora_add(y[:1].expand(50, 96), x[:1].expand(50, 128), a, b, ids, scale=scale))
    at, bt = a.transpose(1, 2).contiguous().transpose(1, 2), b.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(ops().lora_add(y, x, at, bt, ids, scale=scale), ops().lora_add(y, x, a, b, ids, scale=scale))
    odd = torch.empty(a.numel() + 1, dtype=BF, device="cuda")[1:].view_as(a).copy_(a)
    check(y, x, odd, b, ids, scale, ops().lora_add(y, x, odd, b, ids, scale=scale))
    cols = x.t().contiguous().t()
    assert torch.equal(ops().lora_add(y, cols, a, b, ids, scale=scale), ops().lora_add(y, x, a, b, ids, scale=scale))


@pytest.mark.parametrize("dtype", [BF, HF])
def test_scales_of_activations(dtype):
    """A x beyond the range of f16, and tiny: rows of very different sizes."""
    y, x, a, b, ids, _ = make(5, 40, 256, 128, 16, 3, dtype, FP)
    size = torch.logspace(-6, 4 if dtype == HF else 8, 40, device="cuda")[:, None]
    x, a = (x.float() * size).to(dtype), (a.float() * 100).to(dtype)
    check(y, x, a, b, ids, 1e-3, ops().lora_add(y, x, a, b, ids, scale=1e-3))
    x = x.clone()
    x[7, 3], x[9, 0] = float("inf"), float("nan")
    ids[7] = ids[9] = 1
    ids[8] = 1
    out = ops().lora_add(y, x, a, b, ids)
    assert not torch.isfinite(out[7]).any() and torch.isnan(out[9]).all() and torch.isfinite(out[8]).all()


@pytest.mark.parametrize("tokens", [1, 40, 100, 700])
def test_infinities_stay_with_their_adapter(tokens):
    """An adapter whose weights hold infinities and NaN beside others in the same tiles; so does a token's x, and y without an adapter."""
    y, x, a, b, _, scale = make(9, tokens, 128, 136, 16, 3, BF)
    ids = (torch.arange(tokens, device="cuda") * 2 // 64 % 4 - 1).to(torch.int32)
    ids[::7] = 2
    a[1, 3, 5], b[1, 20], b[1, :, 2] = float("inf"), float("nan"), float("-inf")
    x[tokens // 2, 0] = float("nan")
    bad = ids == 1
    bad[tokens // 2] = ids[tokens // 2] >= 0
    y[ids < 0, 0] = float("inf")
    out = ops().lora_add(y, x, a, b, ids, scale=scale)
    good = ~bad & (ids >= 0)
    assert torch.equal(out[ids < 0], y[ids < 0])
    if good.any():
        check(y[good], x[good], a, b, ids[good], scale, out[good])
    assert torch.isnan(out[bad][:, 20]).all()


def test_refusals():
    from spark_b200._lib import SparkError
    y, x, a, b, ids, scale = make(6, 12, 64, 32, 8, 3, BF)
    f = ops().lora_add
    for args, kw, error in [
        ((y.cpu(), x, a, b, ids), {}, RuntimeError), ((y, x.cpu(), a, b, ids), {}, RuntimeError), ((y, x, a, b, ids.cpu()), {}, RuntimeError),
        ((y, x.half(), a, b, ids), {}, TypeError), ((y.half(), x, a, b, ids), {}, TypeError), ((y, x.float(), a.float(), b.float(), ids), {}, TypeError),
        ((y, x, a, b, ids.long()), {}, TypeError), ((y, x, a, b, ids[:5]), {}, ValueError), ((y, x, a, b, ids[:0]), {}, ValueError),
        ((y[:5], x, a, b, ids), {}, ValueError), ((y, x, a[:, :, :32], b, ids), {}, ValueError), ((y, x, a[:2], b, ids), {}, ValueError),
        ((y, x, a[:, :4], b, ids), {}, ValueError), ((y, x, a[0], b, ids), {}, ValueError), ((y, x, a[:, :0], b[:, :, :0], ids), {}, ValueError),
        ((y, x, a, b, ids), dict(scale=scale.double()), TypeError), ((y, x, a, b, ids), dict(scale=scale[:2]), TypeError),
        ((y, x, a, b, ids), dict(out=y.float()), ValueError), ((y, x, a, b, ids), dict(out=y[:5]), ValueError),
        ((y, x, a, b, ids), dict(out=torch.empty(32, 12, dtype=BF, device="cuda").t()), ValueError),
        ((y, x, a, b, ids), dict(out=y[:1].expand(12, 32)), SparkError),
    ]:
        with pytest.raises(error):
            f(*args, **kw)
    big = torch.zeros(1, 257, 64, dtype=BF, device="cuda"), torch.zeros(1, 32, 257, dtype=BF, device="cuda")
    with pytest.raises(SparkError, match="256"):
        f(y, x, *big, ids)


def test_captured_and_on_another_stream():
    y, x, a, b, ids, scale = make(7, 48, 512, 384, 16, 8, BF)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops().lora_add(y, x, a, b, ids, scale=scale)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, ops().lora_add(y, x, a, b, ids, scale=scale))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops().lora_add(y, x, a, b, ids, scale=scale)
    for seed in (1, 2):
        x.copy_(randn(gen(seed), 48, 512))
        ids.copy_(torch.randint(-1, 8, (48,), generator=gen(seed), device="cuda"))
        scale.mul_(0.7)
        graph.replay()
        check(y, x, a, b, ids, scale, out)


def test_a_pool_of_one_captured():
    y, x, a, b, ids, scale = make(8, 5, 64, 48, 8, 1, BF)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops().lora_add(y, x, a, b, ids, scale=scale)
    scale.fill_(1.75)
    graph.replay()
    check(y, x, a, b, ids, scale, out)


@pytest.mark.parametrize("tokens,oc", [(1, 512), (40, 2048), (200, 1000), (4096, 2304)])
def test_a_chain_of_calls_without_a_pause(tokens, oc):
    """What a call reads (y, x, the numbers of the adapters) is written by the launch before it, and what it writes is read by the
    next: one graph of twelve steps gives what the steps give one by one."""
    y, x, a, b, ids, scale = make(tokens, tokens, 256, oc, 16, 6, BF)
    ys, xs = (torch.stack([v * (i + 1) for i in range(12)]) for v in (y, x))
    ids = torch.stack([(ids + i).remainder(7) - 1 for i in range(12)]).to(torch.int32)
    if tokens > 1000:
        ids = ids[:, ::tokens // 8].contiguous()
    now = [torch.empty_like(v[0]) for v in (ys, xs, ids)]
    out = torch.empty(12, tokens, oc, dtype=BF, device="cuda")

    def step(i, wait):
        for to, v in zip(now, (ys, xs, ids)):
            to.copy_(v[i])
            if wait:
                torch.cuda.synchronize()
        ops().lora_add(now[0], now[1], a, b, now[2], scale=scale, out=now[0])
        if wait:
            torch.cuda.synchronize()
        ops().lora_add(now[0], now[1] * 0.5, a, b, now[2], scale=scale, out=out[i])

    for i in range(12):
        step(i, True)
    torch.cuda.synchronize()
    want, graph = out.clone(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for i in range(12):
            step(i, False)
    for _ in range(5):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


@pytest.mark.parametrize("tokens", [512, 2048])
def test_two_streams_at_once(tokens):
    """Calls on two streams have workspaces of their own."""
    sets = [make(s, tokens, 512, 4096, 16, 4, BF, ids=torch.randint(-1, 4, (tokens // 64,), device="cuda").repeat_interleave(64)) for s in (1, 2)]
    want = [ops().lora_add(*v[:5], scale=v[5]) for v in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sets], [[], []]
    for _ in range(10):
        for i, (s, v) in enumerate(zip(streams, sets)):
            with torch.cuda.stream(s):
                got[i].append(ops().lora_add(*v[:5], scale=v[5]))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in (0, 1) for g in got[i])


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("tokens,rank,ic,oc", [(8400, 24, 96, 1000), (8389, 64, 40, 1000), (61700, 40, 64, 136), (21411, 12, 72, 392), (1050000, 4, 16, 8)])
def test_as_many_values_as_tensor_memory_takes(tokens, rank, ic, oc, dtype):
    """The tiles of test_many_tokens, again and again at other offsets, where y has 2^23 values or more; rows with a gap; an adapter
    of infinities."""
    y, x, a, b, _, scale = make(rank, tokens, ic, oc, rank, 12, dtype)
    ids = torch.zeros(900, dtype=torch.int32, device="cuda")
    ids[128:200], ids[200:256] = 3, 5
    ids[256:384] = torch.arange(128, device="cuda") // 32 + 6
    ids[384:512] = -1
    ids[512:600], ids[600:640] = 2, -1
    ids[640:768] = torch.arange(128, device="cuda") * 5 % 12
    ids[768:900] = torch.arange(132, device="cuda") % 3 - 1
    ids = ids.repeat(tokens // 900 + 1)[:tokens].contiguous()
    out = ops().lora_add(y, x, a, b, ids, scale=scale)
    check(y, x, a, b, ids, scale, out)
    none = ids < 0
    assert torch.equal(out[none], y[none])
    wide = torch.cat([y[:, :8], y, y[:, :8]], 1)
    part = wide[:, 8:8 + oc]
    ops().lora_add(part, x, a, b, ids, scale=scale, out=part)
    assert torch.equal(part, out) and torch.equal(wide[:, :8], y[:, :8]) and torch.equal(wide[:, -8:], y[:, :8])
    a[3, rank - 1] = float("inf")
    b[5, oc // 2] = float("nan")
    bad = ops().lora_add(y, x, a, b, ids, scale=scale)
    others = (ids != 3) & (ids != 5)
    assert torch.equal(bad[others], out[others]) and not bad[ids == 3].isfinite().all() and bad[ids == 5][:, oc // 2].isnan().all()
    ops().check_device_errors()
