"""Norms of q and k with rotary positions (ops.qk_norm_rope, rotary.apply_qk_norm_rope)
against the formula in 64 bits.

Tolerances, with e = 2^-24 and u the unit roundoff of the tensors' type (2^-24 fp32,
2^-11 f16, 2^-8 bf16), D <= 256 values a head:
  forward   the sum of squares adds non-negative terms in chains of at most 16 and 8 of
            those in a tree: 24 e relative, 12 e after the root, and 3 for division, addition and
            root; n = x s w two more roundings: 17 e |n|.  The rotation rounds three times
            at most |a| + |b|: 20 e (|a| + |b|) in all, where a and b are the pair of n
            (c, s at most 1).  Then u |y|.
  dx        with m = sum |w d n| / D (n the unit row): d is off by 3 e (|a| + |b|), which
            bounds |d| too; products, sums and s add 36 e of s (w dd + |n| m), with
            dd = |a| + |b|: 48 e s (w dd + |n| mean(w dd |n|)).  Then u |dx|.
  dw        sums of d n, each off by 3 e dd |n| + 18 e |d n|; a chain has at most 64 of the
            terms of the cases here, then come 5 + 8 + 8 + 37 additions: 160 e sum dd |n|.
            Then u |dw|, u of the weight's type.
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


def rotary():
    from spark_b200 import rotary as _rotary
    return _rotary


def turned(y, positions, table, interleaved, back=False, size=False):
    """The rotation in 64 bits; size: |a| + |b| of each value's pair (|y| where it is not turned)."""
    rot = table.shape[1]
    row = table.double()[positions.long()][..., None, :]
    c, s = row[..., :rot // 2], row[..., rot // 2:] * (-1 if back else 1)
    a, b = (y[..., 0:rot:2], y[..., 1:rot:2]) if interleaved else (y[..., :rot // 2], y[..., rot // 2:rot])
    ya, yb = (a.abs() + b.abs(),) * 2 if size else (a * c - b * s, b * c + a * s)
    part = torch.stack([ya, yb], -1).flatten(-2) if interleaved else torch.cat([ya, yb], -1)
    return torch.cat([part, y[..., rot:].abs() if size else y[..., rot:]], -1)


def check_forward(x, w, y, positions, table, interleaved, eps):
    z = x.double()
    n = z / (z.square().mean(-1, keepdim=True) + eps).sqrt() * (1 if w is None else w.double())
    want, size = turned(n, positions, table, interleaved), turned(n, positions, table, interleaved, size=True)
    assert y.dtype == x.dtype and y.shape == x.shape
    off = (y.double() - want).abs() - (U[x.dtype] * want.abs() + 20 * E * size) * 1.001
    assert float(off.max()) <= 2.0 ** -25 if x.dtype == HF else float(off.max()) <= 0, float(off.max())


def check_backward(x, w, g, dx, dw, positions, table, interleaved, eps):
    z, ww = x.double(), torch.ones(x.shape[-1], dtype=torch.float64, device=x.device) if w is None else w.double()
    s = (z.square().mean(-1, keepdim=True) + eps).rsqrt()
    n = z * s
    d, dd = (turned(g.double(), positions, table, interleaved, back=True, size=f) for f in (False, True))
    want = s * (ww * d - n * (ww * d * n).mean(-1, keepdim=True))
    room = s * (ww.abs() * dd + n.abs() * (ww.abs() * dd * n.abs()).mean(-1, keepdim=True))
    if dx is not None:
        off = (dx.double() - want).abs() - (U[x.dtype] * want.abs() + 48 * E * room) * 1.001
        assert float(off.max()) <= (2.0 ** -25 if x.dtype == HF else 0), float(off.max())
    if dw is not None:
        want, room = (d * n).flatten(0, -2).sum(0), (dd * n.abs()).flatten(0, -2).sum(0)
        assert dw.dtype == w.dtype
        off = (dw.double() - want).abs() - (U[w.dtype] * want.abs() + 160 * E * room) * 1.001
        assert float(off.max()) <= (2.0 ** -25 if w.dtype == HF else 0), float(off.max())


def make(seed, b, t, hq, hk, d, rot, dtype, wtype, rows=97, views=True):
    g = gen(seed)
    qkv = randn(g, b, t, (hq + 2 * hk) * d, dtype=dtype)
    q, k = qkv[..., :hq * d].unflatten(-1, (hq, d)), qkv[..., hq * d:(hq + hk) * d].unflatten(-1, (hk, d))
    if not views:
        q, k = q.contiguous(), k.contiguous()
    qw, kw = ((1 + 0.4 * randn(g, d)).to(wtype) for _ in range(2))
    positions = torch.randint(0, rows, (b, t), generator=g, device="cuda")
    return g, q, k, qw, kw, positions, rotary().rope_table(rows, rot)


SIZES = [  # b, t, hq, hk, d, rot
    (1, 1, 1, 1, 2, 2), (1, 1, 32, 8, 128, 128), (2, 3, 5, 2, 64, 64), (3, 7, 6, 2, 80, 40), (1, 19, 7, 1, 112, 28),
    (2, 5, 4, 4, 256, 64), (1, 33, 9, 3, 96, 96), (4, 2, 3, 3, 250, 6), (1, 130, 8, 2, 128, 32), (2, 9, 2, 1, 34, 34),
]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype,wtype", [(BF, BF), (HF, FP), (FP, FP), (BF, FP), (FP, BF)])
@pytest.mark.parametrize("size", SIZES)
def test_forward_and_backward(size, dtype, wtype, interleaved):
    b, t, hq, hk, d, rot = size
    g, q, k, qw, kw, positions, table = make(7, b, t, hq, hk, d, rot, dtype, wtype)
    eps = 1e-5
    y, z = ops().qk_norm_rope(q, k, qw, kw, positions, table, eps=eps, interleaved=interleaved)
    check_forward(q, qw, y, positions, table, interleaved, eps)
    check_forward(k, kw, z, positions, table, interleaved, eps)
    leaves = [x.detach().requires_grad_() for x in (q, k, qw, kw)]
    y2, z2 = rotary().apply_qk_norm_rope(*leaves, positions, table, eps=eps, interleaved=interleaved)
    assert torch.equal(y, y2) and torch.equal(z, z2)
    gy, gz = randn(g, *y.shape, dtype=dtype), randn(g, *z.shape, dtype=dtype)
    dq, dk, dqw, dkw = torch.autograd.grad((y2, z2), leaves, (gy, gz))
    check_backward(q, qw, gy, dq, dqw, positions, table, interleaved, eps)
    check_backward(k, kw, gz, dk, dkw, positions, table, interleaved, eps)
    again = torch.autograd.grad(rotary().apply_qk_norm_rope(*leaves, positions, table, eps=eps, interleaved=interleaved), leaves, (gy, gz))
    assert all(torch.equal(a, b) for a, b in zip(again, (dq, dk, dqw, dkw)))
    ops().check_device_errors()


def test_many_tokens():
    """More items than groups on the GPU: the sums of the weights' gradients go over both parts."""
    g, q, k, qw, kw, positions, table = make(8, 2, 1031, 8, 3, 128, 128, BF, FP)
    leaves = [x.detach().requires_grad_() for x in (q, k, qw, kw)]
    y, z = rotary().apply_qk_norm_rope(*leaves, positions, table)
    check_forward(q, qw, y.detach(), positions, table, False, 1e-6)
    gy, gz = randn(g, *y.shape, dtype=BF), randn(g, *z.shape, dtype=BF)
    dq, dk, dqw, dkw = torch.autograd.grad((y, z), leaves, (gy, gz))
    check_backward(q, qw, gy, dq, dqw, positions, table, False, 1e-6)
    check_backward(k, kw, gz, dk, dkw, positions, table, False, 1e-6)


@pytest.mark.parametrize("interleaved", [False, True])
def test_views_and_addresses(interleaved):
    """Strides and addresses that fit shorter vectors or none; expanded inputs; heads and tokens in another order."""
    g, q, k, qw, kw, positions, table = make(9, 2, 5, 4, 2, 64, 32, BF, BF)
    flat = randn(g, 2 * 5 * 4 * 68 + 9, dtype=BF)
    for at, step in ((1, 67), (2, 66), (4, 68), (3, 65)):
        x = flat[at:].as_strided((2, 5, 4, 64), (5 * 4 * step, 4 * step, step, 1))
        y, _ = ops().qk_norm_rope(x, None, qw, None, positions, table, interleaved=interleaved)
        check_forward(x, qw, y, positions, table, interleaved, 1e-6)
    x = q.transpose(1, 2).contiguous().transpose(1, 2)
    y, z = ops().qk_norm_rope(x, k[:, :, :1].expand(2, 5, 3, 64), None, kw, positions.int(), table, interleaved=interleaved)
    check_forward(x, None, y, positions, table, interleaved, 1e-6)
    check_forward(k[:, :, :1].expand(2, 5, 3, 64), kw, z, positions, table, interleaved, 1e-6)
    # a table at an odd address, a head of every other value
    odd = torch.empty(table.numel() + 1, device="cuda")[1:].view_as(table).copy_(table)
    y, _ = ops().qk_norm_rope(q, None, qw, None, positions, odd, interleaved=interleaved)
    check_forward(q, qw, y, positions, table, interleaved, 1e-6)
    wide = randn(g, 2, 5, 4, 128, dtype=BF)[..., ::2]
    y, _ = ops().qk_norm_rope(wide, None, qw, None, positions, table, interleaved=interleaved)
    check_forward(wide, qw, y, positions, table, interleaved, 1e-6)


def test_in_place_and_without_a_batch():
    _, q, k, qw, kw, positions, table = make(10, 1, 12, 6, 2, 128, 64, HF, HF)
    want = ops().qk_norm_rope(q, k, qw, kw, positions, table)
    rest = q.clone(), k.clone()
    y, z = ops().qk_norm_rope(q[0], k[0], qw, kw, positions[0], table)
    assert torch.equal(y, want[0][0]) and torch.equal(z, want[1][0])
    y, z = ops().qk_norm_rope(q, k, qw, kw, positions, table, out=(q, k))
    assert y.data_ptr() == q.data_ptr() and torch.equal(q, want[0]) and torch.equal(k, want[1])
    assert not torch.equal(rest[0], q)


def test_no_tokens():
    _, q, k, qw, kw, positions, table = make(11, 2, 4, 2, 1, 64, 64, BF, FP)
    leaves = [x.detach().requires_grad_() for x in (q[:, :0], k[:, :0], qw, kw)]
    y, z = rotary().apply_qk_norm_rope(*leaves, positions[:, :0], table)
    assert y.shape == (2, 0, 2, 64)
    grads = torch.autograd.grad((y, z), leaves, (torch.zeros_like(y), torch.zeros_like(z)))
    assert grads[0].shape == y.shape and (grads[2] == 0).all() and (grads[3] == 0).all()


def test_positions_outside_the_table():
    from spark_b200._lib import SparkError
    g, q, k, qw, kw, positions, table = make(12, 1, 6, 3, 2, 64, 64, BF, FP)
    good = positions.clone()
    positions[0, 2], positions[0, 4] = table.shape[0], -1
    leaves = [x.detach().requires_grad_() for x in (q, k, qw, kw)]
    y, z = rotary().apply_qk_norm_rope(*leaves, positions, table)
    with pytest.raises(SparkError, match="position"):
        ops().check_device_errors()
    keep = [0, 1, 3, 5]
    assert (y[0, [2, 4]] == 0).all() and (z[0, [2, 4]] == 0).all()
    check_forward(q[:, keep], qw, y.detach()[:, keep], good[:, keep], table, False, 1e-6)
    gy, gz = randn(g, *y.shape, dtype=BF), randn(g, *z.shape, dtype=BF)
    dq, _, dqw, _ = torch.autograd.grad((y, z), leaves, (gy, gz))
    with pytest.raises(SparkError, match="position"):
        ops().check_device_errors()
    assert (dq[0, [2, 4]] == 0).all()
    check_backward(q[:, keep], qw, gy[:, keep], dq[:, keep], dqw, good[:, keep], table, False, 1e-6)


def test_some_gradients_only():
    """One output's gradient alone, some leaves alone, parts without weights."""
    g, q, k, qw, kw, positions, table = make(13, 2, 6, 3, 2, 64, 32, FP, FP)
    gy, gz = randn(g, *q.shape), randn(g, *k.shape)

    def leaf(x, yes):
        return None if x is None else x.detach().requires_grad_(yes)

    for need in ((1, 0, 0, 0), (0, 1, 0, 1), (0, 0, 1, 0), (0, 0, 0, 1), (1, 1, 0, 1)):
        leaves = [leaf(x, bool(n)) for x, n in zip((q, k, qw, kw), need)]
        out = rotary().apply_qk_norm_rope(*leaves, positions, table)
        pairs = [(o, d) for o, d in zip(out, (gy, gz)) if o.requires_grad]
        got = torch.autograd.grad([p[0] for p in pairs], [x for x in leaves if x.requires_grad], [p[1] for p in pairs])
        got = iter(got)
        dq, dk, dqw, dkw = (next(got) if n else None for n in need)
        check_backward(q, qw, gy, dq, dqw, positions, table, False, 1e-6)
        check_backward(k, kw, gz, dk, dkw, positions, table, False, 1e-6)
    # only y takes part in what is differentiated
    leaves = [leaf(x, True) for x in (q, k, qw, kw)]
    y, _ = rotary().apply_qk_norm_rope(*leaves, positions, table)
    dq, dk, dqw, dkw = torch.autograd.grad(y, leaves, gy, allow_unused=True)
    assert dk is None and dkw is None
    check_backward(q, qw, gy, dq, dqw, positions, table, False, 1e-6)
    # without weights, without k
    for k_, kw_ in ((k, kw), (k, None), (None, None)):
        leaves = [leaf(x, True) for x in (q, k_, None, kw_)]
        out = rotary().apply_qk_norm_rope(*leaves, positions, table)
        got = torch.autograd.grad([o for o in out if o is not None], [x for x in leaves if x is not None], [gy, gz][:2 if k_ is not None else 1])
        check_backward(q, None, gy, got[0], None, positions, table, False, 1e-6)
        if k_ is not None:
            check_backward(k, kw_, gz, got[1], got[2] if kw_ is not None else None, positions, table, False, 1e-6)


def test_shared_weight_and_broadcast_inputs():
    """One weight for both parts, q the same for all sequences, gradients in other layouts."""
    g, q, k, qw, _, positions, table = make(14, 3, 4, 4, 2, 64, 64, FP, FP)
    base, w = q[:1].detach().clone().requires_grad_(), qw.clone().requires_grad_()
    y, z = rotary().apply_qk_norm_rope(base.expand(3, 4, 4, 64), k, w, w, positions, table)
    gy = randn(g, 3, 4, 64, 4).transpose(2, 3)
    gz = randn(g, 1, 1, 1, 64).expand(3, 4, 2, 64)
    dq, dw = torch.autograd.grad((y, z), (base, w), (gy, gz))
    base64, k64, w64 = base.detach().double().requires_grad_(), k.double(), w.detach().double().requires_grad_()

    def forward(x):
        return turned(x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w64, positions, table, False)

    want = torch.autograd.grad((forward(base64.expand(3, 4, 4, 64)), forward(k64)), (base64, w64), (gy.double(), gz.double()))
    assert torch.allclose(dq.double(), want[0], rtol=0, atol=float(1e-5 * want[0].abs().max()))
    assert torch.allclose(dw.double(), want[1], rtol=0, atol=float(1e-5 * want[1].abs().max()))


def test_gradients_are_differences():
    """L = sum of g y along a direction: the central difference of step h is off by O(h^2) of third
    derivatives of order L, and by 40 e |g| |y| / h from the roundings: within 2e-3 of the scale."""
    g, q, k, qw, kw, positions, table = make(15, 1, 3, 2, 1, 32, 16, FP, FP)
    gy, gz = randn(g, *q.shape), randn(g, *k.shape)
    tensors = [x.detach().contiguous() for x in (q, k, qw, kw)]
    leaves = [x.clone().requires_grad_() for x in tensors]
    grads = torch.autograd.grad(rotary().apply_qk_norm_rope(*leaves, positions, table, interleaved=True), leaves, (gy, gz))
    h = 1e-2
    for i in range(4):
        v = randn(g, *tensors[i].shape)

        def value(step):
            x = [t + step * v if j == i else t for j, t in enumerate(tensors)]
            y, z = ops().qk_norm_rope(*x, positions, table, interleaved=True)
            return float((y.double() * gy.double()).sum() + (z.double() * gz.double()).sum())

        scale = float((grads[i].double() * v.double()).abs().sum())
        assert abs((value(h) - value(-h)) / (2 * h) - float((grads[i].double() * v.double()).sum())) < 2e-3 * scale


def test_large_small_and_empty_values():
    """Zeros give zeros; values whose squares overflow or vanish in 16 bits do not in 32."""
    _, q, _, qw, _, positions, table = make(16, 1, 4, 2, 1, 64, 64, BF, FP)
    q = q.contiguous()
    q[0, 0] = 0
    q[0, 1] *= 1e15
    q[0, 2] *= 1e-12
    y, _ = ops().qk_norm_rope(q, None, qw, None, positions, table)
    assert (y[0, 0] == 0).all()
    check_forward(q, qw, y, positions, table, False, 1e-6)


def test_refusals():
    _, q, k, qw, kw, positions, table = make(17, 1, 4, 2, 1, 64, 64, BF, BF)
    f = ops().qk_norm_rope
    from spark_b200._lib import SparkError
    for args, error in [
        ((q.cpu(), k, qw, kw, positions, table), RuntimeError),
        ((q, k.float(), qw, kw, positions, table), TypeError),
        ((q, k[:, :3], qw, kw, positions, table), ValueError),
        ((q, k, qw[:32], kw, positions, table), ValueError),
        ((q, k, qw.double(), kw, positions, table), TypeError),
        ((q, k, qw.cpu(), kw, positions, table), RuntimeError),
        ((q, None, qw, kw, positions, table), ValueError),
        ((q, k, qw, kw, positions.float(), table), TypeError),
        ((q, k, qw, kw, positions[:, :2], table), ValueError),
        ((q, k, qw, kw, positions, table.half()), TypeError),
        ((q, k, qw, kw, positions, table[:, :63].contiguous()), SparkError),
        ((q[..., :63], k[..., :63], qw[:63], kw[:63], positions, table[:, :32].contiguous()), SparkError),
        ((q.double(), None, None, None, positions, table), TypeError),
    ]:
        with pytest.raises(error):
            f(*args)
    for eps in (-1e-6, float("nan"), float("inf")):
        with pytest.raises(SparkError):
            f(q, k, qw, kw, positions, table, eps=eps)
    big = torch.zeros(1, 4, 2, 258, dtype=BF, device="cuda")
    with pytest.raises(SparkError, match="256"):
        f(big, None, None, None, positions, table)
    with pytest.raises(ValueError):
        f(q, k, qw, kw, positions, table, out=(q.float(), k))
    with pytest.raises(SparkError):
        f(q, k, qw, kw, positions, table, out=(q[:, :, :1].expand(1, 4, 2, 64), k))
    with pytest.raises(SparkError):
        f(q[:, :, :1], k, qw, kw, positions, table, out=(k, None))


def test_gradients_of_gradients_and_forward_mode_are_refused():
    _, q, k, qw, kw, positions, table = make(18, 1, 4, 2, 1, 64, 64, FP, FP)
    leaves = [x.detach().clone().requires_grad_() for x in (q, k, qw, kw)]
    y, z = rotary().apply_qk_norm_rope(*leaves, positions, table)
    grads = torch.autograd.grad(y.square().sum() + z.sum(), leaves, create_graph=True)
    check_backward(q, qw, 2 * y.detach(), grads[0].detach(), grads[2].detach(), positions, table, False, 1e-6)
    with pytest.raises(NotImplementedError):
        torch.autograd.grad(grads[0].sum(), leaves[0])
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level():
        dual = fwd.make_dual(leaves[2].detach(), torch.ones_like(leaves[2]))
        with pytest.raises(NotImplementedError):
            rotary().apply_qk_norm_rope(leaves[0], leaves[1], dual, leaves[3], positions, table)


def test_captured_and_on_another_stream():
    """Forward and backward in a graph, replayed on new values; a call on a stream of its own."""
    g, q, k, qw, kw, positions, table = make(19, 1, 40, 4, 2, 128, 128, BF, FP)
    q, k = q.contiguous(), k.contiguous()
    gy, gz = randn(g, *q.shape, dtype=BF), randn(g, *k.shape, dtype=BF)
    leaves = [x.detach().clone().requires_grad_() for x in (q, k, qw, kw)]

    def both():
        out = rotary().apply_qk_norm_rope(*leaves, positions, table)
        return [o.detach() for o in out], torch.autograd.grad(out, leaves, (gy, gz))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = both()
    torch.cuda.current_stream().wait_stream(side)
    plain = both()
    assert all(torch.equal(a, b) for a, b in zip(want[0] + list(want[1]), plain[0] + list(plain[1])))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, grads = both()
    with torch.no_grad():
        leaves[0].mul_(-0.5).add_(0.25)
    graph.replay()
    now = leaves[0].detach().clone()
    check_forward(now, qw, out[0], positions, table, False, 1e-6)
    check_backward(now, qw, gy, grads[0], grads[2], positions, table, False, 1e-6)
    ops().check_device_errors()


def test_capture_beside_a_living_graph():
    """Leaves of which an eager graph lives: refused under capture if it is the default stream's, and taken once it is gone."""
    g, q, k, qw, kw, positions, table = make(23, 1, 24, 4, 2, 64, 64, BF, FP)
    leaves = [x.detach().clone().requires_grad_() for x in (q, k, qw, kw)]
    gy, gz = randn(g, *q.shape, dtype=BF), randn(g, *k.shape, dtype=BF)
    out = rotary().apply_qk_norm_rope(*leaves, positions, table)
    want = torch.autograd.grad(out, leaves, (gy, gz), retain_graph=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="default stream"):
            rotary().apply_qk_norm_rope(*leaves, positions, table)
        with torch.no_grad():
            plain = rotary().apply_qk_norm_rope(*leaves, positions, table)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(plain, out))
    del out
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = rotary().apply_qk_norm_rope(*leaves, positions, table)
        got = torch.autograd.grad(out, leaves, (gy, gz))
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
