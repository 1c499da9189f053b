"""The tree-decoding operators (rope, tree_attention, tree_verify, kv_append)
against plain 64-bit implementations.

Tolerances, with u the unit roundoff of the tensors' type (2^-24 fp32, 2^-11
f16, 2^-8 bf16):
  rope       a c - b s in fp32: three roundings of at most (|a| + |b|) 2^-24
             each, then one rounding of the result: u |y|;
  attention  the weights may be rounded to 16 bits before they meet V, and the
             result is: u max|v| each; fp32 scores and sums get another
             u max|v|; over all values the two roundings are independent, their
             root mean square is 0.41 u each: Frobenius norm within u;
             lse: a score of D products in fp32 is off by about
             sqrt(D) 2^-24 sum|q k| < 1e-4 here;
  verify     whole numbers: equal, unless the 64-bit decision itself is closer
             than 1e-5 (relative), where fp32 may decide otherwise;
  append     equal.
"""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def ops():
    from spark_b200 import ops as _ops
    return _ops


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=FP):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


# ------------------------------------------------------------------ rope
def rope64(x, positions, table, interleaved, inverse):
    rot = table.shape[1]
    row = table.double()[positions.long()][..., None, :]
    c, s = row[..., :rot // 2], row[..., rot // 2:] * (-1 if inverse else 1)
    x = x.double()
    y = x.clone()
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])
    ya, yb = a * c - b * s, b * c + a * s
    if interleaved:
        y[..., 0:rot:2], y[..., 1:rot:2] = ya, yb
    else:
        y[..., :rot // 2], y[..., rot // 2:rot] = ya, yb
    return y


def check_rope(x, y, want):
    tol = U[x.dtype] * want.abs() * 1.0001 + 3 * 2.0 ** -24 * 2 * x.double().abs().amax(-1, keepdim=True) + 2.0 ** -25 * (x.dtype == HF)
    assert ((y.double() - want).abs() <= tol).all(), (y.double() - want).abs().max().item()


ROPE = [
    # batch, tokens, q heads, kv heads, head_dim, rot_dim
    (1, 1, 1, 1, 64, 64),
    (1, 16, 16, 16, 256, 64),      # a quarter of the head
    (3, 37, 5, 1, 80, 40),
    (2, 129, 8, 2, 128, 128),
    (2, 5, 3, 3, 66, 6),           # rows that no 16-byte access fits
    (1, 7, 2, 1, 34, 2),
    (4, 511, 32, 8, 128, 96),
]


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("b,t,hq,hkv,d,rot", ROPE)
def test_rope(b, t, hq, hkv, d, rot, interleaved, dtype):
    from spark_b200.rotary import rope_table
    g = gen(b * 1000 + t)
    table = rope_table(70000, rot, base=500000.0)
    qkv = randn(g, b, t, (hq + 2 * hkv) * d, dtype=dtype)
    q, k = qkv[..., :hq * d].unflatten(-1, (hq, d)), qkv[..., hq * d:(hq + hkv) * d].unflatten(-1, (hkv, d))
    pos = torch.randint(0, 70000, (b, t), generator=g, device="cuda")
    before = qkv.clone()
    for inverse in (False, True):
        y, z = ops().rope(q, k, pos, table, interleaved=interleaved, inverse=inverse)
        check_rope(q, y, rope64(q, pos, table, interleaved, inverse))
        check_rope(k, z, rope64(k, pos, table, interleaved, inverse))
        assert torch.equal(y[..., rot:], q[..., rot:])
    # int32 positions, no k, tokens without a batch: the same bits
    assert torch.equal(ops().rope(q[0], None, pos[0].int(), table, interleaved, True)[0], y[0])
    # a head-major q: other strides, the same bits
    qh = q.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(ops().rope(qh, k, pos, table, interleaved, True)[0], y)
    # a base address that is not 16-byte aligned
    odd = torch.empty(q.numel() + 1, dtype=dtype, device="cuda")[1:].view(q.shape).copy_(q)
    assert torch.equal(ops().rope(odd, k, pos, table, interleaved, True)[0], y)
    assert torch.equal(qkv, before)
    # in place
    ops().rope(q, k, pos, table, interleaved, True, out=(q, k))
    assert torch.equal(q, y) and torch.equal(k, z)
    assert torch.equal(qkv[..., (hq + hkv) * d:], before[..., (hq + hkv) * d:])
    ops().check_device_errors()


@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_gradient(interleaved):
    """The gradient against the transposed rotation and against differences (the
    operator is linear: a difference over any step is exact but for rounding)."""
    from spark_b200.rotary import apply_rope, rope_table
    g = gen(5)
    table = rope_table(100, 12)
    q, k = randn(g, 2, 9, 3, 20).requires_grad_(), randn(g, 2, 9, 1, 20).requires_grad_()
    pos = torch.randint(0, 100, (2, 9), generator=g, device="cuda")
    wq, wk = randn(g, 2, 9, 3, 20), randn(g, 2, 9, 1, 20)

    def loss(q, k):
        y, z = apply_rope(q, k, pos, table, interleaved)
        return (y.double() * wq).sum() + (z.double() * wk).sum()

    dq, dk = torch.autograd.grad(loss(q, k), (q, k))
    check_rope(wq, dq, rope64(wq, pos, table, interleaved, True))
    check_rope(wk, dk, rope64(wk, pos, table, interleaved, True))
    for x, dx, other in ((q, dq, k), (k, dk, q)):
        step = randn(g, *x.shape)
        at = (lambda v: loss(v, other)) if x is q else (lambda v: loss(other, v))
        diff = (at(x + step) - at(x - step)).item() / 2
        # each of the outputs is off by at most 3 * 2^-24 (|a| + |b|), weighted and summed
        tol = 2.0 ** -24 * 12 * ((x.abs() + step.abs()).amax() * (wq if x is q else wk).abs().sum()).item()
        assert abs(diff - (dx.double() * step).sum().item()) <= tol
    # only one of the two needs a gradient
    y, z = apply_rope(q.detach(), k, pos, table, interleaved)
    (d,) = torch.autograd.grad(z, k, wk)
    assert torch.equal(d, dk)
    y, z = apply_rope(q, None, pos, table, interleaved)
    assert z is None and torch.equal(torch.autograd.grad(y, q, wq)[0], dq)


@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_gradient_of_a_gradient(interleaved):
    """The gradient is linear in what comes back: its own gradient turns forward again."""
    from spark_b200.rotary import apply_rope, rope_table
    g = gen(6)
    table = rope_table(50, 8, scaling="yarn", factor=4.0)
    q, k = (randn(g, 7, n, 8).requires_grad_() for n in (3, 2))
    wq, wk = (randn(g, 7, n, 8).requires_grad_() for n in (3, 2))
    pos = torch.randint(0, 50, (7,), generator=g, device="cuda")
    with torch.no_grad():
        y, z = apply_rope(q, k, pos, table, interleaved)
    assert not y.requires_grad and not z.requires_grad
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y, z = apply_rope(q, k, pos, table, interleaved)
        dq, dk = torch.autograd.grad((y, z), (q, k), (wq, wk), create_graph=True)
        vq, vk = randn(g, *q.shape), randn(g, *k.shape)
        hq, hk = torch.autograd.grad((dq, dk), (wq, wk), (vq, vk))
    torch.cuda.current_stream().wait_stream(s)
    check_rope(q, y, rope64(q, pos, table, interleaved, False))
    check_rope(wk, dk, rope64(wk, pos, table, interleaved, True))
    check_rope(vq, hq, rope64(vq, pos, table, interleaved, False))
    check_rope(vk, hk, rope64(vk, pos, table, interleaved, False))
    ops().check_device_errors()


def test_errors_outlast_a_larger_workspace():
    from spark_b200 import SparkError
    from spark_b200.rotary import rope_table
    g = gen(8)
    q, kt, vt, kc, vc, table, lens, _ = make(g, 8, 16, 32, 8, 128, [4000] * 8, 16, BF)
    parents = torch.arange(-1, 15, dtype=torch.int32, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        bad = torch.full((8, 16), 99, device="cuda")
        ops().rope(q, None, bad, rope_table(10, 16))
        ops().tree_attention(q, kt, vt, kc, vc, table, lens, parents)
    with pytest.raises(SparkError, match="rotary table"):
        ops().check_device_errors()
    ops().check_device_errors()


def test_rope_position_outside_the_table_is_reported():
    from spark_b200.rotary import rope_table
    q = randn(gen(1), 4, 2, 64, dtype=BF)
    table = rope_table(10, 32)
    pos = torch.tensor([3, 10, -1, 9], device="cuda")
    y, _ = ops().rope(q, None, pos, table)
    assert (y[1:3] == 0).all()
    assert torch.equal(y[[0, 3]], ops().rope(q[[0, 3]], None, pos[[0, 3]], table)[0])
    from spark_b200 import SparkError
    with pytest.raises(SparkError, match="rotary table"):
        ops().check_device_errors()
    ops().check_device_errors()
    assert ops().rope(q[:0], q[:0], pos[:0], table)[0].shape == (0, 2, 64)


# ------------------------------------------------------------------ attention
def random_tree(b, t, g):
    """Parents of random trees; about a tenth of the nodes unused."""
    pick = torch.rand(b, t, generator=g, device="cuda")
    at = torch.arange(t, device="cuda")
    p = (pick * (at + 1)).long() - 1
    p = torch.where(torch.rand(b, t, generator=g, device="cuda") < 0.1, -2, p)
    p[:, 0] = -1
    return p.int()


def sees(parents):
    """Nodes that each node sees, [] for an unused one."""
    out = []
    for t in range(len(parents)):
        chain, n = [], t
        while n >= 0:
            chain.append(n)
            up = parents[n]
            n = up if up < n else -2
        out.append(chain if n == -1 else [])
    return out


def attention64(q, kt, vt, kc, vc, table, lens, parents, scale):
    b, t, hq, d = q.shape
    hkv, page = kt.shape[2], kc.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    lse = torch.full((b, t, hq), -math.inf, dtype=torch.float64, device="cuda")
    for i in range(b):
        n = int(lens[i])
        at = torch.arange(n, device="cuda")
        pages = table[i, at // page].long()
        kk = kc[pages, at % page].double()
        vv = vc[pages, at % page].double()
        for j, chain in enumerate(sees((parents if parents.dim() == 1 else parents[i]).tolist())):
            if not chain:
                continue
            keys = torch.cat([kk, kt[i, chain].double()]).repeat_interleave(hq // hkv, 1)
            vals = torch.cat([vv, vt[i, chain].double()]).repeat_interleave(hq // hkv, 1)
            s = torch.einsum("hd,nhd->hn", q[i, j].double(), keys) * scale
            lse[i, j] = torch.logsumexp(s, -1)
            out[i, j] = torch.einsum("hn,nhd->hd", torch.softmax(s, -1), vals)
    return out, lse


def make(g, b, t, hq, hkv, d, lens, page, dtype, spare=3):
    need = [-(-n // page) for n in lens]
    total = sum(need) + spare
    order = torch.randperm(total, generator=g, device="cuda").int()
    table = torch.full((b, max(max(need), 1)), -7, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    kc, vc = randn(g, total, page, hkv, d, dtype=dtype), randn(g, total, page, hkv, d, dtype=dtype)
    q = randn(g, b, t, hq, d, dtype=FP).mul(2).to(dtype)
    kt, vt = randn(g, b, t, hkv, d, dtype=dtype), randn(g, b, t, hkv, d, dtype=dtype)
    return q, kt, vt, kc, vc, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), random_tree(b, t, g)


def check_attention(out, lse, want, want_lse, vmax):
    u = U[out.dtype]
    none = want_lse == -math.inf
    assert torch.equal(lse == -math.inf, none) and (out[none] == 0).all()
    assert ((lse.double() - want_lse)[~none].abs() <= 1e-4).all(), (lse.double() - want_lse)[~none].abs().max().item()
    off = (out.double() - want).abs()
    assert (off <= 3 * u * vmax).all(), (off.max().item(), 3 * u * vmax)
    assert off.norm() <= u * want.norm(), (off.norm() / want.norm()).item()


ATTENTION = [
    # nodes, q heads, kv heads, head_dim, page, context lengths
    (1, 1, 1, 64, 16, [0]),
    (1, 16, 16, 256, 64, [1000]),
    (1, 8, 1, 128, 16, [1, 127, 128, 129, 255, 257]),
    (5, 6, 2, 64, 8, [63, 64, 65, 0, 1]),
    (13, 4, 4, 128, 48, [777, 47, 48, 49, 300]),
    (16, 32, 8, 128, 32, [2049, 1, 500]),
    (16, 8, 8, 256, 24, [513, 64, 191]),
    (33, 10, 2, 128, 64, [700, 0]),
    (64, 8, 1, 128, 128, [1500, 3]),
    (64, 4, 4, 64, 256, [1024, 40, 4000]),
    (64, 16, 2, 256, 32, [600]),
    (40, 14, 2, 80, 40, [333, 90]),
    (7, 5, 5, 112, 16, [257, 12]),
    (3, 12, 3, 16, 8, [130, 7]),
    (2, 40, 1, 128, 64, [20000]),
]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("t,hq,hkv,d,page,lens", ATTENTION)
def test_tree_attention(t, hq, hkv, d, page, lens, dtype):
    g = gen(t * 100 + d)
    x = make(g, len(lens), t, hq, hkv, d, lens, page, dtype)
    scale = d ** -0.5
    want, want_lse = attention64(*x, scale)
    out, lse = ops().tree_attention(*x, return_lse=True)
    vmax = max(x[2].abs().max().item(), x[4].abs().max().item())
    check_attention(out, lse, want, want_lse, vmax)
    again, lse2 = ops().tree_attention(*x, scale=scale, return_lse=True)
    assert torch.equal(out, again) and torch.equal(lse, lse2)
    ops().check_device_errors()


def test_tree_attention_many_ragged_sequences():
    g = gen(77)
    lens = [(i * 37) % 400 for i in range(70)]
    x = make(g, 70, 4, 8, 2, 64, lens, 16, BF)
    want, want_lse = attention64(*x, 0.2)
    out, lse = ops().tree_attention(*x, scale=0.2, return_lse=True)
    check_attention(out, lse, want, want_lse, 5.0)
    # one tree for all, and the same sequence alone
    out1 = ops().tree_attention(*x[:7], x[7][5], scale=0.2)
    one = ops().tree_attention(*(v[5:6] for v in x[:3]), x[3], x[4], x[5][5:6], x[6][5:6], x[7][5], scale=0.2)
    assert (out1[5:6].float() - one.float()).abs().max() <= 3 * U[BF] * 5.0


def test_tree_attention_layouts_and_streams():
    """Head-major caches, merged projections, page tables with a shared row, an output
    view, unaligned inputs and another stream give what contiguous inputs give."""
    g = gen(12)
    b, t, hq, hkv, d = 2, 6, 8, 2, 128
    q, kt, vt, kc, vc, table, lens, parents = make(g, b, t, hq, hkv, d, [300, 170], 32, BF)
    want, want_lse = attention64(q, kt, vt, kc, vc, table, lens, parents, d ** -0.5)
    merged = torch.cat([q.flatten(2), kt.flatten(2), vt.flatten(2)], -1)
    q2 = merged[..., :hq * d].unflatten(-1, (hq, d))
    kt2 = merged[..., hq * d:(hq + hkv) * d].unflatten(-1, (hkv, d))
    vt2 = merged[..., (hq + hkv) * d:].unflatten(-1, (hkv, d))
    both = torch.stack([kc, vc], 1)                       # one tensor for keys and values
    kc2, vc2 = both[:, 0], both[:, 1]
    kc3, vc3 = (c.transpose(1, 2).contiguous().transpose(1, 2) for c in (kc, vc))   # head-major pages
    buf = torch.zeros(b, t, hq + 3, d, dtype=BF, device="cuda")
    for args in ((q2, kt2, vt2, kc, vc), (q, kt, vt, kc2, vc2), (q2, kt, vt2, kc3, vc3)):
        out, lse = ops().tree_attention(*args, table, lens, parents, return_lse=True, out=buf[:, :, 1:hq + 1])
        check_attention(out, lse, want, want_lse, 5.0)
        assert out.data_ptr() == buf[:, :, 1:].data_ptr() and (buf[:, :, 0] == 0).all() and (buf[:, :, hq + 1:] == 0).all()
    odd = [torch.empty(v.numel() + 1, dtype=BF, device="cuda")[1:].view(v.shape).copy_(v) for v in (q, kt, vt)]
    out, lse = ops().tree_attention(*odd, kc, vc, table, lens, parents, return_lse=True)
    check_attention(out, lse, want, want_lse, 5.0)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        out, lse = ops().tree_attention(q, kt, vt, kc, vc, table, lens, parents, return_lse=True)
    torch.cuda.current_stream().wait_stream(stream)
    check_attention(out, lse, want, want_lse, 5.0)
    # parallel samples of one prompt: the table's row and the length are shared
    shared, n = table[:1].expand(2, -1), lens[:1].repeat(2)
    out, lse = ops().tree_attention(q, kt, vt, kc, vc, shared, n, parents, return_lse=True)
    want, want_lse = attention64(q, kt, vt, kc, vc, shared, n, parents, d ** -0.5)
    check_attention(out, lse, want, want_lse, 5.0)


@pytest.mark.parametrize("t,hq,hkv,d", [(1, 8, 1, 128), (9, 4, 2, 64), (20, 8, 1, 128), (12, 2, 2, 256)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf, "lowest"])
def test_tree_attention_masked_places_do_not_matter(t, hq, hkv, d, bad):
    """What a node does not see may hold anything: the cache behind the context, pages
    of others, unused nodes, and nodes that are no ancestors."""
    g = gen(3)
    dtype = BF
    bad = torch.finfo(dtype).min if bad == "lowest" else bad
    q, kt, vt, kc, vc, table, lens, parents = make(g, 3, t, hq, hkv, d, [130, 0, 61], 16, dtype)
    want, want_lse = attention64(q, kt, vt, kc, vc, table, lens, parents, d ** -0.5)
    page = kc.shape[1]
    keep = torch.zeros(kc.shape[:2], dtype=torch.bool, device="cuda")
    for i in range(3):
        at = torch.arange(int(lens[i]), device="cuda")
        keep[table[i, at // page].long(), at % page] = True
    for c in (kc, vc):
        c[~keep] = bad
    out, lse = ops().tree_attention(q, kt, vt, kc, vc, table, lens, parents, return_lse=True)
    check_attention(out, lse, want, want_lse, 5.0)
    # node j of the tree goes bad: the nodes that do not see it stay what they were
    for j in range(0, t, 4):
        kt2, vt2 = kt.clone(), vt.clone()
        kt2[:, j], vt2[:, j] = bad, bad
        out, lse = ops().tree_attention(q, kt2, vt2, kc, vc, table, lens, parents, return_lse=True)
        blind = torch.tensor([[j not in chain for chain in sees(parents[i].tolist())] for i in range(3)], device="cuda")
        if blind.any():
            check_attention(out[blind], lse[blind], want[blind], want_lse[blind], 5.0)
    # only its values go bad: who sees it gets what the formula gives, a NaN or an infinity
    if not math.isfinite(bad):
        vt2 = vt.clone()
        vt2[:, 0, :, 3] = bad
        out = ops().tree_attention(q, kt, vt2, kc, vc, table, lens, parents)
        seen = torch.tensor([[0 in chain for chain in sees(parents[i].tolist())] for i in range(3)], device="cuda")
        assert not torch.isfinite(out[..., 3][seen]).any()
        assert torch.isfinite(out[~seen]).all() and torch.isfinite(out[..., 4:]).all()
    ops().check_device_errors()


def test_tree_attention_long_cache_offsets():
    """A cache of more than 2^31 values and more than 4 GB: the last pages are used."""
    page, hkv, d = 64, 8, 128
    pages = (1 << 31) // (page * hkv * d) + 40
    kc = torch.zeros(pages, page, hkv, d, dtype=BF, device="cuda")
    vc = torch.zeros_like(kc)
    g = gen(8)
    n = 30
    kc[-n:], vc[-n:] = randn(g, n, page, hkv, d, dtype=BF), randn(g, n, page, hkv, d, dtype=BF)
    table = torch.arange(pages - n, pages, dtype=torch.int32, device="cuda").flip(0)[None]
    lens = torch.tensor([n * page - 5], dtype=torch.int32, device="cuda")
    q, kt, vt = randn(g, 1, 4, 16, d, dtype=BF), randn(g, 1, 4, hkv, d, dtype=BF), randn(g, 1, 4, hkv, d, dtype=BF)
    parents = torch.tensor([-1, 0, 0, 2], dtype=torch.int32, device="cuda")
    want, want_lse = attention64(q, kt, vt, kc, vc, table, lens, parents, d ** -0.5)
    out, lse = ops().tree_attention(q, kt, vt, kc, vc, table, lens, parents, return_lse=True)
    check_attention(out, lse, want, want_lse, 5.0)
    before = [kc[-n:].clone(), vc[-n:].clone()]
    new = ops().kv_append(kt, vt, kc, vc, table, lens)
    assert new.tolist() == [n * page - 1]
    before[0][0, -5:-1], before[1][0, -5:-1] = kt[0], vt[0]
    assert torch.equal(kc[-n:], before[0]) and torch.equal(vc[-n:], before[1])


def test_tree_attention_bad_pages_and_lengths_are_reported():
    from spark_b200 import SparkError
    g = gen(2)
    q, kt, vt, kc, vc, table, lens, parents = make(g, 1, 2, 4, 2, 64, [100], 16, BF)
    for t2, l2 in ((table.clone().index_fill_(1, torch.tensor([1], device="cuda"), 10 ** 6), lens), (table, lens + 1000),
                   (table, lens * 0 - 1)):
        ops().tree_attention(q, kt, vt, kc, vc, t2, l2, parents)
        with pytest.raises(SparkError, match="outside the cache"):
            ops().check_device_errors()
    ops().check_device_errors()


def test_tree_attention_in_a_graph():
    """Captured once, replayed with longer contexts and another tree."""
    g = gen(21)
    q, kt, vt, kc, vc, table, lens, parents = make(g, 2, 8, 8, 2, 128, [900, 400], 32, BF)
    now, tree = torch.tensor([5, 0], dtype=torch.int32, device="cuda"), parents.clone()
    ops().tree_attention(q, kt, vt, kc, vc, table, now, tree)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = ops().tree_attention(q, kt, vt, kc, vc, table, now, tree, return_lse=True)
    for n, p in ((lens, parents), (lens // 2, random_tree(2, 8, g)), (lens * 0, parents)):
        now.copy_(n)
        tree.copy_(p)
        graph.replay()
        want, want_lse = attention64(q, kt, vt, kc, vc, table, n, p, 128 ** -0.5)
        check_attention(out, lse, want, want_lse, 5.0)


# ------------------------------------------------------------------ verification
def verify64(logits, tokens, parents, uniforms, noise, draft, temperature):
    """One sequence: (path, next token, the smallest relative margin of a decision)."""
    t = logits.shape[0]
    cur, path, margin = 0, [0], 1.0

    def near(a, b):
        nonlocal margin
        margin = min(margin, abs(a - b) / max(abs(a), abs(b), 1e-30))

    while True:
        row = logits[cur].double()
        if row.isnan().any() or row.max() in (math.inf, -math.inf):
            return path, -1, margin
        best = int((row == row.max()).nonzero()[0])
        r = None if temperature == 0 else torch.softmax(row / temperature, 0)
        step = None
        for c in [j for j in range(cur + 1, t) if parents[j] == cur]:
            x = tokens[c]
            if not 0 <= x < row.numel():
                continue
            if r is None:
                yes = x == best
            else:
                left = uniforms[c] * (1.0 if draft is None else float(draft[cur, x]))
                near(left, float(r[x]))
                yes = left < float(r[x])
            if yes:
                step = c
                break
            if r is not None:
                rest = r.clone()
                if draft is None:
                    rest[x] = 0
                else:
                    rest = (r - draft[cur].double()).clamp(min=0)
                if rest.sum() > 0:
                    r = rest / rest.sum()
        if step is None:
            break
        path.append(step)
        cur = step
    if r is None:
        return path, best, margin
    score = r / noise.double()
    top = score.topk(min(2, score.numel())).values.tolist()
    if len(top) > 1:
        near(*top)
    return path, int(score.argmax()), margin


def verify_inputs(g, b, t, v, dtype, sampled, spread=4.0, shift=0.7):
    logits = torch.randn(b, t, v, generator=g, device="cuda") * spread
    draft = torch.softmax(logits + shift * torch.randn(b, t, v, generator=g, device="cuda"), -1)
    parents = random_tree(b, t, g)
    up = parents.clamp(min=0).long()
    rows = draft.gather(1, up[..., None].expand(b, t, v))
    if sampled:
        tokens = torch.multinomial(rows.reshape(-1, v), 1, generator=g).view(b, t)
    else:
        tokens = rows.topk(min(2, v), -1).indices[..., -1]
    u = torch.rand(b, t, generator=g, device="cuda")
    noise = torch.empty(b, v, device="cuda").exponential_(generator=g)
    return logits.to(dtype), tokens, parents, u, noise, draft if sampled else None


def check_verify(x, got, temperature):
    logits, tokens, parents, u, noise, draft = (v.cpu() if v is not None else None for v in x)
    path, accepted, token = (v.cpu() for v in got)
    t, close = logits.shape[1], 0
    for i in range(logits.shape[0]):
        temp = float(temperature[i]) if isinstance(temperature, torch.Tensor) else temperature
        want, last, margin = verify64(logits[i], tokens[i].tolist(), parents[i].tolist(), u[i].double().tolist(), noise[i],
                                      draft[i] if draft is not None else None, temp)
        if margin < 1e-5:
            close += 1
            continue
        assert accepted[i] == len(want) and path[i].tolist() == want + [-1] * (t - len(want)), (i, path[i], want)
        assert token[i] == last, (i, token[i], last)
    assert close <= max(1, logits.shape[0] // 20)


@pytest.mark.parametrize("dtype", [FP, BF, HF])
@pytest.mark.parametrize("sampled", [True, False])
@pytest.mark.parametrize("b,t,v", [(1, 1, 5), (3, 8, 1), (40, 12, 33), (5, 16, 1000), (7, 9, 32001), (2, 64, 4099), (1, 5, 160000),
                                   (70, 6, 2001), (130, 4, 509), (300, 3, 77)])
def test_tree_verify(b, t, v, sampled, dtype):
    g = gen(b + t + v)
    x = verify_inputs(g, b, t, v, dtype, sampled)
    for temperature in (1.0, 0.0, torch.tensor([(1.0, 0.0, 0.6, 1.5)[i % 4] for i in range(b)], device="cuda")):
        got = ops().tree_verify(*x[:5], draft_probs=x[5], temperature=temperature)
        check_verify(x, got, temperature)
        again = ops().tree_verify(*x[:5], draft_probs=x[5], temperature=temperature)
        assert all(torch.equal(a, b) for a, b in zip(got, again))
    ops().check_device_errors()


def test_tree_verify_layouts():
    """16-bit draft probabilities, strided rows, one tree for all."""
    g = gen(31)
    b, t, v = 6, 10, 777
    logits, tokens, _, u, noise, draft = verify_inputs(g, b, t, v, FP, True)
    parents = random_tree(1, t, g)[0]
    wide = torch.randn(b, t, v + 5, generator=g, device="cuda")
    wide[..., 3:v + 3] = logits
    draft = draft.to(BF)
    x = (wide[..., 3:v + 3], tokens, parents.expand(b, t), u, noise, draft)
    got = ops().tree_verify(x[0], tokens, parents, u, noise, draft_probs=draft)
    check_verify(x, got, 1.0)


@pytest.mark.parametrize("sampled", [True, False])
def test_tree_verify_samples_the_target(sampled):
    """The first new token is distributed as the target's softmax whatever the draft
    is: 100000 sequences with the same logits, every frequency within 5 standard
    deviations."""
    g = gen(4)
    b, v = 100000, 7
    parents = torch.tensor([-1, 0, 0, 0], dtype=torch.int32, device="cuda")
    logits = torch.randn(1, 4, v, generator=g, device="cuda").expand(b, 4, v)
    p = torch.softmax(logits[0, 0].double(), 0)
    if sampled:
        q = torch.softmax(torch.randn(v, generator=g, device="cuda") * 1.5, 0)
        tokens = torch.multinomial(q, b * 4, replacement=True, generator=g).view(b, 4)
        draft = q.expand(b, 4, v)
    else:
        tokens, draft = torch.tensor([0, 2, 5, 1], device="cuda").expand(b, 4), None
    u = torch.rand(b, 4, generator=g, device="cuda")
    noise = torch.empty(b, v, device="cuda").exponential_(generator=g)
    path, n, last = ops().tree_verify(logits, tokens, parents, u, noise, draft_probs=draft)
    first = torch.where(n > 1, tokens.gather(1, path[:, 1:2].clamp(min=0).long())[:, 0], last)
    share = torch.bincount(first, minlength=v).double() / b
    assert ((share - p).abs() <= 5 * (p * (1 - p) / b).sqrt()).all(), (share, p)
    assert 0.2 < (n > 1).double().mean() < 0.99


def test_tree_verify_rows_without_a_distribution():
    """NaN, +inf and all -inf end a sequence with -1; single -inf values are probability
    zero; a draft equal to the target accepts; a bad token id is reported."""
    from spark_b200 import SparkError
    g = gen(6)
    b, t, v = 8, 3, 300
    logits = torch.randn(b, t, v, generator=g, device="cuda")
    tokens = torch.randint(0, v, (b, t), generator=g, device="cuda")
    parents = torch.tensor([-1, 0, 1], dtype=torch.int32, device="cuda")
    u, noise = torch.full((b, t), 0.5, device="cuda"), torch.empty(b, v, device="cuda").exponential_(generator=g)
    logits[0, 0, 250] = math.nan
    logits[1, 0] = -math.inf
    logits[2, 0, 7] = math.inf
    logits[3, 0] = -math.inf
    logits[3, 0, 123] = 2.0
    tokens[3, 1] = 9
    logits[4, 0], tokens[4, 1] = -math.inf, 77
    logits[4, 0, 77] = 1.0
    logits[4, 1, 5] = math.nan
    draft = torch.softmax(logits, -1)
    for temperature in (1.0, 0.0):
        path, n, last = ops().tree_verify(logits, tokens, parents, u, noise, temperature=temperature)
        assert last[:5].tolist() == [-1, -1, -1, 123, -1] and n[:5].tolist() == [1, 1, 1, 1, 2]
    path, n, last = ops().tree_verify(logits[5:], tokens[5:], parents, u[5:], noise[5:], draft_probs=draft[5:])
    assert n.tolist() == [3, 3, 3]
    ops().check_device_errors()
    tokens[6, 1] = v
    path, n, last = ops().tree_verify(logits, tokens, parents, u, noise)
    assert n[6] == 1 and 0 <= last[6] < v
    with pytest.raises(SparkError, match="vocabulary"):
        ops().check_device_errors()


# ------------------------------------------------------------------ append
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("b,t,hkv,d,page,ctx", [(1, 1, 1, 64, 16, 0), (5, 16, 8, 128, 32, 100), (3, 7, 3, 50, 5, 11),
                                                (2, 300, 4, 80, 24, 1), (4, 9, 2, 8, 1, 17), (2, 45, 1, 8, 7, 3), (2, 70, 3, 24, 16, 9)])
def test_kv_append(b, t, hkv, d, page, ctx, dtype):
    g = gen(t)
    lens = [(ctx + 13 * i) % (ctx + 40) for i in range(b)]
    _, _, _, kc, vc, table, n, _ = make(g, b, 1, hkv, hkv, d, [v + t for v in lens], page, dtype)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    merged = randn(g, b, t, 2 * hkv * d, dtype=dtype)
    k, v = merged[..., :hkv * d].unflatten(-1, (hkv, d)), merged[..., hkv * d:].unflatten(-1, (hkv, d))
    index = torch.rand(b, t, generator=g, device="cuda").argsort(-1).int()
    counts = torch.randint(0, t + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
    for idx, cnt in ((None, None), (index, counts), (index, None), (None, counts), (index[:, :1], None)):
        for head_major in (False, True):
            k2, v2 = kc.clone(), vc.clone()
            if head_major:
                k2, v2 = (c.transpose(1, 2).contiguous().transpose(1, 2) for c in (k2, v2))
            new = ops().kv_append(k, v, k2, v2, table, n, index=idx, counts=cnt)
            wk, wv, m = kc.clone(), vc.clone(), []
            for i in range(b):
                many = int(cnt[i]) if cnt is not None else t if idx is None else idx.shape[1]
                m.append(lens[i] + many)
                for j in range(many):
                    at = lens[i] + j
                    src = int(idx[i, j]) if idx is not None else j
                    wk[table[i, at // page], at % page], wv[table[i, at // page], at % page] = k[i, src], v[i, src]
            assert torch.equal(k2, wk) and torch.equal(v2, wv) and new.tolist() == m
    ops().check_device_errors()


def test_kv_append_out_of_room_and_bad_indexes_are_reported():
    from spark_b200 import SparkError
    g = gen(9)
    _, _, _, kc, vc, table, n, _ = make(g, 2, 1, 2, 2, 64, [30, 20], 16, BF)
    table[1, 1:] = -1
    k, v = randn(g, 2, 6, 2, 64, dtype=BF), randn(g, 2, 6, 2, 64, dtype=BF)
    before = kc.clone()
    new = ops().kv_append(k, v, kc, vc, table, n)      # 0: room for two; 1: its second page is bad
    assert new.tolist() == [32, 26]
    page = int(table[0, 1])
    before[page, 14:] = k[0, :2]
    assert torch.equal(kc, before)
    with pytest.raises(SparkError, match="outside the cache"):
        ops().check_device_errors()
    idx = torch.tensor([[6], [-1]], dtype=torch.int32, device="cuda")
    ops().kv_append(k, v, kc, vc, table, torch.zeros_like(n), index=idx)
    assert torch.equal(kc, before)
    with pytest.raises(SparkError, match="outside the cache"):
        ops().check_device_errors()
    assert ops().kv_append(k[:0], v[:0], kc, vc, table[:0], n[:0]).shape == (0,)


# ------------------------------------------------------------------ refusals
def test_refusals():
    g = gen(1)
    o = ops()
    from spark_b200 import SparkError
    from spark_b200.rotary import rope_table
    x = q, kt, vt, kc, vc, table, lens, parents = make(g, 2, 4, 8, 2, 64, [30, 20], 16, BF)

    def attention(**kw):
        names = ("q", "k_tree", "v_tree", "k_cache", "v_cache", "page_table", "context_lens", "parents")
        return o.tree_attention(**{**dict(zip(names, x)), **kw})

    for err, kw in ((TypeError, {"q": q.half()}), (TypeError, {"k_cache": kc.half()}), (TypeError, {"parents": parents.long()}),
                    (TypeError, {"parents": parents[:1]}), (TypeError, {"context_lens": lens.long()}),
                    (TypeError, {"page_table": table.long()}), (ValueError, {"k_tree": kt[:, :3]}),
                    (ValueError, {"q": q[..., :32]}), (ValueError, {"v_cache": vc[:, :8]}),
                    (ValueError, {"out": q[:, :1].clone()}), (RuntimeError, {"q": q.cpu()}),
                    (RuntimeError, {"page_table": table.cpu()}), (RuntimeError, {"k_cache": kc.cpu()}),
                    (SparkError, {"q": q[:, :, :7]}), (SparkError, {"scale": 0.0}), (SparkError, {"scale": -1.0})):
        with pytest.raises(err):
            attention(**kw)
    y = make(g, 1, 65, 2, 2, 64, [30], 16, BF)
    with pytest.raises(SparkError, match="64 nodes"):
        o.tree_attention(*y)
    y = make(g, 1, 2, 129, 1, 64, [30], 16, BF)
    with pytest.raises(SparkError, match="at most 128"):
        o.tree_attention(*y)
    y = make(g, 1, 2, 2, 2, 64, [30], 12, BF)
    with pytest.raises(SparkError, match="page_size"):
        o.tree_attention(*y)
    y = make(g, 1, 2, 2, 2, 264, [30], 16, BF)
    with pytest.raises(SparkError, match="head_dim"):
        o.tree_attention(*y)

    t2, pos = rope_table(50, 32), torch.zeros(2, 4, dtype=torch.int64, device="cuda")
    for err, a in ((TypeError, (q, kt.half(), pos, t2)), (ValueError, (q, kt[:, :3], pos, t2)), (ValueError, (q, kt, pos[0], t2)),
                   (TypeError, (q, kt, pos.float(), t2)), (TypeError, (q, kt, pos, t2.double())),
                   (TypeError, (q.int(), None, pos, t2)), (RuntimeError, (q.cpu(), None, pos, t2)),
                   (RuntimeError, (q, kt, pos.cpu(), t2)), (SparkError, (q, kt, pos, t2[:, :31].contiguous())),
                   (SparkError, (q[..., :16], None, pos, t2)), (ValueError, (q[0, 0], None, pos[0], t2))):
        with pytest.raises(err):
            o.rope(*a)
    with pytest.raises(ValueError):
        o.rope(q, None, pos, t2, out=(q[:1], None))

    for err, a in ((TypeError, (kt, vt.half())), (ValueError, (kt, vt[:, :2])), (ValueError, (kt[..., :32], vt[..., :32]))):
        with pytest.raises(err):
            o.kv_append(*a, kc, vc, table, lens)
    with pytest.raises(TypeError):
        o.kv_append(kt, vt, kc, vc, table, lens, index=parents.long())
    with pytest.raises(TypeError):
        o.kv_append(kt, vt, kc, vc, table, lens, counts=lens.long())
    with pytest.raises(ValueError):
        o.kv_append(kt[:1], vt[:1], kc, vc, table, lens)

    z = logits, tokens, par, u, noise, draft = verify_inputs(g, 2, 4, 50, FP, True)
    for err, i, bad in ((ValueError, 0, logits[0]), (ValueError, 1, tokens[:1]), (TypeError, 1, tokens.int()),
                        (TypeError, 2, par.long()), (TypeError, 3, u.double()), (ValueError, 4, noise[:, :9]),
                        (RuntimeError, 4, noise.cpu()), (TypeError, 0, logits.double())):
        with pytest.raises(err):
            o.tree_verify(*[bad if j == i else w for j, w in enumerate(z[:5])])
    with pytest.raises(ValueError):
        o.tree_verify(*z[:5], draft_probs=draft[:, :2])
    with pytest.raises(TypeError):
        o.tree_verify(*z[:5], temperature=torch.ones(3, device="cuda"))
