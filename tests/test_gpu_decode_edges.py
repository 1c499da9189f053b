"""Norms, sampling and adapters at the edges of their definitions, against 64 bits."""
from __future__ import annotations

import math

import pytest
import torch

from test_gpu_lora import E, check, make
from test_gpu_sample import check_sample, noise_of
from test_gpu_tree_decode import BF, FP, HF, U, gen, randn

pytestmark = pytest.mark.gpu


def ops():
    from spark_b200 import ops as _ops
    return _ops


# ------------------------------------------------------------------ adapters
# few tokens, more, and as many values of y as the tensor memory takes
MANY = [(40, 136), (64, 136), (65, 136), (300, 264), (8400, 1000)]


def runs(tokens, pool):
    """Adapters in runs of 96 tokens, or of an eighth of a few; one run in pool + 1 without one."""
    return (torch.arange(tokens, device="cuda") // min(96, tokens // 8) % (pool + 1) - 1).flip(0).to(torch.int32)


@pytest.mark.parametrize("dtype,y_dtype", [(BF, BF), (HF, HF), (BF, FP), (HF, FP)])
@pytest.mark.parametrize("tokens,oc", MANY)
def test_infinite_weights_of_b(tokens, oc, dtype, y_dtype):
    """One infinity in a row of B: y + scale B h has its sign times that of h, whose error is below its size in the rows that are
    looked at; the row's other columns are what they are without it."""
    y, x, a, b, _, scale = make(tokens, tokens, 128, oc, 16, 3, dtype, y_dtype)
    ids = runs(tokens, 3)
    at = {2: (3, math.inf), 70: (0, -math.inf), 71: (15, math.inf), oc - 1: (7, -math.inf)}
    for column, (rank, value) in at.items():
        b[1, column, rank] = value
    out = ops().lora_add(y, x, a, b, ids, scale=scale)
    mine = ids == 1
    rest = [c for c in range(oc) if c not in at]
    check(y[:, rest], x, a, b[:, rest], ids, scale, out[:, rest])
    assert out[~mine].isfinite().all()
    for column, (rank, value) in at.items():
        h, size = x[mine].double() @ a[1, rank].double(), x[mine].double().abs() @ a[1, rank].double().abs()
        sure = h.abs() > 2 * E * (128 / 8 + 24) * size
        assert int(sure.sum()) > int(mine.sum()) * 0.9
        assert torch.equal(out[mine, column][sure].double(), (value * scale[1].double().sign() * h.sign())[sure])
    assert int(mine.sum()) >= tokens // 5
    ops().check_device_errors()


@pytest.mark.parametrize("dtype,y_dtype", [(BF, BF), (HF, HF), (BF, FP), (HF, FP)])
@pytest.mark.parametrize("tokens,oc", MANY)
def test_infinite_values_of_h(tokens, oc, dtype, y_dtype):
    """One infinity in A, and beside it components beyond the range of f16: every column is infinite by the sign of B alone.  Two
    infinities of one sign in a row of h: NaN where B has them on different sides, infinite elsewhere."""
    y, x, a, b, _, scale = make(tokens + 1, tokens, 128, oc, 16, 3, dtype, y_dtype)
    ids = runs(tokens, 3)
    x = torch.where(x == 0, 1, x).abs().to(dtype)
    a = a.abs()
    a[:, 1:9] *= 30000
    b = torch.where(b == 0, 1, b)
    a[0, 4, 10] = math.inf
    a[2, 5, 1], a[2, 12, 100] = math.inf, math.inf
    out = ops().lora_add(y, x, a, b, ids, scale=scale)
    sign = scale.double().sign()
    got = out.double()
    assert torch.equal(got[ids == 0], (sign[0] * b[0, :, 4].double().sign() * math.inf).expand(int((ids == 0).sum()), oc))
    p, q = b[2, :, 5].double().sign(), b[2, :, 12].double().sign()
    alike = p == q
    two = got[ids == 2]
    assert two[:, ~alike].isnan().all() and int(alike.sum()) > 10 and int((~alike).sum()) > 10
    assert torch.equal(two[:, alike], (sign[2] * p[alike] * math.inf).expand(two.shape[0], -1))
    # (in f16 the sums of adapter 1 are beyond its range)
    others = ids < 0 if y_dtype == HF else (ids == 1) | (ids < 0)
    check(y[others], x[others], a, b, ids[others], scale, out[others])
    ops().check_device_errors()


@pytest.mark.parametrize("tokens,oc", MANY)
@pytest.mark.parametrize("y_dtype", [HF, FP])
def test_ranks_of_very_different_sizes(tokens, oc, y_dtype):
    """f16, the ranks of one token's h from 1 down to 2^-30 of the largest, and columns of B that are zero up to one of them.  A row
    is brought to 2^15 or more; a component's first term is cut at 2^-10 of it, the second rounded at 2^-22 of it (a third at 2^-32), or
    at f16's last step, 2^-24, which is 2^-39 of the largest; a rest of 0 counts as a step, that of the third term as another."""
    y, x, a, b, _, _ = make(tokens, tokens, 128, oc, 16, 3, HF, y_dtype)
    ids = runs(tokens, 3)
    size = 2.0 ** (-2 * torch.arange(16, device="cuda"))[:, None]
    a = (a.float() * 2 ** 6 * size).to(HF)
    for column in range(64):
        b[:, column, :column // 4] = 0
    y = y * 0 if y_dtype == FP else y
    out = ops().lora_add(y, x, a, b, ids).double()
    X, want, room = x.double(), y.double(), E * y.double().abs()
    for i in range(3):
        rows = ids == i
        A, B = a[i].double(), b[i].double()
        h, hh = X[rows] @ A.T, X[rows].abs() @ A.T.abs()
        off = h.abs() * 2.0 ** -22 + 2.0 ** -38 * h.abs().amax(1, keepdim=True) + 2 * E * (128 / 8 + 24) * hh
        want[rows] += h @ B.T
        room[rows] += off @ B.T.abs() + 2 * E * (3 * 16 + 4) * (hh @ B.T.abs()) + 2 * E * (h @ B.T).abs()
    bad = (out - want).abs() - (U[y_dtype] * want.abs() + room) * 1.001
    assert float(bad.max()) <= (2.0 ** -25 if y_dtype == HF else 0), float(bad.max())


# ------------------------------------------------------------------ sampling
@pytest.mark.parametrize("vocab,dtype", [(409600, FP), (409600, BF), (100003, BF), (32000, FP)])
@pytest.mark.parametrize("s", [dict(), dict(temperature=2.0), dict(min_p=1e-6)])
def test_log_of_the_probability_of_a_whole_row(vocab, dtype, s):
    """Nothing is listed: the sum is of all entries.  Its terms are good to 2^-22 + 3 2^-24 |z|, and are added in multiples of 2^-44 (n 2^-45
    of a sum of 1 or more): within 1e-5."""
    g = gen(vocab)
    logits, noise = (randn(g, 3, vocab) * 2).to(dtype), noise_of(g, 3, vocab)
    logits[2, 1:] = -0.5      # (the same term again and again)
    logits[2, 0] = 0.25
    token, logprob = ops().sample(logits, noise, **s, return_logprob=True)
    check_sample(logits, noise, token, logprob, s)


@pytest.mark.parametrize("vocab,dtype", [(100003, BF), (32000, FP), (60001, HF), (210011, FP)])
@pytest.mark.parametrize("s", [dict(), dict(top_k=100), dict(top_p=0.9), dict(min_p=1e-5, temperature=1.5)])
def test_a_row_is_the_same_in_every_batch(vocab, dtype, s):
    """Tokens and the bits of their probabilities, however many CTAs take a row."""
    g = gen(vocab)
    logits, noise = (randn(g, 150, vocab) * 3).to(dtype), noise_of(g, 150, vocab)
    whole = ops().sample(logits, noise, **s, return_logprob=True)
    for rows in (1, 9, 36, 70):
        part = ops().sample(logits[:rows], noise[:rows], **s, return_logprob=True)
        assert torch.equal(part[0], whole[0][:rows]) and torch.equal(part[1], whole[1][:rows])
    assert torch.equal(ops().sample(logits, noise, **s), whole[0])


@pytest.mark.parametrize("vocab", [7, 3001, 100003])
@pytest.mark.parametrize("s", [dict(), dict(top_k=1), dict(top_k=5, top_p=0.8), dict(top_p=0.5), dict(min_p=1.0), dict(min_p=0.3), dict(temperature=0.0)])
def test_noise_that_leaves_no_chance(vocab, s):
    """Variates of infinity: e / noise is 0 for every entry that stays, and the lowest index of the tie is the token; where one other
    stays with a finite variate it wins."""
    g = gen(vocab)
    logits = randn(g, 4, vocab) * 2
    logits[1, :vocab // 2] = -math.inf
    logits[2].clamp_(max=1.0)
    logits[3, 0] = logits[3, vocab - 1] = -math.inf
    noise = torch.full_like(logits, math.inf)
    cut = ops().filter_logits(logits, **s)
    first = (cut > -math.inf).int().argmax(1)
    token, logprob = ops().sample(logits, noise, **s, return_logprob=True)
    assert torch.equal(token, first)
    check_sample(logits, torch.where(torch.arange(vocab, device="cuda") == first[:, None], 1.0, 1e30), token, logprob, s)
    assert torch.equal(ops().sample(logits, torch.full_like(noise, math.nan), **s), first)
    last = vocab - 1 - (cut > -math.inf).flip(1).int().argmax(1)
    noise.scatter_(1, last[:, None], 3.0)
    if s.get("temperature") != 0:
        assert torch.equal(ops().sample(logits, noise, **s), last)


# ------------------------------------------------------------------ outputs
def test_outputs_that_overlap_are_refused():
    """Views of one buffer: on the input by some values, or rows on one another; parts side by side are taken."""
    from spark_b200._lib import SparkError
    from spark_b200 import rotary
    g = gen(1)
    flat = randn(g, 4 * 200 + 8)
    with pytest.raises(SparkError, match="overlaps"):
        ops().filter_logits(flat[:800].view(4, 200), top_k=3, out=flat[8:].view(4, 200))
    with pytest.raises(SparkError, match="one place"):
        ops().filter_logits(flat[:800].view(4, 200), top_k=3, out=torch.empty_like(flat).as_strided((4, 200), (100, 1)))
    both = randn(g, 4, 400)
    want = ops().filter_logits(both[:, :200].clone(), top_k=3)
    assert torch.equal(ops().filter_logits(both[:, :200], top_k=3, out=both[:, 200:]), want) and torch.equal(both[:, 200:], want)
    y, x, a, b, _, scale = make(3, 20, 64, 64, 8, 3, BF)
    ids = runs(20, 3)
    with pytest.raises(SparkError, match="overlaps"):
        ops().lora_add(y[:16], x[:16], a, b, ids[:16], scale=scale, out=y[4:])
    wide = torch.cat([x, y, y], 1)
    want = ops().lora_add(y, x, a, b, ids, scale=scale)
    assert torch.equal(ops().lora_add(wide[:, 64:128], wide[:, :64], a, b, ids, scale=scale, out=wide[:, 128:]), want)
    assert torch.equal(wide[:, :128], torch.cat([x, y], 1)) and torch.equal(wide[:, 128:], want)
    q, table, positions = randn(g, 1, 9, 4, 64, dtype=BF), rotary.rope_table(32, 64), torch.arange(8, device="cuda")[None]
    with pytest.raises(SparkError, match="overlaps"):
        ops().qk_norm_rope(q[:, :8], None, None, None, positions, table, out=(q[:, 1:], None))
    with pytest.raises(SparkError, match="output"):
        ops().qk_norm_rope(q[:, :8, :2], q[:, :8, 2:], None, None, positions, table, out=(q[:, :8, :2], q[:, :8, 1:3]))
    want = ops().qk_norm_rope(q[:, :8, :2], q[:, :8, 2:], None, None, positions, table)
    ops().qk_norm_rope(q[:, :8, :2], q[:, :8, 2:], None, None, positions, table, out=(q[:, :8, :2], q[:, :8, 2:]))
    assert torch.equal(q[:, :8, :2], want[0]) and torch.equal(q[:, :8, 2:], want[1])
