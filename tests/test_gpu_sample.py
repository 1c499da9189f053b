"""Sampling and the cut of logits (ops.sample, ops.filter_logits) against the definition in
64 bits.

What stays is a set of entries: equal, unless a border is closer than the sums are good.
A sum of n exponentials in multiples of 2^-44 of the largest is off by at most n 2^-45;
where the mass before an entry is within 2 n 2^-45 of top_p times the whole, either side is
right.  min_p's border, an exponent in 64 bits that is rounded up to a logit of 32 bits, is
never closer than that in the cases here.
The token is argmax e / noise in fp32: the exponent is off by 3 2^-24 |z| (a difference, a factor and a
product), the exponential by 2^-22 and the quotient by 2^-23; a token that wins has |z| < 25 here: 4.9e-6
each.  Equal, unless the two largest quotients are within 1e-5.  logprob: z in 64 bits less the log of a sum of
such terms, most of the mass at |z| < 10: 2^-22 + 30 2^-24, and chains of at most 100 terms with trees of 10,
110 2^-24: within 1e-5 + 2^-22 |logprob|.
"""
from __future__ import annotations

import math

import pytest
import torch

from test_gpu_tree_decode import BF, FP, HF, gen, randn

pytestmark = pytest.mark.gpu


def ops():
    from spark_b200 import ops as _ops
    return _ops


def cut64(row, temperature, top_k, top_p, min_p):
    """(indices that stay, in falling order; their exponentials; indices of a border too close to call) of a row in
    64 bits; None without a distribution."""
    row = row.double().cpu() + 0.0
    top = row.max()
    if torch.isnan(row).any() or not math.isfinite(top) or not temperature >= 0:
        return None
    order = torch.argsort(row, descending=True, stable=True)
    if temperature == 0:
        return order[:1], torch.ones(1, dtype=torch.float64), []
    e = ((row[order] - top) / min(max(temperature, 1e-30), 1e30)).exp()
    n, vague = len(order), []
    if 0 < top_k < n:
        order, e, n = order[:top_k], e[:top_k], top_k
    if top_p < 1:
        before, whole = e.cumsum(0) - e, e.sum()
        near = (before - top_p * whole).abs() <= 2 * len(row) * 2.0 ** -45 * 1.01
        near[0] = False
        vague = order[near].tolist()
        n = max(1, int((before < top_p * whole).sum()))
    if min_p > 0:
        n = max(1, min(n, int((e >= min(min_p, 1.0)).sum())))
    return order[:n], e[:n], vague


def settings_of(s, i):
    return [float(v[i]) if isinstance(v, torch.Tensor) else v for v in (s.get("temperature", 1.0), s.get("top_k", 0), s.get("top_p", 1.0), s.get("min_p", 0.0))]


def check_filter(logits, out, s):
    assert out.shape == logits.shape and out.dtype == logits.dtype
    rows = logits.shape[1] if logits.dim() == 3 else 1
    x, y = logits.flatten(0, -2), out.flatten(0, -2)
    for i in range(x.shape[0]):
        temperature, k, p, least = settings_of(s, i // rows)
        cut = cut64(x[i], temperature, int(k), p, least)
        if cut is None:
            assert torch.equal(x[i].view(torch.int16 if x.element_size() == 2 else torch.int32), y[i].view(torch.int16 if x.element_size() == 2 else torch.int32))
            continue
        order, _, vague = cut
        want = torch.full((x.shape[1],), -math.inf, dtype=torch.float64)
        want[order] = x[i].double().cpu()[order]
        got = y[i].double().cpu()
        if vague:
            want[vague] = got[vague] = 0
        assert torch.equal(got, want), (i, temperature, k, p, least, (got != want).nonzero()[:5], len(order))


def check_sample(logits, noise, token, logprob, s):
    for i in range(logits.shape[0]):
        temperature, k, p, least = settings_of(s, i)
        cut = cut64(logits[i], temperature, int(k), p, least)
        if cut is None:
            assert int(token[i]) == -1 and math.isnan(float(logprob[i]))
            continue
        order, e, vague = cut
        chance = e / noise[i].double().cpu()[order] if temperature else e
        best = chance.max()
        likely = order[chance >= best * (1 - 1e-5)].tolist()
        t = int(token[i])
        if len(likely) == 1 or bool((chance == best).sum() == len(likely)):
            assert t == min(likely) or t in vague, (i, t, likely)
        else:
            assert t in likely or t in vague
        if t not in vague:
            want = float((e[order == t][0] / e.sum()).log())
            assert abs(float(logprob[i]) - want) <= 1e-5 + 2.0 ** -22 * abs(want), (float(logprob[i]), want)


KINDS = [dict(), dict(temperature=0.7), dict(temperature=0.0), dict(top_k=1), dict(top_k=50), dict(top_k=700), dict(top_p=0.9),
         dict(top_p=0.01, temperature=2.0), dict(min_p=0.05, temperature=1.3), dict(temperature=0.7, top_k=40, top_p=0.95, min_p=0.02),
         dict(top_k=2000, top_p=0.999), dict(top_p=0.9999999), dict(top_p=0.0), dict(min_p=1.0), dict(temperature=0.05, top_k=300),
         dict(temperature=30.0, top_p=0.5), dict(temperature=30.0, top_k=5000, top_p=0.5)]


def noise_of(g, *shape):
    return torch.empty(*shape, device="cuda").exponential_(generator=g).clamp_(min=1e-30)


@pytest.mark.parametrize("dtype", [FP, BF, HF])
@pytest.mark.parametrize("vocab", [1, 2, 5, 17, 128, 1000, 8191, 32000, 100003])
def test_cut_and_token(vocab, dtype):
    g = gen(vocab)
    logits = (randn(g, 3, vocab) * 4).to(dtype)
    noise = noise_of(g, 3, vocab)
    for s in KINDS:
        out = ops().filter_logits(logits, **s)
        check_filter(logits, out, s)
        token, logprob = ops().sample(logits, noise, **s, return_logprob=True)
        check_sample(logits, noise, token, logprob, s)
        assert torch.equal(token, ops().sample(logits, noise, **s))
        assert torch.equal(out, ops().filter_logits(logits, **s))


@pytest.mark.parametrize("rows", [1, 40, 300])
def test_rows_with_their_own_settings(rows):
    """Clusters of every size: few and many rows, settings of each as tensors."""
    g = gen(rows)
    for vocab, dtype in ((1003, FP), (20001, BF), (60000, FP)):
        logits, noise = (randn(g, rows, vocab) * 3).to(dtype), noise_of(g, rows, vocab)
        pick = [KINDS[i % len(KINDS)] for i in range(rows)]
        s = {"temperature": torch.tensor([k.get("temperature", 1.0) for k in pick], device="cuda"),
             "top_k": torch.tensor([k.get("top_k", 0) for k in pick], dtype=torch.int32, device="cuda"),
             "top_p": torch.tensor([k.get("top_p", 1.0) for k in pick], device="cuda"),
             "min_p": torch.tensor([k.get("min_p", 0.0) for k in pick], device="cuda")}
        check_filter(logits[:60], ops().filter_logits(logits, **s)[:60], s)
        token, logprob = ops().sample(logits, noise, **s, return_logprob=True)
        check_sample(logits[:60], noise, token, logprob, s)
        # the same row alone, its settings as numbers
        for i in (0, rows - 1):
            alone, lp = ops().sample(logits[i:i + 1], noise[i:i + 1], **pick[i], return_logprob=True)
            check_sample(logits[i:i + 1], noise[i:i + 1], alone, lp, pick[i])


@pytest.mark.parametrize("dtype", [FP, BF, HF])
def test_ties(dtype):
    """Equal logits, more of them than are compared at once: the lowest indices stay."""
    g = gen(3)
    vocab = 6000
    rows = [torch.zeros(vocab, device="cuda"), randn(g, vocab).round(), (randn(g, vocab) * 0.3).round(), randn(g, vocab).clamp(max=0.5),
            torch.where(torch.arange(vocab, device="cuda") % 2 == 0, 0.0, -0.0), torch.full((vocab,), -7.25, device="cuda")]
    rows[3][4000] = 2
    logits, noise = torch.stack(rows).to(dtype), noise_of(g, len(rows), vocab)
    for s in [dict(top_k=k) for k in (1, 511, 513, 700, 3001, 5999, 6000)] + [dict(top_p=p) for p in (0.001, 0.1, 0.3337, 0.5, 0.97)] + \
             [dict(top_k=3000, top_p=0.4), dict(top_k=600, top_p=0.999), dict(min_p=1.0), dict(temperature=0.0)]:
        check_filter(logits, ops().filter_logits(logits, **s), s)
        token, logprob = ops().sample(logits, noise, **s, return_logprob=True)
        check_sample(logits, noise, token, logprob, s)
    same = torch.ones_like(noise)
    assert ops().sample(logits, same).tolist() == [int((r.double() + 0.0).argmax()) for r in logits]


@pytest.mark.parametrize("dtype", [FP, BF, HF])
def test_masked_and_extreme_rows(dtype):
    g = gen(4)
    vocab, inf, low = 3001, math.inf, torch.finfo(dtype).min
    x = (randn(g, 12, vocab) * 3).to(dtype)
    x[0, 5:] = -inf
    x[1, :] = -inf
    x[1, 77] = -3.0
    x[2, :] = -inf
    x[3, 100] = math.nan
    x[4, 9] = inf
    x[5, 100:] = low
    x[6, :] = low
    x[7, :2500] = -inf
    x[8, :] = torch.finfo(dtype).max
    x[8, 7:] = low
    x[9] *= 1000
    x[10] *= 1e-3
    x[11, ::3] = low
    noise = noise_of(g, 12, vocab)
    for s in KINDS + [dict(temperature=1e-35, top_p=0.9), dict(temperature=1e35, top_p=0.25), dict(temperature=1e-35, top_k=3),
                      dict(temperature=1e20, top_k=100, top_p=0.5), dict(temperature=math.inf, min_p=0.5), dict(top_k=2999)]:
        check_filter(x, ops().filter_logits(x, **s), s)
        token, logprob = ops().sample(x, noise, **s, return_logprob=True)
        check_sample(x, noise, token, logprob, s)


def test_settings_that_mean_nothing():
    """Tensors are not looked at on the host: a negative or NaN temperature gives no token, NaN and out-of-range
    settings count as the nearest that means something."""
    g = gen(5)
    x, noise = randn(g, 9, 2000) * 3, noise_of(g, 9, 2000)
    nan = math.nan
    s = {"temperature": torch.tensor([-1.0, nan, 1, 1, 1, 1, 1, 1, math.inf], device="cuda"),
         "top_k": torch.tensor([0, 0, -5, 2 ** 31 - 1, 0, 0, 0, 0, 0], dtype=torch.int32, device="cuda"),
         "top_p": torch.tensor([1, 1, 1, 1, nan, -1, 2, 1, 1], device="cuda"),
         "min_p": torch.tensor([0, 0, 0, 0, 0, 0, 0, nan, 0], device="cuda")}
    token, logprob = ops().sample(x, noise, **s, return_logprob=True)
    assert token[:2].tolist() == [-1, -1] and torch.isnan(logprob[:2]).all()
    plain = ops().sample(x, noise)
    assert torch.equal(token[[2, 3, 4, 6, 7]], plain[[2, 3, 4, 6, 7]]) and int(token[5]) == int(x[5].argmax())
    out = ops().filter_logits(x, **s)
    assert torch.equal(out[[0, 1, 2, 3, 4, 6, 7, 8]], x[[0, 1, 2, 3, 4, 6, 7, 8]])
    assert torch.isfinite(out[5]).sum() == 1
    assert int(token[8]) == int(noise[8].argmin())
    s["min_p"][:] = 7.0
    out = ops().filter_logits(x, **s)
    assert (torch.isfinite(out[2:]).sum(1)[:6] == 1).all()


def test_layouts():
    """Rows at odd addresses, strided rows and nodes, a vocabulary of every other value, in place."""
    g = gen(6)
    s = dict(temperature=0.8, top_k=100, top_p=0.9)
    for dtype in (FP, BF):
        big = (randn(g, 4, 3, 1013) * 4).to(dtype)
        for view in (big[..., 3:1003], big[:, 1:, 1:], big.transpose(0, 1), big[..., ::2], big[:1].expand(4, 3, 1013)):
            out = ops().filter_logits(view, **s)
            check_filter(view, out, s)
            into = torch.full((*view.shape[:2], view.shape[2] + 5), 9.0, dtype=dtype, device="cuda")
            ops().filter_logits(view, **s, out=into[..., 2:-3])
            assert torch.equal(into[..., 2:-3], out) and (into[..., :2] == 9).all() and (into[..., -3:] == 9).all()
        noise = noise_of(g, 3, 4, 1010).transpose(0, 1)[:, 1]
        token, logprob = ops().sample(big[:, 1, 2:1012], noise, **s, return_logprob=True)
        check_sample(big[:, 1, 2:1012], noise, token, logprob, s)
        copy = big.clone()
        got = ops().filter_logits(copy, **s, out=copy)
        assert got.data_ptr() == copy.data_ptr()
        check_filter(big, copy, s)


def test_largest_vocabulary_and_no_rows():
    g = gen(7)
    for dtype in (FP, BF):
        x, noise = (randn(g, 2, 409600) * 2).to(dtype), noise_of(g, 2, 409600)
        for s in (dict(top_p=0.9), dict(top_k=2000, top_p=0.95), dict(top_k=300000), dict()):
            check_filter(x, ops().filter_logits(x, **s), s)
            token, logprob = ops().sample(x, noise, **s, return_logprob=True)
            if s:   # (the log of a sum of so many terms in fp32 is not covered by the bound above)
                check_sample(x, noise, token, logprob, s)
    assert ops().sample(torch.zeros(0, 10, device="cuda"), torch.zeros(0, 10, device="cuda")).shape == (0,)
    assert ops().filter_logits(torch.zeros(3, 0, 10, device="cuda")).shape == (3, 0, 10)


def test_refusals():
    from spark_b200._lib import SparkError
    x, e = torch.zeros(2, 10, device="cuda"), torch.ones(2, 10, device="cuda")
    f, cut = ops().sample, ops().filter_logits
    for args, kw, error in [
        ((x.cpu(), e), {}, RuntimeError), ((x, e.cpu()), {}, RuntimeError), ((x, e.half()), {}, TypeError), ((x, e[:, :5]), {}, ValueError),
        ((x[0], e[0]), {}, ValueError), ((x.double(), e), {}, TypeError), ((x[:, :0], e[:, :0]), {}, ValueError),
        ((x, e), dict(temperature=-1.0), ValueError), ((x, e), dict(temperature=math.nan), ValueError), ((x, e), dict(top_k=-1), ValueError),
        ((x, e), dict(top_p=1.5), ValueError), ((x, e), dict(top_p=math.nan), ValueError), ((x, e), dict(min_p=-0.1), ValueError),
        ((x, e), dict(min_p=1.1), ValueError), ((x, e), dict(temperature=torch.ones(3, device="cuda")), TypeError),
        ((x, e), dict(top_k=torch.ones(2, device="cuda")), TypeError), ((x, e), dict(top_p=torch.ones(2)), TypeError),
        ((x, e), dict(top_k=2.5), TypeError),
    ]:
        with pytest.raises(error):
            f(*args, **kw)
    for out in (x.half(), x[:, :5], torch.zeros(10, 2, device="cuda").t()):
        with pytest.raises(ValueError):
            cut(x, out=out)
    with pytest.raises(SparkError):
        cut(x, out=x[:1].expand(2, 10))
    with pytest.raises(SparkError, match="409600"):
        cut(torch.zeros(1, 409601, dtype=BF, device="cuda"))


def test_captured_and_on_another_stream():
    g = gen(8)
    x, noise = (randn(g, 5, 32000) * 4).to(BF), noise_of(g, 5, 32000)
    t = torch.tensor([0.5, 1.0, 0.0, 0.9, 2.0], device="cuda")
    s = dict(temperature=t, top_k=60, top_p=0.9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops().sample(x, noise, **s)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, ops().sample(x, noise, **s))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cut = ops().filter_logits(x, **s)
        token, logprob = ops().sample(cut, noise, temperature=t, return_logprob=True)
    for seed in (1, 2):
        x.copy_(randn(gen(seed), 5, 32000) * 4)
        t.mul_(0.8)
        graph.replay()
        check_filter(x, cut, s)
        check_sample(x, noise, token, logprob, s)


def test_settings_of_one_sequence_stay_on_the_device():
    """Tensors of one value each, in a graph: replays follow them."""
    g = gen(9)
    x, noise = randn(g, 1, 5000) * 3, noise_of(g, 1, 5000)
    s = {"temperature": torch.tensor([0.7], device="cuda"), "top_k": torch.tensor([20], dtype=torch.int32, device="cuda"),
         "top_p": torch.tensor([0.9], device="cuda"), "min_p": torch.tensor([0.01], device="cuda")}
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cut = ops().filter_logits(x, **s)
        token, logprob = ops().sample(x, noise, **s, return_logprob=True)
    for k in (20, 3, 1000):
        s["top_k"].fill_(k)
        graph.replay()
        check_filter(x, cut, s)
        check_sample(x, noise, token, logprob, s)


@pytest.mark.parametrize("vocab,dtype", [(3000, FP), (32000, FP), (32000, BF), (120000, FP)])
def test_borders_that_only_good_sums_tell(vocab, dtype):
    """top_p within 1e-8 of the mass before an entry, on either side: sums in 32 bits of what is far below would not do."""
    x = (randn(gen(vocab), 1, vocab) * 4).to(dtype)
    row = x[0].double().cpu()
    e = (row.sort(descending=True).values - row.max()).exp()
    before = (e.cumsum(0) - e) / e.sum()
    for share in (0.5, 0.8, 0.93):
        i = int((before < share).sum())
        for p in (float(before[i]) * (1 + 1e-8), float(before[i]) * (1 - 1e-8)):
            assert cut64(row, 1.0, 0, p, 0.0)[2] == [] and len(cut64(row, 1.0, 0, p, 0.0)[0]) == (i + 1 if p > before[i] else i)
            check_filter(x, ops().filter_logits(x, top_p=p), dict(top_p=p))


@pytest.mark.parametrize("dtype", [FP, BF, HF])
@pytest.mark.parametrize("vocab", [1001, 70003])
def test_rows_of_the_lowest_value(vocab, dtype):
    """Masks of the type's lowest value beside -inf, in rows that begin inside a vector: fewer entries than top_k."""
    low = torch.finfo(dtype).min
    logits = torch.full((5, vocab), -math.inf, dtype=dtype, device="cuda")
    for i in range(4):
        logits[i, [0, vocab - 1, vocab // 2, 7][i]] = low
    logits[4] = low
    noise = noise_of(gen(5), 5, vocab)
    for s in (dict(top_k=5), dict(top_k=900), dict(top_p=0.9), dict(top_k=40, top_p=0.5, temperature=3.0), dict(top_k=5, temperature=1e30), dict()):
        check_filter(logits, ops().filter_logits(logits, **s), s)
        token, logprob = ops().sample(logits, noise, **s, return_logprob=True)
        check_sample(logits, noise, token, logprob, s)


@pytest.mark.parametrize("dtype", [FP, BF])
def test_many_rows_of_wide_distributions(dtype):
    """Rows whose top_p takes more entries than the first list has, whole rows, and borders that sums in fp32 leave open."""
    g = gen(17)
    logits = (randn(g, 160, 20011) * torch.tensor([0.5, 2.0, 3.0, 4.0], device="cuda").repeat(40)[:, None]).to(dtype)
    p = torch.rand(160, generator=g, device="cuda") * 0.2 + 0.79
    s = dict(top_p=p)
    check_filter(logits, ops().filter_logits(logits, **s), s)
    check_filter(logits[:8], ops().filter_logits(logits[:8], top_p=p[:8]), dict(top_p=p[:8]))


@pytest.mark.parametrize("rows,vocab,dtype", [(1, 50021, BF), (10, 50021, HF), (30, 30011, FP), (40, 90001, BF), (64, 100003, HF), (70, 90001, BF),
                                              (150, 30011, FP), (300, 20011, BF), (20, 110003, FP), (40, 110003, FP), (2, 210011, FP)])
def test_rows_by_ctas_and_clusters(rows, vocab, dtype):
    """Numbers and lengths of rows that one CTA takes, and clusters of 4 and 8, alone on an SM and two of them."""
    g = gen(rows)
    logits, noise = (randn(g, rows, vocab) * 4).to(dtype), noise_of(g, rows, vocab)
    kinds = [(1.0, 0, 0.95, 0.0), (0.7, 50, 0.9, 0.0), (1.2, 900, 0.99, 0.01), (2.0, 0, 0.9, 0.0), (0.9, 0, 1.0, 0.0)]
    values = list(zip(*(kinds[i % 5] for i in range(rows))))
    s = {n: torch.tensor(v, dtype=torch.int32 if n == "top_k" else FP, device="cuda") for n, v in zip(("temperature", "top_k", "top_p", "min_p"), values)}
    out = ops().filter_logits(logits, **s)
    token, logprob = ops().sample(logits, noise, **s, return_logprob=True)
    some = torch.randperm(rows, generator=torch.Generator().manual_seed(rows))[:8].cuda()
    cut = {n: v[some] for n, v in s.items()}
    check_filter(logits[some], out[some], cut)
    check_sample(logits[some], noise[some], token[some], logprob[some], cut)


@pytest.mark.parametrize("rows,vocab,dtype", [(200, 20011, BF), (3, 100003, FP)])
def test_the_same_inputs_give_the_same_bits(rows, vocab, dtype):
    """Tokens and their probabilities whatever the order of atomics."""
    g = gen(29)
    logits, noise = (randn(g, rows, vocab) * 3).to(dtype), noise_of(g, rows, vocab)
    for s in (dict(top_k=300), dict(top_k=2000, top_p=0.95), dict(top_p=0.9), dict(top_p=0.99, temperature=2.0), dict()):
        first = ops().sample(logits, noise, **s, return_logprob=True)
        for _ in range(20):
            assert all(torch.equal(u, v) for u, v in zip(first, ops().sample(logits, noise, **s, return_logprob=True)))
