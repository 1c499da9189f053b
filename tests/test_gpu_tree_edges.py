"""The tree-decoding operators where their inputs are at the edge of what they
take: unused nodes, workspaces shared by graphs, sequences without pages, draws
from what little a rejection leaves, temperatures and contexts at the ends.

Tolerances as in test_gpu_tree_decode: u the unit roundoff of the tensors' type,
attention within 3 u max|v| and, over all values, within u of the norm.
"""
from __future__ import annotations

import importlib.util
import math
import os

import pytest
import torch

from test_gpu_tree_decode import (BF, FP, HF, attention64, check_attention, check_verify, gen,
                                  make, ops, randn, sees, verify_inputs)

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ rope
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rot", [(64, 32), (256, 64), (112, 28), (66, 6), (64, 64)])
def test_rope_in_place_outside_the_table_gives_zero_rows(d, rot, interleaved, dtype):
    from spark_b200 import SparkError
    from spark_b200.rotary import rope_table
    g = gen(2)
    table, pos = rope_table(10, rot), torch.tensor([3, 10, -1, 9], device="cuda")
    for both in (False, True):
        for shift in (0, 1):      # an address of whole 16 bytes, one that is none
            q, k = (torch.empty(4 * n * d + shift, dtype=dtype, device="cuda")[shift:].view(4, n, d).copy_(randn(g, 4, n, d, dtype=dtype))
                    for n in (6, 3))
            y, z = ops().rope(q, k if both else None, pos, table, interleaved)
            ops().rope(q, k if both else None, pos, table, interleaved, out=(q, k if both else None))
            assert torch.equal(q, y) and (q[1:3] == 0).all()
            assert not both or (torch.equal(k, z) and (k[1:3] == 0).all())
            with pytest.raises(SparkError, match="rotary table"):
                ops().check_device_errors()
    ops().check_device_errors()


def test_forward_mode_is_refused():
    """No tangent is lost in silence, with and without a gradient in reverse."""
    import torch.autograd.forward_ad as fwd
    from spark_b200.rotary import apply_rope, rope_table
    g = gen(3)
    table, pos = rope_table(20, 16), torch.arange(5, device="cuda")
    q, k, tangent = randn(g, 5, 2, 16), randn(g, 5, 1, 16), randn(g, 5, 2, 16)
    with fwd.dual_level():
        for x in (q, q.clone().requires_grad_()):
            dual = fwd.make_dual(x, tangent)
            for args in ((dual, k), (dual, None), (k, dual)):
                with pytest.raises(NotImplementedError, match="forward"):
                    apply_rope(*args, pos, table)
        apply_rope(q, k, pos, table)
        apply_rope(q, None, pos, table)


# ------------------------------------------------------------------ attention
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("b,t,hq,hkv,d,n", [
    (40, 6, 8, 8, 128, 60), (2, 6, 8, 2, 128, 900),       # most items whole; all in parts
    (60, 20, 32, 4, 64, 60), (3, 20, 32, 4, 64, 700),     # more than 128 rows an item
    (40, 5, 8, 8, 256, 70), (1, 5, 4, 4, 256, 900),
])
def test_unused_nodes_give_zero_rows(b, t, hq, hkv, d, n, dtype):
    """Whatever their queries and the values that others see hold."""
    g = gen(t)
    q, kt, vt, kc, vc, table, lens, parents = make(g, b, t, hq, hkv, d, [n] * b, 16, dtype)
    parents[:, t - 1] = -2
    want, want_lse = attention64(q, kt, vt, kc, vc, table, lens, parents, d ** -0.5)
    used = torch.tensor([[len(chain) > 0 for chain in sees(p)] for p in parents.tolist()], device="cuda")
    vmax = max(vt.abs().max().item(), vc.abs().max().item())
    for bad in (math.nan, math.inf, -math.inf):
        q2 = q.clone()
        q2[~used] = bad
        out, lse = ops().tree_attention(q2, kt, vt, kc, vc, table, lens, parents, return_lse=True)
        check_attention(out, lse, want, want_lse, vmax)
        # a value of the context that the used nodes see: theirs is what the formula gives, no number
        v2 = vc.clone()
        v2[table[:, 0].long(), 5, :, 3] = bad
        out, lse = ops().tree_attention(q, kt, vt, kc, v2, table, lens, parents, return_lse=True)
        assert (out[~used] == 0).all() and (lse[~used] == -math.inf).all()
        assert not torch.isfinite(out[..., 3][used]).any()
        assert torch.isfinite(out[..., 4:]).all() and torch.isfinite(lse[used]).all()
    ops().check_device_errors()


def test_tree_attention_of_expanded_inputs():
    """Queries, keys or values that a batch, the nodes or the heads share (stride 0) give
    what their copies give; an output or a cache of that kind is refused."""
    from spark_b200 import SparkError
    g = gen(14)
    q, kt, vt, kc, vc, table, lens, parents = make(g, 3, 4, 8, 2, 64, [100, 30, 0], 16, BF)
    args = (kc, vc, table, lens, parents)
    for dim in range(3):
        x, k, v = (t.narrow(dim, 0, 1).expand_as(t) for t in (q, kt, vt))
        for tree in ((x, kt, vt), (q, k, vt), (q, kt, v), (x, k, v)):
            assert torch.equal(ops().tree_attention(*tree, *args), ops().tree_attention(*(t.contiguous() for t in tree), *args))
        with pytest.raises(SparkError, match="strides"):
            ops().tree_attention(q, kt, vt, *args, out=x)
        with pytest.raises(SparkError, match="strides"):
            ops().tree_attention(q, kt, vt, kc.narrow(dim, 0, 1).expand_as(kc), *args[1:])
    ops().check_device_errors()


def test_a_workspace_as_the_header_asks_for_it():
    """Zeros where the C header says so, every bit set behind them, and nothing else done
    between calls; items in parts of several CTAs."""
    import ctypes
    from spark_b200 import _lib
    L = _lib.lib()
    g = gen(15)
    for b, t, hq, hkv, d, n in ((1, 1, 16, 16, 256, 1000), (2, 64, 8, 1, 128, 5000), (3, 9, 4, 2, 64, 900)):
        x = q, kt, vt, kc, vc, table, lens, parents = make(g, b, t, hq, hkv, d, [n] * b, 16, BF)
        want, lse = ops().tree_attention(*x, return_lse=True)
        out, lse2 = torch.empty_like(q), torch.empty_like(lse)
        c = _lib.SparkPagedCache(k=kc.data_ptr(), v=vc.data_ptr(), pages=kc.shape[0], page_size=16, kv_heads=hkv, head_dim=d,
                                 page_table=table.data_ptr(), page_table_stride=table.stride(0), max_pages=table.shape[1],
                                 lens=lens.data_ptr(), dtype=_lib.DTYPE_BF16)
        c.k_stride[:], c.v_stride[:] = kc.stride()[:3], vc.stride()[:3]
        a = _lib.SparkTreeAttention(cache=c, batch=b, nodes=t, q_heads=hq, q=q.data_ptr(), k=kt.data_ptr(), v=vt.data_ptr(),
                                    out=out.data_ptr(), parents=parents.data_ptr(), parents_stride=parents.stride(0),
                                    lse=lse2.data_ptr(), scale=d ** -0.5)
        a.q_stride[:], a.out_stride[:] = q.stride()[:3], out.stride()[:3]
        a.kn_stride[:], a.vn_stride[:] = kt.stride()[:3], vt.stride()[:3]
        size = L.spark_tree_attention_workspace_size(ctypes.byref(a))
        ws = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
        ws[:_lib.TREE_ATTENTION_ZEROED] = 0
        stream = torch.cuda.current_stream().cuda_stream
        for _ in range(3):
            out.zero_()
            assert L.spark_tree_attention(ctypes.byref(a), ctypes.c_void_p(ws.data_ptr()), size, ctypes.c_void_p(stream)) == _lib.OK
            assert torch.equal(out, want) and torch.equal(lse2, lse)
        assert int(ws[:_lib.TREE_ATTENTION_ZEROED].count_nonzero()) == 0


# ------------------------------------------------------------------ workspaces
def test_workspaces_born_in_a_capture(monkeypatch):
    """Their zeros are there before any replay, and no replay makes them anew: graphs of
    one stream are replayed in any order, and errors stay."""
    from spark_b200 import SparkError
    from spark_b200.rotary import rope_table
    g = gen(21)
    for name in ("_ws", "_chain_ws", "_tree_ws"):
        monkeypatch.setattr(ops(), name, {})
    stream = torch.cuda.Stream()
    rope_in, table = (randn(g, 4, 2, 64, dtype=BF), torch.tensor([3, 10, -1, 9], device="cuda")), rope_table(10, 32)
    cases, graphs = [], []
    for b, hq, n in ((2, 8, 900), (3, 8, 2000), (8, 32, 700)):
        x = make(g, b, 8, hq, 2, 128, [n] * b, 32, BF)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            turned = ops().rope(rope_in[0], None, rope_in[1], table)[0] if len(graphs) == 1 else None
            out, lse = ops().tree_attention(*x, return_lse=True)
            if not graphs:
                scratch = ops().workspace(x[0].device, 1 << 20)
        cases.append((x, out, lse, turned))
        graphs.append(graph)
    tree = [v for (_, s), v in [*ops()._tree_ws.items(), *ops()._tree_outgrown] if s == stream.cuda_stream]
    assert len(tree) >= 2 and all(int(v.count_nonzero()) == 0 for v in tree + [scratch])
    for i in (2, 1, 0, 1, 0, 2):
        x, out, lse, _ = cases[i]
        out.zero_()
        graphs[i].replay()
        want, want_lse = attention64(*x, 128 ** -0.5)
        check_attention(out, lse, want, want_lse, 5.0)
    # the second graph's bad positions, with a replay of each graph since
    with pytest.raises(SparkError, match="rotary table"):
        ops().check_device_errors()
    ops().check_device_errors()


def test_two_streams_at_once():
    """Each with a workspace of its own, their launches between one another's."""
    g = gen(22)
    cases = [make(g, 2, 8, 8, 2, 128, [900, 3000], 32, BF), make(g, 3, 20, 16, 4, 64, [1500, 10, 400], 16, BF)]
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        for s, x, to in zip(streams, cases, got):
            with torch.cuda.stream(s):
                to.append(ops().tree_attention(*x, return_lse=True))
    for s, x, to in zip(streams, cases, got):
        torch.cuda.current_stream().wait_stream(s)
        want, want_lse = attention64(*x, x[0].shape[-1] ** -0.5)
        check_attention(*to[0], want, want_lse, 5.0)
        assert all(torch.equal(a, b) for other in to for a, b in zip(to[0], other))
    ops().check_device_errors()


def test_errors_are_cleared_on_the_workspace_s_own_stream():
    """Work that the current stream still has to do neither holds the clearing back nor
    lets it fall on a later launch of the workspace's stream."""
    from spark_b200 import SparkError
    from spark_b200.rotary import rope_table
    q, bad, table = randn(gen(4), 4, 2, 64, dtype=BF), torch.full((4,), 99, device="cuda"), rope_table(10, 32)
    for stream in (torch.cuda.Stream(), torch.cuda.default_stream()):
        with torch.cuda.stream(stream):
            stream.wait_stream(torch.cuda.default_stream())
            ops().rope(q, None, bad, table)
        other = torch.cuda.Stream()
        with torch.cuda.stream(other):
            torch.cuda._sleep(200_000_000)       # about 0.1 s
            with pytest.raises(SparkError, match="rotary table"):
                ops().check_device_errors()
        with torch.cuda.stream(stream):
            ops().rope(q, None, bad, table)
        other.synchronize()
        with pytest.raises(SparkError, match="rotary table"):
            ops().check_device_errors()
        ops().check_device_errors()


def test_errors_of_a_replay_on_another_stream():
    """The check waits for the replay, which is not on the stream of its capture."""
    from spark_b200 import SparkError
    from spark_b200.rotary import rope_table
    q, bad, table = randn(gen(4), 4, 2, 64, dtype=BF), torch.full((4,), 99, device="cuda"), rope_table(10, 32)
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    ops().rope(q, None, bad * 0, table)
    with torch.cuda.graph(graph):
        ops().rope(q, None, bad, table)
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        torch.cuda._sleep(200_000_000)       # about 0.1 s
        graph.replay()
    with pytest.raises(SparkError, match="rotary table"):
        ops().check_device_errors()
    ops().check_device_errors()


def test_a_workspace_is_zero_on_the_stream_it_is_for(monkeypatch):
    """Not only once the current stream has got there."""
    monkeypatch.setattr(ops(), "_ws", {})
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        torch.full((1 << 20,), 255, dtype=torch.uint8, device="cuda")
    torch.full((1 << 20,), 255, dtype=torch.uint8, device="cuda")
    torch.cuda._sleep(200_000_000)       # about 0.1 s
    ws = ops().workspace(torch.device("cuda", torch.cuda.current_device()), 1 << 20, stream=stream)
    with torch.cuda.stream(stream):
        assert int(ws.count_nonzero()) == 0


# ------------------------------------------------------------------ verification
@pytest.mark.parametrize("dtype", [FP, BF])
@pytest.mark.parametrize("left,times", [(1e-4, 1), (0.1, 4), (0.02, 2)])
def test_what_a_rejection_leaves_is_summed_anew(left, times, dtype):
    """`times` children that leave `left` of the distribution each are rejected; the next
    one's chance is known to a part in 10000, the draws are that far from it.  (In fp32
    a chance is off by the rounding of logits below 32, 2^-20, a few times over; 1 minus
    the rejected ones would be off by 2^-24 / left^times, 6 parts in 10000 and more.)"""
    g = gen(17)
    b, v, t = 256, 1000, times + 2
    logits = torch.randn(b, 1, v, generator=g, device="cuda", dtype=torch.float64)
    logits[..., :times + 1] -= 20
    tokens = torch.zeros(b, t, dtype=torch.int64, device="cuda")
    for i in reversed(range(times)):
        # token i holds 1 - left of what the tokens after it leave
        rest = torch.cat([logits[:, 0, i + 1:times], logits[:, 0, times:]], 1) if i + 1 < times else logits[:, 0, times:]
        logits[:, 0, i] = torch.logsumexp(rest, -1) + math.log((1 - left) / left)
        tokens[:, 1 + i] = i
    logits = logits.expand(b, t, v).to(dtype)
    x = logits[:, 0].double()
    tokens[:, times + 1] = x[:, times:].argmax(-1) + times
    rest = x.clone()
    for i in range(times):
        rest[:, i] = -math.inf
    chance = torch.softmax(rest, -1).gather(1, tokens[:, times + 1:])[:, 0]
    sign = torch.where(torch.arange(b, device="cuda") % 2 == 0, 1.0, -1.0)
    u = torch.full((b, t), 1 - left / 10, device="cuda")
    u[:, times + 1] = (chance * (1 + 1e-4 * sign)).float()
    parents = torch.tensor([-1] + [0] * (t - 1), dtype=torch.int32, device="cuda")
    noise = torch.empty(b, v, device="cuda").exponential_(generator=g)
    path, n, _ = ops().tree_verify(logits, tokens, parents, u, noise)
    taken = sign < 0
    wrong = (n == 2) != taken
    assert not wrong.any(), int(wrong.sum())
    assert (path[:, 1] == torch.where(taken, times + 1, -1)).all()
    ops().check_device_errors()


def test_bad_token_ids_are_reported_at_any_temperature():
    from spark_b200 import SparkError
    g = gen(6)
    logits, u = torch.randn(1, 3, 300, generator=g, device="cuda"), torch.zeros(1, 3, device="cuda")
    noise = torch.empty(1, 300, device="cuda").exponential_(generator=g)
    parents = torch.tensor([-1, 0, 0], dtype=torch.int32, device="cuda")
    best = int(logits[0, 0].argmax())
    for temperature in (0.0, 1.0):
        for bad in (300, -1, 1 << 40, best + (1 << 32)):
            tokens = torch.tensor([[0, bad, best]], device="cuda")
            path, n, _ = ops().tree_verify(logits, tokens, parents, u, noise, temperature=temperature)
            assert path.tolist() == [[0, 2, -1]] and n.tolist() == [2]
            with pytest.raises(SparkError, match="vocabulary"):
                ops().check_device_errors()
    ops().check_device_errors()


@pytest.mark.parametrize("sampled", [True, False])
@pytest.mark.parametrize("v", [5, 300, 4096, 32768])
def test_temperatures_at_the_ends(v, sampled):
    """An infinite one is the uniform distribution of what is above -inf, the smallest
    ones are the argmax, a negative one turns the logits round."""
    g = gen(v)
    x = verify_inputs(g, 24, 6, v, FP, sampled)
    got = ops().tree_verify(*x[:5], draft_probs=x[5], temperature=math.inf)
    check_verify(x, got, math.inf)
    assert (got[2] >= 0).all()
    got = ops().tree_verify(*x[:5], draft_probs=x[5], temperature=-1.5)
    check_verify(x, got, -1.5)
    for tiny in (1e-20, 1e-37, 1e-44):
        check_verify(x, ops().tree_verify(*x[:5], draft_probs=x[5], temperature=tiny), tiny)
    logits = x[0].clone()
    logits[..., v // 2:] = -math.inf
    parents = torch.tensor([-1] + [-2] * 5, dtype=torch.int32, device="cuda")
    _, _, last = ops().tree_verify(logits, x[1], parents, x[3], x[4], temperature=math.inf)
    assert torch.equal(last, x[4][:, :v // 2].argmin(-1))
    got = ops().tree_verify(*x[:5], draft_probs=x[5], temperature=math.nan)
    assert (got[1] == 1).all() and (got[2] == -1).all()
    ops().check_device_errors()


# ------------------------------------------------------------------ the cache
def example():
    spec = importlib.util.spec_from_file_location(
        "example_tree_decode", os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "tree_decode.py"))
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    return ex


def test_rows_without_pages_leave_the_others_alone():
    """A batch whose first sequence is gone, and whose last never came, decodes what the
    second decodes by itself, and its pages are the same to the bit."""
    from spark_b200.tree_decode import PagedKVCache, tree_depths
    ex = example()
    model = ex.build()
    tree = torch.tensor([-1, 0, 0, 1], dtype=torch.int32, device="cuda")
    depths = tree_depths(tree.tolist()).cuda()
    prompt = torch.randint(0, 2048, (1, 21), generator=gen(1), device="cuda").expand(3, -1)
    tokens = torch.randint(0, 2048, (1, 4), generator=gen(2), device="cuda").expand(3, -1)
    u, noise = torch.full((3, 4), 0.5, device="cuda"), torch.ones(3, 2048, device="cuda")
    got = []
    for before in (True, False):
        c = PagedKVCache(2, 3, 64, 2, 64, page_size=8, pages=8)
        if before:
            c.reserve(0, 64)
            c.release(0)
        c.reserve(1, 40)
        model.prefill(prompt, c)
        if before:
            c.reserve(0, 16)
            c.release(0)
        pages = c.page_table[1, :5].long()
        path, n, last = model.step(tokens, tree, depths, c, u, noise, temperature=0.0)
        assert c.lens.tolist() == [0, 21 + int(n[1]), 0]
        got.append([path[1], last[1]] + [x[pages].clone() for x in c.k + c.v])
        others = torch.ones(8, dtype=torch.bool, device="cuda").index_fill_(0, pages, False)
        assert all((x[others] == 0).all() for x in c.k + c.v)
    assert all(torch.equal(a, b) for a, b in zip(*got))
    ops().check_device_errors()


def test_an_append_beyond_the_reserved_pages_is_reported():
    from spark_b200 import SparkError
    from spark_b200.tree_decode import PagedKVCache
    g = gen(3)
    c = PagedKVCache(1, 2, 64, 2, 64, page_size=8)
    c.reserve(0, 16)
    c.reserve(1, 32)
    k = randn(g, 2, 20, 2, 64, dtype=BF)
    c.append([(k, k)])
    with pytest.raises(SparkError, match="outside the cache"):
        ops().check_device_errors()
    for i, n in ((0, 16), (1, 20)):
        rows = c.k[0][c.page_table[i, :-(-n // 8)].long()].flatten(0, 1)
        assert torch.equal(rows[:n], k[i, :n]) and (rows[n:] == 0).all()
    kept = torch.zeros(16, dtype=torch.bool, device="cuda")
    kept[c.page_table[c.page_table >= 0].long()] = True
    assert (c.k[0][~kept] == 0).all()
    ops().check_device_errors()


def test_a_prompt_of_one_token():
    """Its prefill has no tokens."""
    ex = example()
    model = ex.build()
    new, steps = ex.generate(model, torch.tensor([[5], [9]], device="cuda"), 6, [-1])
    assert steps == 6 and [len(t) for t in new] == [6, 6]


# ------------------------------------------------------------------ append
def test_an_index_without_columns_appends_nothing():
    g = gen(5)
    _, _, _, kc, vc, table, n, _ = make(g, 2, 1, 2, 2, 64, [30, 20], 16, BF)
    k = randn(g, 2, 3, 2, 64, dtype=BF)
    before = kc.clone(), vc.clone()
    new = ops().kv_append(k, k, kc, vc, table, n, index=torch.zeros(2, 0, dtype=torch.int32, device="cuda"))
    assert torch.equal(new, n) and torch.equal(kc, before[0]) and torch.equal(vc, before[1])
    ops().check_device_errors()
