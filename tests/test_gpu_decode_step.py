"""The decode step's operators together: a small packed decoder with norms of q and k,
adapters for each sequence and sampling, against a dense model of the decoded weights.

Logits as in the tree decoder's own tests: of order 1, off by the roundings of some
bf16 operations, so that a greedy token's dense logit lies within 0.3 of the largest.
What stays of a distribution and which token is drawn is checked on the logits that the
model itself gives, in 64 bits."""
from __future__ import annotations

import pytest
import torch

from test_gpu_sample import cut64
from test_gpu_tree_model import dense_weight, example

pytestmark = pytest.mark.gpu

HIDDEN, VOCAB, Q_HEADS, KV_HEADS, D, POOL, RANK = 512, 2048, 8, 2, 64, 4, 8


def build(seed=0):
    """The example's decoder with norms in its attention blocks and adapters on q|k|v (none on k), out and down."""
    from spark_b200.inference_v3 import V3LoRALinear
    ex = example()
    model = ex.build(seed=seed)
    g = torch.Generator("cuda").manual_seed(seed + 1)

    def pair(out_features, in_features):
        a = (torch.randn(POOL, RANK, in_features, generator=g, device="cuda") * in_features ** -0.5).bfloat16()
        return a, (torch.randn(POOL, out_features, RANK, generator=g, device="cuda") * 0.2).bfloat16()

    scale = torch.rand(POOL, generator=g, device="cuda") + 0.5
    for block in model.blocks:
        attention, _, down = block
        attention.q_norm, attention.k_norm = ((1 + 0.3 * torch.randn(D, generator=g, device="cuda")).bfloat16() for _ in range(2))
        attention.qkv = V3LoRALinear(attention.qkv, [pair(Q_HEADS * D, HIDDEN), None, pair(KV_HEADS * D, HIDDEN)], scale=scale)
        attention.out_proj = V3LoRALinear(attention.out_proj, *pair(HIDDEN, Q_HEADS * D), scale=0.75)
        block[2] = V3LoRALinear(down, *pair(HIDDEN, down.in_features), scale=scale)
    return ex, model


def weight(layer, adapter):
    """The dense weight of a layer with a sequence's adapter (the parts of a merged one stacked)."""
    from spark_b200.inference_v3 import V3LoRALinear
    if not isinstance(layer, V3LoRALinear):
        return dense_weight(getattr(layer, "merged", layer))
    w = dense_weight(getattr(layer.base, "merged", layer.base)).float().clone()
    if adapter < 0:
        return w
    at = 0
    for i, width in enumerate(getattr(layer, "splits", [w.shape[0]])):
        if i in layer._parts:
            s = float(layer.scale[adapter]) if isinstance(layer.scale, torch.Tensor) else layer.scale
            w[at:at + width] += s * getattr(layer, f"b{i}")[adapter].float() @ getattr(layer, f"a{i}")[adapter].float()
        at += width
    return w


def dense_logits(model, text, adapter):
    rms = lambda x, eps=torch.finfo(torch.bfloat16).eps: x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)  # noqa: E731
    n, rot = text.numel(), model.table.shape[1]
    x = model.embed(text).float()
    c, s = model.table[:n, None, :rot // 2], model.table[:n, None, rot // 2:]

    def turn(u):
        a, b = u[..., :rot // 2], u[..., rot // 2:rot]
        return torch.cat([a * c - b * s, b * c + a * s, u[..., rot:]], -1)

    for attention, gate_up, down in model.blocks:
        q, k, v = (rms(x) @ weight(attention.qkv, adapter).T).split(attention.qkv.splits, -1)
        q, k, v = (u.reshape(n, -1, D) for u in (q, k, v))
        q, k = turn(rms(q, 1e-6) * attention.q_norm.float()), turn(rms(k, 1e-6) * attention.k_norm.float())
        k, v = (u.repeat_interleave(Q_HEADS // KV_HEADS, 1) for u in (k, v))
        score = torch.einsum("qhd,khd->hqk", q, k) * D ** -0.5
        score = score.masked_fill(torch.ones(n, n, device="cuda").triu(1).bool(), float("-inf"))
        x = x + torch.einsum("hqk,khd->qhd", score.softmax(-1), v).reshape(n, -1) @ weight(attention.out_proj, adapter).T
        gu = (rms(x) @ weight(gate_up, -1).T).view(n, -1, 2, 8)
        x = x + (torch.nn.functional.silu(gu[:, :, 0]) * gu[:, :, 1]).reshape(n, -1) @ weight(down, adapter).T
    return rms(x) @ weight(model.head, -1).T


def cache_of(model, prompts, room):
    from spark_b200.tree_decode import PagedKVCache
    cache = PagedKVCache(len(model.blocks), prompts.shape[0], room, KV_HEADS, D, page_size=16)
    for i in range(prompts.shape[0]):
        cache.reserve(i, room)
    model.prefill(prompts[:, :-1], cache)
    return cache


ADAPTERS = [2, -1, 0]


def test_decoding_follows_the_dense_model():
    """Greedy tokens, one at a time and by trees, each sequence with its own adapter (one with none)."""
    ex, model = build()
    prompts = torch.randint(0, VOCAB, (3, 70), generator=torch.Generator("cuda").manual_seed(7), device="cuda")
    model.use_adapters(torch.tensor(ADAPTERS, dtype=torch.int32, device="cuda"))
    cache = cache_of(model, prompts, 120)
    noise = torch.ones(3, VOCAB, device="cuda")
    last, plain = prompts[:, -1], []
    for _ in range(24):
        last, logprob = model.decode(last, cache, noise, temperature=0.0, return_logprob=True)
        assert (logprob == 0).all()
        plain.append(last)
    plain = torch.stack(plain, 1).tolist()
    by_trees, steps = ex.generate(model, prompts, 24, ex.PARENTS)
    assert steps <= 24
    for new in (plain, by_trees):
        for i, adapter in enumerate(ADAPTERS):
            text = torch.tensor(prompts[i].tolist() + new[i], device="cuda")
            logits = dense_logits(model, text[:-1], adapter)[69:]
            behind = logits.amax(-1) - logits.gather(1, text[70:, None])[:, 0]
            assert (behind <= 0.3).all(), (i, behind.max().item())
    # the adapters matter: without them other tokens come
    model.use_adapters(None)
    without = ex.generate(model, prompts, 24, [-1])[0]
    assert without[0] != plain[0] and without[2] != plain[2]


def test_sampling_keeps_to_what_stays():
    """Drawn tokens, and those accepted from a tree, are among what the settings leave of the model's own logits."""
    from spark_b200 import ops
    from spark_b200.tree_decode import tree_depths
    ex, model = build(3)
    g = torch.Generator("cuda").manual_seed(11)
    prompts = torch.randint(0, VOCAB, (3, 33), generator=g, device="cuda")
    model.use_adapters(torch.tensor([1, 3, -1], dtype=torch.int32, device="cuda"))
    cache = cache_of(model, prompts, 200)
    settings = [(0.8, 20, 0.9, 0.0), (1.1, 0, 0.7, 0.01), (0.6, 5, 1.0, 0.0)]
    t, k, p, least = (torch.tensor(v, dtype=d, device="cuda") for v, d in zip(zip(*settings), (torch.float32, torch.int32, torch.float32, torch.float32)))
    last = prompts[:, -1]
    for _ in range(4):
        logits, _ = model(last[:, None], model.root, model.root + 1, cache)
        noise = torch.empty(3, VOCAB, device="cuda").exponential_(generator=g)
        last = model.decode(last, cache, noise, temperature=t, top_k=k, top_p=p, min_p=least)
        for i, s in enumerate(settings):
            order, e, vague = cut64(logits[i, 0], s[0], s[1], float(p[i]), float(least[i]))
            chance = e / noise[i].double().cpu()[order]
            likely = order[chance >= chance.max() * (1 - 1e-4)].tolist()
            assert int(last[i]) in likely + vague
    tree, depths = torch.tensor(ex.PARENTS, dtype=torch.int32, device="cuda"), tree_depths(ex.PARENTS).cuda()
    for _ in range(4):
        tokens = ex.draft(model, cache, last, ex.PARENTS)
        logits, _ = model(tokens, tree, depths, cache)
        u, noise = torch.rand(3, len(ex.PARENTS), generator=g, device="cuda"), torch.empty(3, VOCAB, device="cuda").exponential_(generator=g)
        path, accepted, last = model.step(tokens, tree, depths, cache, u, noise, temperature=t, top_k=k, top_p=p, min_p=least)
        for i, s in enumerate(settings):
            nodes = path[i, :int(accepted[i])].tolist()
            for at, node in enumerate(nodes):
                took = int(tokens[i, nodes[at + 1]]) if at + 1 < len(nodes) else int(last[i])
                order, _, vague = cut64(logits[i, node], s[0], s[1], float(p[i]), float(least[i]))
                assert took in order.tolist() + vague
    ops.check_device_errors()


def test_adapters_of_layers():
    from spark_b200.inference_v3 import V3GateUpSiLU, V3LoRALinear, V3MergedLinear
    ex = example()
    g = torch.Generator("cuda").manual_seed(2)
    lin = [ex.linear("nvfp4", n, 256, g) for n in (128, 64)]
    a, b = torch.randn(3, 4, 256, generator=g, device="cuda").bfloat16(), torch.randn(3, 128, 4, generator=g, device="cuda").bfloat16()
    x = torch.randn(6, 256, generator=g, device="cuda").bfloat16()
    layer = V3LoRALinear(lin[0], a, b, scale=0.5)
    assert torch.equal(layer(x), lin[0](x))
    ids = torch.tensor([2, -1], dtype=torch.int32, device="cuda")
    layer.use(ids)
    y = lin[0](x)
    want = y.float()
    want[:3] += 0.5 * (x[:3].float() @ a[2].float().T) @ b[2].float().T
    assert torch.allclose(layer(x).float(), want, rtol=2.0 ** -8, atol=2.0 ** -8) and torch.equal(layer(x)[3:], y[3:])
    merged = V3LoRALinear(V3MergedLinear(lin), [(a, b), None])
    merged.use(ids)
    first, second = merged(x)
    assert torch.equal(second, V3MergedLinear(lin)(x)[1]) and not torch.equal(first[:3], V3MergedLinear(lin)(x)[0][:3])
    with pytest.raises(TypeError):
        V3LoRALinear(V3GateUpSiLU(lin[0], lin[0]), a, b)
    for bad in ((a[:, :, :8], b), (a, b[:, :64]), (a[:2], b), (a[0], b[0])):
        with pytest.raises(ValueError):
            V3LoRALinear(lin[0], *bad)
    with pytest.raises(ValueError):
        V3LoRALinear(V3MergedLinear(lin), [(a, b)])
    layer.use(torch.zeros(4, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError):
        layer(x)


def test_rows_that_have_ended():
    """A batch's sequence without pages, and one whose last draw gave nothing, leave the others' tokens as they are."""
    from spark_b200 import ops
    _, model = build(5)
    prompts = torch.randint(0, VOCAB, (3, 40), generator=torch.Generator("cuda").manual_seed(1), device="cuda")
    model.use_adapters(torch.tensor(ADAPTERS, dtype=torch.int32, device="cuda"))
    noise, got = torch.ones(3, VOCAB, device="cuda"), []
    for ended in (False, True):
        cache = cache_of(model, prompts, 60)
        last, tokens = prompts[:, -1].clone(), []
        if ended:
            cache.release(1)
            last[1] = -1
        for _ in range(8):
            last = model.decode(last, cache, noise, temperature=0.0)
            if ended:
                last[1] = -1
            tokens.append(last)
        got.append(torch.stack(tokens, 1))
    ops.check_device_errors()
    assert torch.equal(got[0][::2], got[1][::2]) and int(cache.lens[1]) == 0


def test_a_captured_step_takes_new_numbers():
    """One graph of a step: other adapters, settings, tokens and noise at each replay, and what the same calls give one by one."""
    from spark_b200 import ops
    _, model = build(6)
    g = torch.Generator("cuda").manual_seed(3)
    prompts = torch.randint(0, VOCAB, (4, 50), generator=g, device="cuda")
    ids = torch.zeros(4, dtype=torch.int32, device="cuda")
    model.use_adapters(ids)
    cache = cache_of(model, prompts, 64)
    last, noise = torch.zeros(4, dtype=torch.long, device="cuda"), torch.ones(4, VOCAB, device="cuda")
    heat, p = torch.ones(4, device="cuda"), torch.ones(4, device="cuda")
    k = torch.zeros(4, dtype=torch.int32, device="cuda")

    def step():
        logits, _ = model(last[:, None], model.root, model.root_depth, cache)
        return ops.sample(logits[:, 0], noise, temperature=heat, top_k=k, top_p=p, return_logprob=True)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(6):
        ids.copy_(torch.randint(-1, POOL, (4,), generator=g, device="cuda"))
        last.copy_(torch.randint(0, VOCAB, (4,), generator=g, device="cuda"))
        noise.exponential_(generator=g)
        heat.copy_(torch.tensor([0.0, 0.5, 1.0, 2.0], device="cuda").roll(i))
        p.copy_(torch.tensor([1.0, 0.9, 0.3, 0.99], device="cuda").roll(-i))
        k.copy_(torch.tensor([0, 3, 100, VOCAB], device="cuda").roll(i // 2))
        graph.replay()
        torch.cuda.synchronize()
        got = [u.clone() for u in out]
        assert all(torch.equal(u, v) for u, v in zip(got, step()))
