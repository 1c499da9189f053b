"""The tree operators together: a small packed decoder generates with a tree of
drafted tokens what it generates token by token, checked against a dense model.

The dense model has the decoded weights and computes in fp32; the packed one has
bf16 activations.  Its logits are of order 1 (unit-RMS input, weights of variance
1 / hidden) and off by the roundings of about ten bf16 operations on the way,
2^-8 each: 0.04 is one standard deviation at most, so that a greedy token's dense
logit lies within 0.3 of the largest."""
from __future__ import annotations

import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def example():
    spec = importlib.util.spec_from_file_location("example_tree_decode", os.path.join(ROOT, "examples", "tree_decode.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def dense_weight(lin):
    from spark_b200 import ops
    oc, ic = lin.out_features, lin.in_features
    if lin.fmt == "spfp2":
        return ops.spfp2_unpack(lin.w_packed, oc * ic).view(oc, ic)
    unpack = ops.fp3_unpack if lin.fmt == "fp3" else ops.nvfp4_unpack
    return unpack(lin.w_packed, lin.w_scales.view(torch.float8_e4m3fn), oc, ic)


def dense_logits(model, text, q_heads, kv_heads, d):
    """fp32 logits of every position of text [n]."""
    rms = lambda x: x * torch.rsqrt(x.square().mean(-1, keepdim=True) + torch.finfo(torch.bfloat16).eps)  # noqa: E731
    n = text.numel()
    x = model.embed(text).float()
    rot = model.table.shape[1]
    c, s = model.table[:n, None, :rot // 2], model.table[:n, None, rot // 2:]

    def turn(u):
        a, b = u[..., :rot // 2], u[..., rot // 2:rot]
        return torch.cat([a * c - b * s, b * c + a * s, u[..., rot:]], -1)

    for attention, gate_up, down in model.blocks:
        q, k, v = (rms(x) @ dense_weight(attention.qkv.merged).T).split(attention.qkv.splits, -1)
        q, k, v = turn(q.view(n, -1, d)), turn(k.view(n, -1, d)), v.view(n, -1, d)
        k, v = k.repeat_interleave(q_heads // kv_heads, 1), v.repeat_interleave(q_heads // kv_heads, 1)
        score = torch.einsum("qhd,khd->hqk", q, k) * d ** -0.5
        score = score.masked_fill(torch.ones(n, n, device="cuda").triu(1).bool(), float("-inf"))
        y = torch.einsum("hqk,khd->qhd", score.softmax(-1), v).reshape(n, -1)
        x = x + y @ dense_weight(attention.out_proj).T
        gu = (rms(x) @ dense_weight(gate_up.merged).T).view(n, -1, 2, 8)
        x = x + (torch.nn.functional.silu(gu[:, :, 0]) * gu[:, :, 1]).reshape(n, -1) @ dense_weight(down).T
    return rms(x) @ dense_weight(model.head).T


@pytest.mark.parametrize("batch", [1, 3])
def test_tree_generation_is_greedy_generation(batch):
    ex = example()
    model = ex.build()
    prompts = torch.randint(0, 2048, (batch, 75), generator=torch.Generator("cuda").manual_seed(batch), device="cuda")
    plain, plain_steps = ex.generate(model, prompts, 40, [-1])
    tree, steps = ex.generate(model, prompts, 40, ex.PARENTS)
    assert plain_steps == 40 and steps <= 40
    for new in (plain, tree):
        for i in range(batch):
            assert len(new[i]) == 40
            text = torch.tensor(prompts[i].tolist() + new[i], device="cuda")
            logits = dense_logits(model, text[:-1], 8, 2, 64)[74:]
            behind = logits.amax(-1) - logits.gather(1, text[75:, None])[:, 0]
            assert (behind <= 0.3).all(), behind.max().item()


def test_a_drafted_continuation_is_accepted_whole():
    """Drafts that are the model's own greedy tokens: every step takes all of them."""
    from spark_b200.tree_decode import PagedKVCache, tree_depths
    ex = example()
    model = ex.build(seed=3)
    prompt = torch.randint(0, 2048, (1, 20), generator=torch.Generator("cuda").manual_seed(5), device="cuda")
    known = ex.generate(model, prompt, 24, [-1])[0][0]
    cache = PagedKVCache(2, 1, 80, 2, 64, page_size=8)
    cache.reserve(0, 80)
    model.prefill(prompt[:, :-1], cache)
    parents = list(range(-1, 7))
    tree, depths = torch.tensor(parents, dtype=torch.int32, device="cuda"), tree_depths(parents).cuda()
    text = prompt[0].tolist()[-1:] + known
    noise, u = torch.ones(1, 2048, device="cuda"), torch.zeros(1, 8, device="cuda")
    for at in (0, 8):
        tokens = torch.tensor([text[at:at + 8]], device="cuda")
        path, n, last = model.step(tokens, tree, depths, cache, u, noise, temperature=0.0)
        assert n.tolist() == [8] and path.tolist() == [list(range(8))] and last.tolist() == [text[at + 8]]
    assert cache.lens.tolist() == [35]


def test_cache_pages_are_taken_and_given_back():
    from spark_b200.tree_decode import PagedKVCache
    c = PagedKVCache(1, 2, 64, 1, 64, page_size=16, pages=5)
    c.reserve(0, 33)
    c.reserve(0, 20)
    c.reserve(1, 30)
    assert len(set(c.page_table[0, :3].tolist() + c.page_table[1, :2].tolist())) == 5
    with pytest.raises(RuntimeError):
        c.reserve(1, 33)
    with pytest.raises(ValueError):
        c.reserve(0, 65)
    c.release(0)
    c.reserve(1, 64)
    with pytest.raises(ValueError):
        PagedKVCache(1, 1, 64, 1, 64, page_size=12)
