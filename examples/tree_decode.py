"""Generation with a tree of drafted tokens on packed weights: a random decoder
(NVFP4 embedding and head, FP3 attention, SPFP2 MLP), drafts by its first layer
alone, the tree verified against the whole model's logits.

    python examples/tree_decode.py [--tokens 64] [--temperature 0.0] [--top-k 0] [--top-p 1.0]

Prints the steps that the tokens took: with one token a step there would be as many
steps as tokens."""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from spark_b200 import ops  # noqa: E402
from spark_b200.inference_v3 import V3GateUpSiLU, V3MergedLinear, V3NVFP4Embedding, V3PackedLinear  # noqa: E402
from spark_b200.tree_decode import PagedKVCache, TreeAttention, TreeDecoder, tree_depths  # noqa: E402

# by depth: node 0 the last token, three guesses for the next one, continued one to three tokens deep
PARENTS = [-1, 0, 0, 0, 1, 2, 3, 4, 5, 7]


def linear(fmt: str, out_features: int, in_features: int, gen) -> V3PackedLinear:
    w = torch.randn(out_features, in_features, generator=gen, device="cuda") * in_features ** -0.5
    packed, scales = ops.spfp2_pack(w)[0], None
    if fmt != "spfp2":
        packed, scales = (ops.fp3_pack if fmt == "fp3" else ops.nvfp4_pack)(w)
    return V3PackedLinear(fmt, packed, out_features, in_features, scales=scales)


def build(vocab=2048, hidden=512, inter=1024, layers=2, q_heads=8, kv_heads=2, head_dim=64, rot_dim=32, seed=0) -> TreeDecoder:
    gen = torch.Generator("cuda").manual_seed(seed)
    embed = V3NVFP4Embedding(*ops.nvfp4_pack(torch.randn(vocab, hidden, generator=gen, device="cuda")), vocab, hidden,
                             dtype=torch.bfloat16)
    blocks = []
    for _ in range(layers):
        qkv = V3MergedLinear([linear("fp3", n * head_dim, hidden, gen) for n in (q_heads, kv_heads, kv_heads)])
        attention = TreeAttention(qkv, linear("nvfp4", hidden, q_heads * head_dim, gen), head_dim)
        gate_up = V3GateUpSiLU(linear("spfp2", inter, hidden, gen), linear("spfp2", inter, hidden, gen))
        blocks.append((attention, gate_up, linear("spfp2", hidden, inter, gen)))
    return TreeDecoder(embed, blocks, linear("nvfp4", vocab, hidden, gen), rot_dim, max_positions=4096)


def draft(first_layer: TreeDecoder, cache: PagedKVCache, last: torch.Tensor, parents: list[int]) -> torch.Tensor:
    """Tokens [batch, nodes] of the tree: the likeliest continuations by the model's
    first layer alone.  It shares the model's cache, whose first layer it would fill
    alike; the tree grows by one level a pass."""
    tree, depths = torch.tensor(parents, dtype=torch.int32, device=last.device), tree_depths(parents)
    tokens = torch.zeros(last.shape[0], len(parents), dtype=torch.int64, device=last.device)
    tokens[:, 0] = last
    for level in range(1, int(depths.max()) + 1):
        n = int((depths < level).sum())
        logits, _ = first_layer(tokens[:, :n], tree[:n], depths[:n].to(last.device), cache)
        for node in (depths == level).nonzero()[:, 0].tolist():
            rank = sum(p == parents[node] for p in parents[:node])
            tokens[:, node] = logits[:, parents[node]].topk(rank + 1).indices[:, rank]
    return tokens


def generate(model: TreeDecoder, prompts: torch.Tensor, n_tokens: int, parents: list[int], temperature=0.0, seed=0,
             vocab=2048, top_k=0, top_p=1.0):
    """([batch] lists of new tokens, steps)."""
    batch, dev = prompts.shape[0], prompts.device
    attention = model.blocks[0][0]
    room = prompts.shape[1] + n_tokens + len(parents)
    cache = PagedKVCache(len(model.blocks), batch, room, attention.kv_heads, attention.head_dim, page_size=16, device=dev)
    for i in range(batch):
        cache.reserve(i, room)
    model.prefill(prompts[:, :-1], cache)
    gen = torch.Generator(dev).manual_seed(seed)
    tree, depths = torch.tensor(parents, dtype=torch.int32, device=dev), tree_depths(parents).to(dev)
    first_layer = TreeDecoder(model.embed, list(model.blocks)[:1], model.head, model.table.shape[1], model.table.shape[0])
    text, steps = prompts.tolist(), 0
    while min(len(t) for t in text) < prompts.shape[1] + n_tokens:
        tokens = draft(first_layer, cache, torch.tensor([t[-1] for t in text], device=dev), parents)
        u = torch.rand(batch, len(parents), generator=gen, device=dev)
        noise = torch.empty(batch, vocab, device=dev).exponential_(generator=gen)
        path, accepted, last = model.step(tokens, tree, depths, cache, u, noise, temperature=temperature, top_k=top_k,
                                          top_p=top_p)
        steps += 1
        for i, (nodes, n, token) in enumerate(zip(path.tolist(), accepted.tolist(), last.tolist())):
            text[i] += [int(tokens[i, k]) for k in nodes[1:n]] + [token]
            if len(text[i]) >= prompts.shape[1] + n_tokens:
                # done: the others go on, this one keeps its last token
                text[i] = text[i][:prompts.shape[1] + n_tokens]
                cache.lens[i] = len(text[i]) - 1
    ops.check_device_errors()
    return [t[prompts.shape[1]:] for t in text], steps


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--tokens", type=int, default=64)
    ap.add_argument("--batch", type=int, default=1)
    ap.add_argument("--temperature", type=float, default=0.0)
    ap.add_argument("--top-k", type=int, default=0)
    ap.add_argument("--top-p", type=float, default=1.0)
    a = ap.parse_args()
    model = build()
    prompts = torch.randint(0, 2048, (a.batch, 40), generator=torch.Generator("cuda").manual_seed(1), device="cuda")
    how = {"temperature": a.temperature, "top_k": a.top_k, "top_p": a.top_p}
    _, plain = generate(model, prompts, a.tokens, [-1], **how)
    _, steps = generate(model, prompts, a.tokens, PARENTS, **how)
    print(f"{a.tokens} tokens a sequence: {plain} steps with one token a step, {steps} steps with a tree of {len(PARENTS)} nodes")


if __name__ == "__main__":
    main()
