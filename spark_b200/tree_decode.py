"""Decoding with a tree of drafted tokens: the paged K/V cache, one attention
block and a small decoder around the operators of ops (rope or qk_norm_rope,
tree_attention, filter_logits, tree_verify, sample, kv_append) and the packed
linears, with or without adapters (inference_v3.V3LoRALinear).

A step takes T tokens a sequence (node 0 the last accepted token, the others
drafted, `parents` says on which node each hangs), runs the layers on all of
them at once -- the packed linears read their weights once for up to 16 tokens --
and verifies the tree against the resulting logits; the K/V rows of accepted
nodes go into the cache.  T = 1 is plain decoding, a chain of T prompt tokens is
prefill.  The reference generates token by token through its model library
(04_scripts/inference_v3.py:108-123).
"""
from __future__ import annotations

import torch
from torch import nn

from . import ops
from .inference_v3 import V3LoRALinear
from .rotary import rope_table


class PagedKVCache:
    """K and V of `layers` layers in pages of `page_size` tokens that sequences
    take from a common pool; the page table and the lengths are shared by the
    layers.  k[l], v[l]: [pages, page_size, kv_heads, head_dim]; page_table int32
    [batch, max_pages], -1 where a sequence has no page (nothing is written or read
    there: an append beyond what is reserved is reported); lens int32 [batch]; held
    int32 [batch], 1 where a sequence has pages: a batch's other rows take part in a
    step, but nothing of theirs is kept."""

    def __init__(self, layers: int, batch: int, max_tokens: int, kv_heads: int, head_dim: int, page_size: int = 64,
                 pages: int | None = None, dtype=torch.bfloat16, device="cuda"):
        if page_size % 8 or head_dim % 8:
            raise ValueError("PagedKVCache: page_size and head_dim must be multiples of 8")
        self.page_size, self.max_pages = page_size, -(-max_tokens // page_size)
        pages = batch * self.max_pages if pages is None else pages
        shape = (pages, page_size, kv_heads, head_dim)
        self.k = [torch.zeros(shape, dtype=dtype, device=device) for _ in range(layers)]
        self.v = [torch.zeros(shape, dtype=dtype, device=device) for _ in range(layers)]
        self.page_table = torch.full((batch, self.max_pages), -1, dtype=torch.int32, device=device)
        self.lens = torch.zeros(batch, dtype=torch.int32, device=device)
        self.held = torch.zeros(batch, dtype=torch.int32, device=device)
        self._free = list(range(pages - 1, -1, -1))
        self._taken: list[list[int]] = [[] for _ in range(batch)]

    def reserve(self, sequence: int, tokens: int) -> None:
        """Gives the sequence pages for `tokens` tokens in all."""
        need = -(-tokens // self.page_size) - len(self._taken[sequence])
        if need <= 0:
            return
        if tokens > self.max_pages * self.page_size:
            raise ValueError(f"PagedKVCache: {tokens} tokens, a sequence holds {self.max_pages * self.page_size}")
        if need > len(self._free):
            raise RuntimeError(f"PagedKVCache: {need} pages wanted, {len(self._free)} free")
        at = len(self._taken[sequence])
        new = [self._free.pop() for _ in range(need)]
        self._taken[sequence] += new
        self.page_table[sequence, at:at + need] = torch.tensor(new, dtype=torch.int32, device=self.page_table.device)
        self.held[sequence] = 1

    def release(self, sequence: int) -> None:
        """Takes the sequence's pages back and empties it."""
        self._free += reversed(self._taken[sequence])
        self._taken[sequence] = []
        self.page_table[sequence] = -1
        self.lens[sequence] = self.held[sequence] = 0

    def attend(self, layer: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, parents: torch.Tensor, **kw):
        return ops.tree_attention(q, k, v, self.k[layer], self.v[layer], self.page_table, self.lens, parents, **kw)

    def append(self, new: list, index: torch.Tensor | None = None, counts: torch.Tensor | None = None) -> None:
        """Every layer's (k, v) of a step [batch, nodes, kv_heads, head_dim]: the rows
        that index and counts name (ops.kv_append) go behind each sequence's tokens; none
        of a sequence without pages."""
        lens = self.lens
        width = (new[0][0] if index is None else index).shape[1]
        counts = self.held * (width if counts is None else counts)
        for layer, (k, v) in enumerate(new):
            lens = ops.kv_append(k, v, self.k[layer], self.v[layer], self.page_table, self.lens, index=index, counts=counts)
        self.lens = lens


def tree_depths(parents) -> torch.Tensor:
    """int32 depth of each node of a tree given as a list of parents (0 on the context)."""
    depth = []
    for p in parents:
        depth.append(depth[p] + 1 if p >= 0 else 0)
    return torch.tensor(depth, dtype=torch.int32)


class TreeAttention(nn.Module):
    """Attention block: q|k|v (an inference_v3.V3MergedLinear, or one with adapters), rotary
    positions, with q_norm and k_norm [head_dim] after RMS norms of each head, tree
    attention, output projection."""

    def __init__(self, qkv, out_proj, head_dim: int, interleaved: bool = False, q_norm: torch.Tensor | None = None,
                 k_norm: torch.Tensor | None = None, eps: float = 1e-6):
        super().__init__()
        if (q_norm is None) != (k_norm is None):
            raise ValueError("TreeAttention: q_norm and k_norm come together")
        self.qkv, self.out_proj, self.eps = qkv, out_proj, eps
        self.register_buffer("q_norm", q_norm)
        self.register_buffer("k_norm", k_norm)
        self.head_dim, self.interleaved = head_dim, interleaved
        self.kv_heads = qkv.splits[1] // head_dim

    def forward(self, x: torch.Tensor, positions: torch.Tensor, table: torch.Tensor, parents: torch.Tensor,
                cache: PagedKVCache, layer: int):
        """x [batch, nodes, hidden] -> (y, (k, v)); k and v are the nodes', not yet in the cache."""
        b, t, _ = x.shape
        q, k, v = (u.unflatten(-1, (-1, self.head_dim)).unflatten(0, (b, t)) for u in self.qkv(x.reshape(b * t, -1)))
        # in place: q and k are parts of the projection's output
        if self.q_norm is None:
            q, k = ops.rope(q, k, positions, table, interleaved=self.interleaved, out=(q, k))
        else:
            q, k = ops.qk_norm_rope(q, k, self.q_norm, self.k_norm, positions, table, eps=self.eps,
                                    interleaved=self.interleaved, out=(q, k))
        y = cache.attend(layer, q, k, v, parents)
        return self.out_proj(y.reshape(b * t, -1)).reshape(b, t, -1), (k, v)


class TreeDecoder(nn.Module):
    """A decoder of packed layers for tree decoding.  embed: token ids -> bf16
    [.., hidden]; blocks: a list of (TreeAttention, gate_up, down), gate_up an
    inference_v3.V3GateUpSiLU; head: hidden -> logits; RMS norms without weights."""

    def __init__(self, embed, blocks: list, head, rot_dim: int, max_positions: int, base: float = 10000.0, **scaling):
        super().__init__()
        self.embed, self.head = embed, head
        self.blocks = nn.ModuleList(nn.ModuleList(b) for b in blocks)
        self.register_buffer("table", rope_table(max_positions, rot_dim, base, **scaling), persistent=False)
        # the tree of one node, which hangs on the context
        self.register_buffer("root", torch.full((1,), -1, dtype=torch.int32, device=self.table.device), persistent=False)
        self.register_buffer("root_depth", torch.zeros(1, dtype=torch.int32, device=self.table.device), persistent=False)

    @staticmethod
    def norm(x: torch.Tensor) -> torch.Tensor:
        return nn.functional.rms_norm(x, x.shape[-1:])

    def use_adapters(self, adapter: torch.Tensor | None) -> None:
        """The adapter of each sequence of the batch (int32 [batch], negative for none) in all
        layers that have some; None takes them off."""
        for m in self.modules():
            if isinstance(m, V3LoRALinear):
                m.use(adapter)

    def forward(self, tokens: torch.Tensor, parents: torch.Tensor, depths: torch.Tensor, cache: PagedKVCache):
        """tokens [batch, nodes] -> (logits [batch, nodes, vocab], every layer's (k, v)).
        depths [nodes] or [batch, nodes]: tree_depths of parents."""
        b, t = tokens.shape
        positions = cache.lens[:, None] + depths
        x, new = self.embed(tokens), []
        for layer, (attention, gate_up, down) in enumerate(self.blocks):
            y, kv = attention(self.norm(x), positions, self.table, parents, cache, layer)
            x = x + y
            x = x + down(gate_up(self.norm(x).reshape(b * t, -1))).reshape(b, t, -1)
            new.append(kv)
        return self.head(self.norm(x).reshape(b * t, -1)).reshape(b, t, -1), new

    def prefill(self, tokens: torch.Tensor, cache: PagedKVCache) -> None:
        """Puts tokens [batch, n] into the cache, 64 at a time as a chain."""
        if tokens.shape[1] == 0:
            return
        for part in tokens.split(ops.MAX_TREE_NODES, dim=1):
            chain = torch.arange(-1, part.shape[1] - 1, dtype=torch.int32, device=part.device)
            _, new = self(part, chain, chain + 1, cache)
            cache.append(new)

    def step(self, tokens: torch.Tensor, parents: torch.Tensor, depths: torch.Tensor, cache: PagedKVCache,
             uniforms: torch.Tensor, noise: torch.Tensor, draft_probs: torch.Tensor | None = None, temperature=1.0,
             top_k=0, top_p=1.0, min_p=0.0):
        """One step: forward, verification, append of the accepted nodes.  Returns
        ops.tree_verify's (path, accepted, next); those of a row whose sequence has no
        pages mean nothing.  top_k, top_p and min_p (numbers, or tensors [batch], as in ops.sample)
        cut the distributions that the tokens are samples of."""
        logits, new = self(tokens, parents, depths, cache)
        if any(isinstance(s, torch.Tensor) or s != off for s, off in ((top_k, 0), (top_p, 1.0), (min_p, 0.0))):
            logits = ops.filter_logits(logits, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p, out=logits)
        path, accepted, last = ops.tree_verify(logits, tokens, parents, uniforms, noise, draft_probs=draft_probs,
                                               temperature=temperature)
        cache.append(new, index=path, counts=accepted)
        return path, accepted, last

    def decode(self, last: torch.Tensor, cache: PagedKVCache, noise: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0,
               min_p=0.0, return_logprob: bool = False):
        """One token a sequence: forward of the last ones [batch], whose K/V rows go into the
        cache, and the next ones, drawn by ops.sample with its settings.  A negative one (a
        row that had no distribution gives -1) stands for token 0, and what follows it means
        nothing, as in a row whose sequence has no pages."""
        logits, new = self(last.clamp(min=0)[:, None], self.root, self.root_depth, cache)
        cache.append(new)
        return ops.sample(logits[:, 0], noise, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p,
                          return_logprob=return_logprob)
