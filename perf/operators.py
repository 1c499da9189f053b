"""Measured cases of the tree-decoding operators: rotary positions, attention of
a tree of drafted tokens over a paged K/V cache, verification of the tree, and
the append of accepted tokens to the cache.

``run`` computes them in plain torch (32-bit) where ``own`` is false and through
the framework's entry points where it is true.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
ITEM = {"bf16": 2, "f16": 2, "f32": 4}


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # rotary positions of one decode step's 16 tree nodes, half layout, a quarter of the 256-wide head
        {"name": "rope tree nodes", "op": "rope", "b": 1, "t": 16, "hq": 16, "hkv": 16, "d": 256, "rot": 64,
         "interleaved": False, "train": False, "dtype": "bf16", "positions": 32768},
        # prefill of 2048 tokens, interleaved layout, the whole 128-wide head
        {"name": "rope prefill", "op": "rope", "b": 1, "t": 2048, "hq": 32, "hkv": 32, "d": 128, "rot": 128,
         "interleaved": True, "train": False, "dtype": "f16", "positions": 8192},
        # a training micro-batch of 8 x 4096 tokens, shared key heads, forward and backward
        {"name": "rope train", "op": "rope", "b": 8, "t": 4096, "hq": 32, "hkv": 8, "d": 128, "rot": 128,
         "interleaved": False, "train": True, "dtype": "bf16", "positions": 4096},
        # plain decode: one token of one sequence, 16 heads of 256
        {"name": "attention one token", "op": "attention", "b": 1, "t": 1, "hq": 16, "hkv": 16, "d": 256,
         "ctx": 1000, "page": 64, "dtype": "bf16"},
        # eight sequences with 16-node trees over ragged contexts of a few thousand tokens
        {"name": "attention 16 nodes", "op": "attention", "b": 8, "t": 16, "hq": 32, "hkv": 8, "d": 128,
         "ctx": 4097, "page": 32, "dtype": "bf16"},
        # one key head per query head, an odd tree, small pages that end inside a tile
        {"name": "attention odd tree", "op": "attention", "b": 3, "t": 13, "hq": 32, "hkv": 32, "d": 128,
         "ctx": 7777, "page": 48, "dtype": "f16"},
        # large trees of two long sequences, eight query heads per key head
        {"name": "attention long context", "op": "attention", "b": 2, "t": 64, "hq": 32, "hkv": 4, "d": 128,
         "ctx": 65536, "page": 64, "dtype": "bf16"},
        # a serving batch: 16 sequences of up to 32k tokens, 32-node trees
        {"name": "attention batch", "op": "attention", "b": 16, "t": 32, "hq": 32, "hkv": 8, "d": 128,
         "ctx": 32768, "page": 64, "dtype": "bf16"},
        # one sequence, a chain of drafted tokens sampled from the draft's distribution
        {"name": "verify chain", "op": "verify", "b": 1, "t": 8, "branch": 1, "vocab": 32000, "dtype": "f32",
         "sampled": True, "temperature": "one"},
        # a serving batch with the draft's most likely tokens as a tree, an odd vocabulary, mixed temperatures
        {"name": "verify batch", "op": "verify", "b": 64, "t": 16, "branch": 3, "vocab": 100003, "dtype": "bf16",
         "sampled": False, "temperature": "mixed"},
        # the accepted path of every sequence's tree goes into the cache
        {"name": "append accepted", "op": "append", "b": 32, "t": 16, "hkv": 8, "d": 128, "ctx": 2048, "page": 32,
         "path": True, "dtype": "bf16"},
        # prompts of 2048 tokens, one key head per query head
        {"name": "append prompt", "op": "append", "b": 4, "t": 2048, "hkv": 32, "d": 128, "ctx": 500, "page": 64,
         "path": False, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _fit(case):
    """Fewer sequences, then fewer tokens, until a pass costs no more than the largest listed one of its kind."""
    most = [work(c) for c in listed() if c["op"] == case["op"]]
    while any(work(case)[x] > max(m[x] for m in most) for x in ("bytes", "flops")):
        if case["b"] > 1:
            case["b"] -= max(1, case["b"] // 8)
        elif case["t"] > 1 and case["op"] != "attention":
            case["t"] -= max(1, case["t"] // 8)
        else:
            case["ctx"] -= max(1, case["ctx"] // 8)
    # round lengths are the listed cases': the drawn ones stay off them
    return {x: n - 1 if x in ("t", "ctx", "vocab", "positions") and n > 0 and n % 1024 == 0 else n for x, n in case.items()}


def draw(rng):
    op = rng.choice(["rope", "attention", "attention", "attention", "verify", "append"])
    if op == "rope":
        d = rng.choice([64, 80, 112, 128, 256])
        hkv = rng.choice([1, 2, 4, 8, 32])
        hq = hkv * rng.choice([1, 2, 4, 8]) if hkv < 32 else 32
        return _fit({"op": op, "b": _log(rng, 1, 64), "t": _log(rng, 1, 4096), "hq": hq, "hkv": hkv, "d": d,
                     "rot": rng.choice([d, d // 2, d // 4 // 2 * 2]), "interleaved": rng.random() < 0.5,
                     "train": rng.random() < 0.4, "dtype": rng.choice(["bf16", "f16", "f32"]),
                     "positions": _log(rng, 4096, 131072)})
    if op == "attention":
        hkv = rng.choice([1, 2, 4, 8, 16, 32])
        return _fit({"op": op, "b": _log(rng, 1, 32), "t": _log(rng, 1, 64), "hq": hkv * rng.choice([1, 2, 4, 5, 8][:6 - hkv // 8]),
                     "hkv": hkv, "d": rng.choice([64, 80, 112, 128, 128, 256]), "ctx": _log(rng, 1, 65536) - 1,
                     "page": rng.choice([8, 16, 24, 32, 48, 64, 128, 256]), "dtype": rng.choice(["bf16", "f16"])})
    if op == "verify":
        case = {"op": op, "b": _log(rng, 1, 128), "t": _log(rng, 1, 64), "branch": rng.choice([1, 2, 3, 4]),
                "vocab": _log(rng, 1000, 160000), "dtype": rng.choice(["f32", "bf16", "f16"]),
                "sampled": rng.random() < 0.5, "temperature": rng.choice(["one", "warm", "zero", "mixed"])}
        case["b"] = max(1, min(case["b"], 64 * 16 * 100003 // (case["vocab"] * case["t"])))
        return _fit(case)
    path = rng.random() < 0.5
    return _fit({"op": op, "b": _log(rng, 1, 64), "t": _log(rng, 1, 64 if path else 4096), "hkv": rng.choice([1, 2, 4, 8, 32]),
                 "d": rng.choice([64, 80, 128, 256]), "ctx": _log(rng, 1, 4096) - 1,
                 "page": rng.choice([8, 16, 24, 32, 64, 128]), "path": path, "dtype": rng.choice(["bf16", "f16", "f32"])})


def lengths(case):
    """The context length of each sequence: the first is the longest, the others are ragged."""
    b, ctx = case["b"], case["ctx"]
    return [ctx - (ctx * ((5 * i) % b)) // (2 * b) for i in range(b)]


def counts(case):
    """How many of its new tokens each sequence appends."""
    return [1 + (3 * i) % min(case["t"], 6) if case["path"] else case["t"] for i in range(case["b"])]


# ------------------------------------------------------------------ the inputs
def _tree(b, t, gen):
    """Random trees: node 0 hangs on the context, node i on an earlier one; the
    last nodes of some sequences are unused."""
    pick = torch.rand(b, t, generator=gen)
    at = torch.arange(t)
    back = 1 + (pick * pick * at.clamp(max=12)).long()
    parents = (at - back).clamp(min=0)
    parents[:, 0] = -1
    used = t - (torch.rand(b, generator=gen) * 0.3 * t).long()
    used[0] = t
    return torch.where(at < used[:, None], parents, -2).to(torch.int32)


def _pages(case, extra, gen):
    page = case["page"]
    need = [-(-(n + extra) // page) for n in lengths(case)]
    total, width = sum(need) + 3, max(max(need), 1)
    order = torch.randperm(total, generator=gen)
    table, at = torch.zeros(len(need), width, dtype=torch.int32), 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n].to(torch.int32)
        at += n
    return total, table


def prepare(case, seed):
    dev = torch.device("cuda")
    gen, host = torch.Generator(dev).manual_seed(seed), torch.Generator().manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    op, b, t = case["op"], case["b"], case["t"]

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=dev, dtype=dt if dt != torch.float16 else torch.float32).to(dt)

    s = {"op": op, "case": case}
    if op == "rope":
        hq, hkv, d, rot = case["hq"], case["hkv"], case["d"], case["rot"]
        # q and k are parts of a merged q|k|v projection's rows
        qkv = randn(b, t, (hq + 2 * hkv) * d)
        s["q"] = qkv[..., :hq * d].unflatten(-1, (hq, d))
        s["k"] = qkv[..., hq * d:(hq + hkv) * d].unflatten(-1, (hkv, d))
        start = torch.randint(0, max(1, case["positions"] - t), (b, 1), generator=gen, device=dev)
        s["positions"] = start + torch.arange(t, device=dev)
        freq = 500000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=dev) / rot)
        angle = torch.arange(max(case["positions"], t), dtype=torch.float64, device=dev)[:, None] * (freq / 4.0)
        s["table"] = torch.cat([angle.cos(), angle.sin()], 1).float()
        if case["train"]:
            s["q"], s["k"] = s["q"].detach().requires_grad_(), s["k"].detach().requires_grad_()
            s["dq"], s["dk"] = randn(b, t, hq, d), randn(b, t, hkv, d)
    elif op == "attention":
        hq, hkv, d = case["hq"], case["hkv"], case["d"]
        total, table = _pages(case, 0, host)
        s["k_cache"], s["v_cache"] = randn(total, case["page"], hkv, d), randn(total, case["page"], hkv, d)
        s["page_table"] = table.to(dev)
        s["lens"] = torch.tensor(lengths(case), dtype=torch.int32, device=dev)
        s["parents"] = _tree(b, t, host).to(dev)
        # queries with some spread, so that a few tokens carry much of the weight
        s["q"] = randn(b, t, hq, d) * 2
        s["k_tree"], s["v_tree"] = randn(b, t, hkv, d), randn(b, t, hkv, d)
        s["scale"] = d ** -0.5
    elif op == "verify":
        v, branch = case["vocab"], case["branch"]
        logits = torch.randn(b, t, v, generator=gen, device=dev) * 4
        draft = torch.softmax(logits + 0.7 * torch.randn(b, t, v, generator=gen, device=dev), -1)
        at = torch.arange(t)
        parents = torch.where(at > 0, (at - 1).clamp(min=0) // branch, -1)
        s["parents"] = parents.to(torch.int32).expand(b, t).contiguous().to(dev)
        up = parents.clamp(min=0).to(dev)
        if case["sampled"]:
            inner = int(up.max()) + 1
            drawn = torch.multinomial(draft[:, :inner].reshape(-1, v), branch, replacement=True, generator=gen)
            s["draft_probs"] = draft
        else:
            inner = int(up.max()) + 1
            drawn = draft[:, :inner].topk(branch, -1).indices.reshape(-1, branch)
            s["draft_probs"] = None
        drawn = drawn.reshape(b, inner, branch)
        rank = (at - 1).clamp(min=0).to(dev) % branch
        s["tokens"] = drawn[:, up, rank].contiguous()
        s["logits"] = logits.to(dt)
        s["uniforms"] = torch.rand(b, t, generator=gen, device=dev)
        s["noise"] = torch.empty(b, v, device=dev).exponential_(generator=gen).clamp_(min=1e-30)
        kind = case["temperature"]
        values = {"one": [1.0], "warm": [0.7], "zero": [0.0], "mixed": [1.0, 0.0, 0.6, 1.3]}[kind]
        s["temperature"] = torch.tensor([values[i % len(values)] for i in range(b)], device=dev)
    else:
        hkv, d, n = case["hkv"], case["d"], counts(case)
        total, table = _pages(case, max(n), host)
        s["k_cache"], s["v_cache"] = randn(total, case["page"], hkv, d), randn(total, case["page"], hkv, d)
        s["page_table"] = table.to(dev)
        s["lens"] = torch.tensor(lengths(case), dtype=torch.int32, device=dev)
        s["k_new"], s["v_new"] = randn(b, t, hkv, d), randn(b, t, hkv, d)
        s["path"] = s["counts"] = None
        if case["path"]:
            # an accepted path: increasing node numbers, -1 after its end
            order = torch.rand(b, t, generator=host).argsort(-1)
            path = torch.full((b, t), -1, dtype=torch.int32)
            for i, k in enumerate(n):
                path[i, :k] = order[i, :k].sort().values.to(torch.int32)
            s["path"] = path.to(dev)
            s["counts"] = torch.tensor(n, dtype=torch.int32, device=dev)
    return s


# ------------------------------------------------------------------ plain forms
def _rotate(x, cos, sin, interleaved):
    """Both values of each pair of the first part of the head, the rest unchanged."""
    rot, y = 2 * cos.shape[-1], x.float()
    if interleaved:
        a, b = y[..., 0:rot:2], y[..., 1:rot:2]
        part = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = y[..., :rot // 2], y[..., rot // 2:rot]
        part = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([part, y[..., rot:]], -1).to(x.dtype)


def _plain_rope(s):
    inter = s["case"]["interleaved"]
    row = s["table"][s["positions"]][:, :, None]
    cos, sin = row.chunk(2, -1)
    out = {"q": _rotate(s["q"], cos, sin, inter), "k": _rotate(s["k"], cos, sin, inter)}
    if "dq" in s:
        out["dq"], out["dk"] = _rotate(s["dq"], cos, -sin, inter), _rotate(s["dk"], cos, -sin, inter)
    return out


def _ancestors(parents):
    """[B, T, T]: whether node j is node i or one of its ancestors; used nodes [B, T]."""
    t = parents.shape[1]
    own_node = torch.eye(t, device=parents.device)
    step = own_node + (parents[:, :, None] == torch.arange(t, device=parents.device)).float()
    for _ in range(max(1, (t - 1).bit_length())):
        step = (step @ step).clamp(max=1)
    used = ~((step > 0) & (parents < -1)[:, None]).any(-1)
    return (step > 0) & used[:, :, None], used


def _plain_attention(s):
    q, lens, table = s["q"], s["lens"], s["page_table"]
    b, t, hq, d = q.shape
    hkv = s["k_tree"].shape[2]
    page = s["k_cache"].shape[1]
    at = torch.arange(table.shape[1] * page, device=q.device)
    where = table[:, at // page].long()
    inside = at[None] < lens[:, None]
    sees, used = _ancestors(s["parents"])
    mask = torch.cat([inside[:, None] & used[:, :, None], sees], 2)

    def rows(cache, tree):
        ctx = cache[where, at % page].float()
        return torch.cat([torch.where(inside[:, :, None, None], ctx, 0.0), tree.float()], 1).transpose(1, 2)

    k, v = rows(s["k_cache"], s["k_tree"]), rows(s["v_cache"], s["v_tree"])
    # [B, Hkv, group * T, D]: the query heads of one key head together
    x = q.float().reshape(b, t, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, -1, d)
    p = (x @ k.transpose(2, 3)).mul_(s["scale"]).view(b, hkv, hq // hkv, t, -1)
    p.masked_fill_(~mask[:, None, None], -math.inf)
    top = p.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p.view(b, hkv, -1, p.shape[-1]) @ v).view(b, hkv, hq // hkv, t, d) / torch.where(total == 0, 1.0, total)
    lse = (total.log() + top).squeeze(-1)
    return {"out": out.permute(0, 3, 1, 2, 4).reshape(b, t, hq, d).to(q.dtype),
            "lse": lse.permute(0, 3, 1, 2).reshape(b, t, hq)}


def _plain_verify(s):
    logits, tokens, parents, draft = s["logits"], s["tokens"], s["parents"], s["draft_probs"]
    b, t, v = logits.shape
    dev, seq = logits.device, torch.arange(b, device=logits.device)
    temp = s["temperature"][:, None]
    greedy = temp[:, 0] == 0
    lowest = torch.arange(v, 0, -1, device=dev)

    def first_max(x):
        return ((x == x.amax(-1, keepdim=True)) * lowest).argmax(-1)

    def target(node):
        x = logits[seq, node].float()
        best = torch.nn.functional.one_hot(first_max(x), v).float()
        x = x / torch.where(temp == 0, 1.0, temp)
        e = (x - x.amax(-1, keepdim=True)).exp()
        return torch.where(greedy[:, None], best, e / e.sum(-1, keepdim=True))

    cur = torch.zeros(b, dtype=torch.long, device=dev)
    r, n = target(cur), torch.ones(b, dtype=torch.long, device=dev)
    path = torch.full((b, t), -1, dtype=torch.int32, device=dev)
    path[:, 0] = 0
    for i in range(1, t):
        child, x = parents[:, i] == cur, tokens[:, i]
        one_hot = torch.nn.functional.one_hot(x, v).float()
        q = one_hot if draft is None else torch.where(greedy[:, None], one_hot, draft[seq, cur].float())
        yes = child & (s["uniforms"][:, i] * q[seq, x] < r[seq, x])
        # rejected: what is left of the target's distribution
        left = (r - q).clamp(min=0)
        if draft is None:
            left = r * (1 - one_hot)
        mass = left.sum(-1, keepdim=True)
        left = torch.where(mass > 0, left / mass, r)
        left = torch.where(greedy[:, None], r, left)
        r = torch.where((child & ~yes)[:, None], left, r)
        path[seq, torch.where(yes, n, t - 1)] = torch.where(yes, i, path[seq, torch.where(yes, n, t - 1)]).to(torch.int32)
        n = n + yes
        cur = torch.where(yes, i, cur)
        r = torch.where(yes[:, None], target(cur), r)
    return {"path": path, "accepted": n.to(torch.int32), "next": first_max(torch.where(r > 0, r / s["noise"], -1.0))}


def _plain_append(s):
    k, v, page = s["k_new"], s["v_new"], s["k_cache"].shape[1]
    b, t = k.shape[:2]
    dev, seq = k.device, torch.arange(b, device=k.device)
    n = s["counts"] if s["counts"] is not None else torch.full((b,), t, dtype=torch.int32, device=dev)
    at = torch.arange(t, device=dev)[None]
    take = s["path"].long().clamp(min=0) if s["path"] is not None else at.expand(b, t)
    who, which = (at < n[:, None]).nonzero(as_tuple=True)
    spot = s["lens"][who].long() + which
    pages = s["page_table"][who, spot // page].long()
    s["k_cache"][pages, spot % page] = k[who, take[who, which]]
    s["v_cache"][pages, spot % page] = v[who, take[who, which]]
    return {"k_cache": s["k_cache"], "v_cache": s["v_cache"], "lens": s["lens"] + n}


def run(s):
    op = s["op"]
    if not own:
        return {"rope": _plain_rope, "attention": _plain_attention, "verify": _plain_verify, "append": _plain_append}[op](s)
    from spark_b200 import ops, rotary
    if op == "rope":
        inter = s["case"]["interleaved"]
        if "dq" not in s:
            q, k = ops.rope(s["q"], s["k"], s["positions"], s["table"], interleaved=inter)
            return {"q": q, "k": k}
        q, k = rotary.apply_rope(s["q"], s["k"], s["positions"], s["table"], interleaved=inter)
        dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
        return {"q": q, "k": k, "dq": dq, "dk": dk}
    if op == "attention":
        out, lse = ops.tree_attention(s["q"], s["k_tree"], s["v_tree"], s["k_cache"], s["v_cache"], s["page_table"],
                                      s["lens"], s["parents"], scale=s["scale"], return_lse=True)
        return {"out": out, "lse": lse}
    if op == "verify":
        path, n, token = ops.tree_verify(s["logits"], s["tokens"], s["parents"], s["uniforms"], s["noise"],
                                         draft_probs=s["draft_probs"], temperature=s["temperature"])
        return {"path": path, "accepted": n, "next": token}
    lens = ops.kv_append(s["k_new"], s["v_new"], s["k_cache"], s["v_cache"], s["page_table"], s["lens"],
                         index=s["path"], counts=s["counts"])
    return {"k_cache": s["k_cache"], "v_cache": s["v_cache"], "lens": lens}


# ------------------------------------------------------------------ what a pass needs
def work(case):
    b, t, e = case["b"], case["t"], ITEM[case["dtype"]]
    if case["op"] == "rope":
        values = b * t * (case["hq"] + case["hkv"]) * case["d"]
        table = min(b * t, case["positions"]) * case["rot"] * 4
        times = 2 if case["train"] else 1
        return {"bytes": times * (2 * values * e + table + 8 * b * t), "flops": times * 3 * values * case["rot"] // case["d"]}
    if case["op"] == "attention":
        ctx, kv, q = sum(lengths(case)), case["hkv"] * case["d"], case["hq"] * case["d"]
        return {"bytes": 2 * e * (ctx + b * t) * kv + 2 * e * b * t * q + 4 * b * t * (case["hq"] + 1),
                "flops": 4 * t * q * (ctx + b * (t + 1) // 2)}
    if case["op"] == "verify":
        # the root's distribution and the noise of the last draw; deeper nodes are read as the path goes
        return {"bytes": b * case["vocab"] * (e + 4), "flops": 4 * b * case["vocab"]}
    n = sum(counts(case))
    return {"bytes": 4 * n * case["hkv"] * case["d"] * e + 12 * b, "flops": 0}


# ------------------------------------------------------------------ 64 bits
def _exact_rope(s):
    case, out = s["case"], {}
    half = case["rot"] // 2
    z = s["table"].double()[s["positions"]][:, :, None]
    turn = torch.complex(z[..., :half].contiguous(), z[..., half:].contiguous())
    for name in ("q", "k", "dq", "dk"):
        if name not in s:
            continue
        x = s[name].detach().double()
        part = x[..., :case["rot"]].unflatten(-1, (half, 2) if case["interleaved"] else (2, half))
        a, b = part.unbind(-1 if case["interleaved"] else -2)
        y = torch.complex(a.contiguous(), b.contiguous()) * (turn.conj() if name[0] == "d" else turn)
        y = torch.stack([y.real, y.imag], -1 if case["interleaved"] else -2).flatten(-2)
        out[name] = torch.cat([y, x[..., case["rot"]:]], -1)
    return out


def _exact_attention(s):
    """One sequence and key head at a time, the mask by walking up from each node."""
    q = s["q"].double()
    b, t, hq, d = q.shape
    hkv, page = s["k_tree"].shape[2], s["k_cache"].shape[1]
    group = hq // hkv
    out, lse = torch.zeros_like(q), torch.full((b, t, hq), -math.inf, dtype=torch.float64, device=q.device)
    for i, n in enumerate(s["lens"].tolist()):
        parents = s["parents"][i].tolist()
        chains = []
        for node in range(t):
            chain = []
            while node >= 0:
                chain.append(node)
                node = parents[node]
            chains.append(chain if node == -1 else None)
        used = [j for j in range(t) if chains[j] is not None]
        if not used:
            continue
        mask = torch.zeros(len(used), n + t, dtype=torch.bool)
        mask[:, :n] = True
        for j, node in enumerate(used):
            mask[j, [n + a for a in chains[node]]] = True
        mask, pick = mask.to(q.device), torch.tensor(used, device=q.device)
        pages = s["page_table"][i, :-(-n // page)].long()
        k = torch.cat([s["k_cache"][pages].flatten(0, 1)[:n], s["k_tree"][i]]).double()
        v = torch.cat([s["v_cache"][pages].flatten(0, 1)[:n], s["v_tree"][i]]).double()
        for h in range(hkv):
            heads = slice(h * group, (h + 1) * group)
            x = q[i, pick][:, heads].transpose(0, 1)
            score = (x @ k[:, h].T * s["scale"]).masked_fill(~mask, -math.inf)
            z = torch.logsumexp(score, -1, keepdim=True)
            out[i, pick, heads] = ((score - z).exp() @ v[:, h]).transpose(0, 1)
            lse[i, pick, heads] = z.squeeze(-1).T
    return {"out": out, "lse": lse}


def _exact_verify(s):
    """One sequence at a time, from node to node."""
    b, t, v = s["logits"].shape
    parents, tokens, u = s["parents"].tolist(), s["tokens"].tolist(), s["uniforms"].double().tolist()
    temp = s["temperature"].double().tolist()
    path, n, last = torch.full((b, t), -1, dtype=torch.int32), torch.ones(b, dtype=torch.int32), torch.zeros(b, dtype=torch.int64)
    for i in range(b):
        cur, walked, token = 0, [0], None
        while token is None:
            row = s["logits"][i, cur].double().cpu()
            best = int((row == row.max()).nonzero()[0])
            r = torch.softmax(row / temp[i], 0) if temp[i] else None
            q = s["draft_probs"][i, cur].double().cpu() if s["draft_probs"] is not None else None
            step = None
            for c in [j for j in range(1, t) if parents[i][j] == cur]:
                x = tokens[i][c]
                if r is None:
                    yes = x == best
                else:
                    yes = u[i][c] * (1.0 if q is None else float(q[x])) < float(r[x])
                if yes:
                    step = c
                    break
                if r is not None:
                    left = r.clone()
                    if q is None:
                        left[x] = 0
                    else:
                        left = (r - q).clamp(min=0)
                    r = left / left.sum() if float(left.sum()) > 0 else r
            if step is not None:
                cur = step
                walked.append(step)
            elif r is None:
                token = best
            else:
                token = int((r / s["noise"][i].double().cpu()).argmax())
        path[i, :len(walked)] = torch.tensor(walked, dtype=torch.int32)
        n[i], last[i] = len(walked), token
    return {"path": path, "accepted": n, "next": last}


def _exact_append(s):
    """One token at a time of the cache's own values: they are moved, not computed."""
    page, table, lens = s["k_cache"].shape[1], s["page_table"].cpu(), s["lens"].cpu()
    k, v = s["k_cache"].cpu().double(), s["v_cache"].cpu().double()
    new_k, new_v = s["k_new"].cpu().double(), s["v_new"].cpu().double()
    n = counts(s["case"])
    for i, many in enumerate(n):
        for j in range(many):
            at = int(lens[i]) + j
            spot = (int(table[i, at // page]), at % page)
            node = int(s["path"][i, j]) if s["path"] is not None else j
            k[spot], v[spot] = new_k[i, node], new_v[i, node]
    return {"k_cache": k, "v_cache": v, "lens": lens + torch.tensor(n, dtype=torch.int32)}


def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _exact_rope, "attention": _exact_attention, "verify": _exact_verify, "append": _exact_append}[case["op"]](s)
