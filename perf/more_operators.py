"""Measured cases of what a decoding step does around its projections, its cache
and its attention: norms of q and k with the rotary positions in one pass
(forward and backward), sampling with temperature, top-k, top-p and min-p from
given random numbers, the same filter as logits (in front of a tree's
verification), and low-rank adapters of many requests beside a shared projection.

``run`` computes them in plain torch where ``own`` is false and through the
framework's entry points where it is true.
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
        # one decode step's 16 tree nodes: 32 query and 8 key heads of 128, views of a merged projection
        {"name": "norm rope tree nodes", "op": "norm", "b": 1, "t": 16, "hq": 32, "hkv": 8, "d": 128, "rot": 128,
         "interleaved": False, "train": False, "dtype": "bf16", "wtype": "bf16", "positions": 32768},
        # prefill of 2048 tokens, interleaved layout
        {"name": "norm rope prefill", "op": "norm", "b": 1, "t": 2048, "hq": 32, "hkv": 8, "d": 128, "rot": 128,
         "interleaved": True, "train": False, "dtype": "f16", "wtype": "f32", "positions": 8192},
        # a training micro-batch of 8 x 4096 tokens, forward and backward with the norms' weights
        {"name": "norm rope train", "op": "norm", "b": 8, "t": 4096, "hq": 32, "hkv": 8, "d": 128, "rot": 128,
         "interleaved": False, "train": True, "dtype": "bf16", "wtype": "bf16", "positions": 4096},
        # odd sizes, half of an 80-wide head turned, all of it in 32 bits
        {"name": "norm rope train odd", "op": "norm", "b": 3, "t": 777, "hq": 6, "hkv": 2, "d": 80, "rot": 40,
         "interleaved": False, "train": True, "dtype": "f32", "wtype": "f32", "positions": 1000},
        # the next token of one sequence with the usual chat settings
        {"name": "sample one", "op": "sample", "b": 1, "t": 1, "vocab": 32000, "dtype": "f32", "kind": "k and p"},
        # a serving batch whose requests differ in their settings, an odd vocabulary
        {"name": "sample batch", "op": "sample", "b": 64, "t": 1, "vocab": 100003, "dtype": "bf16", "kind": "mixed"},
        # the logits of a chain of 8 drafted tokens, cut to the nucleus before their verification
        {"name": "filter chain", "op": "filter", "b": 1, "t": 8, "vocab": 32000, "dtype": "f32", "kind": "p"},
        # trees of 16 nodes of 16 sequences with different settings
        {"name": "filter trees", "op": "filter", "b": 16, "t": 16, "vocab": 32000, "dtype": "bf16", "kind": "mixed"},
        # one token of one request beside the q projection
        {"name": "adapters one token", "op": "adapters", "requests": 1, "t": 1, "ic": 2560, "oc": 4096, "r": 16, "pool": 8,
         "dtype": "bf16"},
        # a decoding batch, a token of each of 48 requests, beside the gate and up projections' width
        {"name": "adapters decode", "op": "adapters", "requests": 48, "t": 48, "ic": 2560, "oc": 9728, "r": 16, "pool": 32,
         "dtype": "bf16"},
        # 77 tokens of ragged requests, sizes that fit no tile and no 16 bytes
        {"name": "adapters odd", "op": "adapters", "requests": 9, "t": 77, "ic": 1001, "oc": 1030, "r": 12, "pool": 5,
         "dtype": "f16"},
        # the prompts of five requests, 4096 tokens in all
        {"name": "adapters prompts", "op": "adapters", "requests": 5, "t": 4096, "ic": 2560, "oc": 9728, "r": 32, "pool": 8,
         "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _fit(case):
    """Fewer sequences, then fewer tokens, then smaller sizes, until a pass costs no more than the largest listed one of its kind."""
    most = [work(c) for c in listed() if c["op"] == case["op"]]
    while any(work(case)[x] > max(m[x] for m in most) for x in ("bytes", "flops")):
        if case.get("b", 1) > 1:
            case["b"] -= max(1, case["b"] // 8)
        elif case["t"] > 1:
            case["t"] -= max(1, case["t"] // 8)
            case["requests"] = min(case.get("requests", 1), case["t"])
        else:
            for x in ("pool", "r"):
                case[x] = max(1, case[x] * 7 // 8)
    if case["op"] != "adapters":
        case.pop("requests", None)
    # round lengths are the listed cases': the drawn ones stay off them
    return {x: n - 1 if x in ("t", "vocab", "positions", "ic", "oc") and n > 0 and n % 1024 == 0 else n for x, n in case.items()}


def draw(rng):
    op = rng.choice(["norm", "norm", "sample", "filter", "adapters", "adapters"])
    if op == "norm":
        d = rng.choice([64, 80, 96, 112, 128, 128, 256])
        hkv = rng.choice([1, 2, 4, 8, 32])
        hq = hkv * rng.choice([1, 2, 4, 5, 8]) if hkv < 32 else 32
        dtype = rng.choice(["bf16", "f16", "f32"])
        return _fit({"op": op, "b": _log(rng, 1, 64), "t": _log(rng, 1, 4096), "hq": hq, "hkv": hkv, "d": d,
                     "rot": rng.choice([d, d // 2, d // 4 // 2 * 2]), "interleaved": rng.random() < 0.5,
                     "train": rng.random() < 0.5, "dtype": dtype, "wtype": rng.choice([dtype, "f32"]),
                     "positions": _log(rng, 4096, 131072)})
    if op in ("sample", "filter"):
        case = {"op": op, "b": _log(rng, 1, 128), "t": 1 if op == "sample" else _log(rng, 1, 32), "vocab": _log(rng, 1000, 160000),
                "dtype": rng.choice(["f32", "bf16", "f16"]), "kind": rng.choice(list(KINDS))}
        return _fit(case)
    t = _log(rng, 1, 6000)
    return _fit({"op": op, "requests": max(1, min(t, _log(rng, 1, 128))), "t": t, "ic": _log(rng, 256, 12000),
                 "oc": _log(rng, 256, 16000), "r": rng.choice([4, 8, 12, 16, 24, 32, 64, 100, 128]), "pool": _log(rng, 1, 64),
                 "dtype": rng.choice(["bf16", "f16"])})


# temperature, top_k, top_p, min_p of the requests in turn
KINDS = {
    "k and p": [(0.7, 50, 0.9, 0.0)],
    "p": [(1.0, 0, 0.95, 0.0)],
    "k": [(1.0, 40, 1.0, 0.0)],
    "min": [(1.3, 0, 1.0, 0.05)],
    "plain": [(0.9, 0, 1.0, 0.0)],
    "mixed": [(0.7, 50, 0.9, 0.0), (1.0, 0, 0.95, 0.0), (0.0, 0, 1.0, 0.0), (1.3, 0, 1.0, 0.05), (0.9, 0, 1.0, 0.0),
              (1.0, 1000, 0.8, 0.02), (0.6, 20, 1.0, 0.0), (1.0, 0, 0.5, 0.0)],
}


def settings(case):
    """(temperature, top_k, top_p, min_p) of each sequence."""
    kind = KINDS[case["kind"]]
    return [kind[i % len(kind)] for i in range(case["b"])]


# ------------------------------------------------------------------ the inputs
def segments(case):
    """The tokens of each request: one in a decoding batch, else ragged runs, each at least one."""
    n, t = case["requests"], case["t"]
    weight = [1 + (7 * i) % 5 for i in range(n)]
    out = [1 + (t - n) * w // sum(weight) for w in weight]
    out[0] += t - sum(out)
    return out


def prepare(case, seed):
    dev = torch.device("cuda")
    gen, host = torch.Generator(dev).manual_seed(seed), torch.Generator().manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    op, t = case["op"], case["t"]

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=dev, dtype=dt if dt != torch.float16 else torch.float32).to(dt)

    s = {"op": op, "case": case}
    if op == "norm":
        b, hq, hkv, d, rot = case["b"], case["hq"], case["hkv"], case["d"], case["rot"]
        # q and k are parts of a merged q|k|v projection's rows
        qkv = randn(b, t, (hq + 2 * hkv) * d)
        s["q"] = qkv[..., :hq * d].unflatten(-1, (hq, d))
        s["k"] = qkv[..., hq * d:(hq + hkv) * d].unflatten(-1, (hkv, d))
        wt = DTYPES[case["wtype"]]
        s["qw"], s["kw"] = ((1 + 0.3 * torch.randn(d, generator=gen, device=dev)).to(wt) for _ in range(2))
        start = torch.randint(0, max(1, case["positions"] - t), (b, 1), generator=gen, device=dev)
        s["positions"] = start + torch.arange(t, device=dev)
        freq = 1000000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=dev) / rot)
        angle = torch.arange(max(case["positions"], t), dtype=torch.float64, device=dev)[:, None] * freq
        s["table"] = torch.cat([angle.cos(), angle.sin()], 1).float()
        s["eps"] = 1e-6
        if case["train"]:
            for x in ("q", "k", "qw", "kw"):
                s[x] = s[x].detach().requires_grad_()
            s["dq"], s["dk"] = randn(b, t, hq, d), randn(b, t, hkv, d)
    elif op in ("sample", "filter"):
        b, v = case["b"], case["vocab"]
        shape = (b, v) if op == "sample" else (b, t, v)
        s["logits"] = (torch.randn(*shape, generator=gen, device=dev) * 4).to(dt)
        temp, k, p, least = zip(*settings(case))
        s["settings"] = {"temperature": torch.tensor(temp, device=dev), "top_k": torch.tensor(k, dtype=torch.int32, device=dev),
                         "top_p": torch.tensor(p, device=dev), "min_p": torch.tensor(least, device=dev)}
        if op == "sample":
            s["noise"] = torch.empty(b, v, device=dev).exponential_(generator=gen).clamp_(min=1e-30)
    else:
        ic, oc, r, pool = case["ic"], case["oc"], case["r"], case["pool"]
        s["x"], s["y"] = randn(t, ic), randn(t, oc)
        s["a"] = (torch.randn(pool, r, ic, generator=gen, device=dev) * ic ** -0.5).to(dt)
        s["b"] = (torch.randn(pool, oc, r, generator=gen, device=dev) * 0.2).to(dt)
        s["scale"] = 16.0 / r * (1 + torch.rand(pool, generator=gen, device=dev))
        # an adapter of the pool for each request; one in eight has none
        which = torch.randint(0, pool, (case["requests"],), generator=host)
        which = torch.where((torch.arange(case["requests"]) % 8 == 7), -1, which)
        s["adapter"] = which.repeat_interleave(torch.tensor(segments(case))).to(torch.int32).to(dev)
    return s


# ------------------------------------------------------------------ plain forms
def _turned(y, cos, sin, interleaved):
    """Both values of each pair of the first part of the head turned, the rest unchanged."""
    rot = 2 * cos.shape[-1]
    if interleaved:
        a, b = y[..., 0:rot:2], y[..., 1:rot:2]
        part = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = y[..., :rot // 2], y[..., rot // 2:rot]
        part = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([part, y[..., rot:]], -1)


def _plain_norm(s):
    inter = s["case"]["interleaved"]
    cos, sin = s["table"][s["positions"]][:, :, None].chunk(2, -1)
    out = {}
    with torch.no_grad():
        for name in ("q", "k"):
            x, w = s[name].float(), s[name + "w"].float()
            rstd = ((x * x).mean(-1, keepdim=True) + s["eps"]).rsqrt()
            unit = x * rstd
            out[name] = _turned(unit * w, cos, sin, inter).to(s[name].dtype)
            if "d" + name in s:
                g = _turned(s["d" + name].float(), cos, -sin, inter)
                out["d" + name + "w"] = (g * unit).flatten(0, 2).sum(0, dtype=torch.float64).to(s[name + "w"].dtype)
                g = g * w
                out["d" + name] = (rstd * (g - unit * (g * unit).mean(-1, keepdim=True))).to(s[name].dtype)
    return out


def _kept(s):
    """[rows, vocab]: what top-k, top-p and min-p leave; e = exp((logit - largest) / temperature), both in 64 bits."""
    x = s["logits"]
    rows = x.shape[1] if x.dim() == 3 else 1
    x = x.flatten(0, -2).double()
    per_row = {n: v.repeat_interleave(rows)[:, None] for n, v in s["settings"].items()}
    temp, top_p, v = per_row["temperature"].double(), per_row["top_p"].double(), x.shape[-1]
    greedy = temp == 0
    value, order = torch.sort(x, dim=-1, descending=True, stable=True)
    e = ((value - value[:, :1]) / torch.where(greedy, 1.0, temp)).exp()
    rank = torch.arange(v, device=x.device)
    keep = (rank < per_row["top_k"]) | (per_row["top_k"] <= 0)
    part = e * keep
    mass = part.cumsum(-1)
    keep &= (mass - part < top_p * mass[:, -1:]) | (top_p >= 1)
    keep &= e >= per_row["min_p"].double().clamp(max=1)
    keep = torch.where(greedy, rank == 0, keep | (rank == 0))
    back = torch.zeros_like(keep).scatter_(1, order, keep)
    return back, torch.zeros_like(e).scatter_(1, order, e)


def _plain_sample(s):
    keep, e = _kept(s)
    chance = torch.where(keep, e / s["noise"], -1.0)
    lowest = torch.arange(keep.shape[-1], 0, -1, device=keep.device)
    token = ((chance == chance.amax(-1, keepdim=True)) * lowest).argmax(-1)
    # a temperature of 0 leaves one token, drawn for certain
    e = torch.where(keep, e, 0.0)
    return {"token": token, "logprob": (e.gather(1, token[:, None]).squeeze(1) / e.sum(-1)).log().float()}


def _plain_filter(s):
    keep, _ = _kept(s)
    return {"logits": torch.where(keep.view(s["logits"].shape), s["logits"], -math.inf)}


def _plain_adapters(s):
    x, adapter = s["x"].float(), s["adapter"].long()
    pool, r, ic = s["a"].shape
    # every adapter's products, those of the others than a token's own set to zero
    mine = (adapter[:, None] == torch.arange(pool, device=x.device)).float() * s["scale"]
    h = (x @ s["a"].float().reshape(-1, ic).T).view(-1, pool, r) * mine[:, :, None]
    return {"y": (s["y"].float() + h.flatten(1) @ s["b"].float().transpose(1, 2).reshape(pool * r, -1)).to(s["y"].dtype)}


def run(s):
    op = s["op"]
    if not own:
        return {"norm": _plain_norm, "sample": _plain_sample, "filter": _plain_filter, "adapters": _plain_adapters}[op](s)
    from spark_b200 import ops, rotary
    if op == "norm":
        args = (s["q"], s["k"], s["qw"], s["kw"], s["positions"], s["table"])
        how = {"eps": s["eps"], "interleaved": s["case"]["interleaved"]}
        if "dq" not in s:
            q, k = ops.qk_norm_rope(*args, **how)
            return {"q": q, "k": k}
        q, k = rotary.apply_qk_norm_rope(*args, **how)
        dq, dk, dqw, dkw = torch.autograd.grad((q, k), (s["q"], s["k"], s["qw"], s["kw"]), (s["dq"], s["dk"]))
        return {"q": q, "dqw": dqw, "dq": dq, "k": k, "dkw": dkw, "dk": dk}
    if op == "sample":
        token, logprob = ops.sample(s["logits"], s["noise"], **s["settings"], return_logprob=True)
        return {"token": token, "logprob": logprob}
    if op == "filter":
        return {"logits": ops.filter_logits(s["logits"], **s["settings"])}
    return {"y": ops.lora_add(s["y"], s["x"], s["a"], s["b"], s["adapter"], scale=s["scale"])}


# ------------------------------------------------------------------ what a pass needs
def work(case):
    t, e = case["t"], ITEM[case["dtype"]]
    if case["op"] == "norm":
        b = case["b"]
        values, table = b * t * (case["hq"] + case["hkv"]) * case["d"], min(b * t, case["positions"]) * case["rot"] * 4
        n = 2 * values * e + table + 8 * b * t
        if not case["train"]:
            return {"bytes": n, "flops": 7 * values}
        return {"bytes": n + 3 * values * e + table + 8 * b * t, "flops": 21 * values}
    if case["op"] in ("sample", "filter"):
        rows, v = case["b"] * t, case["vocab"]
        if case["op"] == "filter":
            return {"bytes": 2 * rows * v * e, "flops": 4 * rows * v}
        # the noise of every token where nothing is cut, else of the few that are left
        whole = sum(k == 0 and p >= 1 and least == 0 and temp > 0 for temp, k, p, least in settings(case))
        return {"bytes": rows * v * e + 4 * whole * v + 12 * rows, "flops": 4 * rows * v}
    ic, oc, r = case["ic"], case["oc"], case["r"]
    n = min(case["pool"], case["requests"])
    return {"bytes": e * (t * (ic + 2 * oc) + n * r * (ic + oc)) + 4 * t, "flops": 2 * t * r * (ic + oc)}


# ------------------------------------------------------------------ 64 bits
def _exact_norm(s):
    """Through complex numbers; the gradients by reverse differentiation of the definition in 64 bits."""
    case, out = s["case"], {}
    half = case["rot"] // 2
    z = s["table"].double()[s["positions"]][:, :, None]
    turn = torch.complex(z[..., :half].contiguous(), z[..., half:].contiguous())

    def forward(x, w):
        n = w * x / (x.square().mean(-1, keepdim=True) + s["eps"]).sqrt()
        part = n[..., :case["rot"]].unflatten(-1, (half, 2) if case["interleaved"] else (2, half))
        a, b = part.unbind(-1 if case["interleaved"] else -2)
        y = torch.complex(a.contiguous(), b.contiguous()) * turn
        y = torch.stack([y.real, y.imag], -1 if case["interleaved"] else -2).flatten(-2)
        return torch.cat([y, n[..., case["rot"]:]], -1)

    for name in ("q", "k"):
        x, w = s[name].detach().double(), s[name + "w"].detach().double()
        if "dq" not in s:
            out[name] = forward(x, w)
            continue
        # one sequence at a time
        parts, dw = [], torch.zeros_like(w)
        whole = turn
        for i in range(x.shape[0]):
            turn = whole[i:i + 1]
            leaf, lw = x[i:i + 1].clone().requires_grad_(), w.clone().requires_grad_()
            y = forward(leaf, lw)
            dx, g = torch.autograd.grad(y, (leaf, lw), s["d" + name][i:i + 1].double())
            parts.append((y.detach(), dx))
            dw += g
        turn = whole
        out[name], out["d" + name + "w"] = torch.cat([p[0] for p in parts]), dw
        out["d" + name] = torch.cat([p[1] for p in parts])
    return out


def _exact_rows(s):
    """One row at a time: (row, kept indices in falling order, their exponentials, all of them)."""
    x = s["logits"].double().cpu()
    rows = x.shape[1] if x.dim() == 3 else 1
    for n, row in enumerate(x.flatten(0, -2)):
        temp, k, p, least = (float(s["settings"][name][n // rows]) for name in ("temperature", "top_k", "top_p", "min_p"))
        order = torch.argsort(row, descending=True, stable=True)
        if temp == 0:
            yield n, order[:1], torch.ones(1, dtype=torch.float64)
            continue
        if k > 0:
            order = order[:int(k)]
        prob = torch.softmax(row[order] / temp, 0)
        count = len(order)
        if p < 1:
            # how many it takes for a mass of p
            count = int((prob.cumsum(0) < p).sum()) + 1
        count = max(1, min(count, int((prob >= least * prob[0]).sum())))
        yield n, order[:count], prob[:count]


def _exact_sample(s):
    token = torch.zeros(s["logits"].shape[0], dtype=torch.int64)
    logprob = torch.zeros(token.shape, dtype=torch.float64)
    noise = s["noise"].double().cpu()
    for n, order, prob in _exact_rows(s):
        chance = prob / noise[n][order]
        token[n] = order[chance == chance.max()].min()
        logprob[n] = torch.log(prob[order == token[n]][0] / prob.sum())
    return {"token": token, "logprob": logprob}


def _exact_filter(s):
    x = s["logits"].double().cpu()
    out = torch.full_like(x, -math.inf).flatten(0, -2)
    for n, order, _ in _exact_rows(s):
        out[n, order] = x.flatten(0, -2)[n, order]
    return {"logits": out.view(x.shape)}


def _exact_adapters(s):
    """One adapter at a time, its tokens alone."""
    y = s["y"].double()
    for i in range(s["a"].shape[0]):
        rows = (s["adapter"] == i).nonzero()[:, 0]
        h = torch.einsum("ti,ri->tr", s["x"][rows].double(), s["a"][i].double())
        y[rows] += float(s["scale"][i]) * torch.einsum("tr,or->to", h, s["b"][i].double())
    return {"y": y}


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "sample": _exact_sample, "filter": _exact_filter, "adapters": _exact_adapters}[case["op"]](s)
