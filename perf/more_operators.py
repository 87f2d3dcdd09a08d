"""Mixtures of experts and linears over merged INT8 weights, as cases to be timed and compared.

A model whose weights are stored in INT8 with one scale per output channel (and had their LoRAs merged there) runs its
linears over them as they are stored, either with its inputs in 16 bits or with every token's inputs quantised to INT8,
one scale per token.  A mixture of experts first routes its tokens, brings the rows of one expert side by side, and
adds up what the experts return.

``listed()`` names cases of each, ``draw()`` gives more over the same ranges.  A case is a dict of plain values:

* ``op``: int8 (one weight) | grouped (one INT8 weight per group of consecutive rows) | route | rows
* ``dtype``: bf16 | f16 | f32 (logits only);  ``train``: gradients too
* int8, grouped: ``tokens``, ``rows``, ``cols``: x is [tokens, cols], a weight [rows, cols], y [tokens, rows];
  ``quant``: x is quantised for the product; ``bias``; ``experts``, ``used``: groups, and the rows of x that belong to one
* route: ``tokens``, ``used`` (the rest of a fixed-size batch is padding), ``experts``, ``best`` (experts of a token),
  ``score`` (softmax | sigmoid), ``bias`` (added for the choice alone), ``groups``, ``top_groups``, ``group_best``,
  ``renormalize``, ``scale``
* rows: ``tokens``, ``used``, ``cols``, ``experts``, ``best``: rows taken to their experts, and back as weighted sums
"""

from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # decode of one token through a small projection (k / v of the 8B-shaped model): latency counts
        dict(name="int8 decode small", op="int8", tokens=1, rows=1024, cols=4096, dtype="bf16", quant=True, bias=False,
             train=False),
        # decode of one token through the largest projection (gate / up), inputs in 16 bits: the weight's bytes count
        dict(name="int8 decode gate", op="int8", tokens=1, rows=14336, cols=4096, dtype="bf16", quant=False, bias=False,
             train=False),
        # a prompt of odd length through a layer of odd sizes with a bias, fp16
        dict(name="int8 prompt odd", op="int8", tokens=777, rows=2001, cols=2083, dtype="f16", quant=True, bias=True,
             train=False),
        # prefill through the largest projection, 8-bit inputs
        dict(name="int8 prefill", op="int8", tokens=4096, rows=14336, cols=4096, dtype="bf16", quant=True, bias=False,
             train=False),
        # training in front of a frozen weight: forward with 16-bit inputs and the input's gradient
        dict(name="int8 train", op="int8", tokens=2048, rows=14336, cols=4096, dtype="bf16", quant=False, bias=False,
             train=True),
        # decode through experts in buffers of a fixed size, as a captured graph has them
        dict(name="experts int8 decode", op="grouped", tokens=128, used=100, rows=2048, cols=1408, experts=64,
             dtype="bf16", quant=True, train=False),
        # training in front of frozen experts, 8-bit inputs in the forward
        dict(name="experts int8 train", op="grouped", tokens=4096, used=4096, rows=2816, cols=2048, experts=32,
             dtype="bf16", quant=True, train=True),
        # routing of a decode batch: latency counts
        dict(name="route decode", op="route", tokens=8, used=8, experts=32, best=4, score="softmax", bias=False, groups=1,
             top_groups=1, group_best=1, renormalize=True, scale=1.0, dtype="bf16", train=False),
        # routing of a prefill among many experts: balance bias, groups of experts, scaled weights, some padding
        dict(name="route prefill groups", op="route", tokens=16384, used=16000, experts=256, best=8, score="sigmoid",
             bias=True, groups=8, top_groups=4, group_best=2, renormalize=True, scale=2.5, dtype="f32", train=False),
        # routing in training, with the gradient to the logits
        dict(name="route train", op="route", tokens=8192, used=8192, experts=64, best=4, score="softmax", bias=False,
             groups=1, top_groups=1, group_best=1, renormalize=False, scale=1.0, dtype="bf16", train=True),
        # a decode batch's rows to their experts and back
        dict(name="rows decode", op="rows", tokens=16, used=16, cols=2048, experts=32, best=4, dtype="bf16", train=False),
        # a training batch's rows to their experts and back, with all gradients
        dict(name="rows train", op="rows", tokens=8192, used=8192, cols=2048, experts=32, best=4, dtype="bf16",
             train=True),
    ]


def _spread(rng, lo, hi):
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


def _size(rng, lo, hi, unit=1):
    return max(unit, int(_spread(rng, lo, hi)) // unit * unit)


def _draw_product(rng, op):
    train = rng.random() < 0.35
    case = dict(op=op, dtype=rng.choice(["bf16", "bf16", "f16"]), quant=rng.random() < 0.6, train=train)
    rows = _size(rng, 64, 16384, rng.choice([1, 8, 64, 128, 128]))
    cols = _size(rng, 64, 16384, rng.choice([1, 8, 16, 64, 128, 128]))
    experts = 1
    if op == "grouped":
        experts = rng.choice([2, 4, 8, 16, 24, 32, 64])
        experts = max(1, min(experts, (1 << 28) // (rows * cols)))
    else:
        case |= dict(bias=not train and rng.random() < 0.3)
    rows = min(rows, (1 << 27) // cols)
    tokens = max(1, min(_size(rng, 1, 8192), int(2e11 / (rows * cols * (2 if train else 1)))))
    if op == "grouped":
        case |= dict(experts=experts, used=tokens if rng.random() < 0.7 else rng.randint(tokens // 2, tokens))
    return case | dict(tokens=tokens, rows=rows, cols=cols)


def _draw_route(rng):
    tokens = _size(rng, 1, 32768)
    groups = rng.choice([1, 1, 2, 4, 8])
    each = _size(rng, 2 if groups > 1 else 4, 512 // groups)
    experts = groups * each
    tokens = min(tokens, (1 << 22) // experts)
    top_groups = rng.randint(1, groups)
    best = rng.randint(1, min(12, top_groups * each))
    return dict(op="route", tokens=tokens, used=tokens if rng.random() < 0.6 else rng.randint(tokens // 2, tokens),
                experts=experts, best=best, score=rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.5,
                groups=groups, top_groups=top_groups, group_best=rng.randint(1, min(2, each)),
                renormalize=rng.random() < 0.6, scale=rng.choice([1.0, 1.0, 2.5]),
                dtype=rng.choice(["bf16", "f16", "f32"]), train=rng.random() < 0.5)


def _draw_rows(rng):
    cols = _size(rng, 64, 8192, rng.choice([1, 8, 64, 128]))
    experts = _size(rng, 4, 256)
    best = rng.randint(1, min(8, experts))
    tokens = max(1, min(_size(rng, 1, 16384), (1 << 26) // (cols * best)))
    return dict(op="rows", tokens=tokens, used=tokens if rng.random() < 0.6 else rng.randint(tokens // 2, tokens),
                cols=cols, experts=experts, best=best, dtype=rng.choice(["bf16", "bf16", "f16"]), train=rng.random() < 0.5)


def draw(rng: random.Random):
    op = rng.choice(["int8", "grouped", "route", "rows"])
    if op == "route":
        return _draw_route(rng)
    if op == "rows":
        return _draw_rows(rng)
    return _draw_product(rng, op)


# ---------------------------------------------------------------------------
# inputs, in plain torch
# ---------------------------------------------------------------------------
def _sizes(case, seed):
    """Rows per expert: a skewed choice for every row, some experts never chosen; the seed says which expert is which."""
    n = case["experts"]
    rng = random.Random(case["tokens"] * 1000 + n)
    likely = [math.exp(rng.gauss(0.0, 0.5)) if i % 7 else 0.0 for i in range(1, n + 1)]
    sizes = [0] * n
    for i in rng.choices(range(n), likely, k=case["used"]):
        sizes[i] += 1
    turn = seed % n
    return sizes[turn:] + sizes[:turn]


def _activations(normal, uniform, t, k, dtype):
    """A scale of its own for every token, and a few channels that stand out, as after a norm."""
    return (normal(t, k) * torch.exp(0.3 * normal(t, 1)) * (1 + 7 * (uniform(k) < 0.01))).to(dtype)


def _prepare_product(case, state, seed, normal, uniform):
    t, n, k, dtype = case["tokens"], case["rows"], case["cols"], DTYPES[case["dtype"]]
    state["x"] = _activations(normal, uniform, t, k, dtype)
    shape = (n, k)
    if case["op"] == "grouped":
        sizes = _sizes(case, seed)
        state["cap"] = max(1, max(sizes))  # the plain form's padding
        state["ends"] = torch.tensor(sizes, device="cuda").cumsum(0).to(torch.int32)
        shape = (case["experts"], n, k)
    w = normal(*shape) * 0.02
    scale = w.abs().amax(-1, keepdim=True) / 127
    state["qdata"], state["scale"] = torch.round(w / scale).clamp(-128, 127).to(torch.int8), scale
    if case.get("bias"):
        state["bias"] = (normal(n) * 0.1).to(dtype)
    if case["train"]:
        state["dy"] = (normal(t, n) * 0.01).to(dtype)


def _prepare_route(case, state, normal):
    t, e = case["tokens"], case["experts"]
    logits = normal(t, e) * 1.5 + normal(e) * 0.5  # some experts are liked by most tokens
    logits[case["used"]:] = -math.inf  # padding: no expert at all
    state["logits"] = logits.to(DTYPES[case["dtype"]])
    if case["bias"]:
        state["bias"] = normal(e) * 0.05
    if case["train"]:
        state["dweight"] = normal(t, case["best"]) * 0.1


def _prepare_rows(case, state, normal, uniform):
    t, k, e, dtype = case["tokens"], case["cols"], case["experts"], DTYPES[case["dtype"]]
    state["x"] = _activations(normal, uniform, t, k, dtype)
    logits = normal(t, e) + normal(e) * 0.5
    value, expert = logits.topk(case["best"], -1)
    state["weight"] = value.softmax(-1)
    live = torch.arange(t, device="cuda") < case["used"]
    expert = torch.where(live[:, None], expert, e).reshape(-1)
    state["weight"][case["used"]:] = 0
    place = torch.empty_like(expert)
    place[expert.argsort(stable=True)] = torch.arange(expert.numel(), device="cuda")
    state["position"] = place.to(torch.int32).view(t, -1)
    state["ends"] = torch.bincount(expert, minlength=e + 1)[:e].cumsum(0).to(torch.int32)
    # what the experts return; padding gives zeros
    h = normal(t * case["best"], k)
    h[case["used"] * case["best"]:] = 0
    state["h"] = h.to(dtype)
    if case["train"]:
        state["dout"] = (normal(t, k) * 0.01).to(dtype)
        state["drows"] = (normal(t * case["best"], k) * 0.01).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    def uniform(*shape):
        return torch.rand(shape, generator=g, device="cuda")

    state = dict(case=case)
    if case["op"] == "route":
        _prepare_route(case, state, normal)
    elif case["op"] == "rows":
        _prepare_rows(case, state, normal, uniform)
    else:
        _prepare_product(case, state, seed, normal, uniform)
    return state


# ---------------------------------------------------------------------------
# the plain form: elementary operations in 32 bits
# ---------------------------------------------------------------------------
def _plain_quantised(x):
    """Codes and the scale of every row: the largest magnitude / 127; the quotients (in 64 bits, for those next to a
    border) rounded to the nearest whole number, ties to even."""
    scale = x.float().abs().amax(-1, keepdim=True) / 127
    q = torch.round(x.double() / torch.where(scale > 0, scale, 1.0).double()).clamp(-127, 127)
    return q.float(), scale


def _plain_product(state):
    case, x = state["case"], state["x"]
    dtype = x.dtype
    w = state["qdata"].float() * state["scale"]
    x32 = x.float()
    if case["quant"]:
        q, s = _plain_quantised(x)
        x32 = q * s
    if case["op"] == "int8":
        y = x32 @ w.t()
        if case["bias"]:
            y = y + state["bias"].float()
        if not case["train"]:
            return y.to(dtype)
        return {"y": y.to(dtype), "dx": (state["dy"].float() @ w).to(dtype)}
    # groups: rows gathered into [experts, cap, .], products over the batch of experts, rows taken back
    ends = state["ends"].long()
    t, cap = x.shape[0], state["cap"]
    starts = torch.cat((ends.new_zeros(1), ends[:-1]))
    slot = torch.arange(cap, device=x.device)
    row = starts[:, None] + slot
    inside = (row < ends[:, None])[..., None]
    row = row.clamp(max=t - 1)
    expert = (torch.arange(t, device=x.device)[:, None] >= ends).sum(1)
    routed = (expert < ends.numel())[:, None]
    expert = expert.clamp(max=ends.numel() - 1)
    place = (torch.arange(t, device=x.device) - starts[expert]).clamp(max=cap - 1)

    def batched(rows):
        return torch.where(inside, rows[row], 0.0)

    def back(y):
        return torch.where(routed, y[expert, place], 0.0).to(dtype)

    y = back(torch.bmm(batched(x32), w.transpose(1, 2).contiguous()))
    if not case["train"]:
        return y
    return {"y": y, "dx": back(torch.bmm(batched(state["dy"].float()), w))}


def _plain_route(state):
    case = state["case"]
    logits = state["logits"].double()  # (64 bits: scores next to each other decide between experts)
    t, e = logits.shape
    k = case["best"]
    open_ = logits > -math.inf
    if case["score"] == "softmax":
        top = logits.amax(-1, keepdim=True)
        s = torch.exp(logits - torch.where(top > -math.inf, top, 0.0))
        s = s / s.sum(-1, keepdim=True).clamp_min(1e-300)
    else:
        s = 1 / (1 + torch.exp(-logits))
    choice = s + state["bias"].double() if case["bias"] else s
    choice = torch.where(open_, choice, -math.inf)
    if case["groups"] > 1:
        each = choice.view(t, case["groups"], -1).sort(-1, descending=True).values[..., :case["group_best"]]
        value = each[..., 0]
        if case["group_best"] == 2:
            value = value + torch.where(each[..., 1] > -math.inf, each[..., 1], 0.0)
        kept = value.sort(dim=-1, descending=True, stable=True).indices[:, :case["top_groups"]]
        keep = torch.zeros_like(value).scatter_(1, kept, 1.0) > 0
        choice = torch.where(keep.repeat_interleave(e // case["groups"], 1), choice, -math.inf)
    value, expert = choice.sort(dim=-1, descending=True, stable=True)
    chosen, expert = value[:, :k] > -math.inf, expert[:, :k]
    picked = torch.where(chosen, s.gather(1, expert), 0.0)
    total = picked.sum(-1, keepdim=True).clamp_min(1e-300)
    weight = (picked / total if case["renormalize"] else picked) * case["scale"]
    # rows of one expert side by side, in the order of the tokens; choices that no expert takes come last
    key = torch.where(chosen, expert, e).reshape(-1)
    place = torch.empty_like(key)
    place[key.sort(dim=-1, stable=True).indices] = torch.arange(t * k, device=key.device)
    ends = (key[:, None] == torch.arange(e, device=key.device)).sum(0).cumsum(0)
    out = {"weight": weight.float(), "expert": torch.where(chosen, expert, -1).int(), "position": place.view(t, k).int(),
           "ends": ends.int()}
    if case["train"]:
        g = torch.where(chosen, state["dweight"].double(), 0.0)
        if case["renormalize"]:
            ds = case["scale"] * (g - (g * picked).sum(-1, keepdim=True) / total) / total
        else:
            ds = case["scale"] * g
        ds = torch.zeros_like(s).scatter_(1, expert, torch.where(chosen, ds, 0.0))
        dl = s * (ds - (s * ds).sum(-1, keepdim=True)) if case["score"] == "softmax" else s * (1 - s) * ds
        out["dlogits"] = dl.to(state["logits"].dtype)
    return out


def _plain_rows(state):
    case, x, h = state["case"], state["x"], state["h"]
    t, k = state["position"].shape
    position = state["position"].long()
    live = (position < state["ends"][-1]).reshape(-1, 1)
    source = torch.empty_like(position.view(-1))
    source[position.view(-1)] = torch.arange(t * k, device=x.device)
    taken = live[source]
    rows = torch.where(taken, x[source // k], 0.0)
    back = torch.where(live, h.float()[position.view(-1)], 0.0).view(t, k, -1)
    y = (state["weight"][..., None] * back).sum(1).to(x.dtype)
    if not case["train"]:
        return {"rows": rows, "y": y}
    dx = torch.where(live, state["drows"].float()[position.view(-1)], 0.0).view(t, k, -1).sum(1)
    dy = state["dout"].float()
    dh = torch.where(taken, state["weight"].view(-1)[source, None] * dy[source // k], 0.0)
    dweight = (back * dy[:, None]).sum(-1)
    return {"rows": rows, "y": y, "dx": dx.to(x.dtype), "dh": dh.to(x.dtype), "dweight": dweight}


def _plain(state):
    op = state["case"]["op"]
    return _plain_route(state) if op == "route" else _plain_rows(state) if op == "rows" else _plain_product(state)


# ---------------------------------------------------------------------------
# the framework's operators
# ---------------------------------------------------------------------------
def _kernels():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "piper-offload_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from piper_offload_amd import kernels

    return kernels


def _own(state):
    k = _kernels()
    case = state["case"]
    if case["op"] == "route":
        how = dict(score=case["score"], renormalize=case["renormalize"], scale=case["scale"])
        r = k.route_topk(state["logits"], case["best"], bias=state.get("bias"), groups=case["groups"],
                         top_groups=case["top_groups"], group_best=case["group_best"], **how)
        out = {"weight": r.weight, "expert": r.expert, "position": r.position, "ends": r.ends}
        if case["train"]:
            out["dlogits"] = k.route_topk_grad(state["dweight"], state["logits"], r.expert, **how)
        return out
    if case["op"] == "rows":
        at = (state["position"], state["ends"])
        out = {"rows": k.dispatch_rows(state["x"], *at), "y": k.combine_rows(state["h"], state["weight"], *at)}
        if case["train"]:
            out["dx"] = k.dispatch_rows_grad(state["drows"], *at)
            out["dh"], out["dweight"] = k.combine_rows_grad(state["dout"], state["h"], state["weight"], *at)
        return out
    x, q, s = state["x"], state["qdata"], state["scale"]
    eight = dict(activation_dtype=torch.int8 if case["quant"] else None)
    if case["op"] == "int8":
        y = k.int8_matmul(x, q, s, bias=state.get("bias"), **eight)
        return {"y": y, "dx": k.int8_matmul_input_grad(state["dy"], q, s)} if case["train"] else y
    y = k.grouped_int8_matmul(x, q, s, state["ends"], **eight)
    if not case["train"]:
        return y
    return {"y": y, "dx": k.grouped_int8_matmul_input_grad(state["dy"], q, s, state["ends"])}


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    """Inputs read once, outputs written once; weights of experts that no row chose are not read."""
    t, size = case["tokens"], 4 if case["dtype"] == "f32" else 2
    if case["op"] == "route":
        e, k = case["experts"], case["best"]
        moved = t * e * size + t * k * 12 + e * 4 + (e * 4 if case["bias"] else 0)
        # (the gradient reads the logits of softmax again, and writes as many)
        if case["train"]:
            moved += t * k * 4 + t * e * size
        return {"bytes": moved, "flops": t * e * (16 if case["train"] else 8)}
    if case["op"] == "rows":
        n, k = case["cols"], case["best"]
        one, many = t * n * 2, t * k * n * 2
        moved = 2 * (one + many) + t * k * 8
        if case["train"]:
            moved += one + many + one + many + t * k * 4  # dx from drows; dh and dweight from dout (h is in already)
        return {"bytes": moved, "flops": t * k * n * (6 if case["train"] else 2)}
    n, k = case["rows"], case["cols"]
    used, read = t, 1
    if case["op"] == "grouped":
        used, read = case["used"], sum(s > 0 for s in _sizes(case, 0))
    moved = used * k * 2 + read * (n * k + n * 4) + t * n * 2 + (n * 2 if case.get("bias") else 0)
    if case["train"]:
        moved += used * n * 2 + t * k * 2
    return {"bytes": moved, "flops": 2 * used * n * k * (2 if case["train"] else 1)}


# ---------------------------------------------------------------------------
# 64 bits, from the definition
# ---------------------------------------------------------------------------
def _exact_product(case, state):
    t, n, k = case["tokens"], case["rows"], case["cols"]
    w = state["qdata"].double()
    w *= state["scale"].double()
    x = state["x"].double()
    if case["quant"]:
        # the scale is a stored number of 32 bits; a row of zeros stays one
        top = x.abs().max(-1, keepdim=True).values
        s = (top.float() / 127).double()
        whole = (x / s).nan_to_num(0.0)
        low = whole.floor()
        part = whole - low
        up = (part > 0.5) | ((part == 0.5) & (low.remainder(2) == 1))
        x = (low + up).clamp(-127, 127) * s
    dy = state["dy"].double() if case["train"] else None
    if case["op"] == "int8":
        y = x @ w.t() + (state["bias"].double() if case["bias"] else 0.0)
        return {"y": y, "dx": dy @ w} if case["train"] else y
    y, dx = x.new_zeros(t, n), x.new_zeros(t, k)
    begin = 0
    for e, end in enumerate(state["ends"].tolist()):
        if end > begin:
            y[begin:end] = x[begin:end] @ w[e].t()
            if case["train"]:
                dx[begin:end] = dy[begin:end] @ w[e]
        begin = end
    return {"y": y, "dx": dx} if case["train"] else y


def _first_best(value):
    """The lowest index of the largest value of each row."""
    index = torch.arange(value.shape[-1], device=value.device)
    top = value.amax(-1, keepdim=True)
    return torch.where(value == top, index, value.shape[-1]).amin(-1)


def _exact_route(case, state):
    l = state["logits"].double()
    t, e = l.shape
    k, groups = case["best"], case["groups"]
    none = l == -math.inf
    if case["score"] == "softmax":
        p = torch.where(none.all(-1, keepdim=True), 0.0, torch.softmax(l, -1))
    else:
        p = torch.sigmoid(l)
    rank = (p + (state["bias"].double() if case["bias"] else 0.0)).masked_fill(none, -math.inf)
    if groups > 1:
        member = rank.reshape(t, groups, e // groups).clone()
        score = torch.full((t, groups), -math.inf, dtype=torch.double, device=l.device)
        for i in range(case["group_best"]):
            at = _first_best(member)[..., None]
            best = member.gather(-1, at)[..., 0]
            score = best if i == 0 else torch.where(best == -math.inf, score, score + best)
            member.scatter_(-1, at, -math.inf)
        allowed = torch.zeros(t, groups, dtype=torch.bool, device=l.device)
        for _ in range(case["top_groups"]):
            at = _first_best(score)[:, None]
            allowed |= torch.zeros_like(allowed).scatter_(1, at, True) & (score > -math.inf)
            score.scatter_(1, at, -math.inf)
        rank = rank.reshape(t, groups, -1).masked_fill(~allowed[..., None], -math.inf).reshape(t, e)
    rank = rank.clone()
    expert = torch.empty(t, k, dtype=torch.long, device=l.device)
    for j in range(k):
        at = _first_best(rank)
        some = rank.amax(-1) > -math.inf
        expert[:, j] = torch.where(some, at, -1)
        rank.scatter_(1, at[:, None], -math.inf)
    on = expert >= 0
    at = expert.clamp_min(0)
    w = torch.where(on, p.gather(1, at), 0.0)
    total = w.sum(1, keepdim=True)
    if case["renormalize"]:
        w = torch.where(on, w / torch.where(total > 0, total, 1.0), 0.0)
    w = w * case["scale"]
    # a choice's place: the choices of lower experts, and those of the same expert before it
    which = torch.where(on, expert, e).reshape(-1)
    count = torch.bincount(which, minlength=e + 1)
    first = count.cumsum(0) - count
    place = torch.empty_like(which)
    for i in range(e + 1):
        mine = (which == i).nonzero().view(-1)
        place[mine] = first[i] + torch.arange(mine.numel(), device=l.device)
    out = {"weight": w, "expert": expert, "position": place.view(t, k), "ends": count.cumsum(0)[:e]}
    if case["train"]:
        # through the derivatives of the weights to the logits, one choice at a time
        g = torch.where(on, state["dweight"].double(), 0.0)
        dl = torch.zeros_like(l)
        mean = (g * w).sum(1, keepdim=True)  # sum of g_j w_j
        for j in range(k):
            pj, wj, gj = p.gather(1, at[:, j:j + 1]), w[:, j:j + 1], g[:, j:j + 1]
            log = torch.ones_like(pj) if case["score"] == "softmax" else 1 - pj  # d log p_j / d l_j, the own part
            own_part = wj * (gj - mean / case["scale"]) if case["renormalize"] else wj * gj
            dl.scatter_add_(1, at[:, j:j + 1], torch.where(on[:, j:j + 1], own_part * log, 0.0))
        if case["score"] == "softmax" and not case["renormalize"]:
            dl -= p * mean
        out["dlogits"] = dl
    return out


def _exact_rows(case, state):
    x, h, position = state["x"].double(), state["h"].double(), state["position"].long()
    t, k = position.shape
    limit = int(state["ends"][-1])
    rows, dh = x.new_zeros(t * k, x.shape[1]), x.new_zeros(t * k, x.shape[1])
    y, dx, dweight = torch.zeros_like(x), torch.zeros_like(x), x.new_zeros(t, k)
    weight = state["weight"].double()
    for j in range(k):
        token = (position[:, j] < limit).nonzero().view(-1)
        at = position[token, j]
        rows[at] = x[token]
        y[token] += weight[token, j, None] * h[at]
        if case["train"]:
            dx[token] += state["drows"].double()[at]
            dout = state["dout"].double()[token]
            dh[at] = weight[token, j, None] * dout
            dweight[token, j] = torch.linalg.vecdot(dout, h[at])
    out = {"rows": rows, "y": y}
    return out | {"dx": dx, "dh": dh, "dweight": dweight} if case["train"] else out


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "route":
        return _exact_route(case, state)
    return _exact_rows(case, state) if case["op"] == "rows" else _exact_product(case, state)
