"""Products with packed and expert-stacked weights, as cases to be timed and compared.

A model whose weights are stored in MXFP4 (and had their LoRAs merged there) is used in three ways: a few tokens at a time
(decode), many at once (prefill), and with gradients to its inputs (training of adapters in front of frozen weights).
Mixture-of-experts layers and batches with one adapter per request do the same with one weight per group of rows.

``listed()`` names cases of each, ``draw()`` gives more over the same ranges.  A case is a dict of plain values:

* ``op``: mx (one MXFP4 weight) | grouped (one weight per group of consecutive rows of x)
* ``weight``: mxfp4 | dense (experts in ``dtype``)
* ``tokens``, ``rows``, ``cols``: x is [tokens, cols], a weight [rows, cols], y [tokens, rows]
* ``experts``, ``used``: groups, and the rows of x that belong to one (the rest is padding of a fixed-size buffer)
* ``dtype``: bf16 | f16 of x and y;  ``quant``: x is quantised to MXFP4 for the product
* ``swizzled``: scales in the 128x4 order;  ``bias``;  ``train``: gradients too
"""

from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # decode of one token through a small projection (k / v of the 8B-shaped model): latency counts
        dict(name="mx decode small", op="mx", weight="mxfp4", tokens=1, rows=1024, cols=4096, dtype="bf16", quant=False,
             swizzled=False, bias=False, train=False),
        # decode of one token through the largest projection (gate / up): the weight's bytes count
        dict(name="mx decode gate", op="mx", weight="mxfp4", tokens=1, rows=14336, cols=4096, dtype="bf16", quant=False,
             swizzled=True, bias=False, train=False),
        # decode of a batch of 24 requests through the down projection, 4-bit inputs
        dict(name="mx decode batch", op="mx", weight="mxfp4", tokens=24, rows=4096, cols=14336, dtype="bf16", quant=True,
             swizzled=False, bias=False, train=False),
        # prefill with 4-bit inputs, the largest projection
        dict(name="mx prefill 4-bit", op="mx", weight="mxfp4", tokens=4096, rows=14336, cols=4096, dtype="bf16",
             quant=True, swizzled=True, bias=False, train=False),
        # a prompt of odd length through a layer of odd sizes with a bias, fp16, inputs not quantised
        dict(name="mx prompt odd", op="mx", weight="mxfp4", tokens=777, rows=2001, cols=2080, dtype="f16", quant=False,
             swizzled=False, bias=True, train=False),
        # training in front of a frozen packed weight: forward and the input's gradient
        dict(name="mx train", op="mx", weight="mxfp4", tokens=2048, rows=14336, cols=4096, dtype="bf16", quant=False,
             swizzled=False, bias=False, train=True),
        # decode through experts: 8 tokens, two experts each
        dict(name="experts decode", op="grouped", weight="mxfp4", tokens=16, used=16, rows=2816, cols=2048, experts=32,
             dtype="bf16", quant=False, swizzled=False, train=False),
        # decode in buffers of a fixed size, as a captured graph has them, 4-bit inputs
        dict(name="experts decode padded", op="grouped", weight="mxfp4", tokens=128, used=100, rows=2048, cols=1408,
             experts=64, dtype="bf16", quant=True, swizzled=True, train=False),
        # prefill through experts, 4-bit inputs
        dict(name="experts prefill 4-bit", op="grouped", weight="mxfp4", tokens=8192, used=8192, rows=2816, cols=2048,
             experts=32, dtype="bf16", quant=True, swizzled=False, train=False),
        # training in front of frozen packed experts
        dict(name="experts train packed", op="grouped", weight="mxfp4", tokens=4096, used=4096, rows=2048, cols=1408,
             experts=16, dtype="bf16", quant=False, swizzled=False, train=True),
        # training of dense experts: forward, the input's gradient and the weights'
        dict(name="experts train dense", op="grouped", weight="dense", tokens=4096, used=4096, rows=4096, cols=2048,
             experts=8, dtype="bf16", quant=False, swizzled=False, train=True),
        # one LoRA per request: the down factors (rank 16) of 24 adapters, trained
        dict(name="adapters train", op="grouped", weight="dense", tokens=2048, used=2048, rows=16, cols=4096, experts=24,
             dtype="bf16", quant=False, swizzled=False, train=True),
    ]


def _spread(rng, lo, hi):
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


def _size(rng, lo, hi, unit):
    return max(unit, int(_spread(rng, lo, hi)) // unit * unit)


def draw(rng: random.Random):
    op = rng.choice(["mx", "grouped"])
    weight = "mxfp4" if op == "mx" else rng.choice(["mxfp4", "mxfp4", "dense"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f16"])
    train = rng.random() < 0.35
    quant = weight == "mxfp4" and not train and rng.random() < 0.5
    tokens = _size(rng, 1, 8192, 1)
    if weight == "dense" and rng.random() < 0.4:  # LoRA factors: a rank on one side
        rank, wide = rng.choice([4, 8, 16, 24, 32, 64]), _size(rng, 256, 8192, rng.choice([1, 8, 64, 128]))
        rows, cols = (rank, wide) if rng.random() < 0.5 else (wide, rank)
    else:
        rows = _size(rng, 64, 16384, rng.choice([1, 8, 64, 128, 128]))
        cols = _size(rng, 128, 16384, rng.choice([128, 128, 32]) if weight == "mxfp4" else rng.choice([128, 64, 8, 1]))
    products = (3 if weight == "dense" else 2) if train else 1
    case = dict(op=op, weight=weight, dtype=dtype, quant=quant, train=train)
    if op == "mx":
        rows = min(rows, (1 << 27) // cols)
        case |= dict(bias=not train and rng.random() < 0.3)
        experts = 1
    else:
        experts = rng.choice([1, 2, 4, 8, 16, 24, 32, 64])
        experts = max(1, min(experts, (1 << 27) // (rows * cols)))
        rows = min(rows, (1 << 27) // cols)
    tokens = max(1, min(tokens, int(1.2e11 / (rows * cols * products))))
    if op == "grouped":
        case |= dict(experts=experts, used=tokens if rng.random() < 0.7 else rng.randint(tokens // 2, tokens))
    return case | dict(tokens=tokens, rows=rows, cols=cols, swizzled=weight == "mxfp4" and rng.random() < 0.5)


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


def _swizzle(s):
    """[n, c] -> the order of 128-row by 4-column tiles, padded with zeros: 32 groups of 4 rows x 4 columns a tile."""
    n, c = s.shape[-2:]
    s = torch.nn.functional.pad(s, (0, -c % 4, 0, -n % 128))
    lead, (n, c) = s.shape[:-2], s.shape[-2:]
    s = s.reshape(-1, n // 128, 4, 32, c // 4, 4).permute(0, 1, 4, 3, 2, 5)
    return s.reshape(*lead, n // 4, c * 4).contiguous()


def _encode(w):
    """MXFP4 codes and scales of a dense weight [..., n, k] (any encoder would do: these are the stored weights)."""
    blocks = w.unflatten(-1, (-1, 32))
    amax = blocks.abs().amax(-1, keepdim=True).clamp_min(1e-30)
    e = torch.floor(torch.log2(amax)) - 2
    v = blocks * torch.exp2(-e)
    a = v.abs()
    code = sum((a > t).to(torch.uint8) for t in (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0))
    code = (code | ((v < 0).to(torch.uint8) << 3)).flatten(-2)
    return code[..., 0::2] | code[..., 1::2] << 4, (e.squeeze(-1) + 127).to(torch.uint8)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    t, n, k = case["tokens"], case["rows"], case["cols"]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    state = dict(case=case)
    # activations: a scale of its own for every token, and a few channels that stand out, as after a norm
    loud = 1 + 7 * (torch.rand(k, generator=g, device="cuda") < 0.01)
    state["x"] = (normal(t, k) * torch.exp(0.3 * normal(t, 1)) * loud).to(dtype)
    if case["op"] == "grouped":
        sizes = _sizes(case, seed)
        state["cap"] = max(1, max(sizes))  # the plain form's padding
        state["ends"] = torch.tensor(sizes, device="cuda").cumsum(0).to(torch.int32)
    shape = (case["experts"], n, k) if case["op"] == "grouped" else (n, k)
    if case["weight"] == "dense":
        state["weight"] = (normal(*shape) * k ** -0.5).to(dtype)
    else:
        qdata, scale = _encode(normal(*shape) * 0.02)
        state["qdata"], state["scale"] = qdata, _swizzle(scale) if case["swizzled"] else scale
    if case.get("bias"):
        state["bias"] = (normal(n) * 0.1).to(dtype)
    if case["train"]:
        state["dy"] = (normal(t, n) * 0.01).to(dtype)
    return state


# ---------------------------------------------------------------------------
# the plain form: elementary operations in 32 bits
# ---------------------------------------------------------------------------
_E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _plain_scales(scale, n, c, swizzled):
    if not swizzled:
        return scale
    rows, cols = -(-n // 128) * 128, -(-c // 4) * 4
    s = scale.reshape(-1, rows // 128, cols // 4, 32, 4, 4).permute(0, 1, 4, 3, 2, 5).reshape(-1, rows, cols)
    return s[:, :n, :c].reshape(scale.shape[:-2] + (n, c))


def _plain_weight(state):
    """The weight's values in 32 bits."""
    case = state["case"]
    if case["weight"] == "dense":
        return state["weight"].float()
    q = state["qdata"]
    table = torch.tensor(_E2M1 + [-v for v in _E2M1], device=q.device)
    v = torch.stack((table[(q & 15).int()], table[(q >> 4).int()]), -1).flatten(-2)
    s = _plain_scales(state["scale"], case["rows"], case["cols"] // 32, case["swizzled"])
    return (v.unflatten(-1, (-1, 32)) * torch.exp2(s.float() - 127).unsqueeze(-1)).flatten(-2)


def _plain_quantised(x):
    """x [t, k] on the MXFP4 grid: blocks of 32, the scale 2^(floor(log2 max) - 2), nearest with ties to even, up to 6."""
    blocks = x.float().unflatten(-1, (-1, 32))
    amax = blocks.abs().amax(-1, keepdim=True)
    exponent = (amax.view(torch.int32) >> 23) - 127 - 2
    scale = torch.exp2(exponent.clamp_min(-126).float())
    v = blocks / scale
    a = v.abs()
    code = (a > 0.25).int() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)
    q = torch.tensor(_E2M1, device=x.device)[code]
    return (torch.where(v < 0, -q, q) * scale).flatten(-2)


def _plain(state):
    case, x = state["case"], state["x"]
    dtype = x.dtype
    w = _plain_weight(state)
    x32 = _plain_quantised(x) if case["quant"] else x.float()
    if case["op"] == "mx":
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

    xs = batched(x32)
    y = back(torch.bmm(xs, w.transpose(1, 2)))
    if not case["train"]:
        return y
    dys = batched(state["dy"].float())
    out = {"y": y, "dx": back(torch.bmm(dys, w))}
    if case["weight"] == "dense":
        out["dw"] = torch.bmm(dys.transpose(1, 2), xs).to(dtype)
    return out


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
    case, x = state["case"], state["x"]
    packed = dict(swizzled=case["swizzled"])
    four = dict(packed, activation_dtype=torch.float4_e2m1fn_x2 if case["quant"] else None)
    if case["op"] == "mx":
        q, s = state["qdata"], state["scale"]
        y = k.mx_matmul(x, q, s, bias=state.get("bias"), **four)
        return {"y": y, "dx": k.mx_matmul_input_grad(state["dy"], q, s, **packed)} if case["train"] else y
    ends = state["ends"]
    if case["weight"] == "dense":
        y = k.grouped_matmul(x, state["weight"], ends)
        if not case["train"]:
            return y
        return {"y": y, "dx": k.grouped_matmul_input_grad(state["dy"], state["weight"], ends),
                "dw": k.grouped_matmul_weight_grad(state["dy"], x, ends)}
    q, s = state["qdata"], state["scale"]
    y = k.grouped_mx_matmul(x, q, s, ends, **four)
    return {"y": y, "dx": k.grouped_mx_matmul_input_grad(state["dy"], q, s, ends, **packed)} if case["train"] else y


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    """Inputs read once, outputs written once; weights of experts that no row chose are not read."""
    t, n, k = case["tokens"], case["rows"], case["cols"]
    used, read, experts = t, 1, 1
    if case["op"] == "grouped":
        used, experts = case["used"], case["experts"]
        read = sum(s > 0 for s in _sizes(case, 0))
    weight = n * k * 2 if case["weight"] == "dense" else n * k // 2 + n * k // 32
    size = used * k * 2 + read * weight + t * n * 2 + (n * 2 if case.get("bias") else 0)
    products = 1
    if case["train"]:
        products = 2
        size += used * n * 2 + t * k * 2
        if case["weight"] == "dense":
            products = 3
            size += experts * n * k * 2
    return {"bytes": size, "flops": 2 * used * n * k * products}


# ---------------------------------------------------------------------------
# 64 bits, from the definition
# ---------------------------------------------------------------------------
def _exact_weight(state):
    case = state["case"]
    if case["weight"] == "dense":
        return state["weight"].double()
    n, k = case["rows"], case["cols"]
    q = state["qdata"]
    shifts = torch.tensor([0, 4], device=q.device, dtype=torch.uint8)
    code = (q.unsqueeze(-1) >> shifts).bitwise_and(15).reshape(*q.shape[:-1], k)
    mantissa, exponent = (code & 1).double(), ((code >> 1) & 3).double()
    v = torch.where(exponent == 0, mantissa / 2, (1 + mantissa / 2) * 2 ** (exponent - 1))
    v = torch.where(code >= 8, -v, v)
    # the place of the scale of (row, block): tiles of 128 x 4, rows r, r + 32, r + 64, r + 96 side by side
    r, c = torch.arange(n, device=q.device)[:, None], torch.arange(k // 32, device=q.device)[None]
    if case["swizzled"]:
        at = ((r // 128) * (-(-k // 128)) + c // 4) * 512 + (r % 32) * 16 + (r % 128) // 32 * 4 + c % 4
    else:
        at = r * (k // 32) + c
    s = state["scale"].reshape(*q.shape[:-2], -1)[..., at.reshape(-1)].reshape(*q.shape[:-1], k // 32)
    v *= torch.pow(2.0, s.double() - 127).repeat_interleave(32, -1)
    return v


def _exact_quantised(x):
    blocks = x.double().reshape(x.shape[0], -1, 32)
    _, p = torch.frexp(blocks.abs().amax(-1, keepdim=True))  # max = m 2^p, 1/2 <= m < 1
    scale = torch.pow(2.0, (p - 3).clamp(-127, 127).double())
    v = blocks / scale
    a = v.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).double()
    return (torch.sign(v) * (torch.round(a / step) * step).clamp(max=6) * scale).reshape(x.shape)


def exact(case, seed):
    state = prepare(case, seed)
    w = _exact_weight(state)
    x = _exact_quantised(state["x"]) if case["quant"] else state["x"].double()
    dy = state["dy"].double() if case["train"] else None
    t, n, k = case["tokens"], case["rows"], case["cols"]
    if case["op"] == "mx":
        y = x @ w.t() + (state["bias"].double() if case["bias"] else 0.0)
        return {"y": y, "dx": dy @ w} if case["train"] else y
    y, dx, dw = x.new_zeros(t, n), x.new_zeros(t, k), torch.zeros_like(w)
    begin = 0
    for e, end in enumerate(state["ends"].tolist()):
        if end > begin:
            y[begin:end] = x[begin:end] @ w[e].t()
            if case["train"]:
                dx[begin:end] = dy[begin:end] @ w[e]
                dw[e] = dy[begin:end].t() @ x[begin:end]
        begin = end
    if not case["train"]:
        return y
    return {"y": y, "dx": dx, "dw": dw} if case["weight"] == "dense" else {"y": y, "dx": dx}
