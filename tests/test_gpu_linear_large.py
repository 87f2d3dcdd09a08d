"""Products with MXFP4 weights and grouped products at the sizes where their larger tiles, split sums and wide workgroups
run, against sums in 64 bits on the same stored values (float64 products of whole matrices, also on the GPU).

Tolerance of one output: half a unit in the last place of its type (up to 2^-8 of it in bfloat16, 2^-11 in float16) and, for
an fp32 sum of n products in any order, at most n + 2 roundings of 2^-23 of the sum of magnitudes.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

K = pytest.importorskip("piper_offload_amd.kernels")

DEV = "cuda"
FP4 = getattr(torch, "float4_e2m1fn_x2", None)
BF16, F16 = torch.bfloat16, torch.float16


def _normal(seed, *shape, std=1.0, dtype=BF16):
    return (torch.randn(*shape, generator=torch.Generator(DEV).manual_seed(seed), device=DEV) * std).to(dtype)


def _decode(q, s, swizzled):
    n, blocks = q.shape[0], q.shape[1] // 16
    if swizzled:
        r, c = torch.arange(n, device=DEV)[:, None], torch.arange(blocks, device=DEV)[None]
        s = s.reshape(-1)[((r // 128) * (-(-blocks // 4)) + c // 4) * 512 + (r % 32) * 16 + (r % 128) // 32 * 4 + c % 4]
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64, device=DEV)
    v = grid[torch.stack((q & 15, q >> 4), -1).reshape(n, -1).int()]
    return v * torch.pow(2.0, s.double() - 127).repeat_interleave(32, 1)


def _weight(seed, n, k, swizzled):
    q, s = K.requantize_mx(_normal(seed, n, k, std=0.02), FP4, swizzled=swizzled)
    return q, s, _decode(q, s, swizzled)


def _quantised(x):
    """x on the MXFP4 grid: scale 2^(floor(log2 max) - 2), nearest (ties to even), up to 6."""
    b = x.double().reshape(x.shape[0], -1, 32)
    scale = torch.pow(2.0, (torch.frexp(b.abs().amax(-1, keepdim=True))[1] - 3).double())
    v = b / scale
    step = torch.where(v.abs() < 2, 0.5, torch.where(v.abs() < 4, 1.0, 2.0)).double()
    return (torch.sign(v) * (torch.round(v.abs() / step) * step).clamp(max=6) * scale).reshape(x.shape)


def _check(got, a, b):
    """got against a @ b in 64 bits."""
    a, b = a.double().contiguous(), b.double().contiguous()
    want, size = a @ b, a.abs() @ b.abs()
    half, tiny = (2.0**-8, 1e-38) if got.dtype is BF16 else (2.0**-11, 2.0**-25)
    tol = (1 + 2.0**-8) * half * want.abs() + (a.shape[1] + 2) * 2.0**-23 * size + tiny
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    assert (off <= tol).all(), f"{int((off > tol).sum())} of {off.numel()} off, worst {(off / tol).max():.3g} tolerances"


# few rows: columns past 256, 512 and 2048 workgroups of 16, contractions below and above 32 units of 128;
# tiles: 64, 128 and 256 rows, whole rounds of 256 tiles and a rest, contractions split over workgroups
MX_SHAPES = [(1, 4112, 4128), (3, 8208, 4128), (9, 4112, 4160), (12, 8208, 4256), (16, 4112, 1056), (50, 8200, 512),
             (60, 16400, 544), (150, 2064, 4128), (257, 4112, 2080), (520, 1040, 8224), (1030, 2064, 1056),
             (2050, 2320, 544), (4100, 4352, 1056), (4090, 4112, 288), (4100, 4112, 4128)]


@pytest.mark.parametrize("shape", MX_SHAPES, ids=str)
@pytest.mark.parametrize("dtype,swizzled", [(BF16, False), (BF16, True), (F16, True)], ids=["bf16", "bf16-swizzled", "f16"])
def test_mx(shape, dtype, swizzled):
    t, n, k = shape
    q, s, w = _weight(t + n, n, k, swizzled)
    x = _normal(t, t, k, dtype=dtype)
    _check(K.mx_matmul(x, q, s, swizzled=swizzled), x, w.t())
    _check(K.mx_matmul(x, q, s, swizzled=swizzled, activation_dtype=FP4), _quantised(x), w.t())
    dy = _normal(k, t, n, dtype=dtype)
    _check(K.mx_matmul_input_grad(dy, q, s, swizzled=swizzled), dy, w)


def _spans(sizes):
    end = 0
    for e, size in enumerate(sizes):
        yield e, end, end + size
        end += size


# sizes, N, K: the rests of the groups' tiles, groups of one row beside large ones, rows after the last group
GROUPS = [([1500, 0, 1, 2000, 700], 4112, 1568), ([255, 257, 0, 512, 1], 1040, 2080), ([9] * 20 + [0, 200], 1040, 4128),
          ([12, 1, 0, 40, 20] * 5, 528, 1056), ([3, 0, 1] * 10, 2064, 1056), ([130, 0, 900], 2064, 544),
          ([4000, 90], 4112, 2080)]
GIDS = [f"{'-'.join(map(str, s[:4]))}:{n}x{k}" for s, n, k in GROUPS]


@pytest.mark.parametrize("case", GROUPS, ids=GIDS)
@pytest.mark.parametrize("swizzled", [False, True], ids=["plain", "swizzled"])
def test_grouped_mx(case, swizzled):
    sizes, n, k = case
    stored = [_weight(e, n, k, swizzled) for e in range(len(sizes))]
    q, s = torch.stack([w[0] for w in stored]), torch.stack([w[1] for w in stored])
    t, ends = sum(sizes) + 5, torch.tensor(sizes).cumsum(0).to(torch.int32).to(DEV)
    x, dy = _normal(1, t, k), _normal(2, t, n)
    x[t - 5:] = float("nan")
    dy[t - 5:] = float("nan")
    y = K.grouped_mx_matmul(x, q, s, ends, swizzled=swizzled)
    y4 = K.grouped_mx_matmul(x, q, s, ends, swizzled=swizzled, activation_dtype=FP4)
    dx = K.grouped_mx_matmul_input_grad(dy, q, s, ends, swizzled=swizzled)
    for e, b, end in _spans(sizes):
        if end > b:
            _check(y[b:end], x[b:end], stored[e][2].t())
            _check(y4[b:end], _quantised(x[b:end]), stored[e][2].t())
            _check(dx[b:end], dy[b:end], stored[e][2])
    assert not y[t - 5:].any() and not y4[t - 5:].any() and not dx[t - 5:].any()


DENSE = [(s, n, k + d) for (s, n, k), d in zip(GROUPS, (0, 8, 0, 7, 0, 1, 4))] + \
    [([0, 4000], 130, 264), ([1], 4112, 4128), ([16], 2048, 4096), ([7000], 96, 64), ([64] * 130, 64, 256), ([40], 16400, 520),
     ([1000, 0, 5100, 2100], 2040, 2024)]


@pytest.mark.parametrize("case", DENSE, ids=[f"{'-'.join(map(str, s[:4]))}:{n}x{k}" for s, n, k in DENSE])
@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
def test_grouped_dense(case, dtype):
    sizes, n, k = case
    t, ends = sum(sizes) + 5, torch.tensor(sizes).cumsum(0).to(torch.int32).to(DEV)
    w = _normal(3, len(sizes), n, k, std=k**-0.5, dtype=dtype)
    x, dy = _normal(1, t, k, dtype=dtype), _normal(2, t, n, dtype=dtype)
    x[t - 5:] = float("nan")
    dy[t - 5:] = float("nan")
    y, dx, dw = K.grouped_matmul(x, w, ends), K.grouped_matmul_input_grad(dy, w, ends), \
        K.grouped_matmul_weight_grad(dy, x, ends)
    for e, b, end in _spans(sizes):
        if end > b:
            _check(y[b:end], x[b:end], w[e].t())
            _check(dx[b:end], dy[b:end], w[e])
            _check(dw[e], dy[b:end].t(), x[b:end])
        else:
            assert not dw[e].any()
    assert not y[t - 5:].any() and not dx[t - 5:].any()


def test_weights_past_32_bits():
    """A stack of experts whose bytes and elements pass 2^31 and 2^32: offsets of the last experts hold 64 bits."""
    n, k, groups = 16384, 16384, 34  # 4.5e9 bytes of codes, 9.1e9 elements
    q = torch.zeros(groups, n, k // 2, dtype=torch.uint8, device=DEV)
    s = torch.full((groups, n, k // 32), 127, dtype=torch.uint8, device=DEV)
    for e in (0, groups - 1):
        q[e].random_(0, 256, generator=torch.Generator(DEV).manual_seed(e))
    for rows in (3, 300):
        x = _normal(rows, 2 * rows, k, std=0.1)
        ends = torch.tensor([rows] * (groups - 1) + [2 * rows], dtype=torch.int32, device=DEV)
        y = K.grouped_mx_matmul(x, q, s, ends)
        dy = _normal(rows + 1, 2 * rows, n, std=0.1)
        dx = K.grouped_mx_matmul_input_grad(dy, q, s, ends)
        for e, b in ((0, 0), (groups - 1, rows)):
            at = slice(b, b + 3)  # some rows and columns: a whole 64-bit product of this size is not needed
            w = torch.cat([_decode(q[e, i:i + 64], s[e, i:i + 64], False) for i in (0, n - 64)])
            cols = torch.cat([torch.arange(64), torch.arange(n - 64, n)]).to(DEV)
            _check(y[at][:, cols], x[at], w.t())
            ks = torch.cat([torch.arange(64), torch.arange(k - 64, k)]).to(DEV)
            wk = torch.cat([_decode(q[e, :, i // 2:i // 2 + 32], s[e, :, i // 32:i // 32 + 2], False) for i in (0, k - 64)], 1)
            _check(dx[at][:, ks], dy[at], wk)
