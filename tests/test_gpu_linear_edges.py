"""Products with MXFP4 weights and grouped products where a tile, a group or the stored scales end, against sums in 64 bits.

Tolerance of one output: half a unit in the last place of its type (up to 2^-8 of it in bfloat16, 2^-11 in float16) and, for
an fp32 sum of n products in any order, at most n + 2 roundings of 2^-23 of the sum of magnitudes.
"""

from __future__ import annotations

import ctypes

import pytest
import torch

from piper_offload_amd import _lib as L

pytestmark = pytest.mark.gpu

K = pytest.importorskip("piper_offload_amd.kernels")

DEV = "cuda"
FP4 = getattr(torch, "float4_e2m1fn_x2", None)
BF16, F16 = torch.bfloat16, torch.float16


def _normal(seed, *shape, std=1.0, dtype=BF16):
    return (torch.randn(*shape, generator=torch.Generator(DEV).manual_seed(seed), device=DEV) * std).to(dtype)


def _scale_places(n, blocks):
    """Byte of (row, block) in swizzled scales."""
    r, c = torch.arange(n, device=DEV)[:, None], torch.arange(blocks, device=DEV)[None]
    return ((r // 128) * (-(-blocks // 4)) + c // 4) * 512 + (r % 32) * 16 + (r % 128) // 32 * 4 + c % 4


def _decode(q, s, swizzled=False):
    n, blocks = q.shape[0], q.shape[1] // 16
    s = s.reshape(-1)[_scale_places(n, blocks)] if swizzled else s
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64, device=DEV)
    v = grid[torch.stack((q & 15, q >> 4), -1).reshape(n, -1).int()]
    return v * torch.pow(2.0, s.double() - 127).repeat_interleave(32, 1)


def _weight(seed, n, k, swizzled=False):
    q, s = K.requantize_mx(_normal(seed, n, k, std=0.02), FP4, swizzled=swizzled)
    return q, s, _decode(q, s, swizzled)


def _quantised(x):
    """x on the MXFP4 grid: scale 2^(floor(log2 max) - 2), nearest (ties to even), up to 6."""
    b = x.double().reshape(x.shape[0], -1, 32)
    scale = torch.pow(2.0, (torch.frexp(b.abs().amax(-1, keepdim=True))[1] - 3).double())
    v = b / scale
    step = torch.where(v.abs() < 2, 0.5, torch.where(v.abs() < 4, 1.0, 2.0)).double()
    return (torch.sign(v) * (torch.round(v.abs() / step) * step).clamp(max=6) * scale).reshape(x.shape)


def _check(got, a, b, bias=None):
    """got against a @ b + bias in 64 bits."""
    a, b = a.double().contiguous(), b.double().contiguous()
    want, size = a @ b, a.abs() @ b.abs()
    if bias is not None:
        want, size = want + bias.double(), size + bias.double().abs()
    half, tiny = (2.0**-8, 1e-38) if got.dtype is BF16 else (2.0**-11, 2.0**-25)
    tol = (1 + 2.0**-8) * half * want.abs() + (a.shape[1] + 2) * 2.0**-23 * size + tiny
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    assert (off <= tol).all(), f"{int((off > tol).sum())} of {off.numel()} off, worst {(off / tol).max():.3g} tolerances"


def _spans(sizes):
    end = 0
    for e, size in enumerate(sizes):
        yield e, end, end + size
        end += size


# rows of the groups, rows after the last of them, N, K; whether the sums are split over workgroups.  The last row of a group
# times an odd N ends inside the four sums that a thread adds up.
BIASED = [([9], 11, 64, 512, False), ([100], 29, 1000, 128, False), ([2000, 0, 7], 60, 2001, 544, False),
          ([200], 100, 1024, 8192, True), ([199, 0, 33], 68, 1021, 8224, True), ([0], 300, 1021, 8192, True)]


@pytest.mark.parametrize("case", BIASED, ids=[f"{'-'.join(map(str, s))}+{r}:{n}x{k}" for s, r, n, k, _ in BIASED])
@pytest.mark.parametrize("kind", ["mxfp4", "fp4-inputs", "dense"])
def test_bias_leaves_rows_of_no_group_zero(case, kind):
    sizes, rest, n, k, split = case
    t, groups = sum(sizes) + rest, len(sizes)
    x, bias, ends = _normal(1, t, k), _normal(2, n), torch.tensor(sizes).cumsum(0).to(torch.int32).to(DEV)
    if kind == "dense":
        w = _normal(3, groups, n, k, std=k**-0.5)
        scale, stored = None, list(w.double())
    else:
        made = [_weight(e, n, k) for e in range(groups)]
        w, scale, stored = torch.stack([m[0] for m in made]), torch.stack([m[1] for m in made]), [m[2] for m in made]
    weight = L.WeightStruct(w.data_ptr(), None if scale is None else scale.data_ptr(), n, k,
                            L.LM_BF16 if kind == "dense" else L.LM_E2M1, 0, groups, 0)
    input_id = L.LM_E2M1 if kind == "fp4-inputs" else L.LM_BF16
    need = L.lib().lm_linear_workspace_size(0, t, k, 0, n, k, groups, weight.dtype, input_id, 1)
    if kind == "mxfp4":
        assert (need > 0) == split
    space, y = L.workspace(need, x.device), torch.full((t, n), float("nan"), dtype=BF16, device=DEV)
    L.check(L.lib().lm_linear(x.data_ptr(), k, ctypes.byref(weight), bias.data_ptr(), ends.data_ptr(), y.data_ptr(), t,
                              L.LM_BF16, input_id, L.aligned_ptr(space), need, torch.cuda.current_stream().cuda_stream))
    for e, b, end in _spans(sizes):
        if end > b:
            _check(y[b:end], _quantised(x[b:end]) if kind == "fp4-inputs" else x[b:end], stored[e].t(), bias)
    assert not y[t - rest:].any()


def _pad(s, n, blocks, value):
    """Swizzled scales with `value` in every byte that belongs to no row or no block."""
    out = torch.full_like(s, value)
    at = _scale_places(n, blocks).reshape(-1)
    out.view(-1)[at] = s.reshape(-1)[at]
    return out


# one tile and many, sums split in three from 1030 rows on; N that ends inside a run of 32 rows, K with and without whole words of scales
PADDED = [(3, 1, 64), (40, 33, 96), (20, 100, 4128), (70, 100, 160), (150, 1100, 4128), (300, 257, 416), (300, 130, 32),
          (1030, 2050, 1056), (2050, 2325, 544)]


@pytest.mark.parametrize("shape", PADDED, ids=str)
@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("groups", [1, 3])
def test_padding_of_swizzled_scales_is_not_read(shape, dtype, groups):
    """The padding may hold anything, the code of NaN too: the results are those with zeros there, bit for bit."""
    t, n, k = shape
    made = [_weight(e, n, k, True) for e in range(groups)]
    q = torch.stack([m[0] for m in made])
    zeros, nans = (torch.stack([_pad(m[1], n, k // 32, v) for m in made]) for v in (0, 255))
    x, dy = _normal(1, t, k, dtype=dtype), _normal(2, t, n, dtype=dtype)
    ends = torch.tensor([t // 3, t // 3, t][-groups:], dtype=torch.int32, device=DEV)
    for quant in (None, FP4):
        if groups == 1:
            y = [K.mx_matmul(x, q[0], s[0], swizzled=True, activation_dtype=quant) for s in (zeros, nans)]
        else:
            y = [K.grouped_mx_matmul(x, q, s, ends, swizzled=True, activation_dtype=quant) for s in (zeros, nans)]
        assert torch.equal(y[0], y[1])
    if groups == 1:
        dx = [K.mx_matmul_input_grad(dy, q[0], s[0], swizzled=True) for s in (zeros, nans)]
    else:
        dx = [K.grouped_mx_matmul_input_grad(dy, q, s, ends, swizzled=True) for s in (zeros, nans)]
    assert torch.equal(dx[0], dx[1])
    b = 0
    for e, end in enumerate(ends.tolist()):
        if end > b:
            _check(dx[1][b:end], dy[b:end], made[e][2])
        b = end


@pytest.mark.parametrize("k", [32, 64, 96])
@pytest.mark.parametrize("n", [1, 2, 3, 129, 130, 131, 257])
@pytest.mark.parametrize("t", [65, 100, 300])
@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
def test_last_columns_with_fewer_than_four_scales(t, n, k, dtype):
    """The last column tile has 1 to 9 bytes of scales, not always a whole word: of one weight, and of each in a stack."""
    made = [_weight(10 * e + k, n, k) for e in range(3)]
    x = _normal(t, t, k, dtype=dtype)
    _check(K.mx_matmul(x, made[0][0], made[0][1]), x, made[0][2].t())
    ends = torch.tensor([t // 2, t - 20, t], dtype=torch.int32, device=DEV)
    y = K.grouped_mx_matmul(x, torch.stack([m[0] for m in made]), torch.stack([m[1] for m in made]), ends)
    b = 0
    for e, end in enumerate(ends.tolist()):
        _check(y[b:end], x[b:end], made[e][2].t())
        b = end


def test_raw_products_refuse_to_lose_a_gradient():
    """The raw operators return no graph: with gradients on they refuse what requires one, and run under no_grad."""
    q, s, _ = _weight(1, 64, 128)
    x, dy, bias = _normal(2, 4, 128), _normal(3, 4, 64), _normal(4, 64)
    w, ends = _normal(5, 2, 64, 128), torch.tensor([1, 3], dtype=torch.int32, device=DEV)
    stack = q.view(2, 32, 64), s.view(2, 32, 4)
    calls = [(lambda x: K.mx_matmul(x, q, s), x), (lambda b: K.mx_matmul(x, q, s, bias=b), bias),
             (lambda dy: K.mx_matmul_input_grad(dy, q, s), dy), (lambda x: K.grouped_matmul(x, w, ends), x),
             (lambda w: K.grouped_matmul(x, w, ends), w), (lambda dy: K.grouped_matmul_input_grad(dy, w, ends), dy),
             (lambda w: K.grouped_matmul_input_grad(dy, w, ends), w),
             (lambda dy: K.grouped_matmul_weight_grad(dy, x, ends), dy),
             (lambda x: K.grouped_matmul_weight_grad(dy, x, ends), x),
             (lambda x: K.grouped_mx_matmul(x, *stack, ends), x),
             (lambda dy: K.grouped_mx_matmul_input_grad(dy, *stack, ends), dy[:, :32].contiguous())]
    for i, (call, tensor) in enumerate(calls):
        want = call(tensor)
        leaf = tensor.clone().requires_grad_()
        with pytest.raises(NotImplementedError):
            call(leaf)
            pytest.fail(f"call {i} was taken")
        with torch.no_grad():
            assert torch.equal(call(leaf), want)


# tiles of 64, 128 and 256 rows, whole rounds of tiles with a rest, split sums; N a multiple of 8 and not
MANY = [(100, 1000, 128), (128, 256, 256), (777, 2001, 2080), (150, 2064, 4128), (300, 1021, 8192), (1030, 2064, 1056),
        (2050, 2325, 544), (4100, 4352, 1056), (4100, 4353, 1056)]


@pytest.mark.parametrize("shape", MANY, ids=str)
@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("quant", [False, True], ids=["wide", "fp4"])
def test_bias_of_many_rows(shape, dtype, quant):
    """Every column its own bias, of the size of the sums."""
    t, n, k = shape
    q, s, w = _weight(n, n, k)
    x, bias = _normal(t, t, k, dtype=dtype), _normal(n + 1, n, dtype=dtype)
    act = FP4 if quant else None
    a = _quantised(x) if quant else x
    _check(K.mx_matmul(x, q, s, bias=bias, activation_dtype=act), a, w.t(), bias)
    _check(K.mx_matmul(x, q, s, activation_dtype=act), a, w.t())


def _whole(seed, *shape, blocks):
    """Whole numbers of the 4-bit grid up to 4; the first of every block of 32 is 4 (blocks: its scale is 2^0)."""
    g = torch.Generator(DEV).manual_seed(seed)
    v = torch.randint(-4, 5, shape, generator=g, device=DEV).double()
    if blocks:
        v[..., ::32] = 4
    return v


def _whole_weight(seed, n, k):
    w = _whole(seed, n, k, blocks=True)
    q, s = K.requantize_mx(w.to(BF16), FP4)
    assert torch.equal(_decode(q, s), w)
    return q, s, w


def _same(got, want):
    """want is exact, and so is a sum of whole numbers in fp32: one rounding is left, and one right value."""
    assert want.abs().max() < 2**24 and (got.dtype is BF16 or want.abs().max() < 65504)
    assert torch.equal(got, want.to(got.dtype))


@pytest.mark.parametrize("shape", MANY, ids=str)
@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
def test_whole_numbers_of_many_rows_are_exact(shape, dtype):
    t, n, k = shape
    q, s, w = _whole_weight(n, n, k)
    x, dy = _whole(t, t, k, blocks=True), _whole(k, t, n, blocks=False)
    xd, wt = x.to(dtype), w.t().contiguous()
    _same(K.mx_matmul(xd, q, s), x @ wt)
    _same(K.mx_matmul(xd, q, s, activation_dtype=FP4), x @ wt)
    _same(K.mx_matmul_input_grad(dy.to(dtype), q, s), dy @ w)


@pytest.mark.parametrize("case", [([1500, 0, 1, 2000, 700], 4112, 1568), ([255, 257, 0, 512, 1], 1040, 2080),
                                  ([130, 0, 900], 2061, 544)], ids=lambda c: f"{'-'.join(map(str, c[0]))}:{c[1]}x{c[2]}")
def test_whole_numbers_of_groups_are_exact(case):
    sizes, n, k = case
    t, ends = sum(sizes) + 3, torch.tensor(sizes).cumsum(0).to(torch.int32).to(DEV)
    made = [_whole_weight(e, n, k) for e in range(len(sizes))]
    q, s, w = (torch.stack(m) for m in zip(*made))
    x, dy = _whole(1, t, k, blocks=True), _whole(2, t, n, blocks=False)
    xd, dyd, wd = x.to(BF16), dy.to(BF16), w.to(BF16)
    y, dx, dw = x.new_zeros(t, n), x.new_zeros(t, k), torch.zeros_like(w)
    for e, b, end in _spans(sizes):
        y[b:end], dx[b:end], dw[e] = x[b:end] @ w[e].t().contiguous(), dy[b:end] @ w[e], dy[b:end].t().contiguous() @ x[b:end]
    _same(K.grouped_mx_matmul(xd, q, s, ends), y)
    _same(K.grouped_mx_matmul(xd, q, s, ends, activation_dtype=FP4), y)
    _same(K.grouped_mx_matmul_input_grad(dyd, q, s, ends), dx)
    _same(K.grouped_matmul(xd, wd, ends), y)
    _same(K.grouped_matmul_input_grad(dyd, wd, ends), dx)
    _same(K.grouped_matmul_weight_grad(dyd, xd, ends), dw)
