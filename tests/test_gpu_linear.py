"""Products with MXFP4 weights and grouped products against plain sums in 64 bits.

Tolerance of one output: half a unit in the last place of its type (up to 2^-8 of it in bfloat16, which has 8 significant
bits, and 2^-11 in float16, with half of float16's subnormal spacing, 2^-25), and for the fp32 sum of n products at most n + 2 roundings of 2^-23 of the sum of magnitudes (2^-24 each
if they round to nearest, twice that if the matrix unit truncates).  Both sides see the same stored values.
"""

from __future__ import annotations

import pytest
import torch

from piper_offload_amd import MXWeight, expert_view, grouped_linear, mx_linear

pytestmark = pytest.mark.gpu

K = pytest.importorskip("piper_offload_amd.kernels")

DEV = "cuda"
FP4 = getattr(torch, "float4_e2m1fn_x2", None)
BF16, F16 = torch.bfloat16, torch.float16
E2M1 = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64)


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _normal(g, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=g) * std).to(dtype)


def _plain_scale(s, n, blocks):
    """Swizzled scale bytes of one weight back in rows."""
    r, c = torch.arange(n)[:, None], torch.arange(blocks)[None]
    at = ((r // 128) * (-(-blocks // 4)) + c // 4) * 512 + (r % 32) * 16 + (r % 128) // 32 * 4 + c % 4
    return s.reshape(-1)[at]


def _decode(q, s, swizzled=False):
    """64-bit values of MXFP4 storage [n, k/2]."""
    n, k = q.shape[0], q.shape[1] * 2
    code = torch.stack((q & 15, q >> 4), -1).reshape(n, k).long()
    s = _plain_scale(s, n, k // 32) if swizzled else s
    return E2M1[code] * torch.pow(2.0, s.double() - 127).repeat_interleave(32, 1)


def _weight(g, n, k, swizzled=False, std=0.02):
    w = _normal(g, n, k, std=std, dtype=BF16)
    q, s = K.requantize_mx(w.to(DEV), FP4, swizzled=swizzled)
    return q, s, _decode(q.cpu(), s.cpu(), swizzled)


def _quantised(x):
    """x on the MXFP4 grid, in 64 bits: scale 2^(floor(log2 max) - 2), nearest (ties to even), up to 6."""
    b = x.double().reshape(x.shape[0], -1, 32)
    scale = torch.pow(2.0, (torch.frexp(b.abs().amax(-1, keepdim=True))[1] - 3).double())
    v = b / scale
    step = torch.where(v.abs() < 2, 0.5, torch.where(v.abs() < 4, 1.0, 2.0)).double()
    return (torch.sign(v) * (torch.round(v.abs() / step) * step).clamp(max=6) * scale).reshape(x.shape)


def _check(got, a, b, bias=None):
    """got (GPU) against a @ b (64 bits, CPU)."""
    a, b = a.double().cpu(), b.double().cpu()
    want, size = a @ b, a.abs() @ b.abs()
    if bias is not None:
        want, size = want + bias.double().cpu(), size + bias.double().cpu().abs()
    half, tiny = (2.0**-8, 1e-38) if got.dtype is BF16 else (2.0**-11, 2.0**-25)
    tol = (1 + 2.0**-8) * half * want.abs() + (a.shape[1] + 2) * 2.0**-23 * size + tiny
    off = (got.double().cpu() - want).abs()
    assert torch.isfinite(got).all()
    assert (off <= tol).all(), f"{int((off > tol).sum())} of {off.numel()} off, worst {(off / tol).max():.3g} tolerances"


MX_SHAPES = [(1, 16, 32), (1, 1, 64), (1, 257, 4096), (2, 100, 96), (3, 64, 128), (5, 1, 32), (7, 130, 288), (15, 48, 512),
             (16, 128, 1024), (17, 33, 160), (31, 256, 384), (33, 300, 544), (63, 129, 2080), (64, 512, 256), (65, 96, 768),
             (100, 1000, 128), (128, 256, 256), (129, 257, 640), (255, 255, 1056), (300, 520, 2048), (513, 2001, 416)]


@pytest.mark.parametrize("shape", MX_SHAPES, ids=str)
@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("swizzled", [False, True], ids=["plain", "swizzled"])
@pytest.mark.parametrize("quant", [False, True], ids=["wide", "fp4"])
def test_mx_matmul(shape, dtype, swizzled, quant):
    t, n, k = shape
    g = _gen(t * 1000 + n + k)
    q, s, w = _weight(g, n, k, swizzled)
    x = _normal(g, t, k, dtype=dtype)
    bias = _normal(g, n, dtype=dtype) if (t + n) % 2 else None
    y = K.mx_matmul(x.to(DEV), q, s, swizzled=swizzled, bias=None if bias is None else bias.to(DEV),
                    activation_dtype=FP4 if quant else None)
    assert y.dtype is dtype and y.shape == (t, n)
    _check(y, _quantised(x) if quant else x, w.t(), bias)


@pytest.mark.parametrize("shape", MX_SHAPES, ids=str)
@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("swizzled", [False, True], ids=["plain", "swizzled"])
def test_mx_input_grad(shape, dtype, swizzled):
    t, n, k = shape
    g = _gen(t + n * 1000 + k)
    q, s, w = _weight(g, n, k, swizzled)
    dy = _normal(g, t, n, dtype=dtype)
    dx = K.mx_matmul_input_grad(dy.to(DEV), q, s, swizzled=swizzled)
    assert dx.dtype is dtype and dx.shape == (t, k)
    _check(dx, dy, w)


# sizes of the groups, and rows after the last of them
GROUPS = [([1], 0), ([0], 3), ([5], 0), ([0, 1, 0, 2, 0], 0), ([16, 16], 0), ([3, 0, 17, 130, 1], 7), ([0, 0, 64, 65], 0),
          ([200, 0, 300], 5), ([1] * 40, 2), ([0] * 30 + [257, 3], 0), ([2, 1, 3] * 7, 0), ([129, 128, 127, 1], 0)]
GIDS = ["-".join(map(str, g[:5])) + f"+{r}" for g, r in GROUPS]


def _spans(sizes):
    end = 0
    for e, size in enumerate(sizes):
        yield e, end, end + size
        end += size


def _ends(sizes):
    return torch.tensor(sizes).cumsum(0).to(torch.int32).to(DEV)


@pytest.mark.parametrize("groups", GROUPS, ids=GIDS)
@pytest.mark.parametrize("nk", [(40, 96), (256, 512), (129, 288)], ids=str)
@pytest.mark.parametrize("mode", ["wide", "fp4", "grad"])
@pytest.mark.parametrize("dtype,swizzled", [(BF16, False), (BF16, True), (F16, False)], ids=["bf16", "bf16-swizzled", "f16"])
def test_grouped_mx(groups, nk, mode, dtype, swizzled):
    (sizes, rest), (n, k) = groups, nk
    g = _gen(len(sizes) + n)
    stored = [_weight(g, n, k, swizzled) for _ in sizes]
    q, s = torch.stack([w[0] for w in stored]), torch.stack([w[1] for w in stored])
    t = sum(sizes) + rest
    x = _normal(g, t, n if mode == "grad" else k, dtype=dtype)
    if mode == "grad":
        got = K.grouped_mx_matmul_input_grad(x.to(DEV), q, s, _ends(sizes), swizzled=swizzled)
    else:
        got = K.grouped_mx_matmul(x.to(DEV), q, s, _ends(sizes), swizzled=swizzled,
                                  activation_dtype=FP4 if mode == "fp4" else None)
    assert got.shape == (t, k if mode == "grad" else n)
    for e, b, end in _spans(sizes):
        if end > b:
            rows = _quantised(x[b:end]) if mode == "fp4" else x[b:end]
            _check(got[b:end], rows, stored[e][2] if mode == "grad" else stored[e][2].t())
    assert not got[t - rest:].any()


@pytest.mark.parametrize("groups", GROUPS, ids=GIDS)
@pytest.mark.parametrize("nk", [(16, 256), (256, 16), (40, 33), (1, 7), (136, 264), (300, 1)], ids=str)
@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
def test_grouped_dense(groups, nk, dtype):
    (sizes, rest), (n, k) = groups, nk
    g = _gen(len(sizes) * 7 + n)
    w = _normal(g, len(sizes), n, k, std=k**-0.5, dtype=dtype)
    t = sum(sizes) + rest
    x, dy = _normal(g, t, k, dtype=dtype), _normal(g, t, n, dtype=dtype)
    xd, dyd, wd, ends = x.to(DEV), dy.to(DEV), w.to(DEV), _ends(sizes)
    y, dx, dw = K.grouped_matmul(xd, wd, ends), K.grouped_matmul_input_grad(dyd, wd, ends), \
        K.grouped_matmul_weight_grad(dyd, xd, ends)
    assert dw.shape == w.shape and dw.dtype is dtype
    for e, b, end in _spans(sizes):
        if end > b:
            _check(y[b:end], x[b:end], w[e].t())
            _check(dx[b:end], dy[b:end], w[e])
            _check(dw[e], dy[b:end].t(), x[b:end])
        else:
            assert not dw[e].any()
    assert not y[t - rest:].any() and not dx[t - rest:].any()


@pytest.mark.parametrize("shape", [(1, 64, 128), (40, 96, 160), (200, 384, 512), (513, 256, 1024)], ids=str)
@pytest.mark.parametrize("quant", [False, True], ids=["wide", "fp4"])
def test_whole_numbers_are_exact(shape, quant):
    """Small whole numbers: every product and sum is exact, so every place of every layout has one right value."""
    t, n, k = shape
    g = _gen(t)
    grid = torch.tensor([0.0, 1, 2, 3, 4, 6, -1, -2, -3, -4, -6])
    x = grid[torch.randint(11, (t, k), generator=g)].to(BF16)
    x[:, ::32] = 4  # the block's scale is 2^0
    x[x.abs() == 6] = 4
    w = grid[torch.randint(11, (n, k), generator=g)]
    w[:, ::32] = 6
    w[torch.rand(n, k, generator=g) < 0.9] = 0  # sums below 256
    w[:, ::32] = 6 * (torch.rand(n, k // 32, generator=g) < 0.1)
    q, s = K.requantize_mx(w.to(BF16).to(DEV), FP4)
    w = _decode(q.cpu(), s.cpu())
    got = K.mx_matmul(x.to(DEV), q, s, activation_dtype=FP4 if quant else None)
    assert torch.equal(got.cpu(), (x.double() @ w.t()).to(BF16))
    dy = grid[torch.randint(11, (t, n), generator=g)].to(BF16)
    dx = K.mx_matmul_input_grad(dy.to(DEV), q, s)
    assert torch.equal(dx.cpu(), (dy.double() @ w).to(BF16))


@pytest.mark.parametrize("t", [1, 20, 300])
def test_quantised_input_is_the_weights_encode(t):
    """The input's quantisation equals requantize_mx: the product of the decoded codes is the same, bit for bit."""
    g = _gen(t)
    k = 512
    x = _normal(g, t, k, dtype=BF16) * torch.exp(3 * _normal(g, t, 1)).to(BF16)
    x[0, 32:64] = 0
    x[0, 64:96] *= 2.0**-60
    q, s, w = _weight(g, 96, k)
    xq, xs = K.requantize_mx(x.to(DEV), FP4)
    _check(K.mx_matmul(x.to(DEV), q, s, activation_dtype=FP4), _decode(xq.cpu(), xs.cpu()), w.t())


@pytest.mark.parametrize("t", [3, 40, 260])
@pytest.mark.parametrize("quant", [False, True], ids=["wide", "fp4"])
def test_scales_at_the_ends_of_their_range(t, quant):
    """e8m0 codes 0 and 254 decode to 2^-127 and 2^127; 255 is NaN and reaches the outputs of its row alone."""
    n, k = 70, 256
    g = _gen(5)
    q, s, _ = _weight(g, n, k)
    x = _normal(g, t, k, dtype=BF16)
    s = s.clone()
    s[3] = 0
    s[5, 2] = 0
    x32 = x.float()
    small = K.mx_matmul(x.to(DEV), q, s, activation_dtype=FP4 if quant else None)
    w = _decode(q.cpu(), s.cpu())
    got = small.double().cpu()
    want = (_quantised(x) if quant else x32.double()) @ w.t()
    keep = [i for i in range(n) if i != 3]
    _check(small[:, keep], _quantised(x) if quant else x, w[keep].t())
    assert (got[:, 3] - want[:, 3]).abs().max() <= 2.0**-126  # subnormal or flushed
    s[7, 1] = 255
    nan = K.mx_matmul(x.to(DEV), q, s, activation_dtype=FP4 if quant else None)
    assert nan[:, 7].isnan().all() and torch.equal(nan[:, keep[:6]], small[:, keep[:6]])
    dy = torch.zeros(t, n, dtype=BF16)
    dy[1] = 1
    dx = K.mx_matmul_input_grad(dy.to(DEV), q, s)
    assert dx[:, 32:64].isnan().all() and dx[:, :32].isfinite().all()


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")], ids=str)
@pytest.mark.parametrize("t", [4, 70])
def test_non_finite_inputs_reach_their_row_alone(bad, t):
    g = _gen(6)
    q, s, w = _weight(g, 64, 160)
    x = _normal(g, t, 160, dtype=BF16)
    x[2, 133] = bad
    rest = [i for i in range(t) if i != 2]
    for quant in (False, True):
        y = K.mx_matmul(x.to(DEV), q, s, activation_dtype=FP4 if quant else None)
        assert not y[2].isfinite().any() if quant else not y[2, w[:, 133].to(DEV) != 0].isfinite().any()
        _check(y[rest], _quantised(x[rest]) if quant else x[rest], w.t())
    # and rows of other groups, or of none, do not see them
    wd = _normal(g, 2, 24, 160, dtype=BF16)
    ends = torch.tensor([1, 3], dtype=torch.int32, device=DEV)
    y = K.grouped_matmul(x.to(DEV), wd.to(DEV), ends)
    _check(y[:1], x[:1], wd[0].t())
    assert not y[3:].any()
    dw = K.grouped_matmul_weight_grad(torch.ones(t, 8, dtype=BF16, device=DEV), x.to(DEV), ends)
    _check(dw[0], torch.ones(8, 1), x[:1])
    assert not dw[1, :, 133].isfinite().any()
    x[2, 133] = 0
    x[3:] = bad
    dw = K.grouped_matmul_weight_grad(torch.ones(t, 8, dtype=BF16, device=DEV), x.to(DEV), ends)
    _check(dw[1], torch.ones(8, 2), x[1:3])


def test_strides_and_offsets():
    """Rows with a stride, rows that start off 16 bytes, expanded rows, a transposed view, leading dimensions."""
    g = _gen(7)
    t, n, k = 37, 96, 256
    q, s, w = _weight(g, n, k)
    for quant in (None, FP4):
        def ref(v):
            return _quantised(v) if quant else v

        wide = _normal(g, t, k + 24, dtype=BF16).to(DEV)
        for begin in (0, 3, 8):
            x = wide[:, begin:begin + k]
            _check(K.mx_matmul(x, q, s, activation_dtype=quant), ref(x.cpu()), w.t())
        x = _normal(g, k, t, dtype=BF16).to(DEV).t()
        _check(K.mx_matmul(x, q, s, activation_dtype=quant), ref(x.cpu()), w.t())
        x = _normal(g, 1, k, dtype=BF16).to(DEV).expand(t, k)
        _check(K.mx_matmul(x, q, s, activation_dtype=quant), ref(x.cpu()), w.t())
        x = _normal(g, 3, 5, k, dtype=BF16).to(DEV)
        y = K.mx_matmul(x, q, s, activation_dtype=quant)
        assert y.shape == (3, 5, n)
        _check(y.reshape(15, n), ref(x.cpu().reshape(15, k)), w.t())
    dy = _normal(g, t, n + 7, dtype=BF16).to(DEV)[:, 5:5 + n]
    _check(K.mx_matmul_input_grad(dy, q, s), dy, w)
    ends = _ends([10, 20])
    x = _normal(g, t, k + 3, dtype=BF16).to(DEV)[:, 1:1 + k]
    dw = K.grouped_matmul_weight_grad(dy, x, ends)
    _check(dw[1], dy[10:30].t(), x[10:30])


def test_no_rows():
    q, s, _ = _weight(_gen(8), 32, 64)
    ends = torch.zeros(1, dtype=torch.int32, device=DEV)
    for quant in (None, FP4):
        assert K.mx_matmul(torch.empty(0, 64, dtype=BF16, device=DEV), q, s, activation_dtype=quant).shape == (0, 32)
    assert K.mx_matmul_input_grad(torch.empty(0, 32, dtype=BF16, device=DEV), q, s).shape == (0, 64)
    x, dy = torch.empty(0, 8, dtype=BF16, device=DEV), torch.empty(0, 4, dtype=BF16, device=DEV)
    dw = K.grouped_matmul_weight_grad(dy, x, ends)
    assert dw.shape == (1, 4, 8) and not dw.any()


@pytest.mark.parametrize("ends", [[5, 3, 40], [-4, 10, 10], [0, 1 << 30, -1], [40, 41, 42], [0, 0, 0]], ids=str)
def test_ends_out_of_order_stay_inside(ends):
    """Ends that fall or pass the rows are clamped: every row belongs to one group or none, and nothing else is touched."""
    g = _gen(9)
    t, n, k = 40, 24, 64
    w = _normal(g, 3, n, k, dtype=BF16)
    x = _normal(g, t, k, dtype=BF16)
    y = K.grouped_matmul(x.to(DEV), w.to(DEV), torch.tensor(ends, dtype=torch.int32, device=DEV))
    begin = 0
    for e, end in enumerate(ends):
        end = max(begin, min(end, t))
        if end > begin:
            _check(y[begin:end], x[begin:end], w[e].t())
        begin = end
    assert not y[begin:].any()


def _mx_weight(g, n, k, swizzled=False):
    q, s, w = _weight(g, n, k, swizzled)
    return MXWeight(q, s, FP4, 32, BF16, swizzled), w


def test_mx_linear_gradient_by_differences():
    """The loss is linear in x, so its gradient is its difference along any direction."""
    g = _gen(10)
    weight, w = _mx_weight(g, 48, 96, True)
    x = _normal(g, 6, 96, dtype=BF16).to(DEV).requires_grad_()
    bias = _normal(g, 48, dtype=BF16).to(DEV)
    dy = _normal(g, 6, 48, dtype=BF16).to(DEV)
    y = mx_linear(x, weight, bias)
    _check(y.detach(), x.detach(), w.t(), bias)
    y.backward(dy)
    _check(x.grad, dy, w)
    for i in range(4):
        d = torch.zeros(6, 96, dtype=torch.float64)
        d[i, 17 * i] = 1.0
        difference = (dy.double().cpu() * ((x.detach().double().cpu() + d) @ w.t() - x.detach().double().cpu() @ w.t())).sum()
        assert abs(float(x.grad[i, 17 * i]) - float(difference)) <= 2.0**-8 * abs(float(difference)) + 1e-4
    # straight through the rounding of a quantised input
    x2 = x.detach().clone().requires_grad_()
    mx_linear(x2, weight, activation_dtype=FP4).backward(dy)
    assert torch.equal(x2.grad, x.grad)


def test_grouped_linear_gradients():
    g = _gen(11)
    sizes = [4, 0, 9]
    ends = _ends(sizes)
    w = _normal(g, 3, 20, 40, dtype=BF16)
    x = _normal(g, 15, 40, dtype=BF16)
    xd, wd = x.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    dy = _normal(g, 15, 20, dtype=BF16)
    grouped_linear(xd, wd, ends).backward(dy.to(DEV))
    for e, b, end in _spans(sizes):
        if end > b:
            _check(xd.grad[b:end], dy[b:end], w[e])
            _check(wd.grad[e], dy[b:end].t(), x[b:end])
    assert not wd.grad[1].any() and not xd.grad[13:].any()
    # a weight shared by a broadcast: its gradient is the sum over the groups
    shared = _normal(g, 20, 40, dtype=BF16).to(DEV).requires_grad_()
    grouped_linear(xd.detach(), shared.expand(3, 20, 40).contiguous(), ends).backward(dy.to(DEV))
    want = dy[:13].double().t() @ x[:13].double()
    assert (shared.grad.double().cpu() - want).abs().max() <= 2.0**-7 * want.abs().max()


@pytest.mark.parametrize("swizzled", [False, True], ids=["plain", "swizzled"])
def test_stacked_experts_are_merged_and_multiplied(swizzled):
    """expert_view shares the stack's storage: a LoRA merged into one expert shows in the products of its rows."""
    from piper_offload_amd import MxAdapter

    g = _gen(12)
    groups, n, k = 3, 128, 256
    stack, w = _mx_weight(g, groups * n, k, swizzled)
    sizes = [5, 8, 6]
    x = _normal(g, 19, k, dtype=BF16)
    before = grouped_linear(x.to(DEV), stack, _ends(sizes))
    for e, b, end in _spans(sizes):
        _check(before[b:end], x[b:end], w[e * n:(e + 1) * n].t())
    view = expert_view(stack, 1, groups)
    MxAdapter.merge_lora_(view, _normal(g, n, 8, std=0.1, dtype=BF16).to(DEV), _normal(g, 8, k, dtype=BF16).to(DEV), 1.0)
    after = grouped_linear(x.to(DEV), stack, _ends(sizes))
    merged = _decode(view.qdata.cpu(), view.scale.cpu(), swizzled)
    _check(after[5:13], x[5:13], merged.t())
    assert torch.equal(after[:5], before[:5]) and torch.equal(after[13:], before[13:])
    assert not torch.equal(after[5:13], before[5:13])


def test_other_streams():
    """Calls follow the current stream, and what they free is theirs."""
    g = _gen(13)
    q, s, w = _weight(g, 256, 512)
    x = _normal(g, 200, 512, dtype=BF16)
    side = torch.cuda.Stream()
    xd = x.to(DEV)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [K.mx_matmul(xd, q, s, activation_dtype=FP4) for _ in range(8)]
    torch.cuda.current_stream().wait_stream(side)
    for y in outs:
        assert torch.equal(y, outs[0])
    _check(outs[0], _quantised(x), w.t())


def test_graph_replays():
    """Captured once, replayed with other rows and other groups: nothing is read on the host."""
    g = _gen(14)
    sizes = [9, 0, 12]
    stored = [_weight(g, 128, 256) for _ in sizes]
    q, s = torch.stack([w[0] for w in stored]), torch.stack([w[1] for w in stored])
    x, ends = torch.zeros(24, 256, dtype=BF16, device=DEV), _ends(sizes)

    def step():
        return (K.grouped_mx_matmul(x, q, s, ends), K.grouped_mx_matmul(x, q, s, ends, activation_dtype=FP4),
                K.grouped_mx_matmul_input_grad(x[:, :128].contiguous(), q, s, ends))

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(4):
        x.copy_(_normal(g, 24, 256, dtype=BF16))
        ends.copy_(_ends([[9, 0, 12], [0, 24, 0], [1, 1, 1], [0, 0, 24]][i]))
        graph.replay()
        replayed = [o.clone() for o in outs]
        for a, b in zip(replayed, step()):
            assert torch.equal(a, b)
        torch.cuda.synchronize()


@pytest.mark.parametrize("case", ["forward", "fp4", "grad", "weight"])
def test_results_do_not_change_between_calls(case):
    """No atomics whose order shows: the same call gives the same bits."""
    g = _gen(15)
    q, s, _ = _weight(g, 272, 4096)
    x = _normal(g, 20, 4096, dtype=BF16).to(DEV)
    dy = _normal(g, 20, 272, dtype=BF16).to(DEV)
    ends = _ends([3, 17])
    run = {"forward": lambda: K.mx_matmul(x, q, s), "fp4": lambda: K.mx_matmul(x, q, s, activation_dtype=FP4),
           "grad": lambda: K.mx_matmul_input_grad(dy, q, s), "weight": lambda: K.grouped_matmul_weight_grad(dy, x, ends)}[case]
    first = run()
    for _ in range(5):
        assert torch.equal(run(), first)


def test_refusals():
    g = _gen(16)
    q, s, _ = _weight(g, 64, 128)
    x = _normal(g, 4, 128, dtype=BF16).to(DEV)
    dy = _normal(g, 4, 64, dtype=BF16).to(DEV)
    w = _normal(g, 2, 64, 128, dtype=BF16).to(DEV)
    ends = _ends([1, 3])
    bad = [
        lambda: K.mx_matmul(x.float(), q, s),
        lambda: K.mx_matmul(x[:, :96], q, s),
        lambda: K.mx_matmul(x, q.t(), s),
        lambda: K.mx_matmul(x, q, s, swizzled=True),
        lambda: K.mx_matmul(x, q.float(), s),
        lambda: K.mx_matmul(x, q, s.float()),
        lambda: K.mx_matmul(x, q[:, :-8].contiguous(), s),
        lambda: K.mx_matmul(x, q, s, activation_dtype=torch.float8_e4m3fn),
        lambda: K.mx_matmul(x, q, s, bias=torch.zeros(64, device=DEV)),
        lambda: K.mx_matmul(x, q, s, bias=torch.zeros(63, dtype=BF16, device=DEV)),
        lambda: K.mx_matmul(x, q.cpu(), s),
        lambda: K.mx_matmul_input_grad(x, q, s),
        lambda: K.grouped_matmul(x, w[0], ends),
        lambda: K.grouped_matmul(x, w.half(), ends),
        lambda: K.grouped_matmul(x, w.transpose(0, 1), ends),
        lambda: K.grouped_matmul(x, w, ends.long()),
        lambda: K.grouped_matmul(x, w, ends[:1]),
        lambda: K.grouped_matmul(x, w, ends.cpu()),
        lambda: K.grouped_matmul_weight_grad(dy[:3], x, ends),
        lambda: K.grouped_matmul_weight_grad(dy.half(), x, ends),
        lambda: K.grouped_mx_matmul(x, q, s, ends),
        lambda: K.grouped_mx_matmul(x, q.view(2, 32, 64), s.view(2, 32, 4), ends[:1]),
        lambda: grouped_linear(x, w, ends, activation_dtype=FP4),
        lambda: grouped_linear(x, MXWeight(q, s, FP4), _ends([1, 1, 1])),
        lambda: mx_linear(x, MXWeight(q, s, FP4), torch.zeros(64, dtype=BF16, device=DEV, requires_grad=True)),
        lambda: mx_linear(x, MXWeight(torch.zeros(64, 128, device=DEV, dtype=torch.float8_e4m3fn), s, torch.float8_e4m3fn)),
        lambda: expert_view(MXWeight(q, s, FP4), 2, 2),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was taken")
