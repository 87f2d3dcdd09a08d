"""Products with INT8 weights against plain sums in 64 bits.

Tolerances of one output: half a unit in the last place of its type (2^-8 of it in bfloat16, 2^-11 in float16 with half of
its subnormal spacing, 2^-25) and

* 8-bit inputs: the sum is exact, so four roundings of 2^-24 of it (to fp32, two scales, the bias);
* 16-bit inputs: n + 4 roundings of 2^-23 of the sum of magnitudes (2^-24 each if they round to nearest, twice that if the
  matrix unit truncates);
* input gradient: besides that each weight's rounding to 16 bits, 2^-8 or 2^-11 of the sum of magnitudes (and float16's
  subnormal spacing, 2^-25 of the sum of |dy|).
"""

from __future__ import annotations

import pytest
import torch

from piper_offload_amd import Int8Adapter, Int8Weight, expert_view, grouped_linear, int8_linear

pytestmark = pytest.mark.gpu

K = pytest.importorskip("piper_offload_amd.kernels")

DEV = "cuda"
BF16, F16, I8 = torch.bfloat16, torch.float16, torch.int8


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _normal(g, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=g) * std).to(dtype)


def _weight(g, *shape, scale_dtype=torch.float32):
    q = torch.randint(-128, 128, shape, generator=g, dtype=torch.int8)
    s = (torch.rand(*shape[:-1], 1, generator=g) * 2e-4 + 1e-5).to(scale_dtype)
    return q, s, q.double() * s.double()


def _codes(x):
    """Codes and scale of every row in 64 bits: the quotients by the fp32 scale, to nearest, ties to even.

    The scale is the largest magnitude times the number of 32 bits next to 1 / 127, as torch divides by 127 on the GPU (on the
    CPU it rounds the quotient)."""
    s = (x.float().abs().amax(-1, keepdim=True) * (torch.ones(()) / 127)).double()
    return torch.round(x.double() / torch.where(s > 0, s, 1.0)).clamp(-127, 127), s


def _half(dtype):
    return (2.0**-8, 1e-38) if dtype is BF16 else (2.0**-11, 2.0**-25)


def _close(got, want, slack):
    half, tiny = _half(got.dtype)
    off, tol = (got.double().cpu() - want).abs(), (1 + 2.0**-8) * half * want.abs() + slack + tiny
    assert torch.isfinite(got).all()
    assert (off <= tol).all(), f"{int((off > tol).sum())} of {off.numel()} off, worst {(off / tol).max():.3g} tolerances"


def _want(x, q, s, quant, bias=None):
    """The product in 64 bits and the slack of its sum."""
    x64, rs = _codes(x) if quant else (x.double(), 1.0)
    y = (x64 @ q.double().t()) * rs * s.double().t()
    size = y.abs() if quant else (x64.abs() @ q.double().abs().t()) * s.double().t()
    if bias is not None:
        y, size = y + bias.double(), size + bias.double().abs()
    return y, (4 * 2.0**-24 if quant else (x.shape[1] + 4) * 2.0**-23) * size


def _check(x, q, s, got, quant, bias=None):
    _close(got, *_want(x, q, s, quant, bias))


def _check_grad(dy, w, got):
    half, tiny = _half(dy.dtype)
    dy = dy.double()
    size = dy.abs() @ w.abs()
    _close(got, dy @ w, ((dy.shape[1] + 4) * 2.0**-23 + half) * size + tiny * dy.abs().sum(-1, keepdim=True))


SHAPES = [(1, 1, 1), (1, 16, 64), (1, 7, 4096), (1, 257, 100), (2, 100, 96), (3, 64, 128), (5, 1, 33), (7, 130, 288), (15, 48, 500),
          (16, 128, 1024), (17, 33, 161), (31, 256, 384), (33, 300, 545), (63, 129, 2083), (64, 512, 256), (65, 96, 768),
          (100, 1000, 130), (128, 256, 256), (129, 257, 641), (255, 255, 1056), (300, 520, 2048), (513, 2001, 415), (600, 640, 72)]


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("quant", [False, True], ids=["x16", "x8"])
@pytest.mark.parametrize("t,n,k", SHAPES)
def test_forward(t, n, k, quant, dtype):
    g = _gen(t * 7 + n + k)
    q, s, _ = _weight(g, n, k)
    x = _normal(g, t, k, dtype=dtype)
    bias = _normal(g, n, std=0.1, dtype=dtype) if (t + n) % 2 else None
    got = K.int8_matmul(x.to(DEV), q.to(DEV), s.to(DEV), bias=None if bias is None else bias.to(DEV),
                        activation_dtype=I8 if quant else None)
    assert got.dtype is dtype and got.shape == (t, n)
    _check(x, q, s, got, quant, bias)


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("t,n,k", SHAPES)
def test_input_grad(t, n, k, dtype):
    g = _gen(t * 5 + n + k)
    q, s, w = _weight(g, n, k)
    dy = _normal(g, t, n, dtype=dtype)
    got = K.int8_matmul_input_grad(dy.to(DEV), q.to(DEV), s.to(DEV))
    assert got.dtype is dtype and got.shape == (t, k)
    _check_grad(dy, w, got)


def _ends(sizes):
    return torch.tensor(sizes).cumsum(0).to(torch.int32)


GROUPS = [([1], 1, 32, 64), ([0, 3, 0, 1], 5, 48, 96), ([5, 0, 0, 16, 1, 17], 39, 130, 161), ([64, 64], 128, 128, 256),
          ([100, 0, 300, 7, 0], 500, 257, 320), ([0, 0, 0], 9, 32, 64), ([1] * 70, 75, 40, 144), ([700, 1, 333], 1034, 264, 520),
          ([2, 0, 1, 3] * 8, 64, 2048, 1408)]


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("quant", [False, True], ids=["x16", "x8"])
@pytest.mark.parametrize("sizes,t,n,k", GROUPS, ids=lambda v: str(v) if isinstance(v, int) else f"g{len(v)}")
def test_grouped(sizes, t, n, k, quant, dtype):
    g = _gen(t + n + k)
    e = len(sizes)
    q, s, w = _weight(g, e, n, k)
    x, dy = _normal(g, t, k, dtype=dtype), _normal(g, t, n, dtype=dtype)
    ends = _ends(sizes)
    args = q.to(DEV), s.to(DEV), ends.to(DEV)
    y = K.grouped_int8_matmul(x.to(DEV), *args, activation_dtype=I8 if quant else None)
    dx = K.grouped_int8_matmul_input_grad(dy.to(DEV), *args)
    begin = 0
    for i, end in enumerate(ends.tolist()):
        if end > begin:
            _check(x[begin:end], q[i], s[i], y[begin:end], quant)
            _check_grad(dy[begin:end], w[i], dx[begin:end])
        begin = end
    assert (y[begin:] == 0).all() and (dx[begin:] == 0).all()


def test_whole_numbers_are_exact():
    """Sums of codes past 2^24, which fp32 sums would round."""
    g = _gen(5)
    for t, n, k in ((3, 40, 8192), (200, 300, 16384), (40, 64, 132104)):
        q = torch.randint(100, 128, (n, k), generator=g, dtype=torch.int8)
        x = torch.randint(100, 128, (t, k), generator=g).to(BF16)
        x[:, 0] = 127
        s = torch.full((n, 1), 2.0**-20)
        got = K.int8_matmul(x.to(DEV), q.to(DEV), s.to(DEV), activation_dtype=I8)
        want = ((x.double() @ q.double().t()).float() * 2.0**-20).to(BF16)
        assert (got.cpu() == want).all()


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
def test_codes_next_to_a_border(dtype):
    """Quotients at and next to halves, read off through a weight of one: y = r * code."""
    g = _gen(9)
    k = 4096
    x = _normal(g, 64, k, dtype=dtype)
    x[::3] *= 64
    for i in range(0, 64, 4):  # the largest makes the scale a power of two: every odd half is a tie
        top = 127 * 2.0 ** (i % 8 - 4)
        x[i] = ((torch.randint(-253, 254, (k,), generator=g) / 2) * 2.0 ** (i % 8 - 4)).to(dtype)
        x[i, 0] = top
    eye = torch.zeros(128, k, dtype=torch.int8)
    for start in range(0, k, 1024):
        eye.zero_()
        eye[torch.arange(128), start + 8 * torch.arange(128)] = 1
        got = K.int8_matmul(x.to(DEV), eye.to(DEV), torch.ones(128, 1, device=DEV), activation_dtype=I8)
        c, r = _codes(x)
        want = (c.float() * r.float()).to(dtype)[:, start:start + 1024:8]
        assert (got.cpu() == want).all()


def test_extreme_rows():
    g = _gen(11)
    n, k = 70, 200
    q, s, _ = _weight(g, n, k)
    x = _normal(g, 9, k, dtype=BF16)
    x[1] = 0
    x[2] = 0
    x[2, 5] = 1e-40  # (subnormal: the scale is one too)
    x[3] *= 1e36
    x[4, 7] = float("inf")
    x[5, 199] = float("nan")
    x[6, 0] = float("-inf")
    x[7] = x[7] * 1e-38
    y = K.int8_matmul(x.to(DEV), q.to(DEV), (s * 100).to(DEV), activation_dtype=I8).cpu()
    assert torch.isnan(y[[4, 5, 6]]).all()
    assert (y[1] == 0).all()
    rows = [0, 2, 3, 7, 8]
    want, slack = _want(x[rows], q, s * 100, True)
    _close(y[rows], want, slack + 2.0**-133)  # (results below bfloat16's normal numbers)


@pytest.mark.parametrize("quant", [False, True], ids=["x16", "x8"])
@pytest.mark.parametrize("t", [1, 5, 40, 300])
def test_strides_and_alignment(t, quant):
    g = _gen(t)
    n, k = 160, 320
    q, s, w = _weight(g, n, k)
    act = I8 if quant else None
    big = _normal(g, t, k + 13, dtype=BF16).to(DEV)
    store = torch.empty(n * k + 64, dtype=torch.int8, device=DEV)
    for off in (0, 1, 3, 8):
        view = store[off:off + n * k].view(n, k).copy_(q.to(DEV))
        for x in (big[:, :k], big[:, 5:k + 5], big[:, 8:k + 8], big[:, :k].t().contiguous().t()):
            _check(x.cpu(), q, s, K.int8_matmul(x, view, s.to(DEV), activation_dtype=act), quant)
        dy = _normal(g, t, n + 3, dtype=BF16).to(DEV)[:, 1:n + 1]
        _check_grad(dy.cpu(), w, K.int8_matmul_input_grad(dy, view, s.to(DEV)))
    x = big[:, :k].reshape(1, t, k).expand(2, t, k)
    y = K.int8_matmul(x, q.to(DEV), s.to(DEV), activation_dtype=act)
    assert y.shape == (2, t, n) and (y[0] == y[1]).all()


def test_scales_in_bfloat16_and_flat():
    g = _gen(3)
    for t in (1, 90):
        q, s, w = _weight(g, 140, 96, scale_dtype=BF16)
        x, dy = _normal(g, t, 96, dtype=BF16), _normal(g, t, 140, dtype=BF16)
        for quant in (False, True):
            a = K.int8_matmul(x.to(DEV), q.to(DEV), s.to(DEV), activation_dtype=I8 if quant else None)
            b = K.int8_matmul(x.to(DEV), q.to(DEV), s.view(-1).to(DEV), activation_dtype=I8 if quant else None)
            assert (a == b).all()
            _check(x, q, s, a, quant)
        _check_grad(dy, w, K.int8_matmul_input_grad(dy.to(DEV), q.to(DEV), s.to(DEV)))


def test_layers_and_gradients():
    g = _gen(21)
    q, s, w = _weight(g, 192, 160)
    weight = Int8Weight(q.to(DEV), s.to(DEV), (1, 160))
    x = _normal(g, 4, 10, 160, dtype=BF16).to(DEV).requires_grad_()
    dy = _normal(g, 4, 10, 192, dtype=BF16)
    for act in (None, I8):
        x.grad = None
        y = int8_linear(x, weight, activation_dtype=act)
        y.backward(dy.to(DEV))
        _check(x.detach().cpu().view(-1, 160), q, s, y.detach().view(-1, 192), act is I8)
        _check_grad(dy.view(-1, 192), w, x.grad.view(-1, 160))
    # experts one below the other
    ends = _ends([13, 0, 20]).to(DEV)
    x = _normal(g, 40, 160, dtype=BF16).to(DEV).requires_grad_()
    y = grouped_linear(x, weight, ends, activation_dtype=I8)
    y.backward(dy[:, :, :64].reshape(40, 64).to(DEV))
    _check(x.detach().cpu()[13:33], q[128:], s[128:], y.detach()[13:33], True)
    _check_grad(dy[:, :, :64].reshape(40, 64)[:13], w[:64], x.grad[:13])
    assert (x.grad[33:] == 0).all() and (y[33:] == 0).all()


def test_gradient_against_differences():
    """<dx, u> against the difference of <y, dy> along u (the product is linear in x)."""
    g = _gen(31)
    q, s, _ = _weight(g, 96, 128)
    x, u, dy = (_normal(g, 20, n, dtype=BF16) for n in (128, 128, 96))
    f = lambda v: (K.int8_matmul(v.to(DEV), q.to(DEV), s.to(DEV)).double().cpu() * dy.double()).sum()  # noqa: E731
    dx = K.int8_matmul_input_grad(dy.to(DEV), q.to(DEV), s.to(DEV)).double().cpu()
    a, b = (x.float() + 0.5 * u.float()).to(BF16), (x.float() - 0.5 * u.float()).to(BF16)
    along = (dx * (a.double() - b.double())).sum()
    # 2^-8 of every product's magnitude from the roundings of y, the weights and dx
    ya, yb = (_want(v, q, s, False)[0].abs() for v in (a, b))
    bound = 2.0**-8 * ((ya + yb) * dy.double().abs()).sum() + 2.0**-7 * ((a.double() - b.double()).abs() * (dy.double().abs() @ (q.double() * s.double()).abs())).sum()
    assert abs(f(a) - f(b) - along) <= bound


def test_merged_weight_is_used_as_stored():
    g = _gen(41)
    n, k = 256, 512
    w = _normal(g, n, k, std=0.02, dtype=BF16).to(DEV)
    q, s, _ = K.requantize_int8(w, (1, k))
    stack = Int8Weight(q, s, (1, k))
    one = expert_view(stack, 1, 2)
    Int8Adapter.merge_lora_(one, _normal(g, 128, 8, dtype=BF16).to(DEV), _normal(g, 8, k, std=0.05, dtype=BF16).to(DEV), 0.7)
    x = _normal(g, 30, k, dtype=BF16)
    for act in (None, I8):
        _check(x, stack.qdata.cpu(), stack.scale.cpu(), int8_linear(x.to(DEV), stack, activation_dtype=act), act is I8)


def test_graph_replays_and_other_streams():
    g = _gen(51)
    q, s, _ = _weight(g, 300, 272)
    q, s = q.to(DEV), s.to(DEV)
    ends = _ends([20, 0, 40]).to(DEV)
    x = _normal(g, 64, 272, dtype=BF16).to(DEV)
    dy = _normal(g, 64, 100, dtype=BF16).to(DEV)

    def work():
        a = K.int8_matmul(x, q, s, activation_dtype=I8)
        b = K.int8_matmul(x, q, s)
        c = K.grouped_int8_matmul(x, q.view(3, 100, 272), s.view(3, 100, 1), ends, activation_dtype=I8)
        return a, b, c, K.grouped_int8_matmul_input_grad(dy, q.view(3, 100, 272), s.view(3, 100, 1), ends)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = work()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, work()):
        assert (a == b).all()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for i in range(4):
        x.copy_(_normal(g, 64, 272, dtype=BF16) * (i + 1))
        ends.copy_(_ends([i, 30, 3 * i]))
        graph.replay()
        want = work()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert (a == b).all()


def test_no_rows():
    q, s, _ = _weight(_gen(1), 32, 64)
    q, s = q.to(DEV), s.to(DEV)
    x = torch.empty(0, 64, dtype=BF16, device=DEV)
    assert K.int8_matmul(x, q, s, activation_dtype=I8).shape == (0, 32)
    assert K.int8_matmul_input_grad(x.new_empty(0, 32), q, s).shape == (0, 64)


def test_refusals():
    g = _gen(2)
    q, s, _ = _weight(g, 32, 64)
    q, s, x = q.to(DEV), s.to(DEV), _normal(g, 4, 64, dtype=BF16).to(DEV)
    bad = [
        (x.float(), q, s, {}), (x[:, :60], q, s, {}), (x, q.float(), s, {}), (x, q[:, ::2], s, {}), (x, q, s.half(), {}),
        (x, q, s[:30], {}), (x, q, s.expand(32, 2), {}), (x, q.view(2, 16, 64), s, {}), (x, q, s, dict(activation_dtype=torch.float16)),
        (x, q, s, dict(activation_dtype=torch.float8_e4m3fn)), (x, q, s, dict(bias=torch.zeros(31, dtype=BF16, device=DEV))),
        (x, q, s, dict(bias=torch.zeros(32, device=DEV))), (x, q.cpu(), s, {}), (x.cpu(), q, s, {}), (x, q[:0], s[:0], {}),
    ]
    for a, b, c, kw in bad:
        with pytest.raises(ValueError):
            K.int8_matmul(a, b, c, **kw)
    wide = torch.zeros(16, 132120, dtype=torch.int8, device=DEV)
    with pytest.raises(ValueError, match="columns"):
        K.int8_matmul(torch.zeros(1, 132120, dtype=BF16, device=DEV), wide, torch.ones(16, 1, device=DEV), activation_dtype=I8)
    assert (K.int8_matmul(torch.zeros(1, 132120, dtype=BF16, device=DEV), wide, torch.ones(16, 1, device=DEV)) == 0).all()
    with pytest.raises(NotImplementedError):
        K.int8_matmul(x.clone().requires_grad_(), q, s)
    ends = torch.tensor([1, 4], dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError):
        K.grouped_int8_matmul(x, q.view(2, 16, 64), s.view(2, 16, 1), ends.long())
    with pytest.raises(ValueError):
        K.grouped_int8_matmul(x, q.view(2, 16, 64), s, ends)
    with pytest.raises(ValueError, match="per row"):
        int8_linear(x, Int8Weight(q, s.expand(32, 2).contiguous(), (1, 32)))
    with pytest.raises(ValueError, match="zero points"):
        int8_linear(x, Int8Weight(q, s, (1, 64), zero_point=torch.zeros(32, 1, dtype=torch.int8, device=DEV)))
    with pytest.raises(ValueError, match="pre-scale"):
        int8_linear(x, Int8Weight(q, s, (1, 64), act_pre_scale=torch.ones(64, device=DEV)))
    with pytest.raises(ValueError, match="frozen"):
        int8_linear(x, Int8Weight(q, s, (1, 64)), torch.zeros(32, dtype=BF16, device=DEV, requires_grad=True))
    with pytest.raises(ValueError):
        grouped_linear(x, Int8Weight(q, s, (1, 64)), torch.zeros(3, dtype=torch.int32, device=DEV))


# up to four rows are quantised by the product's own workgroups while their codes fit; the last but one are too long
OWN = [(1, 300, 4095), (1, 48, 4104), (2, 4200, 130), (3, 130, 4097), (4, 96, 8192), (4, 70, 8208), (1, 50, 32768), (1, 48, 32784),
       (4, 4200, 1056), (5, 4200, 300)]


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("t,n,k", OWN)
def test_few_rows_with_8_bit_inputs(t, n, k, dtype):
    g = _gen(t + 3 * n + k)
    q, s, _ = _weight(g, n, k)
    x = _normal(g, t, k, dtype=dtype)
    x[0, k // 2] = 17.0  # (its largest value in the middle)
    if t > 2:
        x[1] = 0.0
    bias = _normal(g, n, std=0.1, dtype=dtype)
    args = q.to(DEV), s.to(DEV)
    got = K.int8_matmul(x.to(DEV), *args, bias=bias.to(DEV), activation_dtype=I8)
    _check(x, q, s, got, True, bias)
    big = torch.full((t, k + 9), 1e4, dtype=dtype, device=DEV)
    view = big[:, 3:3 + k].copy_(x.to(DEV))
    assert (K.int8_matmul(view, *args, bias=bias.to(DEV), activation_dtype=I8) == got).all()


# 16-bit inputs: every shape of workgroup (few and many columns, up to and above 8 rows, long rows)
@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("t,n,k", [(1, 4097, 200), (8, 4200, 640), (9, 4200, 640), (16, 5000, 129), (40, 4100, 512), (3, 4112, 8200), (20, 4100, 8192)])
def test_few_rows_with_16_bit_inputs(t, n, k, dtype):
    g = _gen(t + n + 5 * k)
    q, s, _ = _weight(g, n, k)
    x = _normal(g, t, k, dtype=dtype)
    _check(x, q, s, K.int8_matmul(x.to(DEV), q.to(DEV), s.to(DEV)), False)


@pytest.mark.parametrize("quant", [False, True], ids=["x16", "x8"])
@pytest.mark.parametrize("sizes,t,n,k", [([0, 1, 0, 2, 1], 4, 200, 1408), ([0, 1, 1], 3, 64, 520), ([1, 0, 0, 0], 4, 4100, 144), ([2, 3] * 20, 100, 2050, 136),
                                         ([40, 50] * 3, 270, 6200, 72)])
def test_few_rows_of_groups(sizes, t, n, k, quant):
    g = _gen(t + n + k)
    q, s, _ = _weight(g, len(sizes), n, k)
    x, ends = _normal(g, t, k, dtype=BF16), _ends(sizes)
    x[int(ends[-1]):] = float("nan")  # (rows of no group are not looked at)
    y = K.grouped_int8_matmul(x.to(DEV), q.to(DEV), s.to(DEV), ends.to(DEV), activation_dtype=I8 if quant else None)
    begin = 0
    for i, end in enumerate(ends.tolist()):
        if end > begin:
            _check(x[begin:end], q[i], s[i], y[begin:end], quant)
        begin = end
    assert (y[begin:] == 0).all()


def test_bad_rows_of_few():
    """An infinity or a NaN makes its own row NaN, also where the rows are quantised by the product's workgroups."""
    g = _gen(19)
    q, s, _ = _weight(g, 500, 4300)
    x = _normal(g, 4, 4300, dtype=BF16)
    x[1, 4299] = float("inf")
    x[3, 7] = float("nan")
    y = K.int8_matmul(x.to(DEV), q.to(DEV), s.to(DEV), activation_dtype=I8)
    assert torch.isnan(y[[1, 3]]).all()
    _check(x[[0, 2]], q, s, y[[0, 2]], True)


def test_few_rows_in_a_graph_on_another_stream():
    g = _gen(52)
    q, s, _ = _weight(g, 700, 1000)
    q, s = q.to(DEV), s.to(DEV)
    x = _normal(g, 3, 1000, dtype=BF16).to(DEV)
    K.int8_matmul(x, q, s, activation_dtype=I8)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = K.int8_matmul(x, q, s, activation_dtype=I8)
    for _ in range(3):
        x.copy_(_normal(g, 3, 1000, dtype=BF16))
        graph.replay()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            want = K.int8_matmul(x, q, s, activation_dtype=I8)
        torch.cuda.current_stream().wait_stream(side)
        assert (y == want).all()


# many rows, weights whose rows start and end anywhere: the last 16 codes of a row in each place of a tile
@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("k", [1, 9, 15, 16, 17, 31, 33, 129, 136, 255, 257, 264, 511, 1041])
def test_rows_of_any_length(k, dtype):
    g = _gen(k)
    for t, n in ((70, 100), (300, 4200), (1100, 520), (30, 33)):
        q, s, w = _weight(g, n, k)
        store = torch.full((n * k + 37,), 127, dtype=I8, device=DEV)
        codes = store[5:5 + n * k].view(n, k).copy_(q.to(DEV))
        x, dy = _normal(g, t, k, dtype=dtype), _normal(g, t, n, dtype=dtype)
        _check(x, q, s, K.int8_matmul(x.to(DEV), codes, s.to(DEV)), False)
        _check(x, q, s, K.int8_matmul(x.to(DEV), codes, s.to(DEV), activation_dtype=I8), True)
        _check_grad(dy, w, K.int8_matmul_input_grad(dy.to(DEV), codes, s.to(DEV)))
    sizes = [5, 0, 130, 1, 64]
    q, s, w = _weight(g, len(sizes), 72, k)
    ends, t = _ends(sizes), 210
    x, dy = _normal(g, t, k, dtype=dtype), _normal(g, t, 72, dtype=dtype)
    args = q.to(DEV), s.to(DEV), ends.to(DEV)
    y, dx = K.grouped_int8_matmul(x.to(DEV), *args), K.grouped_int8_matmul_input_grad(dy.to(DEV), *args)
    begin = 0
    for i, end in enumerate(ends.tolist()):
        if end > begin:
            _check(x[begin:end], q[i], s[i], y[begin:end], False)
            _check_grad(dy[begin:end], w[i], dx[begin:end])
        begin = end
    assert (y[begin:] == 0).all() and (dx[begin:] == 0).all()


def test_the_same_call_gives_the_same_bits():
    """Columns that two tiles have in common, split sums, rows quantised by every workgroup."""
    g = _gen(71)
    for t, n, k in ((300, 260, 1041), (40, 3000, 257), (3, 500, 999), (700, 96, 4099)):
        q, s, _ = _weight(g, n, k)
        q, s = q.to(DEV), s.to(DEV)
        x, dy = _normal(g, t, k, dtype=BF16).to(DEV), _normal(g, t, n, dtype=BF16).to(DEV)
        first = None
        for _ in range(5):
            out = K.int8_matmul(x, q, s), K.int8_matmul(x, q, s, activation_dtype=I8), K.int8_matmul_input_grad(dy, q, s)
            first = first or out
            assert all((a == b).all() for a, b in zip(first, out))


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
def test_codes_are_those_of_a_program_that_quantises_by_itself(dtype):
    """Read off through a weight of one, against torch on the GPU: no code differs, in launches of few and of many rows."""
    g = _gen(83)
    eye = torch.eye(256, dtype=torch.int8, device=DEV)
    one = torch.ones(256, device=DEV)
    for t in (2, 4, 60, 4000):
        x = (_normal(g, t, 256) * torch.exp(_normal(g, t, 1))).to(dtype).to(DEV)
        s = x.float().abs().amax(-1, keepdim=True) / 127
        codes = torch.round(x.double() / s.double()).clamp(-127, 127)
        y = K.int8_matmul(x, eye, one, activation_dtype=I8)
        assert (y == (codes.float() * s).to(dtype)).all()


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("sizes,n,k", [([60, 0, 64, 20, 3, 100, 40, 64], 2050, 1037), ([30] * 40, 700, 1041), ([50, 62] * 6, 1030, 2051),
                                       ([40] * 3 + [70] * 30, 640, 515), ([33] * 64, 256, 272)])
def test_groups_of_rows_of_any_length(sizes, n, k, dtype):
    """8-bit inputs, many groups: weights whose rows are no whole pieces, or start anywhere, are not copied."""
    g = _gen(n + k)
    e, t = len(sizes), sum(sizes) + 7
    q, s, _ = _weight(g, e, n, k)
    store = torch.full((e * n * k + 19,), 111, dtype=I8, device=DEV)
    codes = store[3:3 + e * n * k].view(e, n, k).copy_(q.to(DEV))
    x, ends = _normal(g, t, k, dtype=dtype), _ends(sizes)
    y = K.grouped_int8_matmul(x.to(DEV), codes, s.to(DEV), ends.to(DEV), activation_dtype=I8)
    begin = 0
    for i, end in enumerate(ends.tolist()):
        if end > begin:
            _check(x[begin:end], q[i], s[i], y[begin:end], True)
        begin = end
    assert (y[begin:] == 0).all()


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("scale_dtype", [torch.float32, BF16], ids=["s32", "s16"])
@pytest.mark.parametrize("s0,d0", [(1e-9, 2.0**13), (1e-12, 2.0**14), (1e3, 2.0**-12), (2e4, 2.0**-14), (1.0, 1.0)])
@pytest.mark.parametrize("t,n,k", [(1, 16, 64), (40, 300, 129), (200, 512, 257), (300, 2000, 256)])
def test_input_grad_with_scales_of_any_size(t, n, k, s0, d0, scale_dtype, dtype):
    """Weights below and above float16's own range.

    Their largest scale counts as 128 to 256, and no scale here is less than a quarter of it, so the weights (codes of 1 too)
    are float16's normal numbers and each is off by half a step: 2^-11 of its magnitude.
    """
    g = _gen(t + n + k)
    q = torch.randint(-128, 128, (n, k), generator=g, dtype=torch.int8)
    s = ((0.25 + 0.75 * torch.rand(n, 1, generator=g)) * s0).to(scale_dtype)
    s[n // 2] = s0
    dy = _normal(g, t, n, std=d0).clamp(-3 * d0, 3 * d0).to(dtype)
    got = K.int8_matmul_input_grad(dy.to(DEV), q.to(DEV), s.to(DEV))
    w = q.double() * s.double()
    half, _ = _half(dtype)
    _close(got, dy.double() @ w, ((n + 4) * 2.0**-23 + half) * (dy.double().abs() @ w.abs()))


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
def test_input_grad_of_groups_with_scales_of_any_size(dtype):
    """Every group's scales of a size of their own; a scale that is not finite makes its own group's rows so."""
    g = _gen(52)
    sizes, n, k = [70, 0, 3, 130, 64], 264, 272
    size = torch.tensor([1e-9, 1.0, 2e3, 1e-4, 1e-6])
    d0 = torch.tensor([2.0**13, 1.0, 2.0**-12, 1.0, 2.0**6])
    e, t = len(sizes), sum(sizes) + 5
    q = torch.randint(-128, 128, (e, n, k), generator=g, dtype=torch.int8)
    s = (0.25 + 0.75 * torch.rand(e, n, 1, generator=g)) * size[:, None, None]
    ends = _ends(sizes)
    of = torch.repeat_interleave(torch.arange(e), torch.tensor(sizes))
    dy = _normal(g, t, n)
    dy[:t - 5] *= d0[of][:, None]
    dy = dy.to(dtype)
    half, _ = _half(dtype)
    for bad in (False, True):
        if bad:
            s[3, 7] = float("inf")
            s[4, 100] = float("nan")
        got = K.grouped_int8_matmul_input_grad(dy.to(DEV), q.to(DEV), s.to(DEV), ends.to(DEV))
        begin = 0
        for i, end in enumerate(ends.tolist()):
            if bad and i >= 3:
                assert not torch.isfinite(got[begin:end]).any()
            else:
                w, rows = q[i].double() * s[i].double(), dy[begin:end].double()
                _close(got[begin:end], rows @ w, ((n + 4) * 2.0**-23 + half) * (rows.abs() @ w.abs()))
            begin = end
        assert (got[begin:] == 0).all()


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
def test_input_grad_with_scales_of_zero(dtype):
    g = _gen(53)
    q = torch.randint(-128, 128, (96, 144), generator=g, dtype=torch.int8)
    dy = _normal(g, 20, 96, dtype=dtype)
    s = torch.zeros(96, 1)
    assert (K.int8_matmul_input_grad(dy.to(DEV), q.to(DEV), s.to(DEV)) == 0).all()
    s[5] = -3e-9  # (signs count)
    dy[:, 5] *= 1e4
    w, rows = q.double() * s.double(), dy.double()
    _close(K.int8_matmul_input_grad(dy.to(DEV), q.to(DEV), s.to(DEV)), rows @ w, (100 * 2.0**-23 + _half(dtype)[0]) * (rows.abs() @ w.abs()))


def test_fp16_gradients_follow_their_scales():
    """A captured gradient whose scales change between replays, through the layers, on another stream than its tensors'."""
    g = _gen(54)
    n, k, t = 200, 272, 90
    q = torch.randint(-128, 128, (2, n, k), generator=g, dtype=torch.int8)
    s0 = (0.25 + 0.75 * torch.rand(2, n, 1, generator=g)) * 1e-3
    ends = torch.tensor([40, t - 3], dtype=torch.int32)
    dy, x = _normal(g, t, n, dtype=F16), _normal(g, t, k, dtype=F16)
    q1, s1 = q.view(2 * n, k).to(DEV), s0.view(2 * n, 1).to(DEV)
    weight, one, at = Int8Weight(q1, s1, (1, k)), Int8Weight(q1[:n], s1[:n], (1, k)), ends.to(DEV)
    rows, dy1, factor = x.to(DEV).requires_grad_(), dy.to(DEV), torch.ones((), device=DEV)

    def work():
        y = grouped_linear(rows, weight, at)
        a, = torch.autograd.grad(y, rows, dy1 * factor.to(F16))
        b, = torch.autograd.grad(int8_linear(rows, one), rows, dy1 * factor.to(F16))
        return a, b

    def want(scale, f):
        w, d = q.double() * scale.double(), (dy * f).double()
        size = torch.cat((d[:40].abs() @ w[0].abs(), d[40:t - 3].abs() @ w[1].abs(), torch.zeros(3, k)))
        a = torch.cat((d[:40] @ w[0], d[40:t - 3] @ w[1], torch.zeros(3, k, dtype=torch.double)))
        return (a, size), (d @ w[0], d.abs() @ w[0].abs())

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = work()
    torch.cuda.current_stream().wait_stream(side)
    for down, f in ((1.0, 1.0), (1e-6, 2.0**12), (1e5, 2.0**-10), (1.0, 1.0)):
        s1.copy_((s0 * down).view(2 * n, 1))
        factor.fill_(f)
        graph.replay()
        got = [o.clone() for o in out]
        eager = work()
        for o, e, (a, size) in zip(got, eager, want(s1.cpu().view(2, n, 1), f)):
            assert (o == e).all()
            _close(o, a, ((n + 4) * 2.0**-23 + 2.0**-11) * size)
