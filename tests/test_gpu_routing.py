"""Routing to experts, and rows to their experts and back, against plain code in 64 bits.

Experts, places and ends have to be equal.  Tolerances, with D the largest difference of two logits that matter to a
weight: an exponential is off by 4 + D units of 2^-24 (2 units in its last place, and the rounding of its argument), a
sum of at most 1024 terms by 22 (a tree of 6 levels over at most 16 terms of a lane), a sigmoid's quotient by 8, and
3 roundings join them, above and below the fraction line: at most (60 + 2 D) 2^-24 of a weight.  A gradient is a sum of
terms, each of which has two such factors.  Outputs in 16 bits are off by half a unit in their last place besides.
Weighted sums of n terms are off by n + 1 roundings of 2^-24 of the sum of magnitudes.
"""

from __future__ import annotations

import math

import pytest
import torch

from piper_offload_amd import combine_experts, dispatch_experts, grouped_linear, route_experts

pytestmark = pytest.mark.gpu

K = pytest.importorskip("piper_offload_amd.kernels")

DEV = "cuda"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
INF = math.inf


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _normal(g, *shape, std=1.0, dtype=F32):
    return (torch.randn(*shape, generator=g) * std).to(dtype)


def _order(row, n):
    """Indices of the n largest entries above -inf, ties by index."""
    return [i for i in sorted(range(len(row)), key=lambda i: (-row[i], i)) if row[i] > -INF][:n]


def _scores(logits, score):
    x = logits.double()
    if score == "sigmoid":
        return 1 / (1 + torch.exp(-x))
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(top > -INF, top, 0.0))
    return e / e.sum(-1, keepdim=True).clamp_min(1e-300)


def _plain(logits, k, bias=None, score="softmax", groups=1, top_groups=1, group_best=1, renormalize=True, scale=1.0):
    t, e = logits.shape
    p = _scores(logits, score)
    # (without a bias the scores are in the order of the logits, also where they are equal in 64 bits)
    c = (p + bias.double() if bias is not None else p)
    c = torch.where(logits == -INF, -INF, c)
    rank = c if bias is not None else logits.double()
    expert = torch.full((t, k), -1)
    for i in range(t):
        row, values = c[i].tolist(), rank[i].tolist()
        if groups > 1:
            per = e // groups
            value = []
            for j in range(groups):
                best = sorted((v for v in row[j * per:(j + 1) * per] if v > -INF), reverse=True)[:group_best]
                value.append(sum(best) if best else -INF)
            kept = _order(value, top_groups)
            values = [v if n // per in kept else -INF for n, v in enumerate(values)]
        best = _order(values, k)
        expert[i, :len(best)] = torch.tensor(best, dtype=torch.long)
    on = expert >= 0
    picked = torch.where(on, logits.double().gather(1, expert.clamp_min(0)), 0.0)
    if renormalize:  # (from logarithms, for scores that are 0 in 64 bits)
        log = picked if score == "softmax" else torch.nn.functional.logsigmoid(picked)
        w = torch.softmax(torch.where(on, log, -INF), -1).nan_to_num(0.0)
    else:
        w = torch.where(on, p.gather(1, expert.clamp_min(0)), 0.0)
    key = torch.where(on, expert, e).reshape(-1)
    place = torch.empty_like(key)
    place[key.argsort(stable=True)] = torch.arange(key.numel())
    ends = torch.bincount(key, minlength=e + 1)[:e].cumsum(0)
    return w * scale, expert, place.view(t, k), ends


def _spread(logits):
    x = torch.where(logits > -1e30, logits.float(), 0.0)
    return float((x.amax(-1) - x.amin(-1)).max()) if x.numel() else 0.0


def _check(logits, k, bias=None, **how):
    got = K.route_topk(logits.to(DEV), k, bias=None if bias is None else bias.to(DEV), **how)
    w, expert, place, ends = _plain(logits.cpu(), k, bias, **how)
    assert got.weight.dtype is F32 and {got.expert.dtype, got.position.dtype, got.ends.dtype} == {torch.int32}
    assert (got.expert.cpu() == expert).all()
    assert (got.position.cpu() == place).all()
    assert (got.ends.cpu() == ends).all()
    tol = (60 + 2 * _spread(logits)) * 2.0**-24 * w.abs() + 2.0**-126
    off = (got.weight.double().cpu() - w).abs()
    assert (off <= tol).all(), f"worst {(off / tol).max():.3g} tolerances"
    return got


SIZES = [(1, 1, 1), (1, 8, 2), (3, 5, 5), (8, 32, 4), (17, 64, 6), (32, 65, 8), (33, 100, 1), (64, 128, 8), (100, 129, 7), (257, 256, 8),
         (1000, 60, 4), (40, 300, 12), (70, 512, 64), (50, 1024, 10), (5000, 16, 2), (20000, 8, 2)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("t,e,k", SIZES)
def test_route(t, e, k, score, dtype):
    g = _gen(t + e + k)
    logits = _normal(g, t, e, std=1.5, dtype=dtype)
    _check(logits, k, score=score, renormalize=(t + k) % 2 == 0, scale=2.5 if t % 3 else 1.0)
    _check(logits, k, _normal(g, e, std=0.1), score=score, renormalize=(t + k) % 2 == 1)


GROUPED = [(1, 8, 2, 2, 1, 1), (9, 32, 4, 8, 3, 2), (40, 256, 8, 8, 4, 2), (33, 160, 6, 8, 3, 1), (20, 60, 5, 3, 2, 2), (31, 64, 2, 64, 5, 1),
           (50, 1024, 8, 16, 4, 2), (300, 96, 3, 12, 12, 2), (45, 21, 6, 7, 2, 2), (12, 126, 4, 63, 9, 2)]


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("t,e,k,groups,top,best", GROUPED)
def test_groups(t, e, k, groups, top, best, score, dtype):
    g = _gen(t + e + k + groups)
    logits = _normal(g, t, e, std=1.5, dtype=dtype)
    logits[_normal(g, t, e) > 1.5] = -INF  # some closed ones, whole groups among them
    how = dict(score=score, groups=groups, top_groups=top, group_best=best)
    _check(logits, k, **how)
    _check(logits, k, _normal(g, e, std=0.1), scale=2.5, **how)


@pytest.mark.parametrize("bias", [None, "zero", "same", "steps"])
def test_ties_go_to_the_lowest_index(bias):
    """Few values of the logits, so that most choices are between equals; biases that keep them so."""
    g = _gen(3)
    for t, e, k, groups in ((40, 64, 8, 1), (40, 256, 8, 8), (200, 24, 5, 4)):
        logits = torch.randint(0, 3, (t, e), generator=g).to(BF16)
        b = None if bias is None else torch.zeros(e) if bias == "zero" else torch.full((e,), 0.25)
        if bias == "steps":
            b = torch.randint(0, 2, (e,), generator=g).float() / 4
        for score in ("softmax", "sigmoid"):
            _check(logits, k, b, score=score, groups=groups, top_groups=max(1, groups // 2), group_best=min(2, groups))


def test_choices_between_scores_that_agree_in_32_bits():
    """Pairs of experts whose biased scores differ by less than a rounding of 2^-24."""
    g = _gen(8)
    t, e = 300, 64
    logits = _normal(g, t, e)
    logits[:, 32:] = logits[:, :32] + _normal(g, t, 32, std=2e-7)
    bias = _normal(g, 32, std=0.05).repeat(2)
    for score in ("softmax", "sigmoid"):
        _check(logits, 8, bias, score=score)
        _check(logits, 8, bias, score=score, groups=2, top_groups=1, group_best=2)
        _check(logits, 8, None, score=score, groups=2, top_groups=1, group_best=2)


def test_closed_experts_and_padding():
    g = _gen(4)
    logits = _normal(g, 50, 40)
    logits[10:20] = -INF
    logits[20:25, 3:] = -INF
    logits[25, 1:] = -INF
    logits[26] = torch.finfo(F32).min  # (a mask of the type's lowest value closes nothing: all alike)
    logits[27, 5:] = torch.finfo(F32).min
    logits[28] = -200.0  # sigmoid: scores that are 0 in 32 bits
    logits[29] = 200.0
    for bias in (None, _normal(g, 40, std=0.1)):
        for score in ("softmax", "sigmoid"):
            for dtype in (F32, BF16, F16):
                x = logits.clamp_min(torch.finfo(dtype).min).to(dtype)
                x[logits == -INF] = -INF
                r = _check(x, 6, bias, score=score)
                assert (r.expert[10:20] == -1).all() and (r.weight[10:20] == 0).all()
                assert torch.isfinite(r.weight).all()
    b = torch.zeros(40)
    b[7] = -INF
    r = K.route_topk(torch.full((3, 40), 1.0, device=DEV), 40, bias=b.to(DEV))
    want = [i for i in range(40) if i != 7] + [-1]
    assert r.expert.tolist() == [want] * 3 and r.ends[-1] == 117


def test_not_a_number_stays_in_its_row():
    g = _gen(6)
    logits = _normal(g, 20, 30)
    logits[3, 4] = float("nan")
    logits[9, 29] = float("nan")
    logits[11, 2] = INF
    for bias in (None, _normal(g, 30, std=0.1)):
        for score in ("softmax", "sigmoid"):
            for groups in (1, 3):
                how = dict(score=score, groups=groups, top_groups=max(1, groups - 1), group_best=1)
                r = K.route_topk(logits.to(DEV), 4, bias=None if bias is None else bias.to(DEV), **how)
                bad = [3, 9] + ([11] if score == "softmax" else [])
                assert torch.isnan(r.weight[bad]).all()
                assert all(len(set(row)) == 4 and 0 <= min(row) and max(row) < 30 for row in r.expert.tolist())
                rest = [i for i in range(20) if i not in bad]
                w, expert, _, _ = _plain(logits[rest], 4, bias, **how)
                assert (r.expert.cpu()[rest] == expert).all() and torch.isfinite(r.weight[rest]).all()
                assert sorted(r.position.view(-1).tolist()) == list(range(80)) and int(r.ends[-1]) == 80


def test_strides():
    g = _gen(12)
    big = _normal(g, 70, 99, dtype=BF16).to(DEV)
    for x in (big[:, :64], big[:, 7:71], big[::2, :64], big[:, ::3], big[:64, :64].t(), big[:1, 3:60]):
        _check(x, 4)
        dw = _normal(g, x.shape[0], 4).to(DEV)
        e = K.route_topk(x, 4).expert
        a, b = K.route_topk_grad(dw, x, e), K.route_topk_grad(dw, x.contiguous(), e)
        assert a.is_contiguous() and (a == b).all()


def _grad_want(logits, expert, dw, score, renormalize, scale):
    """By autograd in 64 bits, and the sum of the terms' magnitudes."""
    x = logits.double().clone().requires_grad_()
    on = expert >= 0
    at = expert.clamp_min(0).long()
    if renormalize:
        log = x if score == "softmax" else torch.nn.functional.logsigmoid(x)
        w = torch.softmax(torch.where(on, log.gather(1, at), -1e300), -1)
    else:
        p = torch.softmax(torch.where(x == -INF, -1e300, x), -1) if score == "softmax" else torch.sigmoid(x)
        w = p.gather(1, at)
    w = torch.where(on, w, 0.0) * scale
    g = torch.where(on, dw.double(), 0.0)
    (w * g).sum().backward()
    total = (g * w).abs().sum(-1, keepdim=True)
    size = torch.zeros_like(x).scatter_add(1, at, torch.where(on, (g * w).abs(), 0.0)).detach()
    if renormalize:
        size += torch.zeros_like(x).scatter_add(1, at, w.abs() / abs(scale) * total).detach()
    elif score == "softmax":
        size += (torch.softmax(torch.where(x == -INF, -1e300, x), -1) * total).detach()
    return x.grad.nan_to_num(0.0), size


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_gradient(score, renormalize, dtype):
    for t, e, k in ((1, 1, 1), (5, 8, 2), (40, 64, 4), (33, 130, 8), (20, 256, 6), (9, 500, 64), (7, 1024, 10)):
        g = _gen(t + e)
        logits = _normal(g, t, e, std=1.5, dtype=dtype)
        if e > 8:
            logits[2, 3:] = -INF
            logits[3] = -INF
        dw = _normal(g, t, k)
        expert = K.route_topk(logits.to(DEV), k, score=score).expert
        got = K.route_topk_grad(dw.to(DEV), logits.to(DEV), expert, score=score, renormalize=renormalize, scale=2.5)
        want, size = _grad_want(logits, expert.cpu(), dw, score, renormalize, 2.5)
        half, tiny = {F32: (2.0**-24, 2.0**-120), BF16: (2.0**-8, 2.0**-120), F16: (2.0**-11, 2.0**-25)}[dtype]
        tol = (1 + 2.0**-8) * half * want.abs() + 2 * (60 + 2 * _spread(logits)) * 2.0**-24 * size + tiny
        assert got.dtype is dtype
        off = (got.double().cpu() - want).abs()
        assert (off <= tol).all(), f"{t} {e} {k}: worst {(off / tol).max():.3g} tolerances"


def test_gradient_against_differences():
    """The loss sum(w dw) along a direction, by central differences, whose error is of the third order."""
    g = _gen(14)
    logits, u, dw = _normal(g, 30, 48), _normal(g, 30, 48), _normal(g, 30, 5)
    for score in ("softmax", "sigmoid"):
        for renormalize in (True, False):
            how = dict(score=score, renormalize=renormalize)
            bias = torch.where(torch.arange(48) < 5, 100.0, 0.0).to(DEV)  # (the choice does not change)

            def loss(x):
                return (K.route_topk(x.to(DEV), 5, bias=bias, **how).weight.double().cpu() * dw.double()).sum()

            h = 2.0**-6
            r = K.route_topk(logits.to(DEV), 5, bias=bias, **how)
            along = (K.route_topk_grad(dw.to(DEV), logits.to(DEV), r.expert, **how).double().cpu() * u.double()).sum()
            diff = (loss(logits + h * u) - loss(logits - h * u)) / (2 * h)
            # third derivative of a weight along u: at most 6 of |u|^3, h^2 / 6 of it; fp32 weights' errors over 2 h
            u3 = (u.abs().amax(-1, keepdim=True) ** 3 * dw.abs()).sum()
            bound = h * h * u3 + 2 * (60 + 20) * 2.0**-24 * dw.abs().sum() / (2 * h)
            assert abs(along - diff) <= bound, (score, renormalize, float(along), float(diff))


def _case(g, t, e, k, cols, dtype, padded=0):
    logits = _normal(g, t, e)
    logits[t - padded:] = -INF
    r = K.route_topk(logits.to(DEV), k)
    x, dy = _normal(g, t, cols, dtype=dtype), _normal(g, t, cols, dtype=dtype)
    h, dh = _normal(g, t * k, cols, dtype=dtype), _normal(g, t * k, cols, dtype=dtype)
    return r, x, dy, h, dh


ROWS = [(1, 4, 1, 1, 0), (1, 8, 2, 7, 0), (5, 8, 3, 64, 2), (16, 32, 4, 2048, 0), (33, 20, 6, 513, 5), (70, 64, 8, 1000, 70), (9, 40, 33, 129, 1),
        (300, 16, 2, 4100, 17), (6, 64, 64, 24, 0)]


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("t,e,k,cols,padded", ROWS)
def test_rows(t, e, k, cols, padded, dtype):
    g = _gen(t + cols)
    r, x, dy, h, dh = _case(g, t, e, k, cols, dtype, padded)
    live = t - padded
    if padded:  # what padding holds is not looked at
        x[live:] = float("nan")
        h[live * k:] = float("nan")
        dh[live * k:] = INF
    at = (r.position, r.ends)
    place, w = r.position.cpu().long(), r.weight.double().cpu()
    assert sorted(place.view(-1).tolist()) == list(range(t * k)) and int(r.ends[-1]) == live * k
    rows = K.dispatch_rows(x.to(DEV), *at).cpu()
    want = torch.zeros_like(rows)
    want[place[:live].reshape(-1)] = x[:live].repeat_interleave(k, 0)
    assert (rows == want).all()

    half, tiny = (2.0**-8, 1e-38) if dtype is BF16 else (2.0**-11, 2.0**-25)

    def close(got, want, size, n, half=half, tiny=tiny):
        off = (got.double().cpu() - want).abs()
        assert (off <= (1 + 2.0**-8) * half * want.abs() + (n + 1) * 2.0**-24 * size + tiny).all()

    h64, d64, y64 = h.double(), dh.double(), dy.double()
    y = K.combine_rows(h.to(DEV), r.weight, *at)
    mine = torch.zeros(t, k, cols, dtype=torch.float64)
    mine[:live] = h64[place[:live]]
    w = torch.where((torch.arange(t) < live)[:, None], w, 0.0)
    close(y, (w[..., None] * mine).sum(1), (w[..., None] * mine).abs().sum(1), k)
    back = torch.zeros(t, k, cols, dtype=torch.float64)
    back[:live] = d64[place[:live]]
    close(K.dispatch_rows_grad(dh.to(DEV), *at), back.sum(1), back.abs().sum(1), k)
    gh, gw = K.combine_rows_grad(dy.to(DEV), h.to(DEV), r.weight, *at)
    wh = torch.zeros(t * k, cols, dtype=torch.float64)
    wh[place[:live].reshape(-1)] = (w[:live, :, None] * y64[:live, None]).reshape(-1, cols)
    close(gh, wh, wh.abs(), 1)
    terms = y64[:, None] * mine
    close(gw, terms.sum(-1), terms.abs().sum(-1), cols, half=2.0**-24)


def test_rows_of_other_strides():
    g = _gen(77)
    r, x, dy, h, dh = _case(g, 20, 8, 3, 200, BF16)
    at = (r.position, r.ends)

    def wide(v, off):
        out = torch.empty(v.shape[0], v.shape[1] + 11, dtype=v.dtype, device=DEV)[:, off:off + v.shape[1]]
        return out.copy_(v.to(DEV))

    for off in (0, 1, 8):
        assert (K.dispatch_rows(wide(x, off), *at) == K.dispatch_rows(x.to(DEV), *at)).all()
        assert (K.dispatch_rows_grad(wide(dh, off), *at) == K.dispatch_rows_grad(dh.to(DEV), *at)).all()
        assert (K.combine_rows(wide(h, off), r.weight, *at) == K.combine_rows(h.to(DEV), r.weight, *at)).all()
        a = K.combine_rows_grad(wide(dy, off), wide(h, off), r.weight, *at)
        b = K.combine_rows_grad(dy.to(DEV), h.to(DEV), r.weight, *at)
        assert (a[0] == b[0]).all() and (a[1] == b[1]).all()


def test_places_outside_are_passed_over():
    """Positions that are no places: nothing is read or written for them."""
    x = torch.ones(4, 16, dtype=BF16, device=DEV)
    ends = torch.tensor([3, 8], dtype=torch.int32, device=DEV)
    bad = torch.tensor([[0, 1], [-5, 2], [8, 3], [4, 1 << 30]], dtype=torch.int32, device=DEV)
    h = torch.ones(8, 16, dtype=BF16, device=DEV)
    w = torch.ones(4, 2, device=DEV)
    rows = K.dispatch_rows(x, bad, ends)
    assert (rows[:5] == 1).all()
    assert K.combine_rows(h, w, bad, ends)[:, 0].tolist() == [2, 1, 1, 1]
    gh, gw = K.combine_rows_grad(x, h, w, bad, ends)
    assert (gh[:5] == 1).all() and gw.tolist() == [[16, 16], [0, 16], [0, 16], [16, 0]]
    for past in (100, -3):  # ends that are not: at most all places, at least none
        out = K.combine_rows(h, w, bad, torch.tensor([3, past], dtype=torch.int32, device=DEV))
        assert out[:, 0].tolist() == ([2, 1, 1, 1] if past > 0 else [0, 0, 0, 0])


def _mixture(x, router, up, down, k, r=None):
    r = route_experts(x @ router.t(), k) if r is None else r
    h = grouped_linear(dispatch_experts(x, r), up, r.ends)
    return combine_experts(grouped_linear(torch.tanh(h), down, r.ends), r)


def test_a_mixture_of_experts_and_its_gradients():
    """All of it together against the same in plain float64, expert by expert; roundings of every step are counted
    as 2^-7 of the sums of magnitudes."""
    g = _gen(99)
    t, hidden, inner, e, k = 50, 64, 96, 6, 2
    x, router = _normal(g, t, hidden), _normal(g, e, hidden, std=hidden**-0.5)
    up, down = _normal(g, e, inner, hidden, std=hidden**-0.5), _normal(g, e, hidden, inner, std=inner**-0.5)
    dy = _normal(g, t, hidden)
    ours = [v.to(BF16).to(DEV).requires_grad_() for v in (x, router, up, down)]
    y = _mixture(*ours, k)
    y.backward(dy.to(BF16).to(DEV))
    plain = [v.detach().cpu().double().requires_grad_() for v in ours]
    px, pr, pu, pd = plain
    logits = (ours[0] @ ours[1].t()).detach().cpu()  # the choice sees rounded logits
    expert = K.route_topk(logits.to(DEV), k).expert.cpu().long()
    w = torch.softmax((px @ pr.t()).gather(1, expert), -1)
    out = torch.zeros(t, hidden, dtype=torch.float64)
    for j in range(k):
        hh = torch.tanh((pu[expert[:, j]] @ px[..., None])[..., 0])
        out = out + w[:, j:j + 1] * (pd[expert[:, j]] @ hh[..., None])[..., 0]
    out.backward(dy.to(BF16).double())
    assert (y.detach().cpu().double() - out.detach()).abs().max() <= 2.0**-7 * 4 * out.abs().max()
    for a, b in zip(ours, plain):
        assert (a.grad.cpu().double() - b.grad).norm() <= 2.0**-6 * b.grad.norm()


def test_graph_replays_and_other_streams():
    g = _gen(101)
    router = _normal(g, 8, 64, std=0.125, dtype=BF16).to(DEV)
    up, down = _normal(g, 8, 96, 64, std=0.1, dtype=BF16).to(DEV), _normal(g, 8, 64, 96, std=0.1, dtype=BF16).to(DEV)
    for t in (3, 200):
        x = _normal(g, t, 64, dtype=BF16).to(DEV)
        logits = (x @ router.t()).clone()

        def work():
            r = K.route_topk(logits, 2)
            y = _mixture(x, router, up, down, 2, r)
            return *r, y, K.route_topk_grad(r.weight, logits, r.expert)

        with torch.no_grad():
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
                x.copy_(_normal(g, t, 64, dtype=BF16))
                logits.copy_(x @ router.t())
                logits[t - min(i, t):] = -INF
                graph.replay()
                want = work()
                torch.cuda.synchronize()
                for a, b in zip(out, want):
                    assert (a == b).all()


def test_no_tokens():
    for e in (3, 100):
        r = K.route_topk(torch.empty(0, e, device=DEV), 2)
        assert r.expert.shape == (0, 2) and r.ends.tolist() == [0] * e
    x = torch.empty(0, 16, dtype=BF16, device=DEV)
    assert K.dispatch_rows(x, r.position, r.ends).shape == (0, 16) and K.dispatch_rows_grad(x, r.position, r.ends).shape == (0, 16)
    assert K.combine_rows(x, r.weight, r.position, r.ends).shape == (0, 16)
    assert K.combine_rows_grad(x, x, r.weight, r.position, r.ends)[1].shape == (0, 2)
    assert K.route_topk_grad(r.weight, torch.empty(0, e, device=DEV), r.expert).shape == (0, e)


def test_gradients_are_not_lost():
    x = torch.zeros(4, 8, device=DEV, requires_grad=True)
    with pytest.raises(NotImplementedError):
        K.route_topk(x, 2)
    r = route_experts(x, 2)
    assert r.weight.requires_grad and not r.expert.requires_grad
    h = torch.zeros(8, 16, dtype=BF16, device=DEV)
    with pytest.raises(NotImplementedError):
        K.combine_rows(h, r.weight, r.position, r.ends)
    with pytest.raises(NotImplementedError):
        K.dispatch_rows(torch.zeros(4, 16, dtype=BF16, device=DEV, requires_grad=True), r.position, r.ends)
    with pytest.raises(ValueError, match="detach"):
        route_experts(x, 2, bias=torch.zeros(8, device=DEV, requires_grad=True))


def _places_of(expert, e):
    """Places and ends of given choices, by a stable sort."""
    key = torch.where(expert < 0, e, expert).reshape(-1).long()
    place = torch.empty_like(key)
    place[key.argsort(stable=True)] = torch.arange(key.numel())
    return place.view(expert.shape), torch.bincount(key, minlength=e + 1)[:e].cumsum(0)


@pytest.mark.parametrize("t,e,k", [(4096, 70, 3), (4097, 70, 3), (32768, 12, 2), (32769, 12, 2), (70000, 33, 5), (6000, 1024, 4), (33000, 513, 2)])
def test_many_tokens(t, e, k):
    """Around the numbers of tokens where workgroups get larger and places are found another way; closed tokens in between.
    The logits of a row are whole numbers, so that many are equal: ties go to the lowest index."""
    g = _gen(t + e)
    logits = torch.randint(-40, 40, (t, e), generator=g).to(BF16)
    logits[torch.rand(t, generator=g) < 0.1] = -INF
    logits[t - 100:] = -INF
    logits[t // 2, 1:] = -INF
    r = K.route_topk(logits.to(DEV), k)
    value, index = logits.float().sort(dim=-1, descending=True, stable=True)
    expert = torch.where(value[:, :k] > -INF, index[:, :k], -1)
    assert (r.expert.cpu() == expert).all()
    place, ends = _places_of(expert, e)
    assert (r.position.cpu() == place).all() and (r.ends.cpu() == ends).all()


@pytest.mark.parametrize("many", [3, 20, 60, 64, 65, 100, 300])
def test_runs_of_scores_that_agree_in_32_bits(many):
    """`many` experts whose scores differ by less than a rounding of 2^-24, above the others: some of them are chosen."""
    g = _gen(many)
    t, e = 40, 320
    logits = _normal(g, t, e) - 6.0
    for i in range(t):
        logits[i, torch.randperm(e, generator=g)[:many]] = 1.0 + 1e-7 * torch.randint(0, 8, (many,), generator=g).float()
    bias = 1e-9 * _normal(g, e)
    for score in ("softmax", "sigmoid"):
        for k in (1, 8, 64):
            _check(logits, k, bias, score=score)
        _check(logits, 8, bias, score=score, groups=8, top_groups=3, group_best=2)
        _check(logits, 8, torch.full((e,), 0.5), score=score)  # (the same for all)


@pytest.mark.parametrize("e,groups", [(12, 3), (128, 64), (128, 2), (96, 1), (640, 5), (1020, 60), (64, 32), (72, 18), (1000, 8)])
def test_sizes_of_groups(e, groups):
    g = _gen(e + groups)
    logits = _normal(g, 60, e, std=1.5)
    per = e // groups
    for top in {1, (groups + 1) // 2, groups}:
        k = min(6, top * per)
        for best in (1, 2) if per > 1 else (1,):
            _check(logits, k, _normal(g, e, std=0.1), score="sigmoid", groups=groups, top_groups=top, group_best=best)
            _check(logits, k, score="softmax", groups=groups, top_groups=top, group_best=best)


@pytest.mark.parametrize("cols", [1, 8, 509, 1023, 1024, 1025, 2048, 2055, 4104, 9000])
def test_rows_there_and_back(cols):
    """Whole numbers, weights of one: rows and their sums come back exactly, whatever part of a row a wave has."""
    g = _gen(cols)
    for t, k in ((1, 1), (3, 5), (41, 4), (2300, 2)):
        if t * cols > 3e6:
            continue
        r = K.route_topk(_normal(g, t, 9).to(DEV), k)
        x = torch.randint(-8, 9, (t, cols), generator=g).to(BF16).to(DEV)
        at = (r.position, r.ends)
        rows = K.dispatch_rows(x, *at)
        assert (rows[r.position.long().view(-1)] == x.repeat_interleave(k, 0)).all()
        one = torch.ones_like(r.weight)
        assert (K.combine_rows(rows, one, *at) == x * k).all() and (K.dispatch_rows_grad(rows, *at) == x * k).all()
        dh, dw = K.combine_rows_grad(x, rows, one, *at)
        assert (dh == rows).all()
        assert (dw == (x.float() ** 2).sum(-1, keepdim=True)).all()


def test_backward_through_sums_and_views():
    """Gradients that come as broadcast or transposed views, captured into a graph as well."""
    g = _gen(55)
    logits = _normal(g, 60, 12).to(DEV).requires_grad_()
    x = _normal(g, 60, 80, dtype=BF16).to(DEV).requires_grad_()

    def grads(dy):
        r = route_experts(logits, 3, score="sigmoid")
        y = combine_experts(dispatch_experts(x, r), r)
        return torch.autograd.grad(y, (logits, x), dy)

    dy = _normal(g, 80, 60, dtype=BF16).to(DEV).t()
    for a, b in zip(grads(dy), grads(dy.contiguous())):
        assert (a == b).all()
    one = torch.ones((), dtype=BF16, device=DEV).expand(60, 80)
    want = grads(one.contiguous())
    for a, b in zip(grads(one), want):
        assert (a == b).all()
    static = dy.contiguous().clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        grads(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = grads(static)
    for _ in range(3):
        static.copy_(_normal(g, 60, 80, dtype=BF16))
        graph.replay()
        want = grads(static)
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert (a == b).all()


def test_refusals():
    logits = torch.zeros(6, 12, device=DEV)
    zeros = torch.zeros
    for args, how, text in (((zeros(12, device=DEV), 2), {}, "tokens, experts"), ((logits.double(), 2), {}, "supports"), ((logits, 0), {}, "top_k"),
                            ((logits, 13), {}, "top_k"), ((logits, 2), dict(score="tanh"), "score"), ((logits, 2), dict(groups=5), "divide"),
                            ((logits, 2), dict(groups=3, top_groups=4), "top_groups"), ((logits, 5), dict(groups=3, top_groups=1), "top_k"),
                            ((logits, 2), dict(groups=3, group_best=3), "group_best"), ((logits, 2), dict(groups=12, group_best=2), "group_best"),
                            ((logits, 2), dict(scale=math.nan), "scale"), ((logits, 2), dict(bias=zeros(11, device=DEV)), "bias"),
                            ((logits, 2), dict(bias=zeros(12, dtype=BF16, device=DEV)), "bias"), ((logits, 2), dict(bias=zeros(12)), "one GPU"),
                            ((zeros(2, 1025, device=DEV), 2), {}, "experts"), ((zeros(2, 0, device=DEV), 2), {}, "experts")):
        with pytest.raises(ValueError, match=text):
            K.route_topk(*args, **how)
    r = K.route_topk(logits, 2)
    for dw, expert, text in ((r.weight[:5], r.expert, "dweight"), (r.weight.double(), r.expert, "dweight"), (r.weight, r.expert.long(), "expert"),
                             (r.weight, r.expert[:5], "expert"), (r.weight, r.expert.cpu(), "one GPU")):
        with pytest.raises(ValueError, match=text):
            K.route_topk_grad(dw, logits, expert)
    x, h = zeros(6, 16, dtype=BF16, device=DEV), zeros(12, 16, dtype=BF16, device=DEV)
    at = (r.position, r.ends)
    bad = (r.position.long(), r.ends), (r.position.view(-1), r.ends), (r.position[:, :0], r.ends), (r.position, r.ends.long()), (r.position, r.ends[:0])
    for p, e in bad:
        for call in (lambda: K.dispatch_rows(x, p, e), lambda: K.dispatch_rows_grad(h, p, e), lambda: K.combine_rows(h, r.weight, p, e),
                     lambda: K.combine_rows_grad(x, h, r.weight, p, e)):
            with pytest.raises(ValueError):
                call()
    for call, text in ((lambda: K.dispatch_rows(h, *at), "6 rows"), (lambda: K.dispatch_rows(x.float(), *at), "supports"),
                       (lambda: K.dispatch_rows(x[:, :0], *at), "non-empty"), (lambda: K.dispatch_rows_grad(x, *at), "12 rows"),
                       (lambda: K.combine_rows(x, r.weight, *at), "12 rows"), (lambda: K.combine_rows(h, r.weight.half(), *at), "weight"),
                       (lambda: K.combine_rows(h, r.weight[:, :1], *at), "weight"), (lambda: K.combine_rows(h.cpu(), r.weight, *at), "GPU"),
                       (lambda: K.combine_rows_grad(x.half(), h, r.weight, *at), "differ"), (lambda: K.combine_rows_grad(x[:, :8], h, r.weight, *at), "differ"),
                       (lambda: K.combine_rows_grad(x[0], h, r.weight, *at), "rows")):
        with pytest.raises(ValueError, match=text):
            call()


def test_places_that_do_not_exist_are_passed_over():
    """Places outside the rows and ends that pass them: nothing is read or written out of range."""
    g = _gen(63)
    x, h, dy = (_normal(g, n, 40, dtype=BF16).to(DEV) for n in (5, 10, 5))
    w = torch.rand(5, 2, generator=g).to(DEV)
    position = torch.tensor([[0, 1], [2, 99], [-7, 3], [4, 2**31 - 1], [5, 6]], dtype=torch.int32, device=DEV)
    for last in (7, 10, 1000, 2**31 - 1):
        ends = torch.tensor([3, last], dtype=torch.int32, device=DEV)
        rows = K.dispatch_rows(x, position, ends)
        assert (rows[0] == x[0]).all() and (rows[4] == x[3]).all() and (rows[6] == x[4]).all()
        y = K.combine_rows(h, w, position, ends).double()
        want = w[3, 0].double() * h[4].double()
        assert ((y[3] - want).abs() <= 2.0**-8 * want.abs() + 1e-30).all()
        assert (K.dispatch_rows_grad(h, position, ends)[1] == h[2]).all()
        dh, dw = K.combine_rows_grad(dy, h, w, position, ends)
        assert (dw[[1, 2, 3], [1, 0, 1]] == 0).all() and torch.isfinite(dw).all()
    for last in (0, -5):
        ends = torch.tensor([0, last], dtype=torch.int32, device=DEV)
        assert (K.combine_rows(h, w, position, ends) == 0).all() and (K.dispatch_rows_grad(h, position, ends) == 0).all()


def test_experts_in_int8_from_logits_to_the_sum_and_back():
    """Routing, rows to experts, products with INT8 weights and 8-bit inputs, weighted sums; gradients of rows and logits.

    Roundings to bfloat16, half a step 2^-8 each: of a product's row and of the sum forward; backward of a row of w dy, a weight, a
    product's row and the sum (four, of the sum of magnitudes); a weight's gradient sees the rounded product (2^-8 of its
    magnitudes), a logit's is w_j (g_j - sum_i w_i g_i).  2^-6 of each bound is left for products of roundings and fp32 sums.
    """
    from piper_offload_amd import Int8Weight

    g = _gen(131)
    for t, e, k, n, cols, padded in ((1, 4, 2, 40, 48, 0), (70, 12, 3, 96, 160, 9), (400, 8, 4, 72, 130, 0)):
        q = torch.randint(-127, 128, (e * n, cols), generator=g, dtype=torch.int8)
        s = torch.rand(e * n, 1, generator=g) * 1e-3 + 1e-4
        weight = Int8Weight(q.to(DEV), s.to(DEV), (1, cols))
        x, logits, dy = _normal(g, t, cols, dtype=BF16), _normal(g, t, e), _normal(g, t, n, dtype=BF16)
        if padded:
            logits[t - padded:] = -INF
        ours = x.to(DEV).requires_grad_(), logits.to(DEV).requires_grad_()
        r = route_experts(ours[1], k)
        h = grouped_linear(dispatch_experts(ours[0], r), weight, r.ends, activation_dtype=torch.int8)
        y = combine_experts(h, r)
        dx, dl = torch.autograd.grad(y, ours, dy.to(DEV))

        live, expert = t - padded, r.expert.cpu().long()
        w64 = (q.double() * s.double()).view(e, n, cols)
        scale = (x.float().abs().amax(-1, keepdim=True) * (torch.ones(()) / 127)).double()  # (torch's / 127 on the GPU)
        codes = torch.round(x.double() / scale).clamp(-127, 127) * scale
        of = w64[expert.clamp_min(0)]  # [t, k, n, cols]
        p = torch.where(expert >= 0, r.weight.detach().double().cpu(), 0.0)
        hh = (of @ codes[:, None, :, None])[..., 0]
        want, size = (p[..., None] * hh).sum(1), (p[..., None] * hh).abs().sum(1)
        more = 1 + 2.0**-6
        assert ((y.detach().double().cpu() - want).abs() <= more * 2.0**-8 * (size + want.abs()) + 1e-30).all()
        wdy = p[..., None] * dy.double()[:, None]
        want, size = (wdy[:, :, None] @ of).sum((1, 2)), (wdy.abs()[:, :, None] @ of.abs()).sum((1, 2))
        assert ((dx.double().cpu() - want).abs() <= more * 4 * 2.0**-8 * size + 1e-30).all()
        grad, err = (dy.double()[:, None] * hh).sum(-1), 2.0**-8 * (dy.double()[:, None] * hh).abs().sum(-1)
        want = p * (grad - (p * grad).sum(-1, keepdim=True))
        bound = more * p * (err + (p * err).sum(-1, keepdim=True)) + 2.0**-20 * p * (grad.abs() + (p * grad.abs()).sum(-1, keepdim=True))
        at = expert.clamp_min(0)
        got = dl.double().cpu()
        assert ((got.gather(1, at)[:live] - want[:live]).abs() <= bound[:live] + 1e-30).all()
        assert (got.scatter(1, at, 0.0)[:live] == 0).all() and (got[live:] == 0).all() and (dx[live:] == 0).all() and (y[live:] == 0).all()


@pytest.mark.parametrize("bound", [100.0, 1e3, 1e4, 1e5])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_values_of_groups_that_cancel(score, bound):
    """Biases of opposite sign inside every group: its value is of the size of a score, its two addends, rounded to 32 bits,
    are of the size of the bias."""
    g = _gen(41)
    e = 16
    bias = torch.tensor([bound, -bound]).repeat(e // 2)
    for t in (20, 6000):
        logits = _normal(g, t, e, std=0.05)
        _check(logits, 2, bias, score=score, groups=8, top_groups=4, group_best=2)
    more = bias.clone()
    more[4:6] = -1e30  # a group that its bias all but closes
    more[9] = -INF  # one of a single open expert
    _check(logits[:500], 2, more, score=score, groups=8, top_groups=4, group_best=2)


def test_a_bias_that_is_the_same_for_all_is_a_bias():
    """With one the numbers p + bias decide, and those of far logits are equal in 64 bits: the lowest index has them."""
    rows = {"sigmoid": [[40.0, 50.0, 45.0, -3.0], [50.0, 40.0, 60.0, 41.0], [-60.0, -50.0, -70.0, -55.0], [-2.0, 60.0, 1.0, 70.0]],
            "softmax": [[-900.0, -800.0, 0.0, -1000.0], [0.0, -900.0, -800.0, -850.0], [-800.0, -790.0, -780.0, 5.0], [1.0, 2.0, -800.0, 900.0]]}
    for score, logits in rows.items():
        logits = torch.tensor(logits)
        for t in (1, 50):
            for value in (0.0, 0.25):
                bias = torch.full((4,), value)
                x = logits.repeat(t, 1)
                for how in ({}, dict(groups=2, top_groups=1, group_best=1), dict(groups=2, top_groups=1, group_best=2)):
                    _check(x, 2, bias, score=score, **how)
                    _check(x, 2, None, score=score, **({} if how.get("group_best") == 1 else how))
            more = torch.tensor([0.0, 0.0, 0.0, 1e-30])  # (nothing beside a score of 1)
            _check(logits.repeat(t, 1), 2, more, score=score)
    many = torch.linspace(40.0, 90.0, 300).flip(0).repeat(3, 1)  # (more equal ones than a wave has lanes)
    r = _check(many, 5, torch.zeros(300), score="sigmoid")
    assert r.expert.tolist() == [[0, 1, 2, 3, 4]] * 3
