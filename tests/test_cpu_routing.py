"""Routing and INT8 products without a GPU: the structs' layouts, host-side checks of the C entries, refusals."""

from __future__ import annotations

import ctypes
import os
import subprocess

import pytest
import torch

from piper_offload_amd import Int8Weight, combine_experts, dispatch_experts, expert_view, grouped_linear, int8_linear, route_experts
from piper_offload_amd import _lib as L
from piper_offload_amd import kernels as K

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("struct,name,extra", [
    (L.RouteStruct, "lm_route", {"LM_ROUTE_MAX_BEST": K._MAX_BEST, "LM_ROUTE_MAX_GROUPS": K._MAX_GROUPS,
                                 "LM_ROUTE_SIGMOID": K._SCORES["sigmoid"], "LM_I8": L.LM_I8}),
    (L.RowsStruct, "lm_rows", {}),
])
def test_structs_match_a_c_compiler(tmp_path, struct, name, extra):
    fields = [f for f, _ in struct._fields_]
    src = "#include <stdio.h>\n#include <stddef.h>\n#include \"lora_merge.h\"\nint main(void) {\n"
    src += "".join(f'printf("%zu\\n", offsetof({name}, {f}));\n' for f in fields) + f'printf("%zu\\n", sizeof({name}));\n'
    src += "".join(f'printf("%d\\n", (int){c});\n' for c in extra) + "return 0; }\n"
    (tmp_path / "w.c").write_text(src)
    exe = tmp_path / "w"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), "-o", str(exe), str(tmp_path / "w.c")], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [getattr(struct, f).offset for f in fields] + [ctypes.sizeof(struct), *extra.values()]


# nothing here reaches the GPU
@pytest.mark.parametrize("over", [
    dict(logits=None), dict(ld=15), dict(T=-1), dict(T=1 << 30, top_k=4), dict(experts=0), dict(experts=1025, ld=2000), dict(dtype=L.LM_E4M3),
    dict(score=2), dict(score=-1), dict(top_k=0), dict(top_k=17), dict(top_k=65, experts=128, ld=128), dict(groups=0), dict(groups=3),
    dict(groups=128, experts=128, ld=128), dict(groups=4, top_groups=5), dict(groups=4, top_groups=0), dict(group_best=0), dict(group_best=3),
    dict(groups=16, group_best=2), dict(groups=4, top_groups=1, top_k=5),
], ids=str)
def test_c_routing_refuses(over):
    fields = dict(logits=4096, bias=None, ld=16, T=4, experts=16, dtype=L.LM_BF16, score=0, top_k=2, groups=1, top_groups=1, group_best=1,
                  renormalize=1, scale=1.0, reserved=0) | over
    r = L.RouteStruct(**fields)
    handle = L.load_library()
    assert handle.lm_route_topk(ctypes.byref(r), 4096, 4096, 4096, 4096, None, 0, None) in (L.LM_EINVAL, L.LM_EUNSUPPORTED)
    assert handle.lm_last_error()
    assert handle.lm_route_topk_grad(ctypes.byref(r), 4096, 4096, 4096, None) in (L.LM_EINVAL, L.LM_EUNSUPPORTED)


def test_c_routing_refuses_pointers_and_workspaces():
    r = L.RouteStruct(4096, None, 16, 1000, 16, L.LM_BF16, 0, 2, 1, 1, 1, 1, 1.0, 0)
    handle, p = L.load_library(), ctypes.byref(r)
    need = handle.lm_route_workspace_size(1000, 16)
    assert need > 0
    for outs in ((None, 4096, 4096, 4096), (4096, None, 4096, 4096), (4096, 4096, None, 4096), (4096, 4096, 4096, None)):
        assert handle.lm_route_topk(p, *outs, 4096, need, None) == L.LM_EINVAL
    assert handle.lm_route_topk(p, 4096, 4096, 4096, 4096, None, 0, None) == L.LM_EWORKSPACE
    assert handle.lm_route_topk(p, 4096, 4096, 4096, 4096, 4096, need - 1, None) == L.LM_EWORKSPACE
    assert handle.lm_route_topk(p, 4096, 4096, 4096, 4096, 4100, need, None) == L.LM_EINVAL
    assert handle.lm_route_topk(None, 4096, 4096, 4096, 4096, None, 0, None) == L.LM_EINVAL


@pytest.mark.parametrize("over", [dict(T=-1), dict(N=0), dict(top_k=0), dict(experts=0), dict(experts=1025), dict(dtype=L.LM_F32), dict(position=None),
                                  dict(ends=None), dict(T=1 << 30, top_k=2), dict(N=1 << 31)], ids=str)
def test_c_rows_refuse(over):
    r = L.RowsStruct(**(dict(position=4096, ends=4096, T=4, N=16, top_k=2, experts=3, dtype=L.LM_BF16, reserved=0) | over))
    handle, p = L.load_library(), ctypes.byref(r)
    bad = (L.LM_EINVAL, L.LM_EUNSUPPORTED)
    assert handle.lm_dispatch_rows(p, 4096, 1 << 32, 4096, None) in bad
    assert handle.lm_dispatch_rows_grad(p, 4096, 1 << 32, 4096, None) in bad
    assert handle.lm_combine_rows(p, 4096, 1 << 32, 4096, 4096, None) in bad
    assert handle.lm_combine_rows_grad(p, 4096, 1 << 32, 4096, 1 << 32, 4096, 4096, 4096, None) in bad


def test_c_rows_refuse_pointers_and_strides():
    r = L.RowsStruct(4096, 4096, 4, 16, 2, 3, L.LM_BF16, 0)
    handle, p = L.load_library(), ctypes.byref(r)
    assert handle.lm_dispatch_rows(p, None, 16, 4096, None) == handle.lm_dispatch_rows(p, 4096, 15, 4096, None) == L.LM_EINVAL
    assert handle.lm_dispatch_rows_grad(p, 4096, 16, None, None) == handle.lm_combine_rows(p, 4096, 16, None, 4096, None) == L.LM_EINVAL
    for i in (1, 3, 5, 6, 7):
        args = [p, 4096, 16, 4096, 16, 4096, 4096, 4096, None]
        args[i] = None
        assert handle.lm_combine_rows_grad(*args) == L.LM_EINVAL
    assert handle.lm_combine_rows_grad(p, 4096, 15, 4096, 16, 4096, 4096, 4096, None) == L.LM_EINVAL
    assert handle.lm_combine_rows_grad(p, 4096, 16, 4096, 15, 4096, 4096, 4096, None) == L.LM_EINVAL


@pytest.mark.parametrize("weight,input_dtype", [
    (dict(scale=None), L.LM_BF16), (dict(reserved=L.LM_F16), L.LM_BF16), (dict(reserved=7), L.LM_BF16), ({}, L.LM_E2M1), (dict(K=132105), L.LM_I8),
    (dict(dtype=L.LM_BF16), L.LM_I8), (dict(dtype=L.LM_E2M1), L.LM_I8), (dict(experts=3), L.LM_I8), (dict(q=None), L.LM_I8),
], ids=str)
def test_c_int8_products_refuse(weight, input_dtype):
    w = L.WeightStruct(**(dict(q=4096, scale=4096, N=64, K=128, dtype=L.LM_I8, swizzled=0, experts=1, reserved=0) | weight))
    handle = L.load_library()
    assert handle.lm_linear(4096, 1 << 20, ctypes.byref(w), None, None, 4096, 4, L.LM_BF16, input_dtype, 4096, 1 << 40, None) in (
        L.LM_EINVAL, L.LM_EUNSUPPORTED)
    assert handle.lm_last_error()


def test_c_int8_products_need_their_workspace():
    w = L.WeightStruct(4096, 4096, 64, 128, L.LM_I8, 0, 1, 0)
    handle = L.load_library()
    assert handle.lm_linear_workspace_size(0, 4, 128, 0, 64, 128, 1, L.LM_I8, L.LM_I8, 1) == 0  # (quantised by the product itself)
    need = handle.lm_linear_workspace_size(0, 8, 128, 0, 64, 128, 1, L.LM_I8, L.LM_I8, 1)
    assert need >= 8 * 128
    for ws, size, want in ((None, 0, L.LM_EWORKSPACE), (4096, need - 1, L.LM_EWORKSPACE), (4100, need, L.LM_EINVAL)):
        assert handle.lm_linear(4096, 128, ctypes.byref(w), None, None, 4096, 8, L.LM_BF16, L.LM_I8, ws, size, None) == want


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    q, s = torch.zeros(32, 64, dtype=torch.int8), torch.ones(32, 1)
    p, ends = torch.zeros(4, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    for call in (lambda: K.int8_matmul(x, q, s), lambda: K.int8_matmul_input_grad(x[:, :32], q, s), lambda: int8_linear(x, Int8Weight(q, s, (1, 64))),
                 lambda: K.route_topk(x, 2), lambda: route_experts(x, 2), lambda: K.dispatch_rows(x, p, ends),
                 lambda: K.combine_rows(x[:2].repeat(4, 1), torch.zeros(4, 2), p, ends), lambda: K.dispatch_rows_grad(x.repeat(2, 1), p, ends),
                 lambda: K.combine_rows_grad(x, x.repeat(2, 1), torch.zeros(4, 2), p, ends), lambda: K.route_topk_grad(torch.zeros(4, 2), x, p),
                 lambda: dispatch_experts(x, K.Routing(torch.zeros(4, 2), p, p, ends)),
                 lambda: combine_experts(x.repeat(2, 1), K.Routing(torch.zeros(4, 2), p, p, ends))):
        with pytest.raises(ValueError, match="GPU"):
            call()


def test_expert_views_share_storage():
    q, s = torch.arange(6 * 32, dtype=torch.int8).view(6, 32), torch.arange(6.0).view(6, 1)
    w = Int8Weight(q, s, (1, 32))
    v = expert_view(w, 2, 3)
    assert isinstance(v, Int8Weight) and tuple(v.shape) == (2, 32) and v.block_size == (1, 32)
    assert v.qdata.data_ptr() == q[4:].data_ptr() and v.scale.data_ptr() == s[4:].data_ptr()
    for index, groups in ((3, 3), (-1, 3), (0, 4), (0, 0)):
        with pytest.raises(ValueError):
            expert_view(w, index, groups)
    with pytest.raises(ValueError):
        expert_view(Int8Weight(q, torch.ones(6, 2), (1, 16)), 0, 3)


@pytest.mark.parametrize("over", [
    dict(score="tanh"), dict(groups=0), dict(groups=3), dict(groups=4, top_groups=5), dict(groups=4, top_groups=0), dict(group_best=3),
    dict(group_best=0), dict(groups=16, group_best=2), dict(top_k=0), dict(top_k=17), dict(groups=4, top_groups=1, top_k=5),
    dict(scale=float("nan")), dict(scale=0.0), dict(scale=float("inf")), dict(bias=torch.zeros(15)), dict(bias=torch.zeros(16, dtype=torch.float64)),
    dict(logits=torch.zeros(4, 16, dtype=torch.int32)), dict(logits=torch.zeros(16)), dict(logits=torch.zeros(4, 0)),
    dict(logits=torch.zeros(4, 1025)), dict(logits=torch.zeros(1, 4, 16)),
], ids=str)
def test_routing_arguments_are_checked(over):
    args = dict(logits=torch.zeros(4, 16), top_k=2, bias=None, score="softmax", groups=1, top_groups=1, group_best=1, renormalize=True, scale=1.0) | over
    with pytest.raises(ValueError):
        K._route("Routing", **args)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradients_of_int8_scales_are_refused(dtype):
    """A scale is a number that could be trained; the products have no gradient for it and say so."""
    x, ends = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(4, dtype=torch.int32)
    q, s = torch.zeros(32, 64, dtype=torch.int8), torch.ones(32, 1, dtype=dtype, requires_grad=True)
    w = Int8Weight(q, s, (1, 64))
    for rows in (x, x.clone().requires_grad_()):
        for call in (lambda: int8_linear(rows, w), lambda: grouped_linear(rows, w, ends)):
            with pytest.raises(ValueError, match="scale is frozen"):
                call()
            with torch.no_grad(), pytest.raises(ValueError, match="GPU"):
                call()
    for codes, scale in ((q, s), (q.view(4, 8, 64), s.view(4, 8, 1))):
        with pytest.raises(NotImplementedError, match="gradient"):
            K._int8_weight("INT8 product", codes, scale, codes.ndim == 3)
        with torch.no_grad():
            assert K._int8_weight("INT8 product", codes, scale, codes.ndim == 3).dtype == L.LM_I8
        assert K._int8_weight("INT8 product", codes, scale.detach(), codes.ndim == 3).dtype == L.LM_I8
    expert_view(w, 1, 4)  # (a view is not a product)


def test_c_int8_gradients_in_fp16_need_their_workspace():
    """A power of two for each expert's scales; bf16 needs none."""
    w = L.WeightStruct(4096, 4096, 64, 128, L.LM_I8, 0, 3, 0)
    handle = L.load_library()
    assert handle.lm_linear_workspace_size(1, 4, 64, 0, 64, 128, 3, L.LM_I8, L.LM_BF16, 1) == 0
    need = handle.lm_linear_workspace_size(1, 4, 64, 0, 64, 128, 3, L.LM_I8, L.LM_F16, 1)
    assert need >= 3 * 4
    for ws, size, want in ((None, 0, L.LM_EWORKSPACE), (4096, need - 1, L.LM_EWORKSPACE), (4100, need, L.LM_EINVAL)):
        assert handle.lm_linear_input_grad(4096, 64, ctypes.byref(w), 4096, 4096, 4, L.LM_F16, ws, size, None) == want


def test_tokens_that_one_launch_cannot_hold_are_refused():
    """64 tokens a workgroup of 1024 threads, and fewer than 2^32 threads a launch."""
    handle, most = L.load_library(), (1 << 28) - 64
    for t in (most + 1, 1 << 28):
        r = L.RouteStruct(4096, None, 1, t, 1, L.LM_F32, 0, 1, 1, 1, 1, 1, 1.0, 0)
        assert handle.lm_route_workspace_size(t, 1) == 0
        assert handle.lm_route_topk(ctypes.byref(r), 4096, 4096, 4096, 4096, None, 0, None) == L.LM_EUNSUPPORTED
        assert handle.lm_route_topk_grad(ctypes.byref(r), 4096, 4096, 4096, None) == L.LM_EUNSUPPORTED
        with pytest.raises(ValueError, match="tokens"):
            K._route("Routing", torch.zeros(1, 1).expand(t, 1), 1, None, "softmax", 1, 1, 1, True, 1.0)
    assert handle.lm_route_workspace_size(most, 1) > 0
    r = L.RouteStruct(4096, None, 1, most, 1, L.LM_F32, 0, 1, 1, 1, 1, 1, 1.0, 0)
    assert handle.lm_route_topk(ctypes.byref(r), 4096, 4096, 4096, 4096, None, 0, None) == L.LM_EWORKSPACE


@pytest.mark.parametrize("scale", [1e39, -1e39, 3.5e38, 1e-46, -1e-60, float("nan"), -float("inf"), 0.0])
def test_scales_that_float32_does_not_have_are_refused(scale):
    """The kernels take the scale in float32, where these are infinite or zero."""
    with pytest.raises(ValueError, match="scale"):
        K._route("Routing", torch.zeros(4, 16), 2, None, "softmax", 1, 1, 1, True, scale)


@pytest.mark.parametrize("scale", [2.5, -1, 2.0**-149, torch.finfo(torch.float32).max])
def test_scales_that_float32_has_are_taken(scale):
    r, _ = K._route("Routing", torch.zeros(4, 16), 2, None, "softmax", 1, 1, 1, True, scale)
    assert r.scale == scale
