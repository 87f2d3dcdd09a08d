"""The products' boundary without a GPU: the struct's layout, host-side checks of the C entries, refusals of CPU tensors."""

from __future__ import annotations

import ctypes
import os
import subprocess

import pytest
import torch

from piper_offload_amd import MXWeight, expert_view, grouped_linear, mx_linear
from piper_offload_amd import _lib as L
from piper_offload_amd import kernels as K

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FP4 = getattr(torch, "float4_e2m1fn_x2", None)
BF16 = torch.bfloat16


def test_weight_struct_matches_a_c_compiler(tmp_path):
    fields = [name for name, _ in L.WeightStruct._fields_]
    src = "#include <stdio.h>\n#include <stddef.h>\n#include \"lora_merge.h\"\nint main(void) {\n"
    src += "".join(f'printf("%zu\\n", offsetof(lm_weight, {f}));\n' for f in fields)
    src += 'printf("%zu\\n%d\\n", sizeof(lm_weight), LM_LINEAR_MAX_EXPERTS); return 0; }\n'
    (tmp_path / "w.c").write_text(src)
    exe = tmp_path / "w"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), "-o", str(exe), str(tmp_path / "w.c")], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    want = [getattr(L.WeightStruct, f).offset for f in fields] + [ctypes.sizeof(L.WeightStruct), K._MAX_EXPERTS]
    assert got == want


def _weight(**over):
    fields = dict(q=4096, scale=4096, N=64, K=128, dtype=L.LM_E2M1, swizzled=0, experts=1, reserved=0) | over
    return L.WeightStruct(**fields)


# (what is wrong, the weight's fields, the call's arguments): nothing here reaches the GPU
@pytest.mark.parametrize("over,args", [
    (dict(q=None), {}), (dict(scale=None), {}), (dict(N=0), {}), (dict(K=0), {}), (dict(K=100), {}), (dict(q=4100), {}),
    (dict(experts=0), {}), (dict(experts=1025), {}), (dict(experts=2), {}), (dict(dtype=L.LM_E4M3), {}),
    (dict(dtype=L.LM_F16), {}), ({}, dict(dtype=L.LM_F32)), ({}, dict(T=-1)), ({}, dict(x=None)), ({}, dict(y=None)),
    ({}, dict(ldx=127)),
], ids=str)
def test_c_entries_refuse_bad_arguments(over, args):
    a = dict(x=4096, ldx=128, y=4096, T=4, dtype=L.LM_BF16) | args
    w = _weight(**over)
    handle = L.load_library()
    assert handle.lm_linear(a["x"], a["ldx"], ctypes.byref(w), None, None, a["y"], a["T"], a["dtype"], a["dtype"], None, 0,
                            None) in (L.LM_EINVAL, L.LM_EUNSUPPORTED)
    assert handle.lm_last_error()
    if a["ldx"] == 128:
        assert handle.lm_linear_input_grad(a["x"], a["ldx"], ctypes.byref(w), None, a["y"], a["T"], a["dtype"], None, 0,
                                           None) in (L.LM_EINVAL, L.LM_EUNSUPPORTED)


def test_c_entries_refuse_more():
    handle = L.load_library()
    w = _weight()
    assert handle.lm_linear(4096, 128, None, None, None, 4096, 4, L.LM_BF16, L.LM_BF16, None, 0, None) == L.LM_EINVAL
    # an input dtype that is neither the rows' nor LM_E2M1; 4-bit inputs with a dense weight; without workspace
    assert handle.lm_linear(4096, 128, ctypes.byref(w), None, None, 4096, 4, L.LM_BF16, L.LM_E4M3, None, 0,
                            None) == L.LM_EUNSUPPORTED
    dense = _weight(dtype=L.LM_BF16)
    assert handle.lm_linear(4096, 128, ctypes.byref(dense), None, None, 4096, 4, L.LM_BF16, L.LM_E2M1, None, 0,
                            None) == L.LM_EUNSUPPORTED
    need = handle.lm_linear_workspace_size(0, 300, 128, 0, 64, 128, 1, L.LM_E2M1, L.LM_E2M1, 1)
    assert need >= 300 * (64 + 4)
    assert handle.lm_linear(4096, 128, ctypes.byref(w), None, None, 4096, 300, L.LM_BF16, L.LM_E2M1, 4096, need - 256,
                            None) == L.LM_EWORKSPACE
    assert handle.lm_linear(4096, 128, ctypes.byref(w), None, None, 4096, 300, L.LM_BF16, L.LM_E2M1, 4097, need,
                            None) == L.LM_EINVAL
    for n, k, e, lddy, ldx in ((0, 8, 1, 8, 8), (8, 0, 1, 8, 8), (8, 8, 0, 8, 8), (8, 8, 2, 8, 8), (8, 8, 1, 7, 8),
                               (8, 8, 1, 8, 7)):
        assert handle.lm_linear_weight_grad(4096, lddy, 4096, ldx, None, 4096, 4, n, k, e, L.LM_BF16, None, 0,
                                            None) == L.LM_EINVAL


def test_cpu_tensors_are_refused():
    q, s = torch.zeros(32, 32, dtype=torch.uint8), torch.zeros(32, 2, dtype=torch.uint8)
    x, ends = torch.zeros(2, 64, dtype=BF16), torch.zeros(1, dtype=torch.int32)
    weight = MXWeight(q, s, FP4)
    dense = torch.zeros(1, 32, 64, dtype=BF16)
    for call in (lambda: K.mx_matmul(x, q, s), lambda: mx_linear(x, weight), lambda: K.mx_matmul_input_grad(x, q, s),
                 lambda: K.grouped_matmul(x, dense, ends), lambda: grouped_linear(x, weight, ends),
                 lambda: K.grouped_matmul_weight_grad(x, x, ends)):
        with pytest.raises(ValueError, match="GPU"):
            call()


def test_expert_view_shares_storage():
    q = torch.arange(4 * 128 * 64, dtype=torch.int64).to(torch.uint8).view(512, 64)
    for swizzled in (False, True):
        s = torch.arange(512 * 4, dtype=torch.int64).to(torch.uint8).view((128, 16) if swizzled else (512, 4))
        view = expert_view(MXWeight(q, s, FP4, 32, BF16, swizzled, "even"), 2, 4)
        assert tuple(view.shape) == (128, 128) and view.scaling_mode == "even" and view.is_swizzled_scales is swizzled
        assert view.qdata.data_ptr() == q.data_ptr() + 2 * 128 * 64
        assert view.scale.data_ptr() == s.data_ptr() + 2 * 128 * 4
    with pytest.raises(ValueError):
        expert_view(MXWeight(q, s, FP4, 32, BF16, True), 0, 8)  # 64 rows an expert: half a swizzled tile
    with pytest.raises(ValueError):
        expert_view(MXWeight(q, s, FP4, 32, BF16, True), 4, 4)
    with pytest.raises(ValueError):
        expert_view(MXWeight(q, s, FP4, 32, BF16, True), 0, 5)


@pytest.mark.parametrize("dtype,input_dtype", [(L.LM_BF16, L.LM_BF16), (L.LM_I8, L.LM_BF16), (L.LM_I8, L.LM_I8), (L.LM_E2M1, L.LM_BF16),
                                               (L.LM_E2M1, L.LM_E2M1)])
def test_products_that_one_launch_cannot_hold_are_refused(dtype, input_dtype):
    """2^31 - 1 short rows are a number of rows that the header allows, but more tiles than a launch has threads for."""
    handle, t = L.load_library(), (1 << 31) - 1
    w = _weight(dtype=dtype, N=32, K=32, reserved=L.LM_F32)
    args = 4096, 32, ctypes.byref(w), None
    assert handle.lm_linear(*args, None, 4096, t, L.LM_BF16, input_dtype, 4096, 1 << 60, None) == L.LM_EUNSUPPORTED
    assert b"launch" in handle.lm_last_error()
    if input_dtype == L.LM_BF16:
        assert handle.lm_linear_input_grad(*args, 4096, t, L.LM_BF16, 4096, 1 << 60, None) == L.LM_EUNSUPPORTED
        assert handle.lm_linear_input_grad(4096, 33, ctypes.byref(w), None, 4096, t, L.LM_BF16, 4096, 1 << 60, None) == L.LM_EUNSUPPORTED
