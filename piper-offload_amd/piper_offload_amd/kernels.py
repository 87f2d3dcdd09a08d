"""Drop-in replacements for piper-offload's fused merge functions.

Each public function keeps the exact signature, argument meaning, return
value and ``ValueError`` behaviour of the reference function it replaces
(P/ = the reference's src/piper_offload/), and calls the HIP kernels through
the C ABI:

* :func:`merge_int8_lora`   <- P/_triton_int8_lora.py:267-407
* :func:`merge_float8_lora` <- P/_triton_float8_lora.py:486-588
* :func:`merge_nvfp4_lora`  <- P/_triton_nvfp4_lora.py:515-595
* :func:`merge_mx_lora_`    <- P/_triton_mx_lora.py:333-425
* :func:`merge_q8_0_lora`   -- GGUF Q8_0 merge (no reference counterpart)
* :func:`merge_dense_lora_` <- RegularAdapter.merge_lora_ (P/tensor_adapters.py:686-696)
* :func:`dequantize_gguf`   <- P/gguf_dequant.py:303-331 (all 15 dispatched types)

Products with weights as they are stored (no reference counterpart; with
autograd in :mod:`.linear`, these refuse to lose a gradient):

* :func:`mx_matmul`, :func:`mx_matmul_input_grad` -- one MXFP4 weight
* :func:`grouped_matmul`, :func:`grouped_matmul_input_grad`,
  :func:`grouped_matmul_weight_grad` -- one dense weight per group of rows
* :func:`grouped_mx_matmul`, :func:`grouped_mx_matmul_input_grad` -- one MXFP4
  weight per group of rows
* :func:`int8_matmul`, :func:`int8_matmul_input_grad`,
  :func:`grouped_int8_matmul`, :func:`grouped_int8_matmul_input_grad` -- INT8
  weights with one scale per output channel

Mixtures of experts (likewise; with autograd in :mod:`.routing`):

* :func:`route_topk`, :func:`route_topk_grad` -- the experts of every token,
  their weights, and the places that bring the rows of one expert together
* :func:`dispatch_rows`, :func:`combine_rows` and their gradients -- rows to
  these places, and back as weighted sums

The ``*_into`` variants write into caller-provided (possibly aliasing)
outputs; the adapters use them to merge in place without a copy.
"""

from __future__ import annotations

import ctypes
import math
from typing import Any, NamedTuple

import torch

from . import _lib as L

__all__ = [
    "Routing",
    "combine_rows",
    "combine_rows_grad",
    "dequantize_float8",
    "GGUF_DEQUANT_TYPES",
    "dequantize_gguf",
    "dequantize_int8",
    "dequantize_mx",
    "dequantize_nvfp4",
    "dispatch_rows",
    "dispatch_rows_grad",
    "grouped_int8_matmul",
    "grouped_int8_matmul_input_grad",
    "grouped_matmul",
    "grouped_matmul_input_grad",
    "grouped_matmul_weight_grad",
    "grouped_mx_matmul",
    "grouped_mx_matmul_input_grad",
    "int8_matmul",
    "int8_matmul_input_grad",
    "merge_dense_lora_",
    "merge_float8_lora",
    "merge_float8_lora_into",
    "merge_int8_lora",
    "merge_int8_lora_into",
    "merge_mx_lora_",
    "merge_nvfp4_lora",
    "merge_nvfp4_lora_into",
    "merge_q8_0_lora",
    "mx_matmul",
    "mx_matmul_input_grad",
    "requantize_float8",
    "requantize_int8",
    "requantize_mx",
    "requantize_nvfp4",
    "requantize_q8_0",
    "route_topk",
    "route_topk_grad",
]

GGML_Q8_0 = 8
_Q8_0_BLOCK, _Q8_0_BYTES = 32, 34
_FACTOR_DTYPES = (torch.bfloat16, torch.float16)


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _run(name: str, device: torch.device, ws_bytes: int, *args: object) -> None:
    """Call one C entry point with a fresh workspace on the current stream.

    The workspace comes from torch's caching allocator on the same stream, so
    releasing it after the (asynchronous) launch is stream-ordered.
    """
    entry = getattr(L.lib(), name)
    with L.on_device(device):
        ws = L.workspace(ws_bytes, device)
        rc = entry(*args, L.aligned_ptr(ws), ws_bytes, L.stream_ptr(device))
    if rc:
        L.check(rc)


def _factors(b: torch.Tensor, a: torch.Tensor, rows: int, cols: int, label: str) -> tuple[torch.Tensor, torch.Tensor]:
    if b.ndim != 2 or a.ndim != 2:
        raise ValueError(f"{label} merge expects rank-two tensors.")
    if b.dtype is not a.dtype:
        raise ValueError(f"{label} merge requires matching LoRA factor dtypes.")
    if b.dtype not in _FACTOR_DTYPES:
        raise ValueError(f"{label} HIP merge supports bfloat16 and float16 LoRA factors, got {b.dtype}.")
    rank = a.shape[0]
    if rows == 0 or cols == 0 or rank == 0:
        raise ValueError(f"{label} merge requires non-empty weight and factors.")
    if tuple(b.shape) != (rows, rank) or a.shape[1] != cols:
        raise ValueError(f"LoRA factors do not match the {label} weight shape.")
    if rank > 64:
        raise ValueError(f"{label} HIP merge supports LoRA rank up to 64, got {rank}.")
    return b.contiguous(), a.contiguous()


def _same_device(label: str, *tensors: torch.Tensor | None) -> torch.device:
    first = tensors[0]
    assert first is not None
    if first.device.type != "cuda":
        raise ValueError(f"{label} HIP merge requires GPU tensors.")
    for t in tensors[1:]:
        if t is not None and t.device != first.device:
            raise ValueError(f"{label} HIP merge requires all tensors on one GPU device.")
    return first.device


# ---------------------------------------------------------------------------
# INT8
# ---------------------------------------------------------------------------
def _group_ok(cols: int, group: int) -> bool:
    """Per-group sizes the group kernels take: 16, 32 or a multiple of 64, dividing the columns."""
    return 0 < group < cols and cols % group == 0 and (group in (16, 32) or group % 64 == 0)


def _int8_group(shape: tuple[int, int], block_size: tuple[int, ...]) -> int:
    """Elements per qparam: per-tensor, per-row or per-group (1, g) layouts (P/_triton_int8_lora.py:251-264)."""
    rows, cols = shape
    block_size = tuple(block_size)
    if block_size == (rows, cols):
        return rows * cols
    if block_size == (1, cols):
        return cols
    if len(block_size) == 2 and block_size[0] == 1 and _group_ok(cols, block_size[1]):
        return block_size[1]
    raise ValueError(
        "HIP INT8 merge supports two-dimensional per-tensor, per-row and per-group layouts (group 16, 32 or a "
        f"multiple of 64 dividing the columns), got shape {shape} with block size {block_size}."
    )


def _qparam_shape(shape: tuple[int, int], group: int) -> tuple[int, int]:
    rows, cols = shape
    if group == rows * cols and group != cols:
        return (1, 1)
    return (rows, cols // group)


def merge_int8_lora_into(
    qdata: torch.Tensor, scale: torch.Tensor, zero_point: torch.Tensor | None, block_size: tuple[int, ...],
    b: torch.Tensor, a: torch.Tensor, strength: float, *, asymmetric: bool, reduce_range: bool,
    rounding_seed: int | None, out_qdata: torch.Tensor, out_scale: torch.Tensor, out_zero_point: torch.Tensor | None,
) -> None:
    device = _same_device("INT8", qdata, scale, b, a, zero_point)
    if qdata.dtype is not torch.int8:
        raise ValueError(f"HIP INT8 merge requires int8 weight storage, got {qdata.dtype}.")
    if qdata.ndim != 2:
        raise ValueError("HIP INT8 merge expects rank-two tensors.")
    if scale.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"HIP INT8 merge supports float32 and bfloat16 scales, got {scale.dtype}.")
    rows, cols = qdata.shape
    b, a = _factors(b, a, rows, cols, "INT8")
    group = _int8_group((rows, cols), block_size)
    nq = rows * cols // group
    if scale.numel() != nq:
        raise ValueError("INT8 scale shape does not match the quantization block layout.")
    if zero_point is not None and (zero_point.dtype is not torch.int8 or zero_point.numel() != nq):
        raise ValueError("INT8 zero-point storage does not match the quantization blocks.")
    for t in (qdata, scale, zero_point, out_qdata, out_scale, out_zero_point):
        if t is not None and not t.is_contiguous():
            raise ValueError("HIP INT8 merge requires contiguous storage.")
    lora = L.lora_struct(b, a, strength)
    rnd = L.rounding_struct(rounding_seed)
    ws_bytes = L.workspace_size(rows, cols, a.shape[0])
    _run("lm_int8_merge", device, ws_bytes,
         _ptr(qdata), _ptr(scale), _ptr(zero_point), _ptr(out_qdata), _ptr(out_scale), _ptr(out_zero_point),
         rows, cols, group, L.torch_dtype_id(scale.dtype), int(asymmetric), int(reduce_range),
         ctypes.byref(lora), ctypes.byref(rnd))


def merge_int8_lora(
    qdata: torch.Tensor, scale: torch.Tensor, zero_point: torch.Tensor | None, block_size: tuple[int, int],
    b: torch.Tensor, a: torch.Tensor, strength: float, *, asymmetric: bool, reduce_range: bool,
    rounding_seed: int | None = None,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Return raw affine-INT8 buffers after one LoRA merge (P/_triton_int8_lora.py:267-279)."""
    qdata = qdata.contiguous()
    scale = scale.contiguous()
    zero_point = None if zero_point is None else zero_point.contiguous()
    out_q = torch.empty_like(qdata)
    out_s = torch.empty_like(scale)
    out_z = torch.empty(scale.shape, device=scale.device, dtype=torch.int8)
    merge_int8_lora_into(qdata, scale, zero_point, block_size, b, a, strength, asymmetric=asymmetric,
                         reduce_range=reduce_range, rounding_seed=rounding_seed, out_qdata=out_q, out_scale=out_s,
                         out_zero_point=out_z)
    return out_q, out_s, out_z


def requantize_int8(dense: torch.Tensor, block_size: tuple[int, int], *, scale_dtype: torch.dtype = torch.float32,
                    asymmetric: bool = False, reduce_range: bool = False, rounding_seed: int | None = None
                    ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Encode a dense bf16/fp16 tensor with the fused INT8 requant kernel."""
    device = _same_device("INT8", dense)
    dense = dense.contiguous()
    rows, cols = dense.shape
    group = _int8_group((rows, cols), block_size)
    nq = rows * cols // group
    qshape = _qparam_shape((rows, cols), group)
    out_q = torch.empty((rows, cols), device=device, dtype=torch.int8)
    out_s = torch.empty(qshape, device=device, dtype=scale_dtype)
    out_z = torch.empty(qshape, device=device, dtype=torch.int8)
    assert out_s.numel() == nq
    rnd = L.rounding_struct(rounding_seed)
    ws_bytes = L.workspace_size(rows, cols, 0)
    _run("lm_int8_requant", device, ws_bytes, _ptr(dense), L.torch_dtype_id(dense.dtype), _ptr(out_q), _ptr(out_s),
         _ptr(out_z), rows, cols, group, L.torch_dtype_id(scale_dtype), int(asymmetric), int(reduce_range),
         ctypes.byref(rnd))
    return out_q, out_s, out_z


def dequantize_int8(qdata: torch.Tensor, scale: torch.Tensor, zero_point: torch.Tensor | None,
                    block_size: tuple[int, int], *, dtype: torch.dtype = torch.bfloat16,
                    lora: tuple[torch.Tensor, torch.Tensor, float] | None = None) -> torch.Tensor:
    """Dense INT8 dequantize, or dequantize + LoRA merge without requant when ``lora`` is given."""
    device = _same_device("INT8", qdata, scale)
    qdata = qdata.contiguous()
    rows, cols = qdata.shape
    group = _int8_group((rows, cols), block_size)
    out = torch.empty((rows, cols), device=device, dtype=dtype)
    lora_s, rank = None, 0
    if lora is not None:
        b, a = _factors(lora[0], lora[1], rows, cols, "INT8")
        lora_s, rank = L.lora_struct(b, a, lora[2]), a.shape[0]
    ws_bytes = L.workspace_size(rows, cols, rank)
    _run("lm_int8_dequant", device, ws_bytes, _ptr(qdata), _ptr(scale.contiguous()),
         _ptr(None if zero_point is None else zero_point.contiguous()), rows, cols, group,
         L.torch_dtype_id(scale.dtype), None if lora_s is None else ctypes.byref(lora_s), _ptr(out),
         L.torch_dtype_id(dtype))
    return out


# ---------------------------------------------------------------------------
# scaled FP8
# ---------------------------------------------------------------------------
def _fp8_group(shape: tuple[int, int], block_size: tuple[int, ...], scale: torch.Tensor) -> int:
    """Elements per scale: per-row, per-tensor or per-group (1, g) layouts (P/float8_adapter.py:63-98)."""
    rows, cols = shape
    block_size = tuple(block_size)
    if block_size == (1, cols):
        if tuple(scale.shape) != (rows, 1):
            raise ValueError(f"HIP per-row scaled-FP8 merge expects scale shape {(rows, 1)}, got {tuple(scale.shape)}.")
        return cols
    if block_size == (rows, cols):
        if scale.numel() != 1:
            raise ValueError("HIP per-tensor scaled-FP8 merge expects one scale.")
        return rows * cols
    if len(block_size) == 2 and block_size[0] == 1 and _group_ok(cols, block_size[1]):
        g = block_size[1]
        if tuple(scale.shape) != (rows, cols // g):
            raise ValueError(f"HIP per-group scaled-FP8 merge expects scale shape {(rows, cols // g)}, "
                             f"got {tuple(scale.shape)}.")
        return g
    raise ValueError(
        "HIP scaled-FP8 merge supports per-row, per-tensor and per-group layouts (group 16, 32 or a multiple of 64 "
        f"dividing the columns), got block_size={block_size!r}."
    )


def merge_float8_lora_into(qdata: torch.Tensor, scale: torch.Tensor, block_size: tuple[int, ...], b: torch.Tensor,
                           a: torch.Tensor, strength: float, *, rounding_seed: int | None, out_qdata: torch.Tensor,
                           out_scale: torch.Tensor) -> None:
    device = _same_device("scaled-FP8", qdata, scale, b, a)
    if qdata.dtype not in (torch.float8_e4m3fn, torch.float8_e5m2):
        raise ValueError(f"HIP scaled-FP8 merge supports E4M3FN and E5M2 storage, got {qdata.dtype}.")
    if qdata.ndim != 2:
        raise ValueError("HIP scaled-FP8 merge expects rank-two tensors.")
    if scale.dtype is not torch.float32:
        raise ValueError("HIP scaled-FP8 merge expects float32 scales.")
    rows, cols = qdata.shape
    b, a = _factors(b, a, rows, cols, "scaled-FP8")
    group = _fp8_group((rows, cols), block_size, scale)
    lora = L.lora_struct(b, a, strength)
    rnd = L.rounding_struct(rounding_seed)
    ws_bytes = L.workspace_size(rows, cols, a.shape[0])
    _run("lm_fp8_merge", device, ws_bytes, _ptr(qdata), _ptr(scale), _ptr(out_qdata), _ptr(out_scale), rows, cols,
         group, L.torch_dtype_id(qdata.dtype), ctypes.byref(lora), ctypes.byref(rnd))


def merge_float8_lora(qdata: torch.Tensor, scale: torch.Tensor, block_size: tuple[int, ...], b: torch.Tensor,
                      a: torch.Tensor, strength: float, *, rounding_seed: int | None = None
                      ) -> tuple[torch.Tensor, torch.Tensor]:
    """Return raw scaled-FP8 buffers after one merge (P/_triton_float8_lora.py:486-495)."""
    qdata = qdata.contiguous()
    scale = scale.contiguous()
    out_q = torch.empty_like(qdata)
    out_s = torch.empty_like(scale)
    merge_float8_lora_into(qdata, scale, block_size, b, a, strength, rounding_seed=rounding_seed, out_qdata=out_q,
                           out_scale=out_s)
    return out_q, out_s


def requantize_float8(dense: torch.Tensor, block_size: tuple[int, int], *, fp8_dtype: torch.dtype = torch.float8_e4m3fn,
                      rounding_seed: int | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    device = _same_device("scaled-FP8", dense)
    dense = dense.contiguous()
    rows, cols = dense.shape
    block_size = tuple(block_size)
    if block_size == (1, cols):
        sshape = (rows, 1)
    elif block_size == (rows, cols):
        sshape = (1, 1)
    elif len(block_size) == 2 and block_size[0] == 1 and block_size[1] > 0 and cols % block_size[1] == 0:
        sshape = (rows, cols // block_size[1])
    else:
        sshape = (1, 1)  # rejected by _fp8_group below
    out_q = torch.empty((rows, cols), device=device, dtype=fp8_dtype)
    out_s = torch.empty(sshape, device=device, dtype=torch.float32)
    group = _fp8_group((rows, cols), block_size, out_s)
    rnd = L.rounding_struct(rounding_seed)
    ws_bytes = L.workspace_size(rows, cols, 0)
    _run("lm_fp8_requant", device, ws_bytes, _ptr(dense), L.torch_dtype_id(dense.dtype), _ptr(out_q), _ptr(out_s),
         rows, cols, group, L.torch_dtype_id(fp8_dtype), ctypes.byref(rnd))
    return out_q, out_s


def dequantize_float8(qdata: torch.Tensor, scale: torch.Tensor, block_size: tuple[int, int], *,
                      dtype: torch.dtype = torch.bfloat16,
                      lora: tuple[torch.Tensor, torch.Tensor, float] | None = None) -> torch.Tensor:
    device = _same_device("scaled-FP8", qdata, scale)
    qdata = qdata.contiguous()
    rows, cols = qdata.shape
    group = _fp8_group((rows, cols), block_size, scale)
    out = torch.empty((rows, cols), device=device, dtype=dtype)
    lora_s, rank = None, 0
    if lora is not None:
        b, a = _factors(lora[0], lora[1], rows, cols, "scaled-FP8")
        lora_s, rank = L.lora_struct(b, a, lora[2]), a.shape[0]
    ws_bytes = L.workspace_size(rows, cols, rank)
    _run("lm_fp8_dequant", device, ws_bytes, _ptr(qdata), _ptr(scale.contiguous()), rows, cols, group,
         L.torch_dtype_id(qdata.dtype), None if lora_s is None else ctypes.byref(lora_s), _ptr(out),
         L.torch_dtype_id(dtype))
    return out


# ---------------------------------------------------------------------------
# NVFP4
# ---------------------------------------------------------------------------
def _nvfp4_scale_shape(rows: int, cols: int, swizzled: bool) -> tuple[int, int]:
    if swizzled:
        return (rows + 127) // 128 * 32, (cols + 63) // 64 * 16
    return rows, cols // 16


def merge_nvfp4_lora_into(qdata: torch.Tensor, scale: torch.Tensor, per_tensor_scale: torch.Tensor | None,
                          block_size: int, is_swizzled_scales: bool, b: torch.Tensor, a: torch.Tensor, strength: float,
                          *, rounding_seed: int | None, out_qdata: torch.Tensor, out_scale: torch.Tensor,
                          out_per_tensor_scale: torch.Tensor | None) -> None:
    device = _same_device("NVFP4", qdata, scale, b, a, per_tensor_scale)
    if qdata.dtype is not torch.uint8:
        raise ValueError(f"HIP NVFP4 merge expects packed uint8 data, got {qdata.dtype}.")
    if scale.dtype is not torch.float8_e4m3fn:
        raise ValueError("HIP NVFP4 merge expects E4M3FN block scales.")
    if qdata.ndim != 2 or scale.ndim != 2:
        raise ValueError("HIP NVFP4 merge expects rank-two tensors.")
    if not qdata.is_contiguous() or not scale.is_contiguous():
        raise ValueError("HIP NVFP4 merge requires contiguous packed data and scales.")
    if block_size != 16:
        raise ValueError("HIP NVFP4 merge requires block_size=16.")
    rows, packed_cols = qdata.shape
    cols = packed_cols * 2
    if packed_cols % 8 != 0:
        raise ValueError("HIP NVFP4 merge requires columns divisible by 16.")
    b, a = _factors(b, a, rows, cols, "NVFP4")
    if tuple(scale.shape) != _nvfp4_scale_shape(rows, cols, is_swizzled_scales):
        raise ValueError("NVFP4 scale shape does not match its swizzle metadata.")
    if per_tensor_scale is not None and (per_tensor_scale.dtype is not torch.float32 or per_tensor_scale.numel() != 1):
        raise ValueError("HIP NVFP4 merge expects one float32 per-tensor scale.")
    lora = L.lora_struct(b, a, strength)
    rnd = L.rounding_struct(rounding_seed)
    ws_bytes = L.workspace_size(rows, cols, a.shape[0])
    _run("lm_nvfp4_merge", device, ws_bytes, _ptr(qdata), _ptr(scale.view(torch.uint8)), _ptr(per_tensor_scale),
         _ptr(out_qdata), _ptr(out_scale.view(torch.uint8)), _ptr(out_per_tensor_scale), rows, cols,
         int(is_swizzled_scales), ctypes.byref(lora), ctypes.byref(rnd))


def merge_nvfp4_lora(qdata: torch.Tensor, scale: torch.Tensor, per_tensor_scale: torch.Tensor | None, block_size: int,
                     is_swizzled_scales: bool, b: torch.Tensor, a: torch.Tensor, strength: float, *,
                     rounding_seed: int | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor | None]:
    """Return packed NVFP4 buffers after one merge (P/_triton_nvfp4_lora.py:515-526)."""
    out_q = torch.empty_like(qdata)
    out_s = torch.zeros_like(scale)
    out_pts = None if per_tensor_scale is None else torch.empty_like(per_tensor_scale)
    merge_nvfp4_lora_into(qdata, scale, per_tensor_scale, block_size, is_swizzled_scales, b, a, strength,
                          rounding_seed=rounding_seed, out_qdata=out_q, out_scale=out_s,
                          out_per_tensor_scale=out_pts)
    return out_q, out_s, out_pts


def requantize_nvfp4(dense: torch.Tensor, *, two_level: bool = True, swizzled: bool = False,
                     rounding_seed: int | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor | None]:
    device = _same_device("NVFP4", dense)
    dense = dense.contiguous()
    rows, cols = dense.shape
    out_q = torch.empty((rows, cols // 2), device=device, dtype=torch.uint8)
    out_s = torch.zeros(_nvfp4_scale_shape(rows, cols, swizzled), device=device, dtype=torch.float8_e4m3fn)
    out_pts = torch.empty((), device=device, dtype=torch.float32) if two_level else None
    rnd = L.rounding_struct(rounding_seed)
    ws_bytes = L.workspace_size(rows, cols, 0)
    _run("lm_nvfp4_requant", device, ws_bytes, _ptr(dense), L.torch_dtype_id(dense.dtype), _ptr(out_q),
         _ptr(out_s.view(torch.uint8)), _ptr(out_pts), rows, cols, int(swizzled), ctypes.byref(rnd))
    return out_q, out_s, out_pts


def dequantize_nvfp4(qdata: torch.Tensor, scale: torch.Tensor, per_tensor_scale: torch.Tensor | None, *,
                     swizzled: bool = False, dtype: torch.dtype = torch.bfloat16,
                     lora: tuple[torch.Tensor, torch.Tensor, float] | None = None) -> torch.Tensor:
    device = _same_device("NVFP4", qdata, scale)
    rows, cols = qdata.shape[0], qdata.shape[1] * 2
    out = torch.empty((rows, cols), device=device, dtype=dtype)
    lora_s, rank = None, 0
    if lora is not None:
        b, a = _factors(lora[0], lora[1], rows, cols, "NVFP4")
        lora_s, rank = L.lora_struct(b, a, lora[2]), a.shape[0]
    ws_bytes = L.workspace_size(rows, cols, rank)
    _run("lm_nvfp4_dequant", device, ws_bytes, _ptr(qdata.contiguous()), _ptr(scale.contiguous().view(torch.uint8)),
         _ptr(per_tensor_scale), rows, cols, int(swizzled), None if lora_s is None else ctypes.byref(lora_s),
         _ptr(out), L.torch_dtype_id(dtype))
    return out


# ---------------------------------------------------------------------------
# MX
# ---------------------------------------------------------------------------
_FP4_DTYPE = getattr(torch, "float4_e2m1fn_x2", None)
_E8M0_DTYPE = getattr(torch, "float8_e8m0fnu", None)


def _mx_format(elem_dtype: object) -> int:
    if elem_dtype is torch.float8_e4m3fn:
        return L.LM_E4M3
    if elem_dtype is torch.float8_e5m2:
        return L.LM_E5M2
    if elem_dtype is _FP4_DTYPE and _FP4_DTYPE is not None:
        return L.LM_E2M1
    raise ValueError(f"HIP MX merge does not support element dtype {elem_dtype}.")


def _mx_scale_shape(rows: int, cols: int, swizzled: bool) -> tuple[int, int]:
    if not swizzled:
        return rows, cols // 32
    return (rows + 127) // 128 * 32, (cols + 127) // 128 * 16


def merge_mx_lora_(qdata: torch.Tensor, scale: torch.Tensor, elem_dtype: torch.dtype, block_size: int,
                   orig_dtype: torch.dtype, b: torch.Tensor, a: torch.Tensor, strength: float, *, scaling_mode: int,
                   swizzled: bool, rounding_seed: int | None = None) -> None:
    """Merge one staged update directly into raw MX storage (P/_triton_mx_lora.py:333-346)."""
    device = _same_device("MX", qdata, scale, b, a)
    if qdata.ndim != 2 or scale.ndim != 2 or b.ndim != 2 or a.ndim != 2:
        raise ValueError("HIP MX merge expects rank-two tensors.")
    if block_size != 32:
        raise ValueError("HIP MX merge supports block size 32.")
    if b.dtype is not a.dtype or b.dtype is not orig_dtype:
        raise ValueError("HIP MX merge requires factors in the weight's original dtype.")
    if orig_dtype is not torch.bfloat16:
        raise ValueError(f"HIP MX merge supports bfloat16 weights and factors, got {orig_dtype}.")
    if not qdata.is_contiguous() or not scale.is_contiguous():
        raise ValueError("HIP MX merge requires contiguous MX storage.")
    if scaling_mode not in (0, 1, 2, 3):
        raise ValueError(f"Unsupported MX scaling mode id {scaling_mode}.")
    rows, rank = b.shape
    if a.shape[0] != rank:
        raise ValueError("LoRA factor inner dimensions do not match.")
    cols = a.shape[1]
    if cols % 32 != 0:
        raise ValueError("HIP MX merge requires columns divisible by 32.")
    fmt = _mx_format(elem_dtype)
    expected_q = (rows, cols // 2) if fmt == L.LM_E2M1 else (rows, cols)
    if tuple(qdata.shape) != expected_q:
        raise ValueError("MX qdata shape does not match its element format and LoRA factors.")
    if tuple(scale.shape) != _mx_scale_shape(rows, cols, swizzled):
        raise ValueError("MX scale shape does not match its block layout.")
    if _E8M0_DTYPE is not None and scale.dtype is not _E8M0_DTYPE and scale.dtype is not torch.uint8:
        raise ValueError(f"HIP MX merge expects E8M0 scales, got {scale.dtype}.")
    b, a = _factors(b, a, rows, cols, "MX")
    lora = L.lora_struct(b, a, strength)
    rnd = L.rounding_struct(rounding_seed)
    ws_bytes = L.workspace_size(rows, cols, rank)
    _run("lm_mx_merge", device, ws_bytes, _ptr(qdata), _ptr(scale), rows, cols, fmt, int(scaling_mode),
         int(swizzled), ctypes.byref(lora), ctypes.byref(rnd))


def requantize_mx(dense: torch.Tensor, elem_dtype: torch.dtype, *, scaling_mode: int = 0, swizzled: bool = False,
                  rounding_seed: int | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    device = _same_device("MX", dense)
    dense = dense.contiguous()
    rows, cols = dense.shape
    fmt = _mx_format(elem_dtype)
    out_q = torch.empty((rows, cols // 2) if fmt == L.LM_E2M1 else (rows, cols), device=device,
                        dtype=torch.uint8 if fmt == L.LM_E2M1 else elem_dtype)
    out_s = torch.zeros(_mx_scale_shape(rows, cols, swizzled), device=device, dtype=torch.uint8)
    rnd = L.rounding_struct(rounding_seed)
    ws_bytes = L.workspace_size(rows, cols, 0)
    _run("lm_mx_requant", device, ws_bytes, _ptr(dense), L.torch_dtype_id(dense.dtype), _ptr(out_q), _ptr(out_s),
         rows, cols, fmt, int(scaling_mode), int(swizzled), ctypes.byref(rnd))
    return out_q, out_s


def dequantize_mx(qdata: torch.Tensor, scale: torch.Tensor, elem_dtype: torch.dtype, cols: int, *,
                  swizzled: bool = False, dtype: torch.dtype = torch.bfloat16,
                  lora: tuple[torch.Tensor, torch.Tensor, float] | None = None) -> torch.Tensor:
    device = _same_device("MX", qdata, scale)
    rows = qdata.shape[0]
    fmt = _mx_format(elem_dtype)
    out = torch.empty((rows, cols), device=device, dtype=dtype)
    lora_s, rank = None, 0
    if lora is not None:
        b, a = _factors(lora[0], lora[1], rows, cols, "MX")
        lora_s, rank = L.lora_struct(b, a, lora[2]), a.shape[0]
    ws_bytes = L.workspace_size(rows, cols, rank)
    _run("lm_mx_dequant", device, ws_bytes, _ptr(qdata.contiguous()), _ptr(scale.contiguous()), rows, cols, fmt,
         int(swizzled), None if lora_s is None else ctypes.byref(lora_s), _ptr(out), L.torch_dtype_id(dtype))
    return out


# ---------------------------------------------------------------------------
# GGUF Q8_0
# ---------------------------------------------------------------------------
def q8_0_logical_shape(packed_shape: tuple[int, ...]) -> tuple[int, ...]:
    """P/gguf_dequant.py:297-300 for Q8_0: 34 bytes hold 32 elements."""
    return (*packed_shape[:-1], packed_shape[-1] // _Q8_0_BYTES * _Q8_0_BLOCK)


def merge_q8_0_lora(packed: torch.Tensor, b: torch.Tensor, a: torch.Tensor, strength: float, *,
                    rounding_seed: int | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Merge into GGUF Q8_0 bytes: dequantize (bf16), add strength*B@A, re-block per ggml."""
    device = _same_device("Q8_0", packed, b, a)
    if packed.dtype is not torch.uint8 or packed.ndim != 2:
        raise ValueError("HIP Q8_0 merge expects rank-two uint8 GGUF bytes.")
    if packed.shape[1] % _Q8_0_BYTES != 0:
        raise ValueError("Q8_0 rows must hold whole 34-byte blocks.")
    packed = packed.contiguous()
    rows, cols = q8_0_logical_shape(tuple(packed.shape))
    b, a = _factors(b, a, rows, cols, "Q8_0")
    out = torch.empty_like(packed) if out is None else out
    lora = L.lora_struct(b, a, strength)
    rnd = L.rounding_struct(rounding_seed)
    ws_bytes = L.workspace_size(rows, cols, a.shape[0])
    _run("lm_q8_0_merge", device, ws_bytes, _ptr(packed), _ptr(out), rows, cols, ctypes.byref(lora),
         ctypes.byref(rnd))
    return out


def requantize_q8_0(dense: torch.Tensor, *, rounding_seed: int | None = None) -> torch.Tensor:
    device = _same_device("Q8_0", dense)
    dense = dense.contiguous()
    rows, cols = dense.shape
    if cols % _Q8_0_BLOCK != 0:
        raise ValueError("Q8_0 requires columns divisible by 32.")
    out = torch.empty((rows, cols // _Q8_0_BLOCK * _Q8_0_BYTES), device=device, dtype=torch.uint8)
    rnd = L.rounding_struct(rounding_seed)
    ws_bytes = L.workspace_size(rows, cols, 0)
    _run("lm_q8_0_requant", device, ws_bytes, _ptr(dense), L.torch_dtype_id(dense.dtype), _ptr(out), rows, cols,
         ctypes.byref(rnd))
    return out


# block elements and bytes of every type P/gguf_dequant.py:278-294 dispatches
# (ggml block structs; keys are gguf.GGMLQuantizationType values)
GGUF_DEQUANT_TYPES: dict[int, tuple[int, int]] = {
    0: (1, 4), 1: (1, 2), 30: (1, 2),                      # F32, F16, BF16
    2: (32, 18), 3: (32, 20), 6: (32, 22), 7: (32, 24),    # Q4_0, Q4_1, Q5_0, Q5_1
    8: (32, 34), 20: (32, 18),                             # Q8_0, IQ4_NL
    10: (256, 84), 11: (256, 110), 12: (256, 144),         # Q2_K, Q3_K, Q4_K
    13: (256, 176), 14: (256, 210), 23: (256, 136),        # Q5_K, Q6_K, IQ4_XS
}
_GGUF_OUT_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def dequantize_gguf(data: torch.Tensor, quant_type: int, *, dtype: torch.dtype = torch.bfloat16,
                    lora: tuple[torch.Tensor, torch.Tensor, float] | None = None) -> torch.Tensor:
    """GGUF dequantize on the GPU (P/gguf_dequant.py:303-331) for every type
    the reference dispatches; ``lora`` (Q8_0 only) adds strength*B@A."""
    sizes = GGUF_DEQUANT_TYPES.get(int(quant_type))
    if sizes is None:
        raise NotImplementedError(f"Unsupported GGUF quant type: {quant_type!r}")
    if dtype not in _GGUF_OUT_DTYPES:
        raise ValueError(f"HIP GGUF dequant computes in bf16, fp16 or fp32, not {dtype}.")
    block, nbytes = sizes
    device = _same_device("GGUF", data)
    if data.ndim == 0:
        raise ValueError("GGUF data must have at least one dimension.")
    shape = (*data.shape[:-1], data.shape[-1] // nbytes * block)  # P/gguf_dequant.py:297-300 on data.shape
    raw = data.view(torch.uint8)
    if raw.shape[-1] % nbytes != 0:
        raise ValueError(f"GGUF rows must hold whole {nbytes}-byte blocks of type {quant_type}.")
    raw = raw.contiguous()
    elements = raw.numel() // nbytes * block
    if math.prod(shape) != elements:
        raise ValueError(f"GGUF bytes of shape {tuple(data.shape)} do not give a tensor of shape {shape}.")
    out = torch.empty(shape, device=device, dtype=dtype)
    if elements == 0:
        return out
    cols = shape[-1]
    rows = elements // cols
    lora_s, rank = None, 0
    if lora is not None:
        if int(quant_type) != GGML_Q8_0:
            raise ValueError("GGUF dequant with LoRA factors supports Q8_0 only.")
        b, a = _factors(lora[0], lora[1], rows, cols, "GGUF")
        lora_s, rank = L.lora_struct(b, a, lora[2]), a.shape[0]
    ws_bytes = L.workspace_size(rows, cols, rank) if lora is not None else 0
    _run("lm_gguf_dequant", device, ws_bytes, _ptr(raw), int(quant_type), rows, cols,
         None if lora_s is None else ctypes.byref(lora_s), _ptr(out), L.torch_dtype_id(dtype))
    return out


# ---------------------------------------------------------------------------
# plain dense weight
# ---------------------------------------------------------------------------
def merge_dense_lora_(weight: torch.Tensor, b: torch.Tensor, a: torch.Tensor, strength: float) -> None:
    """``weight.addmm_(b, a, alpha=strength)`` for bf16/fp16 weights on the GPU."""
    device = _same_device("dense", weight, b, a)
    if weight.ndim != 2 or weight.stride(1) != 1:
        raise ValueError("HIP dense merge expects a row-major rank-two weight.")
    if weight.dtype is not b.dtype:
        raise ValueError("HIP dense merge requires factors in the weight dtype.")
    rows, cols = weight.shape
    b, a = _factors(b, a, rows, cols, "dense")
    lora = L.lora_struct(b, a, strength)
    ws_bytes = L.workspace_size(rows, cols, a.shape[0])
    _run("lm_dense_merge", device, ws_bytes, _ptr(weight), rows, cols, weight.stride(0), ctypes.byref(lora))


# ---------------------------------------------------------------------------
# Products with stored weights
# ---------------------------------------------------------------------------
_MAX_EXPERTS = 1024
_MAX_INT8_COLS = 132104  # products of codes, 127 * 128 each, add up below 2^31


_LAYERS = "mx_linear, int8_linear, grouped_linear, route_experts, dispatch_experts or combine_experts"


# (These calls are as short as 5 us on the GPU: the checks below look at each tensor once.)
def _raw(label: str, *tensors: torch.Tensor) -> None:
    """Refuse what would lose a gradient: the result has no graph, the layers of :mod:`.linear` give it one."""
    for t in tensors:
        if t.requires_grad and torch.is_grad_enabled():
            raise NotImplementedError(f"{label} records no gradient; call {_LAYERS}, or run it under torch.no_grad().")


def _rows(label: str, x: torch.Tensor, cols: int) -> tuple[torch.Tensor, int, int]:
    """``x`` [..., cols] as [rows, cols] whose rows are contiguous, the number of rows, and their stride."""
    shape = x.shape
    if not shape or shape[-1] != cols:
        raise ValueError(f"{label}: expected rows of {cols} elements, got shape {tuple(shape)}.")
    if x.dtype not in _FACTOR_DTYPES:
        raise ValueError(f"{label} supports bfloat16 and float16 rows, got {x.dtype}.")
    if x.requires_grad:
        _raw(label, x)
    if len(shape) != 2:
        x = x.reshape(-1, cols)
        shape = x.shape
    rows = shape[0]
    if x.is_contiguous():
        return x, rows, cols
    stride, step = x.stride()
    if (cols > 1 and step != 1) or (rows > 1 and stride < cols):
        return x.contiguous(), rows, cols
    return x, rows, stride if rows > 1 else cols  # (the stride of a single row may be anything)


def _on_gpu(label: str, first: torch.Tensor, *others: torch.Tensor | None) -> None:
    """All tensors on the GPU of the first."""
    if not first.is_cuda:
        raise ValueError(f"{label} requires GPU tensors.")
    index = first.get_device()
    for t in others:
        if t is not None and t.get_device() != index:
            raise ValueError(f"{label} requires all tensors on one GPU device.")


def _ends(label: str, ends: torch.Tensor, experts: int) -> torch.Tensor:
    if ends.dtype is not torch.int32 or ends.ndim != 1 or ends.shape[0] != experts:
        raise ValueError(f"{label}: ends must be int32 [{experts}] (the end of each group's rows), got "
                         f"{ends.dtype} {tuple(ends.shape)}.")
    if not 1 <= experts <= _MAX_EXPERTS:
        raise ValueError(f"{label} takes 1 to {_MAX_EXPERTS} groups, got {experts}.")
    return ends.contiguous()


def _mx_weight(label: str, qdata: torch.Tensor, scale: torch.Tensor, swizzled: bool, stacked: bool) -> L.WeightStruct:
    """Check MXFP4 storage ([rows, cols/2], stacked: [groups, rows, cols/2]) and describe it."""
    shape, sshape = qdata.shape, scale.shape
    if len(shape) != 2 + stacked or len(sshape) != 2 + stacked:
        raise ValueError(f"{label} expects rank-{'three' if stacked else 'two'} MXFP4 codes and scales.")
    if qdata.dtype is not torch.uint8 and qdata.dtype is not _FP4_DTYPE:
        raise ValueError(f"{label} expects packed uint8 MXFP4 codes, got {qdata.dtype}.")
    if scale.dtype is not torch.uint8 and scale.dtype is not _E8M0_DTYPE:
        raise ValueError(f"{label} expects E8M0 scales, got {scale.dtype}.")
    if not qdata.is_contiguous() or not scale.is_contiguous():
        raise ValueError(f"{label} requires contiguous MXFP4 storage.")
    rows, cols, groups = shape[-2], shape[-1] * 2, shape[0] if stacked else 1
    if rows == 0 or cols == 0:
        raise ValueError(f"{label} requires a non-empty weight.")
    if cols % 32 != 0:
        raise ValueError(f"{label} requires columns divisible by 32.")
    if sshape[-2:] != _mx_scale_shape(rows, cols, swizzled) or (stacked and sshape[0] != groups):
        raise ValueError(f"{label}: the scale shape {tuple(sshape)} does not match its block layout.")
    return L.WeightStruct(qdata.data_ptr(), scale.data_ptr(), rows, cols, L.LM_E2M1, swizzled, groups, 0)


def _launch(entry: Any, index: int, ws_bytes: int, device: torch.device, *args: object) -> None:
    """Call one C entry on GPU ``index`` with a workspace on the current stream."""
    if torch._C._cuda_getDevice() != index:
        with L.on_device(device):
            _launch(entry, index, ws_bytes, device, *args)
        return
    ws = L.aligned_ptr(keep := L.workspace(ws_bytes, device)) if ws_bytes else None
    rc = entry(*args, ws, ws_bytes, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        L.check(rc)
    if ws_bytes:
        del keep  # released in stream order


def _linear_forward(label: str, x: torch.Tensor, weight: L.WeightStruct, bias: torch.Tensor | None,
                    ends: torch.Tensor | None, activation_dtype: torch.dtype | None) -> torch.Tensor:
    n, k = weight.N, weight.K
    x2, t, ldx = _rows(label, x, k)
    dtype_id = input_id = L.torch_dtype_id(x.dtype)
    if activation_dtype is not None:
        if weight.dtype == L.LM_I8:
            if activation_dtype is not torch.int8:
                raise ValueError(f"{label} quantises its input to int8 only, got {activation_dtype}.")
            if k > _MAX_INT8_COLS:
                raise ValueError(f"{label}: 8-bit products take up to {_MAX_INT8_COLS} columns, got {k}.")
            input_id = L.LM_I8
        else:
            if activation_dtype is not _FP4_DTYPE or _FP4_DTYPE is None:
                raise ValueError(f"{label} quantises its input to float4_e2m1fn_x2 only, got {activation_dtype}.")
            input_id = L.LM_E2M1
    if bias is not None:
        if bias.dtype is not x.dtype or tuple(bias.shape) != (n,):
            raise ValueError(f"{label}: bias must be {x.dtype} [{n}], got {bias.dtype} {tuple(bias.shape)}.")
        _raw(label, bias)
        bias = bias.contiguous()
    y = x2.new_empty(t, n)
    if t:
        px = x2.data_ptr()
        ws_bytes = L.linear_workspace_size(0, t, ldx, 0, n, k, weight.experts, weight.dtype, input_id, not (px | weight.q) & 15)
        _launch(L.lib().lm_linear, x2.get_device(), ws_bytes, x2.device, px, ldx, weight, _ptr(bias), _ptr(ends), y.data_ptr(), t,
                dtype_id, input_id)
    return y if x.ndim == 2 else y.view(*x.shape[:-1], n)


def _linear_input_grad(label: str, dy: torch.Tensor, weight: L.WeightStruct, ends: torch.Tensor | None) -> torch.Tensor:
    n, k = weight.N, weight.K
    dy2, t, ldy = _rows(label, dy, n)
    dx = dy2.new_empty(t, k)
    if t:
        py = dy2.data_ptr()
        dtype_id = L.torch_dtype_id(dy.dtype)
        ws_bytes = L.linear_workspace_size(1, t, ldy, 0, n, k, weight.experts, weight.dtype, dtype_id, not (py | weight.q) & 15)
        _launch(L.lib().lm_linear_input_grad, dy2.get_device(), ws_bytes, dy2.device, py, ldy, weight, _ptr(ends), dx.data_ptr(),
                t, dtype_id)
    return dx if dy.ndim == 2 else dx.view(*dy.shape[:-1], k)


def mx_matmul(x: torch.Tensor, qdata: torch.Tensor, scale: torch.Tensor, *, swizzled: bool = False,
              bias: torch.Tensor | None = None, activation_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``x @ W.T + bias`` with ``W`` stored in MXFP4 (``qdata`` [out, in/2], ``scale`` as in :class:`MXWeight`).

    ``x`` [..., in] bfloat16 or float16; sums in fp32, rounded once to ``x.dtype``.  With
    ``activation_dtype=torch.float4_e2m1fn_x2`` ``x`` is quantised first, as :func:`requantize_mx` does it.
    Weights are exact for bfloat16 and for quantised inputs; float16 inputs see each weight rounded to float16
    (exact from 2^-23 to 49152 in magnitude, infinite above).
    """
    label = "MX product"
    _on_gpu(label, x, qdata, scale, bias)
    return _linear_forward(label, x, _mx_weight(label, qdata, scale, swizzled, False), bias, None, activation_dtype)


def mx_matmul_input_grad(dy: torch.Tensor, qdata: torch.Tensor, scale: torch.Tensor, *,
                         swizzled: bool = False) -> torch.Tensor:
    """``dy @ W``: the input gradient of :func:`mx_matmul` (straight through a quantised input).

    A float16 ``dy`` sees each weight rounded to float16, as there.
    """
    label = "MX product gradient"
    _on_gpu(label, dy, qdata, scale)
    return _linear_input_grad(label, dy, _mx_weight(label, qdata, scale, swizzled, False), None)


def _dense_stack(label: str, rows: torch.Tensor, weight: torch.Tensor) -> L.WeightStruct:
    shape = weight.shape
    if len(shape) != 3 or 0 in shape:
        raise ValueError(f"{label} expects a weight [groups, out, in], got {tuple(shape)}.")
    if weight.dtype is not rows.dtype:
        raise ValueError(f"{label} requires the weight in the rows' dtype {rows.dtype}, got {weight.dtype}.")
    if not weight.is_contiguous():
        raise ValueError(f"{label} requires a contiguous weight.")
    _raw(label, weight)
    return L.WeightStruct(weight.data_ptr(), None, shape[1], shape[2], L.torch_dtype_id(weight.dtype), 0, shape[0], 0)


def grouped_matmul(x: torch.Tensor, weight: torch.Tensor, ends: torch.Tensor) -> torch.Tensor:
    """Rows ``ends[e-1] : ends[e]`` of ``x`` [rows, in] times ``weight[e].T`` (``weight`` [groups, out, in]).

    ``ends`` int32 [groups] stays on the GPU (no synchronization); rows past the last end give zeros.
    """
    label = "Grouped product"
    _on_gpu(label, x, weight, ends)
    w = _dense_stack(label, x, weight)
    return _linear_forward(label, x, w, None, _ends(label, ends, w.experts), None)


def grouped_matmul_input_grad(dy: torch.Tensor, weight: torch.Tensor, ends: torch.Tensor) -> torch.Tensor:
    """The gradient of :func:`grouped_matmul` to ``x``; zeros for rows of no group."""
    label = "Grouped product gradient"
    _on_gpu(label, dy, weight, ends)
    w = _dense_stack(label, dy, weight)
    return _linear_input_grad(label, dy, w, _ends(label, ends, w.experts))


def grouped_matmul_weight_grad(dy: torch.Tensor, x: torch.Tensor, ends: torch.Tensor) -> torch.Tensor:
    """The gradient of :func:`grouped_matmul` to ``weight``: ``dy[group].T @ x[group]``, zeros for empty groups."""
    label = "Grouped product weight gradient"
    _on_gpu(label, dy, x, ends)
    if dy.ndim < 1 or x.ndim < 1 or dy.shape[:-1] != x.shape[:-1]:
        raise ValueError(f"{label}: dy {tuple(dy.shape)} and x {tuple(x.shape)} differ in their rows.")
    if dy.dtype is not x.dtype:
        raise ValueError(f"{label} requires dy and x in one dtype, got {dy.dtype} and {x.dtype}.")
    n, k = dy.shape[-1], x.shape[-1]
    if n == 0 or k == 0:
        raise ValueError(f"{label} requires non-empty rows.")
    (dy2, t, ldy), (x2, _, ldx) = _rows(label, dy, n), _rows(label, x, k)
    ends = _ends(label, ends, ends.shape[0] if ends.ndim == 1 else -1)
    e = ends.shape[0]
    dw = x2.new_empty((e, n, k))
    py, px, dtype_id = dy2.data_ptr(), x2.data_ptr(), L.torch_dtype_id(x.dtype)
    ws_bytes = L.linear_workspace_size(2, t, ldy, ldx, n, k, e, dtype_id, dtype_id, not (py | px) & 15)
    _launch(L.lib().lm_linear_weight_grad, x2.get_device(), ws_bytes, x2.device, py, ldy, px, ldx, ends.data_ptr(), dw.data_ptr(),
            t, n, k, e, dtype_id)
    return dw


def grouped_mx_matmul(x: torch.Tensor, qdata: torch.Tensor, scale: torch.Tensor, ends: torch.Tensor, *,
                      swizzled: bool = False, activation_dtype: torch.dtype | None = None) -> torch.Tensor:
    """:func:`grouped_matmul` with MXFP4 weights: ``qdata`` [groups, out, in/2], scales of each group's weight.

    Roundings as in :func:`mx_matmul`.
    """
    label = "Grouped MX product"
    _on_gpu(label, x, qdata, scale, ends)
    w = _mx_weight(label, qdata, scale, swizzled, True)
    return _linear_forward(label, x, w, None, _ends(label, ends, w.experts), activation_dtype)


def grouped_mx_matmul_input_grad(dy: torch.Tensor, qdata: torch.Tensor, scale: torch.Tensor, ends: torch.Tensor, *,
                                 swizzled: bool = False) -> torch.Tensor:
    """The gradient of :func:`grouped_mx_matmul` to ``x``; zeros for rows of no group."""
    label = "Grouped MX product gradient"
    _on_gpu(label, dy, qdata, scale, ends)
    w = _mx_weight(label, qdata, scale, swizzled, True)
    return _linear_input_grad(label, dy, w, _ends(label, ends, w.experts))


# ---- INT8 weights ----------------------------------------------------------
def _int8_weight(label: str, qdata: torch.Tensor, scale: torch.Tensor, stacked: bool) -> L.WeightStruct:
    """Check INT8 storage (codes [rows, cols], one scale a row; stacked: one such weight per group) and describe it."""
    shape, sshape = qdata.shape, scale.shape
    if len(shape) != 2 + stacked:
        raise ValueError(f"{label} expects rank-{'three' if stacked else 'two'} INT8 codes.")
    if qdata.dtype is not torch.int8:
        raise ValueError(f"{label} expects int8 codes, got {qdata.dtype}.")
    if scale.dtype is not torch.float32 and scale.dtype is not torch.bfloat16:
        raise ValueError(f"{label} supports float32 and bfloat16 scales, got {scale.dtype}.")
    if not qdata.is_contiguous() or not scale.is_contiguous():
        raise ValueError(f"{label} requires contiguous INT8 storage.")
    if 0 in shape:
        raise ValueError(f"{label} requires a non-empty weight.")
    if sshape != shape[:-1] and sshape != (*shape[:-1], 1):
        raise ValueError(f"{label} takes one scale per row of the weight, got scales {tuple(sshape)} for codes {tuple(shape)}.")
    _raw(label, scale)
    return L.WeightStruct(qdata.data_ptr(), scale.data_ptr(), shape[-2], shape[-1], L.LM_I8, 0, shape[0] if stacked else 1,
                          L.torch_dtype_id(scale.dtype))


def int8_matmul(x: torch.Tensor, qdata: torch.Tensor, scale: torch.Tensor, *, bias: torch.Tensor | None = None,
                activation_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``x @ W.T + bias`` with ``W = scale * qdata`` (``qdata`` int8 [out, in], ``scale`` [out] or [out, 1]).

    ``x`` [..., in] bfloat16 or float16.  The sums run over the codes, which are exact, in fp32; they are multiplied by
    the scale and rounded once to ``x.dtype``.  With ``activation_dtype=torch.int8`` every row of ``x`` is quantised
    first: its scale is its largest magnitude times 1 / 127 in fp32, its codes are the exact quotients rounded to nearest (ties
    to even), and the sums of products of codes are exact.  A row with an infinity or a NaN then comes out NaN.
    """
    label = "INT8 product"
    _on_gpu(label, x, qdata, scale, bias)
    return _linear_forward(label, x, _int8_weight(label, qdata, scale, False), bias, None, activation_dtype)


def int8_matmul_input_grad(dy: torch.Tensor, qdata: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """``dy @ W``: the input gradient of :func:`int8_matmul` (straight through a quantised input).

    ``W`` is rounded to ``dy.dtype`` here: its scales lie along the sums.  In float16 that is 11 bits whatever the scales'
    size: the largest counts as 128 to 256 (rows whose scale is below 2^-21 of it lose bits).
    """
    label = "INT8 product gradient"
    _on_gpu(label, dy, qdata, scale)
    return _linear_input_grad(label, dy, _int8_weight(label, qdata, scale, False), None)


def grouped_int8_matmul(x: torch.Tensor, qdata: torch.Tensor, scale: torch.Tensor, ends: torch.Tensor, *,
                        activation_dtype: torch.dtype | None = None) -> torch.Tensor:
    """:func:`grouped_matmul` with INT8 weights: ``qdata`` [groups, out, in], ``scale`` [groups, out] or [groups, out, 1].

    Roundings as in :func:`int8_matmul`.
    """
    label = "Grouped INT8 product"
    _on_gpu(label, x, qdata, scale, ends)
    w = _int8_weight(label, qdata, scale, True)
    return _linear_forward(label, x, w, None, _ends(label, ends, w.experts), activation_dtype)


def grouped_int8_matmul_input_grad(dy: torch.Tensor, qdata: torch.Tensor, scale: torch.Tensor,
                                   ends: torch.Tensor) -> torch.Tensor:
    """The gradient of :func:`grouped_int8_matmul` to ``x``; zeros for rows of no group."""
    label = "Grouped INT8 product gradient"
    _on_gpu(label, dy, qdata, scale, ends)
    w = _int8_weight(label, qdata, scale, True)
    return _linear_input_grad(label, dy, w, _ends(label, ends, w.experts))


# ---------------------------------------------------------------------------
# Routing to experts
# ---------------------------------------------------------------------------
_SCORES = {"softmax": 0, "sigmoid": 1}
_MAX_BEST = 64
_MAX_GROUPS = 64
_MIN_SCALE, _MAX_SCALE = 2.0**-149, (2 - 2.0**-23) * 2.0**127  # of float32
_MAX_TOKENS = (1 << 28) - 64  # what one launch can hold
_LOGIT_DTYPES = (torch.float32, torch.bfloat16, torch.float16)


class Routing(NamedTuple):
    """The choices of every token, the best first.

    ``weight`` float32 [tokens, top_k]; ``expert`` int32 [tokens, top_k], -1 (with weight 0) where no expert was open;
    ``position`` int32 [tokens, top_k]: the place of each choice when the rows of one expert lie side by side, in the
    order of the tokens (those of no expert come last); ``ends`` int32 [experts]: the end of each expert's rows.
    """

    weight: torch.Tensor
    expert: torch.Tensor
    position: torch.Tensor
    ends: torch.Tensor


def _route(label: str, logits: torch.Tensor, top_k: int, bias: torch.Tensor | None, score: str, groups: int, top_groups: int,
           group_best: int, renormalize: bool, scale: float) -> tuple[L.RouteStruct, torch.Tensor]:
    shape = logits.shape
    if len(shape) != 2:
        raise ValueError(f"{label} expects logits [tokens, experts], got {tuple(shape)}.")
    if logits.dtype not in _LOGIT_DTYPES:
        raise ValueError(f"{label} supports float32, bfloat16 and float16 logits, got {logits.dtype}.")
    tokens, experts = shape
    if not 1 <= experts <= _MAX_EXPERTS:
        raise ValueError(f"{label} takes 1 to {_MAX_EXPERTS} experts, got {experts}.")
    if score not in _SCORES:
        raise ValueError(f"{label}: score must be 'softmax' or 'sigmoid', got {score!r}.")
    if not 1 <= groups <= _MAX_GROUPS or experts % groups:
        raise ValueError(f"{label}: {experts} experts do not divide into {groups} groups (1 to {_MAX_GROUPS}).")
    if not 1 <= top_groups <= groups:
        raise ValueError(f"{label}: top_groups must be 1 to {groups}, got {top_groups}.")
    if group_best not in (1, 2) or group_best > experts // groups:
        raise ValueError(f"{label}: group_best must be 1 or 2, and at most the experts of a group, got {group_best}.")
    if not 1 <= top_k <= min(_MAX_BEST, top_groups * (experts // groups)):
        raise ValueError(f"{label}: top_k must be 1 to {min(_MAX_BEST, top_groups * (experts // groups))}, got {top_k}.")
    if tokens > _MAX_TOKENS or tokens * top_k >= 1 << 31:
        raise ValueError(f"{label} takes up to 2^28 - 64 tokens and fewer than 2^31 choices, got {tokens} tokens of {top_k}.")
    if not _MIN_SCALE <= abs(scale) <= _MAX_SCALE:
        raise ValueError(f"{label}: scale must be finite and not zero in float32, got {scale}.")
    if bias is not None:
        if bias.dtype is not torch.float32 or tuple(bias.shape) != (experts,):
            raise ValueError(f"{label}: bias must be float32 [{experts}], got {bias.dtype} {tuple(bias.shape)}.")
        _raw(label, bias)
        bias = bias.contiguous()
    ld = experts
    if tokens > 1:
        ld = logits.stride(0)
        if ld < experts or (experts > 1 and logits.stride(1) != 1):
            logits, ld = logits.contiguous(), experts
    elif not logits.is_contiguous():
        logits = logits.contiguous()
    keep = logits if bias is None else (logits, bias)
    return L.RouteStruct(logits.data_ptr(), _ptr(bias), ld, tokens, experts, L.torch_dtype_id(logits.dtype), _SCORES[score],
                         top_k, groups, top_groups, group_best, renormalize, scale, 0), keep


def _enqueue(entry: Any, index: int, device: torch.device, *args: object) -> None:
    """Call one C entry that needs no workspace on GPU ``index``."""
    if torch._C._cuda_getDevice() != index:
        with L.on_device(device):
            _enqueue(entry, index, device, *args)
        return
    rc = entry(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        L.check(rc)


def route_topk(logits: torch.Tensor, top_k: int, *, bias: torch.Tensor | None = None, score: str = "softmax",
               groups: int = 1, top_groups: int = 1, group_best: int = 1, renormalize: bool = True,
               scale: float = 1.0) -> Routing:
    """The ``top_k`` experts of every token of ``logits`` [tokens, experts], their weights and their places.

    ``score`` 'softmax' or 'sigmoid' of the logits.  ``bias`` (float32 [experts]) is added for the choice alone.  With
    ``groups`` the experts form that many runs; the ``top_groups`` runs with the largest sums of their ``group_best``
    best choices stay open.  The weights are ``scale`` times the scores, divided by the sum of the chosen ones if
    ``renormalize``.  Ties go to the lowest index; scores are compared as numbers of 64 bits (by their logits where
    ``bias`` is None).  An expert whose logit (or bias) is -inf is closed: so is every expert of a padding token whose row is
    -inf.  A row with a NaN (softmax: or +inf) has NaN weights.  float32 throughout.
    """
    label = "Routing"
    _on_gpu(label, logits, bias)
    _raw(label, logits)
    r, keep = _route(label, logits, top_k, bias, score, groups, top_groups, group_best, renormalize, scale)
    (t, e), device = logits.shape, logits.device
    shape, strides = (t, top_k), (top_k, 1)
    weight = torch.empty_strided(shape, strides, dtype=torch.float32, device=device)
    expert = torch.empty_strided(shape, strides, dtype=torch.int32, device=device)
    position = torch.empty_like(expert)
    ends = torch.empty_strided((e,), (1,), dtype=torch.int32, device=device)
    _launch(L.lib().lm_route_topk, logits.get_device(), L.route_workspace_size(t, e), device, r, weight.data_ptr(),
            expert.data_ptr(), position.data_ptr(), ends.data_ptr())
    del keep
    return Routing(weight, expert, position, ends)


def route_topk_grad(dweight: torch.Tensor, logits: torch.Tensor, expert: torch.Tensor, *, score: str = "softmax",
                    renormalize: bool = True, scale: float = 1.0) -> torch.Tensor:
    """The gradient of :func:`route_topk`'s ``weight`` to ``logits``, for the ``expert`` that it chose."""
    label = "Routing gradient"
    _on_gpu(label, dweight, logits, expert)
    _raw(label, dweight, logits)
    shape = expert.shape
    if expert.dtype is not torch.int32 or len(shape) != 2 or shape[0] != logits.shape[0]:
        raise ValueError(f"{label}: expert must be int32 [tokens, top_k], got {expert.dtype} {tuple(shape)}.")
    if dweight.dtype is not torch.float32 or dweight.shape != shape:
        raise ValueError(f"{label}: dweight must be float32 {tuple(shape)}, got {dweight.dtype} {tuple(dweight.shape)}.")
    r, keep = _route(label, logits, shape[1], None, score, 1, 1, 1, renormalize, scale)
    dlogits = logits.new_empty(r.T, r.experts)
    dweight, expert = dweight.contiguous(), expert.contiguous()
    if r.T:
        _enqueue(L.lib().lm_route_topk_grad, logits.get_device(), logits.device, r, dweight.data_ptr(), expert.data_ptr(), dlogits.data_ptr())
    del keep
    return dlogits


def _places(label: str, x: torch.Tensor, of_choices: bool, position: torch.Tensor, ends: torch.Tensor
            ) -> tuple[torch.Tensor, int, L.RowsStruct, tuple[torch.Tensor, torch.Tensor]]:
    """``x``, rows of tokens or of their choices, with contiguous rows, its stride, and the places described."""
    places = position.shape
    if position.dtype is not torch.int32 or len(places) != 2 or places[1] < 1:
        raise ValueError(f"{label}: position must be int32 [tokens, top_k], got {position.dtype} {tuple(places)}.")
    tokens, top_k = places
    if tokens * top_k >= 1 << 31:
        raise ValueError(f"{label} takes fewer than 2^31 choices.")
    rows, shape = tokens * top_k if of_choices else tokens, x.shape
    if len(shape) != 2 or shape[0] != rows:
        raise ValueError(f"{label}: expected {rows} rows, got shape {tuple(shape)}.")
    if shape[1] < 1:
        raise ValueError(f"{label} requires non-empty rows.")
    x, _, ld = _rows(label, x, shape[1])
    ends = _ends(label, ends, ends.shape[0] if ends.ndim == 1 else -1)
    position = position.contiguous()
    return x, ld, L.RowsStruct(position.data_ptr(), ends.data_ptr(), tokens, shape[1], top_k, ends.shape[0],
                               L.torch_dtype_id(x.dtype), 0), (position, ends)


def _choice_weight(label: str, weight: torch.Tensor, position: torch.Tensor) -> torch.Tensor:
    if weight.dtype is not torch.float32 or weight.shape != position.shape:
        raise ValueError(f"{label}: weight must be float32 {tuple(position.shape)}, got {weight.dtype} {tuple(weight.shape)}.")
    _raw(label, weight)
    return weight.contiguous()


def dispatch_rows(x: torch.Tensor, position: torch.Tensor, ends: torch.Tensor) -> torch.Tensor:
    """Rows of tokens [tokens, cols] to the places of their choices: [tokens * top_k, cols], what a grouped product takes.

    ``position`` and ``ends`` as :func:`route_topk` gives them (each place once); places of no expert get zeros.
    """
    label = "Dispatch"
    _on_gpu(label, x, position, ends)
    x, ld, r, keep = _places(label, x, False, position, ends)
    out = x.new_empty(r.T * r.top_k, r.N)
    if r.T:
        _enqueue(L.lib().lm_dispatch_rows, x.get_device(), x.device, r, x.data_ptr(), ld, out.data_ptr())
    del keep
    return out


def dispatch_rows_grad(dy: torch.Tensor, position: torch.Tensor, ends: torch.Tensor) -> torch.Tensor:
    """The gradient of :func:`dispatch_rows` to ``x``: the sum over a token's choices, in fp32, rounded once."""
    label = "Dispatch gradient"
    _on_gpu(label, dy, position, ends)
    dy, ld, r, keep = _places(label, dy, True, position, ends)
    dx = dy.new_empty(r.T, r.N)
    if r.T:
        _enqueue(L.lib().lm_dispatch_rows_grad, dy.get_device(), dy.device, r, dy.data_ptr(), ld, dx.data_ptr())
    del keep
    return dx


def combine_rows(h: torch.Tensor, weight: torch.Tensor, position: torch.Tensor, ends: torch.Tensor) -> torch.Tensor:
    """What the experts return, ``h`` [tokens * top_k, cols], as weighted sums of a token's choices: [tokens, cols].

    ``weight`` float32 [tokens, top_k].  Sums in fp32 in the order of the choices, rounded once to ``h.dtype``; choices
    of no expert are left out, whatever their rows hold.
    """
    label = "Combine"
    _on_gpu(label, h, weight, position, ends)
    h, ld, r, keep = _places(label, h, True, position, ends)
    weight = _choice_weight(label, weight, position)
    out = h.new_empty(r.T, r.N)
    if r.T:
        _enqueue(L.lib().lm_combine_rows, h.get_device(), h.device, r, h.data_ptr(), ld, weight.data_ptr(), out.data_ptr())
    del keep
    return out


def combine_rows_grad(dy: torch.Tensor, h: torch.Tensor, weight: torch.Tensor, position: torch.Tensor, ends: torch.Tensor
                      ) -> tuple[torch.Tensor, torch.Tensor]:
    """The gradients of :func:`combine_rows` to ``h`` (zeros at places of no expert) and to ``weight``."""
    label = "Combine gradient"
    _on_gpu(label, dy, h, weight, position, ends)
    if dy.dtype is not h.dtype or dy.shape[-1:] != h.shape[-1:]:
        raise ValueError(f"{label}: dy {dy.dtype} {tuple(dy.shape)} and h {h.dtype} {tuple(h.shape)} differ.")
    dy, ldy, _, _ = _places(label, dy, False, position, ends)
    h, ldh, r, keep = _places(label, h, True, position, ends)
    weight = _choice_weight(label, weight, position)
    dh, dweight = h.new_empty(r.T * r.top_k, r.N), torch.empty_like(weight)
    if r.T:
        _enqueue(L.lib().lm_combine_rows_grad, h.get_device(), h.device, r, dy.data_ptr(), ldy, h.data_ptr(), ldh, weight.data_ptr(),
                 dh.data_ptr(), dweight.data_ptr())
    del keep
    return dh, dweight
