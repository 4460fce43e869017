"""MXFP4 (microscaled 4-bit floating point) over the sm_100a C ABI.

Blocks of 32 values along the last dimension share a scale 2^e held as the byte e + 127; each
value is a 4-bit E2M1 code (sign, magnitudes 0 0.5 1 1.5 2 3 4 6), two codes a byte, the
even-indexed one in the low half: 4.25 bits a value.  e = floor(log2 of the block's largest
magnitude) - 2, not below -127; values are rounded to nearest, ties to even, and magnitudes
over 6 * 2^e become that.  A block with an infinity or a NaN is NaN throughout (scale byte 255).
"""

from __future__ import annotations

from typing import NamedTuple

from loraforge_b200 import _native
from loraforge_b200.ops._contract import output_is_distinct
from loraforge_b200.ops.experts import MAX_EXPERTS, cuda_tensor, group_tables, packed_table, row_matrix, row_stride

BLOCK = 32


class MxTensor(NamedTuple):
    """A tensor [..., K] in MXFP4."""

    codes: object  # uint8 [..., K / 2]
    scales: object  # uint8 [..., K / 32]


def check_mx(value, name: str, ndim: int, device=None) -> tuple:
    """The shape [..., K] of a contiguous MxTensor of rank `ndim` on `device` if given."""
    import torch

    if not isinstance(value, MxTensor):
        raise TypeError(f"{name} must be an MxTensor")
    cuda_tensor(value.codes, f"{name}.codes", ndim, (torch.uint8,), device)
    *rows, half = value.codes.shape
    if half < BLOCK // 2 or half % (BLOCK // 2) or not value.codes.is_contiguous() or value.codes.data_ptr() % 16:
        raise ValueError(f"{name}.codes must be contiguous and 16-byte aligned with rows of whole blocks of {BLOCK}")
    packed_table(value.scales, f"{name}.scales", (*rows, half * 2 // BLOCK), value.codes.device, torch.uint8)
    return (*rows, 2 * half)


def mxfp4_quantize(x) -> MxTensor:
    """``x`` [..., K] (FP32 / FP16 / BF16, K a multiple of 32) rounded to MXFP4.

    A 2-D ``x`` may have any row stride; one of another rank must be contiguous.
    """
    import torch

    if not isinstance(x, torch.Tensor):
        raise TypeError("x must be a torch.Tensor")
    cuda_tensor(x, "x", max(x.ndim, 1), (torch.float32, torch.float16, torch.bfloat16))
    K = x.shape[-1]
    if K < BLOCK or K % BLOCK:
        raise ValueError(f"x's last dimension must be a positive multiple of {BLOCK}")
    shape = tuple(x.shape[:-1])
    if x.ndim == 2 and x.shape[0] > 1:
        rows, stride = x.shape[0], x.stride(0)
        if x.stride(1) != 1 or stride < K:
            raise ValueError("x must have unit column stride and rows that do not overlap")
    else:
        rows, stride = x.numel() // K, K
        if not x.is_contiguous():
            raise ValueError("x must be contiguous unless it is 2D")
    codes = torch.empty((*shape, K // 2), dtype=torch.uint8, device=x.device)
    scales = torch.empty((*shape, K // BLOCK), dtype=torch.uint8, device=x.device)
    with torch.cuda.device(x.device):
        _native.call("lf_mxfp4_quantize", _native.dtype_code(x.dtype), x.data_ptr(), stride, rows, K,
                     codes.data_ptr(), scales.data_ptr(), _native.stream_of(x.device))
    return MxTensor(codes, scales)


def mxfp4_dequantize(x: MxTensor, dtype=None):
    """The values ``x`` stands for in ``dtype`` (default BF16, which holds all of them exactly)."""
    import torch

    dtype = torch.bfloat16 if dtype is None else dtype
    if dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise ValueError("dtype must be float32, float16 or bfloat16")
    if not isinstance(x, MxTensor):
        raise TypeError("x must be an MxTensor")
    shape = check_mx(x, "x", getattr(x.codes, "ndim", 1))
    out = torch.empty(shape, dtype=dtype, device=x.codes.device)
    with torch.cuda.device(out.device):
        _native.call("lf_mxfp4_dequantize", _native.dtype_code(dtype), x.codes.data_ptr(), x.scales.data_ptr(),
                     out.numel() // shape[-1], shape[-1], out.data_ptr(), _native.stream_of(out.device))
    return out


def expert_linear_mxfp4(x: MxTensor, weight: MxTensor, offsets, *, rows=None, dtype=None, out=None):
    """``expert_linear`` of MXFP4 operands on the block-scaled tensor cores.

    ``x`` [T, K] and ``weight`` [E, N, K] are MxTensors; ``offsets`` int32 [E + 1] and ``rows``
    int32 [R] as in ``expert_linear`` (one expert and offsets (0, T) give a dense product).
    Sums are FP32, rounded once to ``dtype`` (FP32 / FP16 / BF16, default BF16 or out's); rows of
    no group are zeros.  Returns y [R, N] (``out`` when given).
    """
    import torch

    T, K = check_mx(x, "x", 2)
    device = x.codes.device
    E, N, width = check_mx(weight, "weight", 3, device)
    if width != K:
        raise ValueError("x's width must be the weight's")
    if not 1 <= E <= MAX_EXPERTS or N < 1:
        raise ValueError(f"weight must be [experts, out, in] with 1..{MAX_EXPERTS} experts")
    R = group_tables(offsets, rows, E, T, device)
    kinds = (torch.float32, torch.float16, torch.bfloat16)
    if dtype is not None and dtype not in kinds:
        raise ValueError("dtype must be float32, float16 or bfloat16")
    if out is None:
        out = torch.empty((R, N), dtype=torch.bfloat16 if dtype is None else dtype, device=device)
    else:
        row_matrix(out, "out", kinds if dtype is None else (dtype,), device)
        if tuple(out.shape) != (R, N):
            raise ValueError("out must be [rows, out features]")
        output_is_distinct(out, (*x, *weight, offsets) if rows is None else (*x, *weight, offsets, rows))
    room = _native.expert_linear_mxfp4_workspace_bytes(E, R, N, K, rows is not None)
    workspace = torch.empty(room, dtype=torch.uint8, device=device) if room else None
    with torch.cuda.device(device):
        _native.call(
            "lf_expert_linear_mxfp4", _native.dtype_code(out.dtype), x.codes.data_ptr(), x.scales.data_ptr(), T,
            None if rows is None else rows.data_ptr(), weight.codes.data_ptr(), weight.scales.data_ptr(),
            offsets.data_ptr(), E, R, N, K, out.data_ptr(), row_stride(out),
            None if workspace is None else workspace.data_ptr(), room, _native.stream_of(device),
        )
    return out
