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
from loraforge_b200.ops.experts import MAX_EXPERTS, _kinds, cuda_tensor, group_tables, packed_table, row_matrix

BLOCK = 32


class MxTensor(NamedTuple):
    """A tensor [..., K] in MXFP4."""

    codes: object  # uint8 [..., K / 2]
    scales: object  # uint8 [..., K / 32]


def check_mx(value, name: str, ndim: int, index: int | None = None) -> tuple:
    """(shape [..., K], device index) of a contiguous MxTensor of rank `ndim`, on `index` if given."""
    import torch

    if not isinstance(value, MxTensor):
        raise TypeError(f"{name} must be an MxTensor")
    codes = value.codes
    index = cuda_tensor(codes, f"{name}.codes", ndim, (torch.uint8,), index)
    *rows, half = codes.shape
    if half < BLOCK // 2 or half % (BLOCK // 2) or not codes.is_contiguous() or codes.data_ptr() % 16:
        raise ValueError(f"{name}.codes must be contiguous and 16-byte aligned with rows of whole blocks of {BLOCK}")
    packed_table(value.scales, f"{name}.scales", (*rows, half * 2 // BLOCK), index, torch.uint8)
    return (*rows, 2 * half), index


def mxfp4_quantize(x) -> MxTensor:
    """``x`` [..., K] (FP32 / FP16 / BF16, K a multiple of 32) rounded to MXFP4.

    A 2-D ``x`` may have any row stride; one of another rank must be contiguous.
    """
    import torch

    if not isinstance(x, torch.Tensor):
        raise TypeError("x must be a torch.Tensor")
    index = cuda_tensor(x, "x", max(x.ndim, 1), _kinds()[2])
    *shape, K = x.shape
    if K < BLOCK or K % BLOCK:
        raise ValueError(f"x's last dimension must be a positive multiple of {BLOCK}")
    rows, stride = x.numel() // K, K
    if not x.is_contiguous():
        if x.ndim != 2:
            raise ValueError("x must be contiguous unless it is 2D")
        stride = x.stride(0)
        if x.stride(1) != 1 or stride < K:
            raise ValueError("x must have unit column stride and rows that do not overlap")
    codes = x.new_empty((*shape, K // 2), dtype=torch.uint8)
    scales = x.new_empty((*shape, K // BLOCK), dtype=torch.uint8)
    _native.launch("lf_mxfp4_quantize", index, _native.dtype_code(x.dtype), x.data_ptr(), stride, rows, K,
                   codes.data_ptr(), scales.data_ptr())
    return MxTensor(codes, scales)


def mxfp4_dequantize(x: MxTensor, dtype=None):
    """The values ``x`` stands for in ``dtype`` (default BF16).

    BF16 and FP32 hold exactly all that ``mxfp4_quantize`` gives (scale bytes up to 252).  Of the bytes
    253 and 254, which other programs may write, values from 2^128 on become infinite; FP16 rounds.
    """
    import torch

    dtype = torch.bfloat16 if dtype is None else dtype
    if dtype not in _kinds()[2]:
        raise ValueError("dtype must be float32, float16 or bfloat16")
    if not isinstance(x, MxTensor):
        raise TypeError("x must be an MxTensor")
    shape, index = check_mx(x, "x", getattr(x.codes, "ndim", 1))
    out = x.codes.new_empty(shape, dtype=dtype)
    _native.launch("lf_mxfp4_dequantize", index, _native.dtype_code(dtype), x.codes.data_ptr(), x.scales.data_ptr(),
                   out.numel() // shape[-1], shape[-1], out.data_ptr())
    return out


def expert_linear_mxfp4(x: MxTensor, weight: MxTensor, offsets, *, rows=None, dtype=None, out=None):
    """``expert_linear`` of MXFP4 operands on the block-scaled tensor cores.

    ``x`` [T, K] and ``weight`` [E, N, K] are MxTensors; ``offsets`` int32 [E + 1] and ``rows``
    int32 [R] as in ``expert_linear`` (one expert and offsets (0, T) give a dense product).
    Sums are FP32, rounded once to ``dtype`` (FP32 / FP16 / BF16, default BF16 or out's); rows of
    no group are zeros.  Returns y [R, N] (``out`` when given).
    """
    import torch

    (T, K), index = check_mx(x, "x", 2)
    E, N, width = check_mx(weight, "weight", 3, index)[0]
    if width != K:
        raise ValueError("x's width must be the weight's")
    if not 1 <= E <= MAX_EXPERTS or N < 1:
        raise ValueError(f"weight must be [experts, out, in] with 1..{MAX_EXPERTS} experts")
    R = group_tables(offsets, rows, E, T, index)
    if dtype is not None and dtype not in _kinds()[2]:
        raise ValueError("dtype must be float32, float16 or bfloat16")
    out_stride = N
    if out is None:
        out = x.codes.new_empty((R, N), dtype=torch.bfloat16 if dtype is None else dtype)
    else:
        out_stride = row_matrix(out, "out", _kinds()[2] if dtype is None else (dtype,), index)[3]
        if out.shape != (R, N):
            raise ValueError("out must be [rows, out features]")
        output_is_distinct(out, (*x, *weight, offsets) if rows is None else (*x, *weight, offsets, rows))
    room = _native.expert_linear_mxfp4_workspace_bytes(E, R, N, K, rows is not None)
    workspace = x.codes.new_empty(room) if room else None
    _native.launch(
        "lf_expert_linear_mxfp4", index, _native.dtype_code(out.dtype), x.codes.data_ptr(), x.scales.data_ptr(), T,
        None if rows is None else rows.data_ptr(), weight.codes.data_ptr(), weight.scales.data_ptr(),
        offsets.data_ptr(), E, R, N, K, out.data_ptr(), out_stride, workspace.data_ptr() if room else None, room,
    )
    return out
