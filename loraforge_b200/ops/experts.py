"""Mixture-of-experts operators over the sm_100a C ABI: routing, the experts' products, their sum.

A layer with E experts runs ``route_experts`` on its router's logits, multiplies the rows it
gives by their experts' weights (``expert_linear``, which reads the tokens' rows through the
tables), and adds each token's rows up with ``combine_experts``.
Every operator reads its tables on the device, so a layer can be captured in a CUDA graph;
the LoRA operators take the same batch beside it (the rows of a token keep its adapter).
Each forward has an explicit gradient (``*_backward``) and records none: where autograd is
recording, tensors that require a gradient are refused.  The reference has no counterpart.
"""

from __future__ import annotations

from functools import lru_cache
from typing import NamedTuple

from loraforge_b200 import _native
from loraforge_b200.ops._contract import INT32_LIMIT, output_is_distinct

MAX_EXPERTS = 1024
MAX_TOP_K = 32


class ExpertRouting(NamedTuple):
    """Tables of a routed batch: T tokens, k slots each, R = T*k rows sorted by expert."""

    weights: object  # FP32 [T, k], largest first; 0 where no expert was left
    experts: object  # int32 [T, k]; -1 where no expert was left
    offsets: object  # int32 [E + 1]: rows [offsets[e], offsets[e+1]) are expert e's
    rows: object  # int32 [R]: token of each row; -1 beyond offsets[E]
    positions: object  # int32 [T, k]: row of each slot or -1


@lru_cache(maxsize=1)
def _kinds():
    """(torch.Tensor, 16-bit types, floating types), looked up once."""
    import torch

    halves = (torch.float16, torch.bfloat16)
    return torch.Tensor, halves, (torch.float32, *halves)


def _refuse_gradient(name: str) -> None:
    """For a tensor that requires a gradient: an error where autograd would record the call."""
    import torch

    if torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient, which the call does not record: detach it (gradients are "
                         "the *_backward operators) or call under torch.no_grad()")


def cuda_tensor(value, name: str, ndim: int, dtypes, index: int | None = None) -> int:
    """A CUDA tensor of rank `ndim` and one of `dtypes`, int32-indexable, on CUDA device `index`
    if given, that autograd does not follow; the index of its device."""
    if not isinstance(value, _kinds()[0]):
        raise TypeError(f"{name} must be a torch.Tensor")
    if value.ndim != ndim or value.dtype not in dtypes:
        raise ValueError(f"{name} must be {ndim}D with dtype {' or '.join(str(d) for d in dtypes)}")
    if value.numel() >= INT32_LIMIT and max(value.shape) >= INT32_LIMIT:
        raise ValueError(f"{name} dimensions must fit signed int32 indexing")
    found = value.get_device()  # -1: the host
    if found < 0 or not value.is_cuda or (index is not None and found != index):
        raise ValueError(f"{name} must be on the same CUDA GPU")
    if value.requires_grad:
        _refuse_gradient(name)
    return found


def row_matrix(value, name: str, dtypes, index: int | None = None) -> tuple:
    """A 2-D `cuda_tensor` of rows that do not overlap, with unit column stride: its device index,
    rows, width and row stride (a single row's own stride says nothing: its width)."""
    index = cuda_tensor(value, name, 2, dtypes, index)
    rows, width = value.shape
    if value.is_contiguous():
        return index, rows, width, width
    step, unit = value.stride()
    if (rows > 1 and step < width) or (width > 1 and unit != 1):
        raise ValueError(f"{name} must have unit column stride and rows that do not overlap")
    return index, rows, width, step if rows > 1 else width


def packed_table(value, name: str, shape, index: int, dtype) -> None:
    """A contiguous table of exactly `shape` on CUDA device `index`."""
    if (isinstance(value, _kinds()[0]) and value.dtype is dtype and value.shape == shape and value.is_contiguous()
            and value.get_device() == index and value.is_cuda):
        if value.requires_grad:
            _refuse_gradient(name)
        return
    cuda_tensor(value, name, len(shape), (dtype,), index)
    raise ValueError(f"{name} must be contiguous with shape {tuple(shape)}")


def _scale(value) -> float:
    scale = float(value)
    if not 2.0**-150 < scale <= 3.4028234663852886e38:  # what FP32 rounds to 0, and its largest value
        raise ValueError("scale must be positive and finite")
    return scale


def route_experts(logits, top_k: int, *, renormalize: bool = True, scale: float = 1.0,
                  out: ExpertRouting | None = None) -> ExpertRouting:
    """The ``top_k`` experts of each token, their weights, and the rows sorted by expert.

    ``logits`` [T, E] (FP32 / FP16 / BF16, unit column stride).  The experts are those of the
    largest logits, ties to the lowest index; NaN and -inf are never taken (a masked expert;
    a padding token is a row of -inf and gets no rows), +inf counts as the largest finite
    value.  With p = softmax(logits) in FP32 the weights are ``scale * p``, divided by the
    taken experts' sum when ``renormalize``.  ``out``: tables of an earlier call with the
    same sizes to write into (fixed addresses for CUDA graphs).
    """
    import torch

    index, T, E, stride = row_matrix(logits, "logits", _kinds()[2])
    if type(top_k) is not int or not 1 <= top_k <= min(E, MAX_TOP_K):
        raise ValueError(f"top_k must be in 1..min(experts, {MAX_TOP_K})")
    if E > MAX_EXPERTS:
        raise ValueError(f"at most {MAX_EXPERTS} experts")
    if T * top_k >= INT32_LIMIT:
        raise ValueError("tokens * top_k must fit signed int32 indexing")
    if type(renormalize) is not bool:
        raise ValueError("renormalize must be a bool")
    scale = _scale(scale)
    if out is None:
        # The four tables of T * k entries are parts of one allocation.
        parts = torch.unsafe_split_with_sizes(logits.new_empty((4 * T, top_k), dtype=torch.int32), (T, T, T, T))
        out = ExpertRouting(parts[0].view(torch.float32), parts[1], logits.new_empty(E + 1, dtype=torch.int32),
                            parts[2].view(-1), parts[3])
    else:
        for name, shape, dtype in (("weights", (T, top_k), torch.float32), ("experts", (T, top_k), torch.int32),
                                   ("offsets", (E + 1,), torch.int32), ("rows", (T * top_k,), torch.int32),
                                   ("positions", (T, top_k), torch.int32)):
            packed_table(getattr(out, name, None), f"out.{name}", shape, index, dtype)
            output_is_distinct(getattr(out, name), (logits,))
    room = _native.route_experts_workspace_ints(T, E)
    workspace = logits.new_empty(room, dtype=torch.int32) if room else None
    _native.launch(
        "lf_route_experts", index, _native.dtype_code(logits.dtype), logits.data_ptr(), stride, T, E, top_k,
        renormalize, scale, out.weights.data_ptr(), out.experts.data_ptr(), out.offsets.data_ptr(),
        out.rows.data_ptr(), out.positions.data_ptr(), workspace.data_ptr() if room else None, room,
    )
    return out


def route_experts_backward(logits, routing: ExpertRouting, grad_weights, *, renormalize: bool = True,
                           scale: float = 1.0):
    """Gradient of ``route_experts``' weights with respect to the logits, in their dtype.

    ``logits``, ``renormalize`` and ``scale`` as in the forward call, ``routing`` its result,
    ``grad_weights`` FP32 [T, k].  Experts count as fixed; a token without experts gets zeros.
    """
    import torch

    index, T, E, stride = row_matrix(logits, "logits", _kinds()[2])
    if not isinstance(routing, ExpertRouting):
        raise TypeError("routing must be the ExpertRouting of the forward call")
    if getattr(routing.weights, "ndim", 0) != 2:
        cuda_tensor(routing.weights, "routing.weights", 2, (torch.float32,), index)
    k = routing.weights.shape[1]
    packed_table(routing.weights, "routing.weights", (T, k), index, torch.float32)
    packed_table(routing.experts, "routing.experts", (T, k), index, torch.int32)
    grad_stride = row_matrix(grad_weights, "grad_weights", (torch.float32,), index)[3]
    if grad_weights.shape != (T, k):
        raise ValueError("grad_weights must have the weights' shape")
    if not 1 <= k <= min(E, MAX_TOP_K) or E > MAX_EXPERTS:
        raise ValueError("routing does not fit the logits")
    if type(renormalize) is not bool:
        raise ValueError("renormalize must be a bool")
    scale = _scale(scale)
    grad = logits.new_empty((T, E))
    _native.launch(
        "lf_route_experts_backward", index, _native.dtype_code(logits.dtype), logits.data_ptr(), stride,
        routing.weights.data_ptr(), routing.experts.data_ptr(), grad_weights.data_ptr(), grad_stride,
        T, E, k, renormalize, scale, grad.data_ptr(), E,
    )
    return grad


def _combine_tables(positions, weights, index: int):
    import torch

    if getattr(positions, "ndim", 0) != 2:
        cuda_tensor(positions, "positions", 2, (torch.int32,), index)
    T, k = positions.shape
    packed_table(positions, "positions", (T, k), index, torch.int32)
    if weights is not None:
        packed_table(weights, "weights", (T, k), index, torch.float32)
    if not 1 <= k <= MAX_TOP_K or T * k >= INT32_LIMIT:
        raise ValueError(f"positions must have 1..{MAX_TOP_K} columns and fit signed int32 indexing")
    return T, k


def combine_experts(y, weights, positions, *, out=None):
    """``out[t] = sum_j weights[t, j] * y[positions[t, j]]``, summed in FP32, in y's dtype.

    ``y`` [R, N] are the experts' rows, ``weights`` FP32 [T, k] (None: ones, the gradient of
    a gather), ``positions`` int32 [T, k]; a position outside [0, R) adds nothing, so a token
    without experts gets zeros.
    """
    index, R, N, stride = row_matrix(y, "y", _kinds()[2])
    T, k = _combine_tables(positions, weights, index)
    if N < 1:
        raise ValueError("y must have at least one column")
    out_stride = N
    if out is None:
        out = y.new_empty((T, N))
    else:
        out_stride = row_matrix(out, "out", (y.dtype,), index)[3]
        if out.shape != (T, N):
            raise ValueError("out must be [tokens, width]")
        output_is_distinct(out, (y, positions) if weights is None else (y, positions, weights))
    _native.launch(
        "lf_combine_experts", index, _native.dtype_code(y.dtype), y.data_ptr(), stride, R,
        None if weights is None else weights.data_ptr(), positions.data_ptr(), T, k, N, out.data_ptr(), out_stride,
    )
    return out


def combine_experts_backward(grad, y, weights, positions):
    """Gradients of ``combine_experts``: (grad_y [R, N] in y's dtype, grad_weights FP32 [T, k]).

    The positions that are not -1 must be the rows 0 .. n-1, each once, as ``route_experts``
    gives them; the rows behind them get zeros.  ``weights=None`` stands for ones and gives
    None for their gradient.
    """
    import torch

    index, R, N, stride = row_matrix(y, "y", _kinds()[2])
    T, k = _combine_tables(positions, weights, index)
    grad_stride = row_matrix(grad, "grad", (y.dtype,), index)[3]
    if grad.shape != (T, N) or N < 1:
        raise ValueError("grad must be [tokens, width]")
    grad_y = y.new_empty((R, N))
    grad_weights = None if weights is None else y.new_empty((T, k), dtype=torch.float32)
    _native.launch(
        "lf_combine_experts_backward", index, _native.dtype_code(y.dtype), grad.data_ptr(), grad_stride,
        y.data_ptr(), stride, R, None if weights is None else weights.data_ptr(), positions.data_ptr(), T, k, N,
        grad_y.data_ptr(), N, None if weights is None else grad_weights.data_ptr(),
    )
    return grad_y, grad_weights


def _operand(value, name: str, dtypes, index: int | None = None) -> tuple:
    """A `row_matrix` that TMA can read: aligned, its row stride a multiple of 8."""
    found = row_matrix(value, name, dtypes, index)
    _, _, width, stride = found
    if width < 8 or width % 8 or stride % 8 or value.data_ptr() % 16:
        raise ValueError(f"{name} must be 16-byte aligned with a width and row stride that are multiples of 8")
    return found


def _expert_weight(weight, dtype, index: int) -> tuple:
    """(experts, out, in, expert stride, row stride) of a weight tensor that TMA can read."""
    cuda_tensor(weight, "weight", 3, (dtype,), index)
    E, N, K = weight.shape
    if not 1 <= E <= MAX_EXPERTS or N < 8 or N % 8 or K < 8 or K % 8:
        raise ValueError(f"weight must be [experts, out, in] with 1..{MAX_EXPERTS} experts and widths that are multiples of 8")
    by_expert, by_row, unit = weight.stride()
    if E == 1:  # a single expert's own stride says nothing
        by_expert = N * by_row
    if unit != 1 or by_row % 8 or by_row < K or weight.data_ptr() % 16 or by_expert % 8 or by_expert < (N - 1) * by_row + K:
        raise ValueError("weight must be 16-byte aligned with unit inner stride and outer strides that are multiples of 8")
    return E, N, K, by_expert, by_row


def group_tables(offsets, rows, num_experts: int, x_rows: int, index: int) -> int:
    """Checks ``offsets`` [E + 1] and ``rows`` [R] (or None); the number of rows R."""
    import torch

    packed_table(offsets, "offsets", (num_experts + 1,), index, torch.int32)
    if rows is None:
        return x_rows
    if not isinstance(rows, torch.Tensor) or rows.ndim != 1:
        cuda_tensor(rows, "rows", 1, (torch.int32,), index)
    R = rows.numel()
    packed_table(rows, "rows", (R,), index, torch.int32)
    if R and not x_rows:
        raise ValueError("x must have at least one row")
    return R


def expert_linear(x, weight, offsets, *, rows=None, out=None):
    """``y[r] = weight[e] @ x[rows[r]]`` for the rows ``offsets[e] <= r < offsets[e+1]`` of expert e.

    ``x`` [T, K] and ``weight`` [E, N, K] are BF16 or FP16 (both the same; widths multiples of
    8); ``offsets`` int32 [E + 1] and ``rows`` int32 [R] are ``route_experts``' tables.  Without
    ``rows``, x's own rows are the sorted ones.  Sums are FP32, rounded once; rows of no group
    are zeros.  Returns y [R, N] (``out`` when given).
    """
    index, T, width, stride = _operand(x, "x", _kinds()[1])
    E, N, K, by_expert, by_row = _expert_weight(weight, x.dtype, index)
    if width != K:
        raise ValueError("x's width must be the weight's")
    R = group_tables(offsets, rows, E, T, index)
    out_stride = N
    if out is None:
        out = x.new_empty((R, N))
    else:
        out_stride = row_matrix(out, "out", (x.dtype,), index)[3]
        if out.shape != (R, N):
            raise ValueError("out must be [rows, out features]")
        output_is_distinct(out, (x, weight, offsets) if rows is None else (x, weight, offsets, rows))
    workspace, room = _gather_room(x, rows, E, R, K, False)
    _native.launch(
        "lf_expert_linear", index, _native.dtype_code(x.dtype), x.data_ptr(), stride, T,
        None if rows is None else rows.data_ptr(), weight.data_ptr(), by_expert, by_row, offsets.data_ptr(), E, R, N, K,
        out.data_ptr(), out_stride, workspace.data_ptr() if room else None, room,
    )
    return out


def _gather_room(x, rows, E: int, R: int, K: int, weight_grad: bool):
    """Scratch for x's rows in order, where the kernels want them so: (tensor or None, bytes)."""
    import torch

    room = 0 if rows is None else _native.expert_linear_workspace_bytes(E, R, K, weight_grad)
    return (x.new_empty(room, dtype=torch.uint8) if room else None), room


def expert_linear_backward(grad, x, weight, offsets, *, rows=None, weight_grad_dtype=None):
    """Gradients of ``expert_linear``: (grad_x [R, K], grad_weight [E, N, K]).

    ``grad`` [R, N] is the gradient of y.  ``grad_x`` is by row; ``combine_experts(grad_x,
    None, positions)`` adds it up by token.  ``weight_grad_dtype`` is the operands' type
    (default) or FP32.  Experts without rows get zeros.
    """
    import torch

    index, T, width, x_stride = _operand(x, "x", _kinds()[1])
    E, N, K, by_expert, by_row = _expert_weight(weight, x.dtype, index)
    stride = _operand(grad, "grad", (x.dtype,), index)[3]
    if width != K:
        raise ValueError("x's width must be the weight's")
    R = group_tables(offsets, rows, E, T, index)
    if grad.shape != (R, N):
        raise ValueError("grad must be [rows, out features]")
    weight_grad_dtype = x.dtype if weight_grad_dtype is None else weight_grad_dtype
    if weight_grad_dtype not in (x.dtype, torch.float32):
        raise ValueError("weight_grad_dtype must be the operands' type or float32")
    grad_x = x.new_empty((R, K))
    grad_weight = x.new_empty((E, N, K), dtype=weight_grad_dtype)
    dtype = _native.dtype_code(x.dtype)
    _native.launch(
        "lf_expert_linear_input_grad", index, dtype, grad.data_ptr(), stride, weight.data_ptr(), by_expert, by_row,
        offsets.data_ptr(), E, R, N, K, grad_x.data_ptr(), K,
    )
    workspace, room = _gather_room(x, rows, E, R, K, True)
    _native.launch(
        "lf_expert_linear_weight_grad", index, dtype, grad.data_ptr(), stride, x.data_ptr(), x_stride, T,
        None if rows is None else rows.data_ptr(), offsets.data_ptr(), E, R, N, K,
        _native.dtype_code(weight_grad_dtype), grad_weight.data_ptr(), workspace.data_ptr() if room else None, room,
    )
    return grad_x, grad_weight
