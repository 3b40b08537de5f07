"""Root-mean-square norm with the residual's addition, and its gradients.

`rms_norm` adds the residual, norms the sum and writes it in the rows' type, as an
FP8 operand (fp8.Packed) for the layer behind it, or as both, in one pass over the
rows. `rms_norm_backward` gives the gradients of the rows (the residual's is the same)
and of the weight.

Every call launches on the current stream, allocates only the outputs and workspaces
that it is not given, and raises ValueError for tensors that do not fit it.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _native, fp8
from .mx import _workspace, check_output, check_tensor, dtype_code, launch_stream, library, strided_rows


class Normed(NamedTuple):
    """What `rms_norm` gives: the normed rows (None if only an operand was asked for), their operand (None unless it was
    given) and the rows that were normed: x + residual, or x itself."""

    out: object
    packed: object
    total: object


def rms_norm(x, weight, eps: float = 1e-6, residual=None, out=None, packed=None, total=None, stream=None) -> Normed:
    """y = t * weight / sqrt(mean(t^2) + eps) of rows t = x [rows][n], or x + residual rounded to x's type (`total`,
    which may be x or the residual itself).

    y goes to `packed` (fp8.Packed of rows x n), if given, and to `out`, if given or if packed is not.
    """
    code = dtype_code(x, "x")
    rows, n, stride, span = strided_rows(x, "x")
    item, dtype, shape = 2 if code else 4, x.dtype, x.shape
    size = rows * n * item
    check_tensor(weight, "weight", (n,), dtype)
    added, sums, outputs, operand = (None, 0, 0), (None, 0), (None, 0), (None, 0, None, 0)
    tensors = (x, weight)
    if residual is None:
        if total is not None:
            raise ValueError("without a residual the total is x itself")
        total = x
    else:
        if residual.dtype is not dtype or residual.shape != shape:
            raise ValueError(f"the residual must be a {dtype} tensor of {tuple(shape)}, not {residual.dtype} of "
                             f"{tuple(residual.shape)}")
        _, _, residual_stride, residual_span = strided_rows(residual, "residual")
        total = check_output(total, "total", shape, dtype, x, stream)
        added, sums = (residual.data_ptr(), residual_span * item, residual_stride), (total.data_ptr(), size)
        tensors = (x, weight, residual, total)
    if packed is not None:
        packed = fp8._operand(packed, "packed", rows, n, 1, x, stream)
        operand = fp8._parts(packed)
        tensors += (packed.codes, packed.scales)
    if out is not None or packed is None:
        out = check_output(out, "out", shape, dtype, x, stream)
        outputs = (out.data_ptr(), size)
        tensors += (out,)
    handle = launch_stream(stream, *tensors)
    status = library().mb_rms_norm(code, x.data_ptr(), span * item, stride, *added, weight.data_ptr(), n * item, eps,
                                   *sums, *outputs, *operand, rows, n, handle)
    if status:
        _native.check(status)
    return Normed(out, packed, total)


def rms_norm_backward_workspace(rows: int, n: int, device="cuda"):
    """A workspace for `rms_norm_backward`."""
    return torch.empty(library().mb_rms_norm_backward_workspace(rows, n), dtype=torch.uint8, device=device)


def rms_norm_backward(d_out, total, weight, eps: float = 1e-6, d_total=None, d_x=None, d_weight=None, workspace=None,
                      stream=None):
    """(d_x, d_weight) of rms_norm for the gradient d_out [rows][n] of its output, in its type.

    `total` is what was normed (Normed.total); `d_total`, if given, is the gradient that reaches it as an output itself
    and is added. d_x is the gradient of x and of the residual alike, and may be d_out or d_total itself.
    """
    code = dtype_code(total, "total")
    rows, n, stride, span = strided_rows(total, "total")
    item = 2 if code else 4
    check_tensor(weight, "weight", (n,), total.dtype)
    tensors, strides = [d_out, total, weight], []
    for name, tensor in (("d_out", d_out), ("d_total", d_total)):
        if tensor is None:
            strides.append((None, 0, 0))
            continue
        if tensor.dtype is not total.dtype or tensor.shape != total.shape:
            raise ValueError(f"{name} must be a {total.dtype} tensor of {tuple(total.shape)}, not {tensor.dtype} of "
                             f"{tuple(tensor.shape)}")
        _, _, d_stride, d_span = strided_rows(tensor, name)
        strides.append((tensor.data_ptr(), d_span * item, d_stride))
    if d_total is not None:
        tensors.append(d_total)
    d_x = check_output(d_x, "d_x", (rows, n), total.dtype, total, stream)
    d_weight = check_output(d_weight, "d_weight", (n,), total.dtype, total, stream)
    if not rows or not n:
        launch_stream(stream, *tensors, d_x, d_weight)
        with torch.cuda.stream(stream):  # cleared in the order of the call's work
            return d_x, d_weight.zero_()
    native = library()
    workspace = _workspace(workspace, native.mb_rms_norm_backward_workspace(rows, n), total, stream)
    handle = launch_stream(stream, *tensors, d_x, d_weight, workspace)
    status = native.mb_rms_norm_backward(code, *strides[0], total.data_ptr(), span * item, stride,
                                         weight.data_ptr(), n * item, eps, *strides[1], d_x.data_ptr(),
                                         rows * n * item, d_weight.data_ptr(), n * item, rows, n,
                                         workspace.data_ptr(), workspace.numel(), handle)
    if status:
        _native.check(status)
    return d_x, d_weight
