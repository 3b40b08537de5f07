"""MXFP4 operands and linear layers: quantisation, products, gradients.

An operand (`Packed`) is what the MXFP4 GEMM reads: E2M1 codes two per byte
along K and one E8M0 scale per 32 elements, in K-step blocks. `quantize` makes
one from a tensor's rows or columns, `dequantize` gives its values back, and
`linear` multiplies a tensor, quantised on the way, with a weight laid out
once: one weight, or one for each expert that `routing.dispatch` sorted the
rows by. A training step quantises the weight both ways and calls
`linear_backward`, whose products take the gradient and the saved input in
MXFP4 too (straight through: quantisation has the identity's gradient).

Every call launches on the current stream, allocates only the outputs and
workspaces that it is not given, and raises ValueError for tensors that do not
fit it.
"""

from __future__ import annotations

import torch

from . import _native, formats

GROUP = formats.MX_GROUP_SIZE
STEP = 256  # K elements whose scales a row holds together


DTYPE_CODES = {torch.float32: _native.MB_DTYPE_F32, torch.float16: _native.MB_DTYPE_F16,
               torch.bfloat16: _native.MB_DTYPE_BF16}


class Packed:
    """An operand of rows x k: codes [rows][ceil(k/32)*16] and scales [ceil(k/256)][rows][8], contiguous uint8
    tensors; with a leading dimension each, one such matrix for each of `experts`."""

    __slots__ = ("codes", "scales", "k", "rows", "experts")

    def __init__(self, codes, scales, k: int):
        lead = codes.shape[:-2]
        rows = codes.shape[-2] if codes.dim() >= 2 else -1
        if (codes.dtype != torch.uint8 or scales.dtype != torch.uint8 or len(lead) > 1 or not codes.is_contiguous()
                or not scales.is_contiguous() or codes.shape != (*lead, rows, -(-k // GROUP) * (GROUP // 2))
                or scales.shape != (*lead, -(-k // STEP), rows, STEP // GROUP)):
            raise ValueError(f"an operand of k = {k} has contiguous uint8 codes [rows][{-(-k // GROUP) * 16}] and "
                             f"scales [{-(-k // STEP)}][rows][8], not {tuple(codes.shape)} and {tuple(scales.shape)}")
        self.codes, self.scales, self.k, self.rows = codes, scales, k, rows
        self.experts = lead[0] if lead else None


# The checks below run at every call, beside which a kernel takes a few microseconds: get_device and comparisons of
# shapes cost tens of nanoseconds, tensor.device and torch.cuda.current_device several hundred.


def dtype_code(tensor, what: str) -> int:
    code = DTYPE_CODES.get(tensor.dtype)
    if code is None:
        raise ValueError(f"{what} must be float32, float16 or bfloat16, not {tensor.dtype}")
    return code


def check_device(*tensors) -> None:
    device = tensors[0].get_device()
    if device != (torch._C._cuda_getDevice() if torch.cuda.is_initialized() else torch.cuda.current_device()):
        raise ValueError(f"tensors must lie on the current HIP device (cuda:{torch.cuda.current_device()}), not "
                         f"{tensors[0].device}")
    for tensor in tensors:
        if tensor.get_device() != device:
            raise ValueError(f"tensors must lie on one device, cuda:{device}, not {tensor.device}")


def strided_rows(tensor, what: str) -> tuple[int, int]:
    """(row stride, bytes spanned) of a 2-D tensor with contiguous rows."""
    if tensor.dim() != 2:
        raise ValueError(f"{what} must have two dimensions, not {tensor.dim()}")
    rows, columns = tensor.shape
    stride, step = tensor.stride()
    if columns > 1 and step != 1:
        raise ValueError(f"{what} must have contiguous rows (a stride of 1 along its last dimension)")
    if not rows or not columns:
        return columns, 0
    return stride if rows > 1 else columns, ((rows - 1) * stride + columns) * tensor.element_size()


def check_output(tensor, what: str, shape, dtype, device):
    """`tensor`, checked, or a new one in its place."""
    if tensor is None:
        return torch.empty(shape, dtype=dtype, device=device)
    if tensor.shape != shape or tensor.dtype != dtype or not tensor.is_contiguous():
        raise ValueError(f"{what} must be a contiguous {dtype} tensor of {tuple(shape)}, not {tensor.dtype} of "
                         f"{tuple(tensor.shape)}")
    return tensor


def bytes_of(tensor) -> int:
    return tensor.numel() * tensor.element_size()


def empty(rows: int, k: int, device="cuda", experts: int | None = None) -> Packed:
    """An operand's buffers, for `quantize` to fill."""
    lead = () if experts is None else (experts,)
    return Packed(torch.empty((*lead, rows, -(-k // GROUP) * (GROUP // 2)), dtype=torch.uint8, device=device),
                  torch.empty((*lead, -(-k // STEP), rows, STEP // GROUP), dtype=torch.uint8, device=device), k)


def _check_experts(packed: Packed, what: str, experts: int | None) -> None:
    if packed.experts != experts:
        raise ValueError(f"{what} must hold {'one matrix' if experts is None else f'a matrix for each of {experts} experts'},"
                         f" not codes of {tuple(packed.codes.shape)}")


def quantize(x, packed: Packed | None = None, columns: bool = False, stream=None) -> Packed:
    """The MXFP4 operand of x's rows; with `columns`, of its columns (x transposed, groups along its rows)."""
    code = dtype_code(x, "x")
    stride, span = strided_rows(x, "x")
    rows, k = x.shape[::-1] if columns else x.shape
    if packed is None:
        packed = empty(rows, k, x.device)
    _check_experts(packed, "packed", None)
    if (packed.rows, packed.k) != (rows, k):
        raise ValueError(f"packed must be an operand of {rows} x {k}, not {packed.rows} x {packed.k}")
    check_device(x, packed.codes, packed.scales)
    out = (packed.codes.data_ptr(), packed.codes.numel(), packed.scales.data_ptr(), packed.scales.numel(),
           _native.stream_handle(stream))
    if columns:
        _native.call("mb_mx_quantize_columns", code, x.data_ptr(), span, k, rows, stride, *out)
    else:
        _native.call("mb_mx_quantize", code, x.data_ptr(), span, rows, k, stride, None, 0, 1, rows, *out)
    return packed


def dequantize(packed: Packed, out=None, stream=None):
    """The values of an operand [rows][k]: bfloat16 (exact) unless `out` is of another type."""
    _check_experts(packed, "packed", None)
    dtype = torch.bfloat16 if out is None else out.dtype
    out = check_output(out, "out", (packed.rows, packed.k), dtype, packed.codes.device)
    code = dtype_code(out, "out")
    check_device(packed.codes, packed.scales, out)
    _native.call("mb_mx_dequantize", code, packed.codes.data_ptr(), packed.codes.numel(), packed.scales.data_ptr(),
                 packed.scales.numel(), out.data_ptr(), bytes_of(out), packed.rows, packed.k,
                 _native.stream_handle(stream))
    return out


def product(a: Packed, b: Packed, out=None, dtype=None, offsets=None, stream=None):
    """A . B^T of two operands, in `dtype` (bfloat16 unless `out` or `dtype` says otherwise).

    With `offsets` ([experts + 1] int32, on the device) b holds a matrix for each expert, and a's rows offsets[e] ..
    offsets[e + 1] - 1 meet matrix e; output rows from offsets[experts] on are not written.
    """
    experts = None if offsets is None else offsets.numel() - 1
    _check_experts(a, "a", None)
    _check_experts(b, "b", experts)
    if a.k != b.k:
        raise ValueError(f"a and b must have the same k, not {a.k} and {b.k}")
    if dtype is None:
        dtype = torch.bfloat16 if out is None else out.dtype
    out = check_output(out, "out", (a.rows, b.rows), dtype, a.codes.device)
    code = dtype_code(out, "out")
    _check_indices(offsets, "offsets")
    check_device(a.codes, a.scales, b.codes, b.scales, out, *(() if offsets is None else (offsets,)))
    _native.call("mb_mx_product", code, a.codes.data_ptr(), a.codes.numel(), a.scales.data_ptr(), a.scales.numel(),
                 b.codes.data_ptr(), b.codes.numel(), b.scales.data_ptr(), b.scales.numel(), out.data_ptr(),
                 bytes_of(out), a.rows, b.rows, a.k, *_pointer(offsets), experts or 1, _native.stream_handle(stream))
    return out


def _check_indices(tensor, what: str) -> None:
    if tensor is not None and (tensor.dtype != torch.int32 or not tensor.is_contiguous()):
        raise ValueError(f"{what} must be a contiguous int32 tensor, not {tensor.dtype}")


def _pointer(tensor) -> tuple[int | None, int]:
    return (None, 0) if tensor is None else (tensor.data_ptr(), bytes_of(tensor))


def _workspace(tensor, needed: int, device):
    if tensor is None:
        return torch.empty(needed, dtype=torch.uint8, device=device)
    if tensor.dtype != torch.uint8 or not tensor.is_contiguous() or tensor.numel() < needed:
        raise ValueError(f"workspace must be a contiguous uint8 tensor of at least {needed} bytes")
    return tensor


def linear_workspace(rows: int, n: int, k: int, dtype, experts: int = 1, device="cuda"):
    """A workspace for `linear` with `rows` output rows (routed ones, with a plan)."""
    return torch.empty(_native.load().mb_mx_linear_workspace(rows, n, k), dtype=torch.uint8, device=device)


def linear(x, weight: Packed, out=None, plan=None, sorted_rows: bool = False, workspace=None, stream=None):
    """Q(x) . W^T in x's type: x [rows][k], weight an operand of n rows, out [rows][n].

    With a `plan` (routing.dispatch) the weight holds a matrix for each expert: x [tokens][k] gives the routed rows
    out [tokens * top][n] in the plan's order, or, `sorted_rows`, x's rows are routed rows in that order already. Rows
    from plan.offsets[experts] on are not written.
    """
    code = dtype_code(x, "x")
    stride, span = strided_rows(x, "x")
    rows, k = x.shape
    offsets = order = slots = None
    copies, experts = 1, None
    if plan is not None:
        offsets = plan.offsets
        experts = offsets.numel() - 1
        _check_indices(offsets, "plan.offsets")
        if not sorted_rows:
            order, slots = plan.order, plan.slots
            _check_indices(order, "plan.order")
            _check_indices(slots, "plan.slots")
            if slots.dim() != 2 or slots.shape[0] != rows or order.numel() != slots.numel():
                raise ValueError(f"the plan must route {rows} tokens, not slots of {tuple(slots.shape)}")
            copies = slots.shape[1]
        check_device(offsets, *(() if sorted_rows else (order, slots)))
    elif sorted_rows:
        raise ValueError("sorted rows need the plan that they are sorted by")
    _check_experts(weight, "weight", experts)
    if weight.k != k:
        raise ValueError(f"the weight must have k = {k}, not {weight.k}")
    n, routed = weight.rows, rows * copies
    out = check_output(out, "out", (routed, n), x.dtype, x.device)
    library = _native.load()
    workspace = _workspace(workspace, library.mb_mx_linear_workspace(routed, n, k), x.device)
    check_device(x, weight.codes, weight.scales, out, workspace)
    _native.check(library.mb_mx_linear(
        code, x.data_ptr(), span, rows, stride, weight.codes.data_ptr(), weight.codes.numel(),
        weight.scales.data_ptr(), weight.scales.numel(), out.data_ptr(), bytes_of(out), n, k, *_pointer(offsets),
        None if order is None else order.data_ptr(), *_pointer(slots), copies, experts or 1, workspace.data_ptr(),
        workspace.numel(), _native.stream_handle(stream)))
    return out


def _operand_bytes(rows: int, k: int) -> int:
    """Bytes of an operand's codes and scales, each on 16 bytes."""
    return -(-rows * (-(-k // GROUP) * 16) // 16) * 16 + -(-rows * (-(-k // STEP) * 8) // 16) * 16


def _carve(workspace, at: int, rows: int, k: int) -> Packed:
    codes = rows * (-(-k // GROUP) * 16)
    start = at + -(-codes // 16) * 16
    scales = rows * (-(-k // STEP) * 8)
    return Packed(workspace[at:at + codes].view(rows, -(-k // GROUP) * 16),
                  workspace[start:start + scales].view(-(-k // STEP), rows, 8), k)


def linear_backward_workspace(rows: int, n: int, k: int, dtype, device="cuda"):
    """A workspace for `linear_backward`, and for `linear` of the same sizes."""
    needed = max(_backward_bytes(rows, n, k), _native.load().mb_mx_linear_workspace(rows, n, k))
    return torch.empty(needed, dtype=torch.uint8, device=device)


def _backward_bytes(rows: int, n: int, k: int) -> int:
    return _operand_bytes(rows, n) + _operand_bytes(n, rows) + _operand_bytes(k, rows)


def linear_backward(d_out, x, weight_columns: Packed, d_x=None, d_weight=None, workspace=None, stream=None):
    """(d_x, d_weight) of out = Q(x) . Q(w)^T for the gradient d_out [rows][n], in x's type.

    d_x = Q(d_out) . W with `weight_columns` = quantize(w, columns=True); d_weight = d_out^T . x, both quantised
    along the rows that the sum runs over.
    """
    rows, n = d_out.shape
    k = x.shape[1] if x.dim() == 2 else -1
    if d_out.dtype != x.dtype or x.dim() != 2 or x.shape[0] != rows:
        raise ValueError(f"d_out and x must be of one type and number of rows, not {d_out.dtype} of "
                         f"{tuple(d_out.shape)} and {x.dtype} of {tuple(x.shape)}")
    if (weight_columns.rows, weight_columns.k) != (k, n):
        raise ValueError(f"weight_columns must be an operand of {k} x {n} (the weight quantised by columns), not "
                         f"{weight_columns.rows} x {weight_columns.k}")
    workspace = _workspace(workspace, _backward_bytes(rows, n, k), x.device)
    if not rows:
        d_weight = check_output(d_weight, "d_weight", (n, k), x.dtype, x.device)
        return check_output(d_x, "d_x", (rows, k), x.dtype, x.device), d_weight.zero_()
    by_rows = _carve(workspace, 0, rows, n)
    d_columns = _carve(workspace, _operand_bytes(rows, n), n, rows)
    x_columns = _carve(workspace, _operand_bytes(rows, n) + _operand_bytes(n, rows), k, rows)
    quantize(d_out, by_rows, stream=stream)
    quantize(d_out, d_columns, columns=True, stream=stream)
    quantize(x, x_columns, columns=True, stream=stream)
    d_x = product(by_rows, weight_columns, d_x, dtype=x.dtype, stream=stream)
    d_weight = product(d_columns, x_columns, d_weight, dtype=x.dtype, stream=stream)
    return d_x, d_weight
