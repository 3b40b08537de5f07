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


# The checks below run at every call, beside which a kernel takes a few microseconds. They read shapes, types and
# device numbers, tens of nanoseconds each, and compare them; only a refusal builds anything (torch.device objects,
# tuples of sizes and messages cost several hundred).


def dtype_code(tensor, what: str) -> int:
    code = DTYPE_CODES.get(tensor.dtype)
    if code is None:
        raise ValueError(f"{what} must be float32, float16 or bfloat16, not {tensor.dtype}")
    return code


def launch_stream(stream, *tensors) -> int:
    """The raw stream to launch on: `stream`, or the current one; every tensor must lie on the current device."""
    device = tensors[0].get_device()
    for tensor in tensors:
        if tensor.get_device() != device:
            raise ValueError(f"tensors must lie on one device, {tensors[0].device}, not {tensor.device}")
    if device < 0 or device != torch._C._cuda_getDevice():
        raise ValueError(f"tensors must lie on the current HIP device, not {tensors[0].device}")
    if stream is None:
        return torch._C._cuda_getCurrentRawStream(device)
    if stream.device_index != device:
        raise ValueError(f"the stream must be of the tensors' device, {tensors[0].device}, not {stream.device}")
    return stream.cuda_stream


def allocate(shape, dtype, device, stream):
    """A new tensor of the memory of the stream that the call runs on: the current stream's may be memory that it
    still uses for earlier work, or hands out again before the call's work is done."""
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=device)
    with torch.cuda.stream(stream):
        return torch.empty(shape, dtype=dtype, device=device)


def library():
    return _native._library or _native.load()


def strided_rows(tensor, what: str) -> tuple[int, int, int, int]:
    """(rows, columns, row stride, elements spanned) of a 2-D tensor with contiguous rows."""
    if tensor.dim() != 2:
        raise ValueError(f"{what} must have two dimensions, not {tensor.dim()}")
    rows, columns = tensor.shape
    stride, step = tensor.stride()
    if columns > 1 and step != 1:
        raise ValueError(f"{what} must have contiguous rows (a stride of 1 along its last dimension)")
    if rows > 1 and columns:
        return rows, columns, stride, (rows - 1) * stride + columns
    return rows, columns, columns, rows * columns


def check_tensor(tensor, what: str, shape, dtype) -> None:
    if tensor.shape != shape or tensor.dtype is not dtype or not tensor.is_contiguous():
        raise ValueError(f"{what} must be a contiguous {dtype} tensor of {tuple(shape)}, not {tensor.dtype} of "
                         f"{tuple(tensor.shape)}")


def check_output(tensor, what: str, shape, dtype, like, stream):
    """`tensor`, checked, or a new one on the device of `like` in its place."""
    if tensor is None:
        return allocate(shape, dtype, like.device, stream)
    check_tensor(tensor, what, shape, dtype)
    return tensor


def empty(rows: int, k: int, device="cuda", experts: int | None = None, stream=None) -> Packed:
    """An operand's buffers, for `quantize` to fill."""
    lead = () if experts is None else (experts,)
    return Packed(allocate((*lead, rows, -(-k // GROUP) * (GROUP // 2)), torch.uint8, device, stream),
                  allocate((*lead, -(-k // STEP), rows, STEP // GROUP), torch.uint8, device, stream), k)


def _check_experts(packed: Packed, what: str, experts: int | None) -> None:
    if packed.experts != experts:
        raise ValueError(f"{what} must hold {'one matrix' if experts is None else f'a matrix for each of {experts} experts'},"
                         f" not codes of {tuple(packed.codes.shape)}")


def quantize(x, packed: Packed | None = None, columns: bool = False, stream=None) -> Packed:
    """The MXFP4 operand of x's rows; with `columns`, of its columns (x transposed, groups along its rows)."""
    code = dtype_code(x, "x")
    x_rows, x_columns, stride, span = strided_rows(x, "x")
    rows, k = (x_columns, x_rows) if columns else (x_rows, x_columns)
    if packed is None:
        packed = empty(rows, k, x.device, stream=stream)
    _check_experts(packed, "packed", None)
    if packed.rows != rows or packed.k != k:
        raise ValueError(f"packed must be an operand of {rows} x {k}, not {packed.rows} x {packed.k}")
    codes, scales = packed.codes, packed.scales
    handle = launch_stream(stream, x, codes, scales)
    span *= 2 if code else 4
    if columns:
        status = library().mb_mx_quantize_columns(code, x.data_ptr(), span, x_rows, x_columns, stride,
                                                  codes.data_ptr(), codes.numel(), scales.data_ptr(), scales.numel(),
                                                  handle)
    else:
        status = library().mb_mx_quantize(code, x.data_ptr(), span, rows, k, stride, None, 0, 1, rows,
                                          codes.data_ptr(), codes.numel(), scales.data_ptr(), scales.numel(), handle)
    if status:
        _native.check(status)
    return packed


def dequantize(packed: Packed, out=None, stream=None):
    """The values of an operand [rows][k]: bfloat16 (exact) unless `out` is of another type."""
    _check_experts(packed, "packed", None)
    codes, scales, rows, k = packed.codes, packed.scales, packed.rows, packed.k
    out = check_output(out, "out", (rows, k), torch.bfloat16 if out is None else out.dtype, codes, stream)
    code = dtype_code(out, "out")
    handle = launch_stream(stream, codes, scales, out)
    status = library().mb_mx_dequantize(code, codes.data_ptr(), codes.numel(), scales.data_ptr(), scales.numel(),
                                        out.data_ptr(), rows * k * (2 if code else 4), rows, k, handle)
    if status:
        _native.check(status)
    return out


def product_kernel(rows: int, n: int, k: int, dtype=torch.bfloat16, experts: int = 1, linear: bool = False) -> str:
    """Name of the kernel that `product` (with `linear`, `linear` for `rows` rows of output) launches."""
    code = DTYPE_CODES.get(dtype, -1)
    name = library().mb_mx_product_kernel(code, rows, n, k, experts, int(linear))
    if name is None:
        raise _native.NativeError(_native.MB_ERR_INVALID, _native.last_error())
    return name.decode()


def product(a: Packed, b: Packed, out=None, dtype=None, offsets=None, stream=None, kernel: str | None = None):
    """A . B^T of two operands, in `dtype` (bfloat16 unless `out` or `dtype` says otherwise).

    With `offsets` ([experts + 1] int32, on the device) b holds a matrix for each expert, and a's rows offsets[e] ..
    offsets[e + 1] - 1 meet matrix e; output rows from offsets[experts] on are not written. `kernel` names the kernel
    to run on, for tests and measurements.
    """
    experts = None if offsets is None else offsets.numel() - 1
    _check_experts(a, "a", None)
    _check_experts(b, "b", experts)
    if a.k != b.k:
        raise ValueError(f"a and b must have the same k, not {a.k} and {b.k}")
    if dtype is None:
        dtype = torch.bfloat16 if out is None else out.dtype
    out = check_output(out, "out", (a.rows, b.rows), dtype, a.codes, stream)
    code = dtype_code(out, "out")
    _check_indices(offsets, "offsets")
    handle = launch_stream(stream, a.codes, a.scales, b.codes, b.scales, out, *(() if offsets is None else (offsets,)))
    arguments = (code, a.codes.data_ptr(), a.codes.numel(), a.scales.data_ptr(), a.scales.numel(), b.codes.data_ptr(),
                 b.codes.numel(), b.scales.data_ptr(), b.scales.numel(), out.data_ptr(),
                 a.rows * b.rows * (2 if code else 4), a.rows, b.rows, a.k, *_pointer(offsets), experts or 1, handle)
    if kernel is None:
        status = library().mb_mx_product(*arguments)
    else:
        status = library().mb_mx_product_exact(kernel.encode(), *arguments)
    if status:
        _native.check(status)
    return out


def _check_indices(tensor, what: str) -> None:
    if tensor is not None and (tensor.dtype is not torch.int32 or not tensor.is_contiguous()):
        raise ValueError(f"{what} must be a contiguous int32 tensor, not {tensor.dtype}")


def _pointer(tensor) -> tuple[int | None, int]:
    return (None, 0) if tensor is None else (tensor.data_ptr(), 4 * tensor.numel())


def _workspace(tensor, needed: int, like, stream):
    if tensor is None:
        return allocate(needed, torch.uint8, like.device, stream)
    if tensor.dtype is not torch.uint8 or not tensor.is_contiguous() or tensor.numel() < needed:
        raise ValueError(f"workspace must be a contiguous uint8 tensor of at least {needed} bytes")
    return tensor


def linear_workspace(rows: int, n: int, k: int, dtype, experts: int = 1, device="cuda"):
    """A workspace for `linear` with `rows` output rows (routed ones, with a plan)."""
    return torch.empty(library().mb_mx_linear_workspace(rows, n, k), dtype=torch.uint8, device=device)


def linear(x, weight: Packed, out=None, plan=None, sorted_rows: bool = False, workspace=None, stream=None):
    """Q(x) . W^T in x's type: x [rows][k], weight an operand of n rows, out [rows][n].

    With a `plan` (routing.dispatch) the weight holds a matrix for each expert: x [tokens][k] gives the routed rows
    out [tokens * top][n] in the plan's order, or, `sorted_rows`, x's rows are routed rows in that order already. Rows
    from plan.offsets[experts] on are not written.
    """
    code = dtype_code(x, "x")
    rows, k, stride, span = strided_rows(x, "x")
    offsets = order = slots = None
    copies, experts, indices = 1, None, ()
    if plan is not None:
        offsets = plan.offsets
        experts, indices = offsets.numel() - 1, (offsets,)
        _check_indices(offsets, "plan.offsets")
        if not sorted_rows:
            order, slots = plan.order, plan.slots
            _check_indices(order, "plan.order")
            _check_indices(slots, "plan.slots")
            if slots.dim() != 2 or slots.shape[0] != rows or order.numel() != slots.numel():
                raise ValueError(f"the plan must route {rows} tokens, not slots of {tuple(slots.shape)}")
            copies, indices = slots.shape[1], (offsets, order, slots)
    elif sorted_rows:
        raise ValueError("sorted rows need the plan that they are sorted by")
    _check_experts(weight, "weight", experts)
    if weight.k != k:
        raise ValueError(f"the weight must have k = {k}, not {weight.k}")
    n, routed, codes, scales = weight.rows, rows * copies, weight.codes, weight.scales
    out = check_output(out, "out", (routed, n), x.dtype, x, stream)
    native = library()
    workspace = _workspace(workspace, native.mb_mx_linear_workspace(routed, n, k), x, stream)
    handle = launch_stream(stream, x, codes, scales, out, workspace, *indices)
    item = 2 if code else 4
    status = native.mb_mx_linear(
        code, x.data_ptr(), span * item, rows, stride, codes.data_ptr(), codes.numel(), scales.data_ptr(),
        scales.numel(), out.data_ptr(), routed * n * item, n, k, *_pointer(offsets),
        None if order is None else order.data_ptr(), *_pointer(slots), copies, experts or 1, workspace.data_ptr(),
        workspace.numel(), handle)
    if status:
        _native.check(status)
    return out


def linear_backward_workspace(rows: int, n: int, k: int, dtype, device="cuda"):
    """A workspace for `linear_backward`, and for `linear` of the same sizes."""
    native = library()
    return torch.empty(max(native.mb_mx_linear_backward_workspace(rows, n, k),
                           native.mb_mx_linear_workspace(rows, n, k)), dtype=torch.uint8, device=device)


def linear_backward(d_out, x, weight_columns: Packed, d_x=None, d_weight=None, workspace=None, stream=None):
    """(d_x, d_weight) of out = Q(x) . Q(w)^T for the gradient d_out [rows][n], in x's type.

    d_x = Q(d_out) . W with `weight_columns` = quantize(w, columns=True); d_weight = d_out^T . x, both quantised
    along the rows that the sum runs over.
    """
    code = dtype_code(x, "x")
    rows, n, d_stride, d_span = strided_rows(d_out, "d_out")
    x_rows, k, x_stride, x_span = strided_rows(x, "x")
    if d_out.dtype is not x.dtype or x_rows != rows:
        raise ValueError(f"d_out and x must be of one type and number of rows, not {d_out.dtype} of "
                         f"{tuple(d_out.shape)} and {x.dtype} of {tuple(x.shape)}")
    _check_experts(weight_columns, "weight_columns", None)
    if weight_columns.rows != k or weight_columns.k != n:
        raise ValueError(f"weight_columns must be an operand of {k} x {n} (the weight quantised by columns), not "
                         f"{weight_columns.rows} x {weight_columns.k}")
    d_x = check_output(d_x, "d_x", (rows, k), x.dtype, x, stream)
    d_weight = check_output(d_weight, "d_weight", (n, k), x.dtype, x, stream)
    if not rows or not n or not k:
        launch_stream(stream, d_out, x, weight_columns.codes, weight_columns.scales, d_x, d_weight)
        with torch.cuda.stream(stream):  # cleared in the order of the call's work
            return d_x.zero_(), d_weight.zero_()
    native = library()
    workspace = _workspace(workspace, native.mb_mx_linear_backward_workspace(rows, n, k), x, stream)
    codes, scales = weight_columns.codes, weight_columns.scales
    handle = launch_stream(stream, d_out, x, codes, scales, d_x, d_weight, workspace)
    item = 2 if code else 4
    status = native.mb_mx_linear_backward(
        code, d_out.data_ptr(), d_span * item, d_stride, x.data_ptr(), x_span * item, x_stride, codes.data_ptr(),
        codes.numel(), scales.data_ptr(), scales.numel(), d_x.data_ptr(), rows * k * item, d_weight.data_ptr(),
        n * k * item, rows, n, k, workspace.data_ptr(), workspace.numel(), handle)
    if status:
        _native.check(status)
    return d_x, d_weight
