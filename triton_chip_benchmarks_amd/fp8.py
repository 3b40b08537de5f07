"""FP8 operands with block scales, linear layers and the gated pair of projections.

An operand (`Packed`) holds E4M3 codes and one power-of-two scale for each block of
128 along K, of one row (activations) or of 128 rows (weights). `quantize` makes one
of a tensor's rows or columns, `quantize_both` of both in one pass, `dequantize`
gives its values back. `product` multiplies two, `linear` a tensor, quantised on the
way, with a weight laid out once (one, or one for each expert that `routing.dispatch`
sorted the rows by), and `gated` computes silu(x . G^T) * (x . U^T) in one kernel. A
training step calls `linear_backward` and `gated_backward`, whose products take the
gradient and the saved input in FP8 too (straight through: quantisation has the
identity's gradient).

Every call launches on the current stream, allocates only the outputs and workspaces
that it is not given, and raises ValueError for tensors that do not fit it.
"""

from __future__ import annotations

import torch

from . import _native
from .mx import (DTYPE_CODES, _check_indices, _pointer, _workspace, allocate, check_output, check_tensor, dtype_code,
                 launch_stream, library, strided_rows)

BLOCK = 128  # elements along K that share a scale, and rows of a weight that do
STEP = 512   # K elements whose scales a row holds together


class Packed:
    """An operand of rows x k: codes [rows][k rounded up to 16], float8_e4m3fn, and scales [ceil(k/512)][ceil(rows /
    block)][4], uint8 (E8M0), contiguous; `block` rows, 1 or 128, share a scale. With a leading dimension each, one such
    matrix for each of `experts`."""

    __slots__ = ("codes", "scales", "k", "rows", "block", "experts")

    def __init__(self, codes, scales, k: int, block: int = 1):
        if block not in (1, BLOCK):
            raise ValueError(f"a scale stands for 1 or {BLOCK} rows, not {block}")
        lead = codes.shape[:-2]
        rows = codes.shape[-2] if codes.dim() >= 2 else -1
        if (codes.dtype != torch.float8_e4m3fn or scales.dtype != torch.uint8 or len(lead) > 1
                or not codes.is_contiguous() or not scales.is_contiguous() or codes.shape != (*lead, rows, _pitch(k))
                or scales.shape != (*lead, -(-k // STEP), -(-rows // block), STEP // BLOCK)):
            raise ValueError(f"an operand of k = {k} has contiguous float8_e4m3fn codes [rows][{_pitch(k)}] and uint8 "
                             f"scales [{-(-k // STEP)}][ceil(rows/{block})][4], not {tuple(codes.shape)} of "
                             f"{codes.dtype} and {tuple(scales.shape)} of {scales.dtype}")
        self.codes, self.scales, self.k, self.rows, self.block = codes, scales, k, rows, block
        self.experts = lead[0] if lead else None


def _pitch(k: int) -> int:
    return -(-k // 16) * 16


def empty(rows: int, k: int, block: int = 1, device="cuda", experts: int | None = None, stream=None) -> Packed:
    """An operand's buffers, for `quantize` to fill."""
    if block not in (1, BLOCK):
        raise ValueError(f"a scale stands for 1 or {BLOCK} rows, not {block}")
    lead = () if experts is None else (experts,)
    return Packed(allocate((*lead, rows, _pitch(k)), torch.float8_e4m3fn, device, stream),
                  allocate((*lead, -(-k // STEP), -(-rows // block), STEP // BLOCK), torch.uint8, device, stream), k,
                  block)


def _check_experts(packed: Packed, what: str, experts: int | None) -> None:
    if packed.experts != experts:
        wanted = "one matrix" if experts is None else f"a matrix for each of {experts} experts"
        raise ValueError(f"{what} must hold {wanted}, not codes of {tuple(packed.codes.shape)}")


def _operand(packed: Packed | None, what: str, rows: int, k: int, block: int, like, stream) -> Packed:
    """`packed`, checked, or a new one in its place."""
    if packed is None:
        return empty(rows, k, block, like.device, stream=stream)
    _check_experts(packed, what, None)
    if packed.rows != rows or packed.k != k or packed.block != block:
        raise ValueError(f"{what} must be an operand of {rows} x {k} with a scale for {block} rows, not {packed.rows} "
                         f"x {packed.k} with one for {packed.block}")
    return packed


def _parts(packed: Packed) -> tuple[int, int, int, int]:
    return packed.codes.data_ptr(), packed.codes.numel(), packed.scales.data_ptr(), packed.scales.numel()


def quantize(x, packed: Packed | None = None, columns: bool = False, block: int = 1, stream=None) -> Packed:
    """The operand of x's rows; with `columns`, of its columns (x transposed, blocks along its rows). `block` rows of
    the operand, 1 or 128, share a scale."""
    code = dtype_code(x, "x")
    x_rows, x_columns, stride, span = strided_rows(x, "x")
    rows, k = (x_columns, x_rows) if columns else (x_rows, x_columns)
    packed = _operand(packed, "packed", rows, k, block, x, stream)
    handle = launch_stream(stream, x, packed.codes, packed.scales)
    span *= 2 if code else 4
    if columns or block != 1:
        outputs = (None, 0, None, 0, *_parts(packed)) if columns else (*_parts(packed), None, 0, None, 0)
        status = library().mb_fp8_quantize_both(code, x.data_ptr(), span, x_rows, x_columns, stride, block, *outputs,
                                                handle)
    else:
        status = library().mb_fp8_quantize(code, x.data_ptr(), span, rows, k, stride, None, 0, 1, rows,
                                           *_parts(packed), handle)
    if status:
        _native.check(status)
    return packed


def quantize_both(x, rows: Packed | None = None, columns: Packed | None = None, block: int = 1,
                  stream=None) -> tuple[Packed, Packed]:
    """The operands of x's rows and of its columns, in one pass: of a weight with `block` 128 both hold the same
    values."""
    code = dtype_code(x, "x")
    x_rows, x_columns, stride, span = strided_rows(x, "x")
    rows = _operand(rows, "rows", x_rows, x_columns, block, x, stream)
    columns = _operand(columns, "columns", x_columns, x_rows, block, x, stream)
    handle = launch_stream(stream, x, rows.codes, rows.scales, columns.codes, columns.scales)
    status = library().mb_fp8_quantize_both(code, x.data_ptr(), span * (2 if code else 4), x_rows, x_columns, stride,
                                            block, *_parts(rows), *_parts(columns), handle)
    if status:
        _native.check(status)
    return rows, columns


def dequantize(packed: Packed, out=None, stream=None):
    """The values of an operand [rows][k]: bfloat16 unless `out` is of another type."""
    _check_experts(packed, "packed", None)
    rows, k = packed.rows, packed.k
    out = check_output(out, "out", (rows, k), torch.bfloat16 if out is None else out.dtype, packed.codes, stream)
    code = dtype_code(out, "out")
    handle = launch_stream(stream, packed.codes, packed.scales, out)
    status = library().mb_fp8_dequantize(code, *_parts(packed), packed.block, out.data_ptr(),
                                         rows * k * (2 if code else 4), rows, k, handle)
    if status:
        _native.check(status)
    return out


KINDS = {"product": 0, "gated": 1, "gated_kept": 2, "gated_fp8": 3}


def product_kernel(rows: int, n: int, k: int, dtype=torch.bfloat16, experts: int = 1, linear: bool = False,
                   kind: str = "product") -> str:
    """Name of the kernel that `product` or, by `kind`, `gated` (with gate_up, or to an operand) of an operand launches;
    with `linear`, `linear` or `gated` of a tensor for `rows` rows of output."""
    name = library().mb_fp8_product_kernel(DTYPE_CODES.get(dtype, -1), rows, n, k, experts, int(linear), KINDS[kind])
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
    _check_product(a, b, experts)
    if dtype is None:
        dtype = torch.bfloat16 if out is None else out.dtype
    out = check_output(out, "out", (a.rows, b.rows), dtype, a.codes, stream)
    code = dtype_code(out, "out")
    _check_indices(offsets, "offsets")
    handle = launch_stream(stream, a.codes, a.scales, b.codes, b.scales, out, *(() if offsets is None else (offsets,)))
    status = library().mb_fp8_product(code, *_parts(a), a.block, *_parts(b), b.block, out.data_ptr(),
                                      a.rows * b.rows * (2 if code else 4), a.rows, b.rows, a.k, *_pointer(offsets),
                                      experts or 1, None if kernel is None else kernel.encode(), handle)
    if status:
        _native.check(status)
    return out


def _check_product(a: Packed, b: Packed, experts: int | None) -> None:
    _check_experts(a, "a", None)
    _check_experts(b, "b", experts)
    if a.k != b.k:
        raise ValueError(f"a and b must have the same k, not {a.k} and {b.k}")
    if experts is not None and a.block != 1:
        raise ValueError("rows of several experts have a scale each")


def _routes(plan, rows: int, sorted_rows: bool):
    """What a call takes from a plan: (experts, copies of a row, tensors, the C arguments)."""
    if plan is None:
        if sorted_rows:
            raise ValueError("sorted rows need the plan that they are sorted by")
        return None, 1, (), (None, 0, None, None, 0, 1, 1)
    offsets, order, slots = plan.offsets, plan.order, plan.slots
    _check_indices(offsets, "plan.offsets")
    experts = offsets.numel() - 1
    if sorted_rows:
        return experts, 1, (offsets,), (*_pointer(offsets), None, None, 0, 1, experts)
    _check_indices(order, "plan.order")
    _check_indices(slots, "plan.slots")
    if slots.dim() != 2 or slots.shape[0] != rows or order.numel() != slots.numel():
        raise ValueError(f"the plan must route {rows} tokens, not slots of {tuple(slots.shape)}")
    copies = slots.shape[1]
    return (experts, copies, (offsets, order, slots),
            (*_pointer(offsets), order.data_ptr(), *_pointer(slots), copies, experts))


def linear_workspace(rows: int, n: int, k: int, dtype, experts: int = 1, device="cuda"):
    """A workspace for `linear` with `rows` output rows (routed ones, with a plan); for every n, type and number of experts
    the same."""
    return torch.empty(library().mb_fp8_linear_workspace(rows, n, k), dtype=torch.uint8, device=device)


def linear(x, weight: Packed, out=None, plan=None, sorted_rows: bool = False, workspace=None, stream=None):
    """Q(x) . W^T in x's type: x [rows][k], weight an operand of n rows, out [rows][n].

    With a `plan` (routing.dispatch) the weight holds a matrix for each expert: x [tokens][k] gives the routed rows
    out [tokens * top][n] in the plan's order, or, `sorted_rows`, x's rows are routed rows in that order already. Rows
    from plan.offsets[experts] on are not written.
    """
    code = dtype_code(x, "x")
    rows, k, stride, span = strided_rows(x, "x")
    experts, copies, indices, routes = _routes(plan, rows, sorted_rows)
    _check_experts(weight, "weight", experts)
    if weight.k != k:
        raise ValueError(f"the weight must have k = {k}, not {weight.k}")
    n, routed = weight.rows, rows * copies
    out = check_output(out, "out", (routed, n), x.dtype, x, stream)
    native = library()
    workspace = _workspace(workspace, native.mb_fp8_linear_workspace(routed, n, k), x, stream)
    handle = launch_stream(stream, x, weight.codes, weight.scales, out, workspace, *indices)
    item = 2 if code else 4
    status = native.mb_fp8_linear(code, x.data_ptr(), span * item, rows, stride, *_parts(weight), weight.block,
                                  out.data_ptr(), routed * n * item, n, k, *routes, workspace.data_ptr(),
                                  workspace.numel(), handle)
    if status:
        _native.check(status)
    return out


def linear_backward_workspace(rows: int, n: int, k: int, dtype, device="cuda"):
    """A workspace for `linear_backward`, and for `linear` of the same sizes."""
    native = library()
    return torch.empty(max(native.mb_fp8_linear_backward_workspace(rows, n, k),
                           native.mb_fp8_linear_workspace(rows, n, k)), dtype=torch.uint8, device=device)


def _backward(name: str, d_out, gate_up, x, weight_columns: Packed, d_x, d_weight, workspace, stream):
    """(d_x, d_weight) of `linear` or, with gate_up, of `gated`."""
    code = dtype_code(x, "x")
    rows, n, d_stride, d_span = strided_rows(d_out, "d_out")
    x_rows, k, x_stride, x_span = strided_rows(x, "x")
    if d_out.dtype is not x.dtype or x_rows != rows:
        raise ValueError(f"d_out and x must be of one type and number of rows, not {d_out.dtype} of "
                         f"{tuple(d_out.shape)} and {x.dtype} of {tuple(x.shape)}")
    width, saved = n, ()
    if gate_up is not None:
        width, saved = 2 * n, (gate_up,)
        check_tensor(gate_up, "gate_up", (rows, width), x.dtype)
    _check_experts(weight_columns, "weight_columns", None)
    if weight_columns.rows != k or weight_columns.k != width:
        raise ValueError(f"weight_columns must be an operand of {k} x {width} (the weight quantised by columns), not "
                         f"{weight_columns.rows} x {weight_columns.k}")
    d_x = check_output(d_x, "d_x", (rows, k), x.dtype, x, stream)
    d_weight = check_output(d_weight, "d_weight", (width, k), x.dtype, x, stream)
    if not rows or not n or not k:
        launch_stream(stream, d_out, x, weight_columns.codes, weight_columns.scales, d_x, d_weight, *saved)
        with torch.cuda.stream(stream):  # cleared in the order of the call's work
            return d_x.zero_(), d_weight.zero_()
    native = library()
    workspace = _workspace(workspace, getattr(native, name + "_workspace")(rows, n, k), x, stream)
    handle = launch_stream(stream, d_out, x, weight_columns.codes, weight_columns.scales, d_x, d_weight, workspace,
                           *saved)
    item = 2 if code else 4
    kept = (gate_up.data_ptr(), rows * width * item) if saved else ()
    status = getattr(native, name)(code, d_out.data_ptr(), d_span * item, d_stride, *kept, x.data_ptr(), x_span * item,
                                   x_stride, *_parts(weight_columns), weight_columns.block, d_x.data_ptr(),
                                   rows * k * item, d_weight.data_ptr(), width * k * item, rows, n, k,
                                   workspace.data_ptr(), workspace.numel(), handle)
    if status:
        _native.check(status)
    return d_x, d_weight


def linear_backward(d_out, x, weight_columns: Packed, d_x=None, d_weight=None, workspace=None, stream=None):
    """(d_x, d_weight) of out = Q(x) . Q(w)^T for the gradient d_out [rows][n], in x's type.

    d_x = Q(d_out) . W with `weight_columns`, the operand of w's columns; d_weight = d_out^T . x, both quantised along
    the rows that the sum runs over.
    """
    return _backward("mb_fp8_linear_backward", d_out, None, x, weight_columns, d_x, d_weight, workspace, stream)


def gated_workspace(rows: int, n: int, k: int, dtype, experts: int = 1, device="cuda"):
    """A workspace for `gated` with `rows` output rows (routed ones, with a plan)."""
    return linear_workspace(rows, n, k, dtype, experts, device)


def gated(x, weight: Packed, out=None, packed: Packed | None = None, gate_up=None, plan=None,
          sorted_rows: bool = False, dtype=None, workspace=None, stream=None, kernel: str | None = None):
    """silu(x . G^T) * (x . U^T): x [rows][k], a tensor, quantised on the way, or an operand; weight an operand of 2n
    rows, G's and then U's (with a `plan`, a matrix for each expert, as for `linear`; an operand's rows are sorted).

    The result, rounded once from fp32, is `out` [rows][n] of x's type (of an operand: of `dtype`, bfloat16 unless
    given) or, if `packed` is given, that operand, with a scale for each row's 128, its sums those of 16-bit outputs
    whatever x's type (`quantize` of an fp32 `out` has fp32's). `gate_up` [rows][2n], if given, gets
    [x . G^T | x . U^T], which `gated_backward` takes. `kernel` names the kernel to run an operand on, for tests and
    measurements.
    """
    operand = isinstance(x, Packed)
    if operand:
        _check_experts(x, "x", None)
        rows, k, like = x.rows, x.k, x.codes
        dtype = dtype or (torch.bfloat16 if out is None else out.dtype)
        code = _code(dtype)
        if plan is not None and not sorted_rows:
            raise ValueError("an operand's rows are not gathered: they must be sorted by the plan")
    else:
        code = dtype_code(x, "x")
        if dtype is not None and dtype is not x.dtype:
            raise ValueError(f"the output of a tensor of {x.dtype} is of its type, not {dtype}")
        rows, k, stride, span = strided_rows(x, "x")
        like, dtype = x, x.dtype
    experts, copies, indices, routes = _routes(plan, rows, sorted_rows)
    _check_experts(weight, "weight", experts)
    if operand:
        _check_product(x, weight, experts)
    if kernel is not None and not operand:
        raise ValueError("a kernel is named for an operand, not for a tensor")
    if weight.k != k or weight.rows % 2:
        raise ValueError(f"the weight must have k = {k} and an even number of rows, not {weight.k} and {weight.rows}")
    n, routed, item = weight.rows // 2, rows * copies, 2 if code else 4
    if packed is None:
        result = out = check_output(out, "out", (routed, n), dtype, like, stream)
        output, tensors = (out.data_ptr(), routed * n * item, None, 0), (out,)
    else:
        if out is not None or gate_up is not None:
            raise ValueError("the output goes to out or to packed, and gate_up beside out alone")
        result = _operand(packed, "packed", routed, n, 1, like, stream)
        output, tensors = _parts(packed), (packed.codes, packed.scales)
    saved = (None, 0)
    if gate_up is not None:
        check_tensor(gate_up, "gate_up", (routed, 2 * n), dtype)
        saved, tensors = (gate_up.data_ptr(), routed * 2 * n * item), (*tensors, gate_up)
    native = library()
    if operand:
        handle = launch_stream(stream, like, x.scales, weight.codes, weight.scales, *tensors, *indices)
        offsets, size = routes[:2]
        status = native.mb_fp8_gated_product(code, *_parts(x), x.block, *_parts(weight), weight.block, *output, *saved,
                                             rows, n, k, offsets, size, experts or 1,
                                             None if kernel is None else kernel.encode(), handle)
    else:
        workspace = _workspace(workspace, native.mb_fp8_linear_workspace(routed, n, k), x, stream)
        handle = launch_stream(stream, x, weight.codes, weight.scales, workspace, *tensors, *indices)
        status = native.mb_fp8_gated(code, x.data_ptr(), span * item, rows, stride, *_parts(weight), weight.block,
                                     *output, *saved, n, k, *routes, workspace.data_ptr(), workspace.numel(),
                                     handle)
    if status:
        _native.check(status)
    return result


def _code(dtype) -> int:
    code = DTYPE_CODES.get(dtype)
    if code is None:
        raise ValueError(f"the output must be float32, float16 or bfloat16, not {dtype}")
    return code


def gated_backward_workspace(rows: int, n: int, k: int, dtype, device="cuda"):
    """A workspace for `gated_backward`, and for `gated` of the same sizes."""
    native = library()
    return torch.empty(max(native.mb_fp8_gated_backward_workspace(rows, n, k),
                           native.mb_fp8_linear_workspace(rows, n, k)), dtype=torch.uint8, device=device)


def gated_backward(d_out, gate_up, x, weight_columns: Packed, d_x=None, d_weight=None, workspace=None, stream=None):
    """(d_x, d_weight) of out = gated(x, w, gate_up=gate_up) for the gradient d_out [rows][n], in x's type.

    `weight_columns` is the operand of w's columns, w [2n][k]; the gradient of [gate | up] is quantised from fp32, and
    meets it and x as in `linear_backward`.
    """
    if gate_up is None:
        raise ValueError("the gradient needs the gate_up that gated kept")
    return _backward("mb_fp8_gated_backward", d_out, gate_up, x, weight_columns, d_x, d_weight, workspace, stream)
