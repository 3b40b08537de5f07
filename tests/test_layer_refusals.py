"""What the layer operators refuse, on the host and before any launch (pointers here are never dereferenced)."""

import pytest
import torch

from triton_chip_benchmarks_amd import _native, mx, routing

INVALID, UNSUPPORTED, ALIGNMENT = _native.MB_ERR_INVALID, _native.MB_ERR_UNSUPPORTED, _native.MB_ERR_ALIGNMENT
P, BIG = 1 << 20, 1 << 40


def refused(code, name, *arguments, match):
    status = getattr(_native.load(), name)(*arguments)
    assert status == code and match in _native.last_error(), (status, _native.last_error())


def test_quantize():
    # dtype, x, x_bytes, rows, k, row_stride, slots, slots_bytes, copies, out_rows, codes, bytes, scales, bytes, stream
    call = lambda dtype=2, x=P, x_bytes=64 * 32 * 2, rows=64, k=32, stride=32, slots=None, slots_bytes=0, copies=1, out=64, codes=P, codes_bytes=64 * 16, scales=P, scales_bytes=64 * 8: (  # noqa: E731,E501
        dtype, x, x_bytes, rows, k, stride, slots, slots_bytes, copies, out, codes, codes_bytes, scales, scales_bytes,
        None)
    name = "mb_mx_quantize"
    refused(INVALID, name, *call(dtype=3), match="element type")
    refused(INVALID, name, *call(x=None), match="x is NULL")
    refused(INVALID, name, *call(x_bytes=64 * 32 * 2 - 1), match="too small")
    refused(INVALID, name, *call(stride=33), match="too small")
    refused(INVALID, name, *call(stride=1 << 62), match="too small")
    refused(ALIGNMENT, name, *call(x=P + 1), match="elements")
    refused(ALIGNMENT, name, *call(codes=P + 8), match="16 bytes")
    refused(INVALID, name, *call(codes_bytes=64 * 16 - 1), match="too small")
    refused(INVALID, name, *call(scales_bytes=64 * 8 - 1), match="too small")
    refused(UNSUPPORTED, name, *call(rows=(1 << 24) + 1), match="at most")
    refused(INVALID, name, *call(slots=P, slots_bytes=64 * 2 * 4 - 1, copies=2), match="slots")
    refused(INVALID, name, *call(slots=P, slots_bytes=BIG, copies=65), match="slots")
    assert _native.load().mb_mx_quantize(*call(rows=0, x=None, codes=None)) == _native.MB_OK
    refused(INVALID, name, *call(rows=0, dtype=9), match="element type")


def test_quantize_columns_and_dequantize():
    refused(INVALID, "mb_mx_quantize_columns", 2, P, 63 * 64 * 2, 64, 64, 64, P, BIG, P, BIG, None, match="too small")
    refused(UNSUPPORTED, "mb_mx_quantize_columns", 2, P, BIG, 1 << 21, 4, 4, P, BIG, P, BIG, None, match="at most")
    refused(INVALID, "mb_mx_dequantize", 2, P, BIG, P, BIG, P, 64 * 32 * 2 - 1, 64, 32, None, match="too small")
    refused(INVALID, "mb_mx_dequantize", 2, P, 64 * 16 - 1, P, BIG, P, BIG, 64, 32, None, match="too small")
    refused(INVALID, "mb_mx_dequantize", 7, P, BIG, P, BIG, P, BIG, 64, 32, None, match="element type")


def test_product_and_linear():
    product = lambda dtype=2, rows=8, n=64, k=32, offsets=None, offsets_bytes=0, experts=1, c=P, c_bytes=8 * 64 * 2, a_bytes=BIG, b_bytes=BIG: (  # noqa: E731,E501
        dtype, P, a_bytes, P, BIG, P, b_bytes, P, BIG, c, c_bytes, rows, n, k, offsets, offsets_bytes, experts, None)
    refused(INVALID, "mb_mx_product", *product(dtype=-1), match="element type")
    refused(INVALID, "mb_mx_product", *product(experts=2), match="offsets")
    refused(INVALID, "mb_mx_product", *product(experts=0), match="experts")
    refused(INVALID, "mb_mx_product", *product(experts=2, offsets=P, offsets_bytes=8), match="offsets")
    refused(INVALID, "mb_mx_product", *product(k=0), match="K must be positive")
    refused(INVALID, "mb_mx_product", *product(c_bytes=8 * 64 * 2 - 1), match="output")
    refused(INVALID, "mb_mx_product", *product(a_bytes=8 * 16 - 1), match="too small")
    refused(INVALID, "mb_mx_product", *product(experts=2, offsets=P, offsets_bytes=12, b_bytes=2 * 64 * 16 - 1),
            match="too small")
    assert _native.load().mb_mx_product(*product(rows=0, c=None)) == _native.MB_OK
    linear = lambda tokens=8, offsets=None, order=None, slots=None, copies=1, experts=1, workspace=P, workspace_bytes=BIG, y_bytes=BIG, x_bytes=BIG: (  # noqa: E731,E501
        2, P, x_bytes, tokens, 64, P, BIG, P, BIG, P, y_bytes, 64, 64, offsets, BIG if offsets else 0, order, slots,
        BIG if slots else 0, copies, experts, workspace, workspace_bytes, None)
    refused(INVALID, "mb_mx_linear", *linear(x_bytes=8 * 64 * 2 - 1), match="too small")
    refused(INVALID, "mb_mx_linear", *linear(y_bytes=8 * 64 * 2 - 1), match="output")
    refused(INVALID, "mb_mx_linear", *linear(workspace=None), match="workspace")
    refused(INVALID, "mb_mx_linear", *linear(workspace_bytes=15), match="workspace")
    refused(ALIGNMENT, "mb_mx_linear", *linear(workspace=P + 8), match="16 bytes")
    refused(INVALID, "mb_mx_linear", *linear(slots=P, copies=2), match="slots need")
    refused(INVALID, "mb_mx_linear", *linear(slots=P, offsets=P, order=P, copies=65), match="outside 1..64")


def test_linear_backward():
    call = lambda rows=8, d_out_bytes=8 * 64 * 2, x_bytes=8 * 96 * 2, d_x_bytes=8 * 96 * 2, d_w_bytes=64 * 96 * 2, workspace=P, workspace_bytes=BIG, w_bytes=BIG: (  # noqa: E731,E501
        2, P, d_out_bytes, 64, P, x_bytes, 96, P, w_bytes, P, BIG, P, d_x_bytes, P, d_w_bytes, rows, 64, 96, workspace,
        workspace_bytes, None)
    refused(INVALID, "mb_mx_linear_backward", *call(rows=0), match="positive")
    refused(INVALID, "mb_mx_linear_backward", *call(d_out_bytes=8 * 64 * 2 - 1), match="too small")
    refused(INVALID, "mb_mx_linear_backward", *call(x_bytes=8 * 96 * 2 - 1), match="too small")
    refused(INVALID, "mb_mx_linear_backward", *call(w_bytes=96 * 32 - 1), match="too small")
    refused(INVALID, "mb_mx_linear_backward", *call(d_x_bytes=8 * 96 * 2 - 1), match="output")
    refused(INVALID, "mb_mx_linear_backward", *call(d_w_bytes=64 * 96 * 2 - 1), match="output")
    needed = _native.load().mb_mx_linear_backward_workspace(8, 64, 96)
    refused(INVALID, "mb_mx_linear_backward", *call(workspace_bytes=needed - 1), match="workspace")
    refused(UNSUPPORTED, "mb_mx_linear_backward", *call(rows=(1 << 20) + 1, d_out_bytes=BIG, x_bytes=BIG,
                                                       d_x_bytes=BIG), match="at most")


def test_route():
    call = lambda dtype=0, logits=P, logits_bytes=4 * 16 * 4, tokens=4, experts=16, stride=16, bias=None, bias_bytes=0, top=2, scores=0, groups=1, top_groups=1, chosen=P, chosen_bytes=32, weights_bytes=32: (  # noqa: E731,E501
        dtype, logits, logits_bytes, tokens, experts, stride, bias, bias_bytes, top, scores, groups, top_groups, 1, 1.0,
        chosen, chosen_bytes, P, weights_bytes, None)
    refused(INVALID, "mb_route", *call(dtype=5), match="element type")
    refused(INVALID, "mb_route", *call(experts=1025), match="experts")
    refused(INVALID, "mb_route", *call(top=17), match="top")
    refused(INVALID, "mb_route", *call(top=0), match="top")
    refused(INVALID, "mb_route", *call(scores=2), match="scores")
    refused(INVALID, "mb_route", *call(groups=3), match="groups")
    refused(INVALID, "mb_route", *call(groups=4, top_groups=5), match="groups")
    refused(INVALID, "mb_route", *call(groups=8, top_groups=1, top=3), match="exceeds")
    refused(INVALID, "mb_route", *call(bias=P, bias_bytes=60), match="bias")
    refused(INVALID, "mb_route", *call(logits_bytes=255), match="too small")
    refused(INVALID, "mb_route", *call(chosen_bytes=31), match="too small")
    refused(INVALID, "mb_route", *call(weights_bytes=31), match="too small")
    refused(ALIGNMENT, "mb_route", *call(logits=P + 2), match="elements")
    backward = lambda d_bytes=256, top=2: (0, P, 256, 4, 16, 16, P, 32, P, 32, top, 0, 1, 1.0, P, d_bytes, None)  # noqa: E731
    refused(INVALID, "mb_route_backward", *backward(d_bytes=255), match="too small")
    refused(INVALID, "mb_route_backward", *backward(top=3), match="too small")


def test_dispatch_and_combine():
    dispatch = lambda entries=8, experts=4, offsets_bytes=20, order_bytes=32, workspace=None: (  # noqa: E731
        P, 4 * entries, entries, experts, P, offsets_bytes, P, order_bytes, P, 4 * entries, workspace, 0, None)
    refused(INVALID, "mb_dispatch", *dispatch(experts=1025), match="experts")
    refused(INVALID, "mb_dispatch", *dispatch(offsets_bytes=19), match="offsets")
    refused(INVALID, "mb_dispatch", *dispatch(order_bytes=31), match="too small")
    refused(UNSUPPORTED, "mb_dispatch", *dispatch(entries=(1 << 24) + 1), match="at most")
    refused(INVALID, "mb_dispatch", *dispatch(entries=100000, order_bytes=400000), match="workspace")
    combine = lambda dtype=2, y_bytes=8 * 64 * 2, slots_bytes=32, top=2, out_bytes=4 * 64 * 2: (  # noqa: E731
        dtype, P, y_bytes, 8, P, slots_bytes, P, 32, P, out_bytes, 4, top, 64, None)
    refused(INVALID, "mb_combine", *combine(dtype=4), match="element type")
    refused(INVALID, "mb_combine", *combine(y_bytes=8 * 64 * 2 - 1), match="too small")
    refused(INVALID, "mb_combine", *combine(slots_bytes=31), match="too small")
    refused(INVALID, "mb_combine", *combine(top=65), match="outside 1..64")
    refused(INVALID, "mb_combine", *combine(out_bytes=4 * 64 * 2 - 1), match="out is NULL")
    refused(INVALID, "mb_combine_backward", 2, P, BIG, P, BIG, 8, P, BIG, P, BIG, P, 15, P, BIG, 4, 2, 64, None,
            match="d_y")


def test_python_entry_points_refuse_tensors_that_do_not_fit():
    x = torch.zeros(4, 64)
    weight = mx.empty(32, 64, device="cpu")
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        mx.quantize(x.double())
    with pytest.raises(ValueError, match="contiguous rows"):
        mx.quantize(x.t())
    with pytest.raises(ValueError, match="two dimensions"):
        mx.quantize(x[0])
    with pytest.raises(ValueError, match="operand of 4 x 64"):
        mx.quantize(x, mx.empty(5, 64, device="cpu"))
    with pytest.raises(ValueError, match="contiguous uint8"):
        mx.quantize(x, mx.Packed(torch.zeros(4, 31, dtype=torch.uint8), torch.zeros(1, 4, 8, dtype=torch.uint8), 64))
    with pytest.raises(ValueError, match="k = 64"):
        mx.linear(x, mx.empty(32, 96, device="cpu"))
    with pytest.raises(ValueError, match="sorted rows need"):
        mx.linear(x, weight, sorted_rows=True)
    with pytest.raises(ValueError, match="out must be"):
        mx.linear(x, weight, torch.zeros(4, 31))
    plan = routing.Plan(torch.zeros(3, dtype=torch.int32), torch.zeros(8, dtype=torch.int32),
                        torch.zeros(5, 2, dtype=torch.int32))
    with pytest.raises(ValueError, match="route 4 tokens"):
        mx.linear(x, mx.empty(32, 64, device="cpu", experts=2), plan=plan)
    with pytest.raises(ValueError, match="the same k"):
        mx.product(weight, mx.empty(32, 96, device="cpu"))
    with pytest.raises(ValueError, match="weight_columns"):
        mx.linear_backward(torch.zeros(4, 32), x, weight)
    with pytest.raises(ValueError, match="one type and number of rows"):
        mx.linear_backward(torch.zeros(5, 32), x, mx.empty(64, 32, device="cpu"))
    with pytest.raises(ValueError, match="experts must be"):
        routing.route(x, 2, experts=torch.zeros(4, 3, dtype=torch.int32))
    with pytest.raises(ValueError, match="bias must be"):
        routing.route(x, 2, bias=torch.zeros(63))
    with pytest.raises(ValueError, match="experts must be"):
        routing.dispatch(torch.zeros(4, 2, dtype=torch.int64), 8)
    with pytest.raises(ValueError, match="weights must be"):
        routing.combine(x, torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, 3))
