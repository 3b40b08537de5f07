"""What the FP8 operators and the norm refuse, on the host and before any launch (pointers here are never dereferenced)."""

import pytest
import torch

from triton_chip_benchmarks_amd import _native, fp8, norm, routing

INVALID, UNSUPPORTED, ALIGNMENT = _native.MB_ERR_INVALID, _native.MB_ERR_UNSUPPORTED, _native.MB_ERR_ALIGNMENT
P, BIG = 1 << 20, 1 << 50


def refused(code, name, *arguments, match):
    status = getattr(_native.load(), name)(*arguments)
    assert status == code and match in _native.last_error(), (status, _native.last_error())


def accepted(name, *arguments):
    assert getattr(_native.load(), name)(*arguments) == _native.MB_OK, _native.last_error()


def call(**defaults):
    """The arguments in their order, some replaced."""
    def with_(**changed):
        assert set(changed) <= set(defaults), changed
        return tuple({**defaults, **changed}.values())

    return with_


def test_quantize():
    # 64 x 200 of bf16: pitch 208, one dword of scales a row.
    of = call(dtype=2, x=P, x_bytes=64 * 200 * 2, rows=64, k=200, stride=200, slots=None, slots_bytes=0, copies=1,
              out=64, codes=P, codes_bytes=64 * 208, scales=P, scales_bytes=64 * 4, stream=None)
    name = "mb_fp8_quantize"
    refused(INVALID, name, *of(dtype=3), match="element type")
    refused(INVALID, name, *of(x=None), match="x is NULL")
    refused(INVALID, name, *of(x_bytes=64 * 200 * 2 - 1), match="too small")
    refused(INVALID, name, *of(stride=201), match="too small")
    refused(INVALID, name, *of(stride=1 << 62), match="too small")
    refused(ALIGNMENT, name, *of(x=P + 1), match="elements")
    refused(ALIGNMENT, name, *of(codes=P + 8), match="16 bytes")
    refused(ALIGNMENT, name, *of(scales=P + 2), match="scales on 4")
    refused(INVALID, name, *of(codes=None), match="NULL")
    refused(INVALID, name, *of(codes_bytes=64 * 208 - 1), match="too small")
    refused(INVALID, name, *of(scales_bytes=64 * 4 - 1), match="too small")
    refused(UNSUPPORTED, name, *of(rows=(1 << 24) + 1, x_bytes=BIG), match="at most")
    refused(UNSUPPORTED, name, *of(k=(1 << 20) + 1, x_bytes=BIG), match="at most")
    refused(UNSUPPORTED, name, *of(rows=1 << 24, k=1 << 20, stride=0, x_bytes=BIG, codes_bytes=BIG, scales_bytes=BIG),
            match="exceeds one launch")
    refused(INVALID, name, *of(slots=P, slots_bytes=64 * 2 * 4 - 1, copies=2), match="slots")
    refused(INVALID, name, *of(slots=P, slots_bytes=BIG, copies=65), match="slots")
    refused(ALIGNMENT, name, *of(slots=P + 2, slots_bytes=BIG), match="slots")
    accepted(name, *of(rows=0, x=None, codes=None))
    refused(INVALID, name, *of(rows=0, dtype=9), match="element type")


def test_quantize_both_and_dequantize():
    of = call(dtype=0, x=P, x_bytes=BIG, rows=130, columns=70, stride=70, block=1, codes=P, codes_bytes=130 * 80,
              scales=P, scales_bytes=130 * 4, column_codes=P, column_codes_bytes=70 * 144, column_scales=P,
              column_scales_bytes=70 * 4, stream=None)
    name = "mb_fp8_quantize_both"
    refused(INVALID, name, *of(dtype=-1), match="element type")
    refused(INVALID, name, *of(block=64), match="1 or 128")
    refused(INVALID, name, *of(x_bytes=130 * 70 * 4 - 1), match="too small")
    refused(INVALID, name, *of(codes_bytes=130 * 80 - 1), match="too small")
    refused(INVALID, name, *of(column_codes_bytes=70 * 144 - 1), match="too small")
    refused(INVALID, name, *of(column_scales_bytes=70 * 4 - 1), match="too small")
    refused(INVALID, name, *of(block=128, scales_bytes=7), match="too small")
    refused(UNSUPPORTED, name, *of(rows=(1 << 20) + 1, codes=None), match="at most")
    refused(UNSUPPORTED, name, *of(rows=1 << 24, columns=1 << 20, stride=0, codes_bytes=BIG, scales_bytes=BIG,
                                   column_codes=None), match="exceeds one launch")
    accepted(name, *of(codes=None, column_codes=None))
    of = call(dtype=2, codes=P, codes_bytes=64 * 48, scales=P, scales_bytes=256, block=1, out=P, out_bytes=64 * 40 * 2,
              rows=64, k=40, stream=None)
    name = "mb_fp8_dequantize"
    refused(INVALID, name, *of(dtype=7), match="element type")
    refused(INVALID, name, *of(out_bytes=64 * 40 * 2 - 1), match="too small")
    refused(INVALID, name, *of(codes_bytes=64 * 48 - 1), match="too small")
    refused(INVALID, name, *of(block=2), match="1 or 128")
    refused(ALIGNMENT, name, *of(out=P + 1), match="elements")
    refused(UNSUPPORTED, name, *of(rows=1 << 24, k=1 << 20, codes_bytes=BIG, scales_bytes=BIG, out_bytes=BIG),
            match="exceeds one launch")


def test_product_and_gated_product():
    product = call(dtype=2, a=P, a_bytes=BIG, sa=P, sa_bytes=BIG, a_block=1, b=P, b_bytes=BIG, sb=P, sb_bytes=BIG,
                   b_block=128, c=P, c_bytes=8 * 64 * 2, rows=8, n=64, k=40, offsets=None, offsets_bytes=0, experts=1,
                   kernel=None, stream=None)
    gated = call(dtype=2, a=P, a_bytes=BIG, sa=P, sa_bytes=BIG, a_block=1, b=P, b_bytes=BIG, sb=P, sb_bytes=BIG,
                 b_block=128, y=P, y_bytes=8 * 64 * 2, ys=None, ys_bytes=0, gate_up=None, gate_up_bytes=0, rows=8, n=64,
                 k=40, offsets=None, offsets_bytes=0, experts=1, kernel=None, stream=None)
    for name, of, width, output in (("mb_fp8_product", product, 64, {"c_bytes": 8 * 64 * 2 - 1}),
                                    ("mb_fp8_gated_product", gated, 128, {"y_bytes": 8 * 64 * 2 - 1})):
        refused(INVALID, name, *of(dtype=-1), match="element type")
        refused(INVALID, name, *of(experts=2), match="offsets")
        refused(INVALID, name, *of(experts=0), match="experts")
        refused(INVALID, name, *of(experts=4097, offsets=P, offsets_bytes=BIG), match="experts")
        refused(INVALID, name, *of(experts=2, offsets=P, offsets_bytes=8), match="offsets")
        refused(ALIGNMENT, name, *of(experts=2, offsets=P + 2, offsets_bytes=12), match="offsets")
        refused(INVALID, name, *of(k=0), match="K must be positive")
        refused(INVALID, name, *of(a_block=2), match="1 or 128")
        refused(INVALID, name, *of(b_block=0), match="1 or 128")
        refused(UNSUPPORTED, name, *of(a_block=128, experts=2, offsets=P, offsets_bytes=12), match="scale each")
        refused(INVALID, name, *of(**output), match="output")
        refused(INVALID, name, *of(a_bytes=8 * 48 - 1), match="too small")
        refused(INVALID, name, *of(b_bytes=width * 48 - 1), match="too small")
        refused(INVALID, name, *of(sb_bytes=3), match="too small")
        refused(INVALID, name, *of(experts=2, offsets=P, offsets_bytes=12, b_bytes=2 * width * 48 - 1),
                match="too small")
        refused(UNSUPPORTED, name, *of(rows=(1 << 24) + 1), match="at most")
        refused(UNSUPPORTED, name, *of(n=(1 << 20) + 1), match="at most")
        refused(UNSUPPORTED, name, *of(kernel=b"no_such_kernel"), match="no_such_kernel")
        refused(UNSUPPORTED, name, *of(kernel=b"fp8_few_product_f32_f32_2x4"), match="no kernel")
        accepted(name, *of(rows=0, a=None))
    refused(INVALID, "mb_fp8_gated_product", *gated(gate_up=P, gate_up_bytes=8 * 128 * 2 - 1), match="gate_up")
    refused(INVALID, "mb_fp8_gated_product", *gated(ys=P, ys_bytes=31), match="too small")
    refused(UNSUPPORTED, "mb_fp8_gated_product", *gated(ys=P, ys_bytes=BIG, gate_up=P, gate_up_bytes=BIG), match="FP8")


def test_linear_and_gated():
    shared = {"dtype": 2, "x": P, "x_bytes": BIG, "tokens": 8, "stride": 64, "w": P, "w_bytes": BIG, "sw": P,
              "sw_bytes": BIG, "w_block": 128, "y": P, "y_bytes": BIG}
    routes = {"n": 64, "k": 64, "offsets": None, "offsets_bytes": 0, "order": None, "slots": None, "slots_bytes": 0,
              "copies": 1, "experts": 1, "workspace": P, "workspace_bytes": BIG, "stream": None}
    linear = call(**shared, **routes)
    gated = call(**shared, ys=None, ys_bytes=0, gate_up=None, gate_up_bytes=0, **routes)
    for name, of in (("mb_fp8_linear", linear), ("mb_fp8_gated", gated)):
        refused(INVALID, name, *of(x_bytes=8 * 64 * 2 - 1), match="too small")
        refused(INVALID, name, *of(y_bytes=8 * 64 * 2 - 1), match="output")
        refused(INVALID, name, *of(w_block=16), match="1 or 128")
        refused(INVALID, name, *of(workspace=None), match="workspace")
        refused(INVALID, name, *of(workspace_bytes=8 * 64 + 31), match="workspace")
        refused(ALIGNMENT, name, *of(workspace=P + 8), match="16 bytes")
        refused(INVALID, name, *of(slots=P, slots_bytes=BIG, copies=2), match="slots need")
        refused(INVALID, name, *of(slots=P, slots_bytes=63, offsets=P, offsets_bytes=BIG, order=P, copies=2),
                match="slots need")
        refused(INVALID, name, *of(slots=P, slots_bytes=BIG, offsets=P, offsets_bytes=BIG, order=P, copies=65),
                match="outside 1..64")
        refused(UNSUPPORTED, name, *of(tokens=1 << 20, slots=P, slots_bytes=BIG, offsets=P, offsets_bytes=BIG, order=P,
                                       copies=17), match="at most")
        accepted(name, *of(tokens=0, x=None))
    refused(INVALID, "mb_fp8_gated", *gated(w_bytes=128 * 64 - 1), match="too small")


@pytest.mark.parametrize("name", ["mb_fp8_linear_backward", "mb_fp8_gated_backward"])
def test_backward(name):
    kept = {} if "linear" in name else {"gate_up": P, "gate_up_bytes": 8 * 128 * 2}
    width = 128 if kept else 64
    of = call(dtype=2, d=P, d_bytes=8 * 64 * 2, d_stride=64, **kept, x=P, x_bytes=8 * 96 * 2, x_stride=96, w=P,
              w_bytes=96 * width, sw=P, sw_bytes=BIG, w_block=128, dx=P, dx_bytes=8 * 96 * 2, dw=P,
              dw_bytes=width * 96 * 2, rows=8, n=64, k=96, workspace=P, workspace_bytes=BIG, stream=None)
    refused(INVALID, name, *of(rows=0), match="positive")
    refused(INVALID, name, *of(d_bytes=8 * 64 * 2 - 1), match="too small")
    refused(INVALID, name, *of(x_bytes=8 * 96 * 2 - 1), match="too small")
    refused(INVALID, name, *of(w_bytes=96 * width - 1), match="too small")
    refused(INVALID, name, *of(dx_bytes=8 * 96 * 2 - 1), match="d_x")
    refused(INVALID, name, *of(dw_bytes=width * 96 * 2 - 1), match="d_w")
    if kept:
        refused(INVALID, name, *of(gate_up=None), match="gate_up")
        refused(INVALID, name, *of(gate_up_bytes=8 * 128 * 2 - 1), match="gate_up")
        refused(UNSUPPORTED, name, *of(n=(1 << 19) + 1), match="at most")
    needed = getattr(_native.load(), name + "_workspace")(8, 64, 96)
    refused(INVALID, name, *of(workspace_bytes=needed - 1), match="workspace")
    refused(ALIGNMENT, name, *of(workspace=P + 4), match="16 bytes")
    refused(UNSUPPORTED, name, *of(rows=(1 << 20) + 1, d_bytes=BIG, x_bytes=BIG, dx_bytes=BIG), match="at most")


def test_norm():
    of = call(dtype=2, x=P, x_bytes=8 * 64 * 2, x_stride=64, residual=P, residual_bytes=8 * 64 * 2, residual_stride=64,
              weight=P, weight_bytes=128, eps=1e-6, total=P, total_bytes=8 * 64 * 2, out=P, out_bytes=8 * 64 * 2,
              codes=P, codes_bytes=8 * 64, scales=P, scales_bytes=32, rows=8, n=64, stream=None)
    name = "mb_rms_norm"
    refused(INVALID, name, *of(dtype=3), match="element type")
    refused(INVALID, name, *of(eps=-1e-6), match="eps")
    refused(INVALID, name, *of(eps=float("nan")), match="eps")
    refused(INVALID, name, *of(x_bytes=8 * 64 * 2 - 1), match="too small")
    refused(INVALID, name, *of(residual_stride=65), match="too small")
    refused(INVALID, name, *of(residual=None), match="go together")
    refused(INVALID, name, *of(total=None), match="go together")
    refused(INVALID, name, *of(weight_bytes=127), match="weight")
    refused(INVALID, name, *of(out=None, codes=None), match="no output")
    refused(INVALID, name, *of(out_bytes=8 * 64 * 2 - 1), match="too small")
    refused(INVALID, name, *of(codes_bytes=8 * 64 - 1), match="too small")
    refused(ALIGNMENT, name, *of(codes=P + 8), match="16 bytes")
    refused(ALIGNMENT, name, *of(out=P + 1), match="elements")
    refused(UNSUPPORTED, name, *of(n=16385), match="at most 16384")
    large = {key: BIG for key in ("x_bytes", "residual_bytes", "weight_bytes", "total_bytes", "out_bytes",
                                  "codes_bytes", "scales_bytes")}
    # 2^32 - 1 work items a launch: a row of over 8192 takes 1024 of them, of over 1024 256.
    refused(UNSUPPORTED, name, *of(rows=1 << 22, n=8193, x_stride=0, residual_stride=0, **large), match="one launch")
    refused(UNSUPPORTED, name, *of(rows=1 << 24, n=1025, x_stride=0, residual_stride=0, **large), match="one launch")
    accepted(name, *of(rows=0, x=None))
    of = call(dtype=2, d=P, d_bytes=8 * 64 * 2, d_stride=64, total=P, total_bytes=8 * 64 * 2, total_stride=64, weight=P,
              weight_bytes=128, eps=1e-6, d_total=P, d_total_bytes=8 * 64 * 2, d_total_stride=64, dx=P,
              dx_bytes=8 * 64 * 2, dw=P, dw_bytes=128, rows=8, n=64, workspace=P, workspace_bytes=BIG, stream=None)
    name = "mb_rms_norm_backward"
    refused(INVALID, name, *of(dtype=3), match="element type")
    refused(INVALID, name, *of(rows=0), match="positive")
    refused(INVALID, name, *of(d_bytes=8 * 64 * 2 - 1), match="too small")
    refused(INVALID, name, *of(total_stride=65), match="too small")
    refused(INVALID, name, *of(d_total_bytes=8 * 64 * 2 - 1), match="too small")
    refused(INVALID, name, *of(dx_bytes=8 * 64 * 2 - 1), match="too small")
    refused(INVALID, name, *of(dw_bytes=127), match="too small")
    refused(UNSUPPORTED, name, *of(n=16385), match="at most 16384")
    needed = _native.load().mb_rms_norm_backward_workspace(8, 64)
    assert needed == 8 * 64 * 4
    refused(INVALID, name, *of(workspace_bytes=needed - 1), match="workspace")
    refused(ALIGNMENT, name, *of(workspace=P + 8), match="16 bytes")


def _tensor(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype)


def _operand(rows, k, block=1, experts=None):
    return fp8.empty(rows, k, block, "cpu", experts)


def test_operands():
    with pytest.raises(ValueError, match="1 or 128 rows"):
        fp8.empty(4, 16, 64, "cpu")
    good = _operand(130, 70, 128)
    assert good.codes.shape == (130, 80) and good.scales.shape == (1, 2, 4) and good.experts is None
    for codes, scales, k, block in ((good.codes, good.scales, 70, 1), (good.codes, good.scales, 81, 128),
                                    (good.codes.view(torch.uint8), good.scales, 70, 128),
                                    (good.codes[:, :64], good.scales, 64, 128), (good.codes, good.scales[0], 70, 128),
                                    (good.codes, good.scales.int(), 70, 128), (good.codes[0], good.scales, 70, 128)):
        with pytest.raises(ValueError, match="contiguous float8_e4m3fn"):
            fp8.Packed(codes, scales, k, block)


def test_python_refusals():
    x, weight, experts = _tensor(4, 40), _operand(6, 40, 128), _operand(6, 40, 128, experts=3)
    plan = routing.Plan(*(torch.zeros(shape, dtype=torch.int32) for shape in ((4,), (8,), (4, 2))), None)

    def refused_(match, function, *arguments, **options):
        with pytest.raises(ValueError, match=match):
            function(*arguments, **options)

    refused_("current HIP device", fp8.quantize, x)
    refused_("current HIP device", fp8.linear, x, weight, workspace=_tensor(1000, dtype=torch.uint8))
    refused_("current HIP device", norm.rms_norm, x, _tensor(40))
    refused_("float32, float16 or bfloat16", fp8.quantize, x.double())
    refused_("two dimensions", fp8.quantize, x[0])
    refused_("contiguous rows", fp8.quantize, x.t())
    refused_("packed must be an operand of 4 x 40", fp8.quantize, x, _operand(5, 40))
    refused_("packed must be an operand of 4 x 40", fp8.quantize, x, _operand(4, 40, 128))
    refused_("packed must be an operand of 40 x 4", fp8.quantize, x, _operand(4, 40), columns=True)
    refused_("packed must hold one matrix", fp8.quantize, x, _operand(4, 40, experts=1))
    refused_("columns must be an operand", fp8.quantize_both, x, _operand(4, 40), _operand(4, 40))
    refused_("packed must hold one matrix", fp8.dequantize, experts)
    refused_("out must be", fp8.dequantize, weight, _tensor(6, 41))
    refused_("same k", fp8.product, _operand(4, 40), _operand(6, 41))
    refused_("b must hold one matrix", fp8.product, _operand(4, 40), experts)
    refused_("scale each", fp8.product, _operand(4, 40, 128), experts, offsets=torch.zeros(4, dtype=torch.int32))
    refused_("offsets must", fp8.product, _operand(4, 40), experts, offsets=torch.zeros(4, dtype=torch.int64))
    refused_("k = 40", fp8.linear, x, _operand(6, 41, 128))
    refused_("weight must hold one matrix", fp8.linear, x, experts)
    refused_("each of 3 experts", fp8.linear, x, weight, plan=plan)
    refused_("sorted rows need the plan", fp8.linear, x, weight, sorted_rows=True)
    refused_("route 5 tokens", fp8.linear, _tensor(5, 40), experts, plan=plan)
    refused_("out must be", fp8.linear, x, weight, _tensor(4, 5))
    refused_("workspace", fp8.linear, x, weight, workspace=_tensor(8, dtype=torch.uint8))
    refused_("even number of rows", fp8.gated, x, _operand(7, 40, 128))
    refused_("is of its type", fp8.gated, x, weight, dtype=torch.float32)
    refused_("a kernel is named", fp8.gated, x, weight, kernel="fp8")
    refused_("gate_up must be", fp8.gated, x, weight, gate_up=_tensor(4, 7))
    refused_("gate_up beside out", fp8.gated, x, weight, gate_up=_tensor(4, 6), packed=_operand(4, 3))
    refused_("out or to packed", fp8.gated, x, weight, _tensor(4, 3), _operand(4, 3))
    refused_("sorted by the plan", fp8.gated, _operand(4, 40), experts, plan=plan)
    refused_("float32, float16 or bfloat16", fp8.gated, _operand(4, 40), weight, dtype=torch.float64)
    refused_("one type and number of rows", fp8.linear_backward, _tensor(5, 6), x, _operand(40, 6, 128))
    refused_("weight quantised by columns", fp8.linear_backward, _tensor(4, 6), x, weight)
    refused_("gate_up that gated kept", fp8.gated_backward, _tensor(4, 3), None, x, _operand(40, 6, 128))
    refused_("gate_up must be", fp8.gated_backward, _tensor(4, 3), _tensor(4, 5), x, _operand(40, 6, 128))
    refused_("weight must be", norm.rms_norm, x, _tensor(41))
    refused_("weight must be", norm.rms_norm, x, _tensor(40, dtype=torch.float32))
    refused_("residual must be", norm.rms_norm, x, _tensor(40), residual=_tensor(4, 41))
    refused_("without a residual", norm.rms_norm, x, _tensor(40), total=_tensor(4, 40))
    refused_("packed must be an operand", norm.rms_norm, x, _tensor(40), packed=_operand(4, 40, 128))
    refused_("out must be", norm.rms_norm, x, _tensor(40), out=_tensor(5, 40))
    refused_("d_out must be", norm.rms_norm_backward, _tensor(5, 40), x, _tensor(40))
    refused_("d_total must be", norm.rms_norm_backward, x, x, _tensor(40), d_total=_tensor(4, 40, dtype=torch.float32))
    refused_("d_weight must be", norm.rms_norm_backward, x, x, _tensor(40), d_weight=_tensor(41))


def test_names_of_kernels():
    with pytest.raises(_native.NativeError, match="no product"):
        fp8.product_kernel(0, 64, 64)
    with pytest.raises(_native.NativeError, match="experts"):
        fp8.product_kernel(4, 64, 64, experts=5000)
    with pytest.raises(_native.NativeError, match="element type"):
        fp8.product_kernel(4, 64, 64, torch.float64)
