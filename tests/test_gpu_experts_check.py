"""The mixture-of-experts command's own check: right layers of any size pass it, and a wrong weight does not."""

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("apart", [0.0, 2.0**-12, -(2.0**-12)])
@pytest.mark.parametrize("tokens,hidden,inner,count,top", [(1, 64, 33, 4, 1), (1, 256, 96, 8, 2), (9, 96, 1, 3, 2)])
def test_a_right_layer_passes_whatever_codes_its_roundings_move(gpu, monkeypatch, dtype, apart, tokens, hidden, inner,
                                                                count, top):
    """Also against sums that lie a fraction of a rounding apart, after which some values of 16 bits, and then some
    codes, are other ones."""
    import torch

    from triton_chip_benchmarks_amd import experts

    print(f"check {dtype} {tokens}x{hidden}x{inner} experts={count} top={top}, {apart} apart", flush=True)
    kind = {"bf16": torch.bfloat16, "fp16": torch.float16}[dtype]
    right = experts._values
    monkeypatch.setattr(experts, "_values", lambda packed, e: right(packed, e) * (1 + apart))
    worst = max(experts.check(experts.Layer(tokens, hidden, inner, count, top, kind, seed=seed)) for seed in range(150))
    assert worst <= experts.TOLERANCE, worst


@pytest.mark.parametrize("which", ["up_weight", "down_weight"])
def test_another_experts_weight_does_not_pass(gpu, monkeypatch, which):
    import torch

    from triton_chip_benchmarks_amd import experts

    layer = experts.Layer(5, 256, 96, 8, 2, torch.bfloat16)
    right = experts._values
    monkeypatch.setattr(experts, "_values", lambda packed, e: right(packed, (e + 1) % 8) if packed is getattr(layer, which)
                        else right(packed, e))
    assert experts.check(layer) > 0.5
