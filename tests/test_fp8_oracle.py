"""CPU pins of the FP8 operands' and the norm's oracle: known answers, torch's own conversion, gradients against
differences."""

import numpy as np
import pytest
import torch

from oracle import fp8, norm


def test_quantisation_known_answers():
    x = np.zeros((1, 400))
    x[0, :6] = [448, 17, 18.9, 1.0625, -2.0**-9, 2.0**-10]  # scale 2^0: ties to the even code, subnormals
    x[0, 128:130] = [449, 1]  # past 448 * 2^0
    x[0, 256] = 2.0**-140  # below the smallest scale's smallest code
    codes, scales = fp8.quantize(x)
    assert codes.shape == (1, 400) and scales.shape == (1, 1, 4)
    assert scales[0, 0].tolist() == [127, 128, 0, 0]
    assert fp8.values(codes, scales, 400)[0, :6].tolist() == [448, 16, 18, 1, -2.0**-9, 0]
    assert fp8.values(codes, scales, 400)[0, 128:130].tolist() == [448, 1] and codes[0, 256] == 0
    assert fp8.scale_codes(np.array([[448.0], [448.0000001], [224.0], [2.0**-200], [2.0**120]])).ravel().tolist() \
        == [127, 128, 126, 0, 239]


def test_codes_are_those_of_torchs_conversion():
    # Within the format's range, under the scale 2^0, torch rounds the same way.
    x = torch.linspace(-448, 448, 100001, dtype=torch.float64).float()
    scales = np.full((1, -(-len(x) // 128)), 127)
    mine = fp8.element_codes(x.double().numpy()[None], scales)[0]
    assert np.array_equal(mine, x.to(torch.float8_e4m3fn).view(torch.uint8).numpy())


@pytest.mark.parametrize("block", [1, 128])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_a_block_that_is_not_finite_is_nan_alone(bad, block):
    x = np.ones((256, 256))
    x[130, 140] = bad
    values = fp8.rounded(x, block)
    inside = np.zeros(x.shape, bool)
    inside[128 if block == 128 else 130:256 if block == 128 else 131, 128:] = True
    assert np.isnan(values[inside]).all() and (values[~inside] == 1).all()


def test_padding_and_scales_past_the_last_block():
    codes, scales = fp8.quantize(np.ones((3, 520)))
    assert codes.shape == (3, 528) and (codes[:, 520:] == 0).all()
    assert scales.shape == (2, 3, 4) and (scales[1, :, 1:] == 127).all() and (scales[1, :, 0] == 119).all()


def test_linear_gradient_is_the_difference_where_quantisation_changes_nothing():
    # Of a few powers of two every block has the scale of its largest, 1, and every code is exact.
    rng = np.random.default_rng(0)
    lattice = np.array([1.0, 0.5, 0.25, -1, -0.5, -0.125, 0])
    x, w, g = (rng.choice(lattice, size=s) for s in ((40, 150), (130, 150), (40, 130)))
    (d_x, _), (d_w, _) = fp8.linear_backward(g, x, w)
    loss = lambda x, w: (g * fp8.linear(x, w)[0]).sum()  # noqa: E731
    for r, c in ((5, 7), (31, 149), (0, 130)):
        moved = x.copy()
        moved[r, c] += 0.25
        assert loss(moved, w) - loss(x, w) == pytest.approx(d_x[r, c] * 0.25, abs=1e-12)
        moved = w.copy()
        moved[r, c] -= 0.25
        assert loss(x, moved) - loss(x, w) == pytest.approx(-d_w[r, c] * 0.25, abs=1e-12)


def test_gate_and_norm_gradients_against_differences():
    rng = np.random.default_rng(1)
    pair, d_out = rng.standard_normal((3, 10)) * 4, rng.standard_normal((3, 5))
    d_pair = fp8.gate_backward(d_out, pair)
    x, weight, d_y, d_total = (rng.standard_normal(s) for s in ((3, 7), (7,), (3, 7), (3, 7)))
    d_x, d_w = norm.rms_norm_backward(d_y, x, weight, 1e-3, d_total)
    h = 1e-6

    def difference(loss, values, at):
        losses = []
        for sign in (1, -1):
            moved = values.copy()
            moved[at] += sign * h
            losses.append(loss(moved))
        return (losses[0] - losses[1]) / (2 * h)

    for at in ((0, 0), (2, 9), (1, 4)):
        assert d_pair[at] == pytest.approx(difference(lambda p: (d_out * fp8.gate(p)).sum(), pair, at), rel=1e-6, abs=1e-8)
    of_x = lambda x: (d_y * norm.rms_norm(x, weight, 1e-3)).sum() + (d_total * x).sum()  # noqa: E731
    for at in ((0, 0), (2, 6), (1, 3)):
        assert d_x[at] == pytest.approx(difference(of_x, x, at), rel=1e-6, abs=1e-8)
    of_w = lambda w: (d_y * norm.rms_norm(x, w, 1e-3)).sum()  # noqa: E731
    assert d_w[2] == pytest.approx(difference(of_w, weight, 2), rel=1e-6)


def test_gate_of_extremes():
    pair = np.array([[-1e4, 0.0, 800.0, -800.0, 3.0, 2.0, 1.0, 1.0]])
    assert fp8.gate(pair)[0].tolist() == [0.0, 0.0, 800.0, pytest.approx(0, abs=1e-300)]
