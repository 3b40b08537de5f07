"""CPU pins of the layer operators' oracle: known answers, torch's own operations, gradients against differences."""

import numpy as np
import pytest

from oracle import mx, routing


def test_quantisation_known_answers():
    x = np.zeros((1, 96))
    x[0, :10] = [6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -0.2500001, -5.0]  # scale 2^0: ties to the even code
    x[0, 32:35] = [7.9, 6.9, -1e-30]  # still 2^0: 7.9 lies in [4, 8) and saturates at 6
    x[0, 64:66] = [2.0**-140, 2.0**-128]  # 2^-130 clamps to 2^-127
    codes, scales = mx.quantize(x)
    assert scales.shape == (1, 1, 8) and scales[0, 0].tolist() == [127, 127, 0, 127, 127, 127, 127, 127]
    assert mx.values(codes, scales, 96)[0, :10].tolist() == [6, 0, 1, 1, 2, 2, 4, 4, -0.5, -4]
    assert mx.values(codes, scales, 96)[0, 32:35].tolist() == [6, 6, 0] and codes[0, 17] & 15 == 8  # minus zero
    assert mx.values(codes, scales, 96)[0, 64:66].tolist() == [0.0, 2.0**-128]
    assert codes[0, 0] == 7 | 0 << 4  # even k in the low nibble


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_a_group_that_is_not_finite_is_nan_alone(bad):
    x = np.ones((2, 64))
    x[1, 40] = bad
    values = mx.rounded(x)
    assert np.isnan(values[1, 32:]).all() and (values[0] == 1).all() and (values[1, :32] == 1).all()


def test_every_value_is_the_nearest_of_the_groups_lattice():
    x = np.random.default_rng(0).standard_normal((7, 100)) * np.exp2(np.arange(7) * 9.0 - 30)[:, None]
    scales = mx.scale_codes(x).astype(np.float64)
    values = mx.rounded(x)
    for r in range(7):
        for i in range(100):
            lattice = np.concatenate([mx.MAGNITUDES, -mx.MAGNITUDES]) * np.exp2(scales[r, i // 32] - 127)
            assert abs(values[r, i] - x[r, i]) <= np.abs(lattice - x[r, i]).min() * (1 + 1e-12)
            assert 4 <= np.abs(x[r, i // 32 * 32:i // 32 * 32 + 32]).max() * np.exp2(127 - scales[r, i // 32]) < 8


def test_linear_gradient_is_the_difference_where_quantisation_changes_nothing():
    # On the lattice the layer is its product, so a step from code to code changes the loss by its gradient.
    rng = np.random.default_rng(1)
    lattice = np.concatenate([mx.MAGNITUDES, -mx.MAGNITUDES])
    x, w, g = (rng.choice(lattice, size=s) for s in ((32, 64), (96, 64), (32, 96)))
    for m in (x, w, g):
        m[::32, :] = 6
        m[:, ::32] = 6  # every group's scale, along rows and columns, is 2^0
    d_x, d_w = (part[0] for part in mx.linear_backward(g, x, w))
    loss = lambda x, w: (g * mx.linear(x, w)[0]).sum()  # noqa: E731
    for r, c in ((5, 7), (31, 63), (1, 33)):
        moved = x.copy()
        moved[r, c] = 3.0 if x[r, c] != 3.0 else 2.0
        assert loss(moved, w) - loss(x, w) == d_x[r, c] * (moved[r, c] - x[r, c])
        moved = w.copy()
        moved[r, c] = -1.5 if w[r, c] != -1.5 else 0.5
        assert loss(x, moved) - loss(x, w) == d_w[r, c] * (moved[r, c] - w[r, c])


@pytest.mark.parametrize("kind", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [False, True])
def test_route_gradient_against_differences_and_autograd(kind, renormalize):
    import torch

    rng = np.random.default_rng(2)
    logits, g = rng.standard_normal((3, 12)), rng.standard_normal((3, 4))
    logits[0, 5] = -np.inf
    logits[2] = -np.inf
    options = {"kind": kind, "renormalize": renormalize, "scale": 2.5}
    experts, _ = routing.route(logits, 4, **options)
    assert (experts[2] == -1).all()
    d_logits = routing.route_backward(logits, experts, g, **options)
    assert (d_logits[2] == 0).all() and d_logits[0, 5] == 0
    for t, e in ((0, experts[0, 0]), (0, experts[0, 3]), (1, experts[1, 1]), (1, int(logits[1].argmin()))):
        h = 1e-6
        losses = []
        for sign in (1, -1):
            moved = logits.copy()
            moved[t, e] += sign * h
            chosen, weights = routing.route(moved, 4, **options)
            assert (chosen == experts).all()
            losses.append((weights * g).sum())
        assert abs((losses[0] - losses[1]) / (2 * h) - d_logits[t, e]) < 1e-8
    leaf = torch.tensor(logits[:2], requires_grad=True)
    s = torch.softmax(leaf, 1) if kind == "softmax" else torch.sigmoid(leaf)
    w = s.gather(1, torch.tensor(experts[:2]).long())
    w = w / w.sum(1, keepdim=True) if renormalize else w
    (2.5 * w * torch.tensor(g[:2])).sum().backward()
    assert np.allclose(np.nan_to_num(leaf.grad.numpy()), d_logits[:2], rtol=1e-12, atol=1e-15)


def test_route_known_answers():
    logits = np.array([[1.0, 3.0, 3.0, 0.0, 2.0, -np.inf]])
    experts, weights = routing.route(logits, 3)
    assert experts.tolist() == [[1, 2, 4]] and np.isclose(weights.sum(), 1)  # equal logits: the lower index first
    experts, _ = routing.route(logits, 3, bias=np.array([0, 0, 0, 2.0, 0, 5.0]))
    assert experts.tolist() == [[3, 1, 2]]  # the bias moves the choice; masked stays masked
    # Groups {0,1} {2,3} {4,5}: sums of two 4, 3, 2 (the masked one counts for nothing).
    experts, _ = routing.route(logits, 3, kind="sigmoid", groups=3, top_groups=1)
    assert experts.tolist() == [[1, 0, -1]]


def test_dispatch_and_combine_known_answers():
    experts = np.array([[2, 0], [-1, 2], [0, 7]])
    offsets, order, slots = routing.dispatch(experts, 3)
    assert offsets.tolist() == [0, 2, 2, 4] and order.tolist() == [1, 4, 0, 3, -1, -1]
    assert slots.tolist() == [[2, 0], [-1, 3], [1, -1]]
    y = np.arange(8.0).reshape(4, 2)
    weights = np.array([[0.5, 2.0], [9.0, 1.0], [3.0, 9.0]])
    out, _ = routing.combine(y, slots, weights)
    assert out.tolist() == [[2.0, 4.5], [6.0, 7.0], [6.0, 9.0]]
    d_out = np.array([[1.0, 2.0], [0.0, 1.0], [1.0, 0.0]])
    d_y, d_weights, _ = routing.combine_backward(d_out, y, slots, weights)
    assert d_weights.tolist() == [[14.0, 2.0], [0.0, 7.0], [2.0, 0.0]]
    h = 1e-6  # linear: differences are the gradient
    for index in np.ndindex(y.shape):
        moved = y.copy()
        moved[index] += h
        change = ((routing.combine(moved, slots, weights)[0] - out) * d_out).sum() / h
        assert abs(change - d_y[index]) < 1e-8
