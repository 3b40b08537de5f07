"""Routing's gradients and weights where scores are far from 1: each value against its own size, not the row's.

A score is one exponential, one addition and one division (together under 8 roundings of 2^-24, and one of 2^-150
where it is below 2^-126), a sum of `top` scores adds log2(64) + top, and a renormalised gradient is a difference of
values up to the sum of the magnitudes of `g`, times a share and a complement: 64 roundings of 2^-23 cover every chain.
"""

import numpy as np
import pytest

from oracle import routing as oracle

pytestmark = pytest.mark.gpu

ROUNDINGS = 64 * 2.0**-23


def _host(tensor):
    return tensor.double().cpu().numpy()


def _gradient(logits, chosen, g, **options):
    """(d_logits on the device, the float64 oracle's, and the size of the terms that each element is the sum of)."""
    import torch

    from triton_chip_benchmarks_amd import routing

    on_device = [torch.tensor(part, device="cuda") for part in (logits, chosen, g)]
    got = _host(routing.route_backward(*on_device, **options))
    kind, scale = options.get("scores", "softmax"), options.get("scale", 1.0)
    exact = oracle.route_backward(logits, chosen, g, kind=kind, renormalize=options.get("renormalize", True),
                                  scale=scale)
    return got, exact


def _size(logits, chosen, g, scores, renormalize, scale):
    """scale * share * complement * sum |g| of the chosen elements, 0 elsewhere."""
    size = np.zeros(logits.shape)
    for t in range(logits.shape[0]):
        # In units of the row's largest exponential, so that float64 holds every share.
        l = logits[t].astype(np.float64)
        s = np.exp(l - l.max()) if scores == "softmax" else 1 / (1 + np.exp(-l))
        s = s / s.sum() if scores == "softmax" else s
        rest = 1.0 if scores == "softmax" else 1 / (1 + np.exp(l))
        part = s / s[chosen[t]].sum() if renormalize else s
        size[t, chosen[t]] = (scale * part * rest * np.abs(g[t]).sum())[chosen[t]]
    return size


@pytest.mark.parametrize("tokens", [3, 4100])
@pytest.mark.parametrize("scores", ["sigmoid", "softmax"])
def test_gradient_of_shares_of_scores_near_the_smallest(gpu, scores, tokens):
    """Chosen scores of 1e-38: their shares, and the gradient, are of the size of any others'."""
    print(f"gradient of small scores, {scores}, {tokens} tokens", flush=True)
    row = np.array([-88.0, -88.2, -95.0, -95.5, -87.5, -90.0, -91.0, -96.0], dtype=np.float32)
    logits = np.tile(row, (tokens, 1))
    if scores == "softmax":
        logits[:, 7] = 0.0  # takes the whole sum; not chosen
    chosen = np.tile(np.array([0, 1], dtype=np.int32), (tokens, 1))
    chosen[1] = 4, 0
    g = np.tile(np.array([3.0, -3.0], dtype=np.float32), (tokens, 1))
    got, exact = _gradient(logits, chosen, g, scores=scores, scale=2.5)
    # The unchosen have no part in renormalised weights; the oracle's differences leave 2^-53 of the choices' there.
    unchosen = np.ones(logits.shape, dtype=bool)
    np.put_along_axis(unchosen, chosen, False, axis=1)
    assert (got[unchosen] == 0).all()
    # A score of e^-88.2 is 3.5e6 units of 2^-149: two more roundings of 2^-22.
    bound = (ROUNDINGS + 2.0**-21) * _size(logits, chosen, g, scores, True, 2.5)
    assert np.abs(exact).max() > 1
    assert (np.abs(got - exact) <= bound)[~unchosen].all(), (got[:2], exact[:2])


@pytest.mark.parametrize("tokens", [2, 4100])
@pytest.mark.parametrize("renormalize", [True, False])
def test_sigmoid_gradient_of_scores_near_one(gpu, renormalize, tokens):
    """The gradient goes with 1 - s, which is far below a score's last bit from a logit of 17 on."""
    print(f"gradient of scores near one, renormalize={renormalize}, {tokens} tokens", flush=True)
    row = np.array([14.0, 16.0, 17.5, 20.0, 30.0, 86.0, -3.0, 0.5], dtype=np.float32)
    logits = np.tile(row, (tokens, 1))
    chosen = np.tile(np.array([5, 3, 0, 1, 2, 4, 6], dtype=np.int32), (tokens, 1))
    g = np.tile(np.array([3.0, -3.0, 0.5, 1.0, -2.0, 1.5, 0.25], dtype=np.float32), (tokens, 1))
    got, exact = _gradient(logits, chosen, g, scores="sigmoid", renormalize=renormalize, scale=2.5)
    # The oracle's 1 - s is good to 2^-53; here the complement is the sigmoid of the logit's negative.
    s = 1 / (1 + np.exp(-row.astype(np.float64)))
    exact = exact * np.divide(1 / (1 + np.exp(row.astype(np.float64))), 1 - s, where=s < 1, out=np.ones(8))
    part = s[chosen[0]] / s[chosen[0]].sum()
    terms = 2.5 * ((g[0] - (g[0] * part).sum()) * part if renormalize else g[0] * s[chosen[0]])
    exact[:, chosen[0]] = terms / (1 + np.exp(row[chosen[0]].astype(np.float64)))
    bound = ROUNDINGS * _size(logits, chosen, g, "sigmoid", renormalize, 2.5) + 2.0**-149
    assert (np.abs(got - exact) <= bound).all(), (got[0], exact[0])


@pytest.mark.parametrize("tokens", [3, 4100])
@pytest.mark.parametrize("renormalize", [True, False])
def test_sigmoid_scores_down_to_the_smallest(gpu, renormalize, tokens):
    """Logits whose scores fp32 still holds (from about -103 on) are told apart, and their shares are finite."""
    import torch

    from triton_chip_benchmarks_amd import routing

    print(f"sigmoid scores near the smallest, renormalize={renormalize}, {tokens} tokens", flush=True)
    row = np.array([-96.0, -89.5, -94.0, -88.9, -92.0, -90.5, -95.0, -200.0], dtype=np.float32)
    logits = np.tile(row, (tokens, 1))
    chosen, weights = routing.route(torch.tensor(logits, device="cuda"), 4, scores="sigmoid", renormalize=renormalize)
    expected, exact = oracle.route(logits, 4, kind="sigmoid", renormalize=renormalize)
    assert np.array_equal(chosen.cpu().numpy(), expected)
    smallest = np.exp(row[expected[0]].astype(np.float64)).min()
    bound = (ROUNDINGS + 2 * 2.0**-150 / smallest) * exact + (0 if renormalize else 2.0**-150)
    assert (np.abs(_host(weights) - exact) <= bound).all(), (weights[0], exact[0])
    assert (exact > 0).all()


@pytest.mark.parametrize("tokens", [5, 4100])
def test_far_scores_of_a_token_leave_its_neighbours_alone(gpu, tokens):
    """Tokens of far logits among ordinary and masked ones, in groups and with a bias: each as if it were alone."""
    import torch

    from triton_chip_benchmarks_amd import routing

    print(f"far and near tokens, {tokens}", flush=True)
    rng = np.random.default_rng(0)
    logits = np.stack([rng.permutation(np.arange(32) / 8.0 - 2) for _ in range(tokens)]).astype(np.float32)
    logits[1::3] -= 94.0
    logits[1::3, 4:8] = -np.inf
    logits[2::5] = -np.inf
    logits[3::7, 16:] -= 300.0
    options = {"scores": "sigmoid", "groups": 4, "top_groups": 2}
    bias = np.zeros(32, dtype=np.float32)
    bias[10:12] = 2.0  # chosen whatever they score
    for offset in (None, bias):
        on_device = None if offset is None else torch.tensor(offset, device="cuda")
        chosen, weights = routing.route(torch.tensor(logits, device="cuda"), 5, on_device, **options)
        kept = list(range(0, tokens, 1 if tokens < 100 else 89))
        expected, exact = oracle.route(logits[kept], 5, offset, kind="sigmoid", groups=4, top_groups=2)
        assert np.array_equal(chosen.cpu().numpy()[kept], expected)
        # A score of e^-98 is 196 units of 2^-149.
        assert (np.abs(_host(weights)[kept] - exact) <= (ROUNDINGS + 2.0**-6) * exact + 1e-30).all()
        alone = [routing.route(torch.tensor(logits[t:t + 1], device="cuda"), 5, on_device, **options) for t in kept]
        assert np.array_equal(chosen.cpu().numpy()[kept], np.concatenate([a[0].cpu().numpy() for a in alone]))
