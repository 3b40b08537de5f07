"""Routing of many tokens, a quarter of a wave each, in every type: against the oracle, and against the same tokens in
calls so small that each has a wave."""

import numpy as np
import pytest

from oracle import routing as oracle

pytestmark = pytest.mark.gpu

UNIT = {"fp32": 2.0**-24, "fp16": 2.0**-11, "bf16": 2.0**-8}
# A score: an exponential, an addition, a division and a sum of up to 256 in a tree; see the routing tests.
SCORE_TOLERANCE = (32 + 24 + 8) * 2.0**-23


def _host(tensor):
    return tensor.double().cpu().numpy()


# The experts of 4, 8 and 16 a lane: as many as fit, and ones that end inside a lane's.
@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts,top,groups,top_groups", [(64, 16, 1, 1), (50, 3, 1, 1), (128, 8, 8, 3),
                                                           (117, 5, 1, 1), (256, 16, 16, 4), (229, 8, 1, 1)])
def test_many_tokens(gpu, dtype, scores, experts, top, groups, top_groups):
    import torch

    from triton_chip_benchmarks_amd import routing

    print(f"route {dtype} 4103x{experts} top {top} of {groups}/{top_groups} {scores}", flush=True)
    tokens = 4103  # the last of them end inside a workgroup
    rng = np.random.default_rng(experts)
    ladder = (np.arange(experts) - experts // 2) / 32.0  # exact in every type, and no two scores alike in 32 bits
    values = np.stack([rng.permutation(ladder) for _ in range(tokens)])
    values[4::9] = -np.inf
    values[:, 7] = -np.inf
    kind = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}[dtype]
    wide = torch.zeros(tokens, experts + 5, device="cuda", dtype=kind)
    logits = wide[:, 3:experts + 3]  # off every vector's alignment
    logits.copy_(torch.tensor(values))
    sample = np.r_[0:20, 2000:2010, tokens - 20:tokens]
    assert np.array_equal(_host(logits)[sample], values[sample])
    options = {"scores": scores, "groups": groups, "top_groups": top_groups, "scale": 1.5}
    chosen, weights = routing.route(logits, top, **options)
    expected, exact = oracle.route(values[sample], top, kind=scores, groups=groups, top_groups=top_groups, scale=1.5)
    if groups == 1:  # sums of two scores may be closer than 32 bits tell apart
        assert np.array_equal(chosen.cpu().numpy()[sample], expected)
        assert np.allclose(_host(weights)[sample], exact, rtol=SCORE_TOLERANCE, atol=0)
    few = [routing.route(logits[i:i + 1500], top, **options) for i in range(0, tokens, 1500)]
    assert torch.equal(chosen, torch.cat([part[0] for part in few]))
    assert torch.allclose(weights, torch.cat([part[1] for part in few]), rtol=SCORE_TOLERANCE, atol=0)
    for renormalize in (True, False):
        g = torch.randn(tokens, top, device="cuda", generator=torch.Generator(device="cuda").manual_seed(top))
        d_logits = routing.route_backward(logits, chosen, g, scores=scores, renormalize=renormalize, scale=1.5)
        exact = oracle.route_backward(values[sample], chosen.cpu().numpy()[sample], _host(g)[sample], kind=scores,
                                      renormalize=renormalize, scale=1.5)
        bound = 6 * SCORE_TOLERANCE * np.abs(_host(g)[sample]).sum(axis=1, keepdims=True) + UNIT[dtype] * np.abs(exact)
        assert (np.abs(_host(d_logits)[sample] - exact) <= bound + 2.0**-25).all()
        part = torch.cat([routing.route_backward(logits[i:i + 1500], chosen[i:i + 1500], g[i:i + 1500], scores=scores,
                                                 renormalize=renormalize, scale=1.5) for i in range(0, tokens, 1500)])
        assert np.abs(_host(part) - _host(d_logits)).max() <= 12 * SCORE_TOLERANCE * float(g.abs().sum(1).max()) + \
            2 * UNIT[dtype] * float(d_logits.abs().max())
