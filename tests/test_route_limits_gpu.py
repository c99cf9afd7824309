"""The general routing and its gradient where the ordinary tests do not reach.  Tolerances as in
test_route_experts_gpu: indices equal, weights within REL of themselves (those made in 64 bits
within half a step, less), gradients within REL of the largest term."""
import numpy as np
import pytest
import torch

import candle_moe as cm
import route_testlib as rt
from test_route_experts_gpu import check_route, make_logits

pytestmark = pytest.mark.gpu

# a shape for each of the three kernels: several rows per warp, a warp per row, 64-bit keys
SHAPES = [(24, 1, 1, 4), (100, 1, 1, 12), (510, 5, 2, 4)]


@pytest.mark.parametrize("E,n,kg,k", SHAPES + [(12, 1, 1, 4), (50, 1, 1, 10), (60, 5, 2, 11),
                                               (64, 4, 2, 8), (63, 1, 1, 30)])
@pytest.mark.parametrize("scoring", [0, 1])
@pytest.mark.parametrize("group_score", [0, 1])
def test_bias_of_plus_infinity(E, n, kg, k, scoring, group_score):
    """Experts that a bias of +inf forces on: one, as many as there are slots, more, and all; in
    shapes whose number of candidates is no multiple of four."""
    x = make_logits(E, 37, E, "f32")
    x[5, 3] = float("-inf")  # not available, whatever its bias
    for count in (1, 2, k, min(k + 3, E), E):
        bias = np.round(np.random.default_rng(count).normal(size=E) * 0.1, 3)
        bias[np.random.default_rng(E).permutation(E)[:count]] = np.inf
        check_route(x, k, bias=bias, scoring=cm.Scoring(scoring), num_groups=n, topk_groups=kg,
                    group_score=cm.GroupScore(group_score), renormalize=True)
