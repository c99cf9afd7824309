"""The general routing and its gradient where the ordinary tests do not reach.  Tolerances as in
test_route_experts_gpu: indices equal, weights within REL of themselves (those made in 64 bits
within half a step, less), gradients within REL of the largest term."""
import numpy as np
import pytest
import torch

import candle_moe as cm
import route_testlib as rt
from test_route_experts_gpu import DT, REL, check_route, make_logits

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


@pytest.mark.parametrize("E,n,kg,k", SHAPES)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("with_bias", [False, True])
def test_small_sigmoid_scores_renormalise(E, n, kg, k, dtype, with_bias):
    """exp(-l) passes the largest f32 at l = -88.7; the picks' share of their sum does not depend
    on how small they are, down to the last 64-bit score (l = -709.8: the sum is 0 below)."""
    base = torch.tensor([0.0, -60.0, -86.0, -88.0, -89.0, -100.0, -300.0, -650.0, -800.0])
    x = torch.rand(9, E, generator=torch.Generator().manual_seed(E)) * 4 + base[:, None]
    x = x.repeat(5, 1).to(DT[dtype]).cuda()
    bias = np.zeros(E) if with_bias else None
    for scaling in (1.0, 2.5, 1e6):
        w, idx = check_route(x, k, bias=bias, scoring=cm.Scoring.Sigmoid, num_groups=n,
                             topk_groups=kg, renormalize=True, scaling=scaling)
        assert (w[8] == 0).all() and (idx[8] < E).all()
        g = torch.randn(w.shape, generator=torch.Generator().manual_seed(1)).cuda()
        keep = [t for t in range(45) if t % 9 != 8]
        d = cm.route_experts_backward(g, x, w, idx, cm.Scoring.Sigmoid, True, scaling)
        ref = rt.backward(g.double().cpu().numpy(), x.double().cpu().numpy(), idx.cpu().numpy(), 1,
                          True, scaling)
        tol = 4 * REL * scaling * g.abs().amax(1, keepdim=True).double().cpu().numpy()
        if dtype != "f32":
            tol = tol + torch.finfo(DT[dtype]).eps / 2 * np.abs(ref)
        assert (np.abs(d.double().cpu().numpy() - ref) <= tol)[keep].all()


@pytest.mark.parametrize("E,n,kg,k", SHAPES)
def test_small_softmax_scores_renormalise(E, n, kg, k):
    """A bias may lift experts far below the row's largest logit into the picks."""
    x = torch.rand(8, E, generator=torch.Generator().manual_seed(E)) * 4
    top = torch.tensor([0.0, 60.0, 80.0, 88.0, 100.0, 300.0, 700.0, 900.0])
    x[:, 0] = top
    bias = np.full(E, 4.0)
    bias[0] = 0.0
    for scaling in (1.0, 1e6):
        w, idx = check_route(x.cuda(), k, bias=bias, scoring=cm.Scoring.Softmax, num_groups=n,
                             topk_groups=kg, renormalize=True, scaling=scaling)
        assert (idx != 0).all() and (w[7] == 0).all() and (w[:7] > 0).all()


def test_small_scores_between_ordinary_rows():
    """Only the rows that need 64 bits are redone: their neighbours in the warp keep theirs."""
    x = make_logits(2, 333, 128, "f32")
    ordinary, _ = cm.route_experts(x, 8, cm.Scoring.Sigmoid, renormalize=True)
    low = x.clone()
    low[::7] -= 120.0
    w, idx = check_route(low, 8, scoring=cm.Scoring.Sigmoid, renormalize=True)
    keep = [t for t in range(333) if t % 7]
    assert torch.equal(w[keep], ordinary[keep])
