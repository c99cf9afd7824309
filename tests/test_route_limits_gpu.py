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


# ---- batches of which every warp takes several groups of rows ------------------------------------
# One pass of the gradient covers at most num_sms x 16 blocks x 4 warps x 32 / LPR rows, LPR the
# lanes of a row (8, 16 or 32 by k): 37888, 18944 and 9472 on 148 SMs; the dense one and the
# 64-bit kernel 9472 and 4736, the forward one with 4 lanes a row 75776.

def scores64(x, scoring):
    """Scores in 64 bits; logits of -inf score 0."""
    return torch.sigmoid(x) if scoring == 1 else torch.softmax(x, 1)


def route64(x, k, scoring, renormalize, scaling, bias=None):
    """Stable sorts of a 64-bit key: ties go to the lower id, as everywhere."""
    s = scores64(x.double(), scoring)
    key = x.double() if bias is None else s + bias.double()
    idx = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :k]
    r = s.gather(1, idx)
    if renormalize:
        r = r / r.sum(1, keepdim=True)
    return r * scaling, idx.int()


def backward64(g, x, idx, scoring, renormalize, scaling):
    s = scores64(x.double(), scoring)
    at = idx.long()
    r, d = s.gather(1, at), g.double() * scaling
    if renormalize:
        R = r.sum(1, keepdim=True)
        d = (d - (d * r).sum(1, keepdim=True) / R) / R
    ds = torch.zeros_like(s).scatter_add_(1, at, d)
    return ds * s * (1 - s) if scoring == 1 else s * (ds - (ds * s).sum(1, keepdim=True))


def spread(seed, T, E, dtype):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(T, E, generator=g, device="cuda") * 1.5
    return (x + torch.randn(E, generator=g, device="cuda") * 0.5).to(DT[dtype])


# E: rows of whole 16-byte pieces, tiles of whole pieces only, neither
@pytest.mark.parametrize("T,E,k", [(80001, 64, 8), (80003, 36, 5), (80001, 33, 3), (40001, 64, 12),
                                   (40003, 23, 10), (20011, 72, 20), (20011, 61, 17)])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("scoring,renormalize", [(0, True), (1, True), (1, False), (0, False)])
def test_gradients_of_several_passes(T, E, k, dtype, scoring, renormalize):
    """Zeros of the second tile, places cleared between passes, picks loaded a pass ahead, a short
    last tile behind full ones: all rows against the formula."""
    x = spread(E, T, E, dtype)
    w, idx = cm.route_experts(x, k, cm.Scoring(scoring), renormalize=renormalize, scaling=1.5)
    g = torch.randn(w.shape, generator=torch.Generator(device="cuda").manual_seed(k), device="cuda")
    d = cm.route_experts_backward(g, x, w, idx, cm.Scoring(scoring), renormalize, 1.5)
    ref = backward64(g, x, idx, scoring, renormalize, 1.5)
    tol = 2 * REL * 2 * 1.5 * g.abs().amax(1, keepdim=True).double()
    if dtype != "f32":
        tol = tol + torch.finfo(x.dtype).eps / 2 * ref.abs() + 2.0 ** -25
    assert ((d.double() - ref).abs() <= tol).all()
    if scoring == 1 or renormalize:  # zero but at the picks
        rest = torch.ones_like(d, dtype=torch.bool).scatter_(1, idx.long(), False)
        assert (d[rest] == 0).all()


@pytest.mark.parametrize("T,E,k,n,kg", [(160001, 64, 8, 1, 1), (160003, 30, 4, 1, 1),
                                        (80001, 128, 8, 1, 1), (80001, 16, 3, 1, 1),
                                        (40003, 256, 8, 1, 1), (40001, 100, 12, 1, 1),
                                        (20001, 480, 7, 12, 12)])
@pytest.mark.parametrize("scoring,with_bias", [(0, False), (1, False), (1, True), (0, True)])
def test_routing_of_several_passes(T, E, k, n, kg, scoring, with_bias):
    """All rows against stable 64-bit sorts (every group stays open where there are groups)."""
    x = spread(E + k, T, E, "f32" if E % 4 == 0 else "bf16")
    bias = None
    if with_bias:
        gen = torch.Generator(device="cuda").manual_seed(5)
        bias = torch.round(torch.randn(E, generator=gen, device="cuda") * 100) / 1000
    w, idx = cm.route_experts(x, k, cm.Scoring(scoring), bias=bias, num_groups=n, topk_groups=kg,
                              renormalize=True, scaling=2.5)
    w_ref, i_ref = route64(x, k, scoring, True, 2.5, bias)
    assert torch.equal(idx, i_ref)
    assert ((w.double() - w_ref).abs() <= REL * w_ref).all()


# ---- shapes that are ranked with 64-bit keys: more than 16 experts of a group to a lane -----------

@pytest.mark.parametrize("E,n,kg,k", [(510, 5, 2, 4), (510, 5, 3, 20), (480, 12, 5, 8), (480, 12, 1, 9),
                                      (510, 17, 4, 6), (511, 7, 2, 32), (510, 3, 1, 8),
                                      (510, 30, 30, 11)])
@pytest.mark.parametrize("scoring", [0, 1])
@pytest.mark.parametrize("group_score", [0, 1])
@pytest.mark.parametrize("with_bias", [False, True])
def test_groups_ranked_in_64_bits(E, n, kg, k, group_score, with_bias, scoring):
    bias = None
    if with_bias:
        bias = np.round(np.random.default_rng(E + n).normal(size=E) * 0.1, 3)
        bias[7], bias[8] = -np.inf, np.nan
    for dtype in ("f32", "bf16", "f16"):
        x = make_logits(E * 7 + kg, 29, E, dtype)
        x[:, 6::7] = float("-inf")          # out of service
        x[3] = float("-inf")                # padding
        x[4, 2:] = float("nan")
        x[5] = 0.25                         # all equal
        x[6, : E // n] = float("-inf")      # a whole group
        check_route(x, k, bias=bias, scoring=cm.Scoring(scoring), num_groups=n, topk_groups=kg,
                    group_score=cm.GroupScore(group_score), renormalize=(E % 2 == 0), scaling=2.5)
