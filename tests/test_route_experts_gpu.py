"""General expert routing and its gradient on the GPU against a 64-bit restatement.

Tolerances.  The indices have to be equal.  A softmax weight goes through l - m (off by
|l - m| 2^-24, which the exponential turns into a relative error), expf (2 ulp), a sum of at most
16 terms a lane and 5 across lanes, a division, the sum over the picks (5 more), a division and
the scaling: under (D + 2*4 + 21 + 5 + 4) 2^-24 relative for picks at most D below the maximum;
D < 40 here, so 80 * 2^-24.  A sigmoid weight has fewer steps.  The gradient takes differences
of such values, so it is off by the same share of the largest term, 2 scaling max|g|; another
factor two covers the products.  16-bit gradients add half a step of rounding (f16: and half a
step of its smallest subnormal, 2^-25)."""
import numpy as np
import pytest
import torch

import candle_moe as cm
import route_testlib as rt

pytestmark = pytest.mark.gpu
REL = 80 * 2.0 ** -24
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def make_logits(seed, T, E, dtype, spread=1.5):
    rng = np.random.default_rng(seed)
    x = rng.normal(size=(T, E)) * spread + rng.normal(size=E) * 0.5
    return torch.from_numpy(x).to(DT[dtype]).cuda()


def check_route(x, k, bias=None, **kw):
    b = None if bias is None else torch.from_numpy(bias.astype(np.float32)).cuda()
    w, idx = cm.route_experts(x, k, bias=b, **kw)
    b64 = None if bias is None else bias.astype(np.float32).astype(np.float64)
    okw = {a: (int(v) if a in ("scoring", "group_score") else v) for a, v in kw.items()}
    w_ref, i_ref = rt.route(x.double().cpu().numpy(), k, bias=b64, **okw)
    np.testing.assert_array_equal(idx.cpu().numpy(), i_ref)
    err = np.abs(w.double().cpu().numpy() - w_ref)
    assert (err <= REL * np.abs(w_ref) + 1e-37).all(), err.max()
    return w, idx


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 128, 8), (3, 5, 5), (33, 60, 4), (129, 256, 8),
                                   (70, 7, 2), (65, 384, 22), (40, 512, 32), (257, 33, 1)])
@pytest.mark.parametrize("scoring", [0, 1])
def test_plain(dtype, T, E, k, scoring):
    x = make_logits(T * 1000 + E, T, E, dtype)
    check_route(x, k, scoring=cm.Scoring(scoring), renormalize=(T % 2 == 1), scaling=1.0)


@pytest.mark.parametrize("scoring", [0, 1])
@pytest.mark.parametrize("group_score", [0, 1])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("E,n,kg,k", [(256, 8, 4, 8), (160, 8, 3, 6), (64, 4, 1, 3), (60, 5, 2, 4),
                                      (96, 32, 7, 12), (34, 17, 2, 3), (512, 2, 1, 32),
                                      (32, 32, 5, 5), (66, 3, 3, 9), (256, 1, 1, 8), (60, 1, 1, 4),
                                      (100, 1, 1, 12), (512, 16, 4, 8), (8, 2, 1, 2)])
def test_groups(E, n, kg, k, group_score, with_bias, scoring):
    T = 61
    rng = np.random.default_rng(E + n)
    bias = np.round(rng.normal(size=E) * 0.1, 3) if with_bias else None
    for dtype in ("f32", "bf16", "f16"):
        x = make_logits(E * 7 + kg, T, E, dtype)
        check_route(x, k, bias=bias, scoring=cm.Scoring(scoring), num_groups=n, topk_groups=kg,
                    group_score=cm.GroupScore(group_score), renormalize=True, scaling=2.5)


@pytest.mark.parametrize("scoring", [0, 1])
@pytest.mark.parametrize("with_bias", [False, True])
def test_ties_and_near_ties(scoring, with_bias):
    """Equal logits, and logits one f32 step apart, whose f32 scores often coincide."""
    rng = np.random.default_rng(11)
    T, E, k = 200, 96, 8
    base = rng.normal(size=(T, 1)).astype(np.float32) + 2.0
    steps = rng.integers(-2, 3, size=(T, E))
    x = base + steps.astype(np.float32) * np.float32(2.0 ** -22)
    x[:, ::5] = base  # ties
    bias = np.zeros(E) if with_bias else None
    check_route(torch.from_numpy(x.astype(np.float32)).cuda(), k, bias=bias,
                scoring=cm.Scoring(scoring), renormalize=True)
    if with_bias:  # scores that meet only through the bias
        b = rng.integers(-2, 3, size=E) * 2.0 ** -25
        check_route(torch.from_numpy(x.astype(np.float32)).cuda(), k, bias=b,
                    scoring=cm.Scoring(scoring), num_groups=8, topk_groups=3,
                    group_score=cm.GroupScore.Top2)


@pytest.mark.parametrize("scoring", [0, 1])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("n,kg", [(1, 1), (4, 2)])
def test_masked_rows(scoring, with_bias, n, kg):
    """Rows with fewer available experts than picks, or none; NaN counts as unavailable; the
    type's lowest finite value does not."""
    T, E, k = 64, 24, 6
    x = make_logits(3, T, E, "f32")
    x[:, 3] = float("-inf")
    x[0] = float("-inf")
    x[1, 2:] = float("-inf")
    x[2, 5:] = float("nan")
    x[3] = float("nan")
    x[4, 1:] = torch.finfo(torch.float32).min
    x[5] = torch.finfo(torch.float32).min
    x[6, 6:] = float("-inf")
    bias = None
    if with_bias:
        bias = np.linspace(-0.3, 0.3, E)
        bias[7], bias[8] = -np.inf, np.nan
    w, idx = check_route(x, k, bias=bias, scoring=cm.Scoring(scoring), num_groups=n,
                         topk_groups=kg, group_score=cm.GroupScore.Top2, renormalize=True)
    assert (idx[0] == E).all() and (w[0] == 0).all()
    assert (idx[3] == E).all() and (w[3] == 0).all()
    assert torch.isfinite(w).all()


def test_extreme_logits():
    x = torch.tensor([[100.0, -100.0, 30.0, 0.0], [-90.0, -95.0, -80.0, -85.0],
                      [88.0, 87.0, 3e38, -3e38]], device="cuda")
    check_route(x, 2, scoring=cm.Scoring.Softmax)
    w, idx = cm.route_experts(x, 4, scoring=cm.Scoring.Sigmoid)
    assert idx.tolist() == [[0, 2, 3, 1], [2, 3, 0, 1], [2, 0, 1, 3]]
    assert torch.isfinite(w).all()
    # +inf is a valid logit for sigmoid scores
    x[0, 1] = float("inf")
    w, idx = cm.route_experts(x, 1, scoring=cm.Scoring.Sigmoid)
    assert idx[0, 0] == 1 and w[0, 0] == 1


def test_strided_rows_and_offsets():
    wide = make_logits(9, 37, 200, "bf16")
    for lo, E in ((0, 64), (3, 60), (8, 128), (1, 5)):
        view = wide[:, lo:lo + E]
        w, idx = cm.route_experts(view, 4, renormalize=True)
        w2, idx2 = cm.route_experts(view.contiguous(), 4, renormalize=True)
        assert torch.equal(idx, idx2) and torch.equal(w, w2)
        g = torch.randn_like(w)
        d = cm.route_experts_backward(g, view, w, idx, renormalize=False)
        d2 = cm.route_experts_backward(g, view.contiguous(), w, idx, renormalize=False)
        assert torch.equal(d, d2)
    every_other = wide[::2]
    w, idx = cm.route_experts(every_other, 3)
    w2, idx2 = cm.route_experts(every_other.contiguous(), 3)
    assert torch.equal(idx, idx2) and torch.equal(w, w2)


def test_many_tokens_agree_with_few():
    x = make_logits(17, 40000, 72, "f32")
    b = torch.randn(72, device="cuda") * 0.1
    kw = dict(scoring=cm.Scoring.Sigmoid, bias=b, num_groups=6, topk_groups=3,
              group_score=cm.GroupScore.Top2, renormalize=True)
    w, idx = cm.route_experts(x, 5, **kw)
    w2, idx2 = cm.route_experts(x[39990:], 5, **kw)
    assert torch.equal(idx[39990:], idx2) and torch.equal(w[39990:], w2)
    w_ref, i_ref = rt.route(x[:300].double().cpu().numpy(), 5, 1, b.double().cpu().numpy(), 6, 3,
                            1, True)
    np.testing.assert_array_equal(idx[:300].cpu().numpy(), i_ref)


def check_backward(x, k, scoring, renormalize, scaling, idx=None, seed=0):
    w, i = cm.route_experts(x, k, scoring=cm.Scoring(scoring), renormalize=renormalize,
                            scaling=scaling)
    if idx is not None:
        i = idx
        w64 = np.stack([rt.weights(l, np.where((r >= 0) & (r < x.shape[1]), r, x.shape[1]),
                                   scoring, renormalize, scaling)
                        for l, r in zip(x.double().cpu().numpy(), i.cpu().numpy())])
        w = torch.from_numpy(w64).float().cuda()
    g = torch.from_numpy(np.random.default_rng(seed).normal(size=tuple(w.shape))).float().cuda()
    d = cm.route_experts_backward(g, x, w, i, scoring=cm.Scoring(scoring),
                                  renormalize=renormalize, scaling=scaling)
    assert d.dtype == x.dtype and d.shape == x.shape
    ref = rt.backward(g.double().cpu().numpy(), x.double().cpu().numpy(), i.cpu().numpy(), scoring,
                      renormalize, scaling)
    gmax = np.abs(g.double().cpu().numpy()).max(axis=1, keepdims=True)
    tol = 2 * REL * 2 * scaling * gmax * (1 if idx is None else k)
    if x.dtype != torch.float32:
        tol = tol + torch.finfo(x.dtype).eps / 2 * np.abs(ref) + 2.0 ** -25
    err = np.abs(d.double().cpu().numpy() - ref)
    assert (err <= tol).all(), (err - tol).max()
    return d


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 128, 8), (33, 60, 4), (130, 256, 8), (9, 5, 5),
                                   (40, 512, 32), (77, 97, 3)])
@pytest.mark.parametrize("scoring", [0, 1])
@pytest.mark.parametrize("renormalize", [False, True])
def test_backward(dtype, T, E, k, scoring, renormalize):
    check_backward(make_logits(T + E, T, E, dtype), k, scoring, renormalize, 2.5, seed=T)


@pytest.mark.parametrize("scoring", [0, 1])
@pytest.mark.parametrize("renormalize", [False, True])
def test_backward_masked_and_repeated(scoring, renormalize):
    """Masked experts and empty rows have zero gradients; ids outside [0, E) count for nothing;
    an id that a token holds twice contributes twice."""
    T, E, k = 12, 20, 4
    x = make_logits(4, T, E, "f32")
    x[:, 2] = float("-inf")
    x[0] = float("-inf")
    x[1, 3:] = float("nan")
    d = check_backward(x, k, scoring, renormalize, 1.0)
    assert (d[:, 2] == 0).all() and (d[0] == 0).all() and (d[1, 3:] == 0).all()
    idx = torch.from_numpy(np.random.default_rng(1).integers(3, 8, size=(T, k))).int().cuda()
    idx[2, 1] = E
    idx[3, 2] = -1
    idx[4, 0] = 2 ** 31 - 1
    x = make_logits(5, T, E, "f32")
    check_backward(x, k, scoring, renormalize, 1.5, idx=idx)


def test_backward_is_deterministic_and_whole():
    x = make_logits(8, 5000, 100, "f32")
    w, i = cm.route_experts(x, 8, renormalize=True)
    g = torch.randn_like(w)
    a = cm.route_experts_backward(g, x, w, i, renormalize=True)
    for _ in range(3):
        junk = torch.full((5000, 100), float("nan"), device="cuda")
        del junk
        assert torch.equal(a, cm.route_experts_backward(g, x, w, i, renormalize=True))


def test_refusals():
    x = make_logits(1, 4, 8, "f32")
    with pytest.raises(cm.MoeError):
        cm.route_experts(x, 9)
    with pytest.raises(cm.MoeError):
        cm.route_experts(x, 0)
    with pytest.raises(cm.MoeError):
        cm.route_experts(x, 2, num_groups=3)
    with pytest.raises(cm.MoeError):
        cm.route_experts(x, 2, scaling=0.0)
    with pytest.raises(cm.MoeError):
        cm.route_experts(torch.zeros(2, 600, device="cuda"), 2)
    with pytest.raises(ValueError, match="bias"):
        cm.route_experts(x, 2, bias=torch.zeros(7, device="cuda"))
    with pytest.raises(ValueError, match="cuda"):
        cm.route_experts(x, 2, bias=torch.zeros(8))
    with pytest.raises(TypeError):
        cm.route_experts(x.double(), 2)
    with pytest.raises(ValueError, match="contiguous rows"):
        cm.route_experts(torch.zeros(8, 4, device="cuda").t(), 2)
    with pytest.raises(ValueError, match="contiguous rows"):
        cm.route_experts(torch.zeros(1, 8, device="cuda").expand(4, 8), 2)
    w, i = cm.route_experts(x, 2)
    with pytest.raises(ValueError, match="grad_weights"):
        cm.route_experts_backward(w[:, :1], x, w, i)
    with pytest.raises(TypeError, match="indices"):
        cm.route_experts_backward(w, x, w, i.long())
    assert cm.route_experts(x[:0], 2)[0].shape == (0, 2)
    assert cm.route_experts_backward(w[:0], x[:0], w[:0], i[:0]).shape == (0, 8)


def test_on_another_stream_and_in_a_graph():
    x = make_logits(21, 300, 64, "bf16")
    w0, i0 = cm.route_experts(x, 6, renormalize=True)
    g = torch.randn_like(w0)
    d0 = cm.route_experts_backward(g, x, w0, i0, renormalize=True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        w1, i1 = cm.route_experts(x, 6, renormalize=True)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(w0, w1) and torch.equal(i0, i1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w2, i2 = cm.route_experts(x, 6, renormalize=True)
        d2 = cm.route_experts_backward(g, x, w2, i2, renormalize=True)
    for seed in (22, 23):
        x.copy_(make_logits(seed, 300, 64, "bf16"))
        graph.replay()
        w3, i3 = cm.route_experts(x, 6, renormalize=True)
        assert torch.equal(w2, w3) and torch.equal(i2, i3)
        assert torch.equal(d2, cm.route_experts_backward(g, x, w3, i3, renormalize=True))
    assert not torch.equal(d0, d2)


@pytest.mark.parametrize("E,n,kg,k", [(128, 1, 1, 8), (256, 8, 4, 8), (60, 1, 1, 10), (40, 5, 2, 3),
                                      (512, 1, 1, 32), (4, 1, 1, 4)])
@pytest.mark.parametrize("scoring", [0, 1])
@pytest.mark.parametrize("with_bias", [False, True])
def test_constant_rows(E, n, kg, k, scoring, with_bias):
    """Every logit the same (an untrained router, a padded batch): the first experts of the first
    groups, at equal weights."""
    x = torch.zeros(70, E, device="cuda", dtype=torch.bfloat16)
    x[30:50] = 3.0
    bias = np.zeros(E) if with_bias else None
    w, idx = check_route(x, k, bias=bias, scoring=cm.Scoring(scoring), num_groups=n,
                         topk_groups=kg, group_score=cm.GroupScore.Top2, renormalize=True)
    assert (idx == torch.arange(k, device="cuda")).all()


def test_few_distinct_logits():
    """16-bit logits of a handful of values, with a bias of a handful: ties in every row."""
    rng = np.random.default_rng(8)
    x = torch.from_numpy(rng.integers(-3, 4, size=(300, 64)) * 0.5).bfloat16().cuda()
    bias = rng.integers(-1, 2, size=64) * 0.125
    for k in (4, 8, 20):
        for kw in (dict(), dict(num_groups=4, topk_groups=2, group_score=cm.GroupScore.Top2)):
            check_route(x, k, bias=bias, scoring=cm.Scoring.Sigmoid, renormalize=True, **kw)
            check_route(x, k, bias=bias, scoring=cm.Scoring.Softmax, **kw)
            check_route(x, k, scoring=cm.Scoring.Sigmoid, **kw)


@pytest.mark.parametrize("E,k", [(64, 4), (256, 8), (60, 3), (512, 32)])
def test_bias_off_its_alignment(E, k):
    x = make_logits(E, 50, E, "bf16")
    long = torch.randn(E + 3, device="cuda") * 0.1
    for lo in (1, 2, 3):
        b = long[lo:lo + E]
        w, idx = cm.route_experts(x, k, cm.Scoring.Sigmoid, bias=b)
        w2, idx2 = cm.route_experts(x, k, cm.Scoring.Sigmoid, bias=b.clone())
        assert torch.equal(idx, idx2) and torch.equal(w, w2)


@pytest.mark.parametrize("E,k", [(512, 32), (511, 31), (300, 17)])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_gradient_straight_from_the_library(E, k, dtype):
    """The most experts and slots, and a gradient that does not start on 16 bytes."""
    x = make_logits(E, 77, E, dtype)
    for scoring, renorm in ((0, False), (0, True), (1, True)):
        w, idx = cm.route_experts(x, k, cm.Scoring(scoring), renormalize=bool(renorm))
        g = torch.randn_like(w)
        ref = cm.route_experts_backward(g, x, w, idx, cm.Scoring(scoring), bool(renorm))
        out = torch.full((77 * E + 2,), 7.0, dtype=x.dtype, device="cuda")
        at = out[1:]
        code = {"f16": 0, "bf16": 1, "f32": 2}[dtype]
        st = cm.lib().moe_route_experts_backward(
            g.data_ptr(), x.data_ptr(), code, E, w.data_ptr(), idx.data_ptr(), 77, E, k, scoring,
            int(renorm), 1.0, at.data_ptr(), torch.cuda.current_stream().cuda_stream)
        assert st == 0
        assert torch.equal(at[:77 * E].view(77, E), ref)
        assert out[0] == 7 and out[-1] == 7
