"""SparseMoeBlock with general routing and with 4-bit experts: router projection, routing and
experts together, against the 64-bit restatements of the two (bounds: int4_testlib)."""
import numpy as np
import pytest
import torch

import candle_moe as cm
import route_testlib as rt
from int4_testlib import DT, check, random_weights, reference

pytestmark = pytest.mark.gpu


def block(seed, E, H, I, k, G, dtype, nomic=False, **kw):
    rng = np.random.default_rng(seed)
    mats = (random_weights(rng, E, H, I, G, dtype, True),
            None if nomic else random_weights(rng, E, H, I, G, dtype, True),
            random_weights(rng, E, I, H, G, dtype, True))
    router = torch.from_numpy(rng.normal(size=(E, H)) * 0.05).to(DT[dtype]).cuda()
    b = cm.SparseMoeBlock(router, None, None, None, k,
                          activation=cm.Activation.Gelu if nomic else cm.Activation.Silu,
                          int4_experts=cm.Int4Experts(*mats), **kw)
    return b, mats


def route_ref(logits, k, kw):
    bias = kw.get("correction_bias")
    return rt.route(logits.double().cpu().numpy(), k, int(kw.get("scoring", 0)),
                    None if bias is None else bias.double().cpu().numpy(), kw.get("num_groups", 1),
                    kw.get("topk_groups", 1), int(kw.get("group_score", 0)),
                    kw.get("norm_topk_prob", True), kw.get("routed_scaling", 1.0))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("T", [1, 5, 90, 700])
@pytest.mark.parametrize("E,k,groups", [(16, 4, 4), (12, 3, 1), (8, 2, 1)])
def test_block(dtype, T, E, k, groups):
    H, I, G = 256, 128, 64
    kw = {}
    if E != 8:
        kw = dict(scoring=cm.Scoring.Sigmoid, routed_scaling=2.5, num_groups=groups,
                  topk_groups=max(1, groups // 2), group_score=cm.GroupScore.Top2,
                  correction_bias=torch.linspace(-0.2, 0.2, E, device="cuda"))
    b, mats = block(E + T, E, H, I, k, G, dtype, nomic=(E == 12), **kw)
    x = torch.from_numpy(np.random.default_rng(T).normal(size=(T, H))).to(DT[dtype]).cuda()
    out, logits = b.forward(x, return_router_logits=True)
    assert logits.shape == (T, E) and logits.dtype == torch.float32
    # a logit sums H exact products in f32
    ref = x.double() @ b.router_weight.double().t()
    slack = 64 * 2.0 ** -23 * (x.double().abs() @ b.router_weight.double().abs().t())
    assert ((logits.double() - ref).abs() <= slack).all()
    w, idx, again = b.route(x)
    assert torch.equal(again, logits)
    w_ref, i_ref = route_ref(logits, k, kw)
    np.testing.assert_array_equal(idx.cpu().numpy(), i_ref)
    assert np.allclose(w.double().cpu().numpy(), w_ref, rtol=80 * 2.0 ** -24, atol=0)
    y, bound = reference(x, mats, w, idx, int(b.experts.activation), weights_rounded=True)
    assert check(out, y, bound) <= torch.finfo(x.dtype).eps


def test_block_with_16_bit_experts_and_general_routing():
    torch.manual_seed(0)
    T, E, H, I, k = 40, 6, 128, 256, 2
    r = (torch.randn(E, H, device="cuda") * 0.05).bfloat16()
    g, u = [(torch.randn(E, H, I, device="cuda") * 0.05).bfloat16() for _ in range(2)]
    d = (torch.randn(E, I, H, device="cuda") * 0.05).bfloat16()
    x = torch.randn(T, H, device="cuda").bfloat16()
    b = cm.SparseMoeBlock(r, g, u, d, k, scoring=cm.Scoring.Sigmoid)
    out, logits = b.forward(x, return_router_logits=True)
    w, idx = cm.route_experts(logits, k, cm.Scoring.Sigmoid, renormalize=True)
    assert torch.equal(out, cm.FusedMoE(E, k).forward(x, g, u, d, w, idx, 0))


def test_default_block_keeps_the_fused_router():
    torch.manual_seed(1)
    E, H, k = 8, 128, 2
    r = (torch.randn(E, H, device="cuda") * 0.05).bfloat16()
    g = (torch.randn(E, H, 128, device="cuda") * 0.05).bfloat16()
    b = cm.SparseMoeBlock(r, g, g, None, k)
    assert not b.general_routing
    x = torch.randn(9, H, device="cuda").bfloat16()
    w, idx, logits = b.route(x)
    w2, idx2, _, l2 = cm.router_project_topk(x, r, k, renormalize=True, return_logits=True)
    assert torch.equal(w, w2) and torch.equal(idx, idx2) and torch.equal(logits, l2)


def test_tokens_without_experts_in_the_block():
    """Rows whose logits leave no expert (here: all masked by a bias of -inf) come out as zero."""
    b, _ = block(3, 8, 128, 64, 2, 32, "bf16", correction_bias=torch.full((8,), -float("inf"),
                                                                        device="cuda"))
    x = torch.randn(7, 128, device="cuda").bfloat16()
    assert (b.forward(x) == 0).all()


def test_router_training_step():
    """The gradient of a loss on the routing weights reaches the router's weight: route_experts
    and route_experts_backward around the projection, against differentiation in 64 bits."""
    torch.manual_seed(2)
    T, E, H, k = 50, 20, 64, 4
    x = torch.randn(T, H, device="cuda")
    r = torch.randn(E, H, device="cuda") * 0.1
    target = torch.rand(T, k, device="cuda")
    logits = x @ r.t()
    w, idx = cm.route_experts(logits, k, cm.Scoring.Sigmoid, renormalize=True, scaling=1.5)
    grad_w = 2 * (w - target)
    grad_r = cm.route_experts_backward(grad_w, logits, w, idx, cm.Scoring.Sigmoid, True, 1.5).t() @ x
    l64 = logits.double().requires_grad_(True)
    s = torch.sigmoid(l64).gather(1, idx.long())
    w64 = 1.5 * s / s.sum(1, keepdim=True)
    (g64,) = torch.autograd.grad(w64, l64, grad_w.double())
    ref = g64.t() @ x.double()
    # the gradient's own bound (2 * 80 * 2^-24 of 2 * 1.5 * max|g|) and T f32 additions
    tol = (160 + T) * 2.0 ** -24 * 3 * grad_w.abs().max().double() * x.abs().double().sum(0)
    assert ((grad_r.double() - ref).abs() <= tol).all()


def test_block_refusals():
    b, mats = block(1, 8, 128, 64, 2, 32, "bf16")
    r = b.router_weight
    with pytest.raises(ValueError, match="takes the place"):
        cm.SparseMoeBlock(r, r, None, None, 2, int4_experts=b.int4_experts)
    with pytest.raises(ValueError, match="experts"):
        cm.SparseMoeBlock(r[:4], None, None, None, 2, int4_experts=b.int4_experts)
    with pytest.raises(cm.MoeError):
        cm.SparseMoeBlock(r, None, None, None, 2, num_groups=3, int4_experts=b.int4_experts).forward(
            torch.zeros(2, 128, dtype=torch.bfloat16, device="cuda"))


@pytest.mark.parametrize("E,kw", [(8, {}), (12, {"scoring": cm.Scoring.Sigmoid})])
def test_zero_tokens_in_the_block(E, kw):
    b, _ = block(4, E, 128, 64, 2, 32, "bf16", **kw)
    out, logits = b.forward(torch.zeros(0, 128, dtype=torch.bfloat16, device="cuda"),
                            return_router_logits=True)
    assert out.shape == (0, 128) and logits.shape == (0, E)


def test_4_bit_block_with_a_shared_expert():
    """The shared expert's contribution is added to the 4-bit experts'."""
    torch.manual_seed(5)
    b, mats = block(6, 8, 128, 64, 2, 32, "bf16")
    sg, su = [(torch.randn(1, 128, 192, device="cuda") * 0.05).bfloat16() for _ in range(2)]
    sd = (torch.randn(1, 192, 128, device="cuda") * 0.05).bfloat16()
    both = cm.SparseMoeBlock(b.router_weight, None, None, None, 2, int4_experts=b.int4_experts,
                             shared_gate=sg, shared_up=su, shared_down=sd)
    alone = cm.SparseMoeBlock(b.router_weight[:1], sg, su, sd, 1)
    x = torch.randn(21, 128, device="cuda").bfloat16()
    a, c, got = b.forward(x), alone.forward(x), both.forward(x)
    # two sums, each rounded by half a step, against one of the rounded parts
    size = a.abs().double() + c.abs().double()
    assert ((got.double() - a.double() - c.double()).abs() <= 3 * 2.0 ** -8 * size).all()
