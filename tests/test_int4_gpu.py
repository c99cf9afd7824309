"""The expert FFN on 4-bit weights against a 64-bit restatement (bounds: int4_testlib)."""
import numpy as np
import pytest
import torch

import candle_moe as cm
from int4_testlib import DT, check, dequantise, random_weights, reference, routing, unpack

pytestmark = pytest.mark.gpu


def make(seed, T, E, k, H, I, G, dtype, zeros, nomic, skip=0.0):
    rng = np.random.default_rng(seed)
    mats = (random_weights(rng, E, H, I, G, dtype, zeros),
            None if nomic else random_weights(rng, E, H, I, G, dtype, zeros),
            random_weights(rng, E, I, H, G, dtype, zeros))
    x = torch.from_numpy(rng.normal(size=(T, H))).to(DT[dtype]).cuda()
    w, idx = routing(rng, T, E, k, skip)
    return x, mats, w, idx


def run(x, mats, w, idx, act, rounded=False):
    got = cm.fused_moe_int4(x, cm.Int4Experts(*mats), w, idx, act)
    y, b = reference(x, mats, w, idx, act, rounded)
    rel = check(got, y, b)
    assert rel <= torch.finfo(x.dtype).eps, rel
    return got


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("T,E,k,H,I,G", [
    (1, 1, 1, 64, 64, 32), (1, 8, 2, 256, 128, 64), (1, 16, 8, 512, 384, 128),
    (2, 3, 3, 128, 192, 64), (5, 60, 4, 192, 320, 32), (8, 8, 2, 1024, 256, 128),
    (9, 2, 1, 128, 64, 32), (16, 4, 2, 320, 64, 64), (33, 5, 2, 256, 256, 128),
    (63, 7, 3, 64, 448, 64), (130, 128, 8, 128, 128, 32), (200, 2, 2, 192, 128, 64)])
def test_ffn(T, E, k, H, I, G, dtype, zeros):
    for nomic in (False, True):
        x, mats, w, idx = make(T + E + H, T, E, k, H, I, G, dtype, zeros, nomic)
        run(x, mats, w, idx, cm.Activation.Gelu if nomic else cm.Activation.Silu,
            rounded=T * k > 4 * E)


@pytest.mark.parametrize("act", [0, 1, 2])
def test_activations(act):
    run(*make(act, 6, 4, 2, 128, 128, 32, "bf16", True, False), act)


@pytest.mark.parametrize("T", [1, 4, 40])
def test_skipped_slots(T):
    """Ids >= E contribute nothing; a token with none left, and an expert without rows, work; an
    expert twice in one token counts twice."""
    x, mats, w, idx = make(77, T, 6, 3, 128, 128, 64, "bf16", False, False, skip=0.4)
    idx[0] = 6
    idx[T - 1, 0] = -1
    if T > 3:
        idx[2] = 4
    got = run(x, mats, w, idx, 0, rounded=True)
    if T > 1:
        assert (got[0] == 0).all()
    idx.fill_(6)
    assert (cm.fused_moe_int4(x, cm.Int4Experts(*mats), w, idx) == 0).all()


def test_all_rows_on_one_expert():
    x, mats, w, idx = make(78, 150, 5, 1, 128, 192, 32, "bf16", True, False)
    idx.fill_(3)
    run(x, mats, w, idx, 0, rounded=True)


def test_zero_tokens():
    x, mats, w, idx = make(1, 0, 4, 2, 64, 64, 32, "bf16", False, False)
    assert cm.fused_moe_int4(x, cm.Int4Experts(*mats), w, idx).shape == (0, 64)


@pytest.mark.parametrize("T", [12, 60, 900])
def test_infinities_stay_in_their_rows(T):
    """A token of infinities or NaN does not reach the other tokens' rows."""
    x, mats, w, idx = make(5, T, 4, 2, 128, 128, 64, "bf16", False, False)
    ex = cm.Int4Experts(*mats)
    clean = cm.fused_moe_int4(x, ex, w, idx)
    x[3] = float("inf")
    x[7] = float("nan")
    got = cm.fused_moe_int4(x, ex, w, idx)
    keep = [t for t in range(T) if t not in (3, 7)]
    assert torch.equal(got[keep], clean[keep])


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("E,K,N,G", [(1, 64, 64, 32), (3, 128, 192, 64), (2, 384, 64, 128)])
def test_quantize(E, K, N, G, dtype, symmetric):
    rng = np.random.default_rng(K + N)
    w = rng.normal(size=(E, K, N)) * 0.02
    w[0, :G, 0] = 0.0                       # a group of zeros
    w[0, :G, 1] = np.abs(w[0, :G, 1]) + .01  # one sign only
    w = torch.from_numpy(w).to(DT[dtype]).cuda()
    got = cm.quantize_int4(w, G, symmetric)
    f = w.float().cpu().view(E, K // G, G, N)
    lo, hi = f.amin(2).clamp(max=0), f.amax(2).clamp(min=0)
    s = (torch.maximum(-lo, hi) / 7 if symmetric else (hi - lo) / 15).to(DT[dtype])
    assert torch.equal(got.scales.cpu(), s)
    sf = torch.where(s.float() > 0, s.float(), torch.ones(()))
    z = torch.full_like(sf, 8.0)
    if not symmetric:
        z = torch.where(s.float() > 0, torch.round(-lo / sf).clamp(0, 15), torch.zeros(()))
        assert torch.equal(got.zeros.cpu().float(), z)
    else:
        assert got.zeros is None
    q = (torch.round(f / sf.unsqueeze(2)) + z.unsqueeze(2)).clamp(0, 15).view(E, K, N)
    np.testing.assert_array_equal(unpack(got.q.cpu().numpy()), q.numpy().astype(np.uint8))


def test_quantised_layer_is_near_the_layer():
    """End to end: quantise and run; the reference is the layer on the values the nibbles stand
    for, and those are at most half a step (plus the scale's rounding over 8 steps) off."""
    torch.manual_seed(2)
    E, H, I, k, T = 6, 256, 192, 2, 20
    g, u = [torch.randn(E, H, I, device="cuda").mul_(0.05).bfloat16() for _ in range(2)]
    d = torch.randn(E, I, H, device="cuda").mul_(0.05).bfloat16()
    x = torch.randn(T, H, device="cuda").bfloat16()
    mats = tuple(cm.quantize_int4(m, 64, False) for m in (g, u, d))
    for m, w in zip(mats, (g, u, d)):
        v, _ = dequantise(m)
        step = np.repeat(m.scales.double().cpu().numpy(), 64, axis=1)
        assert (np.abs(v - w.double().cpu().numpy()) <= step * (1.0 + 16 * 2.0 ** -8)).all()
    w, idx = routing(np.random.default_rng(0), T, E, k)
    got = run(x, mats, w, idx, 0, rounded=True)
    again = cm.FusedMoE(E, k).forward_int4(
        x, cm.Int4Experts.quantize(g, u, d, group_size=64, symmetric=False), w, idx)
    assert torch.equal(got, again)


@pytest.mark.parametrize("T", [1, 24, 300])
def test_workspace_stream_graph_and_repeats(T):
    x, mats, w, idx = make(31, T, 9, 3, 256, 128, 64, "f16", True, False)
    ex = cm.Int4Experts(*mats)
    ref = cm.fused_moe_int4(x, ex, w, idx)
    n = cm.int4_workspace_size(T, 256, 128, 9, 3)
    ws = torch.full((n + 512,), 255, dtype=torch.uint8, device="cuda")
    out = torch.full_like(x, float("nan"))
    lo = -ws.data_ptr() % 256
    got = cm.fused_moe_int4(x, ex, w, idx, out=out, workspace=ws[lo:lo + n])
    assert got.data_ptr() == out.data_ptr() and torch.equal(got, ref)
    assert (ws[lo + n:] == 255).all() and (ws[:lo] == 255).all()
    with pytest.raises(cm.MoeError):
        cm.fused_moe_int4(x, ex, w, idx, workspace=ws[lo:lo + n - 1])
    with pytest.raises(cm.MoeError):
        cm.fused_moe_int4(x, ex, w, idx, workspace=ws[lo + 1:lo + 1 + n])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        side = cm.fused_moe_int4(x, ex, w, idx)
    # two calls at once, each with its own pool workspace
    main = cm.fused_moe_int4(x, ex, w, idx)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(side, ref) and torch.equal(main, ref)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = cm.fused_moe_int4(x, ex, w, idx)
        graphs.append((g, o))
    x.neg_()
    idx.copy_(idx.flip(0))
    for g, _ in graphs + graphs[::-1]:
        g.replay()
    ref2 = cm.fused_moe_int4(x, ex, w, idx)
    for _, o in graphs:
        assert torch.equal(o, ref2)


def test_refusals():
    x, mats, w, idx = make(3, 4, 4, 2, 128, 64, 32, "bf16", False, False)
    ex = cm.Int4Experts(*mats)
    other = make(3, 4, 4, 2, 128, 64, 64, "bf16", False, False)[1]
    with pytest.raises(ValueError, match="share"):
        cm.Int4Experts(mats[0], other[1], mats[2])
    with pytest.raises(ValueError, match="down"):
        cm.Int4Experts(mats[0], mats[1], mats[0])
    with pytest.raises(ValueError, match="up"):
        cm.Int4Experts(mats[0], mats[2], mats[2])
    with pytest.raises(TypeError, match="dtype"):
        cm.fused_moe_int4(x.half(), ex, w, idx)
    with pytest.raises(ValueError, match="Hidden"):
        cm.fused_moe_int4(x[:, :64].contiguous(), ex, w, idx)
    with pytest.raises(ValueError, match="tokens"):
        cm.fused_moe_int4(x[:3], ex, w, idx)
    with pytest.raises(ValueError, match="selected"):
        cm.fused_moe_int4(x, ex, w[:, :1].contiguous(), idx)
    with pytest.raises(ValueError, match="contiguous"):
        cm.fused_moe_int4(x.t().contiguous().t(), ex, w, idx)
    with pytest.raises(TypeError, match="expert_indices"):
        cm.fused_moe_int4(x, ex, w, idx.long())
    with pytest.raises(ValueError, match="experts"):
        cm.FusedMoE(5, 2).forward_int4(x, ex, w, idx)
    with pytest.raises(ValueError, match="out"):
        cm.fused_moe_int4(x, ex, w, idx, out=x.float())
    # a row that does not start on 16 bytes
    odd = torch.empty(4 * 128 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(4, 128)
    with pytest.raises(cm.MoeError):
        cm.fused_moe_int4(odd, ex, w, idx)
    with pytest.raises(cm.MoeError):
        cm.fused_moe_int4(x, ex, w, idx, out=odd)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("T,E,k,H,I,G", [(300, 4, 2, 256, 384, 64), (517, 7, 3, 384, 128, 32),
                                         (1500, 16, 3, 128, 192, 64), (400, 1, 1, 128, 256, 128),
                                         (850, 2, 1, 384, 128, 32), (500, 1, 1, 192, 64, 64)])
def test_many_rows(T, E, k, H, I, G, dtype, zeros):
    """Hundreds of rows per expert, on both sides of the 384 from which the weights are expanded to
    16 bits, more than 4096 rows, and a shape that stays packed."""
    for nomic in (False, True):
        x, mats, w, idx = make(T + E, T, E, k, H, I, G, dtype, zeros, nomic, skip=0.1)
        run(x, mats, w, idx, cm.Activation.Gelu if nomic else cm.Activation.Silu, rounded=True)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("T,E,k,H,I,G", [(40, 3, 2, 128, 128, 32), (33, 2, 1, 256, 128, 128),
                                         (64, 4, 1, 128, 384, 64), (150, 9, 3, 512, 256, 64),
                                         (70, 1, 1, 256, 256, 128), (100, 16, 4, 384, 640, 32)])
def test_some_rows_per_expert(T, E, k, H, I, G, dtype, zeros):
    """A few to a few tens of rows per expert, ragged, with experts of none and of many."""
    for nomic in (False, True):
        x, mats, w, idx = make(T + E + G, T, E, k, H, I, G, dtype, zeros, nomic, skip=0.1)
        idx[: T // 2, 0] = 0
        run(x, mats, w, idx, cm.Activation.Gelu if nomic else cm.Activation.Silu, rounded=True)


@pytest.mark.parametrize("T,E,k", [(6, 8, 8), (7, 8, 7), (24, 30, 2), (25, 30, 2), (48, 4, 1)])
def test_around_the_table_limit(T, E, k):
    """48 rows and the first calls beyond, tokens of one expert with more than a chunk of rows."""
    x, mats, w, idx = make(T * k, T, E, k, 192, 128, 64, "f16", True, False)
    run(x, mats, w, idx, 0, rounded=True)
    idx[:, 0] = 1
    run(x, mats, w, idx, 0, rounded=True)


def test_wide_and_long_shapes():
    """More columns than one wave of CTAs takes, and a long reduction with an odd number of blocks."""
    for T in (2, 70):
        x, mats, w, idx = make(T, T, 2, 2, 4416, 64, 64, "bf16", False, False)
        run(x, mats, w, idx, 0, rounded=True)


def test_output_over_the_input_is_refused():
    x, mats, w, idx = make(5, 5, 2, 1, 128, 128, 32, "bf16", False, False)
    ex = cm.Int4Experts(*mats)
    both = torch.zeros(9, 128, dtype=torch.bfloat16, device="cuda")
    for out in (x, both[4:]):
        src = x if out is x else both[:5]
        before = src.clone()
        with pytest.raises(cm.MoeError):
            cm.fused_moe_int4(src, ex, w, idx, out=out)
        assert torch.equal(src, before)
    assert torch.equal(cm.fused_moe_int4(both[:4], ex, w[:4], idx[:4], out=both[4:8]),
                       cm.fused_moe_int4(both[:4], ex, w[:4], idx[:4]))


@pytest.mark.parametrize("T,E,k", [(3, 2048, 8), (300, 2048, 2), (150, 1501, 3), (1100, 513, 4)])
def test_many_experts(T, E, k):
    """Up to the most experts there may be, an odd number, and more than 4096 rows over them."""
    x, mats, w, idx = make(E + T, T, E, k, 64, 64, 32, "bf16", True, False, skip=0.1)
    idx[T - 1, 0] = E - 1
    run(x, mats, w, idx, 0, rounded=True)


def test_one_token_many_times_one_expert():
    """More slots than experts: every slot of the tokens picks the same one or two."""
    for T, k in ((1, 48), (1, 49), (3, 40)):
        x, mats, w, idx = make(T, T, 64, k, 128, 64, 32, "bf16", False, False)
        idx.fill_(63)
        idx[:, ::3] = 0
        run(x, mats, w, idx, 0, rounded=True)
