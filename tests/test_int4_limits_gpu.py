"""The expert FFN on 4-bit weights where the ordinary tests do not reach (bounds: int4_testlib)."""
import numpy as np
import pytest
import torch

import candle_moe as cm
from int4_testlib import random_weights
from test_int4_gpu import make, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("G", [32, 64, 128])
def test_zero_points_out_of_range(G):
    """Refused; straight from the library the low four bits count, for every path alike."""
    E, K, N = 2, 128, 64
    w = random_weights(np.random.default_rng(G), E, K, N, G, "bf16", True)
    high = w.zeros.clone()
    high[1, 0, 5] += 16
    with pytest.raises(ValueError, match="zeros must be in 0..15"):
        cm.Int4Weights(w.q, w.scales, high, G)
    size = cm.lib().moe_int4_packed_size(E, K, N, G, 1, 1)
    out = torch.empty(size, dtype=torch.uint8, device="cuda")
    st = cm.lib().moe_int4_pack(w.q.data_ptr(), w.scales.data_ptr(), high.data_ptr(), E, K, N, G, 1,
                                out.data_ptr(), torch.cuda.current_stream().cuda_stream)
    assert st == 0
    assert torch.equal(out, w._pack())


@pytest.mark.parametrize("T,E,path", [(48, 4, 4), (49, 4, 5), (5000, 16, 5), (900, 2, 2), (30, 4, 4),
                                      (1, 4, 4)])
def test_path_and_phases_are_those_of_the_call(T, E, path):
    x, mats, w, idx = make(T, T, E, 1, 128, 128, 64, "bf16", False, False)
    ex = cm.Int4Experts(*mats)
    g = torch.zeros(E, 128, 128, dtype=torch.bfloat16, device="cuda")
    moe = cm.FusedMoE(E, 1)
    other = x[:1] if path == 2 else x[:1].repeat(64, 1)
    moe.forward(other, g, g, g, w[:1].repeat(len(other), 1), idx[:1].repeat(len(other), 1), 0)
    assert cm.last_gemm_path() not in (path, 0)
    cm.phase_timing(True)
    for _ in range(3):
        cm.fused_moe_int4(x, ex, w, idx)
    assert cm.last_gemm_path() == path
    times, calls = cm.phase_times()
    cm.phase_timing(False)
    assert calls == 3 and times["gemm1"] > 0 and times["gemm2"] > 0
    assert all(t >= 0 for t in times.values())
    with pytest.raises(cm.MoeError):
        cm.fused_moe_int4(x, ex, w, idx, out=x)
    assert cm.last_gemm_path() == 0


def test_weights_stay_packed_where_their_expansion_does_not_fit():
    """Four experts of 90112 x 90112, all matrices one buffer of 17 GB, so that 16-bit copies of
    the three do not fit the GPU.  A matrix is one number s_e (a power of two) and a token one
    number c, so that g = s_e H c is a sum of H small integers, exact in f32, and the output is
    s_e I h.  The bound: h and the output rounded to bf16 (2^-8 each), 2^-17 for the activation,
    and 2^-23 for each of the 5632 additions of 16 products."""
    E, H, T = 4, 90112, 1536
    if 6 * E * H * H < torch.cuda.get_device_properties(0).total_memory:
        pytest.skip("the expansion fits this GPU")
    ex = object.__new__(cm.Int4Experts)
    ex.num_experts, ex.hidden_dim, ex.intermediate_dim = E, H, H
    ex.group_size, ex.dtype, ex.has_zeros, ex.device = 128, torch.bfloat16, False, torch.device(
        "cuda", torch.cuda.current_device())
    scale = 2.0 ** -torch.arange(6.0, 6.0 + E)
    packed = torch.empty(E, H // 16 * (H // 64), 544, dtype=torch.uint8, device="cuda")
    for e in range(E):
        q = torch.full((1, 64, 64), 0x99, dtype=torch.uint8, device="cuda")  # 9 - 8 = 1
        s = torch.full((1, 1, 64), float(scale[e]), dtype=torch.bfloat16, device="cuda")
        packed[e] = cm.Int4Weights(q, s, None, 128)._pack()[:544]
    ex.gate = ex.up = ex.down = packed
    c = 2.0 ** -12 * (1 + torch.arange(T) % 3)
    x = c[:, None].repeat(1, H).to(torch.bfloat16).cuda()
    idx = (torch.arange(T) % E).int()[:, None].cuda()
    w = torch.ones(T, 1, device="cuda")
    got = cm.fused_moe_int4(x, ex, w, idx)
    assert cm.last_gemm_path() == 5
    g = scale[torch.arange(T) % E].double() * H * c.double()
    y = scale[torch.arange(T) % E].double() * H * (g * g / (1 + torch.exp(-g)))
    tol = 2 * 2.0 ** -8 + 2.0 ** -17 + 5632 * 2.0 ** -23
    err = (got.double() - y.cuda()[:, None]).abs().amax(1).cpu()
    assert (err <= tol * y).all()
    del packed, ex, got, x
    torch.cuda.empty_cache()


# ---- calls of few rows: at most 48 rows scale f32 sums, so no weight is rounded ---------------------

FEW_ROWS = 48


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("T,E,k,H,I,G", [
    # chunks of several rows of an expert
    (9, 2, 1, 128, 64, 32), (16, 4, 2, 320, 64, 64), (33, 5, 1, 256, 256, 128),
    (24, 2, 2, 256, 128, 64), (16, 3, 3, 192, 320, 32), (48, 4, 1, 192, 128, 64),
    # K in pieces of which the last ones are empty
    (1, 1, 1, 1536, 768, 128), (1, 4, 2, 1536, 768, 128), (2, 2, 1, 768, 1536, 128),
    (3, 4, 2, 1536, 1536, 128), (1, 2, 1, 640, 896, 128), (2, 3, 2, 1600, 832, 64),
    (1, 1, 1, 1600, 832, 32)])
def test_few_rows_round_no_weight(T, E, k, H, I, G, dtype, zeros):
    assert T * k <= FEW_ROWS
    for nomic in (False, True):
        x, mats, w, idx = make(T + E + I, T, E, k, H, I, G, dtype, zeros, nomic)
        run(x, mats, w, idx, cm.Activation.Gelu if nomic else cm.Activation.Silu, rounded=False)


@pytest.mark.parametrize("T,E,k", [(4, 6, 3), (16, 6, 3), (6, 8, 8), (48, 4, 1), (1, 64, 48),
                                   (3, 64, 16)])
def test_few_rows_of_skipped_and_repeated_experts(T, E, k):
    x, mats, w, idx = make(T * k, T, E, k, 192, 128, 64, "f16", True, False, skip=0.3)
    run(x, mats, w, idx, 0, rounded=False)
    idx[:, 0] = 1
    idx[:, ::3] = E - 1
    idx[T - 1, k - 1] = -1
    run(x, mats, w, idx, 0, rounded=False)
    idx.fill_(E - 1)
    run(x, mats, w, idx, 0, rounded=False)


@pytest.mark.parametrize("T,E,k", [(49, 4, 1), (25, 30, 2), (7, 8, 7)])
def test_the_first_calls_beyond_round_each_weight_once(T, E, k):
    x, mats, w, idx = make(T * k, T, E, k, 192, 128, 64, "bf16", True, False)
    assert T * k == FEW_ROWS + 1 or T * k == 50
    run(x, mats, w, idx, 0, rounded=True)
    assert cm.last_gemm_path() == 5
    run(x[: FEW_ROWS // k].contiguous(), mats, w[: FEW_ROWS // k].contiguous(),
        idx[: FEW_ROWS // k].contiguous(), 0, rounded=False)
    assert cm.last_gemm_path() == 4
