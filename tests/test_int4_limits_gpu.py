"""The expert FFN on 4-bit weights where the ordinary tests do not reach (bounds: int4_testlib)."""
import numpy as np
import pytest
import torch

import candle_moe as cm
from int4_testlib import random_weights
from test_int4_gpu import make

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
