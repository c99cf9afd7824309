"""The expert FFN on 4-bit weights where the ordinary tests do not reach (bounds: int4_testlib)."""
import numpy as np
import pytest
import torch

import candle_moe as cm
from int4_testlib import random_weights

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
