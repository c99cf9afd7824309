"""CPU tests of the 4-bit entry points' argument checks."""
import ctypes

import pytest
import torch

import candle_moe as cm


def test_sizes():
    lib = cm.lib()
    # nibbles, scales and zero points of each 16 columns x 64 k
    for G, per in ((32, 2), (64, 1), (128, 1)):
        assert lib.moe_int4_packed_size(2, 128, 64, G, 1, 0) == 2 * 4 * 2 * (512 + 32 * per)
        assert lib.moe_int4_packed_size(2, 128, 64, G, 1, 1) == 2 * 4 * 2 * (512 + 48 * per)
    for bad in [(0, 128, 64, 64, 1, 0), (2, 96, 64, 32, 1, 0), (2, 128, 72, 64, 1, 0),
                (2, 128, 64, 48, 1, 0), (2, 64, 64, 128, 1, 0), (2, 128, 64, 64, 2, 0),
                (2, 128, 64, 64, 5, 0), (2, 1 << 21, 64, 64, 1, 0), (2, 64, 1 << 21, 64, 1, 0)]:
        assert lib.moe_int4_packed_size(*bad) == 0, bad
    n = cm.int4_workspace_size(64, 256, 128, 8, 2)
    assert n >= 128 * (128 * 2 + 256 * 2) and n % 256 == 0
    assert cm.int4_workspace_size(0, 256, 128, 8, 2) == 0
    assert cm.int4_workspace_size(2 ** 31, 256, 128, 8, 2) == 0


def test_fused_refusals_without_a_gpu():
    lib, p, q = cm.lib(), ctypes.c_void_p(256), ctypes.c_void_p(1 << 40)

    def call(x=p, gate=p, down=p, T=4, H=256, I=128, E=8, k=2, dtype=1, G=64, out=q):
        return lib.moe_fused_int4(x, gate, p, down, p, p, out, T, H, I, E, k, 0, dtype, G, 0, None, 0,
                                  None)
    for kw in [dict(T=-1), dict(k=0), dict(H=0), dict(I=-64), dict(E=0), dict(dtype=4),
               dict(G=16), dict(G=0), dict(I=192, G=128), dict(x=None), dict(gate=None),
               dict(down=None), dict(out=None), dict(out=p), dict(out=ctypes.c_void_p(256 + 2032))]:
        assert call(**kw) == 1, kw
    for kw in [dict(dtype=2), dict(H=96, G=32), dict(I=32, G=32), dict(E=4096), dict(T=2 ** 31),
               dict(x=ctypes.c_void_p(264)), dict(gate=ctypes.c_void_p(264)),
               dict(out=ctypes.c_void_p((1 << 40) + 8))]:
        assert call(**kw) == 2, kw
    assert call(T=0) == 0


def test_quantize_and_pack_refusals_without_a_gpu():
    lib, p = cm.lib(), ctypes.c_void_p(256)
    assert lib.moe_int4_quantize(p, 2, 128, 64, 48, 1, p, p, p, None) == 1
    assert lib.moe_int4_quantize(p, 2, 128, 64, 64, 2, p, p, p, None) == 2
    assert lib.moe_int4_quantize(None, 2, 128, 64, 64, 1, p, p, p, None) == 1
    assert lib.moe_int4_quantize(p, 2, 128, 64, 64, 1, p, None, p, None) == 1
    assert lib.moe_int4_pack(p, p, None, 2, 100, 64, 64, 1, p, None) == 1
    assert lib.moe_int4_pack(None, p, None, 2, 128, 64, 64, 1, p, None) == 1
    assert lib.moe_int4_pack(p, p, None, 2, 128, 64, 64, 1, ctypes.c_void_p(272), None) == 1


def test_python_checks():
    q = torch.zeros(2, 64, 64, dtype=torch.uint8)
    s = torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="must be a cuda tensor"):
        cm.Int4Weights(q, s, group_size=64)
    with pytest.raises(ValueError, match="group_size"):
        cm.Int4Weights(q, s, group_size=16)
    with pytest.raises(ValueError, match="multiples of 64"):
        cm.Int4Weights(q[:, :, :40].contiguous(), s, group_size=64)
    with pytest.raises(ValueError, match="scales must be"):
        cm.Int4Weights(q, s, group_size=128)
    with pytest.raises(TypeError, match="scales"):
        cm.Int4Weights(q, s.float(), group_size=64)
    with pytest.raises(TypeError, match="uint8"):
        cm.Int4Weights(q.int(), s, group_size=64)
    with pytest.raises(ValueError, match="zeros"):
        cm.Int4Weights(q, s, s, group_size=64)
    with pytest.raises(ValueError, match="must be a cuda tensor"):
        cm.quantize_int4(torch.zeros(2, 128, 64, dtype=torch.bfloat16), 64)
