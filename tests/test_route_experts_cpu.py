"""CPU tests of the general routing's argument checks, and of the oracle's gradient against
differences of the oracle's weights."""
import ctypes

import numpy as np
import pytest
import torch

import candle_moe
import route_testlib as rt


def _route(p, dtype=2, stride=8, T=4, E=8, k=2, scoring=0, n=1, kg=1, gs=0, scaling=1.0,
           logits=True, w=True):
    lib = candle_moe.lib()
    return lib.moe_route_experts(p if logits else None, dtype, stride, None, T, E, k, scoring, n,
                                 kg, gs, 0, scaling, p if w else None, p, None)


def test_refusals_without_a_gpu():
    p = ctypes.c_void_p(16)
    bad = [dict(dtype=3), dict(stride=7), dict(T=-1), dict(E=0), dict(k=0), dict(k=9),
           dict(scoring=2), dict(scoring=-1), dict(gs=2), dict(n=3), dict(n=0),
           dict(n=4, kg=0), dict(n=4, kg=5), dict(n=4, kg=1, k=3), dict(scaling=0.0),
           dict(scaling=-1.0), dict(scaling=float("nan")), dict(scaling=float("inf")),
           dict(logits=False), dict(w=False)]
    for kw in bad:
        assert _route(p, **kw) == 1, kw
    assert _route(p, E=513, stride=513) == 2
    assert _route(p, E=512, stride=512, k=33) == 2
    assert _route(p, E=66, stride=66, n=33, kg=33) == 2
    assert _route(p, T=0) == 0
    assert _route(p, T=0, logits=False) == 0


def test_backward_refusals_without_a_gpu():
    lib, p = candle_moe.lib(), ctypes.c_void_p(16)

    def call(dtype=2, stride=8, T=4, E=8, k=2, scoring=0, scaling=1.0, g=p, out=p):
        return lib.moe_route_experts_backward(g, p, dtype, stride, p, p, T, E, k, scoring, 1,
                                              scaling, out, None)
    for kw in [dict(dtype=9), dict(stride=4), dict(T=-3), dict(E=-1), dict(k=0), dict(k=9),
               dict(scoring=5), dict(scaling=0.0), dict(g=None), dict(out=None)]:
        assert call(**kw) == 1, kw
    assert call(E=600, stride=600) == 2
    assert call(E=100, stride=100, k=40) == 2
    assert call(T=0) == 0


def test_python_checks():
    x, w, i = torch.zeros(4, 8), torch.zeros(4, 2), torch.zeros(4, 2, dtype=torch.int32)
    with pytest.raises(ValueError, match="must be a cuda tensor"):
        candle_moe.route_experts(x, 2)
    with pytest.raises(ValueError, match="must be a cuda tensor"):
        candle_moe.route_experts_backward(w, x, w, i)


@pytest.mark.parametrize("scoring", [0, 1])
@pytest.mark.parametrize("renormalize", [False, True])
def test_oracle_gradient_against_differences(scoring, renormalize):
    """Central differences at step h are off by h^2/6 of a third derivative of order 1 (1e-11)
    and by rounding, 2^-53 / h of values of order 1 (1e-11 at h = 1e-5): 1e-9 leaves room."""
    rng = np.random.default_rng(5)
    T, E, k, h = 3, 7, 3, 1e-5
    l = rng.normal(size=(T, E))
    l[0, 2] = -np.inf
    g = rng.normal(size=(T, k))
    _, idx = rt.route(l, k, scoring, renormalize=renormalize, scaling=1.7)
    idx[1, 2] = E
    got = rt.backward(g, l, idx, scoring, renormalize, 1.7)

    def loss(x):
        return sum((g[t] * rt.weights(x[t], idx[t], scoring, renormalize, 1.7)).sum()
                   for t in range(T))
    for t in range(T):
        for e in range(E):
            if not np.isfinite(l[t, e]):
                assert got[t, e] == 0
                continue
            a, b = l.copy(), l.copy()
            a[t, e] += h
            b[t, e] -= h
            assert abs((loss(a) - loss(b)) / (2 * h) - got[t, e]) < 1e-9
