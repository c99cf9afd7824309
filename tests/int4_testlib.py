"""Plain 64-bit restatement of the 4-bit expert FFN, with a bound on what its kernels may differ."""
import numpy as np
import torch

import candle_moe as cm

DT = {"bf16": torch.bfloat16, "f16": torch.float16}


def unpack(q):
    """[E, K/2, N] bytes -> [E, K, N] values 0..15."""
    E, half, N = q.shape
    out = np.empty((E, 2 * half, N), dtype=np.uint8)
    out[:, 0::2], out[:, 1::2] = q & 15, q >> 4
    return out


def dequantise(w):
    """Int4Weights -> (values, (32 + q + z) * scale) [E, K, N] float64; the second bounds the
    terms that the kernels sum."""
    q = unpack(w.q.cpu().numpy()).astype(np.float64)
    s = np.repeat(w.scales.double().cpu().numpy(), w.group_size, axis=1)
    z = 8.0 if w.zeros is None else np.repeat(w.zeros.cpu().numpy().astype(np.float64),
                                              w.group_size, axis=1)
    return (q - z) * s, (32 + q + z) * np.abs(s)


def random_weights(rng, E, K, N, G, dtype, zeros):
    q = rng.integers(0, 256, size=(E, K // 2, N), dtype=np.uint8)
    s = (rng.uniform(0.5, 1.5, size=(E, K // G, N)) / (5.0 * np.sqrt(K)))
    z = rng.integers(0, 16, size=s.shape, dtype=np.uint8) if zeros else None
    return cm.Int4Weights(torch.from_numpy(q).cuda(), torch.from_numpy(s).to(DT[dtype]).cuda(),
                          None if z is None else torch.from_numpy(z).cuda(), G)


def act64(x, act):
    if act == 1:
        return 0.5 * x * (1 + np.tanh(np.sqrt(2 / np.pi) * (x + 0.044715 * x ** 3)))
    if act == 2:
        return np.maximum(x, 0)
    return x / (1 + np.exp(-x))


def reference(x, mats, w, idx, act, weights_rounded=False):
    """(y, bound) in 64 bits.  mats: (gate, up or None, down) Int4Weights.

    The bound, with u = eps / 2 of the 16-bit type.  A product sums K exact terms of at most
    (32 + q + z) s |x|; a tensor-core step of 16 terms and each later f32 addition is off by at
    most 2^-23 of what it adds up, and an output passes through fewer than 32 of them per group
    and warp: 64 * 2^-23 of the sum of the terms.  The activation's slope is below 1.13 and its
    fast exponential and division are off by less than 2^-18 relative.  h is rounded once (u), the
    output once (u).  weights_rounded: the weights and each slot's contribution are rounded to
    the 16-bit type as well (calls of many rows)."""
    u = torch.finfo(x.dtype).eps / 2
    tiny = 2.0 ** -25 if x.dtype == torch.float16 else 0.0  # half a step of f16's subnormals
    f32 = 64 * 2.0 ** -23
    X, W, ID = x.double().cpu().numpy(), w.double().cpu().numpy(), idx.cpu().numpy()
    ID = ID.astype(np.int64) & 0xffffffff
    G, GA = dequantise(mats[0])
    D, DA = dequantise(mats[2])
    if mats[1] is not None:
        U, UA = dequantise(mats[1])
    E = G.shape[0]
    y, b = np.zeros(X.shape), np.zeros(X.shape)
    for e in range(E):
        t, j = np.nonzero(ID == e)
        if t.size == 0:
            continue
        xa = np.abs(X[t])
        g = X[t] @ G[e]
        eg = f32 * (xa @ GA[e]) + (u * (xa @ np.abs(G[e])) if weights_rounded else 0)
        h = act64(g, act)
        eh = 1.13 * eg + 2.0 ** -18 * np.abs(h)
        if mats[1] is not None:
            up = X[t] @ U[e]
            eu = f32 * (xa @ UA[e]) + (u * (xa @ np.abs(U[e])) if weights_rounded else 0)
            eh = eh * (np.abs(up) + eu) + np.abs(h) * eu
            h = h * up
        eh = eh * (1 + u) + u * np.abs(h) + tiny
        c = h @ D[e]
        ec = eh @ np.abs(D[e]) + f32 * ((np.abs(h) + eh) @ DA[e])
        if weights_rounded:
            ec = ec + u * ((np.abs(h) + eh) @ np.abs(D[e])) + tiny * (np.abs(h).sum(1)[:, None] + 1)
        s = W[t, j][:, None]
        if weights_rounded:
            ec = ec * (1 + u) + u * np.abs(c) + tiny
        np.add.at(y, t, s * c)
        np.add.at(b, t, np.abs(s) * ec)
    b = b * (1 + u) + u * np.abs(y) + 2.0 ** -20 * np.abs(y) + tiny
    return y, b


def routing(rng, T, E, k, skip=0.0):
    idx = np.stack([rng.permutation(E)[:k] for _ in range(T)]).astype(np.int32) if T else \
        np.zeros((0, k), np.int32)
    w = rng.uniform(0.05, 1.0, size=(T, k)).astype(np.float32)
    if skip:
        idx[rng.uniform(size=idx.shape) < skip] = E
    return torch.from_numpy(w).cuda(), torch.from_numpy(idx).cuda()


def check(got, y, bound):
    got = got.double().cpu().numpy()
    err = np.abs(got - y)
    assert np.isfinite(got).all()
    assert (err <= bound).all(), (err - bound).max()
    # at most six roundings of rms u/sqrt(3) each act on the result: below 2 u in the 2-norm
    return np.linalg.norm(err) / max(np.linalg.norm(y), 1e-30)
