"""Plain 64-bit restatement of the general expert routing, one token at a time."""
import numpy as np


def scores(l, scoring):
    """l [E] float64; -inf and NaN are unavailable and score 0."""
    ok = l > -np.inf
    s = np.zeros_like(l)
    if not ok.any():
        return s
    if scoring == 1:
        with np.errstate(over="ignore"):
            s[ok] = 1.0 / (1.0 + np.exp(-l[ok]))
        return s
    p = np.exp(l[ok] - l[ok].max())
    s[ok] = p / p.sum()
    return s


def picks(l, k, scoring, bias, num_groups, topk_groups, group_score):
    E = l.size
    s = scores(l, scoring)
    ok = l > -np.inf
    total = s + (0.0 if bias is None else bias)
    ok &= total > -np.inf
    total = np.where(ok, total, -np.inf)
    key = total.copy() if bias is not None else np.where(ok, l, -np.inf)
    if num_groups > 1:
        per = E // num_groups
        value = np.full(num_groups, -np.inf)
        for g in range(num_groups):
            part = (key if group_score == 0 else total)[g * per:(g + 1) * per]
            best = np.sort(part[part > -np.inf])[::-1]
            if best.size:
                value[g] = best[0] if group_score == 0 else best[:2].sum()
        order = np.argsort(-value, kind="stable")[:topk_groups]
        keep = np.zeros(E, dtype=bool)
        for g in order:
            if value[g] > -np.inf:
                keep[g * per:(g + 1) * per] = True
        key = np.where(keep, key, -np.inf)
    order = np.argsort(-key, kind="stable")[:k]
    return np.array([e if key[e] > -np.inf else E for e in order], dtype=np.int64)


def weights(l, idx, scoring, renormalize, scaling):
    s = np.append(scores(l, scoring), 0.0)
    r = s[idx]
    if renormalize and r.sum() > 0:
        r = r / r.sum()
    return r * scaling


def route(logits, k, scoring=0, bias=None, num_groups=1, topk_groups=1, group_score=0,
          renormalize=False, scaling=1.0):
    """logits [T,E] float64 -> (weights [T,k] float64, indices [T,k])."""
    T = logits.shape[0]
    idx = np.zeros((T, k), dtype=np.int64)
    w = np.zeros((T, k))
    for t in range(T):
        idx[t] = picks(logits[t], k, scoring, bias, num_groups, topk_groups, group_score)
        w[t] = weights(logits[t], idx[t], scoring, renormalize, scaling)
    return w, idx


def backward(g, logits, idx, scoring=0, renormalize=False, scaling=1.0):
    """Gradient by the formula, in 64 bits; idx entries outside [0, E) contribute nothing."""
    T, E = logits.shape
    out = np.zeros((T, E))
    for t in range(T):
        s = scores(logits[t], scoring)
        ok = (idx[t] >= 0) & (idx[t] < E)
        at, gt = idx[t][ok], g[t][ok] * scaling
        r = s[at]
        if renormalize:
            R = r.sum()
            gt = (gt - (gt * r).sum() / R) / R if R > 0 else np.zeros_like(gt)
        ds = np.zeros(E)
        np.add.at(ds, at, gt)
        out[t] = ds * s * (1 - s) if scoring == 1 else s * (ds - (ds * s).sum())
    return out
