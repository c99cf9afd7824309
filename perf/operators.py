"""Workloads of the expert routing and of the 4-bit expert FFN, for measuring them.

Three operators: the general expert routing (softmax or sigmoid scores, a balance bias, groups,
top-k, renormalised weights), its backward pass, and the fused expert FFN on 4-bit weights with
group scales.  Each has a plain form here in elementary torch operations; with `own` set, run()
makes the calls of the candle_moe module instead.
"""
import math
import os
import sys

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _library():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    pkg = os.path.join(root, "candle-moe_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import candle_moe
    return candle_moe


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------

def _route(name, T, E, k, dtype="f32", scoring="softmax", bias=False, groups=1, topk_groups=1,
           top2=False, renormalize=True, scaling=1.0, masked=False, op="route"):
    c = dict(op=op, T=T, E=E, k=k, dtype=dtype, scoring=scoring, bias=bias, groups=groups,
             topk_groups=topk_groups, top2=top2, renormalize=renormalize, scaling=scaling,
             masked=masked)
    return dict(c, name=name) if name else c


def _int4(name, T, E, k, H, I, dtype="bf16", group=128, zeros=False, nomic=False):
    c = dict(op="int4", T=T, E=E, k=k, H=H, I=I, dtype=dtype, group=group, zeros=zeros,
             nomic=nomic)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one decoded token through the router of a 128-expert layer: latency
        _route("route_one_token", 1, 128, 8),
        # a prefill batch through a router with 256 experts in 8 groups, sigmoid scores and a
        # balance bias
        _route("route_groups", 16384, 256, 8, scoring="sigmoid", bias=True, groups=8,
               topk_groups=4, top2=True, scaling=2.5),
        # an odd expert count, 16-bit logits, experts that are out of service and padded tokens
        _route("route_masked_odd", 5001, 60, 4, dtype="bf16", renormalize=False, masked=True),
        # the 65536-token batch of the 128-expert layer
        _route("route_large", 65536, 128, 8),
        # training with unnormalised softmax weights: every logit gets a gradient
        _route("backward_softmax_dense", 8191, 64, 6, dtype="bf16", renormalize=False,
               op="route_backward"),
        # training with sigmoid scores and renormalised weights
        _route("backward_sigmoid", 16384, 256, 8, scoring="sigmoid", bias=True, scaling=2.5,
               op="route_backward"),
        # training on the 65536-token batch of the 128-expert layer
        _route("backward_large", 65536, 128, 8, op="route_backward"),
        # one decoded token through the 128-expert layer: eight experts' weights are read
        _int4("int4_one_token", 1, 128, 8, 2048, 768),
        # eight decoding sequences on the 8-expert layer; weights with zero points
        _int4("int4_decode_batch", 8, 8, 2, 4096, 1536, zeros=True),
        # an odd batch, two-matrix experts with GELU, f16, small groups
        _int4("int4_nomic_odd", 77, 60, 4, 1152, 1472, dtype="f16", group=64, nomic=True),
        # a server's mixed batch: every expert is touched by a few tens of rows
        _int4("int4_mixed_batch", 512, 128, 8, 2048, 768),
        # prefill on the 128-expert layer
        _int4("int4_prefill", 16384, 128, 8, 2048, 768),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["route", "route_backward", "int4"])
    if op == "int4":
        group = rng.choice([32, 64, 128])
        step = max(group, 64)
        dtype, nomic, zeros = (rng.choice(["bf16", "f16"]), rng.random() < 0.3,
                               rng.random() < 0.5)
        H = step * _log_int(rng, 256 // step, 4096 // step)
        I = step * _log_int(rng, max(1, 128 // step), 2048 // step)
        E = min(_log_int(rng, 2, 160), 128 * 2048 * 768 // (H * I))
        k = rng.randint(1, min(E, 8))
        T = _log_int(rng, 1, max(1, min(8192, 4096 * 8 * 2048 * 768 // (k * H * I))))
        return _int4("", T, E, k, H, I, dtype, group, zeros, nomic)
    groups = rng.choice([1, 1, 2, 4, 5, 8])
    per = _log_int(rng, 3, 512 // groups)
    E = groups * per
    topk_groups = rng.randint(1, groups)
    k = rng.randint(1, min(16, topk_groups * per))
    T = _log_int(rng, 1, min(65536, 65536 * 128 // E))
    bias = rng.random() < 0.5
    return _route("", T, E, k, rng.choice(["f32", "bf16", "f16"]),
                  rng.choice(["softmax", "sigmoid"]), bias, groups, topk_groups,
                  rng.random() < 0.5, rng.random() < 0.6, rng.choice([1.0, 2.5, 0.7]),
                  rng.random() < 0.3, op)


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------

def _logits(c, g):
    """Router logits: noise over the tokens plus a preference per expert that unbalances the
    loads; with `masked`, every seventh expert out of service and every 50th token padding."""
    x = torch.randn((c["T"], c["E"]), generator=g, device="cuda") * 1.5
    x += torch.randn((c["E"],), generator=g, device="cuda") * 0.5
    if c["masked"]:
        x[:, 6::7] = float("-inf")
        x[49::50] = float("-inf")
    return x.to(_DTYPES[c["dtype"]])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    c = dict(case)
    if c["op"] == "int4":
        return _prepare_int4(c, g)
    s = dict(c, logits=_logits(c, g), bias_values=None)
    if c["bias"]:
        # a balance bias moves in steps of 0.001 per update
        b = torch.randn((c["E"],), generator=g, device="cuda") * (0.1 if c["scoring"] == "sigmoid"
                                                                  else 0.01)
        s["bias_values"] = torch.round(b * 1000) / 1000
    if c["op"] == "route_backward":
        s["weights"], s["indices"] = _plain_route(s)
        s["grad"] = torch.randn((c["T"], c["k"]), generator=g, device="cuda") * 0.1
    return s


def _prepare_int4(c, g):
    T, E, k, H, I, G, dt = (c["T"], c["E"], c["k"], c["H"], c["I"], c["group"],
                            _DTYPES[c["dtype"]])

    def weights(K, N):
        q = torch.randn((E, K, N), generator=g, device="cuda", dtype=torch.bfloat16)
        q = (q * 3).round_().clamp_(-8, 7).add_(8).to(torch.uint8)
        packed = q[:, 0::2] | (q[:, 1::2] << 4)
        scales = torch.randn((E, K // G, N), generator=g, device="cuda")
        scales = (0.02 / 3) * torch.exp(scales * 0.25)
        zeros = None
        if c["zeros"]:
            zeros = torch.randint(6, 11, (E, K // G, N), generator=g, device="cuda",
                                  dtype=torch.uint8)
        return packed, scales.to(dt), zeros

    raw = {"gate": weights(H, I), "up": None if c["nomic"] else weights(H, I),
           "down": weights(I, H)}
    x = torch.randn((T, H), generator=g, device="cuda").to(dt)
    logits = torch.randn((T, E), generator=g, device="cuda")
    logits += torch.randn((E,), generator=g, device="cuda") * 0.5
    top, idx = torch.topk(torch.softmax(logits, dim=1), k, dim=1)
    s = dict(c, x=x, weights=(top / top.sum(1, keepdim=True)).contiguous(),
             indices=idx.to(torch.int32).contiguous())
    if own:
        m = _library()
        s["experts"] = m.Int4Experts(*[None if w is None else m.Int4Weights(*w, group_size=G)
                                       for w in (raw["gate"], raw["up"], raw["down"])])
        s["moe"] = m.FusedMoE(E, k, m.Activation.Gelu if c["nomic"] else m.Activation.Silu)
    else:
        s["raw"] = raw
    return s


# ---------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------

def _scores(x, scoring):
    """Softmax or sigmoid in x's type; an expert with logit -inf scores 0."""
    if scoring == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-x))
    m = x.amax(dim=1, keepdim=True)
    p = torch.exp(x - torch.where(torch.isinf(m), torch.zeros_like(m), m))
    total = p.sum(dim=1, keepdim=True)
    return p / torch.where(total > 0, total, torch.ones_like(total))


def _first_k(keys, k):
    """The k largest of each row and their places, ties to the lower place."""
    v, at = torch.sort(keys, dim=1, descending=True, stable=True)
    return v[:, :k], at[:, :k]


def _plain_route(s):
    T, E, k, groups = s["T"], s["E"], s["k"], s["groups"]
    x = s["logits"].float()
    none = float("-inf")
    # picks compare scores that may be close: 64 bits, unless the logits themselves decide
    wide = _scores(x.double(), s["scoring"]) if s["bias"] or (s["top2"] and groups > 1) else None
    if s["bias"]:
        keys = (wide + s["bias_values"].double()).masked_fill(x == none, none)
    else:
        keys = x
    if groups > 1:
        if s["top2"]:
            sums = keys if s["bias"] else wide.masked_fill(x == none, none)
            two = _first_k(sums.view(T * groups, E // groups), 2)[0]
            value = two.masked_fill(two == none, 0.0).sum(1)
            value = value.masked_fill(two[:, 0] == none, none).view(T, groups)
        else:
            value = keys.view(T, groups, E // groups).amax(dim=2)
        v, at = _first_k(value, s["topk_groups"])
        chosen = torch.zeros((T, groups), dtype=torch.bool, device=x.device)
        chosen.scatter_(1, at, v > none)
        keys = keys.masked_fill(~chosen.repeat_interleave(E // groups, dim=1), none)
    v, at = _first_k(keys, k)
    free = v == none  # a slot no available expert is left for
    picked = _scores(x, s["scoring"]).gather(1, at).masked_fill(free, 0.0)
    if s["renormalize"]:
        total = picked.sum(dim=1, keepdim=True)
        picked = picked / torch.where(total > 0, total, torch.ones_like(total))
    return picked * s["scaling"], at.to(torch.int32).masked_fill(free, E)


def _plain_route_backward(s):
    T, E = s["T"], s["E"]
    score = _scores(s["logits"].float(), s["scoring"])
    # column E takes what the empty slots would give
    wide = torch.cat([score, torch.zeros_like(score[:, :1])], dim=1)
    at = s["indices"].long()
    r, g = wide.gather(1, at), s["grad"] * s["scaling"]
    if s["renormalize"]:
        total = r.sum(dim=1, keepdim=True)
        total = torch.where(total > 0, total, torch.ones_like(total))
        g = (g - (g * r / total).sum(dim=1, keepdim=True)) / total
    ds = torch.zeros_like(wide).scatter_add_(1, at, g)[:, :E]
    if s["scoring"] == "sigmoid":
        dx = ds * score * (1.0 - score)
    else:
        dx = score * (ds - (ds * score).sum(dim=1, keepdim=True))
    return dx.to(s["logits"].dtype)


def _dequantise(raw, used, group, dtype):
    """The used experts' weights [U, K, N] in `dtype`."""
    packed, scales, zeros = raw
    packed, scales = packed[used], scales[used].to(dtype)
    q = torch.stack([packed & 15, packed >> 4], dim=2).flatten(1, 2).to(dtype)
    U, K, N = q.shape
    z = 8.0 if zeros is None else zeros[used].to(dtype).unsqueeze(2)
    return ((q.view(U, K // group, group, N) - z) * scales.unsqueeze(2)).view(U, K, N)


def _activation(x, nomic):
    if nomic:  # GELU in its tanh form
        return 0.5 * x * (1.0 + torch.tanh(0.7978845608028654 * (x + 0.044715 * x * x * x)))
    return x / (1.0 + torch.exp(-x))


def _plain_int4(s):
    T, k, G = s["T"], s["k"], s["group"]
    used, place, counts = torch.unique(s["indices"].long().flatten(), return_inverse=True,
                                       return_counts=True)
    # the routed rows of each used expert, padded to the longest list
    order = torch.argsort(place, stable=True)
    first = torch.cumsum(counts, 0) - counts
    slot = torch.arange(T * k, device=place.device) - first[place[order]]
    rows = torch.zeros((used.numel(), int(counts.max()), s["H"]), device=place.device)
    rows[place[order], slot] = s["x"].float()[order // k]
    h = torch.bmm(rows, _dequantise(s["raw"]["gate"], used, G, torch.float32))
    h = _activation(h, s["nomic"])
    if s["raw"]["up"] is not None:
        h = h * torch.bmm(rows, _dequantise(s["raw"]["up"], used, G, torch.float32))
    y = torch.bmm(h, _dequantise(s["raw"]["down"], used, G, torch.float32))
    back = torch.empty_like(order)
    back[order] = slot
    y = y[place, back].view(T, k, s["H"]) * s["weights"].unsqueeze(2)
    return y.sum(dim=1).to(s["x"].dtype)


def run(state):
    s = state
    if own:
        m = _library()
        scoring = m.Scoring.Sigmoid if s.get("scoring") == "sigmoid" else m.Scoring.Softmax
        if s["op"] == "int4":
            return s["moe"].forward_int4(s["x"], s["experts"], s["weights"], s["indices"])
        if s["op"] == "route":
            return m.route_experts(
                s["logits"], s["k"], scoring=scoring, bias=s["bias_values"],
                num_groups=s["groups"], topk_groups=s["topk_groups"],
                group_score=m.GroupScore.Top2 if s["top2"] else m.GroupScore.Max,
                renormalize=s["renormalize"], scaling=s["scaling"])
        return m.route_experts_backward(s["grad"], s["logits"], s["weights"], s["indices"],
                                        scoring=scoring, renormalize=s["renormalize"],
                                        scaling=s["scaling"])
    if s["op"] == "int4":
        return _plain_int4(s)
    return _plain_route(s) if s["op"] == "route" else _plain_route_backward(s)


# ---------------------------------------------------------------------------------------------
# work, and the definition in 64 bits
# ---------------------------------------------------------------------------------------------

def work(case):
    c = case
    T, E, k = c["T"], c["E"], c["k"]
    if c["op"] == "int4":
        H, I = c["H"], c["I"]
        mats = 2 if c["nomic"] else 3
        # distinct experts that T tokens of k picks touch, at even loads
        touched = E * (1.0 - (1.0 - k / E) ** T)
        per = H * I / 2 + (H * I // c["group"]) * (2 + (1 if c["zeros"] else 0))
        return {"bytes": int(touched * mats * per) + T * H * 4 + T * k * 8,
                "flops": 2 * mats * T * k * H * I}
    elt = 4 if c["dtype"] == "f32" else 2
    if c["op"] == "route":
        return {"bytes": T * E * elt + T * k * 8 + (4 * E if c["bias"] else 0),
                "flops": T * E * 8}
    # a renormalised gradient needs the picks' weights alone (and their scores, with sigmoid)
    read = T * k * 12
    if c["scoring"] == "sigmoid":
        read += T * k * elt
    elif not c["renormalize"]:
        read += T * E * elt
    return {"bytes": read + T * E * elt, "flops": T * E * 4}


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "int4":
        return _exact_int4(s)
    x = s["logits"].double()
    if s["op"] == "route":
        at = _exact_picks(s, x)
        return _exact_weights(s, x, at), None
    x.requires_grad_(True)
    w = _exact_weights(s, x, s["indices"].long())
    return torch.autograd.grad(w, x, s["grad"].double())[0]


def _exact_score(s, x):
    if s["scoring"] == "sigmoid":
        return torch.sigmoid(x)
    none = torch.isinf(x).all(dim=1, keepdim=True)
    return torch.softmax(torch.where(none, torch.zeros_like(x), x), dim=1).masked_fill(none, 0.0)


def _exact_picks(s, x):
    """One pick after the other, each the first of the largest."""
    T, E, n = s["T"], s["E"], s["groups"]
    none = float("-inf")
    out = x == none
    score = _exact_score(s, x).masked_fill(out, none)
    if s["bias"]:
        keys = score + s["bias_values"].double()
    else:
        keys = x.clone()
    span = torch.arange(E, device=x.device)
    if n > 1:
        of = keys.view(T, n, E // n)
        if s["top2"]:
            of = (keys if s["bias"] else score).reshape(T, n, E // n)
            two = torch.topk(of, min(2, E // n), dim=2).values
            value = torch.where(two > none, two, torch.zeros_like(two)).sum(2)
            value = torch.where(two[..., 0] > none, value, torch.full_like(value, none))
        else:
            value = of.amax(2)
        open_ = torch.zeros((T, E), dtype=torch.bool, device=x.device)
        for _ in range(s["topk_groups"]):
            best = value.amax(1, keepdim=True)
            at = torch.where(value == best, torch.arange(n, device=x.device),
                             torch.full_like(value, n, dtype=torch.long)).amin(1, keepdim=True)
            open_ |= (span // (E // n) == at) & (best > none)
            value.scatter_(1, at, none)
        keys = torch.where(open_, keys, torch.full_like(keys, none))
    picks = []
    for _ in range(s["k"]):
        best = keys.amax(1, keepdim=True)
        at = torch.where(keys == best, span, torch.full_like(keys, E, dtype=torch.long))
        at = at.amin(1, keepdim=True)
        picks.append(torch.where(best > none, at, torch.full_like(at, E)))
        keys.scatter_(1, at, none)
    return torch.cat(picks, dim=1)


def _exact_weights(s, x, at):
    score = _exact_score(s, x)
    w = torch.cat([score, torch.zeros_like(score[:, :1])], dim=1).gather(1, at)
    if s["renormalize"]:
        total = w.sum(dim=1, keepdim=True)
        w = w / torch.where(total > 0, total, torch.ones_like(total))
    return w * s["scaling"]


def _exact_int4(s):
    raw = s.get("raw")
    if raw is None:
        return None
    T, k, G = s["T"], s["k"], s["group"]
    y = torch.zeros((T, s["H"]), dtype=torch.float64, device="cuda")
    x, w, at = s["x"].double(), s["weights"].double(), s["indices"].long()

    def matrix(name, e):
        packed, scales, zeros = (None if t is None else t[e] for t in raw[name])
        q = torch.empty((packed.shape[0] * 2, packed.shape[1]), dtype=torch.float64,
                        device="cuda")
        q[0::2], q[1::2] = (packed % 16).double(), (packed // 16).double()
        z = 8.0 if zeros is None else zeros.double().repeat_interleave(G, dim=0)
        return (q - z) * scales.double().repeat_interleave(G, dim=0)

    for e in range(s["E"]):
        t, j = torch.nonzero(at == e, as_tuple=True)
        if t.numel() == 0:
            continue
        h = x[t] @ matrix("gate", e)
        if s["nomic"]:
            h = torch.nn.functional.gelu(h, approximate="tanh")
        else:
            h = torch.nn.functional.silu(h) * (x[t] @ matrix("up", e))
        y.index_add_(0, t, (h @ matrix("down", e)) * w[t, j].unsqueeze(1))
    return y
