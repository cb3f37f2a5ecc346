"""What the operators around the W4A16 GEMM are timed and compared on.

Four operators of an inference step with INT4 weights:

* ``linear``   one quantised linear with its epilogue in the same pass: bias,
               activation (or an activated gate times its up column), residual
* ``route``    a router's logits -> each token's experts, their weights, and
               the order of the (token, expert) pairs by expert
* ``experts``  the products of the routed rows with their experts' weights
* ``combine``  each token's expert rows, weighted, summed, plus the residual

With ``own`` false ``run`` computes them in elementary torch operations in 32
bits (the routing's scores in 64), with ``own`` true through the package.

Weights are given as the quantiser leaves them: signed 4-bit codes, two per
byte (element k * N + n, the even one in the low nibble) and FP16 scales
[K / group][N]; the weight's value is half(code * scale). Gated weights hold
their columns in groups of 16: eight gate columns, then their eight up columns.
"""
import math

import numpy as np
import torch

own = False

ACTIVATIONS = ("none", "relu", "silu", "gelu", "gelu_tanh")
MOST_MACS = 8192 * 4096 * 28672      # of the largest listed case
MOST_WEIGHTS = 8 * 4096 * 28672


def listed():
    return [
        # one new token through the fused gate and up projection of an
        # 8B-class MLP (K = 4096, 2 x 14336 columns): latency and HBM
        _linear("linear-token-gate-up", M=1, K=4096, N=28672, group=128, activation="silu",
                gated=True),
        # a small decode batch through the down projection, added to the
        # residual stream
        _linear("linear-batch-down", M=13, K=14336, N=4096, group=64, bias=True, residual=True),
        # a short ragged prompt through a projection with bias and GELU
        _linear("linear-ragged-gelu", M=203, K=4096, N=14336, group=32, bias=True,
                activation="gelu"),
        # a long prompt through the fused gate and up projection
        _linear("linear-prompt-gate-up", M=4096, K=4096, N=28672, group=128, activation="silu",
                gated=True),
        # one token's choice of experts
        _route("route-token", T=1, E=64, k=8, logits="float32"),
        # a long batch with a few padded rows: sigmoid scores, the balancing
        # bias, eight groups of which four stay
        _route("route-prompt-groups", T=16384, E=256, k=8, logits="float32", scoring="sigmoid",
               bias=True, groups=8, keep=4, group_score="top2", scale=2.5, padded=37),
        # one token through its eight experts' gate and up projections
        _experts("experts-token-gate-up", T=1, E=64, k=8, K=2048, N=2048, group=128,
                 activation="silu", gated=True),
        # a decode batch that reaches nearly every expert, on the way down
        # (rows already in expert order)
        _experts("experts-batch-down", T=61, E=64, k=8, K=2048, N=4096, group=64, gather=False),
        # a prompt over many small experts, some tens of rows each
        _experts("experts-prompt-many", T=701, E=64, k=4, K=4096, N=2048, group=32,
                 activation="gelu_tanh", gated=True, bias=True),
        # a long prompt over eight large experts
        _experts("experts-prompt-large", T=4096, E=8, k=2, K=4096, N=28672, group=128,
                 activation="silu", gated=True),
        # the sum of one token's experts, and of a long prompt's
        _combine("combine-token", T=1, k=8, N=4096, residual=True),
        _combine("combine-prompt", T=16384, k=8, N=4096, residual=True),
    ]


def _linear(name, M, K, N, group, activation="none", gated=False, bias=False, residual=False,
            fp32_out=False):
    return {"name": name, "op": "linear", "M": M, "K": K, "N": N, "group": group,
            "activation": activation, "gated": gated, "bias": bias, "residual": residual,
            "fp32_out": fp32_out}


def _route(name, T, E, k, logits, scoring="softmax", bias=False, groups=1, keep=1,
           group_score="max", renormalize=True, scale=1.0, padded=0):
    return {"name": name, "op": "route", "T": T, "E": E, "k": k, "logits": logits,
            "scoring": scoring, "bias": bias, "groups": groups, "keep": keep,
            "group_score": group_score, "renormalize": renormalize, "scale": scale,
            "padded": padded}


def _experts(name, T, E, k, K, N, group, activation="none", gated=False, bias=False, gather=True):
    return {"name": name, "op": "experts", "T": T, "E": E, "k": k, "K": K, "N": N,
            "group": group, "activation": activation, "gated": gated, "bias": bias,
            "gather": gather}


def _combine(name, T, k, N, residual=False):
    return {"name": name, "op": "combine", "T": T, "k": k, "N": N, "residual": residual}


# ------------------------------------------------------------------ drawing

def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _log_multiple(rng, lo, hi, step):
    return step * _log_int(rng, max(1, lo // step), hi // step)


def draw(rng):
    op = rng.choice(("linear", "linear", "route", "experts", "experts", "combine"))
    if op == "linear":
        group = rng.choice((32, 64, 128))
        K = _log_multiple(rng, 256, 14336, max(64, group))
        N = _log_multiple(rng, 256, 28672, 128)
        M = _log_int(rng, 1, max(1, min(4096, MOST_MACS // (K * N))))
        gated = rng.random() < 0.4
        case = _linear("", M, K, N, group, rng.choice(ACTIVATIONS), gated, rng.random() < 0.5,
                       rng.random() < 0.4, rng.random() < 0.2)
    elif op == "route":
        groups = rng.choice((1, 1, 2, 4, 8))
        E = groups * _log_int(rng, max(2, 8 // groups), 256 // groups)
        keep = rng.randint(1, groups)
        T = _log_int(rng, 1, 16384)
        k = min(rng.randint(1, 8), keep * (E // groups))
        case = _route("", T, E, k, rng.choice(("float32", "float16")),
                      rng.choice(("softmax", "sigmoid")), rng.random() < 0.5, groups, keep,
                      rng.choice(("max", "top2")), rng.random() < 0.7, rng.choice((1.0, 2.5)),
                      rng.randint(0, T // 4))
    elif op == "experts":
        group = rng.choice((32, 64, 128))
        E = _log_int(rng, 4, 128)
        K = _log_multiple(rng, 256, 4096, max(64, group))
        N = _log_multiple(rng, 256, max(256, min(14336, MOST_WEIGHTS // (E * K))), 128)
        k = rng.randint(1, min(8, E))
        T = _log_int(rng, 1, max(1, min(4096, MOST_MACS // (k * K * N))))
        case = _experts("", T, E, k, K, N, group, rng.choice(ACTIVATIONS), rng.random() < 0.5,
                        rng.random() < 0.3, rng.random() < 0.5)
    else:
        case = _combine("", _log_int(rng, 1, 16384), rng.randint(1, 8),
                        _log_multiple(rng, 128, 4096, 8), rng.random() < 0.5)
    del case["name"]
    return case


# ------------------------------------------------------------------- inputs

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _weights(g, count, K, N, group):
    """Codes and scales of `count` weights as a quantiser of N(0, 0.02)
    values leaves them: (packed [count, K * N / 2], scales [count, K / group, N])."""
    packed = torch.empty(count, K * N // 2, dtype=torch.uint8, device="cuda")
    for e in range(count):
        q = (_normal(g, K, N // 2, 2) * 2.7).round_().clamp_(-7, 7).to(torch.int8)
        packed[e] = ((q[..., 0] & 15) | (q[..., 1] << 4)).view(torch.uint8).reshape(-1)
    spread = torch.rand(count, K // group, N, generator=g, device="cuda")
    return packed, (0.0075 * (0.8 + 0.4 * spread)).half()


def _pairs(g, T, E, k):
    """A router's choice, some experts being more popular than others: the
    tokens' experts, and the pairs in expert order (stable)."""
    logits = _normal(g, T, E) + 0.5 * _normal(g, E)
    ids = logits.topk(k, dim=1).indices.int()
    weights = torch.softmax(logits.gather(1, ids.long()), dim=1)
    return ids, weights


def _order(ids, E):
    flat = ids.reshape(-1).long()
    chosen = flat >= 0
    key = torch.where(chosen, flat, torch.full_like(flat, E))
    rows = torch.argsort(key, stable=True)
    slots = torch.empty_like(rows)
    slots[rows] = torch.arange(rows.numel(), device=rows.device)
    slots = torch.where(chosen, slots, torch.full_like(slots, -1))
    rows = torch.where(chosen[rows], rows, torch.full_like(rows, -1))
    counts = torch.bincount(flat[chosen], minlength=E)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    return offsets.int(), rows.int(), slots.reshape(ids.shape).int()


def prepare(case, seed):
    g = _generator(seed)
    s = {"case": case}
    op = case["op"]
    if op == "linear":
        M, K, N, group = case["M"], case["K"], case["N"], case["group"]
        out_n = N // 2 if case["gated"] else N
        s["a"] = _normal(g, M, K).half()
        packed, scales = _weights(g, 1, K, N, group)
        s["packed"], s["scales"] = packed[0], scales[0]
        s["bias"] = _normal(g, N).half() if case["bias"] else None
        s["residual"] = _normal(g, M, out_n).half() if case["residual"] else None
        if own:
            from sm_120__gemm_b200 import QuantizedLinear
            s["lin"] = QuantizedLinear.from_packed(s["packed"], s["scales"], K, N, group)
    elif op == "route":
        T, E = case["T"], case["E"]
        logits = (1.5 * _normal(g, T, E) + 0.5 * _normal(g, E)).to(getattr(torch, case["logits"]))
        if case["padded"]:
            rows = torch.randperm(T, generator=g, device="cuda")[:case["padded"]]
            logits[rows] = -math.inf
        s["logits"] = logits
        s["bias"] = 0.1 * _normal(g, E) if case["bias"] else None
    elif op == "experts":
        T, E, k, K, N = case["T"], case["E"], case["k"], case["K"], case["N"]
        ids, weights = _pairs(g, T, E, k)
        offsets, rows, slots = _order(ids, E)
        s["ids"], s["weights"] = ids, weights
        s["offsets"], s["rows"], s["slots"] = offsets, rows, slots
        s["a"] = _normal(g, T if case["gather"] else T * k, K).half()
        s["packed"], s["scales"] = _weights(g, E, K, N, case["group"])
        s["bias"] = _normal(g, E, N).half() if case["bias"] else None
        if own:
            from sm_120__gemm_b200 import QuantizedExperts, Routing
            s["routing"] = Routing(ids, weights, offsets, rows, slots)
            s["experts"] = QuantizedExperts.from_packed(s["packed"], s["scales"], K, N,
                                                        case["group"])
    else:
        T, k, N = case["T"], case["k"], case["N"]
        E = 4 * k
        ids, weights = _pairs(g, T, E, k)
        offsets, rows, slots = _order(ids, E)
        s["y"] = _normal(g, T * k, N).half()
        s["weights"], s["slots"] = weights, slots
        s["residual"] = _normal(g, T, N).half() if case["residual"] else None
        if own:
            from sm_120__gemm_b200 import Routing
            s["routing"] = Routing(ids, weights, offsets, rows, slots)
    return s


# ---------------------------------------------------------------- the passes

def run(state):
    case = state["case"]
    return (_RUN_OWN if own else _RUN_PLAIN)[case["op"]](state, case)


def _own_linear(s, c):
    return s["lin"](s["a"], fp32_out=c["fp32_out"], bias=s["bias"], activation=c["activation"],
                    gated=c["gated"], residual=s["residual"])


def _own_route(s, c):
    from sm_120__gemm_b200 import route
    r = route(s["logits"], c["k"], scoring=c["scoring"], bias=s["bias"], n_group=c["groups"],
              topk_group=c["keep"], group_score=c["group_score"],
              renormalize=c["renormalize"], scale=c["scale"])
    return [r.ids, r.weights, r.offsets, r.rows, r.slots]


def _own_experts(s, c):
    return s["experts"](s["a"], s["routing"], gather=c["gather"], bias=s["bias"],
                        activation=c["activation"], gated=c["gated"])


def _own_combine(s, c):
    from sm_120__gemm_b200 import combine
    return combine(s["y"], s["routing"], residual=s["residual"])


def _plain_weight(packed, scales, K, N, group):
    """half(code * scale), widened to 32 bits."""
    codes = packed.view(torch.int8).view(K, N // 2)
    low = (codes << 4) >> 4
    high = codes >> 4
    q = torch.stack((low, high), dim=2).view(K // group, group, N)
    return (q.float() * scales.float()[:, None, :]).half().float().view(K, N)


def _plain_activation(x, name):
    if name == "relu":
        return torch.maximum(x, torch.zeros_like(x))
    if name == "silu":
        return x / (1 + torch.exp(-x))
    if name == "gelu":
        return 0.5 * x * (1 + torch.erf(x * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x * x * x)))
    return x


def _plain_epilogue(y, bias, activation, gated):
    if bias is not None:
        y = y + bias.float()
    if not gated:
        return _plain_activation(y, activation)
    y = y.view(y.shape[0], -1, 2, 8)
    return (_plain_activation(y[:, :, 0], activation) * y[:, :, 1]).reshape(y.shape[0], -1)


def _plain_linear(s, c):
    w = _plain_weight(s["packed"], s["scales"], c["K"], c["N"], c["group"])
    y = _plain_epilogue(s["a"].float() @ w, s["bias"], c["activation"], c["gated"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y if c["fp32_out"] else y.half()


def _plain_route(s, c):
    x = s["logits"].double()
    T, E, k, G = c["T"], c["E"], c["k"], c["groups"]
    eligible = x > -math.inf
    if c["scoring"] == "sigmoid":
        p = 1 / (1 + torch.exp(-x))
    else:
        top = x.amax(dim=1, keepdim=True)
        top = torch.where(top > -math.inf, top, torch.zeros_like(top))
        p = torch.exp(x - top)
        p = p / p.sum(dim=1, keepdim=True).clamp_min(1e-300)
    by_score = s["bias"] is not None or (G > 1 and c["group_score"] == "top2")
    if by_score:
        choice = p if s["bias"] is None else p + s["bias"].double()
    else:  # the scores rise with the logits
        choice = x
    choice = torch.where(eligible, choice, torch.full_like(choice, -math.inf))
    if G > 1:
        members = choice.view(T, G, E // G)
        best = members.sort(dim=2, descending=True).values
        if c["group_score"] == "top2" and E // G > 1:
            second = best[:, :, 1]
            second = torch.where(second > -math.inf, second, torch.zeros_like(second))
            score = best[:, :, 0] + second
        else:
            score = best[:, :, 0]
        order = torch.sort(score, dim=1, descending=True, stable=True).indices[:, :c["keep"]]
        kept = torch.zeros(T, G, dtype=torch.bool, device=x.device).scatter_(1, order, True)
        members = torch.where(kept[:, :, None], members, torch.full_like(members, -math.inf))
        choice = members.view(T, E)
    best, ids = torch.sort(choice, dim=1, descending=True, stable=True)
    best, ids = best[:, :k], ids[:, :k]
    found = best > -math.inf
    w = torch.where(found, p.gather(1, ids), torch.zeros_like(best))
    if c["renormalize"]:
        total = w.sum(dim=1, keepdim=True)
        w = torch.where(total > 0, w / total.clamp_min(1e-300), torch.zeros_like(w))
    ids = torch.where(found, ids, torch.full_like(ids, -1)).int()
    offsets, rows, slots = _order(ids, E)
    return [ids, (w * c["scale"]).float(), offsets, rows, slots]


def _plain_experts(s, c):
    K, N, E, k = c["K"], c["N"], c["E"], c["k"]
    out = torch.empty(c["T"] * k, N // 2 if c["gated"] else N, dtype=torch.float16,
                      device=s["a"].device)
    edges = s["offsets"].tolist()
    for e in range(E):
        lo, hi = edges[e], edges[e + 1]
        if lo == hi:
            continue
        a = s["a"][s["rows"][lo:hi].long() // k] if c["gather"] else s["a"][lo:hi]
        y = a.float() @ _plain_weight(s["packed"][e], s["scales"][e], K, N, c["group"])
        bias = None if s["bias"] is None else s["bias"][e]
        out[lo:hi] = _plain_epilogue(y, bias, c["activation"], c["gated"]).half()
    return out


def _plain_combine(s, c):
    T, k, N = c["T"], c["k"], c["N"]
    out = torch.zeros(T, N, device=s["y"].device)
    for j in range(k):
        slot = s["slots"][:, j].long()
        out = out + s["weights"][:, j, None] * s["y"][slot].float()
    if s["residual"] is not None:
        out = out + s["residual"].float()
    return out.half()


_RUN_PLAIN = {"linear": _plain_linear, "route": _plain_route, "experts": _plain_experts,
              "combine": _plain_combine}
_RUN_OWN = {"linear": _own_linear, "route": _own_route, "experts": _own_experts,
            "combine": _own_combine}


# ------------------------------------------------------------- cost of a pass

def work(case):
    op = case["op"]
    if op == "linear":
        M, K, N = case["M"], case["K"], case["N"]
        out_n = N // 2 if case["gated"] else N
        b = 2 * M * K + K * N // 2 + 2 * (K // case["group"]) * N
        b += M * out_n * (4 if case["fp32_out"] else 2)
        b += 2 * N * case["bias"] + 2 * M * out_n * case["residual"]
        return {"bytes": b, "flops": 2 * M * K * N}
    if op == "route":
        T, E, k = case["T"], case["E"], case["k"]
        b = T * E * (4 if case["logits"] == "float32" else 2) + 4 * E * case["bias"]
        return {"bytes": b + 16 * T * k + 4 * (E + 1), "flops": 4 * T * E}
    if op == "experts":
        T, E, k, K, N = case["T"], case["E"], case["k"], case["K"], case["N"]
        used = E * (1 - (1 - k / E) ** T)  # experts that T even choices reach
        weights = K * N // 2 + 2 * (K // case["group"]) * N + 2 * N * case["bias"]
        b = int(used * weights) + 2 * K * (T if case["gather"] else T * k)
        b += 2 * T * k * (N // 2 if case["gated"] else N)
        return {"bytes": b, "flops": 2 * T * k * K * N}
    T, k, N = case["T"], case["k"], case["N"]
    b = 2 * T * k * N + 8 * T * k + 2 * T * N + 2 * T * N * case["residual"]
    return {"bytes": b, "flops": 2 * T * k * N}


# --------------------------------------- the definitions, in 64 bits, apart

def exact(case, seed):
    s = prepare(case, seed)
    return {"linear": _exact_linear, "route": _exact_route, "experts": _exact_experts,
            "combine": _exact_combine}[case["op"]](s, case)


def _exact_weight(packed, scales, K, N, group):
    b = packed.to(torch.int16).view(K, N // 2)
    q = torch.empty(K, N, dtype=torch.float64, device=packed.device)
    q[:, 0::2] = ((b & 15) ^ 8) - 8
    q[:, 1::2] = ((b >> 4) ^ 8) - 8
    # a code times an FP16 scale is exact in 64 bits; one rounding to FP16
    return (q * scales.double().repeat_interleave(group, dim=0)).half().double()


def _exact_rows(a, w, bias, activation, gated):
    y = torch.matmul(a.double(), w)
    if bias is not None:
        y += bias.double()
    kinds = {"none": lambda v: v, "relu": lambda v: v.clamp(min=0),
             "silu": lambda v: v * torch.special.expit(v),
             "gelu": lambda v: v * torch.special.ndtr(v),
             # 1 + tanh(u) = 2 / (1 + exp(-2 u))
             "gelu_tanh": lambda v: v * torch.special.expit(
                 math.sqrt(8 / math.pi) * (v + 0.044715 * v ** 3))}
    if not gated:
        return kinds[activation](y)
    column = torch.arange(y.shape[1] // 2, device=y.device)
    gate = 16 * (column // 8) + column % 8
    return kinds[activation](y[:, gate]) * y[:, gate + 8]


def _exact_linear(s, c):
    w = _exact_weight(s["packed"], s["scales"], c["K"], c["N"], c["group"])
    y = _exact_rows(s["a"], w, s["bias"], c["activation"], c["gated"])
    return y if s["residual"] is None else y + s["residual"].double()


def _exact_experts(s, c):
    edges = s["offsets"].cpu().numpy()
    parts = []
    for e in range(c["E"]):
        at = torch.arange(int(edges[e]), int(edges[e + 1]), device=s["a"].device)
        source = torch.div(s["rows"][at], c["k"], rounding_mode="floor") if c["gather"] else at
        w = _exact_weight(s["packed"][e], s["scales"][e], c["K"], c["N"], c["group"])
        parts.append(_exact_rows(s["a"][source], w, None if s["bias"] is None else s["bias"][e],
                                 c["activation"], c["gated"]))
    return torch.cat(parts)


def _exact_combine(s, c):
    y = s["y"].double()[s["slots"].long().reshape(-1)].view(c["T"], c["k"], c["N"])
    out = torch.einsum("tk,tkn->tn", s["weights"].double(), y)
    return out if s["residual"] is None else out + s["residual"].double()


def _exact_route(s, c):
    x = s["logits"].cpu().numpy().astype(np.float64)
    T, E, k, G = c["T"], c["E"], c["k"], c["groups"]
    open_ = x > -np.inf
    with np.errstate(over="ignore", invalid="ignore"):
        if c["scoring"] == "sigmoid":
            p = np.where(open_, 1 / (1 + np.exp(-x)), 0)
        else:
            shifted = x - np.where(open_.any(1), x.max(1), 0)[:, None]
            p = np.where(open_, np.exp(shifted), 0)
            p = p / np.maximum(p.sum(1, keepdims=True), 1e-300)
    scored = s["bias"] is not None or (G > 1 and c["group_score"] == "top2")
    pick = x.copy()
    if scored:
        pick = p + (0 if s["bias"] is None else s["bias"].cpu().numpy().astype(np.float64))
    pick[~open_] = -np.inf
    if G > 1:
        inside = np.sort(pick.reshape(T, G, E // G), axis=2)[:, :, ::-1]
        rank = inside[:, :, 0].copy()
        if c["group_score"] == "top2" and E // G > 1:
            rank += np.where(inside[:, :, 1] > -np.inf, inside[:, :, 1], 0)
        out = np.argsort(-rank, axis=1, kind="stable")[:, c["keep"]:]
        for t in range(out.shape[1]):
            pick.reshape(T, G, E // G)[np.arange(T), out[:, t]] = -np.inf
    ids = np.argsort(-pick, axis=1, kind="stable")[:, :k]
    found = np.take_along_axis(pick, ids, 1) > -np.inf
    w = np.where(found, np.take_along_axis(p, ids, 1), 0)
    if c["renormalize"]:
        total = w.sum(1, keepdims=True)
        w = np.where(total > 0, w / np.maximum(total, 1e-300), 0)
    ids = np.where(found, ids, -1).astype(np.int32)
    flat = ids.reshape(-1)
    rows = np.full(T * k, -1, np.int32)
    slots = np.full(T * k, -1, np.int32)
    offsets = np.zeros(E + 1, np.int32)
    at = 0
    for e in range(E):
        mine = np.nonzero(flat == e)[0]
        rows[at:at + mine.size] = mine
        slots[mine] = np.arange(at, at + mine.size)
        at += mine.size
        offsets[e + 1] = at
    return [ids, w * c["scale"], offsets, rows, slots.reshape(T, k)]
