"""Plain 64-bit implementations and error bounds for the operator tests.

Error bounds. FP32 accumulation: a sum of products whose magnitudes add up to
S is off by at most (number of roundings on a product's way) * 2^-23 * S: the
tensor core adds 16 products per step onto an accumulator that is promoted
every 2048 k, so a product passes at most min(K, 2048) / 16 + K / 2048
roundings there, a few inside its step (16 are counted) and one per part of a
split tile (32 are counted). Rounding to FP16 is off by half a step, 2^-11 of
the value (2^-25 in the subnormal range), to FP32 by 2^-24. Activations have a
slope of at most 1.13 (SiLU 1.10, GELU 1.13); their FP32 evaluation is within
2^-17 of the value (exp of up to |20| within 26 units in the last place of
2^-23, the quotient within 2, plus the argument's roundings).
"""
from __future__ import annotations

import math

import numpy as np
import torch

SLOPE = 1.13
EVAL = 2.0 ** -17


def gamma(K: int) -> float:
    return (min(K, 2048) / 16 + K / 2048 + 16 + 32) * 2.0 ** -23


def activation(x: torch.Tensor, name: str) -> torch.Tensor:
    if name == "relu":
        return x.clamp(min=0)
    if name == "silu":
        return x * torch.special.expit(x)
    if name == "gelu":
        return x * torch.special.ndtr(x)
    if name == "gelu_tanh":
        return x * 0.5 * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)))
    assert name == "none"
    return x


def weight(w: torch.Tensor, group: int) -> torch.Tensor:
    """fp16 [K, N] -> the 64-bit values its codes and scales stand for (CPU oracle)."""
    import oracle
    from parity import u16
    K, N = w.shape
    packed, scales = oracle.quantize(u16(w), K, N, group)
    deq = oracle.dequantize(packed, scales, K, N, group)
    values = np.ascontiguousarray(np.asarray(deq, dtype=np.uint16).reshape(K, N)).view(np.float16)
    return torch.from_numpy(values).to(w.device).double()


def linear(a, w64, act="none", gated=False, bias=None, residual=None, fp32_out=False):
    """(expected, tolerance) of act(a @ w + bias) + residual in 64 bits."""
    K = a.shape[1]
    x = a.double() @ w64
    d = gamma(K) * (a.double().abs() @ w64.abs())
    if bias is not None:
        x = x + bias.double()
        d = d + 2.0 ** -24 * x.abs()
    if gated:
        x, d = x.view(x.shape[0], -1, 2, 8), d.view(d.shape[0], -1, 2, 8)
        g, dg = activation(x[:, :, 0], act), SLOPE * d[:, :, 0]
        dg = dg + EVAL * g.abs()
        u, du = x[:, :, 1], d[:, :, 1]
        y = (g * u).reshape(x.shape[0], -1)
        tol = (dg * (u.abs() + du) + g.abs() * du).reshape(y.shape) + 2.0 ** -24 * y.abs()
    else:
        y = activation(x, act)
        tol = SLOPE * d + (EVAL * y.abs() if act in ("silu", "gelu", "gelu_tanh") else 0)
    if residual is not None:
        y = y + residual.double()
        tol = tol + 2.0 ** -24 * y.abs()
    step = 2.0 ** -24 if fp32_out else 2.0 ** -11
    return y, tol + step * (y.abs() + tol) + (0 if fp32_out else 2.0 ** -25)


def check(got, want, tol):
    err = (got.double() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (int(bad.sum()), float((err / tol)[bad].max()),
                           bad.nonzero()[:4].tolist())
    return float((err / tol).max()) if err.numel() else 0.0


def route(logits, top_k, scoring="softmax", bias=None, n_group=1, topk_group=1,
          group_score="max", renormalize=True, scale=1.0):
    """numpy, one token after another: (ids, weights, offsets, rows, slots)."""
    x = logits.detach().cpu().double().numpy()
    T, E = x.shape
    b = None if bias is None else bias.detach().cpu().double().numpy()
    ids = np.full((T, top_k), -1, np.int32)
    weights = np.zeros((T, top_k))
    for t in range(T):
        row = x[t]
        has = row > -np.inf
        p = np.zeros(E)
        if scoring == "sigmoid":
            with np.errstate(over="ignore"):
                p[has] = 1 / (1 + np.exp(-row[has]))
        elif has.any():
            top = row[has].max()
            with np.errstate(invalid="ignore"):
                p[has] = np.where(row[has] == top, 1.0, np.exp(row[has] - top))
            p /= p.sum()
        by_score = b is not None or (n_group > 1 and group_score == "top2")
        c = p + (0 if b is None else b) if by_score else row.copy()
        open_ = has & (c > -np.inf)
        if n_group > 1:
            size = E // n_group
            score = []
            for g in range(n_group):
                best = sorted((c[e] for e in range(g * size, (g + 1) * size) if open_[e]),
                              reverse=True)
                s = best[0] if best else -np.inf
                if group_score == "top2" and len(best) > 1:
                    s = s + best[1]
                score.append(s)
            keep = sorted(range(n_group), key=lambda g: (-score[g], g))[:topk_group]
            open_ &= np.isin(np.arange(E) // size, keep)
        order = sorted((e for e in range(E) if open_[e]), key=lambda e: (-c[e], e))[:top_k]
        ids[t, :len(order)] = order
        w = p[order]
        if renormalize:
            w = w / w.sum() if w.sum() > 0 else w * 0
        weights[t, :len(order)] = w * scale
    flat = ids.reshape(-1)
    rows = np.full(T * top_k, -1, np.int32)
    slots = np.full(T * top_k, -1, np.int32)
    offsets = np.zeros(E + 1, np.int32)
    at = 0
    for e in range(E):
        mine = np.nonzero(flat == e)[0]
        rows[at:at + mine.size] = mine
        slots[mine] = np.arange(at, at + mine.size)
        at += mine.size
        offsets[e + 1] = at
    return ids, weights, offsets, rows, slots.reshape(T, top_k)


def order(ids, E):
    """(offsets, rows, slots) of given ids [T, k] (numpy)."""
    flat = ids.reshape(-1)
    rows = np.full(flat.size, -1, np.int32)
    slots = np.full(flat.size, -1, np.int32)
    offsets = np.zeros(E + 1, np.int32)
    at = 0
    for e in range(E):
        mine = np.nonzero(flat == e)[0]
        rows[at:at + mine.size] = mine
        slots[mine] = np.arange(at, at + mine.size)
        at += mine.size
        offsets[e + 1] = at
    return offsets, rows, slots.reshape(ids.shape)
