"""CPU restatement in 64 bits of the fp8 linear and the linears of experts (test infrastructure).

numpy float64 throughout, written from the definitions in include/cqfp8.h and include/cqexperts.h; no CUDA library
code.  Each function returns the value before its last rounding to T, and where a caller has to bound rounding
errors also the sum of magnitudes that the value was summed from.
"""
from __future__ import annotations

import numpy as np

BLOCK = 128
E4M3_MAX = 448.0


def e4m3(v):
    """The nearest e4m3 value of each |v| <= 448, halves to even; NaN stays NaN."""
    v = np.asarray(v, np.float64)
    _, e = np.frexp(np.where(np.isfinite(v), v, 0.0))
    step = np.ldexp(1.0, np.maximum(e - 4, -9))
    return np.where(np.isfinite(v), np.round(v / step) * step, np.nan)


def decode(codes):
    """e4m3 bytes -> values: 4 exponent bits of bias 7, 3 fraction bits, 0x7f and 0xff NaN."""
    c = np.asarray(codes, np.uint8).astype(np.int64)
    sign, e, m = np.where(c & 0x80, -1.0, 1.0), (c >> 3) & 15, c & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * np.ldexp(1.0, (e - 10).astype(int)))
    return np.where((c & 0x7F) == 0x7F, np.nan, sign * v)


def scale_of(block):
    """The power of two of one block of values."""
    mags = np.abs(block[np.isfinite(block)])
    top = float(mags.max()) if mags.size else 0.0
    if top == 0.0:
        return 1.0
    f, e = np.frexp(top)
    return float(np.ldexp(1.0, max(int(e) - 9 + (1 if f > 0.875 else 0), -126)))


def quantize_rows(x):
    """x [rows, k] -> (values of the codes [rows, k], scales [blocks, rows])."""
    x = np.asarray(x, np.float64)
    rows, k = x.shape
    nb = -(-k // BLOCK)
    values, scales = np.empty_like(x), np.empty((nb, rows))
    for b in range(nb):
        part = x[:, b * BLOCK:(b + 1) * BLOCK]
        s = np.array([scale_of(r) for r in part])
        scales[b] = s
        values[:, b * BLOCK:(b + 1) * BLOCK] = e4m3(part / s[:, None])
    return values, scales


def quantize_weight(w):
    """w [n, k] -> (values of the codes [n, k], scales [blocks of n, blocks of k])."""
    w = np.asarray(w, np.float64)
    n, k = w.shape
    values, scales = np.empty_like(w), np.empty((-(-n // BLOCK), -(-k // BLOCK)))
    for i in range(scales.shape[0]):
        for j in range(scales.shape[1]):
            at = np.s_[i * BLOCK:(i + 1) * BLOCK, j * BLOCK:(j + 1) * BLOCK]
            scales[i, j] = scale_of(w[at])
            values[at] = e4m3(w[at] / scales[i, j])
    return values, scales


def spread_rows(values, scales):
    return values * np.repeat(scales.T, BLOCK, axis=1)[:, :values.shape[1]]


def spread_weight(values, scales):
    n, k = values.shape
    return values * np.repeat(np.repeat(scales, BLOCK, 0)[:n], BLOCK, 1)[:, :k]


def activate(v, act):
    if act == "silu":
        with np.errstate(over="ignore"):
            return v / (1.0 + np.exp(-v))
    return np.maximum(v, 0.0) if act == "relu" else v


def linear(x, w, bias=None, act="none"):
    """(act(x w^T + b), sum of |x||w| + |b|) for x and w as the values that they stand for."""
    v, mags = x @ w.T, np.abs(x) @ np.abs(w).T
    if bias is not None:
        v, mags = v + bias, mags + np.abs(bias)
    return activate(v, act), mags


def experts(x, w, offsets, bias=None, act="none"):
    """linear() grouped by expert: w [experts, n, k], bias [experts, n]; rows of no expert are zeros."""
    y, mags = np.zeros((x.shape[0], w.shape[1])), np.zeros((x.shape[0], w.shape[1]))
    for e in range(w.shape[0]):
        at = slice(int(offsets[e]), int(offsets[e + 1]))
        y[at], mags[at] = linear(x[at], w[e], None if bias is None else bias[e], act)
    return y, mags


def route(logits, top, renormalize=True):
    """(expert, weight, offsets, token, position) by the definition of cq_route."""
    z = np.asarray(logits, np.float64)
    tokens, n = z.shape
    expert, weight = np.full((tokens, top), -1), np.zeros((tokens, top))
    for t in range(tokens):
        able = [e for e in range(n) if z[t, e] > -np.inf]
        taken = sorted(able, key=lambda e: (-z[t, e], e))[:top]
        if not taken:
            continue
        over = taken if renormalize else able
        best = z[t, taken[0]]
        share = {e: (1.0 if z[t, e] == best else 0.0) if best == np.inf else np.exp(z[t, e] - best) for e in over}
        expert[t, :len(taken)] = taken
        weight[t, :len(taken)] = [share[e] / sum(share.values()) for e in taken]
    token, position = np.full(tokens * top, -1), np.full((tokens, top), -1)
    offsets, at = [0], 0
    for e in range(n):
        for t, j in zip(*np.nonzero(expert == e)):
            token[at], position[t, j], at = t, at, at + 1
        offsets.append(at)
    return expert, weight, np.array(offsets), token, position


def combine(z, position, weight):
    """(sum_j weight z[position], the sum of magnitudes)."""
    y, mags = np.zeros((position.shape[0], z.shape[1])), np.zeros((position.shape[0], z.shape[1]))
    for j in range(position.shape[1]):
        ok = (position[:, j] >= 0) & (position[:, j] < z.shape[0])
        part = weight[ok, j, None] * z[position[ok, j]]
        y[ok] += part
        mags[ok] += np.abs(part)
    return y, mags
