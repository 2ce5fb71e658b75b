"""Plain float64 / integer implementations of the layers with 8-bit weights, the routing and the weighted sum, and how far the
kernels' results may be off."""
import math

import numpy as np

HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 2.0 ** -150, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}   # half a step among the subnormal numbers
U = 2.0 ** -24


def to_store(a, dtype):
    """float64 values in the storage type (bf16 as its bits), rounded to nearest even."""
    a32 = np.asarray(a, np.float32)
    if dtype == "f32":
        return a32
    if dtype == "f16":
        return a32.astype(np.float16)
    b = a32.view(np.uint32)
    out = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(a32), np.uint16(0x7FC0), out)


def to_float(a, dtype):
    if dtype == "bf16":
        return (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return a.astype(np.float64)


def quantize(x):
    """x (T, K) float64: whole numbers nearest to 127 x / max, exactly (Python's integers), and the scales."""
    T, K = x.shape
    q = np.zeros((T, K), np.int8)
    scale = np.zeros(T)
    for t in range(T):
        row = x[t]
        if not np.isfinite(row).all():
            scale[t] = np.nan
            continue
        top = np.abs(row).max() if K else 0.0
        scale[t] = top / 127.0
        if top == 0:
            continue
        n_top, d_top = float(top).as_integer_ratio()
        for j in range(K):
            n, d = abs(float(row[j])).as_integer_ratio()
            a, b = 127 * n * d_top, d * n_top       # the quotient a / b
            w, rest = divmod(a, b)
            w += (2 * rest > b) or (2 * rest == b and w % 2 == 1)
            q[t, j] = w if row[j] >= 0 else -w
    return q, scale


def act(name, x):
    with np.errstate(over="ignore", invalid="ignore"):
        if name == "relu":
            return np.where(x < 0, 0.0, x)
        if name == "silu":
            return x / (1.0 + np.exp(-x))
        if name == "gelu_tanh":
            return x / (1.0 + np.exp(-2.0 * math.sqrt(2.0 / math.pi) * (x + 0.044715 * x ** 3)))
        if name == "gelu_erf":
            return 0.5 * x * np.vectorize(math.erfc, otypes=[float])(-x * math.sqrt(0.5))
        return x


def act_error(name, x, dx):
    """How far the kernel's act(x) may be from act(x), with x off by dx: the steepest slope of any of them is below 1.13; the
    exponent e of exp2 is off by its own two roundings, |e| 2^-23, which moves exp(-e') by as much of itself; exp2, the sum, the
    quotient and the products by at most 1 ulp each."""
    y = np.abs(act(name, x))
    if name in ("none", "relu"):
        return dx
    e = np.abs(x) if name == "silu" else 1.6 * np.abs(x + 0.044715 * x ** 3)
    if name == "gelu_erf":   # erfc is within 16 ulp; its argument's rounding moves it by 2 z^2 of itself, z = x / sqrt 2
        return 1.13 * dx + y * (40 + 2 * x * x) * U
    return 1.13 * dx + y * (4 * e + 16) * U


def layer(x, xs, w, ws, bias, name, gated, dtype):
    """x (T, K) int8, xs (T), w (N, K) int8, ws, bias (N): the result in float64, and the error allowed."""
    sums = x.astype(np.int64) @ w.astype(np.int64).T
    prod = sums * (xs.astype(np.float64)[:, None] * ws.astype(np.float64)[None, :])
    y = prod + (bias.astype(np.float64)[None, :] if bias is not None else 0.0)
    # the sum to 32 bits, the first product, and the last fused step: three roundings
    dy = (2.01 * np.abs(prod) + 1.01 * np.abs(y)) * U + 2 * TINY["f32"]
    if gated:
        half = w.shape[0] // 2
        g, dg = act(name, y[:, :half]), act_error(name, y[:, :half], dy[:, :half])
        u, du = y[:, half:], dy[:, half:]
        out = g * u
        err = np.abs(g) * du + np.abs(u) * dg + dg * du + np.abs(out) * U
    else:
        out, err = act(name, y), act_error(name, y, dy)
    return out, err + (np.abs(out) + err) * HALF_STEP[dtype] + TINY[dtype]


def route(x, top_k, score, bias=None, groups=1, top_groups=1, group_best=1, renormalize=True, scale=1.0):
    """x (T, E) float64: ids and weights (T, top_k), token by token."""
    T, E = x.shape
    ids = np.full((T, top_k), -1, np.int32)
    weights = np.zeros((T, top_k))
    for t in range(T):
        row = x[t]
        b = bias.astype(np.float64) if bias is not None else np.zeros(E)
        if np.isnan(row).any() or (row == np.inf).any() or np.isnan(b).any() or (b == np.inf).any():
            weights[t] = np.nan
            continue
        masked = np.isneginf(row) | np.isneginf(b)
        if score == "softmax":
            top = row.max()
            e = np.exp(row - (top if np.isfinite(top) else 0.0))
            p = e / e.sum() if e.sum() > 0 else e
        else:
            with np.errstate(over="ignore"):
                p = 1.0 / (1.0 + np.exp(-row))
        c = [(-math.inf if masked[e] else p[e] + b[e]) for e in range(E)]
        # where p itself orders as the logits do they tell it apart for longer than 64 bits of p would
        key = (lambda e: (-c[e], e)) if bias is not None else (lambda e: (-row[e], e))
        open_ = set(range(E))
        if top_groups < groups:
            size = E // groups
            counts = []
            for g in range(groups):
                inside = sorted(range(g * size, (g + 1) * size), key=key)[:group_best]
                if group_best == 1 and bias is None:
                    counts.append(row[inside[0]])
                else:
                    counts.append(sum(c[e] for e in inside))
            best = sorted(range(groups), key=lambda g: (-counts[g], g))[:top_groups]
            open_ = {e for g in best for e in range(g * size, (g + 1) * size)}
        left = sorted((e for e in open_ if not masked[e]), key=key)[:top_k]
        ids[t, :len(left)] = left
        if score == "softmax" and renormalize:
            w = np.exp(row[left] - row[left].max()) if left else np.zeros(0)
        elif renormalize:   # relative to the highest logit below 0: exp(-m) p
            m = min(0.0, row[left].max()) if left else 0.0
            with np.errstate(over="ignore"):
                w = 1.0 / (np.exp(m) + np.exp(m - row[left]))
        else:
            w = p[left]
        weights[t, :len(left)] = scale * (w / w.sum() if renormalize and left else w)
    return ids, weights


def plan(ids, experts):
    """offsets (experts + 1) and order of ids (T, top_k)."""
    flat = ids.reshape(-1)
    order = np.full(flat.size, -1, np.int32)
    offsets = np.zeros(experts + 1, np.int32)
    at = 0
    for e in range(experts):
        mine = np.flatnonzero(flat == e)
        order[at:at + mine.size] = mine
        at += mine.size
        offsets[e + 1] = at
    return offsets, order


def combine(y, weights, ids, base, dtype):
    """y (T, k, N), weights (T, k): the sum, and the error allowed: k fused steps of 32 bits, one rounding at the end."""
    T, k, N = y.shape
    out = np.zeros((T, N)) if base is None else base.astype(np.float64).copy()
    size = np.abs(out)
    for j in range(k):
        dead = (ids[:, j] < 0) if ids is not None else np.zeros(T, bool)
        term = np.where(dead[:, None], weights[:, j, None] * 0.0, weights[:, j, None] * np.where(dead[:, None], 0.0, y[:, j]))
        out = out + term
        size = size + np.abs(term)
    err = size * (k + 1) * U
    return out, err + (np.abs(out) + err) * HALF_STEP[dtype] + TINY[dtype]
