"""Plain 64-bit forms of the operators of a step of many requests, and how far
an fp32 computation of the same formulas may be from them."""
import numpy as np

U = 2.0 ** -24                                       # half a step of fp32, relative


def bf16_bits(x):
    """float32 to bfloat16 bits, to nearest even (finite values)."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def to_bits(x, dtype):
    x = np.ascontiguousarray(x, np.float32)
    return x.astype(np.float16).view(np.uint16) if dtype == "f16" else bf16_bits(x)


def from_bits(b, dtype):
    """The values 16-bit patterns stand for, in 64 bits."""
    b = np.ascontiguousarray(b, np.uint16)
    if dtype == "f16":
        return b.view(np.float16).astype(np.float64)
    return (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


HALF = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}         # half a step of the 16-bit types, relative


def rope_tables(half, n, theta=1e4):
    a = np.arange(n)[:, None] * theta ** (-np.arange(half) / half)
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


def rotate(x, c, s):
    """Halved-pair rotation of x [..., hd] in 64 bits, and the sum of the
    absolute products behind each value."""
    h = x.shape[-1] // 2
    a, b, c, s = x[..., :h].astype(np.float64), x[..., h:].astype(np.float64), c.astype(np.float64), s.astype(np.float64)
    size = np.concatenate([np.abs(a * c) + np.abs(b * s), np.abs(a * s) + np.abs(b * c)], -1)
    return np.concatenate([a * c - b * s, b * c + a * s], -1), size


def attend(q, k, v, scale):
    """Attention of the rows q [g, hd] over k, v [n, hd] in 64 bits, and a
    bound of an fp32 evaluation's error per value.

    A score is a sum of hd products of parts that hold q to 2^-21 (two 16-bit
    parts; a rounding each of the scaled product and of the sums): it is off by
    at most (hd + 16) U times the sum of the absolute products. The weights are
    then off by twice that, relatively, with a few roundings of the exponential
    and of the argument (|s| U), and 2^-21 for their own parts; numerator and
    denominator are sums in chains of at most min(n, n / 32 + 64) additions (32
    positions a matrix instruction)."""
    g, hd = q.shape
    if not len(k):
        return np.zeros((g, hd)), np.zeros((g, hd))
    q = q.astype(np.float64)
    s = q @ k.T * scale
    size = (np.abs(q) @ np.abs(k).T * abs(scale)).max(-1, keepdims=True)
    w = np.exp(s - s.max(-1, keepdims=True))
    w /= w.sum(-1, keepdims=True)
    chain = min(len(k), len(k) / 32 + 64)
    rel = 2 * (hd + 24) * U * size + (2 * chain + 32) * U
    return w @ v, rel * (w @ np.abs(v)) + 1e-37


def adjust(logits, hist, n_prompt, rep, presence, frequency, bias, mask, contract=None):
    """One row's rules in fp32, an operation at a time (hist: ids; bias: list
    of (id, value); mask: bool permitted [V] or None). Returns (row, pick)."""
    V = len(logits)
    f = np.float32
    l = logits.astype(f).copy()
    if hist is not None:
        ok = (hist >= 0) & (hist < V)
        seen = np.zeros(V, bool)
        seen[hist[ok]] = True
        made = np.zeros(V, np.int64)
        gen = np.arange(len(hist)) >= n_prompt
        np.add.at(made, hist[ok & gen], 1)
        with np.errstate(all="ignore"):
            if rep is not None:
                l = np.where(seen, np.where(l > 0, l / f(rep), l * f(rep)), l).astype(f)
            if frequency is not None:
                l = np.where(made > 0, l - f(frequency) * made.astype(f), l).astype(f)
            if presence is not None:
                l = np.where(made > 0, l - f(presence), l).astype(f)
    if bias is not None:
        for t, x in dict(bias).items():               # the last entry of an id counts
            if 0 <= t < V:
                with np.errstate(all="ignore"):
                    l[t] = l[t] + f(x)
    permitted = np.arange(V) if mask is None else np.flatnonzero(mask)
    out = np.full(V, -np.inf, f)
    out[permitted] = l[permitted]
    if not len(permitted):
        return out, -1
    best = permitted[0]
    with np.errstate(invalid="ignore"):
        if not np.isnan(l[best]):
            c = np.where(np.isnan(l[permitted]), -np.inf, l[permitted])
            top = c.max()
            if top > l[best]:
                best = permitted[np.flatnonzero(c == top)[0]]
    return out, int(best)


def lora(x, base, a, b, scale, ranks, adapter):
    """y and its fp32 error bound: chains of at most n_in + rank products, each
    rounded once, a rounding of the scale and of the two last sums."""
    y = base.astype(np.float64).copy()
    tol = np.abs(y) * U
    n_in = x.shape[1]
    for r, i in enumerate(adapter):
        if not 0 <= i < len(a):
            continue
        k = min(max(int(ranks[i]), 0), a.shape[1])
        A, B, xr = a[i, :k], b[i, :, :k], x[r].astype(np.float64)
        d = scale[i].astype(np.float64) * (B @ (A @ xr))
        size = abs(float(scale[i])) * (np.abs(B) @ (np.abs(A) @ np.abs(xr)))
        y[r] += d
        tol[r] = (n_in + k + 8) * U * size + 2 * U * np.abs(y[r]) + 1e-37
    return y, tol
