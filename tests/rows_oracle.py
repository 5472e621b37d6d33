"""Plain 64-bit forms of several rows a sequence over a paged cache and of the
cache's upkeep, and how far an fp32 computation may be from them."""
import numpy as np

from serving_oracle import U


def attend(q, k, v, scale, see, cap=0.0, bias=None):
    """Rows q [g, hd] over k, v [n, hd] in 64 bits, row i over the slots that
    see [g, n] marks, and a bound of an fp32 evaluation's error per value. bias
    [g, n]: subtracted from the scores after the cap.

    A score is a sum of hd products of parts that hold q to 2^-21: off by at
    most (hd + 16) U of the sum of absolute products, as serving_oracle.attend
    derives. The cap's derivative is 1 at most, so that error passes it no
    larger; its own evaluation adds 12 U of the score (the quotient, a tanh of a
    few roundings, the product). The bias has 3 roundings (slope times distance,
    the conversion, the subtraction) of its own size and one of the score's. The
    exponential's argument and value round too: 4 U of the score and 4 U. A
    weight is off, relatively, by the sum of these errors, twice (the argument is
    multiplied by log2 e). Numerator and denominator are sums in chains of at most
    min(n, n / 4 + 64) additions; the weights' own parts hold them to 2^-21."""
    g, hd = q.shape
    q = q.astype(np.float64)
    n = len(k)
    if not n:
        return np.zeros((g, hd)), np.zeros((g, hd))
    with np.errstate(all="ignore"):
        kk, vv = np.where(np.isfinite(k), k, 0.0), np.where(np.isfinite(v), v, 0.0)
        s = q @ kk.T * scale
        size = np.abs(q) @ np.abs(kk).T * abs(scale)
        err = (hd + 16) * U * size
        if cap:
            s = cap * np.tanh(s / cap)
            err = err + 12 * U * np.abs(s)
        if bias is not None:
            s = s - bias
            err = err + 3 * U * np.abs(bias) + U * np.abs(s)
        err = 2 * (err + 4 * U * np.abs(s)) + 4 * U
        s = np.where(see, s, -np.inf)
        top = s.max(-1, keepdims=True)
        w = np.exp(s - np.where(np.isfinite(top), top, 0.0))
        # what underflows to nothing in fp32 is off by less than the largest weight's rounding
        total = w.sum(-1, keepdims=True)
        w = w / np.where(total == 0, 1.0, total)
        out = w @ vv
        err = np.where(see, err, 0.0)
        size_v = w @ np.abs(vv)
        chain = min(n, n / 4 + 64)
        tol = (w * err) @ np.abs(vv) + (w * err).sum(-1, keepdims=True) * size_v + (2 * chain + 32) * U * size_v + 1e-37
        # a row that attends to a key or value that is not finite
        bad_k = ~np.isfinite(k).all(-1)
        hit = (see & bad_k[None]).any(-1)
        bad_v = see.astype(float) @ (~np.isfinite(v)).astype(float) > 0
        out[hit] = np.nan
        out[bad_v] = np.nan
    return out, tol


def ancestors(parent):
    """Per row the rows it sees: its ancestors and itself, as whole numbers' bits."""
    bits = []
    for j, p in enumerate(parent):
        bits.append((bits[p] if p >= 0 else 0) | 1 << j)
    return bits


def words(bits, n):
    return np.array([[(int(x) >> (32 * w)) & 0xFFFFFFFF for w in range(n)] for x in bits], np.uint64).astype(np.uint32).reshape(-1, n)


def walk(tok, parent, pick, most):
    """The rows a sequence keeps of its draft."""
    path = [0] if len(tok) else []
    while path and len(path) < most:
        at = path[-1]
        nxt = [j for j in range(at + 1, len(tok)) if parent[j] == at and tok[j] == pick[at]]
        if pick[at] < 0 or not nxt:
            break
        path.append(nxt[0])
    return path
