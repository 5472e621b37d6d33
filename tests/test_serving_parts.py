"""The 16-bit parts that fp32 values meet the matrix cores in: inputs whose
high parts cancel, so that the lowest part alone decides the result. Random
inputs leave a part's loss far inside the worst case that their bounds allow."""
import numpy as np
import pytest

import serving_oracle as so
import sheep_amd as sa
from sheep_amd import serving

PARTS = {"f16": 2, "bf16": 3}
# a - b is what the last part of a holds, b has one part fewer
A = {"f16": 1 + 2.0 ** -13, "bf16": 1 + 2.0 ** -9 + 2.0 ** -18}
B = {"f16": 1.0, "bf16": 1 + 2.0 ** -9}
SHAPES = [("f16", 128), ("f16", 64), ("bf16", 128), ("bf16", 64)]
LN2 = np.float32(np.log(2.0))                        # times log2(e) in fp32 this is 1: weights are powers of two


def cut(x, dtype, n):
    """x as the sum of its first n parts, each the rounding of what is left,
    after a power of two that takes the largest below 2^11."""
    x = np.asarray(x, np.float64)
    top = 2.0 ** (np.frexp(np.abs(x).max())[1] - 11)
    left, out = x / top, np.zeros_like(x)
    for _ in range(n):
        h = so.from_bits(so.to_bits(left, dtype), dtype)
        out, left = out + h, left - h
    return out * top


# ------------------------------------------------------------ the query's parts

def query_case(dtype, hd, heads):
    """Every head's scores are the last part of one of its values: q is a at
    one dim and -b at another, a position's key the same c everywhere. The
    products and their sums are exact in fp32 (c has 4 bits)."""
    n = 70
    q = np.zeros((heads, hd), np.float32)
    for h in range(heads):
        size = 2.0 ** (h % 5 - 2)
        q[h, (37 * h) % hd], q[h, (37 * h + 5 + 11 * h) % hd] = A[dtype] * size, -B[dtype] * size
    c = (np.arange(n) * 7 % 13) / 4 / (A[dtype] - B[dtype])
    k = so.to_bits(np.repeat(c[:, None], hd, 1), dtype)
    v = so.to_bits(np.random.default_rng(hd).integers(-64, 65, (n, hd)) / 64, dtype)
    return q, k, v


def query_want(q, k, v, dtype):
    """In 64 bits; and how far fp32 is off, with exact scores: a weight by a
    step of 2^x (2 U) and 4 U of its parts, the sums by a rounding each (2
    tiles a wave, 4 waves, 3 parts), the quotient by U."""
    k, v = so.from_bits(k, dtype), so.from_bits(v, dtype)
    w = np.exp2(q.astype(np.float64) @ k.T)
    w /= w.sum(-1, keepdims=True)
    return w @ v, 40 * so.U * (w @ np.abs(v))


# ------------------------------------------------------------ the weights' parts

def weight_case(dtype, hd, heads):
    """Half of 32 positions have the weight 1 and the value 1, half a weight
    2^-d and the value -1: the output (1 - 2^-d) / (1 + 2^-d) is what the
    parts behind the first hold. d is the 8-bit number whose weight has the
    largest last part."""
    best = None
    for m in range(128, 256):
        for e in (-14, -15):
            d = m * 2.0 ** e
            w = np.float64(np.float32(2.0 ** -d))
            lost = abs(w - one_cut(w, dtype, PARTS[dtype] - 1))
            if best is None or lost > best[0]:
                best = (lost, d)
    d = best[1]
    rng = np.random.default_rng(hd + heads)
    low = rng.permutation(32) < 16
    q, k = np.zeros((heads, hd), np.float32), np.zeros((32, hd))
    q[np.arange(heads), np.arange(heads) % 3] = 1.0
    k[low, :3] = -d
    v = np.where(low, -1.0, 1.0)[:, None] * np.ones(hd)
    return q, so.to_bits(k, dtype), so.to_bits(v, dtype), 2.0 ** -d


def one_cut(w, dtype, n):
    left, out = w, 0.0
    for _ in range(n):
        h = float(so.from_bits(so.to_bits(np.array([left * 2.0 ** 8]), dtype), dtype)[0]) * 2.0 ** -8
        out, left = out + h, left - h
    return out


# a weight's 2 U, on both sides of a difference of equal shares; roundings of
# sums of which the outputs are differences, 3 parts
WEIGHT_TOL = 8 * so.U


# ------------------------------------------------------------ adapters

LORA = [(1, 64, 40, 16, 1), (8, 520, 300, 64, 8), (20, 256, 70, 16, 3), (40, 264, 33, 256, 2), (100, 520, 130, 24, 7),
        (130, 1032, 65, 64, 2), (300, 264, 130, 64, 4), (290, 512, 70, 256, 2), (600, 520, 70, 128, 5)]


def lora_case(n, n_in, n_out, rank, n_ad, dtype):
    """Pairs of ranks take a and -b from x, an output adds a pair: y is the
    last part, in whole numbers times a - b, and every step exact in fp32."""
    rng = np.random.default_rng(n + rank)
    pairs = rank // 2
    where = np.array([rng.permutation(n_in)[:rank] for _ in range(n_ad)])          # the input of a rank
    a = np.zeros((n_ad, rank, n_in), np.float32)
    b = np.zeros((n_ad, n_out, rank), np.float32)
    which = np.array([rng.permutation(np.arange(n_out) % pairs) for _ in range(n_ad)])     # the pair of an output
    ids = rng.integers(0, n_ad, n)
    x, y = np.zeros((n, n_in), np.float32), np.zeros((n, n_out))
    for i in range(n_ad):
        a[i, np.arange(rank), where[i]] = 1.0
        b[i, np.arange(n_out), 2 * which[i]] = 1.0
        b[i, np.arange(n_out), 2 * which[i] + 1] = 1.0
    for r in range(n):
        i = ids[r]
        s = rng.integers(1, 8, pairs) * rng.choice([-1, 1], pairs)
        x[r, where[i, 0::2]], x[r, where[i, 1::2]] = s * A[dtype], -s * B[dtype]
        y[r] = s[which[i]] * (A[dtype] - B[dtype])
    return x, a, b, ids, y


# ------------------------------------------------------------ a lost part shows

@pytest.mark.parametrize("dtype, hd", SHAPES)
def test_a_lost_part_of_the_query_shows(dtype, hd):
    q, k, v = query_case(dtype, hd, 16)
    want, tol = query_want(q, k, v, dtype)
    for n in (PARTS[dtype], PARTS[dtype] - 1):
        got = query_want(np.array([cut(row, dtype, n) for row in q]), k, v, dtype)[0]
        off = np.abs(got - want) > tol
        assert not off.any() if n == PARTS[dtype] else off.mean() > 0.8


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_a_lost_part_of_the_weights_shows(dtype):
    *_, w = weight_case(dtype, 64, 8)
    w32 = float(np.float32(w))
    for n in (PARTS[dtype], PARTS[dtype] - 1):
        off = abs((1 - one_cut(w32, dtype, n)) / (1 + w) - (1 - w) / (1 + w))
        assert off < 2 * so.U if n == PARTS[dtype] else off > 2 * WEIGHT_TOL


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_a_lost_part_of_the_adapters_shows(dtype):
    x, a, b, ids, y = lora_case(8, 72, 20, 16, 2, dtype)
    P = PARTS[dtype]
    for px, pt in ((P, P), (P - 1, P), (P, P - 1)):
        got = np.empty_like(y)
        for r in range(len(x)):
            t = a[ids[r]].astype(np.float64) @ cut(x[r], dtype, px)
            got[r] = b[ids[r]].astype(np.float64) @ cut(t, dtype, pt)
        assert (got == y).all() if px == pt else (got != y).mean() > 0.4


# ------------------------------------------------------------ the kernels

def attend(q, k, v, dtype):
    """One sequence over the first rows of pages of 16."""
    heads, hd = q.shape
    pages = -(-len(k) // 16)
    pools = [sa.DevBuf.of(np.concatenate([x, np.zeros((16 * pages - len(x), hd), np.uint16)])) for x in (k, v)]
    pg = serving.Pages(*pools, sa.DevBuf.of(np.arange(pages, dtype=np.int32)), pages, 16, 1, pages, 1, hd, dtype)
    out, part = sa.DevBuf(4 * heads * hd), sa.DevBuf(4 * serving.part_floats(1, heads, hd, len(k)))
    serving.attention(pg, sa.DevBuf.of(q), sa.DevBuf.of(np.array([len(k)], np.int32)), len(k), heads, part, out,
                      scale=float(LN2))
    return out.read(np.float32).reshape(heads, hd)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, hd", SHAPES)
def test_attention_holds_the_query_whole(dtype, hd):
    sa.init(0)
    assert np.float32(LN2 * np.float32(1.44269504088896341)) == 1
    q, k, v = query_case(dtype, hd, 16)
    want, tol = query_want(q, k, v, dtype)
    off = np.abs(attend(q, k, v, dtype) - want)
    assert (off <= tol).all(), (off / tol).max()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, hd", SHAPES)
def test_attention_holds_the_weights_whole(dtype, hd):
    sa.init(0)
    q, k, v, w = weight_case(dtype, hd, 8)
    off = np.abs(attend(q, k, v, dtype) - (1 - w) / (1 + w))
    assert (off <= WEIGHT_TOL).all(), off.max() / so.U


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("n, n_in, n_out, rank, n_ad", LORA)
def test_adapters_hold_fp32_whole(n, n_in, n_out, rank, n_ad, dtype):
    sa.init(0)
    x, a, b, ids, y = lora_case(n, n_in, n_out, rank, n_ad, dtype)
    yb, work = sa.DevBuf(4 * n * n_out), sa.DevBuf(4 * serving.lora_work_floats(rank, n))
    ad = serving.Adapters(sa.DevBuf.of(so.to_bits(a, dtype)), sa.DevBuf.of(so.to_bits(b, dtype)), n_ad, rank, n_in, n_out, dtype)
    serving.lora(ad, sa.DevBuf.of(x), n, sa.DevBuf.of(ids.astype(np.int32)), yb, work)
    np.testing.assert_array_equal(yb.read(np.float32).reshape(n, n_out), y.astype(np.float32))
