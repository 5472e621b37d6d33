"""Several rows a sequence and a cache's upkeep at the edges of what their header
allows: parts, far pages, largest counts, streams and graphs, buffers' ends, and a
run of them together."""
import os
import subprocess
import sys

import numpy as np
import pytest

import rows_oracle as ro
import serving_oracle as so
import sheep_amd as sa
from sheep_amd import serving
from test_gpu_rows import by_layer, ints, make_table, rows_case, tree_of, within
from test_gpu_serving import Guarded, Hip

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    sa.init(0)


def attend(q, k, v, dtype, start, lens, heads, scale=0.0, max_len=None, page=16, **rows):
    """One call over sequences whose pages lie one after another: k, v [n_seq][n][kv][hd] bits."""
    n_seq, n, kv, hd = k.shape
    pages = -(-n // page)
    pad = np.zeros((n_seq, pages * page - n, kv, hd), np.uint16)
    pools = [sa.DevBuf.of(np.concatenate([x, pad], 1)) for x in (k, v)]
    pg = serving.Pages(*pools, ints(np.arange(n_seq * pages).reshape(n_seq, pages)), n_seq * pages, page, n_seq, pages, kv, hd, dtype)
    n_row, top = len(q), n if max_len is None else max_len
    out, part = sa.DevBuf.of(np.full((n_row, heads * hd), 7.5, np.float32)), sa.DevBuf(4 * serving.rows_floats(n_seq, n_row, kv, heads, hd, top))
    serving.attention_rows(pg, serving.Rows(ints(start), ints(lens), n_row, top, **rows), sa.DevBuf.of(q.astype(np.float32)), heads,
                           part, out, scale=scale)
    return out.read(np.float32).reshape(n_row, heads, hd)


# ------------------------------------------------------------ parts

@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("dtype, low", [("f16", 2.0 ** -18), ("bf16", 2.0 ** -20)])
def test_the_lowest_part_of_a_query_decides(hd, dtype, low):
    """Two keys whose products with the query's higher parts cancel: the scores
    differ by its lowest part alone, 64 times as large by the scale. q is 1 + low in
    dim 0 and 1 in dim 1, the keys are (1, -1) and (-1, 1): scores +-low * scale. The
    weights' difference is tanh(low * scale), of which fp32 parts of q of 21 bits
    keep all but 2^-21 / low relatively."""
    scale = 2.0 ** 16
    q = np.zeros((3, hd))
    q[:, 0], q[:, 1] = 1 + low, 1
    k, v = np.zeros((1, 2, 1, hd)), np.zeros((1, 2, 1, hd))
    k[0, 0, 0, :2], k[0, 1, 0, :2] = (1, -1), (-1, 1)
    v[0, 0], v[0, 1] = 1, -1
    got = attend(q, so.to_bits(k, dtype), so.to_bits(v, dtype), dtype, [0, 3], [2], 1, scale=scale, first=ints([0] * 3), last=ints([2] * 3))
    want = np.tanh(low * scale)
    assert (np.abs(got - want) <= want * (2.0 ** -21 / low + 2.0 ** -18)).all(), (got[0, 0, 0], want)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_the_lowest_part_of_a_weight_decides(hd, dtype):
    """Weights w and 1 over values 1 and -1 leave their difference, which the
    higher parts do not hold: scores are d and 0, the output is tanh(d / 2), for d
    of about 2^-12 to 2^-9. The weights' parts hold them to 2^-21 (fp16's two of 11
    bits) and the exponential to 4 U: the difference of the two is off by 2^-20 of
    the larger at most."""
    for d in (2.0 ** -9 * 1.37, 2.0 ** -11 * 1.81, 2.0 ** -12 * 1.13):
        q = np.zeros((40, hd))
        q[:, 0] = d
        k, v = np.zeros((1, 50, 1, hd)), np.zeros((1, 50, 1, hd))
        k[0, 0::2, 0, 0] = 1
        v[0, 0::2], v[0, 1::2] = 1, -1
        got = attend(q, so.to_bits(k, dtype), so.to_bits(v, dtype), dtype, [0, 40], [50], 1, scale=1.0, first=ints([0] * 40), last=ints([50] * 40))
        want = np.tanh(float(np.float32(d)) / 2)
        assert (np.abs(got - want) <= 2.0 ** -20).all(), (got[0, 0, 0], want)


def test_norms_of_the_errors():
    """Random rows: the errors' norm is that of fp32's roundings, 2^-19 of the
    outputs' (roundings of scores up to some 2^3 at 2^-24, twice, and of the sums; a
    lost 16-bit part would be 2^-12 or more)."""
    rng = np.random.default_rng(5)
    for dtype, hd, n, m in (("f16", 128, 700, 90), ("bf16", 128, 700, 90), ("f16", 64, 3000, 9), ("bf16", 64, 300, 200)):
        q = rng.standard_normal((m, 4, hd))
        k, v = (so.to_bits(rng.standard_normal((1, n, 2, hd)), dtype) for _ in range(2))
        got = attend(q.reshape(m, -1), k, v, dtype, [0, m], [n], 4)
        see = np.arange(n)[None] <= n - m + np.arange(m)[:, None]
        for h in range(4):
            want, _ = ro.attend(q[:, h].astype(np.float32), so.from_bits(k[0, :, h // 2], dtype), so.from_bits(v[0, :, h // 2], dtype), hd ** -0.5, see)
            assert np.linalg.norm(got[:, h] - want) <= 2.0 ** -19 * np.linalg.norm(want)


# ------------------------------------------------------------ ranges and values

@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_infinite_queries_stay_in_their_heads(dtype):
    rng = np.random.default_rng(3)
    k, v = (so.to_bits(rng.standard_normal((1, 700, 2, 64)), dtype) for _ in range(2))
    q = rng.standard_normal((40, 8, 64)).astype(np.float32)
    clean = attend(q.reshape(40, -1), k, v, dtype, [0, 40], [700], 8)
    bad = [(0, 1), (7, 6), (39, 3), (20, 0)]
    for i, (r, h) in enumerate(bad):
        q[r, h, 5 * i] = [np.inf, -np.inf, np.nan, np.inf][i]
    got = attend(q.reshape(40, -1), k, v, dtype, [0, 40], [700], 8)
    for r, h in bad:
        assert np.isnan(got[r, h]).all()
        got[r, h] = clean[r, h]
    np.testing.assert_array_equal(got, clean)


def test_bf16_largest_values():
    """The largest finite value of the cache comes back from one position; of 70,
    whose weights are all the largest, the weighted sum is 70 * 3.39e38, which fp32
    does not hold: infinities of their signs."""
    v = np.full((1, 70, 1, 64), 0x7F7F, np.uint16)
    v[..., 1::2] = 0xFF7F
    want = so.from_bits(v[0, 0, 0], "bf16")
    q, k = np.zeros((5, 64)), np.zeros((1, 70, 1, 64), np.uint16)
    got = attend(q, k, v, "bf16", [0, 5], [70], 1)
    np.testing.assert_array_equal(got, np.broadcast_to(np.sign(want) * np.inf, got.shape))
    got = attend(q, k, v, "bf16", [0, 5], [70], 1, first=ints(np.arange(5) * 17), last=ints(np.arange(5) * 17 + 1))
    assert np.isfinite(got).all() and (np.abs(got / want - 1) <= 2.0 ** -19).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_scores_that_rise(dtype):
    """The base moves again and again, for some columns and not for others."""
    n, hd = 900, 64
    k = np.zeros((1, n, 1, hd))
    k[0, :, 0, 0] = np.arange(n) / 4
    rng = np.random.default_rng(2)
    vb = so.to_bits(rng.standard_normal((1, n, 1, hd)), dtype)
    q = np.zeros((60, hd))
    q[:, 0] = rng.uniform(-2, 2, 60)
    kb = so.to_bits(k, dtype)
    got = attend(q, kb, vb, dtype, [0, 60], [n], 1, scale=1.0)
    see = np.arange(n)[None] <= n - 60 + np.arange(60)[:, None]
    want, tol = ro.attend(q.astype(np.float32), so.from_bits(kb[0, :, 0], dtype), so.from_bits(vb[0, :, 0], dtype), 1.0, see)
    within(got[:, 0], want, tol)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("m, words", [(33, 2), (64, 2), (65, 3), (100, 4), (300, 10)])
def test_trees_of_many_rows(dtype, m, words):
    assert -(-m // 32) == words
    rows_case([m, 2], [m + 77, 500], 6, 2, 64, dtype, 16, seed=m, mask="tree", idle=0.1, bad_slots={0: [80, 77 + m // 2]})


@pytest.mark.parametrize("hd", [64, 128])
def test_ranges_of_any_numbers(hd):
    """Ranges past both ends of int32's room, alone and beside a tree's bits."""
    rng = np.random.default_rng(12)
    n, m = 200, 40
    k, v = (so.to_bits(rng.standard_normal((1, n, 1, hd)), "f16") for _ in range(2))
    q = rng.standard_normal((m, hd)).astype(np.float32)
    least, most = -2 ** 31, 2 ** 31 - 1
    first = np.array([least, most, 0, -1, 100, most, least, 150] * 5)
    last = np.array([most, least, least, most, least, most, least, -7] * 5)
    tree = [0 if i % 3 == 0 else x for i, x in enumerate(ro.ancestors([-1] + list(range(m - 1))))]
    for bits in (None, sa.DevBuf.of(ro.words(tree, 2))):
        see = (np.arange(n) >= first[:, None]) & (np.arange(n) < last[:, None])
        if bits:
            see[:, n - m:] |= np.array([[x >> j & 1 for j in range(m)] for x in tree], bool)
        got = attend(q, k, v, "f16", [0, m], [n], 1, first=ints(first), last=ints(last), tree=bits, tree_words=2 if bits else 0)
        want, tol = ro.attend(q, so.from_bits(k[0, :, 0], "f16"), so.from_bits(v[0, :, 0], "f16"), hd ** -0.5, see)
        within(got[:, 0], want, tol)


def test_positions_far_apart():
    """A bias of distances past 2^24, which fp32 rounds by half a step, and of 0."""
    rng = np.random.default_rng(8)
    hd, n = 64, 20
    k, v = (so.to_bits(rng.standard_normal((1, n, 1, hd)), "f16") for _ in range(2))
    q = rng.standard_normal((n, hd)).astype(np.float32)
    pos = rng.integers(0, 1 << 30, n)
    pos[5:9] = pos[4]
    got = attend(q, k, v, "f16", [0, n], [n], 1, first=ints([0] * n), last=ints([n] * n), pos=ints(pos),
                 slope=sa.DevBuf.of(np.array([2.0 ** -28], np.float32)))
    far = np.abs(pos[:, None] - pos[None]).astype(np.float64)
    want, tol = ro.attend(q, so.from_bits(k[0, :, 0], "f16"), so.from_bits(v[0, :, 0], "f16"), hd ** -0.5, np.ones((n, n), bool),
                          bias=2.0 ** -28 * far)
    within(got[:, 0], want, tol)


def test_equal_calls_give_equal_bits():
    rng = np.random.default_rng(9)
    k, v = (so.to_bits(rng.standard_normal((5, 900, 2, 128)), "f16") for _ in range(2))
    q = rng.standard_normal((70, 8 * 128))
    start, lens = [0, 20, 20, 55, 60, 70], [900, 3, 400, 5, 700]
    one = attend(q, k, v, "f16", start, lens, 8, cap=20.0)
    for _ in range(3):
        np.testing.assert_array_equal(attend(q, k, v, "f16", start, lens, 8, cap=20.0), one)


def test_rows_of_a_prompt_are_rows_of_their_own():
    """A prompt's chunk gives what its rows give as so many sequences of one token
    over the same pages."""
    rng = np.random.default_rng(10)
    n, m, hd, kv, heads, page = 333, 61, 128, 2, 8, 16
    pages = -(-n // page)
    bits = [so.to_bits(rng.standard_normal((pages, page, kv, hd)), "bf16") for _ in range(2)]
    pools = [sa.DevBuf.of(b) for b in bits]
    q = rng.standard_normal((m, heads * hd)).astype(np.float32)
    table = rng.permutation(pages).astype(np.int32)
    qb, out, part = sa.DevBuf.of(q), sa.DevBuf(4 * m * heads * hd), sa.DevBuf(4 * serving.rows_floats(1, m, kv, heads, hd, n))
    serving.attention_rows(serving.Pages(*pools, ints([table]), pages, page, 1, pages, kv, hd, "bf16"),
                           serving.Rows(ints([0, m]), ints([n]), m, n), qb, heads, part, out)
    got = out.read(np.float32)
    part = sa.DevBuf(4 * serving.part_floats(m, heads, hd, n))
    serving.attention(serving.Pages(*pools, ints(np.tile(table, (m, 1))), pages, page, m, pages, kv, hd, "bf16"), qb,
                      ints(n - m + 1 + np.arange(m)), n, heads, part, out)
    one = out.read(np.float32)
    # the bounds of either against 64 bits, as in the tests of each
    kk, vv = (so.from_bits(b[table], "bf16").reshape(-1, kv, hd)[:n] for b in bits)
    see = np.arange(n)[None] <= n - m + np.arange(m)[:, None]
    for h in range(heads):
        want, tol = ro.attend(q.reshape(m, heads, hd)[:, h], kk[:, h // 4], vv[:, h // 4], hd ** -0.5, see)
        for x in (got, one):
            within(x.reshape(m, heads, hd)[:, h], want, tol)


# ------------------------------------------------------------ sizes

@pytest.mark.parametrize("ms, lens, heads, kv, hd, top", [
    ([1], [1], 8, 2, 128, 1), ([8], [513], 8, 2, 128, 513), ([3], [70001], 4, 4, 64, 70001), ([5, 0, 90], [600, 40, 1000], 16, 1, 64, 1000),
    ([300], [300], 32, 8, 128, 600), ([2] * 257, [600] * 257, 4, 2, 64, 700), ([60] * 40, [200] * 40, 2, 2, 128, 200)])
def test_attention_stays_in_its_buffers(ms, lens, heads, kv, hd, top):
    rng = np.random.default_rng(top)
    page, n_seq, n_row = 64, len(ms), sum(ms)
    pages = -(-top // page)
    bits = [so.to_bits(rng.standard_normal((pages + 1, page, kv, hd)), "f16") for _ in range(2)]
    table = np.tile(rng.permutation(pages + 1)[:pages], (n_seq, 1)).astype(np.int32)
    pg = serving.Pages(*map(sa.DevBuf.of, bits), sa.DevBuf.of(table), pages + 1, page, n_seq, pages, kv, hd)
    part, out = Guarded(4 * serving.rows_floats(n_seq, n_row, kv, heads, hd, top)), Guarded(4 * n_row * heads * hd)
    q = sa.DevBuf.of(rng.standard_normal((n_row, heads * hd)).astype(np.float32))
    start = np.concatenate([[0], np.cumsum(ms)])
    falls = start[::-1].copy()
    for st, ls in ((start, lens), (start, [top + 99] * n_seq), (start, rng.integers(0, top + 1, n_seq)), (start, [0] * n_seq),
                   (start, [-5] * n_seq), (falls, lens), (np.where(np.arange(n_seq + 1) % 2, n_row + 5, -3), [top] * n_seq)):
        serving.attention_rows(pg, serving.Rows(ints(st), ints(ls), n_row, top), q, heads, part, out)
        sa.sync()
        assert part.intact() and out.intact()
        if st is start and ls is lens:
            assert np.isfinite(out.read(np.float32, n_row * heads * hd)).all()


def test_far_pages():
    """Pages whose offset passes 32 bits, in values and in bytes."""
    rng = np.random.default_rng(3)
    stride, hd, page = 1 << 30, 128, 16
    pools = [sa.DevBuf(2 * (4 * stride + page * hd)) for _ in range(2)]
    table = np.array([[4, 1, 3]], np.int32)
    x = [so.to_bits(rng.standard_normal((3 * page, hd)), "f16") for _ in range(2)]

    def put(buf, pid, w):
        sa._chk(sa.lib().sml_hip_h2d(buf.ptr + 2 * int(pid) * stride, w.ctypes.data, w.nbytes))

    def get(buf, pid):
        w = np.empty((page, hd), np.uint16)
        sa._chk(sa.lib().sml_hip_d2h(w.ctypes.data, buf.ptr + 2 * int(pid) * stride, w.nbytes))
        return w
    for b, w in zip(pools, x):
        for i, pid in enumerate(table[0]):
            put(b, pid, w[i * page:(i + 1) * page])
    tb = sa.DevBuf.of(table)
    pg = serving.Pages(*pools, tb, 5, page, 1, 3, 1, hd, page_stride=stride)
    q = rng.standard_normal((6, 4 * hd)).astype(np.float32)
    out, part = sa.DevBuf(4 * 6 * 4 * hd), sa.DevBuf(4 * serving.rows_floats(1, 6, 1, 4, hd, 45))
    serving.attention_rows(pg, serving.Rows(ints([0, 6]), ints([45]), 6, 45), sa.DevBuf.of(q), 4, part, out)
    k, v = (so.from_bits(w, "f16")[:45] for w in x)
    got, see = out.read(np.float32).reshape(6, 4, hd), np.arange(45)[None] <= 39 + np.arange(6)[:, None]
    for h in range(4):
        want, tol = ro.attend(q.reshape(6, 4, hd)[:, h], k, v, hd ** -0.5, see)
        within(got[:, h], want, tol)
    # row 5 of the last six goes to slot 40, page 3; pages 4 and 3 to 0 and 2
    serving.accept(pg, 6, ints([0, 6]), ints([45]), ints([0, 1, 2, 3, 4, 5]), ints([-1, 0, 0, 0, 0, 0]), ints([5] * 6), 4, n_kept=ints([0]))
    for b, w in zip(pools, x):
        w[40] = w[44]
        np.testing.assert_array_equal(get(b, 3), w[32:])
    serving.compact(pg, 2, ints([3, 4]), ints([2, 0]), table=tb)
    assert tb.read(np.int32).tolist() == [0, 1, 2]
    for b, w in zip(pools, x):
        np.testing.assert_array_equal(get(b, 0), w[:16])
        np.testing.assert_array_equal(get(b, 2), w[32:])
    to, ln = ints([[9] * 3]), ints([9])
    serving.fork(pg, ints([37]), 1, ints([0]), ints([4]), to, ln)
    assert to.read(np.int32).tolist() == [0, 1, 4] and ln.read(np.int32)[0] == 37
    for b, w in zip(pools, x):
        np.testing.assert_array_equal(get(b, 4)[:5], w[32:37])


def test_as_many_sequences_as_there_may_be():
    """65535 sequences of a row each, and of none or several, that share their pages."""
    rng = np.random.default_rng(7)
    n, hd, page, pages, top = 65535, 64, 64, 3, 180
    k, v = (so.to_bits(rng.standard_normal((pages, page, 1, hd)), "f16") for _ in range(2))
    table = ints(np.tile(rng.permutation(pages), (n, 1)))
    first = table.read(np.int32, pages)
    pg = serving.Pages(sa.DevBuf.of(k), sa.DevBuf.of(v), table, pages, page, n, pages, 1, hd)
    q = rng.standard_normal(hd).astype(np.float32)
    kk, vv = (so.from_bits(w[first], "f16").reshape(-1, hd) for w in (k, v))
    for ms in (np.ones(n, int), rng.permutation(np.tile([0, 0, 1, 3, 1], n // 5))):
        lens = np.maximum(ms, rng.integers(0, 4, n))
        lens[[0, 1, 40000, n - 1]] = [170, 129, 180, 64]
        start = np.concatenate([[0], np.cumsum(ms)])
        n_row = start[-1]
        out, part = sa.DevBuf.of(np.full((n_row, hd), np.nan, np.float32)), sa.DevBuf(4 * serving.rows_floats(n, n_row, 1, 1, hd, top))
        serving.attention_rows(pg, serving.Rows(ints(start), ints(lens), n_row, top), sa.DevBuf.of(np.tile(q, (n_row, 1))), 1, part, out)
        got = out.read(np.float32).reshape(n_row, hd)
        seen = np.repeat(lens - ms, ms) + np.arange(n_row) - np.repeat(start[:-1], ms) + 1
        for s in np.unique(seen):
            want, tol = so.attend(q[None], kk[:s], vv[:s], hd ** -0.5)
            within(got[seen == s], np.repeat(want, (seen == s).sum(), 0), np.repeat(tol, (seen == s).sum(), 0), f"{s} positions")


def test_as_many_rows_as_there_may_be():
    """A prompt of 65535 rows, some of them looked at."""
    rng = np.random.default_rng(11)
    n, hd, page = 65535, 64, 256
    pages = -(-n // page)
    bits = [so.to_bits(rng.standard_normal((pages, page, 1, hd)), "bf16") for _ in range(2)]
    pg = serving.Pages(*map(sa.DevBuf.of, bits), ints([np.arange(pages)]), pages, page, 1, pages, 1, hd, "bf16")
    q = rng.standard_normal((n, hd)).astype(np.float32)
    out, part = sa.DevBuf.of(np.full((n, hd), np.nan, np.float32)), sa.DevBuf(4 * serving.rows_floats(1, n, 1, 1, hd, n))
    serving.attention_rows(pg, serving.Rows(ints([0, n]), ints([n]), n, n), sa.DevBuf.of(q), 1, part, out)
    got = out.read(np.float32).reshape(n, hd)
    assert np.isfinite(got).all()
    kk, vv = (so.from_bits(b, "bf16").reshape(-1, hd) for b in bits)
    for r in (0, 1, 63, 64, 127, 128, 4095, 30000, 65407, 65534):
        want, tol = ro.attend(q[r:r + 1], kk[:r + 1], vv[:r + 1], hd ** -0.5, np.ones((1, r + 1), bool))
        within(got[r:r + 1], want, tol, f"row {r}")


def test_a_path_as_long_as_may_be_kept():
    """A chain of 1100 drafted rows, all of them picked: 1024 are kept; its rows
    lie behind a first branch that is not."""
    m, most, page, hd = 1101, 1024, 64, 64
    n = m + 5
    rng = np.random.default_rng(1)
    pages = -(-n // page)
    pool = rng.integers(0, 1 << 16, (pages, page, 1, hd)).astype(np.uint16)
    bufs = [sa.DevBuf.of(pool), sa.DevBuf.of(pool ^ 1)]
    pg = serving.Pages(*bufs, ints([np.arange(pages)]), pages, page, 1, pages, 1, hd)
    tok = np.arange(m)
    parent = np.array([-1, 0, 0] + list(range(2, m - 1)))
    pick = np.concatenate([[2, 7], np.arange(3, m + 1)])
    n_kept, kept = ints([0]), ints([0] * most)
    serving.accept(pg, m, ints([0, m]), ints([n]), ints(tok), ints(parent), ints(pick), most, n_kept, kept)
    path = [0] + list(range(2, most + 1))
    assert n_kept.read(np.int32)[0] == most and kept.read(np.int32).tolist() == path
    for b, old in zip(bufs, (pool, pool ^ 1)):
        want = old.reshape(-1, hd).copy()
        want[5:5 + most] = want[5 + np.array(path)]
        np.testing.assert_array_equal(b.read(np.uint16).reshape(-1, hd), want)


@pytest.mark.parametrize("kv", [257, 4096])
def test_as_many_heads_as_there_may_be(kv):
    """More KV heads than there are CUs, some of them looked at."""
    rng = np.random.default_rng(kv)
    n, ms = 150, [2, 0, 5, 1, 3]
    k, v = (so.to_bits(rng.standard_normal((5, n, kv, 64)), "f16") for _ in range(2))
    start = np.concatenate([[0], np.cumsum(ms)])
    q = rng.standard_normal((11, kv, 64)).astype(np.float32)
    got = attend(q.reshape(11, -1), k, v, "f16", start, [n, 5, 70, 129, 3], kv)
    for h in (0, 1, 200, kv - 1):
        for b, (m, ln) in enumerate(zip(ms, [n, 5, 70, 129, 3])):
            see = np.arange(ln)[None] <= ln - m + np.arange(m)[:, None]
            rows = slice(start[b], start[b + 1])
            want, tol = ro.attend(q[rows, h], so.from_bits(k[b, :ln, h], "f16"), so.from_bits(v[b, :ln, h], "f16"), 0.125, see)
            within(got[rows, h], want, tol, f"sequence {b}, head {h}")


@pytest.mark.parametrize("rules", [False, True])
@pytest.mark.parametrize("m, n", [(1601, 1700), (2100, 2100)])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
def test_long_prompts(hd, dtype, m, n, rules):
    """Tiles enough for a CU and a half, and for two workgroups of every CU: 32
    heads over 8, two of them looked at in all rows. With rules, windows, a tree, rows of
    padding, a cap and the bias of distance; infinities where only some rows look."""
    rng = np.random.default_rng(m + hd)
    k, v = (so.to_bits(rng.standard_normal((1, n, 8, hd)), dtype) for _ in range(2))
    q = rng.standard_normal((m, 32, hd)).astype(np.float32)
    row, past = np.arange(m), n - m
    see = np.arange(n)[None] <= past + row[:, None]
    kw = {}
    if rules:
        first = np.where(row % 7 == 3, n, np.maximum(0, row - 300))
        last = np.where(row % 5 == 1, 0, past + row // 2)
        tree = rng.random((m, m)) < 0.05
        tree[row % 11 == 2] = False
        bits = np.packbits(np.pad(tree, ((0, 0), (0, -m % 32))), axis=1, bitorder="little").view(np.uint32)
        see = (np.arange(n) >= first[:, None]) & (np.arange(n) < last[:, None])
        see[:, past:] |= tree
        slope = rng.uniform(0, 0.02, 32).astype(np.float32)
        pos = past + rng.permutation(m)
        kw = dict(first=ints(first), last=ints(last), tree=sa.DevBuf.of(bits), tree_words=bits.shape[1], slope=sa.DevBuf.of(slope), pos=ints(pos),
                  cap=20.0)
        far = np.abs(pos[:, None] - np.concatenate([np.arange(past), pos])[None]).astype(np.float64)
        v[0, [5, 600], :, 1] = 0x7C00 if dtype == "f16" else 0x7F80
    got = attend(q.reshape(m, -1), k, v, dtype, [0, m], [n], 32, **kw)
    for h in (5, 30):
        kk, vv = (so.from_bits(x[0, :, h // 4], dtype) for x in (k, v))
        bad = see[:, [5, 600]].any(1) if rules else np.zeros(m, bool)
        assert np.isnan(got[bad, h]).any(1).all()
        want, tol = ro.attend(q[:, h], kk, np.where(np.isfinite(vv), vv, 0), hd ** -0.5, see, *((20.0, float(slope[h]) * far) if rules else ()))
        within(got[~bad, h], want[~bad], tol[~bad], f"head {h}")
        assert not rules or (0 < bad.sum() < m and (got[~see.any(1), h] == 0).all() and (~see.any(1)).any())


# ------------------------------------------------------------ streams and graphs

def step_state(seed, ms=(9, 1, 30, 4), most=8):
    """The inputs of one drafted step of a small model of two layers: the cache of the past, the rows, their trees."""
    rng = np.random.default_rng(seed)
    H, KV, hd, page, layers, V = 6, 2, 64, 16, 2, 70
    n_seq, ms = len(ms), np.array(ms)
    past = rng.integers(0, 90, n_seq)
    seq_pages = -(-(90 + max(ms)) // page)
    n_pages = n_seq * seq_pages + 9
    n = int(ms.sum())
    start = np.concatenate([[0], np.cumsum(ms)])
    trees = [tree_of(rng, m) for m in ms]
    bits = np.concatenate([ro.words(ro.ancestors(t), 1) for t in trees])
    depth = []
    for t in trees:
        d = []
        for p in t:
            d.append(0 if p < 0 else d[p] + 1)
        depth.append(np.array(d))
    seq = np.repeat(np.arange(n_seq), ms)
    slot = np.concatenate([p + np.arange(m) for p, m in zip(past, ms)])
    pos = np.concatenate([p + d for p, d in zip(past, depth)])
    order = rng.permutation(n_pages).astype(np.int32)
    size = page * KV * hd
    f16 = lambda *sh: so.to_bits(rng.standard_normal(sh), "f16")          # noqa: E731
    return dict(H=H, KV=KV, hd=hd, page=page, layers=layers, V=V, n_seq=n_seq, n=n, seq_pages=seq_pages, n_pages=n_pages, most=most, size=size,
                start=start, lens=past + ms, seq=seq, slot=slot, pos=pos, bits=bits, parent=np.concatenate(trees),
                table=order[:n_seq * seq_pages].reshape(n_seq, seq_pages), fresh=order[n_seq * seq_pages:][:5],
                forked=rng.integers(0, n_seq, 5), src=np.sort(order[:4]), dst=order[-4:],
                k=f16(layers, n_pages, page, KV, hd), v=f16(layers, n_pages, page, KV, hd),
                qkv=rng.standard_normal((layers, n, (H + 2 * KV) * hd)).astype(np.float32), tok=rng.integers(0, V, n),
                logits=rng.standard_normal((n, V)).astype(np.float32), slope=rng.uniform(0, 0.3, H).astype(np.float32))


INTS = ("start", "lens", "seq", "slot", "pos", "parent", "table", "fresh", "forked", "src", "dst", "tok")
VALUES = ("k", "v", "qkv", "logits", "slope", "bits")
MADE = ("q", "out", "part", "pick", "lpart", "n_kept", "kept", "next", "len_out", "to", "ln")


def step_buffers(s):
    d = {k: ints(s[k]) for k in INTS} | {k: sa.DevBuf.of(s[k]) for k in VALUES}
    cos, sin = so.rope_tables(s["hd"] // 2, 200)
    d["cos"], d["sin"] = sa.DevBuf.of(cos), sa.DevBuf.of(sin)
    n, H, hd = s["n"], s["H"], s["hd"]
    sizes = dict(q=4 * n * H * hd, out=4 * s["layers"] * n * H * hd, part=4 * serving.rows_floats(s["n_seq"], n, s["KV"], H, hd, 130), pick=4 * n,
                 lpart=serving.logits_part_bytes(n, s["V"]), n_kept=4 * s["n_seq"], kept=4 * s["n_seq"] * s["most"],
                 next=4 * s["n_seq"] * s["most"], len_out=4 * s["n_seq"], to=4 * 5 * s["seq_pages"], ln=20)
    for k in MADE:
        d[k] = sa.DevBuf.of(np.full(sizes[k], 0xFF, np.uint8))
    return d


class At:
    def __init__(self, p):
        self.ptr = p


def step_run(s, d, stream):
    n, H, KV, hd, L, size = s["n"], s["H"], s["KV"], s["hd"], s["layers"], s["size"]
    layer = lambda name, i, each: At(d[name].ptr + i * each)               # noqa: E731
    geometry = (d["table"], s["n_pages"], s["page"], s["n_seq"], s["seq_pages"], KV, hd)
    for i in range(L):
        pg = serving.Pages(layer("k", i, 2 * size * s["n_pages"]), layer("v", i, 2 * size * s["n_pages"]), *geometry)
        serving.append_axes(pg, layer("qkv", i, 4 * n * (H + 2 * KV) * hd), n, d["slot"], d["pos"], bytes(hd // 2), d["cos"], d["sin"], 200, H,
                            seq=d["seq"], q_out=d["q"], stream=stream)
        rows = serving.Rows(d["start"], d["lens"], n, 130, tree=d["bits"], tree_words=1, pos=d["pos"], slope=d["slope"], cap=30.0)
        serving.attention_rows(pg, rows, d["q"], H, d["part"], layer("out", i, 4 * n * H * hd), stream=stream)
    serving.adjust_logits(d["logits"], n, s["V"], tok=d["pick"], part=d["lpart"], stream=stream)
    pg = serving.Pages(d["k"], d["v"], *geometry)
    lay = dict(n_layer=L, layer_stride=size * s["n_pages"], stream=stream)
    serving.accept(pg, n, d["start"], d["lens"], d["tok"], d["parent"], d["pick"], s["most"], d["n_kept"], d["kept"], d["next"], d["len_out"], **lay)
    serving.fork(pg, d["len_out"], 5, d["forked"], d["fresh"], d["to"], d["ln"], **lay)
    serving.compact(pg, 4, d["src"], d["dst"], table=d["table"], **lay)


def step_outputs(d):
    return {k: d[k].read(np.uint32) for k in ("out", "q", "pick", "n_kept", "kept", "next", "len_out", "to", "ln", "table")} | \
        {k: d[k].read(np.uint16) for k in ("k", "v")}


def test_captured_step_replays():
    """A drafted step on a stream of its own, captured and replayed between eager
    work on new inputs: every replay equals the eager call bit for bit."""
    hip = Hip()
    states = [step_state(i) for i in range(4)]
    want = []
    for s in states:
        d = step_buffers(s)
        step_run(s, d, 0)
        sa.sync()
        want.append(step_outputs(d))
    d, st = step_buffers(states[0]), hip.stream.value
    sa.sync()
    step_run(states[0], d, st)
    hip("hipStreamSynchronize", hip.stream)
    for k, w in want[0].items():
        np.testing.assert_array_equal(step_outputs(d)[k], w, err_msg=k)
    ex = hip.capture(lambda: step_run(states[0], d, st))
    for i in (1, 2, 3, 0, 2):
        s = states[i]
        for k in INTS:
            d[k].write(np.array(s[k], np.int32))
        for k in VALUES:
            d[k].write(s[k])
        for k in MADE:
            d[k].write(np.full(d[k].nbytes, 0xFF, np.uint8))
        sa.sync()
        hip.replay(ex)
        got = step_outputs(d)
        for k, w in want[i].items():
            np.testing.assert_array_equal(got[k], w, err_msg=f"{k} of replay {i}")


def test_two_graphs_with_workspaces_of_their_own():
    hips, ds, exs, want = [Hip(), Hip()], [], [], []
    states = [step_state(10), step_state(11, ms=(3, 25))]
    for s, h in zip(states, hips):
        d = step_buffers(s)
        step_run(s, d, 0)
        sa.sync()
        want.append(step_outputs(d))
        d = step_buffers(s)
        sa.sync()
        ds.append(d)
        exs.append(h.capture(lambda: step_run(s, d, h.stream.value)))
    for _ in range(3):
        for s, d in zip(states, ds):                          # what a step changes
            for k in ("k", "v"):
                d[k].write(s[k])
            d["table"].write(np.array(s["table"], np.int32))
        sa.sync()
        for h, ex in zip(hips, exs):
            h("hipGraphLaunch", ex, h.stream)
        for h in hips:
            h("hipStreamSynchronize", h.stream)
        for d, w in zip(ds, want):
            got = step_outputs(d)
            for k in w:
                np.testing.assert_array_equal(got[k], w[k], err_msg=k)


FIRST = """
import sys
sys.path[:0] = sys.argv[1:]
import numpy as np
import sheep_amd as sa
import test_gpu_rows_edges as t
sa.init(0)
s = t.step_state(1)
d, hip = t.step_buffers(s), t.Hip()
sa.sync()
ex = hip.capture(lambda: t.step_run(s, d, hip.stream.value))
hip.replay(ex)
got = t.step_outputs(d)
d = t.step_buffers(s)
t.step_run(s, d, 0)
sa.sync()
for k, w in t.step_outputs(d).items():
    np.testing.assert_array_equal(got[k], w, err_msg=k)
print("equal")
"""


def test_first_calls_of_a_process_inside_a_capture():
    here = os.path.dirname(os.path.abspath(__file__))
    r = subprocess.run([sys.executable, "-c", FIRST, os.path.dirname(here), here], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and r.stdout.strip().endswith("equal"), r.stdout + r.stderr


# ------------------------------------------------------------ a run of them together

def test_drafted_decoding_gives_what_decoding_gives():
    """Greedy decoding of a small model of two layers, once a token a step and
    once with a tree of drafted tokens a step (some of them right): the same
    tokens. Prompts go through attention_rows in a chunk, sequences fork after it and
    pages are moved in between."""
    rng = np.random.default_rng(42)
    E, H, KV, hd, page, layers, V, steps = 64, 4, 2, 64, 16, 2, 211, 12
    W = (H + 2 * KV) * hd
    emb = rng.standard_normal((V, E))
    wqkv = rng.standard_normal((layers, E, W)) / 8
    wo = rng.standard_normal((layers, H * hd, E)) / 8
    cos, sin = (sa.DevBuf.of(t) for t in so.rope_tables(hd // 2, 256))
    norm = lambda x: x / np.sqrt((x * x).mean(-1, keepdims=True))          # noqa: E731
    prompts = [list(map(int, rng.integers(0, V, m))) for m in (21, 5)]
    n_req, seq_pages, n_pages = 2, 6, 40
    size = page * KV * hd
    lay = dict(n_layer=layers, layer_stride=n_pages * size)

    class Cache:
        def __init__(self, n_seq):
            self.k, self.v = (sa.DevBuf.of(np.full(layers * n_pages * size, 0x7E00, np.uint16)) for _ in range(2))
            self.n_seq, self.free = n_seq, list(rng.permutation(n_pages))
            self.table = np.full((n_seq, seq_pages), -1, np.int32)

        def reach(self, lens):
            for b, n in enumerate(lens):
                for i in range(-(-int(n) // page)):
                    if self.table[b, i] < 0:
                        self.table[b, i] = self.free.pop()

        def pages(self, layer=0):
            o = 2 * layer * n_pages * size
            self.tb = ints(self.table)
            return serving.Pages(At(self.k.ptr + o), At(self.v.ptr + o), self.tb, n_pages, page, self.n_seq, seq_pages, KV, hd)

    def forward(cache, tokens, ms, past, trees=None):
        """The logits of all new rows; they lie in the cache then."""
        past = np.array(past)
        n, start = len(tokens), np.concatenate([[0], np.cumsum(ms)])
        lens = past + np.array(ms)
        cache.reach(lens)
        seq = np.repeat(np.arange(len(ms)), ms)
        slot = np.concatenate([p + np.arange(m) for p, m in zip(past, ms)])
        pos, bits = slot.copy(), None
        if trees is not None:
            depths = []
            for t in trees:
                d = []
                for p in t:
                    d.append(0 if p < 0 else d[p] + 1)
                depths.append(d)
            pos = np.concatenate([p + np.array(d) for p, d in zip(past, depths)])
            bits = sa.DevBuf.of(np.concatenate([ro.words(ro.ancestors(t), 1) for t in trees]))
        x = emb[tokens]
        qo, out = sa.DevBuf(4 * n * H * hd), sa.DevBuf(4 * n * H * hd)
        part = sa.DevBuf(4 * serving.rows_floats(len(ms), n, KV, H, hd, int(max(lens))))
        for i in range(layers):
            pg = cache.pages(i)
            qkv = sa.DevBuf.of((norm(x) @ wqkv[i]).astype(np.float32))
            if trees is None and all(m == 1 for m in ms):                  # plain decoding: the operators of one token a sequence
                serving.append(pg, qkv, n, ints(slot), cos, sin, 256, H, q_out=qo)
                p1 = sa.DevBuf(4 * serving.part_floats(n, H, hd, int(max(lens))))
                serving.attention(pg, qo, ints(lens), int(max(lens)), H, p1, out)
            else:
                serving.append_axes(pg, qkv, n, ints(slot), ints(pos), bytes(hd // 2), cos, sin, 256, H, seq=ints(seq), q_out=qo)
                rows = serving.Rows(ints(start), ints(lens), n, int(max(lens)), tree=bits, tree_words=1 if bits else 0)
                serving.attention_rows(pg, rows, qo, H, part, out)
            x = x + out.read(np.float32).reshape(n, -1).astype(np.float64) @ wo[i]
        return (norm(x) @ emb.T).astype(np.float32)

    def picks(lg):
        n = len(lg)
        tok, part = sa.DevBuf(4 * n), sa.DevBuf(serving.logits_part_bytes(n, V))
        serving.adjust_logits(sa.DevBuf.of(lg), n, V, tok=tok, part=part)
        return tok

    def forked(cache, past, parents):
        """The cache's sequences become these children of theirs, all with pages of their own behind."""
        fresh = [cache.free.pop() for _ in parents]
        to, ln = ints(np.zeros((len(parents), seq_pages))), ints([0] * len(parents))
        serving.fork(cache.pages(), ints(past), len(parents), ints(parents), ints(fresh), to, ln, **lay)
        cache.table, cache.n_seq = to.read(np.int32).reshape(-1, seq_pages).copy(), len(parents)
        return list(ln.read(np.int32))

    # plain decoding: a prompt in one chunk, two samples of the first request and one of the other, which go on differently
    def begin():
        cache = Cache(n_req)
        ms = [len(p) for p in prompts]
        lg = forward(cache, sum(prompts, []), ms, [0] * n_req)
        first = picks(lg[np.cumsum(ms) - 1]).read(np.int32)
        past = forked(cache, ms, [0, 1, 0])
        return cache, past, [int(first[0]), int(first[1]), 3]
    cache, past, last = begin()
    texts = [[t] for t in last]
    for _ in range(steps):
        lg = forward(cache, [t[-1] for t in texts], [1] * 3, past)
        past = [p + 1 for p in past]
        for t, p in zip(texts, picks(lg).read(np.int32)):
            t.append(int(p))

    # the same with drafts: chains and branches around what decoding gave, right and wrong
    cache, past, last = begin()
    got = [[t] for t in last]
    calls = kept_rows = 0
    while min(map(len, got)) <= steps:
        calls += 1
        trees, tokens = [], []
        for b in range(3):
            done = len(got[b])
            guess = texts[b][done:done + 4]
            t, ids = [-1], [got[b][-1]]
            at = 0
            for depth, g in enumerate(guess):
                wrong = int(rng.integers(0, V))
                if rng.random() < 0.5:                        # a wrong branch before the right one
                    t.append(at)
                    ids.append(wrong if wrong != g else (g + 1) % V)
                if rng.random() < 0.25:
                    break
                t.append(at)
                ids.append(g)
                at = len(t) - 1
            trees.append(t)
            tokens += ids
        ms = [len(t) for t in trees]
        lg = forward(cache, tokens, ms, past, trees)
        pick = picks(lg)
        start = np.concatenate([[0], np.cumsum(ms)])
        lens = np.array(past) + ms
        n_kept, kept, nxt, ln = (ints(np.full(s, -9)) for s in (3, (3, 8), (3, 8), 3))
        serving.accept(cache.pages(), len(tokens), ints(start), ints(lens), ints(tokens), ints(np.concatenate(trees)), pick, 8, n_kept, kept, nxt,
                       ln, **lay)
        past = [int(x) for x in ln.read(np.int32)]
        nk = n_kept.read(np.int32)
        for b in range(3):
            assert past[b] == lens[b] - ms[b] + nk[b] and nk[b] >= 1
            kept_rows += nk[b]
            got[b] += [int(x) for x in nxt.read(np.int32).reshape(3, 8)[b, :nk[b]]]
        if calls == 3:                                        # pages move to others, shared ones for all of their sequences
            used = np.unique(cache.table[cache.table >= 0])
            src = np.sort(used[-3:])
            dst = [cache.free.pop() for _ in src]
            pg = cache.pages()
            serving.compact(pg, len(src), ints(src), ints(dst), table=cache.tb, **lay)
            cache.table = cache.tb.read(np.int32).reshape(-1, seq_pages).copy()
            assert not np.isin(cache.table, src).any()
            for buf in (cache.k, cache.v):                    # what lay there is no longer looked at
                x = buf.read(np.uint16).reshape(layers, n_pages, -1)
                x[:, src] = 0x7E00
                buf.write(x)
    assert kept_rows > 1.5 * 3 * calls
    for a, b in zip(got, texts):
        assert a[:steps + 1] == b
