"""Rows' attention where queries, scales and caps lie near the ends of fp32's
range, and over values and keys that are not finite."""
import numpy as np
import pytest

import rows_oracle as ro
import serving_oracle as so
import sheep_amd as sa
from sheep_amd import serving
from test_gpu_rows import ints, rows_case, within
from test_gpu_rows_edges import attend

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    sa.init(0)


# ------------------------------------------------------------ small and large factors

@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads, kv, hd", [(8, 2, 128), (4, 1, 64)])
@pytest.mark.parametrize("mask", ["causal", "tree"])
@pytest.mark.parametrize("q_exp, scale", [(-140, 0.0), (-147, 0.0), (-120, 1e-5), (-20, 2.0 ** -130), (0, 2.0 ** -149), (-60, -2.0 ** -100)])
def test_scores_near_nothing(dtype, heads, kv, hd, mask, q_exp, scale):
    """Scores of some 2^-137 and less, beside masked ones and absent pages: a row is
    the mean of what it attends to, in the general bounds."""
    rows_case([40, 3, 9], [150, 3, 700], heads, kv, hd, dtype, 16, seed=hd, mask=mask, q_exp=q_exp, scale=scale, gone={2: [1, 20]})


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("cap, scale, q_exp, kv_size", [
    (2.0 ** 114, 2.0 ** 15, -38, 9000.0), (2.0 ** 120, -2.0 ** 22, -45, 9000.0), (2.0 ** 90, 0.0, 0, 1.0), (2.0 ** 96, 0.0, -12, 1000.0),
    (2.0 ** 126, 2.0 ** 40, -62, 9000.0), (2.0 ** -40, 2.0 ** -60, 0, 1.0), (2.0 ** -126, 2.0 ** -60, 0, 1.0)])
def test_caps_far_from_their_scores(dtype, hd, bias, cap, scale, q_exp, kv_size):
    """Caps that no score comes near, up to 2^100 times the scale, leave the scores as
    they are, and caps next to nothing leave nothing of them, in the general bounds."""
    rows_case([40, 9], [150, 300], 4, 2, hd, dtype, 16, seed=hd, cap=cap, scale=scale, q_exp=q_exp, kv_size=kv_size, bias=bias)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("cap, scale, q_exp", [(2.0 ** -40, 0.0, 100), (2.0 ** -100, 1.0, 40), (2.0 ** -100, 1.0, 100), (1.0, 2.0 ** 60, 60)])
def test_keys_of_zeros_under_small_caps(dtype, hd, cap, scale, q_exp):
    """Scores of exactly 0, however large the query is over the cap."""
    rng = np.random.default_rng(hd)
    n, m = 150, 40
    k = np.zeros((1, n, 2, hd), np.uint16)
    v = so.to_bits(rng.standard_normal((1, n, 2, hd)), dtype)
    q = (rng.standard_normal((m, 4, hd)) * 2.0 ** q_exp).astype(np.float32)
    got = attend(q.reshape(m, -1), k, v, dtype, [0, m], [n], 4, cap=cap, scale=scale)
    see = np.arange(n) <= n - m + np.arange(m)[:, None]
    for h in range(4):
        want, tol = ro.attend(q[:, h], so.from_bits(k[0, :, 0], dtype), so.from_bits(v[0, :, h // 2], dtype), 1.0, see)
        within(got[:, h], want, tol, f"head {h}")


# ------------------------------------------------------------ values that are not finite

BAD = {"f16": [0x7E00, 0x7C00, 0xFC00], "bf16": [0x7FC0, 0x7F80, 0xFF80]}
# one sequence in splits and in one piece, several (tiles of four waves), prompts (tiles of 128 columns of eight
# and of four waves): the new rows, their positions, heads and KV heads
SHAPES = [([40], [300], 4, 2), ([40], [90], 4, 2), ([9, 40, 1, 30, 3], [300, 190, 210, 230, 90], 4, 2), ([1601], [1650], 32, 8), ([2100], [2100], 32, 8)]


@pytest.mark.parametrize("cap", [0.0, 20.0])
@pytest.mark.parametrize("ms, lens, heads, kv", SHAPES)
@pytest.mark.parametrize("hd, dtype", [(128, "f16"), (64, "bf16"), (128, "bf16"), (64, "f16")])
def test_values_that_are_not_finite_reach_their_dims(ms, lens, heads, kv, hd, dtype, cap):
    """Single values that are NaN or infinite: rows that attend to them have no
    finite output in these dims and the right one in the others, whether every other
    row of the call attends to them too, some do or none but the rows with tree bits do."""
    rng = np.random.default_rng(len(ms) + hd)
    n_seq, n, g = len(ms), max(lens), heads // kv
    k, v = (so.to_bits(rng.standard_normal((n_seq, n, kv, hd)), dtype) for _ in range(2))
    spots = [(5, 3), (17, 3), (70, hd - 1), (71, 40), (85, 0), (n - 2, 33)]
    for i, (slot, dim) in enumerate(spots):
        v[:, slot, kv - 1, dim] = BAD[dtype][i % 3]
    start = np.concatenate([[0], np.cumsum(ms)])
    q = rng.standard_normal((sum(ms), heads, hd)).astype(np.float32)
    row = np.concatenate([np.arange(m) for m in ms])
    top = np.repeat(lens, ms)
    whole = (np.zeros(sum(ms), int), top)
    mixed = (np.where(row % 2, 18, 0), np.where(row % 2, 65, np.where(row % 4, 80, top)))     # odd rows see none of them
    past = np.maximum(0, top - np.repeat(ms, ms) - 6)
    for what, (first, last), bits in (("whole", whole, None), ("mixed", mixed, None), ("tree", (np.minimum(20, past), np.where(row % 3, past, 0)), 0.3)):
        tree = np.zeros((sum(ms), max(ms)), bool)
        if bits:
            tree = (rng.random(tree.shape) < bits) & (row % 5 != 1)[:, None]
        words = -(-max(ms) // 32)
        packed = np.packbits(np.pad(tree, ((0, 0), (0, 32 * words - max(ms)))), axis=1, bitorder="little").view(np.uint32)
        kw = dict(tree=sa.DevBuf.of(packed), tree_words=words) if bits else {}
        got = attend(q.reshape(sum(ms), -1), k, v, dtype, start, lens, heads, first=ints(first), last=ints(last), cap=cap, **kw)
        for b, (m, ln) in enumerate(zip(ms, lens)):
            mine = slice(start[b], start[b + 1])
            see = (np.arange(ln) >= first[mine, None]) & (np.arange(ln) < last[mine, None])
            see[:, ln - m:] |= tree[mine, :m]
            for h in (0, heads - g, heads - 1):
                kk, vv = (so.from_bits(x[b, :ln, h // g], dtype) for x in (k, v))
                hit = see.astype(float) @ ~np.isfinite(vv) > 0
                want, tol = ro.attend(q[mine, h], kk, np.where(np.isfinite(vv), vv, 0), hd ** -0.5, see, cap)
                assert not np.isfinite(got[mine, h][hit]).any(), what
                within(np.where(hit, 0, got[mine, h]), np.where(hit, 0, want), tol, f"{what}, sequence {b}, head {h}")


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("n", [40, 90, 700])
def test_values_that_are_not_finite_of_one_token(n, dtype):
    """The attention of one token a sequence keeps them to their dims as well."""
    rng = np.random.default_rng(n)
    hd, page, pages = 64, 16, 44
    kb, vb = (so.to_bits(rng.standard_normal((pages, page, 2, hd)), dtype) for _ in range(2))
    for i, (slot, dim) in enumerate([(5, 3), (17, 3), (31, 40), (n - 1, 63)]):
        vb[slot // page, slot % page, 1, dim] = BAD[dtype][i % 3]
    q = rng.standard_normal((1, 6, hd)).astype(np.float32)
    out, part = sa.DevBuf(4 * 6 * hd), sa.DevBuf(4 * serving.part_floats(1, 6, hd, n))
    pg = serving.Pages(sa.DevBuf.of(kb), sa.DevBuf.of(vb), ints([np.arange(pages)]), pages, page, 1, pages, 2, hd, dtype)
    serving.attention(pg, sa.DevBuf.of(q), ints([n]), n, 6, part, out)
    got = out.read(np.float32).reshape(6, hd)
    for h in range(6):
        kk, vv = (so.from_bits(x.reshape(-1, 2, hd)[:n, h // 3], dtype) for x in (kb, vb))
        hit = ~np.isfinite(vv).all(0)
        want, tol = ro.attend(q[:, h], kk, np.where(np.isfinite(vv), vv, 0), hd ** -0.5, np.ones((1, n), bool))
        assert not np.isfinite(got[h][hit]).any()
        within(np.where(hit, 0, got[h]), np.where(hit, 0, want[0]), tol[0], f"head {h}")


# ------------------------------------------------------------ keys that are not finite

def key_rule(got, want, tol, other, other_tol, see, up, capped, what):
    """Rows of one head, of which those that see a slot with an infinite key have a
    score that is infinite there (up: upwards) or, of its parts, NaN. NaN and, without a
    cap, an infinity upwards leave nothing but NaN; else the row is `other`."""
    for i in range(len(got)):
        if not see[i]:
            within(got[i], want[i], tol[i], f"{what}, row {i}")
        elif not np.isnan(got[i]).all():
            assert capped or not up[i], f"{what}, row {i}"
            within(got[i], other[i], other_tol[i], f"{what}, row {i}")


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("cap", [0.0, 20.0])
@pytest.mark.parametrize("n", [60, 300])
def test_keys_that_are_not_finite(n, cap, hd, dtype):
    """A key with one infinite dim: rows that do not attend to it know nothing of it,
    of those that do, a score of -infinity has no weight and a capped one is +-cap."""
    rng = np.random.default_rng(hd + n)
    m, heads, g, slot, dim = 40, 4, 2, 30, 7
    k, v = (so.to_bits(rng.standard_normal((1, n, 2, hd)), dtype) for _ in range(2))
    k[0, slot, 1, dim] = BAD[dtype][1]
    q = rng.standard_normal((m, heads, hd)).astype(np.float32)
    first = np.where(np.arange(m) % 3 == 1, 31, 5)
    first[6], last = 30, np.full(m, n)
    last[6] = 31                                              # that slot alone
    got = attend(q.reshape(m, -1), k, v, dtype, [0, m], [n], heads, first=ints(first), last=ints(last), cap=cap)
    see = (np.arange(n) >= first[:, None]) & (np.arange(n) < last[:, None])
    for h in range(heads):
        kk, vv = (so.from_bits(x[0, :, h // g], dtype).copy() for x in (k, v))
        up, bad = q[:, h, dim] > 0, see[:, slot] if h // g else np.zeros(m, bool)
        kk[slot] = np.where(np.isfinite(kk[slot]), kk[slot], 0)
        want, tol = ro.attend(q[:, h], kk, vv, hd ** -0.5, see, cap)
        kk[slot] = 0
        at, rest = np.zeros((m, n)), see.copy()
        at[:, slot] = np.where(up, -cap, cap)
        rest[:, slot] &= cap > 0
        other, other_tol = ro.attend(q[:, h], kk, vv, hd ** -0.5, rest, cap, at)
        key_rule(got[:, h], want, tol, other, other_tol, bad, up, cap > 0, f"head {h}")


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("n", [31, 90, 700])
def test_keys_that_are_not_finite_of_one_token(n, dtype):
    rng = np.random.default_rng(n)
    hd, page, pages, rows, slot, dim = 64, 16, 44, 24, 30, 7
    kb, vb = (so.to_bits(rng.standard_normal((pages, page, 2, hd)), dtype) for _ in range(2))
    kb[slot // page, slot % page, 1, dim] = BAD[dtype][2]
    q = rng.standard_normal((rows, 4, hd)).astype(np.float32)
    out, part = sa.DevBuf(4 * rows * 4 * hd), sa.DevBuf(4 * serving.part_floats(rows, 4, hd, n))
    pg = serving.Pages(sa.DevBuf.of(kb), sa.DevBuf.of(vb), ints(np.tile(np.arange(pages), (rows, 1))), pages, page, rows, pages, 2, hd, dtype)
    lens = np.where(np.arange(rows) % 4 == 1, slot, n)
    serving.attention(pg, sa.DevBuf.of(q), ints(lens), n, 4, part, out)
    got = out.read(np.float32).reshape(rows, 4, hd)
    see = np.arange(n) < lens[:, None]
    for h in range(4):
        kk, vv = (so.from_bits(x.reshape(-1, 2, hd)[:n, h // 2], dtype).copy() for x in (kb, vb))
        kk[slot] = np.where(np.isfinite(kk[slot]), kk[slot], 0)
        want, tol = ro.attend(q[:, h], kk, vv, hd ** -0.5, see)
        rest = see.copy()
        rest[:, slot] = False
        other, other_tol = ro.attend(q[:, h], kk, vv, hd ** -0.5, rest)
        key_rule(got[:, h], want, tol, other, other_tol, see[:, slot] if h // 2 else np.zeros(rows, bool), q[:, h, dim] < 0, False, f"head {h}")
