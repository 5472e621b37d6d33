"""Several rows a sequence over a paged cache, and the cache's upkeep, against
their plain 64-bit forms (rows_oracle.py, which also derives how far fp32 may be
off)."""
import numpy as np
import pytest

import rows_oracle as ro
import serving_oracle as so
import sheep_amd as sa
from sheep_amd import serving

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    sa.init(0)


def ints(x):
    return sa.DevBuf.of(np.array(x, np.int32))


def within(got, want, tol, what=""):
    got = got.astype(np.float64)
    nan = np.isnan(want)
    bad = np.where(nan, np.isfinite(got), ~(np.abs(got - np.where(nan, 0, want)) <= tol))
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, at {np.argwhere(bad)[0]}: " \
        f"{got[tuple(np.argwhere(bad)[0])]} for {want[tuple(np.argwhere(bad)[0])]}, {tol[tuple(np.argwhere(bad)[0])]} allowed"


def make_table(rng, n_seq, seq_pages, n_pages):
    return rng.permutation(n_pages)[:n_seq * seq_pages].reshape(n_seq, seq_pages).astype(np.int32)


# ------------------------------------------------------------ append

def axis_of(hd, kind, n_axis):
    half = hd // 2
    if kind == "sections":
        return serving.sections(*([half // n_axis] * (n_axis - 1) + [half - half // n_axis * (n_axis - 1)]))
    if kind == "turns":
        return bytes(d % n_axis for d in range(half))
    return bytes(d % n_axis if d < half // 2 + 1 else 255 for d in range(half))          # the last pairs stay


@pytest.mark.parametrize("heads, kv, hd, dtype, page", [
    (32, 8, 128, "f16", 16), (12, 2, 128, "bf16", 64), (14, 2, 64, "f16", 32), (3, 3, 64, "bf16", 16)])
@pytest.mark.parametrize("rows, n_axis, kind, in_place, pad", [
    (1, 1, "sections", False, 0), (37, 3, "sections", True, 12), (130, 3, "turns", False, 3), (41, 4, "part", False, 0),
    (9, 2, "part", True, 1)])
def test_append_axes(heads, kv, hd, dtype, page, rows, n_axis, kind, in_place, pad):
    rng = np.random.default_rng(rows + heads + page)
    n_seq, seq_pages, n_rope = 5, 4, 91
    n_pages = n_seq * seq_pages + 3
    table = make_table(rng, n_seq, seq_pages, n_pages)
    table[1, 2], table[2, 0], table[3, 1] = -1, n_pages, -7
    width = (heads + 2 * kv) * hd
    stride = width + pad
    qkv = rng.standard_normal((rows, stride)).astype(np.float32)
    places = rng.permutation(n_seq * seq_pages * page)[:rows]
    seq, slot = places // (seq_pages * page), places % (seq_pages * page)
    pos = rng.integers(0, n_rope, (n_axis, rows))
    if rows > 8:
        slot[3], slot[4], seq[5], seq[6] = -1, seq_pages * page, n_seq, -1
        pos[-1, 7], pos[0, 8] = n_rope, -1
    axis = axis_of(hd, kind, n_axis)
    cos, sin = so.rope_tables(hd // 2, n_rope)
    size = n_pages * page * kv * hd
    was = [rng.integers(0, 1 << 16, size).astype(np.uint16) for _ in range(2)]
    kb, vb = sa.DevBuf.of(was[0]), sa.DevBuf.of(was[1])
    pg = serving.Pages(kb, vb, sa.DevBuf.of(table), n_pages, page, n_seq, seq_pages, kv, hd, dtype)
    qb, qo = sa.DevBuf.of(qkv), sa.DevBuf.of(np.full((rows, heads * hd), 7.5, np.float32))
    serving.append_axes(pg, qb, rows, ints(slot), ints(pos), axis, sa.DevBuf.of(cos), sa.DevBuf.of(sin), n_rope, heads,
                        n_axis=n_axis, seq=ints(seq), q_out=None if in_place else qo, qkv_stride=stride if pad else 0)
    sa.sync()
    k, v = (w.copy().reshape(n_pages, page, kv, hd) for w in was)
    after = qb.read(np.float32).reshape(rows, stride)
    q = after[:, :heads * hd] if in_place else qo.read(np.float32).reshape(rows, heads * hd)
    want_q = (qkv[:, :heads * hd] if in_place else np.full((rows, heads * hd), 7.5)).astype(np.float64)
    tol_q = np.zeros_like(want_q)
    got_k = kb.read(np.uint16).reshape(k.shape)
    turned = np.array([x < n_axis for x in axis])
    for r in range(rows):
        if not (0 <= slot[r] < seq_pages * page and 0 <= seq[r] < n_seq and ((pos[:, r] >= 0) & (pos[:, r] < n_rope)).all()):
            continue
        pid = table[seq[r], slot[r] // page]
        if not 0 <= pid < n_pages:
            continue
        x = qkv[r, :width].reshape(-1, hd)
        c = np.array([cos[pos[a, r], d] if a < n_axis else 1.0 for d, a in enumerate(axis)])
        s = np.array([sin[pos[a, r], d] if a < n_axis else 0.0 for d, a in enumerate(axis)])
        rot, mag = so.rotate(x[:heads + kv], c, s)
        mag = mag * np.concatenate([turned, turned])               # what does not turn stays
        want_q[r] = rot[:heads].reshape(-1)
        tol_q[r] = 2 * so.U * mag[:heads].reshape(-1)
        at = (pid, slot[r] % page)
        v[at] = so.to_bits(x[heads + kv:], dtype)
        within(so.from_bits(got_k[at], dtype), rot[heads:],
               so.HALF[dtype] * (np.abs(rot[heads:]) + 2 * so.U * mag[heads:]) + 2 * so.U * mag[heads:] + 2.0 ** -25, "k")
        k[at] = got_k[at]
    within(q, want_q, tol_q, "q")
    np.testing.assert_array_equal(vb.read(np.uint16).reshape(v.shape), v)
    np.testing.assert_array_equal(got_k, k)
    np.testing.assert_array_equal(after[:, heads * hd if in_place else 0:], qkv[:, heads * hd if in_place else 0:])


@pytest.mark.parametrize("hd, dtype", [(128, "f16"), (64, "bf16")])
def test_one_axis_is_the_plain_append(hd, dtype):
    """With slots that are the positions, the same bits as append."""
    rng = np.random.default_rng(hd)
    H, KV, page, rows = 6, 2, 16, 40
    cos, sin = (sa.DevBuf.of(t) for t in so.rope_tables(hd // 2, 64))
    qkv = rng.standard_normal((rows, H + 2 * KV, hd)).astype(np.float32)
    pos, table = rng.permutation(64)[:rows], ints([[2, 0, 3, 1]])
    got = []
    for axes in (False, True):
        kb, vb = (sa.DevBuf.of(np.zeros(4 * page * KV * hd, np.uint16)) for _ in range(2))
        pg = serving.Pages(kb, vb, table, 4, page, 1, 4, KV, hd, dtype)
        qo = sa.DevBuf(4 * rows * H * hd)
        args = (cos, sin, 64, H)
        if axes:
            serving.append_axes(pg, sa.DevBuf.of(qkv), rows, ints(pos), ints(pos), bytes(hd // 2), *args, seq=ints([0] * rows), q_out=qo)
        else:
            serving.append(pg, sa.DevBuf.of(qkv), rows, ints(pos), *args, seq=ints([0] * rows), q_out=qo)
        got.append([qo.read(np.uint32), kb.read(np.uint16), vb.read(np.uint16)])
    for a, b in zip(*got):
        np.testing.assert_array_equal(a, b)


# ------------------------------------------------------------ attention

BAD = {"f16": [0x7E00, 0x7C00, 0xFC00, 0x7FFF], "bf16": [0x7FC0, 0x7F80, 0xFF80, 0x7FFF]}


def tree_of(rng, m):
    return [-1] + [int(rng.integers(0, j)) for j in range(1, m)]


def rows_case(ms, lens, heads, kv, hd, dtype, page, seed=0, mask="causal", cap=0.0, bias=False, gone=None, scale=0.0,
              q_size=1.0, kv_size=1.0, pad=0, max_len=None, lead=0, behind=0, poison=True, idle=0.0, bad_slots=None,
              q_exp=0, k_exp=0, v_exp=0):
    """One call against the oracle. ms: each sequence's new rows; lens: its
    positions with them. lead, behind: rows that are nobody's. gone: {sequence:
    absent page entries}. poison: NaN and infinities in every slot no row
    attends to. idle: the share of rows that attend to nothing. bad_slots:
    {sequence: slots that hold NaN or infinities whoever attends to them}."""
    rng = np.random.default_rng(seed)
    n_seq = len(lens)
    n_row = lead + sum(ms) + behind
    start = lead + np.concatenate([[0], np.cumsum(ms)])
    seq_pages = max(1, -(-max(lens) // page))
    n_pages = n_seq * seq_pages + 3
    table = make_table(rng, n_seq, seq_pages, n_pages)
    for b, entries in (gone or {}).items():
        for i in entries:
            if i < seq_pages:
                table[b, i] = [-1, n_pages, 1 << 30][i % 3]
    top = max(max(lens), 0) if max_len is None else max_len
    cut = [max(0, min(n, top, seq_pages * page)) for n in lens]
    k, v = (kv_size * rng.standard_normal((n_pages, page, kv, hd)) for _ in range(2))
    kb, vb = so.to_bits(np.clip(k, -3e4, 3e4) * 2.0 ** k_exp, dtype), so.to_bits(np.clip(v, -3e4, 3e4) * 2.0 ** v_exp, dtype)
    first, last, pos = (np.full(n_row, x, np.int64) for x in (0, 0, 7))
    n_words = max(1, -(-max(ms) // 32))
    bits = np.zeros((n_row, n_words), np.uint32)
    see = []                                                  # per sequence [m, n]
    for b, (m, n) in enumerate(zip(ms, cut)):
        past = n - m
        rows = slice(start[b], start[b + 1])
        own = past + np.arange(m)
        lo, hi, at = np.zeros(m, int), own + 1, own.copy()
        if mask == "tree":
            parent = tree_of(rng, m)
            depth = [0] * m
            for j in range(1, m):
                depth[j] = depth[parent[j]] + 1
            hi, at = np.full(m, past), past + np.array(depth, int)
            bits[rows] = ro.words(ro.ancestors(parent), n_words)
        elif mask == "window":
            lo = np.maximum(0, own + 1 - max(1, n // 3))
        elif mask == "prefix":
            hi = np.maximum(hi, past + m // 2)
        elif mask == "docs":
            doc = max(1, m // 3)
            lo = np.where(np.arange(m) >= doc, own - np.arange(m) % doc, 0)
        elif mask == "ragged":
            lo = rng.integers(-5, max(1, n), m)
            hi = lo + rng.integers(-3, max(1, n), m)
        elif mask == "both":                                  # ranges of the past and bits of any rows
            lo = rng.integers(0, max(1, past + 1), m)
            hi = lo + rng.integers(0, max(1, past + 2), m)
            bits[rows] = rng.integers(0, 1 << 32, (m, n_words), dtype=np.uint64).astype(np.uint32)
            at = rng.integers(0, 3 * max(1, n), m)
        none = rng.random(m) < idle
        lo, hi = np.where(none, 0, lo), np.where(none, 0, hi)
        bits[rows][none] = 0
        first[rows], last[rows], pos[rows] = lo, hi, at
        slot = np.arange(n)
        s = (slot >= lo[:, None]) & (slot < hi[:, None])
        for j in range(m):
            if 0 <= past + j < n:
                s[:, past + j] |= (bits[rows][:, j // 32] >> np.uint32(j % 32) & 1).astype(bool)
        there = np.array([0 <= table[b, p // page] < n_pages for p in range(n)], bool)
        see.append(s & there[None, :] if n else s)
    where = lambda b, p: (table[b, p // page], p % page)      # noqa: E731
    if poison:
        keep = np.zeros((n_pages, page), bool)
        for b, s in enumerate(see):
            for p in np.flatnonzero(s.any(0)):
                keep[where(b, p)] = True
        for x in (kb, vb):
            x[~keep] = np.array(BAD[dtype], np.uint16)[rng.integers(0, 4, x[~keep].shape)]
    for b, slots in (bad_slots or {}).items():
        for p in slots:
            for x in (kb, vb):
                x[where(b, p)] = BAD[dtype][p % 4]
    stride = heads * hd + pad
    q = (q_size * rng.standard_normal((n_row, stride))).astype(np.float32)
    q = np.clip(q, -3 * q_size, 3 * q_size) * np.float32(2.0 ** q_exp)
    slope = (2.0 ** rng.uniform(-8, 0, heads)).astype(np.float32)
    out = sa.DevBuf.of(np.full((n_row, heads * hd), 7.5, np.float32))
    part = sa.DevBuf(4 * serving.rows_floats(n_seq, n_row, kv, heads, hd, max(1, top)))
    pg = serving.Pages(sa.DevBuf.of(kb), sa.DevBuf.of(vb), sa.DevBuf.of(table), n_pages, page, n_seq, seq_pages, kv, hd,
                       dtype)
    ranges = mask not in ("causal", "tree") or idle
    rows = serving.Rows(ints(start), ints(lens), n_row, top, first=ints(first) if ranges else None,
                        last=ints(last) if ranges else None, tree=sa.DevBuf.of(bits) if mask in ("tree", "both") else None,
                        tree_words=n_words if mask in ("tree", "both") else 0, pos=ints(pos) if mask in ("tree", "both") else None,
                        slope=sa.DevBuf.of(slope) if bias else None, cap=cap)
    serving.attention_rows(pg, rows, sa.DevBuf.of(q), heads, part, out, scale=scale, q_stride=stride if pad else 0)
    sa.sync()
    got = out.read(np.float32).reshape(n_row, heads, hd)
    sc, g = scale or hd ** -0.5, heads // kv
    assert (got[:lead] == 7.5).all() and (got[lead + sum(ms):] == 7.5).all()
    for b, (m, n) in enumerate(zip(ms, cut)):
        past = n - m
        ids = np.array([(t if 0 <= t < n_pages else 0, o) for t, o in (where(b, p) for p in range(n))], np.int64).reshape(-1, 2)
        mine = slice(start[b], start[b + 1])
        kpos = np.arange(n)
        new = np.arange(n) >= past
        at = pos[mine] if mask in ("tree", "both") else past + np.arange(m)
        kpos[new] = at[np.arange(n)[new] - past]
        far = np.abs(at[:, None] - kpos[None, :]).astype(np.float64)
        for h in range(heads):
            kk, vv = (so.from_bits(x[ids[:, 0], ids[:, 1], h // g], dtype).reshape(-1, hd) for x in (kb, vb))
            want, tol = ro.attend(q[mine, h * hd:(h + 1) * hd], kk, vv, sc, see[b], cap, float(slope[h]) * far if bias else None)
            within(got[mine, h], want, tol, f"sequence {b} of {n}, {m} rows, head {h}")
    return got


HEADS = [(32, 8, 128, "f16", 16), (12, 2, 128, "bf16", 64), (32, 8, 64, "f16", 32), (14, 2, 64, "bf16", 16),
         (4, 4, 128, "f16", 128), (3, 1, 128, "bf16", 16), (16, 1, 64, "f16", 16), (28, 4, 128, "f16", 32)]


@pytest.mark.parametrize("heads, kv, hd, dtype, page", HEADS)
def test_trees(heads, kv, hd, dtype, page):
    rows_case([1, 8, 3, 1, 26, 0, 5], [1, 8, 70, 129, 300, 40, 64], heads, kv, hd, dtype, page, seed=heads, mask="tree")


@pytest.mark.parametrize("heads, kv, hd, dtype, page", HEADS)
@pytest.mark.parametrize("mask", ["causal", "window", "prefix", "docs"])
def test_prompts(heads, kv, hd, dtype, page, mask):
    rows_case([33, 1, 70, 17], [33, 500, 200, 64], heads, kv, hd, dtype, page, seed=heads, mask=mask)


EDGES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 257]


@pytest.mark.parametrize("kv, rep, hd, dtype", [(2, 4, 128, "f16"), (1, 7, 64, "bf16"), (2, 1, 64, "f16")])
def test_rows_of_all_counts(kv, rep, hd, dtype):
    """Counts and lengths on either side of every tile's edge, and rows that are nobody's."""
    rows_case(EDGES, [m + (7 * i) % 50 for i, m in enumerate(EDGES)], kv * rep, kv, hd, dtype, 16, seed=rep, lead=3,
              behind=2)
    rows_case([1, 2, 5, 16, 17], [1, 900, 63, 700, 33], kv * rep, kv, hd, dtype, 32, seed=rep + 1, mask="both", pad=5)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("m, n", [(1, 4095), (8, 4095), (3, 9001), (64, 2500), (300, 1500), (700, 700)])
def test_one_sequence(m, n, dtype):
    rows_case([m], [n], 8, 2, 128, dtype, 16, seed=n, mask="tree" if m < 100 else "causal")


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("cap", [5.0, 30.0, 0.01, 1e4])
@pytest.mark.parametrize("q_size", [1.0, 60.0, 1e-4])
def test_capped_scores(dtype, cap, q_size):
    rows_case([9, 40], [300, 41], 8, 2, 128, dtype, 16, seed=11, mask="tree", cap=cap, q_size=q_size)
    rows_case([40], [150], 6, 3, 64, dtype, 32, seed=12, cap=cap, q_size=q_size, bias=True)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("mask", ["tree", "causal", "prefix", "window", "both"])
def test_bias_of_distance(dtype, mask):
    rows_case([9, 40, 1], [300, 41, 700], 8, 2, 128, dtype, 16, seed=13, mask=mask, bias=True)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("mask", ["tree", "causal", "ragged", "both"])
def test_rows_that_attend_to_nothing(dtype, mask):
    got = rows_case([20, 70, 3], [100, 90, 3], 8, 2, 128, dtype, 16, seed=17, mask=mask, idle=0.5)
    assert (got == 0).all(-1).any()
    got = rows_case([20, 70, 3], [100, 90, 3], 4, 1, 64, dtype, 16, seed=18, mask=mask, idle=1.0)
    assert (got == 0).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_ragged_ranges(dtype):
    for seed in range(3):
        rows_case([50, 7, 130], [200, 300, 140], 8, 2, 128, dtype, 16, seed=seed, mask="ragged", cap=20.0, bias=True)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_absent_pages(dtype):
    rows_case([5, 33, 1, 64, 3], [100, 333, 64, 64, 500], 8, 2, 128, dtype, 16, seed=5, mask="tree",
              gone={0: [0, 1, 2], 1: range(0, 40, 2), 2: range(4), 3: [2], 4: list(range(3, 29))})
    rows_case([50, 200], [700, 2100], 4, 1, 64, dtype, 128, seed=6, gone={0: [5], 1: range(1, 16)})


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("mask", ["tree", "causal", "prefix", "both"])
def test_what_others_attend_to_does_not_count(dtype, mask):
    """Keys and values that are NaN or infinite reach the rows that attend to
    them and no other."""
    rows_case([30, 70, 5], [200, 75, 40], 8, 2, 128, dtype, 16, seed=21, mask=mask,
              bad_slots={0: [180, 199, 175], 1: [20, 74, 40], 2: [36]})
    rows_case([130], [400], 2, 2, 64, dtype, 16, seed=22, mask="window", bad_slots={0: [100, 300, 333]})


def test_many_sequences():
    """Past 256 sequences, whose lengths no workgroup sums."""
    rng = np.random.default_rng(12)
    for n, longest in ((300, 300), (256, 200), (65, 400), (700, 40)):
        ms = [int(x) for x in rng.integers(0, 7, n)]
        lens = [m + int(x) for m, x in zip(ms, rng.integers(0, longest, n))]
        ms[0], lens[0], ms[n // 2], lens[n // 2], ms[-1], lens[-1] = 40, longest + 40, 0, 5, 0, 0
        rows_case(ms, lens, 2, 1, 64, "f16", 16, seed=n, mask="causal" if n % 2 else "tree", lead=n % 3)


def test_lengths_cut():
    rows_case([20, 3, 9], [500, 3, 90], 8, 2, 128, "f16", 32, seed=7, max_len=77)
    rows_case([5, 3], [5, 3], 8, 2, 128, "f16", 32, seed=7, max_len=0)
    rows_case([4, 20], [-3, 40], 8, 2, 128, "f16", 32, seed=8)
    rows_case([40, 20], [3, 25], 8, 2, 128, "bf16", 32, seed=9)                          # fewer positions than rows
    rows_case([40, 20], [3, 25], 8, 2, 128, "f16", 32, seed=9, mask="tree")


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("q_size, scale", [(40.0, 0.0), (1e-3, 0.0), (1.0, 0.7), (3e5, 1e-6), (1e-7, 1e6), (1.0, -0.2)])
def test_query_sizes(dtype, q_size, scale):
    rows_case([20, 17], [300, 17], 8, 2, 128, dtype, 16, seed=9, q_size=q_size, scale=scale, pad=4)


@pytest.mark.parametrize("kv_size, q_size", [(3e-6, 1.0), (3e-6, 2e5), (9000.0, 1.0), (9000.0, 1e-4)])
def test_cache_sizes(kv_size, q_size):
    rows_case([30, 7], [200, 700], 8, 2, 128, "f16", 16, seed=15, kv_size=kv_size, q_size=q_size)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("k_exp, q_exp, v_exp", [(118, -114, 0), (120, -118, 118), (0, 0, 120), (-100, 101, 119), (-110, 111, -100)])
def test_bf16_range(hd, k_exp, q_exp, v_exp):
    rows_case([40, 3], [140, 900], 8, 2, hd, "bf16", 16, seed=hd, k_exp=k_exp, q_exp=q_exp, v_exp=v_exp)


def test_no_rows():
    b = sa.DevBuf(8192)
    pg = serving.Pages(b, b, ints([0]), 1, 16, 1, 1, 1, 128)
    serving.attention_rows(pg, serving.Rows(b, b, 0, 8), b, 1, b, b)
    serving.append_axes(pg, b, 0, b, b, bytes(64), b, b, 1, 1)
    sa.sync()


# ------------------------------------------------------------ the cache's upkeep

def layers_of(rng, n_layer, n_pages, page, kv, hd, shared):
    """Both pools of random bits, and Pages' and the calls' strides of them."""
    size = page * kv * hd
    shape = (n_pages, n_layer, size) if shared else (n_layer, n_pages, size)
    pools = [rng.integers(0, 1 << 16, shape).astype(np.uint16) for _ in range(2)]
    return pools, dict(page_stride=n_layer * size if shared else 0), dict(n_layer=n_layer, layer_stride=size if shared else n_pages * size)


def by_layer(pool, shared, page):
    """[layer][page][position][values] of a pool's bits."""
    x = pool.swapaxes(0, 1) if shared else pool
    return x.reshape(x.shape[0], x.shape[1], page, -1)


@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("n_layer, kv, hd, page, dtype", [(1, 2, 128, 16, "f16"), (5, 3, 64, 32, "bf16"), (32, 8, 128, 16, "f16")])
@pytest.mark.parametrize("most", [1, 3, 40])
def test_accept(shared, n_layer, kv, hd, page, dtype, most):
    rng = np.random.default_rng(n_layer + most)
    ms = [8, 0, 1, 30, 70, 130, 3, 33, 12]
    past = [5, 9, 0, 31, 100, 3, 64, 15, 250]
    n_seq, seq_pages = len(ms), 20
    start = 2 + np.concatenate([[0], np.cumsum(ms)])
    n_row = start[-1] + 4
    n_pages = n_seq * seq_pages if page * n_layer < 200 else 60
    table = np.full((n_seq, seq_pages), -1, np.int32)
    ids = iter(rng.permutation(n_pages))
    for b in range(n_seq):
        for i in range(-(-(past[b] + ms[b]) // page)):
            table[b, i] = next(ids)
    table[8, 15 * 16 // page] = -1                           # some of the new rows' places are absent
    pools, pstride, lay = layers_of(rng, n_layer, n_pages, page, kv, hd, shared)
    tok, pick = rng.integers(0, 4, n_row), rng.integers(0, 4, n_row)
    parent = np.full(n_row, -1)
    for b, m in enumerate(ms):
        if m:
            parent[start[b]:start[b] + m] = tree_of(rng, m) if b % 3 else [-1] + [0] * min(2, m - 1) + list(range(1, max(1, m - 2)))
            for i in range(m):                                # paths go on more often than not, by any of the children
                mine = np.flatnonzero(parent[start[b]:start[b] + m] == i)
                if len(mine) and rng.random() < 0.9:
                    pick[start[b] + i] = tok[start[b] + rng.choice(mine)]
    pick[start[6]] = -1                                       # nothing is permitted behind that root
    tok[start[6] + 1] = -1
    bufs = [sa.DevBuf.of(p) for p in pools]
    pg = serving.Pages(*bufs, sa.DevBuf.of(table), n_pages, page, n_seq, seq_pages, kv, hd, dtype, **pstride)
    lens = [a + m for a, m in zip(past, ms)]
    n_kept, kept, nxt, len_out = (sa.DevBuf.of(np.full(s, -9, np.int32)) for s in (n_seq, (n_seq, most), (n_seq, most), n_seq))
    serving.accept(pg, n_row, ints(start), ints(lens), ints(tok), ints(parent), ints(pick), most, n_kept, kept, nxt,
                   len_out, **lay)
    sa.sync()
    want = [by_layer(p.copy(), shared, page) for p in pools]
    old = [w.copy() for w in want]
    moved = 0
    for b, m in enumerate(ms):
        r = slice(start[b], start[b] + m)
        path = ro.walk(tok[r], parent[r], pick[r], most)
        assert n_kept.read(np.int32)[b] == len(path)
        assert len_out.read(np.int32)[b] == past[b] + len(path)
        row = kept.read(np.int32).reshape(n_seq, most)[b]
        assert row.tolist() == path + [-1] * (most - len(path))
        assert nxt.read(np.int32).reshape(n_seq, most)[b].tolist() == [pick[start[b] + i] for i in path] + [-1] * (most - len(path))
        for j, i in enumerate(path):
            f, t = past[b] + i, past[b] + j
            pf, pt = table[b, f // page], table[b, t // page]
            if pf >= 0 and pt >= 0:
                moved += i != j
                for w, o in zip(want, old):
                    w[:, pt, t % page] = o[:, pf, f % page]
    assert most < 40 or moved > 5
    for w, buf, p in zip(want, bufs, pools):
        np.testing.assert_array_equal(by_layer(buf.read(np.uint16).reshape(p.shape), shared, page), w)


def test_accept_walks_alone():
    """No layers, and outputs left out."""
    n_kept = ints([9])
    pg = serving.Pages(*[sa.DevBuf.of(np.zeros(16 * 64, np.uint16)) for _ in range(2)], ints([[0]]), 1, 16, 1, 1, 1, 64)
    serving.accept(pg, 3, ints([0, 3]), ints([3]), ints([0, 5, 6]), ints([-1, 0, 1]), ints([5, 6, 1]), 8, n_kept=n_kept, n_layer=0)
    assert n_kept.read(np.int32)[0] == 3


def test_accept_parents_that_are_none():
    """Rows that follow themselves, later ones or none are nobody's children."""
    n_kept, kept = ints([9]), ints([9] * 8)
    pg = serving.Pages(*[sa.DevBuf.of(np.zeros(16 * 64, np.uint16)) for _ in range(2)], ints([[0]]), 1, 16, 1, 1, 1, 64)
    serving.accept(pg, 6, ints([0, 6]), ints([6]), ints([1] * 6), ints([0, 1, 5, 99, 0, 4]), ints([1] * 6), 8, n_kept=n_kept,
                   kept=kept)
    assert kept.read(np.int32).tolist() == [0, 4, 5, -1, -1, -1, -1, -1]


@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("n_layer, kv, hd, page", [(1, 2, 128, 16), (5, 3, 64, 64), (24, 8, 128, 32)])
def test_fork(shared, n_layer, kv, hd, page):
    rng = np.random.default_rng(page)
    lens = [0, 1, page - 1, page, page + 1, 3 * page + 5, 4 * page, 4 * page + 3, -2, 2 * page + 7]
    n_seq, seq_pages = len(lens), 4
    n_pages = n_seq * seq_pages + 20
    perm = rng.permutation(n_pages).astype(np.int32)
    table = perm[:n_seq * seq_pages].reshape(n_seq, seq_pages).copy()
    table[9, 2] = -1                                          # a begun page that is absent
    parent = np.array([5, 0, 5, 1, 2, 3, 4, 5, 7, 8, -1, n_seq, 9, 2, 4])
    fresh = perm[n_seq * seq_pages:][:len(parent)].copy()
    fresh[7], fresh[13] = -1, n_pages                         # children that go on in the parent's page
    pools, pstride, lay = layers_of(rng, n_layer, n_pages, page, kv, hd, shared)
    bufs = [sa.DevBuf.of(p) for p in pools]
    pg = serving.Pages(*bufs, sa.DevBuf.of(table), n_pages, page, n_seq, seq_pages, kv, hd, **pstride)
    to, ln = sa.DevBuf.of(np.full((len(parent) + 1, seq_pages), -9, np.int32)), sa.DevBuf.of(np.full(len(parent) + 1, -9, np.int32))
    serving.fork(pg, ints(lens), len(parent), ints(parent), ints(fresh), to, ln, **lay)
    sa.sync()
    want = [by_layer(p.copy(), shared, page) for p in pools]
    got, gl = to.read(np.int32).reshape(-1, seq_pages), ln.read(np.int32)
    for i, b in enumerate(parent):
        n = min(max(lens[b], 0), seq_pages * page) if 0 <= b < n_seq else 0
        full, part = divmod(n, page)
        row = [table[b, p] for p in range(full)] if n else []
        if part:
            f = 0 <= fresh[i] < n_pages
            row.append(fresh[i] if f else table[b, full])
            if f and table[b, full] >= 0:
                for w in want:
                    w[:, fresh[i], :part] = w[:, table[b, full], :part]
        assert got[i].tolist() == row + [-1] * (seq_pages - len(row)), i
        assert gl[i] == n
    assert (got[-1] == -9).all() and gl[-1] == -9
    for w, buf, p in zip(want, bufs, pools):
        np.testing.assert_array_equal(by_layer(buf.read(np.uint16).reshape(p.shape), shared, page), w)


@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("n_layer, kv, hd, page", [(1, 2, 128, 16), (5, 3, 64, 64), (16, 8, 128, 16)])
@pytest.mark.parametrize("n_move, named", [(1, True), (17, True), (30, False)])
def test_compact(shared, n_layer, kv, hd, page, n_move, named):
    rng = np.random.default_rng(n_move)
    n_seq, seq_pages, n_pages = 7, 9, 70
    perm = rng.permutation(n_pages)
    src, dst = np.sort(perm[:n_move]), perm[n_move:2 * n_move].copy()
    table = rng.choice(np.concatenate([np.setdiff1d(np.arange(n_pages), dst), [-1, n_pages, 1 << 30, -7]]), (n_seq, seq_pages)).astype(np.int32)
    table[0, 0] = table[1, 3] = table[6, 8] = src[0]          # a page that several share
    if n_move > 2:
        dst[2] = n_pages                                      # no page: it stays
    pools, pstride, lay = layers_of(rng, n_layer, n_pages, page, kv, hd, shared)
    bufs, tb = [sa.DevBuf.of(p) for p in pools], sa.DevBuf.of(table)
    pg = serving.Pages(*bufs, tb, n_pages, page, n_seq, seq_pages, kv, hd, **pstride)
    serving.compact(pg, n_move, ints(src), ints(dst), table=tb if named else None, **lay)
    sa.sync()
    want, to = [by_layer(p.copy(), shared, page) for p in pools], {}
    for s, d in zip(src, dst):
        if d < n_pages:
            to[s] = d
            for w in want:
                w[:, d] = w[:, s]
    renamed = np.array([[to.get(x, x) for x in row] for row in table]) if named else table
    np.testing.assert_array_equal(tb.read(np.int32).reshape(table.shape), renamed)
    for w, buf, p in zip(want, bufs, pools):
        np.testing.assert_array_equal(by_layer(buf.read(np.uint16).reshape(p.shape), shared, page), w)
