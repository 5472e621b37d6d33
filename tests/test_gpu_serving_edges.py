"""The operators of a step of many requests at the edges of what their header
allows, against the 64-bit forms of serving_oracle.py."""
import ctypes
import os
import subprocess
import sys

import numpy as np
import pytest

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
    off = int((~(np.abs(got.astype(np.float64) - want) <= tol)).sum())
    assert off == 0, f"{what}: {off} of {got.size} off"


# ------------------------------------------------------------ attention

def attend(q, k, v, dtype, scale=0.0):
    """One sequence of all rows k, v [n][kv][hd] (16-bit), pages of 16."""
    (heads, hd), (n, kv, _) = q.shape, k.shape
    pages = -(-n // 16)
    pad = np.zeros((16 * pages - n, kv, hd), np.uint16)
    pg = serving.Pages(*(sa.DevBuf.of(np.concatenate([x, pad])) for x in (k, v)), ints(range(pages)), pages, 16, 1, pages,
                       kv, hd, dtype)
    out, part = sa.DevBuf(4 * heads * hd), sa.DevBuf(4 * serving.part_floats(1, heads, hd, n))
    serving.attention(pg, sa.DevBuf.of(q.astype(np.float32)), ints([n]), n, heads, part, out, scale=scale)
    return out.read(np.float32).reshape(heads, hd)


def check_attend(q, k, v, dtype, scale=0.0):
    q = q.astype(np.float32)
    got = attend(q, k, v, dtype, scale)
    heads, kv, hd = len(q), k.shape[1], q.shape[1]
    g = heads // kv
    for h in range(kv):
        want, tol = so.attend(q[h * g:(h + 1) * g], so.from_bits(k[:, h], dtype), so.from_bits(v[:, h], dtype), scale or hd ** -0.5)
        within(got[h * g:(h + 1) * g], want, tol, f"kv head {h}")


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n", [1, 40, 900])
@pytest.mark.parametrize("k_exp, q_exp, v_exp", [(118, -114, 0), (120, -118, 118), (0, 0, 120), (-100, 101, 119), (-110, 111, -100)])
def test_bf16_range(hd, n, k_exp, q_exp, v_exp):
    """bfloat16 keys, values and queries near fp32's largest and smallest."""
    rng = np.random.default_rng(n + hd)
    k, v = (so.to_bits(np.clip(rng.standard_normal((n, 2, hd)), -3, 3) * 2.0 ** e, "bf16") for e in (k_exp, v_exp))
    check_attend(np.clip(rng.standard_normal((8, hd)), -3, 3) * 2.0 ** q_exp, k, v, "bf16")


def test_bf16_largest_values():
    """The largest finite value of the cache comes back; the largest query
    meets keys that bring it down."""
    k = np.zeros((1, 1, 64), np.uint16)
    v = np.full((1, 1, 64), 0x7F7F, np.uint16)
    v[..., 1::2] = 0xFF7F
    q = np.zeros((4, 64))
    check_attend(q, k, v, "bf16")
    rng = np.random.default_rng(1)
    n = 300
    k = np.zeros((n, 1, 64))
    k[..., 0], k[..., 9] = rng.choice([-1, 1], (2, n, 1)) * rng.uniform(0.5, 1, (2, n, 1)) * 2.0 ** -121
    q[:, 0] = [3.4028234e38, -3.4028234e38, 3.39e38, 3e38]
    q[2, 9] = -3.4028234e38
    check_attend(q, so.to_bits(k, "bf16"), so.to_bits(rng.standard_normal((n, 1, 64)), "bf16"), "bf16", scale=0.02)


def test_bf16_rising_scores_of_large_values():
    """Scores that rise by more than the weights' base leaves room, again and
    again, over values that leave the sums none."""
    n, hd = 900, 64
    k = np.zeros((n, 1, hd))
    k[:, 0, 0] = np.arange(n)
    rng = np.random.default_rng(2)
    q = np.zeros((4, hd))
    q[:, 0] = [0.5, -0.5, 2.0, 0.01]
    check_attend(q, so.to_bits(k, "bf16"), so.to_bits(rng.uniform(-1, 1, (n, 1, hd)) * 2.0 ** 118, "bf16"), "bf16", scale=1.0)


@pytest.mark.parametrize("v_exp", [-116, -122, -125])
def test_bf16_smallest_values(v_exp):
    """Values of one sign and near fp32's smallest normal ones, of 40 keys: the
    weights' and sums' errors (so.attend's), and those of sums that lie in
    fp32's denormals, 2^-149 in each of at most 3 parts x 2 tiles x 2 halves and
    4 waves, for weights from 2^-4."""
    rng = np.random.default_rng(6)
    k = so.to_bits(rng.standard_normal((40, 1, 64)), "bf16")
    v = so.to_bits(rng.uniform(1, 2, (40, 1, 64)) * 2.0 ** v_exp, "bf16")
    q = rng.standard_normal((4, 64)).astype(np.float32)
    want, _ = so.attend(q, so.from_bits(k[:, 0], "bf16"), so.from_bits(v[:, 0], "bf16"), 0.125)
    size = np.abs(q.astype(np.float64)) @ np.abs(so.from_bits(k[:, 0], "bf16")).T * 0.125
    rel = 2 * 88 * so.U * size.max() + (2 * 40 + 32) * so.U
    within(attend(q, k, v, "bf16"), want, rel * np.abs(want) + 48 * 2.0 ** (4 - 149))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_infinite_queries_stay_in_their_heads(dtype):
    rng = np.random.default_rng(3)
    k, v = (so.to_bits(rng.standard_normal((700, 2, 64)), dtype) for _ in range(2))
    q = rng.standard_normal((8, 64)).astype(np.float32)
    clean = attend(q, k, v, dtype)
    q[1, 5], q[6, 0], q[3, 63] = np.inf, -np.inf, np.nan
    got = attend(q, k, v, dtype)
    np.testing.assert_array_equal(got[[0, 2, 4, 5, 7]], clean[[0, 2, 4, 5, 7]])
    assert np.isnan(got[[1, 3, 6]]).all()


def test_as_many_sequences_as_there_may_be():
    """65535 sequences that share their pages: outputs follow from the lengths alone."""
    rng = np.random.default_rng(7)
    n, hd, page, pages, top = 65535, 64, 64, 10, 620
    k, v = (so.to_bits(rng.standard_normal((pages, page, 1, hd)), "f16") for _ in range(2))
    lens = rng.integers(0, 4, n)
    lens[[0, 1, 40000, n - 1]] = [600, 513, 620, 128]
    table = ints(np.tile(rng.permutation(pages), (n, 1)))
    pg = serving.Pages(sa.DevBuf.of(k), sa.DevBuf.of(v), table, pages, page, n, pages, 1, hd)
    q = rng.standard_normal(hd).astype(np.float32)
    out, part = sa.DevBuf.of(np.full((n, hd), np.nan, np.float32)), sa.DevBuf(4 * serving.part_floats(n, 1, hd, top))
    serving.attention(pg, sa.DevBuf.of(np.tile(q, (n, 1))), ints(lens), top, 1, part, out)
    got = out.read(np.float32).reshape(n, hd)
    first = table.read(np.int32, pages)
    kk, vv = (so.from_bits(w[first], "f16").reshape(-1, hd) for w in (k, v))
    for m in np.unique(lens):
        want, tol = so.attend(q[None], kk[:m], vv[:m], hd ** -0.5)
        within(got[lens == m], np.repeat(want, (lens == m).sum(), 0), np.repeat(tol, (lens == m).sum(), 0), f"length {m}")


# ------------------------------------------------------------ append

class At:
    def __init__(self, p):
        self.ptr = p


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("in_place", [False, True])
def test_append_among_other_layers_turns_q(dtype, hd, in_place):
    """The rotated q, and the cache, of the middle of three layers in one pool."""
    rng = np.random.default_rng(hd)
    H, KV, page, layers, rows = 6, 2, 32, 3, 50
    size = page * KV * hd
    cos, sin = so.rope_tables(hd // 2, 128)
    pools = [sa.DevBuf.of(np.full(4 * layers * size, 0x1234, np.uint16)) for _ in range(2)]
    table = np.array([[2, 0, 3, 1]], np.int32)
    pg = serving.Pages(*(At(b.ptr + 2 * size) for b in pools), sa.DevBuf.of(table), 4, page, 1, 4, KV, hd, dtype,
                       page_stride=layers * size)
    qkv = rng.standard_normal((rows, H + 2 * KV, hd)).astype(np.float32)
    pos = rng.permutation(128)[:rows]
    buf, qo = sa.DevBuf.of(qkv), sa.DevBuf.of(np.full(rows * H * hd, np.nan, np.float32))
    serving.append(pg, buf, rows, ints(pos), sa.DevBuf.of(cos), sa.DevBuf.of(sin), 128, H, seq=ints([0] * rows),
                   q_out=None if in_place else qo)
    after = buf.read(np.float32).reshape(qkv.shape)
    want, size_of = so.rotate(qkv[:, :H + KV], cos[pos][:, None], sin[pos][:, None])
    within(after[:, :H] if in_place else qo.read(np.float32).reshape(rows, H, hd), want[:, :H], 2 * so.U * size_of[:, :H], "q")
    np.testing.assert_array_equal(after[:, H if in_place else 0:], qkv[:, H if in_place else 0:])
    ks, vs = (b.read(np.uint16).reshape(4, layers, page, KV, hd) for b in pools)
    place = (table[0, pos // page], 1, pos % page)
    rot, mag = want[:, H:], size_of[:, H:]
    within(so.from_bits(ks[place], dtype), rot, so.HALF[dtype] * (np.abs(rot) + 2 * so.U * mag) + 2 * so.U * mag + 2.0 ** -25, "k")
    np.testing.assert_array_equal(vs[place], so.to_bits(qkv[:, H + KV:], dtype))
    for x in (ks, vs):
        x[place] = 0x1234
        assert (x == 0x1234).all()


def test_append_twice_to_one_place():
    """Rows that share a place, by their positions or by a shared page, leave
    one's value in each of its places, and touch no other."""
    rng = np.random.default_rng(4)
    KV, hd, page, rows = 2, 128, 16, 64
    kb, vb = (sa.DevBuf.of(np.full(2 * page * KV * hd, 0x1234, np.uint16)) for _ in range(2))
    pg = serving.Pages(kb, vb, ints([[1], [1]]), 2, page, 2, 1, KV, hd)
    cos, sin = (sa.DevBuf.of(np.full((page, hd // 2), f, np.float32)) for f in (1.0, 0.0))
    qkv = rng.standard_normal((rows, 1 + 2 * KV, hd)).astype(np.float32)
    qo = sa.DevBuf(4 * rows * hd)
    serving.append(pg, sa.DevBuf.of(qkv), rows, ints([7] * rows), cos, sin, page, 1, seq=ints(np.arange(rows) % 2), q_out=qo)
    np.testing.assert_array_equal(qo.read(np.float32).reshape(rows, hd), qkv[:, 0])
    for buf, first in ((kb, 1), (vb, 1 + KV)):
        got = buf.read(np.uint16).reshape(2, page, KV, hd)
        bits = so.to_bits(qkv[:, first:first + KV], "f16")
        assert (got[1, 7] == bits).any(axis=0).all()
        got[1, 7] = 0x1234
        assert (got == 0x1234).all()


# ------------------------------------------------------------ adapters

def lora(n, n_in, n_out, rank, A, dtype, ids, x, base=None, in_place=False, a=None, b=None, y_pad=0):
    rng = np.random.default_rng(5)
    if a is None:
        a, b = (so.to_bits(rng.standard_normal(s), dtype) for s in ((A, rank, n_in), (A, n_out, rank)))
    bb = sa.DevBuf.of(base) if base is not None else None
    y = bb if in_place else sa.DevBuf.of(np.full((n, n_out + y_pad), 9.0, np.float32))
    work = sa.DevBuf.of(np.full(serving.lora_work_floats(rank, n), np.nan, np.float32))
    ad = serving.Adapters(sa.DevBuf.of(a), sa.DevBuf.of(b), A, rank, n_in, n_out, dtype)
    serving.lora(ad, sa.DevBuf.of(x), n, ints(ids), y, work, base=bb, y_stride=n_out + y_pad)
    return y.read(np.float32).reshape(n, n_out + y_pad), a, b


FORMS = [(8, 256, 70, 16, 4), (16, 520, 301, 64, 16), (20, 256, 70, 16, 3), (100, 256, 70, 16, 9), (130, 1032, 66, 64, 3),
         (300, 264, 131, 256, 4), (600, 264, 67, 24, 5)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("n, n_in, n_out, rank, A", [(65, 1544, 300, 64, 16), (80, 520, 1030, 136, 80), (256, 1032, 301, 32, 33),
                                                     (257, 264, 1500, 256, 16), (500, 520, 517, 200, 9), (513, 72, 600, 256, 40)])
def test_adapters_shared_out(n, n_in, n_out, rank, A, dtype):
    """Mixed batches whose tiles' adapters several workgroups share, as many as
    the LDS of either product's tiles lets run at once."""
    rng = np.random.default_rng(n)
    x, base = rng.standard_normal((n, n_in)).astype(np.float32), rng.standard_normal((n, n_out)).astype(np.float32)
    for ids in (rng.integers(-1, A, n), np.arange(n) % A, np.arange(n) * A // n):
        got, a, b = lora(n, n_in, n_out, rank, A, dtype, ids, x, base)
        want, tol = so.lora(x, base, so.from_bits(a, dtype), so.from_bits(b, dtype), np.ones(A, np.float32), [rank] * A, ids)
        within(got, want, tol)


@pytest.mark.parametrize("n, n_in, n_out, rank, A", FORMS)
def test_bf16_adapters_of_the_largest_inputs(n, n_in, n_out, rank, A):
    """The largest finite inputs, and the same as the first product's results,
    with a second matrix that brings them down."""
    rng = np.random.default_rng(n)
    x = np.zeros((n, n_in), np.float32)
    x[np.arange(n), rng.integers(0, n_in, n)] = rng.choice([3.4028234e38, -3.4028234e38, 3.395e38, 2.0 ** 127], n)
    a = so.to_bits(rng.choice([-1, 1, 2.0 ** -20], (A, rank, n_in)), "bf16")
    b = so.to_bits(rng.choice([-1, 1], (A, n_out, rank)) * rng.uniform(0.5, 1, (A, n_out, rank)) * 2.0 ** -118, "bf16")
    ids = rng.integers(-1, A, n)
    got, _, _ = lora(n, n_in, n_out, rank, A, "bf16", ids, x, a=a, b=b)
    want, tol = so.lora(x, np.zeros((n, n_out)), so.from_bits(a, "bf16"), so.from_bits(b, "bf16"), np.ones(A, np.float32),
                        [rank] * A, ids)
    within(got, want, tol)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("n, n_in, n_out, rank, A", FORMS)
def test_infinite_rows_and_adapters_stay_their_own(n, n_in, n_out, rank, A, dtype):
    """One launch and two, sorted tiles and not: a row with an infinity or a
    NaN, and an adapter with them, reach no other row."""
    rng = np.random.default_rng(n)
    a, b = (so.to_bits(rng.standard_normal(s), dtype) for s in ((A, rank, n_in), (A, n_out, rank)))
    a[1, 3, 5], b[1, 6, 2] = (0x7C00, 0x7E00) if dtype == "f16" else (0x7F80, 0x7FC0)
    x = rng.standard_normal((n, n_in)).astype(np.float32)
    x[4, 7], x[6, 9] = np.inf, np.nan
    ids = rng.integers(-1, A, n)
    ids[4], ids[6] = 0, 2
    ids[7] = 1
    got, _, _ = lora(n, n_in, n_out, rank, A, dtype, ids, x, a=a, b=b)
    clean = [r for r in range(n) if ids[r] != 1 and r not in (4, 6)]
    want, tol = so.lora(x[clean], np.zeros((len(clean), n_out)), so.from_bits(a, dtype), so.from_bits(b, dtype),
                        np.ones(A, np.float32), [rank] * A, ids[clean])
    within(got[clean], want, tol)
    assert not np.isfinite(got[4]).any() and np.isnan(got[6]).all()
    assert not np.isfinite(got[ids == 1]).any()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("n, n_in, n_out, rank, A", FORMS)
@pytest.mark.parametrize("in_place", [False, True])
def test_rows_without_an_adapter_keep_their_bits(n, n_in, n_out, rank, A, dtype, in_place):
    """Zeros of either sign, infinities and NaN of the base come back as they
    are, in the outputs past the last four too."""
    rng = np.random.default_rng(n)
    x = rng.standard_normal((n, n_in)).astype(np.float32)
    base = np.where(rng.random((n, n_out + 3)) < 0.5, -0.0, 1.5).astype(np.float32)
    base[:, 3], base[:, 5], base[:, 6] = np.nan, np.inf, -np.inf
    base[:, -4:] = -0.0
    for ids in (rng.integers(-1, A, n), np.where(np.arange(n) % 5 == 0, 1, -1), np.full(n, A)):
        got, _, _ = lora(n, n_in, n_out, rank, A, dtype, ids, x, base, in_place, y_pad=3)
        none = (ids < 0) | (ids >= A)
        np.testing.assert_array_equal(got[none, :n_out].view(np.uint32), base[none, :n_out].view(np.uint32))


@pytest.mark.parametrize("n, n_in, n_out, rank, A", FORMS)
def test_zeros_do_not_depend_on_other_rows(n, n_in, n_out, rank, A):
    """A row whose product is zero has the same bits, signs of zeros too,
    whatever adapters the others have."""
    rng = np.random.default_rng(n)
    x = rng.standard_normal((n, n_in)).astype(np.float32)
    x[::3] = 0.0
    base = np.full((n, n_out), -0.0, np.float32)
    seen = []
    for _ in range(3):
        ids = rng.integers(-1, A, n)
        ids[::3] = np.arange(len(ids[::3])) % A
        seen.append(lora(n, n_in, n_out, rank, A, "f16", ids, x, base)[0][::3].view(np.uint32))
    np.testing.assert_array_equal(seen[0], seen[1])
    np.testing.assert_array_equal(seen[0], seen[2])


def test_as_many_rows_as_there_may_be():
    """65535 rows of adapters and of logits."""
    rng = np.random.default_rng(9)
    n, n_in, n_out, rank, A = 65535, 16, 9, 8, 3
    x, base = rng.standard_normal((n, n_in)).astype(np.float32), rng.standard_normal((n, n_out)).astype(np.float32)
    ids = rng.integers(-1, A, n)
    got, a, b = lora(n, n_in, n_out, rank, A, "f16", ids, x, base)
    want, tol = so.lora(x, base, so.from_bits(a, "f16"), so.from_bits(b, "f16"), np.ones(A, np.float32), [rank] * A, ids)
    within(got, want, tol)
    logits = rng.integers(-9, 9, (n, n_out)).astype(np.float32)
    out, tok, part = sa.DevBuf(4 * n * n_out), sa.DevBuf(4 * n), sa.DevBuf(serving.logits_part_bytes(n, n_out))
    mask = np.array([0b101010101, 0b000110000], np.uint32)
    which = rng.integers(-1, 3, n)
    serving.adjust_logits(sa.DevBuf.of(logits), n, n_out, out=out, tok=tok, part=part, mask=sa.DevBuf.of(mask), n_mask=2,
                          mask_row=ints(which))
    ok = np.array([mask[0] >> np.arange(n_out) & 1, mask[1] >> np.arange(n_out) & 1, 0 * np.arange(n_out), 0 * np.arange(n_out) + 1]) > 0
    want = np.where(ok[which], logits, -np.inf)
    np.testing.assert_array_equal(out.read(np.float32).reshape(n, n_out), want)
    np.testing.assert_array_equal(tok.read(np.int32), np.where(which == 2, -1, want.argmax(1)))


# ------------------------------------------------------------ beside the products

class Hip:
    """Streams and events of the runtime the library already runs on."""

    def __init__(self):
        sa.lib()
        self.l = ctypes.CDLL("libamdhip64.so")
        self.stream, self.events = ctypes.c_void_p(), [ctypes.c_void_p(), ctypes.c_void_p()]
        self("hipStreamCreateWithFlags", ctypes.byref(self.stream), 1)      # not ordered with the null stream
        for e in self.events:
            self("hipEventCreateWithFlags", ctypes.byref(e), 2)             # no timing

    def __call__(self, name, *args):
        assert getattr(self.l, name)(*args) == 0, name

    def after_null(self):
        """What is enqueued on the stream from here on follows the null stream's work so far."""
        self("hipEventRecord", self.events[0], None)
        self("hipStreamWaitEvent", self.stream, self.events[0], 0)

    def before_null(self):
        self("hipEventRecord", self.events[1], self.stream)
        self("hipStreamWaitEvent", None, self.events[1], 0)


def test_products_and_operators_on_two_streams(tmpdir_s):
    """The documented order of a layer: the shared product on the null stream,
    its adapters, the append and the attention on a stream that does not wait
    for it by itself, the next product after them. Several layers in a row,
    unsynchronized, equal the same calls on the null stream."""
    rng = np.random.default_rng(8)
    n, E, H, KV, hd, page, pages, rank, A, layers = 9, 512, 8, 2, 64, 16, 4, 16, 3, 4
    W = (H + 2 * KV) * hd
    p = tmpdir_s / "serving_streams.ssf"
    sa.synth_matrix(p, W, E, nbits=4, seed=3)
    m = sa.Mat.from_file(p, "w")
    x = rng.standard_normal((n, E)).astype(np.float32)
    act = sa.Act(E * n)
    for r in range(n):
        one = sa.Act(E)
        sa.normq(sa.DevBuf.of(x[r]), one)
        for buf, w, sz in zip((act.q, act.scale, act.sums), one.read(), (E, E // 8, E // 8)):
            sa._chk(sa.lib().sml_hip_h2d(buf.ptr + r * sz, w.ctypes.data, w.nbytes))
    a, b = (so.to_bits(rng.standard_normal(s), "f16") for s in ((A, rank, E), (A, W, rank)))
    ad = serving.Adapters(sa.DevBuf.of(a), sa.DevBuf.of(b), A, rank, E, W)
    cos, sin = (sa.DevBuf.of(t) for t in so.rope_tables(hd // 2, page * pages))
    pos, ids = rng.integers(0, page * pages, n), ints(rng.integers(-1, A, n))
    table, pos_b, len_b = ints(rng.permutation(n * pages).reshape(n, pages)), ints(pos), ints(pos + 1)
    xb, hip = sa.DevBuf.of(x), Hip()
    first = [so.to_bits(rng.standard_normal((n * pages, page, KV, hd)), "f16") for _ in range(2)]

    def run(stream):
        kv = [[sa.DevBuf.of(w) for w in first] for _ in range(layers)]
        qkv, q, out = sa.DevBuf(4 * n * W), sa.DevBuf(4 * n * H * hd), [sa.DevBuf(4 * n * H * hd) for _ in range(layers)]
        part = sa.DevBuf(4 * serving.part_floats(n, H, hd, page * pages))
        work = sa.DevBuf(4 * serving.lora_work_floats(rank, n))
        sa.sync()
        for layer in range(layers):
            sa.gemm(m, act.q, act.scale, act.sums, n, qkv)
            if stream:
                hip.after_null()
            serving.lora(ad, xb, n, ids, qkv, work, base=qkv, stream=stream)
            pg = serving.Pages(*kv[layer], table, n * pages, page, n, pages, KV, hd)
            serving.append(pg, qkv, n, pos_b, cos, sin, page * pages, H, q_out=q, stream=stream)
            serving.attention(pg, q, len_b, page * pages, H, part, out[layer], stream=stream)
            if stream:
                hip.before_null()
        sa.sync()
        return [o.read(np.uint32) for o in out] + [w.read(np.uint16) for pair in kv for w in pair]

    want = run(0)
    for _ in range(3):
        for got, w in zip(run(hip.stream.value), want):
            np.testing.assert_array_equal(got, w)


FIRST = """
import sys
sys.path[:0] = sys.argv[1:]
import numpy as np
import sheep_amd as sa
import test_gpu_serving as t
sa.init(0)
s = t.step_state(1)
d, hip = t.step_buffers(s), t.Hip()
sa.sync()
ex = hip.capture(lambda: t.step_run(s, d, hip.stream.value))
for _ in range(2):
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
    """Nothing but sml_hip_init has to run before a capture."""
    here = os.path.dirname(os.path.abspath(__file__))
    r = subprocess.run([sys.executable, "-c", FIRST, os.path.dirname(here), here], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and r.stdout.strip().endswith("equal"), r.stdout + r.stderr
