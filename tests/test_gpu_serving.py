"""The operators of a step of many requests against their plain 64-bit forms
(serving_oracle.py, which also derives how far fp32 may be off)."""
import ctypes

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
    err = np.abs(got.astype(np.float64) - want)
    bad = ~(err <= tol)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, at {np.argwhere(bad)[0]}: " \
        f"{got[tuple(np.argwhere(bad)[0])]} for {want[tuple(np.argwhere(bad)[0])]}, worst {np.nanmax(err / np.maximum(tol, 1e-300)):.3g} of the bound"


# ------------------------------------------------------------ append

def make_table(rng, n_seq, seq_pages, n_pages):
    """Scattered distinct pages for every entry."""
    return rng.permutation(n_pages)[:n_seq * seq_pages].reshape(n_seq, seq_pages).astype(np.int32)


@pytest.mark.parametrize("heads, kv, hd, dtype, page", [
    (32, 8, 128, "f16", 16), (12, 2, 128, "bf16", 64), (14, 2, 64, "f16", 32), (3, 3, 64, "bf16", 16),
    (16, 1, 128, "f16", 128)])
@pytest.mark.parametrize("rows, in_place, pad", [(1, False, 0), (37, True, 12), (130, False, 4)])
def test_append(heads, kv, hd, dtype, page, rows, in_place, pad):
    rng = np.random.default_rng(rows + heads + page)
    n_seq, seq_pages, n_rope = 5, 4, 4 * page - 3          # the last positions have no angles
    n_pages = n_seq * seq_pages + 3
    table = make_table(rng, n_seq, seq_pages, n_pages)
    table[1, 2], table[2, 0], table[3, 1] = -1, n_pages, -7     # no pages
    width = (heads + 2 * kv) * hd
    stride = width + pad
    qkv = rng.standard_normal((rows, stride)).astype(np.float32)
    # distinct places, then padding and rows that lie outside
    places = rng.permutation(n_seq * seq_pages * page)[:rows]
    seq, pos = places // (seq_pages * page), places % (seq_pages * page)
    if rows > 8:
        pos[3], pos[4], pos[5], seq[6], seq[7] = -1, n_rope, seq_pages * page, n_seq, -1
    cos, sin = so.rope_tables(hd // 2, n_rope)
    size = n_pages * page * kv * hd
    was = [rng.integers(0, 1 << 16, size).astype(np.uint16) for _ in range(2)]
    kb, vb = sa.DevBuf.of(was[0]), sa.DevBuf.of(was[1])
    pg = serving.Pages(kb, vb, sa.DevBuf.of(table), n_pages, page, n_seq, seq_pages, kv, hd, dtype)
    qb, qo = sa.DevBuf.of(qkv), sa.DevBuf.of(np.full((rows, heads * hd), 7.5, np.float32))
    serving.append(pg, qb, rows, ints(pos), sa.DevBuf.of(cos), sa.DevBuf.of(sin), n_rope, heads, seq=ints(seq),
                   q_out=None if in_place else qo, qkv_stride=stride if pad else 0)
    sa.sync()
    k, v = (w.copy().reshape(n_pages, page, kv, hd) for w in was)
    after = qb.read(np.float32).reshape(rows, stride)
    q = after[:, :heads * hd] if in_place else qo.read(np.float32).reshape(rows, heads * hd)
    want_q = (qkv[:, :heads * hd] if in_place else np.full((rows, heads * hd), 7.5)).astype(np.float64)
    tol_q = np.zeros_like(want_q)
    got_k, got_v = kb.read(np.uint16).reshape(k.shape), vb.read(np.uint16).reshape(v.shape)
    near = []
    for r in range(rows):
        if not (0 <= pos[r] < n_rope and pos[r] < seq_pages * page and 0 <= seq[r] < n_seq):
            continue
        pid = table[seq[r], pos[r] // page]
        if not 0 <= pid < n_pages:
            continue
        x = qkv[r, :width].reshape(-1, hd)
        rot, mag = so.rotate(x[:heads + kv], cos[pos[r]], sin[pos[r]])
        want_q[r] = rot[:heads].reshape(-1)
        tol_q[r] = 2 * so.U * mag[:heads].reshape(-1)          # a product's rounding and the sum's
        v[pid, pos[r] % page] = so.to_bits(x[heads + kv:], dtype)
        at = (pid, pos[r] % page)
        near.append((so.from_bits(got_k[at], dtype), rot[heads:], mag[heads:]))
        k[at] = got_k[at]                                      # compared by value below
    within(q, want_q, tol_q, "q")
    for got, rot, mag in near:
        # fp32's roundings, then half a step of the type (2^-25: fp16's denormals)
        within(got, rot, so.HALF[dtype] * (np.abs(rot) + 2 * so.U * mag) + 2 * so.U * mag + 2.0 ** -25, "k")
    np.testing.assert_array_equal(got_v, v)
    np.testing.assert_array_equal(got_k, k)                   # every other place as it was
    if not in_place:
        np.testing.assert_array_equal(after, qkv)
    else:
        np.testing.assert_array_equal(after[:, heads * hd:], qkv[:, heads * hd:])


def test_append_no_rows():
    pg = serving.Pages(sa.DevBuf(8192), sa.DevBuf(8192), ints([0]), 1, 16, 1, 1, 1, 128)
    b = sa.DevBuf(4096)
    serving.append(pg, b, 0, b, b, b, 1, 1)
    sa.sync()


@pytest.mark.parametrize("hd", [128, 64])
def test_append_equals_the_contiguous_cache(hd):
    """An fp16 paged cache holds the bits sml_hip_attention writes, and q is
    rotated alike in a row of the table shared by layers."""
    rng = np.random.default_rng(hd)
    H, KV, n_ctx, page, layers = 8, 2, 128, 32, 3
    cos, sin = so.rope_tables(hd // 2, n_ctx)
    cb, sb = sa.DevBuf.of(cos), sa.DevBuf.of(sin)
    kc, vc = (sa.DevBuf.of(np.zeros(n_ctx * KV * hd, np.uint16)) for _ in range(2))
    part = sa.DevBuf(4 * sa.lib().sml_hip_attn_part_floats(H, hd, n_ctx))
    # the middle layer of pages that three layers share
    size = page * KV * hd
    pools = [sa.DevBuf.of(np.full(4 * layers * size, 0x1234, np.uint16)) for _ in range(2)]

    class At:
        def __init__(self, p):
            self.ptr = p
    mid = [At(b.ptr + 2 * size) for b in pools]
    table = np.array([[2, 0, 3, 1]], np.int32)
    pg = serving.Pages(mid[0], mid[1], sa.DevBuf.of(table), 4, page, 1, 4, KV, hd, page_stride=layers * size)
    out, qo = sa.DevBuf(4 * H * hd), sa.DevBuf(4 * H * hd)
    for p in range(0, 128, 9):
        qkv = rng.standard_normal((H + 2 * KV) * hd).astype(np.float32)
        a, b = sa.DevBuf.of(qkv), sa.DevBuf.of(qkv)
        at = [a.ptr, a.ptr + 4 * H * hd, a.ptr + 4 * (H + KV) * hd]
        assert sa.lib().sml_hip_attention(*at, kc.ptr, vc.ptr, cb.ptr, sb.ptr, ints([p]).ptr, H, KV, hd, n_ctx,
                                          part.ptr, out.ptr) == 0
        serving.append(pg, b, 1, ints([p]), cb, sb, n_ctx, H, q_out=qo)
        sa.sync()
    for c, pool in ((kc, pools[0]), (vc, pools[1])):
        flat = c.read(np.uint16).reshape(n_ctx, KV * hd)
        paged = pool.read(np.uint16).reshape(4, layers, page, KV * hd)
        for p in range(0, 128, 9):
            np.testing.assert_array_equal(paged[table[0, p // page], 1, p % page], flat[p])
        assert (paged[:, 0] == 0x1234).all() and (paged[:, 2] == 0x1234).all()


# ------------------------------------------------------------ attention

def attend_case(lens, heads, kv, hd, dtype, page, seed=0, gone=None, scale=0.0, q_size=1.0, pad=0, max_len=None,
                poison=True, spare=3, kv_size=1.0):
    """One call against the oracle. gone: {sequence: absent page entries};
    poison: NaN and infinities everywhere the call must not look."""
    rng = np.random.default_rng(seed)
    n_seq = len(lens)
    seq_pages = max(1, -(-max(lens) // page))
    n_pages = n_seq * seq_pages + spare
    table = make_table(rng, n_seq, seq_pages, n_pages)
    k, v = (kv_size * rng.standard_normal((n_pages, page, kv, hd)).astype(np.float32) for _ in range(2))
    kb, vb = so.to_bits(k, dtype), so.to_bits(v, dtype)
    cut = [max(0, min(n, max_len if max_len is not None else n)) for n in lens]
    keep = np.zeros((n_pages, page), bool)
    for b in range(n_seq):
        for i in (gone or {}).get(b, ()):
            if i < seq_pages:
                table[b, i] = [-1, n_pages, 1 << 30][i % 3]
        for p in range(cut[b]):
            pid = table[b, p // page]
            if 0 <= pid < n_pages:
                keep[pid, p % page] = True
    if poison:
        bad = np.array([0x7E00, 0x7C00, 0xFC00, 0x7FFF] if dtype == "f16" else [0x7FC0, 0x7F80, 0xFF80, 0x7FFF], np.uint16)
        for x in (kb, vb):
            x[~keep] = bad[rng.integers(0, 4, x[~keep].shape)]
    stride = heads * hd + pad
    q = (q_size * rng.standard_normal((n_seq, stride))).astype(np.float32)
    top = max(1, max(lens)) if max_len is None else max_len
    part = sa.DevBuf(4 * max(1, serving.part_floats(n_seq, heads, hd, max(1, top))))
    out = sa.DevBuf.of(np.full(n_seq * heads * hd, np.nan, np.float32))
    pg = serving.Pages(sa.DevBuf.of(kb), sa.DevBuf.of(vb), sa.DevBuf.of(table), n_pages, page, n_seq, seq_pages, kv, hd,
                       dtype)
    serving.attention(pg, sa.DevBuf.of(q), ints(lens), top, heads, part, out, scale=scale, q_stride=stride if pad else 0)
    sa.sync()
    got = out.read(np.float32).reshape(n_seq, heads, hd)
    sc = scale or hd ** -0.5
    g = heads // kv
    for b in range(n_seq):
        live = [(table[b, p // page], p % page) for p in range(cut[b]) if 0 <= table[b, p // page] < n_pages]
        ids = np.array(live, np.int64).reshape(-1, 2)
        for h in range(kv):
            kk, vv = (so.from_bits(x[ids[:, 0], ids[:, 1], h], dtype).reshape(-1, hd) for x in (kb, vb))
            want, tol = so.attend(q[b, :heads * hd].reshape(heads, hd)[h * g:(h + 1) * g], kk, vv, sc)
            within(got[b, h * g:(h + 1) * g], want, tol, f"sequence {b} of {cut[b]}, kv head {h}")


EDGES = [0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 257, 600]


@pytest.mark.parametrize("heads, kv, hd, dtype, page", [
    (32, 8, 128, "f16", 16), (12, 2, 128, "bf16", 64), (32, 8, 64, "f16", 32), (14, 2, 64, "bf16", 16),
    (8, 8, 128, "f16", 128), (3, 1, 128, "bf16", 16), (16, 1, 64, "f16", 16), (26, 2, 128, "f16", 32)])
def test_attention_lengths(heads, kv, hd, dtype, page):
    attend_case(EDGES, heads, kv, hd, dtype, page, seed=heads + page)


@pytest.mark.parametrize("length", [1, 4095, 9001])
@pytest.mark.parametrize("heads, kv, hd, dtype", [(32, 8, 128, "f16"), (4, 1, 64, "bf16")])
def test_attention_one_sequence(length, heads, kv, hd, dtype):
    attend_case([length], heads, kv, hd, dtype, 16, seed=length)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_attention_absent_pages(dtype):
    attend_case([100, 333, 64, 33, 1, 500], 8, 2, 128, dtype, 16, seed=5,
                gone={0: [0, 1, 2], 1: range(0, 40, 2), 2: range(4), 3: [2], 4: [0], 5: list(range(3, 29))})
    attend_case([700, 2100], 4, 1, 64, dtype, 128, seed=6, gone={0: [5], 1: range(1, 16)})


def test_attention_many_sequences():
    """Past 256 sequences the splits have a fixed size; at and below, the
    lengths are shared out, whole waves of them and part of one."""
    rng = np.random.default_rng(12)
    for n, kv, longest in ((300, 1, 900), (256, 1, 200), (65, 2, 400), (64, 1, 300)):
        lens = [int(x) for x in rng.integers(0, longest, n)]
        lens[n // 2], lens[0] = longest, 0
        attend_case(lens, 2 * kv, kv, 64, "f16", 16, seed=n)


def test_attention_loose_bound():
    """A bound far above the lengths, and sequences that differ much."""
    attend_case([1, 3000, 5, 130], 4, 2, 128, "bf16", 32, seed=13)
    rng = np.random.default_rng(14)
    k, v, q = rng.standard_normal((2, 16, 1, 64)), rng.standard_normal((2, 16, 1, 64)), rng.standard_normal((1, 64))
    kb, vb = so.to_bits(k, "f16"), so.to_bits(v, "f16")
    table = np.full((1, 5000), -1, np.int32)
    table[0, :2] = [1, 0]
    pg = serving.Pages(sa.DevBuf.of(kb), sa.DevBuf.of(vb), sa.DevBuf.of(table), 2, 16, 1, 5000, 1, 64)
    out, part = sa.DevBuf(256), sa.DevBuf(4 * serving.part_floats(1, 1, 64, 1 << 30))
    for n in (20, 1 << 30):                                  # absent pages behind the second
        serving.attention(pg, sa.DevBuf.of(q.astype(np.float32)), ints([n]), 1 << 30, 1, part, out)
        rows = min(n, 32)
        want, tol = so.attend(q.astype(np.float32), so.from_bits(kb[[1, 0]], "f16").reshape(32, 64)[:rows],
                              so.from_bits(vb[[1, 0]], "f16").reshape(32, 64)[:rows], 0.125)
        within(out.read(np.float32).reshape(1, 64), want, tol, str(n))


def test_attention_cut_at_max_len():
    attend_case([500, 3, 90], 8, 2, 128, "f16", 32, seed=7, max_len=77)
    attend_case([5, 3], 8, 2, 128, "f16", 32, seed=7, max_len=0)
    attend_case([-3, 40], 8, 2, 128, "f16", 32, seed=8)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("q_size, scale", [(40.0, 0.0), (1e-3, 0.0), (1.0, 0.7), (3e5, 1e-6), (1e-7, 1e6), (1.0, -0.2)])
def test_attention_query_sizes(dtype, q_size, scale):
    attend_case([300, 17], 8, 2, 128, dtype, 16, seed=9, q_size=q_size, scale=scale, pad=4)


@pytest.mark.parametrize("kv_size, q_size", [(3e-6, 1.0), (3e-6, 2e5), (9000.0, 1.0), (9000.0, 1e-4)])
def test_attention_cache_sizes(kv_size, q_size):
    """fp16's denormals and its largest values in the cache."""
    attend_case([200, 700], 8, 2, 128, "f16", 16, seed=15, kv_size=kv_size, q_size=q_size)


def test_attention_weights_of_all_sizes():
    """Scores spread over the exponential's range: the weights run from 1 to
    below fp16's smallest, and the largest come last."""
    rng = np.random.default_rng(16)
    for dtype in ("f16", "bf16"):
        n, hd, page = 900, 64, 32
        k = np.zeros((n, hd))
        k[:, 0] = np.sort(rng.uniform(-12, 12, n))
        kb, vb = so.to_bits(k, dtype), so.to_bits(rng.standard_normal((n, hd)), dtype)
        pools = [sa.DevBuf.of(np.concatenate([b, np.zeros((29 * page - n, hd), np.uint16)])) for b in (kb, vb)]
        pg = serving.Pages(*pools, sa.DevBuf.of(np.arange(29, dtype=np.int32)), 29, page, 1, 29, 1, hd, dtype)
        q = np.zeros((2, hd), np.float32)
        q[0, 0], q[1, 0] = 8.0, -8.0                         # largest last, largest first
        out, part = sa.DevBuf(4 * 2 * hd), sa.DevBuf(4 * serving.part_floats(1, 2, hd, n))
        serving.attention(pg, sa.DevBuf.of(q), ints([n]), n, 2, part, out)
        want, tol = so.attend(q, so.from_bits(kb, dtype), so.from_bits(vb, dtype), 0.125)
        within(out.read(np.float32).reshape(2, hd), want, tol, dtype)


def test_attention_far_pages():
    """Pages whose offset passes 32 bits, in values and in bytes."""
    rng = np.random.default_rng(3)
    stride, hd, page = 1 << 30, 128, 16
    pools = [sa.DevBuf(2 * (4 * stride + page * hd)) for _ in range(2)]
    table = np.array([[4, 1, 3]], np.int32)
    x = [so.to_bits(rng.standard_normal((3 * page, hd)), "f16") for _ in range(2)]
    for b, w in zip(pools, x):
        for i, pid in enumerate(table[0]):
            sa._chk(sa.lib().sml_hip_h2d(b.ptr + 2 * int(pid) * stride, w[i * page:(i + 1) * page].ctypes.data,
                                         2 * page * hd))
    pg = serving.Pages(pools[0], pools[1], sa.DevBuf.of(table), 5, page, 1, 3, 1, hd, page_stride=stride)
    q = rng.standard_normal((4, hd)).astype(np.float32)
    out, part = sa.DevBuf(4 * 4 * hd), sa.DevBuf(4 * serving.part_floats(1, 4, hd, 45))
    serving.attention(pg, sa.DevBuf.of(q), ints([45]), 45, 4, part, out)
    k, v = (so.from_bits(w, "f16")[:45] for w in x)
    want, tol = so.attend(q, k, v, hd ** -0.5)
    within(out.read(np.float32).reshape(4, hd), want, tol)
    # and the append reaches them: position 33 lies in page 3
    qkv = rng.standard_normal((1, 6 * hd)).astype(np.float32)
    one, zero = (sa.DevBuf.of(np.full((48, hd // 2), f, np.float32)) for f in (1.0, 0.0))
    serving.append(pg, sa.DevBuf.of(qkv), 1, ints([33]), one, zero, 48, 4, q_out=out)
    got = np.empty(hd, np.uint16)
    for b, i in zip(pools, (4, 5)):
        sa._chk(sa.lib().sml_hip_d2h(got.ctypes.data, b.ptr + 2 * (3 * stride + hd), 2 * hd))
        np.testing.assert_array_equal(got, so.to_bits(qkv[0, i * hd:(i + 1) * hd], "f16"))


# ------------------------------------------------------------ logits

def logits_case(n_row, V, seed, lens, n_prompt=True, rep=True, presence=True, frequency=True, biases=0, masks=None,
                mask_row=None, stride=0, in_place=False, only_pick=False, special=False, pick=True, dense=False):
    rng = np.random.default_rng(seed)
    ld = stride or V
    x = (3 * rng.standard_normal((n_row, ld))).astype(np.float32)
    if special:
        x[rng.random(x.shape) < 0.2] = np.nan
        x[rng.random(x.shape) < 0.1] = -np.inf
        x[rng.random(x.shape) < 0.05] = 0.0
        x[rng.random(x.shape) < 0.01] = np.inf
        x[0, 0], x[-1, :] = np.nan, np.nan
    start = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    hist = np.minimum(rng.zipf(1.3, start[-1]) - 1, V + 5).astype(np.int32)
    hist[rng.random(len(hist)) < 0.02] = -4                   # ids that are no tokens
    npr = np.array([rng.integers(0, n + 2) for n in lens], np.int32)
    par = [rng.uniform(a, b, n_row).astype(np.float32) for a, b in ((0.7, 1.6), (-0.5, 0.9), (0.0, 0.4))]
    bs = np.arange(n_row + 1, dtype=np.int32) * biases
    bid = rng.integers(-2, V + 2 if V > 8 else V, n_row * biases).astype(np.int32)
    if biases > 2:
        bid[2::biases] = bid[0::biases]                       # an id listed twice
    bv = (2 * rng.standard_normal(n_row * biases)).astype(np.float32)
    words = -(-V // 32)
    mk = None
    if masks:
        mk = rng.integers(0, 1 << 32, (masks, words), dtype=np.uint64).astype(np.uint32)
        if not dense:
            mk &= rng.integers(0, 1 << 32, mk.shape, dtype=np.uint64).astype(np.uint32)
        mk[-1] = 0                                            # the last permits nothing but bits past the row
        if V % 32:
            mk[-1, -1] = np.uint32((0xFFFFFFFF << (V % 32)) & 0xFFFFFFFF)
    d = lambda a: sa.DevBuf.of(a) if a is not None and a.size else None      # noqa: E731
    xb = sa.DevBuf.of(x)
    out = None if only_pick else xb if in_place else sa.DevBuf.of(np.full((n_row, ld), 9.0, np.float32))
    tok = sa.DevBuf.of(np.full(n_row, -9, np.int32)) if pick else None
    part = sa.DevBuf(serving.logits_part_bytes(n_row, V)) if pick else None
    kw = dict(hist=d(hist), n_hist=len(hist), hist_start=d(start), n_prompt=d(npr) if n_prompt else None,
              rep=d(par[0]) if rep else None, presence=d(par[1]) if presence else None,
              frequency=d(par[2]) if frequency else None)
    if biases:
        kw.update(bias_id=d(bid), bias=d(bv), n_bias=len(bid), bias_start=d(bs))
    if masks:
        kw.update(mask=d(mk), n_mask=masks, mask_row=ints(mask_row) if mask_row is not None else None)
    serving.adjust_logits(xb, n_row, V, out=out, tok=tok, part=part, stride=stride, out_stride=stride, **kw)
    sa.sync()
    got = None if out is None else out.read(np.float32).reshape(n_row, ld)
    toks = tok.read(np.int32) if pick else None
    for b in range(n_row):
        permitted = None
        m = (b if mask_row is None else mask_row[b]) if masks else -1
        if masks and m != -1:
            w = mk[m] if 0 <= m < masks else np.zeros(words, np.uint32)
            permitted = ((w[np.arange(V) // 32] >> (np.arange(V) % 32).astype(np.uint32)) & 1).astype(bool)
        want, t = so.adjust(x[b, :V], hist[start[b]:start[b + 1]], int(npr[b]) if n_prompt else 0,
                            par[0][b] if rep else None, par[1][b] if presence else None,
                            par[2][b] if frequency else None,
                            list(zip(bid[bs[b]:bs[b + 1]].tolist(), bv[bs[b]:bs[b + 1]].tolist())) if biases else None,
                            permitted)
        if got is not None:
            np.testing.assert_array_equal(got[b, :V], want, err_msg=f"row {b}")
            if ld > V:
                np.testing.assert_array_equal(got[b, V:], x[b, V:] if in_place else np.float32(9.0))
        if pick:
            assert toks[b] == t, (b, toks[b], t)


@pytest.mark.parametrize("n_row, V, lens", [
    (1, 1, [3]), (1, 31, [0]), (2, 33, [5, 0]), (3, 4096, [70, 1, 9000]), (2, 4097, [0, 0]), (5, 10007, [10, 200, 3, 0, 44]),
    (2, 128256, [4000, 33]), (1, 151936, [20011])])
def test_logits(n_row, V, lens):
    logits_case(n_row, V, V, lens)
    logits_case(n_row, V, V + 1, lens, biases=5, masks=n_row, n_prompt=False)
    logits_case(n_row, V, V + 2, lens, rep=False, frequency=False, stride=V + 3, in_place=True, biases=1)
    logits_case(n_row, V, V + 3, lens, presence=False, only_pick=True, masks=2, mask_row=[-1, 0, 1, 2, -2][:n_row])
    logits_case(n_row, V, V + 4, lens, special=True, masks=2, mask_row=[0, -1, 1, 0, -1][:n_row], stride=V + 1, dense=True)
    logits_case(n_row, V, V + 5, lens, special=True, pick=False)


def test_logits_many_biases():
    logits_case(3, 5000, 1, [10, 0, 400], biases=6000)


def test_pick_equals_argmax():
    """Without rules the pick is sml_hip_argmax's, ties and NaN included."""
    rng = np.random.default_rng(8)
    for n in (1, 7, 8191, 20000):
        x = rng.integers(0, 50, (4, n)).astype(np.float32)
        x[1, rng.random(n) < 0.3] = np.nan
        x[2, 0] = np.nan
        x[3] = -np.inf
        xb, tok, one = sa.DevBuf.of(x), sa.DevBuf(16), sa.DevBuf(4)
        serving.adjust_logits(xb, 4, n, tok=tok, part=sa.DevBuf(serving.logits_part_bytes(4, n)))
        got = tok.read(np.int32)
        for b in range(4):
            assert sa.lib().sml_hip_argmax(xb.ptr + 4 * n * b, n, one.ptr) == 0
            assert got[b] == one.read(np.int32)[0], (n, b)


def test_logits_bad_starts():
    """Starts that run backwards or past the list stay inside it."""
    rng = np.random.default_rng(2)
    V = 300
    x = rng.standard_normal((3, V)).astype(np.float32)
    hist = rng.integers(0, V, 20).astype(np.int32)
    out = sa.DevBuf(4 * 3 * V)
    serving.adjust_logits(sa.DevBuf.of(x), 3, V, out=out, hist=sa.DevBuf.of(hist), n_hist=20,
                          hist_start=ints([-5, 8, 4, 1 << 30]), presence=sa.DevBuf.of(np.ones(3, np.float32)))
    got = out.read(np.float32).reshape(3, V)
    for b, (lo, hi) in enumerate([(0, 8), (8, 4), (4, 20)]):
        want, _ = so.adjust(x[b], hist[lo:hi], 0, None, 1.0, None, None, None)
        np.testing.assert_array_equal(got[b], want)


# ------------------------------------------------------------ adapters

def lora_case(n, n_in, n_out, rank, A, dtype, adapter, seed=0, base=True, in_place=False, x_pad=0, y_pad=0, ranks=None,
              scale=True, poison=True):
    rng = np.random.default_rng(seed)
    a = so.to_bits(rng.standard_normal((A, rank, n_in)) / np.sqrt(n_in), dtype)
    b = so.to_bits(rng.standard_normal((A, n_out, rank)) / np.sqrt(rank), dtype)
    rk = np.full(A, rank) if ranks is None else np.array(ranks)
    if poison:                                                # what lies past an adapter's rank, and a whole unused one
        for i in range(A):
            a[i, max(0, rk[i]):] = 0x7FFF
            b[i, :, max(0, rk[i]):] = 0x7FFF
            if i not in adapter:
                a[i], b[i] = 0x7FFF, 0x7FFF
    sc = rng.uniform(0.25, 2, A).astype(np.float32) if scale else np.ones(A, np.float32)
    x = rng.standard_normal((n, n_in + x_pad)).astype(np.float32)
    y0 = rng.standard_normal((n, n_out + y_pad)).astype(np.float32)
    yb, bb = sa.DevBuf.of(y0), sa.DevBuf.of(y0)
    work = sa.DevBuf.of(np.full(serving.lora_work_floats(rank, n), np.nan, np.float32))
    ad = serving.Adapters(sa.DevBuf.of(a), sa.DevBuf.of(b), A, rank, n_in, n_out, dtype,
                          scale=sa.DevBuf.of(sc) if scale else None, ranks=ints(rk) if ranks is not None else None)
    serving.lora(ad, sa.DevBuf.of(x), n, ints(adapter), yb, work, base=yb if in_place else bb if base else None,
                 x_stride=n_in + x_pad if x_pad else 0, y_stride=n_out + y_pad if y_pad else 0)
    sa.sync()
    got = yb.read(np.float32).reshape(n, n_out + y_pad)
    want, tol = so.lora(x[:, :n_in], y0[:, :n_out] if base or in_place else np.zeros((n, n_out)), so.from_bits(a, dtype),
                        so.from_bits(b, dtype), sc, rk, adapter)
    within(got[:, :n_out], want, tol, f"{n}x{n_in}x{n_out} rank {rank}")
    np.testing.assert_array_equal(got[:, n_out:], y0[:, n_out:])


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("n, n_in, n_out, rank, A", [
    (1, 8, 1, 8, 1), (1, 1536, 8960, 8, 2), (3, 72, 33, 16, 2), (16, 4096, 1000, 16, 11), (17, 520, 257, 24, 3),
    (33, 264, 130, 64, 4), (64, 1024, 515, 40, 5), (1, 12288, 300, 64, 2), (140, 264, 300, 256, 2), (16, 512, 4000, 64, 9), (100, 136, 65, 256, 2), (130, 2048, 64, 8, 1), (5, 14336, 96, 128, 5)])
def test_lora(dtype, n, n_in, n_out, rank, A):
    rng = np.random.default_rng(n)
    mixed = [int(i) for i in rng.integers(-1, A, n)]
    runs = [r * A // n for r in range(n)]
    lora_case(n, n_in, n_out, rank, A, dtype, mixed, seed=n)
    lora_case(n, n_in, n_out, rank, A, dtype, runs, seed=n + 1, base=False, x_pad=3, y_pad=1,
              ranks=[max(0, rank - 5 * i) for i in range(A)])
    lora_case(n, n_in, n_out, rank, A, dtype, mixed, seed=n + 2, in_place=True, scale=False, y_pad=5, x_pad=8)


@pytest.mark.parametrize("n, A, dtype", [(33, 5, "f16"), (64, 16, "bf16"), (200, 16, "f16"), (257, 255, "bf16"),
                                         (512, 40, "f16"), (513, 40, "f16"), (300, 300, "f16"), (510, 3, "bf16")])
def test_lora_mixed_batches(n, A, dtype):
    """Rows of many adapters in no order, in turn, in runs, and mostly without
    one, around the sizes where tiles take them by adapter."""
    rng = np.random.default_rng(n + A)
    mixed = [int(i) for i in rng.integers(-2, A + 2, n)]
    lora_case(n, 64, 70, 8, A, dtype, mixed, seed=1, y_pad=2)
    lora_case(n, 72, 33, 16, A, dtype, [r % A for r in range(n)], seed=2, in_place=True)
    lora_case(n, 64, 40, 24, A, dtype, [r * A // n for r in range(n)], seed=3, base=False)
    lora_case(n, 64, 40, 8, A, dtype, [0 if r == n - 1 else -1 for r in range(n)], seed=4)
    lora_case(n, 64, 40, 72, A, dtype, [int(i) for i in rng.zipf(1.5, n) - 1], seed=5,
              ranks=[int(i) for i in rng.integers(0, 73, A)])


def test_lora_no_adapters():
    """Ids outside the pool add nothing, and no rows are no work."""
    lora_case(7, 64, 40, 8, 2, "f16", [-1, 2, -5, 1 << 30, 5, -1, 99])
    lora_case(7, 64, 40, 8, 2, "f16", [-1, 2, -5, 1 << 30, 5, -1, 99], base=False)
    ad = serving.Adapters(sa.DevBuf(4096), sa.DevBuf(4096), 1, 8, 64, 40)
    b = sa.DevBuf(1024)
    serving.lora(ad, b, 0, b, b, b)
    sa.sync()


def test_lora_rows_do_not_depend_on_others():
    """A row's bits are the same whatever adapters the other rows have."""
    rng = np.random.default_rng(3)
    for n, A in ((12, 5), (30, 5), (150, 9)):
        n_in, n_out, rank = 520, 90, 16
        a, b = (sa.DevBuf.of(so.to_bits(rng.standard_normal(sh), "f16")) for sh in ((A, rank, n_in), (A, n_out, rank)))
        ad = serving.Adapters(a, b, A, rank, n_in, n_out)
        x = rng.standard_normal((n, n_in)).astype(np.float32)
        got = []
        for other in range(3):
            ids = rng.integers(-1, A, n) if other else np.full(n, 2)
            ids[[0, n // 2, n - 1]] = [2, 1, 4]
            xo = x.copy()
            xo[1] *= 10.0 ** other
            y, work = sa.DevBuf(4 * n * n_out), sa.DevBuf(4 * serving.lora_work_floats(rank, n))
            serving.lora(ad, sa.DevBuf.of(xo), n, ints(ids), y, work)
            got.append(y.read(np.uint32).reshape(n, n_out)[[0, n // 2, n - 1]])
        np.testing.assert_array_equal(got[0], got[1])
        np.testing.assert_array_equal(got[0], got[2])


def test_lora_zero_and_low_ranks():
    lora_case(9, 128, 50, 16, 4, "bf16", [0, 1, 2, 3, 0, 1, 2, 3, -1], ranks=[0, 1, 7, 99])
    lora_case(4, 128, 50, 16, 2, "f16", [0, 1, 0, 1], ranks=[-3, 16])


def test_lora_rows_stand_alone():
    """An infinite or NaN row, or an adapter of them, stays its own."""
    rng = np.random.default_rng(1)
    n, n_in, n_out, rank = 20, 256, 70, 16
    a = so.to_bits(rng.standard_normal((3, rank, n_in)), "f16")
    b = so.to_bits(rng.standard_normal((3, n_out, rank)), "f16")
    a[1, 3, 5], b[1, 6, 2] = 0x7C00, 0x7E00
    x = rng.standard_normal((n, n_in)).astype(np.float32)
    x[4, 7], x[5, 9] = np.inf, np.nan
    ids = [r % 3 for r in range(n)]
    y, work = sa.DevBuf(4 * n * n_out), sa.DevBuf(4 * serving.lora_work_floats(rank, n))
    ad = serving.Adapters(sa.DevBuf.of(a), sa.DevBuf.of(b), 3, rank, n_in, n_out)
    serving.lora(ad, sa.DevBuf.of(x), n, ints(ids), y, work)
    got = y.read(np.float32).reshape(n, n_out)
    clean = [r for r in range(n) if ids[r] != 1 and r not in (4, 5)]
    want, tol = so.lora(x[clean], np.zeros((len(clean), n_out)), so.from_bits(a, "f16"), so.from_bits(b, "f16"),
                        np.ones(3, np.float32), [rank] * 3, [ids[r] for r in clean])
    within(got[clean], want, tol)
    assert np.isnan(got[5]).all() and not np.isfinite(got[4]).any()
    assert not np.isfinite(got[[r for r in range(n) if ids[r] == 1]]).any()


# ------------------------------------------------------------ streams and graphs

class Hip:
    """What these tests need of the runtime the library already runs on."""

    def __init__(self):
        sa.lib()
        self.l = ctypes.CDLL("libamdhip64.so")
        self.stream = ctypes.c_void_p()
        self("hipStreamCreateWithFlags", ctypes.byref(self.stream), 1)      # beside the null stream

    def __call__(self, name, *args):
        assert getattr(self.l, name)(*args) == 0, name

    def capture(self, f):
        graph, ex = ctypes.c_void_p(), ctypes.c_void_p()
        self("hipStreamBeginCapture", self.stream, 1)
        try:
            f()
        finally:
            self("hipStreamEndCapture", self.stream, ctypes.byref(graph))
        self("hipGraphInstantiate", ctypes.byref(ex), graph, None, None, ctypes.c_size_t(0))
        return ex

    def replay(self, ex):
        self("hipGraphLaunch", ex, self.stream)
        self("hipStreamSynchronize", self.stream)


def step_state(seed, n=5, H=8, KV=2, hd=128, V=5000, page=16, seq_pages=8):
    """Buffers of a small step of n requests."""
    rng = np.random.default_rng(seed)
    s = dict(n=n, H=H, KV=KV, hd=hd, V=V, page=page, seq_pages=seq_pages, n_in=256, rank=16, A=3)
    n_pages = n * seq_pages
    s["table"] = make_table(rng, n, seq_pages, n_pages)
    s["lens"] = rng.integers(0, seq_pages * page - 8, n).astype(np.int32)
    width = (H + 2 * KV) * hd
    f = lambda *sh: rng.standard_normal(sh).astype(np.float32)              # noqa: E731
    s["k"], s["v"] = (so.to_bits(f(n_pages, page, KV, hd), "f16") for _ in range(2))
    s["x"], s["qkv"], s["logits"] = f(n, s["n_in"]), f(n, width), 3 * f(n, V)
    s["a"], s["b"] = so.to_bits(f(3, 16, 256) / 16, "f16"), so.to_bits(f(3, width, 16) / 4, "f16")
    s["cos"], s["sin"] = so.rope_tables(hd // 2, seq_pages * page)
    s["hist"] = rng.integers(0, V, (n, 40)).astype(np.int32)
    return s


def step_buffers(s):
    """The state on the device."""
    n, H, KV, hd, V = s["n"], s["H"], s["KV"], s["hd"], s["V"]
    d = {k: sa.DevBuf.of(s[k]) for k in ("table", "k", "v", "x", "qkv", "logits", "a", "b", "cos", "sin", "hist")}
    d["pos"], d["len"] = sa.DevBuf.of(s["lens"]), sa.DevBuf.of(s["lens"] + 1)
    d["ids"], d["start"] = ints([0, -1, 2, 1, 0][:n]), ints([40 * b for b in range(n + 1)])
    d["pen"] = sa.DevBuf.of(np.full(n, 1.2, np.float32))
    d["q"], d["out"], d["y"] = sa.DevBuf(4 * n * H * hd), sa.DevBuf(4 * n * H * hd), sa.DevBuf(s["qkv"].nbytes)
    d["part"] = sa.DevBuf(4 * serving.part_floats(n, H, hd, s["seq_pages"] * s["page"]))
    d["work"] = sa.DevBuf(4 * serving.lora_work_floats(16, n))
    d["adj"], d["tok"] = sa.DevBuf(4 * n * V), sa.DevBuf(4 * n)
    d["lpart"] = sa.DevBuf(serving.logits_part_bytes(n, V))
    return d


def step_run(s, d, stream):
    n, H, V = s["n"], s["H"], s["V"]
    pg = serving.Pages(d["k"], d["v"], d["table"], n * s["seq_pages"], s["page"], n, s["seq_pages"], s["KV"], s["hd"])
    ad = serving.Adapters(d["a"], d["b"], 3, 16, s["n_in"], s["qkv"].shape[1])
    serving.lora(ad, d["x"], n, d["ids"], d["y"], d["work"], base=d["qkv"], stream=stream)
    serving.append(pg, d["y"], n, d["pos"], d["cos"], d["sin"], s["seq_pages"] * s["page"], H, q_out=d["q"], stream=stream)
    serving.attention(pg, d["q"], d["len"], s["seq_pages"] * s["page"], H, d["part"], d["out"], stream=stream)
    serving.adjust_logits(d["logits"], n, V, out=d["adj"], tok=d["tok"], part=d["lpart"], hist=d["hist"],
                          n_hist=40 * n, hist_start=d["start"], rep=d["pen"], presence=d["pen"], stream=stream)


def step_outputs(d):
    return {k: d[k].read(np.uint32) for k in ("y", "q", "out", "adj", "tok")} | {k: d[k].read(np.uint16) for k in ("k", "v")}


def test_captured_step_replays():
    """A step on a stream of its own, captured and replayed between eager work
    on new inputs: every replay equals the eager call bit for bit."""
    hip = Hip()
    states = [step_state(i) for i in range(4)]
    want = []
    for s in states:
        d = step_buffers(s)
        step_run(s, d, 0)
        sa.sync()
        want.append(step_outputs(d))
    d = step_buffers(states[0])
    st = hip.stream.value
    step_run(states[0], d, st)                                # eagerly on that stream
    hip("hipStreamSynchronize", hip.stream)
    for k, w in want[0].items():
        np.testing.assert_array_equal(step_outputs(d)[k], w, err_msg=k)
    ex = hip.capture(lambda: step_run(states[0], d, st))
    for i in (1, 2, 3, 0, 2):
        s = states[i]
        for k in ("table", "k", "v", "x", "qkv", "logits", "a", "b", "hist"):
            d[k].write(s[k])
        d["pos"].write(s["lens"])
        d["len"].write(s["lens"] + 1)
        for k in ("part", "work", "lpart", "adj", "out", "y", "q"):
            d[k].write(np.full(d[k].nbytes, 0xFF, np.uint8))
        sa.sync()
        hip.replay(ex)
        got = step_outputs(d)
        for k, w in want[i].items():
            np.testing.assert_array_equal(got[k], w, err_msg=f"{k} of replay {i}")


def test_two_graphs_with_workspaces_of_their_own():
    """Two captured steps in flight on two streams at once."""
    hips, ds, exs, want = [Hip(), Hip()], [], [], []
    states = [step_state(10, n=3), step_state(11)]
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
        for h, ex in zip(hips, exs):
            h("hipGraphLaunch", ex, h.stream)
        for h in hips:
            h("hipStreamSynchronize", h.stream)
        for d, w in zip(ds, want):
            got = step_outputs(d)
            for k in w:
                np.testing.assert_array_equal(got[k], w[k], err_msg=k)


def test_captured_adapters_take_new_ids():
    """A mixed batch captured once and replayed with other ids, in no order, in
    runs and without any: every replay equals the eager call bit for bit."""
    rng = np.random.default_rng(9)
    n, n_in, n_out, rank, A = 100, 264, 130, 16, 7
    a, b = (sa.DevBuf.of(so.to_bits(rng.standard_normal(sh).astype(np.float32), "f16")) for sh in ((A, rank, n_in), (A, n_out, rank)))
    ad = serving.Adapters(a, b, A, rank, n_in, n_out)
    x, base = (sa.DevBuf.of(rng.standard_normal(sh).astype(np.float32)) for sh in ((n, n_in), (n, n_out)))
    work, y, ids = sa.DevBuf(4 * serving.lora_work_floats(rank, n)), sa.DevBuf(4 * n * n_out), ints(np.zeros(n))
    hip = Hip()
    sa.sync()
    ex = hip.capture(lambda: serving.lora(ad, x, n, ids, y, work, base=base, stream=hip.stream.value))
    for which in (rng.integers(-1, A, n), np.arange(n) * A // n, np.full(n, -1), np.arange(n) % A, np.zeros(n)):
        ids.write(np.array(which, np.int32))
        serving.lora(ad, x, n, ids, y, work, base=base)
        sa.sync()
        want = y.read(np.uint32)
        for buf in (y, work):
            buf.write(np.full(buf.nbytes, 0xFF, np.uint8))
        sa.sync()
        hip.replay(ex)
        np.testing.assert_array_equal(y.read(np.uint32), want)


# ------------------------------------------------------------ sizes

GUARD = 4096


class Guarded(sa.DevBuf):
    """A buffer of exactly the bytes asked for, with a pattern behind them."""

    def __init__(self, nbytes):
        super().__init__(nbytes + GUARD)
        self.write(np.full(nbytes + GUARD, 0xA5, np.uint8))

    def intact(self):
        return (self.read(np.uint8)[-GUARD:] == 0xA5).all()


@pytest.mark.parametrize("n_seq, heads, kv, hd, top", [
    (1, 8, 2, 128, 1), (1, 8, 2, 128, 513), (1, 4, 4, 64, 70001), (7, 16, 1, 64, 1000), (40, 32, 8, 128, 600),
    (257, 4, 2, 64, 700), (300, 2, 2, 128, 64)])
def test_attention_stays_in_its_buffers(n_seq, heads, kv, hd, top):
    rng = np.random.default_rng(top)
    page = 64
    pages = -(-top // page)
    bits = [so.to_bits(rng.standard_normal((pages + 1, page, kv, hd)).astype(np.float32), "f16") for _ in range(2)]
    table = np.tile(rng.permutation(pages + 1)[:pages], (n_seq, 1)).astype(np.int32)       # a prefix that all share
    pg = serving.Pages(*map(sa.DevBuf.of, bits), sa.DevBuf.of(table), pages + 1, page, n_seq, pages, kv, hd)
    part, out = Guarded(4 * serving.part_floats(n_seq, heads, hd, top)), Guarded(4 * n_seq * heads * hd)
    one = rng.standard_normal(heads * hd).astype(np.float32)
    q = sa.DevBuf.of(np.tile(one, (n_seq, 1)))
    for lens in ([top] * n_seq, [top + 99] * n_seq, rng.integers(0, top + 1, n_seq), [0] * (n_seq - 1) + [top], [-1] * n_seq):
        serving.attention(pg, q, ints(lens), top, heads, part, out)
        sa.sync()
        assert part.intact() and out.intact()
        got = out.read(np.float32, n_seq * heads * hd).reshape(n_seq, -1)
        assert np.isfinite(got).all()
        if min(lens) >= top:
            for h in range(heads):
                kk, vv = (so.from_bits(w, "f16").reshape(-1, page, kv, hd)[table[0], :, h * kv // heads].reshape(-1, hd)[:top]
                          for w in bits)
                want, tol = so.attend(one[None, h * hd:(h + 1) * hd], kk, vv, hd ** -0.5)
                within(got[:, h * hd:(h + 1) * hd], np.repeat(want, n_seq, 0), np.repeat(tol, n_seq, 0), f"head {h}")
        assert not got[np.array(lens) <= 0].any()


@pytest.mark.parametrize("n, n_in, n_out, rank, A", [
    (1, 8, 1, 8, 1), (16, 520, 33, 64, 16), (17, 1544, 70, 256, 2), (40, 4096, 65, 8, 5), (200, 264, 257, 24, 16),
    (600, 72, 130, 64, 3)])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_lora_stays_in_its_buffers(n, n_in, n_out, rank, A, dtype):
    rng = np.random.default_rng(n)
    a, b = (sa.DevBuf.of(so.to_bits(rng.standard_normal(sh).astype(np.float32), dtype)) for sh in ((A, rank, n_in), (A, n_out, rank)))
    ad = serving.Adapters(a, b, A, rank, n_in, n_out, dtype)
    x = sa.DevBuf.of(rng.standard_normal((n, n_in)).astype(np.float32))
    y, work = Guarded(4 * n * n_out), Guarded(4 * serving.lora_work_floats(rank, n))
    for ids in (rng.integers(-1, A, n), np.arange(n) * A // n, np.full(n, -1)):
        serving.lora(ad, x, n, ints(ids), y, work)
        sa.sync()
        assert y.intact() and work.intact()
        got = y.read(np.float32, n * n_out).reshape(n, n_out)
        assert not got[ids < 0].any() and (got[ids >= 0] != 0).any(axis=1).all()


@pytest.mark.parametrize("n_row, V", [(1, 1), (3, 2047), (2, 2049), (70, 4098), (600, 2050)])
def test_logits_stay_in_their_buffers(n_row, V):
    rng = np.random.default_rng(V)
    x = rng.standard_normal((n_row, V)).astype(np.float32)
    out, tok, part = Guarded(4 * n_row * V), Guarded(4 * n_row), Guarded(serving.logits_part_bytes(n_row, V))
    serving.adjust_logits(sa.DevBuf.of(x), n_row, V, out=out, tok=tok, part=part)
    sa.sync()
    assert out.intact() and tok.intact() and part.intact()
    np.testing.assert_array_equal(out.read(np.float32, n_row * V).reshape(n_row, V), x)
    np.testing.assert_array_equal(tok.read(np.int32, n_row), x.argmax(1))


# ------------------------------------------------------------ a run of them together

def test_requests_decode_together(tmpdir_s):
    """Requests of different lengths and adapters, one layer, several steps:
    prompts are appended in one ragged call with padding, then every step runs
    the shared projection and its adapters, appends, attends, projects to
    logits, penalizes and picks. Each stage is checked against its 64-bit form
    on the stage's own device inputs, and the cache against all that was
    appended."""
    rng = np.random.default_rng(77)
    n, E, H, KV, hd, page, seq_pages, rank, A = 4, 256, 4, 2, 64, 16, 6, 8, 2
    W, V = (H + 2 * KV) * hd, 700
    paths = []
    for name, rows, cols in (("qkv", W, E), ("head", V, H * hd)):
        p = tmpdir_s / f"serving_{name}.ssf"
        sa.synth_matrix(p, rows, cols, nbits=4, seed=rows)
        paths.append(sa.Mat.from_file(p, "w"))
    n_pages = n * seq_pages + 2
    table = make_table(rng, n, seq_pages, n_pages)
    kb, vb = (sa.DevBuf.of(np.zeros(n_pages * page * KV * hd, np.uint16)) for _ in range(2))
    pg = serving.Pages(kb, vb, sa.DevBuf.of(table), n_pages, page, n, seq_pages, KV, hd)
    cos, sin = so.rope_tables(hd // 2, seq_pages * page)
    cb, sb = sa.DevBuf.of(cos), sa.DevBuf.of(sin)
    a = so.to_bits(rng.standard_normal((A, rank, E)) / 16, "f16")
    b = so.to_bits(rng.standard_normal((A, W, rank)) / 3, "f16")
    sc = np.array([0.5, 2.0], np.float32)
    ad = serving.Adapters(sa.DevBuf.of(a), sa.DevBuf.of(b), A, rank, E, W, scale=sa.DevBuf.of(sc))
    which = [0, 1, -1, 1]
    emb = rng.standard_normal((V, E)).astype(np.float32)
    f16 = lambda x: so.from_bits(x, "f16")                                   # noqa: E731

    def project(m, x, rows):
        q = sa.Act(x.shape[1] * rows)
        for r in range(rows):
            act = sa.Act(x.shape[1])
            sa.normq(sa.DevBuf.of(x[r]), act)
            qq, s, u = act.read()
            for buf, w, sz in ((q.q, qq, x.shape[1]), (q.scale, s, x.shape[1] // 8), (q.sums, u, x.shape[1] // 8)):
                sa._chk(sa.lib().sml_hip_h2d(buf.ptr + r * sz, w.ctypes.data, w.nbytes))
        y = sa.DevBuf(4 * m.rows * rows)
        sa.gemm(m, q.q, q.scale, q.sums, rows, y)
        return y

    def through(ids, rows_seq, rows_pos):
        """Rows through the projection, its adapters and the append; returns their q."""
        rows = len(ids)
        x = emb[ids]
        y = project(paths[0], x, rows)
        base = y.read(np.float32).reshape(rows, W)
        adapter = [which[s] for s in rows_seq]
        serving.lora(ad, sa.DevBuf.of(x), rows, ints(adapter), y, sa.DevBuf(4 * serving.lora_work_floats(rank, rows)), base=y)
        got = y.read(np.float32).reshape(rows, W)
        want, tol = so.lora(x, base, f16(a), f16(b), sc, [rank] * A, adapter)
        within(got, want, tol, "adapters")
        qo = sa.DevBuf.of(np.zeros((rows, H * hd), np.float32))
        serving.append(pg, y, rows, ints(rows_pos), cb, sb, seq_pages * page, H, seq=ints(rows_seq), q_out=qo)
        for r in range(rows):
            if rows_pos[r] >= 0:
                z = got[r].reshape(-1, hd)
                rot, _ = so.rotate(z[H:H + KV], cos[rows_pos[r]], sin[rows_pos[r]])
                caches[rows_seq[r]].append((rows_pos[r], rot, so.to_bits(z[H + KV:], "f16")))
        return qo

    caches = [[] for _ in range(n)]
    prompts = [list(rng.integers(0, V, m)) for m in (33, 1, 16, 50)]
    ids, seqs, poss = [], [], []
    for s, p in enumerate(prompts):                            # the last token of each goes with the first step
        ids += p[:-1] + [0]
        seqs += [s] * len(p)
        poss += list(range(len(p) - 1)) + [-1]                 # and a row of padding in its place
    through(np.array(ids), seqs, poss)
    texts, last = [list(map(int, p)) for p in prompts], np.array([p[-1] for p in prompts])
    part = sa.DevBuf(4 * serving.part_floats(n, H, hd, seq_pages * page))
    out, tok = sa.DevBuf(4 * n * H * hd), sa.DevBuf(4 * n)
    lpart = sa.DevBuf(serving.logits_part_bytes(n, V))
    mask = rng.integers(0, 1 << 32, (1, -(-V // 32)), dtype=np.uint64).astype(np.uint32)
    for _ in range(5):
        pos = [len(t) - 1 for t in texts]
        qo = through(last, list(range(n)), pos)
        serving.attention(pg, qo, ints([p + 1 for p in pos]), max(pos) + 1, H, part, out)
        q, got = qo.read(np.float32).reshape(n, H, hd), out.read(np.float32).reshape(n, H, hd)
        kk, vv = kb.read(np.uint16).reshape(n_pages, page, KV, hd), vb.read(np.uint16).reshape(n_pages, page, KV, hd)
        for s in range(n):
            at = [(table[s, p // page], p % page) for p in range(pos[s] + 1)]
            ks, vs = np.array([kk[i] for i in at]), np.array([vv[i] for i in at])
            assert [c[0] for c in sorted(caches[s], key=lambda c: c[0])] == list(range(pos[s] + 1))
            for p, rot, vbits in caches[s]:
                np.testing.assert_array_equal(vs[p], vbits)
                within(f16(ks[p]), rot, so.HALF["f16"] * 1.01 * np.abs(rot) + 4 * so.U * np.abs(rot).max() + 2.0 ** -25, "k")
            for h in range(KV):
                g = slice(h * H // KV, (h + 1) * H // KV)
                want, tol = so.attend(q[s, g], f16(ks[:, h]), f16(vs[:, h]), hd ** -0.5)
                within(got[s, g], want, tol, "attention")
        lg = project(paths[1], got.reshape(n, -1), n)
        raw = lg.read(np.float32).reshape(n, V)
        lens = [len(t) for t in texts]
        serving.adjust_logits(lg, n, V, out=lg, tok=tok, part=lpart, hist=ints(sum(texts, [])), n_hist=sum(lens),
                              hist_start=ints(np.concatenate([[0], np.cumsum(lens)])),
                              n_prompt=ints([len(p) for p in prompts]),
                              rep=sa.DevBuf.of(np.full(n, 1.3, np.float32)),
                              presence=sa.DevBuf.of(np.full(n, 0.4, np.float32)),
                              frequency=sa.DevBuf.of(np.full(n, 0.2, np.float32)), mask=sa.DevBuf.of(mask), n_mask=1,
                              mask_row=ints([-1, 0, -1, 0]))
        adj, picks = lg.read(np.float32).reshape(n, V), tok.read(np.int32)
        ok = ((mask[0][np.arange(V) // 32] >> (np.arange(V) % 32).astype(np.uint32)) & 1).astype(bool)
        for s in range(n):
            want, t = so.adjust(raw[s], np.array(texts[s]), len(prompts[s]), 1.3, 0.4, 0.2, None, ok if s % 2 else None)
            np.testing.assert_array_equal(adj[s], want)
            assert picks[s] == t
            texts[s].append(int(t))
        last = picks.copy()
