"""The operators of a step that drafts, and of a paged cache's upkeep: their
plain forms beside the calls a program makes of the library
(sheep_amd/serving.py).

New rows are appended with rotary positions of several axes, at slots that the
positions do not give; several rows a sequence (a draft's tree, a prompt's
chunk) attend over the paged cache, with masks, capped scores and a bias of
distance; the drafted rows that the picks accept are kept and moved together;
sequences fork, sharing their full pages; and pages move to others. `own`
chooses which of the two `run` computes.

A case is a dict of plain values; "op" says which operator it takes. Lengths,
trees and masks follow from the case alone, values from the seed.
"""
import hashlib
import math

import torch

own = False

DEV = "cuda"
KV_TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # the drafts of 16 conversations, 8 rows each: slots in order, positions by depth in the tree
        dict(name="axes_16x8_drafts", op="append", heads=32, kv=8, hd=128, type="f16", page=16, seqs=16, rows=8,
             axes=1, at=1024),
        # an image of 37 x 37 patches in a prompt, time, height and width in sections of the pairs
        dict(name="axes_image_37x37", op="append", heads=12, kv=2, hd=128, type="bf16", page=64, seqs=1, rows=1369,
             axes=3, at=100),
        # one conversation's tree of 8 drafted tokens at the end of a 4096-position context: all latency
        dict(name="rows_1x8_tree_at_4095", op="rows", heads=32, kv=8, hd=128, type="f16", page=16, seqs=1, rows=8,
             shortest=4095, longest=4095, mask="tree", cap=0.0, bias=False, idle=False),
        # a server's conversations, 26 drafted tokens each, scores capped
        dict(name="rows_16x26_tree_cap_to_8192", op="rows", heads=32, kv=8, hd=128, type="f16", page=64, seqs=16,
             rows=26, shortest=300, longest=8192, mask="tree", cap=50.0, bias=False, idle=False),
        # a chunk of a prompt behind an earlier part of it
        dict(name="rows_1x509_causal_at_2040", op="rows", heads=32, kv=8, hd=128, type="f16", page=32, seqs=1,
             rows=509, shortest=2040, longest=2040, mask="causal", cap=0.0, bias=False, idle=False),
        # a long prompt of packed documents with a bias of distance, bfloat16, 28 heads over 4
        dict(name="rows_1x2047_docs_bf16", op="rows", heads=28, kv=4, hd=128, type="bf16", page=128, seqs=1, rows=2047,
             shortest=4001, longest=4001, mask="docs", cap=0.0, bias=True, idle=False),
        # one conversation's drafts accepted in 32 layers
        dict(name="accept_1x8_32_layers", op="accept", kv=8, hd=128, type="f16", page=16, seqs=1, rows=8, layers=32,
             longest=900, shared=False),
        # a server's drafts accepted, pages that the layers share
        dict(name="accept_16x26_28_layers", op="accept", kv=4, hd=128, type="bf16", page=32, seqs=16, rows=26,
             layers=28, longest=500, shared=True),
        # four samples of one prompt
        dict(name="fork_4_of_1", op="fork", kv=8, hd=128, type="f16", page=16, seqs=1, forks=4, layers=32, longest=1003,
             shared=False),
        # the beams of 16 requests
        dict(name="fork_64_of_16", op="fork", kv=4, hd=128, type="bf16", page=32, seqs=16, forks=64, layers=28,
             longest=600, shared=True),
        # pages moved down from a pool's end, in all layers: a few, and many
        dict(name="compact_9_pages", op="compact", kv=8, hd=128, type="f16", page=16, seqs=4, moves=9, layers=32,
             longest=300, shared=False),
        dict(name="compact_190_pages", op="compact", kv=2, hd=128, type="bf16", page=64, seqs=24, moves=190, layers=28,
             longest=900, shared=True),
    ]


HEADS = [(32, 8, 128), (12, 2, 128), (16, 8, 128), (28, 4, 128), (32, 8, 64), (14, 2, 64), (32, 2, 128), (4, 4, 128)]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    op = rng.choice(["append", "rows", "rows", "rows", "rows", "accept", "fork", "compact"])
    heads, kv, hd = rng.choice(HEADS)
    kind, page = rng.choice(["f16", "bf16"]), rng.choice([16, 32, 64, 128])
    if op == "append":
        rows = _log(rng, 1, 1400)
        return dict(op=op, heads=heads, kv=kv, hd=hd, type=kind, page=page, seqs=rng.randint(1, max(1, min(24, 1400 // rows))),
                    rows=rows, axes=rng.randint(1, 3), at=rng.randint(0, 2500))
    if op == "rows":
        mask = rng.choice(["tree", "tree", "causal", "window", "prefix", "docs"])
        rows = _log(rng, 1, 90 if mask == "tree" else 1400)
        longest = max(rows, _log(rng, 1, min(8192, 2 ** 21 // rows)))
        # no more pairs than the largest listed case has
        seqs = max(1, min(24, 2 ** 21 // (rows * longest), 60000 // longest))
        return dict(op=op, heads=heads, kv=kv, hd=hd, type=kind, page=page, seqs=rng.randint(1, seqs), rows=rows,
                    shortest=rng.randint(0, longest), longest=longest, mask=mask, cap=rng.choice([0.0, 0.0, 30.0, 50.0]),
                    bias=rng.random() < 0.4, idle=rng.random() < 0.3)
    seqs, layers, shared = rng.randint(1, 16), rng.randint(1, 24), rng.random() < 0.5
    # a pool of at most about 800 MB
    longest = _log(rng, 1, min(1000, 150000 // (seqs * layers)))
    page = min(page, 32)
    some = dict(kv=min(kv, 8), hd=hd, type=kind, page=page, seqs=seqs, layers=layers, longest=longest, shared=shared)
    if op == "accept":
        return dict(op=op, rows=_log(rng, 1, 60), **some)
    if op == "fork":
        return dict(op=op, forks=rng.randint(1, 48), **some)
    return dict(op=op, moves=_log(rng, 1, 60), **some)


# ---------------------------------------------------------------- inputs

class Buf:
    """A torch tensor as one of the library's device buffers."""

    def __init__(self, t):
        self.t = t
        self.ptr = t.data_ptr()


def _gen(seed, salt):
    h = hashlib.sha256(f"{seed}:{salt}".encode()).digest()
    return torch.Generator(device=DEV).manual_seed(int.from_bytes(h[:7], "little"))


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _frac(i):
    return (i * 0.6180339887498949) % 1.0


def _spread(n, lo, hi):
    """n whole numbers from lo to hi, hi among them, even over their logarithm and in no order."""
    return [hi if i == 0 else min(hi, lo + int((hi - lo + 1) ** _frac(i)) - 1) for i in range(n)]


def _rope(half, n):
    f = 5e5 ** (-torch.arange(half, device=DEV, dtype=torch.float64) / half)
    a = torch.arange(n, device=DEV, dtype=torch.float64)[:, None] * f
    return torch.cos(a).float(), torch.sin(a).float()


def _tree(m, b):
    """The parents of m drafted rows of sequence b (-1: the root, row 0), each before its children."""
    return [-1] + [int(j * _frac(7 * j + b)) for j in range(1, m)]


def _depths(parent):
    d = []
    for p in parent:
        d.append(0 if p < 0 else d[p] + 1)
    return d


def _ancestors(parent):
    """Per row the bits of the rows it sees: its ancestors and itself."""
    bits = []
    for j, p in enumerate(parent):
        bits.append((bits[p] if p >= 0 else 0) | 1 << j)
    return bits


def _counts(case):
    """Rows of each sequence, and its length with them: ragged, the first of all rows."""
    m = _spread(case["seqs"], max(1, case["rows"] // 3), case["rows"])
    if case["op"] == "rows":
        n = _spread(case["seqs"], case["shortest"], case["longest"])
    else:
        n = _spread(case["seqs"], max(1, case["longest"] // 6), case["longest"])
    return m, [max(a, b) for a, b in zip(m, n)]


def _starts(m):
    s = [0]
    for x in m:
        s.append(s[-1] + x)
    return s


def _ranges(case):
    """Per row the slots first..last-1 it sees besides its tree's, its own slot and its position."""
    ms, ns = _counts(case)
    out = []
    for b, (m, n) in enumerate(zip(ms, ns)):
        h, kind = n - m, case["mask"]
        depth = _depths(_tree(m, b)) if kind == "tree" else None
        doc = max(1, int(m * 0.37) + 5 * b)
        for i in range(m):
            s = h + i
            lo, hi, pos = 0, s + 1, s
            if kind == "tree":
                hi, pos = h, h + depth[i]
            elif kind == "window":
                lo = max(0, s + 1 - max(1, n // 3))
            elif kind == "prefix":
                hi = max(s + 1, min(n, h + m // 2))
            elif kind == "docs":
                lo = h + i - i % doc if i >= doc else 0
            if case["idle"] and i % 5 == 3:                # a row of padding
                lo = hi = 0
            out.append((lo, hi, s, pos))
    return out


def _bits(case):
    """Per row its tree's bits (none of a row of padding)."""
    ms, _ = _counts(case)
    out = []
    for b, m in enumerate(ms):
        for i, x in enumerate(_ancestors(_tree(m, b))):
            out.append(0 if case["idle"] and i % 5 == 3 else x)
    return out


def _words(bits, n):
    return [[(x >> (32 * w) & 0xFFFFFFFF) - ((x >> (32 * w + 31) & 1) << 32) for w in range(n)] for x in bits]


def _patches(case):
    """The positions of an image's rows after `at` words: time, height and width; of a draft, by depth."""
    out, slots = [[] for _ in range(case["axes"])], []
    for b, m in enumerate(_counts(dict(case, longest=1))[0]):
        depth = _depths(_tree(m, b))
        side = max(1, math.isqrt(m))
        for i in range(m):
            slots.append((b, case["at"] + 13 * b * (case["at"] > 0) + i))
            for a in range(case["axes"]):
                step = depth[i] if case["axes"] == 1 else (0, i // side, i % side)[a]
                out[a].append(case["at"] + 13 * b * (case["at"] > 0) + step)
    return slots, out


def _axis(case):
    """The axis of each rotated pair: sections, the first a quarter of the pairs."""
    half, n = case["hd"] // 2, case["axes"]
    if n == 1:
        return [0] * half
    cut = half // 4 if n == 3 else half // 2
    return [0 if d < cut else 1 + (d - cut) * (n - 1) // (half - cut) for d in range(half)]


def _table(g, pages_of, width, spare):
    """A table of scattered page ids: row b has pages_of[b] of them, -1 behind; and ids that no row has."""
    total = sum(pages_of)
    order = torch.randperm(total + spare, generator=g, device=DEV).int()
    table = torch.full((len(pages_of), max(1, width)), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(pages_of):
        table[b, :n] = order[at:at + n]
        at += n
    return table, order[total:], total + spare


def _pools(case, g, n_pages, s):
    """Both pools of all layers; s["k"], s["v"] are the buffers, s["kl"], s["vl"] the same by layer and page."""
    L, page, kv, hd, dt = case["layers"], case["page"], case["kv"], case["hd"], KV_TYPES[case["type"]]
    size = page * kv * hd
    shape = (n_pages, L) if case["shared"] else (L, n_pages)
    for x in "kv":
        t = torch.empty(*shape, page, kv, hd, dtype=dt, device=DEV).normal_(generator=g)
        s[x], s[x + "l"] = Buf(t), t.transpose(0, 1) if case["shared"] else t
    s["page_stride"], s["layer_stride"] = (L * size, size) if case["shared"] else (0, n_pages * size)
    s["n_pages"] = n_pages


def _floats(seqs, rows, kv, heads, hd):
    """The workspace of the rows' attention, as the header sizes it."""
    return kv * (2 * -(-512 // kv) + min(seqs, rows)) * min(128, rows * (heads // kv)) * (hd + 2)


def prepare(case, seed):
    op, page, dt = case["op"], case["page"], KV_TYPES[case["type"]]
    kv, hd = case["kv"], case["hd"]
    g = _gen(seed, op)
    s = dict(case=case, op=op)
    if op == "append":
        H = case["heads"]
        slots, pos = _patches(case)
        ends = [max(p for q, p in slots if q == b) for b in range(case["seqs"])]
        table, _, n_pages = _table(g, [e // page + 1 for e in ends], max(ends) // page + 1, 5)
        s.update(table=Buf(table), n_pages=n_pages, n=len(slots), axis=bytes(_axis(case)))
        s["seq"], s["slot"] = Buf(_ints([b for b, _ in slots])), Buf(_ints([p for _, p in slots]))
        s["pos"] = Buf(_ints(pos))
        s["qkv"] = Buf(_randn(g, len(slots), (H + 2 * kv) * hd))
        s["cos"], s["sin"] = (Buf(t) for t in _rope(hd // 2, max(max(p) for p in pos) + 1))
        s["k"], s["v"] = (Buf(torch.zeros(n_pages, page, kv, hd, dtype=dt, device=DEV)) for _ in range(2))
        s["q_out"] = Buf(torch.empty(len(slots), H * hd, device=DEV))
        return s
    if op == "rows":
        _from_rows(case, g, s)
        return s
    ms, ns = _counts(dict(case, rows=case.get("rows", 1)))
    tail = 1 if op == "fork" else 0
    of = [-(-n // page) for n in ns]
    spare = case["forks"] if op == "fork" else case["moves"] if op == "compact" else 3
    table, free, n_pages = _table(g, of, max(of) + tail, spare)
    _pools(case, g, n_pages, s)
    s.update(table=Buf(table), len=Buf(_ints(ns)))
    if op == "accept":
        starts = _starts(ms)
        trees = [_tree(m, b) for b, m in enumerate(ms)]
        w = s["most"] = max(_depths(t)[j] for t in trees for j in range(len(t))) + 1
        tok = torch.randint(0, 128256, (starts[-1],), generator=g, device=DEV).int()
        pick = torch.randint(0, 128256, (starts[-1],), generator=g, device=DEV).int()
        toks = tok.cpu().tolist()
        dice = torch.rand(starts[-1], generator=g, device=DEV).cpu().tolist()
        # Each picked token is one of the row's drafted children more often
        # than not. A path whose rows would be moved over rows that it takes is
        # not offered, so that a pass can be made again on what it left.
        for b, t in enumerate(trees):
            i, path = 0, [0]
            while True:
                mine = [j for j in range(1, len(t)) if t[j] == i]
                if not mine or dice[starts[b] + i] < 0.15:
                    break
                j = mine[int(dice[starts[b] + i] * 997) % len(mine)]
                moved = [x for at, x in enumerate(path + [j]) if x != at]
                if moved and min(moved) <= len(path):
                    break
                pick[starts[b] + i] = toks[starts[b] + j]
                path.append(j)
                i = j
        s.update(n=starts[-1], start=Buf(_ints(starts)), tok=Buf(tok), pick=Buf(pick),
                 parent=Buf(_ints([p for t in trees for p in t])))
        s["bits"] = torch.tensor([[[x >> j & 1 for j in range(max(ms))] for x in _ancestors(t)]
                                  + [[0] * max(ms)] * (max(ms) - len(t)) for t in trees], device=DEV).bool()
        for k, shape in (("n_kept", (case["seqs"],)), ("kept", (case["seqs"], w)), ("next", (case["seqs"], w)),
                         ("len_out", (case["seqs"],))):
            s[k] = Buf(torch.empty(shape, dtype=torch.int32, device=DEV))
    elif op == "fork":
        n = case["forks"]
        s["parent"] = Buf(torch.randint(0, case["seqs"], (n,), generator=g, device=DEV).int())
        s["fresh"] = Buf(free[:n].contiguous())
        s["table_out"], s["len_out"] = Buf(torch.empty(n, table.shape[1], dtype=torch.int32, device=DEV)), \
            Buf(torch.empty(n, dtype=torch.int32, device=DEV))
    else:
        used = table[table >= 0].sort().values
        n = min(case["moves"], len(used))
        s["n"] = n
        s["src"], s["dst"] = Buf(used[len(used) - n:].contiguous()), Buf(free.sort().values[:n].contiguous())
        s["was"] = table.clone()
    return s


def _from_rows(case, g, s):
    H, kv, hd, page, dt = case["heads"], case["kv"], case["hd"], case["page"], KV_TYPES[case["type"]]
    ms, ns = _counts(case)
    of = [-(-n // page) for n in ns]
    table, _, n_pages = _table(g, of, max(of), 5)
    rows = _ranges(case)
    s.update(table=Buf(table), n_pages=n_pages, n=len(rows), longest=max(1, max(ns)), most=max(ms))
    s["start"], s["len"] = Buf(_ints(_starts(ms))), Buf(_ints(ns))
    s["seq_of"] = _ints([b for b, m in enumerate(ms) for _ in range(m)]).long()
    s["slot"], s["pos"] = _ints([r[2] for r in rows]), Buf(_ints([r[3] for r in rows]))
    s["first"], s["last"] = Buf(_ints([r[0] for r in rows])), Buf(_ints([r[1] for r in rows]))
    if case["mask"] == "tree":
        s["words"] = -(-max(ms) // 32)
        s["tree"] = Buf(_ints(_words(_bits(case), s["words"])))
    s["k"], s["v"] = (Buf(_randn(g, n_pages, page, kv, hd).to(dt)) for _ in range(2))
    s["q"] = Buf(1.5 * _randn(g, len(rows), H * hd))
    if case["bias"]:
        s["slope"] = Buf(2.0 ** (-8.0 * torch.arange(1, H + 1, device=DEV) / H))
    s["out"] = Buf(torch.empty(len(rows), H * hd, device=DEV))
    s["part"] = Buf(torch.empty(_floats(case["seqs"], len(rows), kv, H, hd), device=DEV))


# ---------------------------------------------------------------- plain forms

def _turn(x, c, sn):
    h = x.shape[-1] // 2
    a, b = x[..., :h], x[..., h:]
    return torch.cat([a * c - b * sn, b * c + a * sn], -1)


def _plain_append(s):
    c = s["case"]
    H, KV, hd, page, n = c["heads"], c["kv"], c["hd"], c["page"], s["n"]
    axis = torch.tensor(list(s["axis"]), device=DEV)
    pos = s["pos"].t.long()[axis].t()                      # [row][pair]
    pair = torch.arange(hd // 2, device=DEV)
    cos, sin = s["cos"].t[pos, pair][:, None], s["sin"].t[pos, pair][:, None]
    rows = s["qkv"].t.view(n, H + 2 * KV, hd)
    slot, seq = s["slot"].t.long(), s["seq"].t.long()
    s["q_out"].t.copy_(_turn(rows[:, :H], cos, sin).view(n, H * hd))
    at = s["table"].t[seq, slot // page].long()
    k, v = s["k"].t, s["v"].t
    k[at, slot % page] = _turn(rows[:, H:H + KV], cos, sin).to(k.dtype)
    v[at, slot % page] = rows[:, H + KV:].to(v.dtype)
    return {"q": s["q_out"].t, "k": k, "v": v}


def _plain_rows(s):
    c = s["case"]
    B, H, KV, hd, page, n, M = c["seqs"], c["heads"], c["kv"], c["hd"], c["page"], s["n"], s["most"]
    table = s["table"].t.long()
    L, G = table.shape[1] * page, H // KV
    k = s["k"].t[table.clamp_min(0)].view(B, L, KV, hd).permute(0, 2, 3, 1).float().contiguous()
    v = s["v"].t[table.clamp_min(0)].view(B, L, KV, hd).permute(0, 2, 1, 3).float().contiguous()
    seq, start, length = s["seq_of"], s["start"].t.long(), s["len"].t.long()
    mine = torch.arange(n, device=DEV) - start[seq]        # a row's number in its sequence
    q = torch.zeros(B, M, H, hd, device=DEV)
    q[seq, mine] = s["q"].t.view(n, H, hd)
    q = q.view(B, M, KV, G, hd).permute(0, 2, 3, 1, 4).reshape(B, KV, G * M, hd)
    score = torch.matmul(q, k).view(B, H, M, L) * hd ** -0.5
    if c["cap"]:
        score = c["cap"] * torch.tanh(score / c["cap"])
    at = torch.arange(L, device=DEV)
    here = (at < length[:, None]) & (table >= 0).repeat_interleave(page, 1)
    see = (at >= s["first"].t[:, None]) & (at < s["last"].t[:, None])
    own_rows = start[1:] - start[:-1]
    j = at[None] - (length - own_rows)[:, None]            # a slot's row in its sequence, below 0 for the past
    if c["mask"] == "tree":
        jr = j[seq].clamp(0, 32 * s["words"] - 1)
        bit = (s["tree"].t.gather(1, jr // 32) >> (jr % 32).int()) & 1
        see = see | ((bit == 1) & (j[seq] >= 0) & (j[seq] < own_rows[seq][:, None]))
    mask = torch.zeros(B, M, L, dtype=torch.bool, device=DEV)
    mask[seq, mine] = see & here[seq]
    if c["bias"]:
        place = torch.where(j >= 0, s["pos"].t[(start[:-1, None] + j).clamp(0, n - 1)].long(), at[None])
        far = torch.zeros(B, M, L, device=DEV)
        far[seq, mine] = (s["pos"].t[:, None].long() - place[seq]).abs().float()
        score = score - s["slope"].t[:, None, None] * far[:, None]
    score = score.masked_fill(~mask[:, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - top.masked_fill(top == -math.inf, 0.0))
    den = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(B, KV, G * M, L), v).view(B, H, M, hd) / den.masked_fill(den == 0, 1.0)
    return {"out": out.permute(0, 2, 1, 3)[seq, mine].reshape(n, H * hd)}


def _plain_accept(s):
    c = s["case"]
    B, page, w = c["seqs"], c["page"], s["most"]
    start, length, table = s["start"].t.long(), s["len"].t.long(), s["table"].t.long()
    M = s["bits"].shape[1]
    count = start[1:] - start[:-1]
    i = torch.arange(M, device=DEV)
    there = i < count[:, None]
    row = (start[:-1, None] + i).clamp_max(s["n"] - 1)
    tok, parent, pick = s["tok"].t.long()[row], s["parent"].t.long()[row], s["pick"].t.long()[row]
    match = (tok == pick.gather(1, parent.clamp_min(0))) & (parent >= 0) & there
    # of siblings with one token the first counts
    twin = match[:, None] & match[:, :, None] & (parent[:, None] == parent[:, :, None]) & (i < i[:, None])
    match = match & ~twin.any(2)
    match[:, 0] = there[:, 0]
    keep = there & ~(s["bits"] & ~match[:, None]).any(2)   # all of its ancestors match
    n_kept = keep.sum(1)
    order = (~keep).int().sort(dim=1, stable=True).indices[:, :w]
    live = torch.arange(order.shape[1], device=DEV) < n_kept[:, None]
    past = (length - count)[:, None]
    src = torch.where(live, past + order, 0)
    dst = torch.where(live, past + torch.arange(order.shape[1], device=DEV), 0)
    owner = torch.arange(B, device=DEV)[:, None].expand_as(src)[live]
    src, dst = src[live], dst[live]
    a, b = table[owner, src // page], table[owner, dst // page]
    for x in (s["kl"], s["vl"]):
        x[:, b, dst % page] = x[:, a, src % page]
    s["n_kept"].t.copy_(n_kept)
    s["kept"].t.copy_(torch.where(live, order, -1))
    s["next"].t.copy_(torch.where(live, pick.gather(1, order), -1))
    s["len_out"].t.copy_(length - count + n_kept)
    return {"n_kept": s["n_kept"].t, "kept": s["kept"].t, "next": s["next"].t, "len": s["len_out"].t, "k": s["k"].t,
            "v": s["v"].t}


def _plain_fork(s):
    page, table = s["case"]["page"], s["table"].t
    parent, fresh = s["parent"].t.long(), s["fresh"].t.long()
    length = s["len"].t[parent]
    full, part = length // page, length % page
    at = torch.arange(table.shape[1], device=DEV)
    out = torch.where(at < full[:, None], table[parent], -1)
    cut = (at == full[:, None]) & (part[:, None] > 0)
    s["table_out"].t.copy_(torch.where(cut, s["fresh"].t[:, None], out))
    s["len_out"].t.copy_(length)
    src = table[parent, full.long().clamp_max(table.shape[1] - 1)].long().clamp_min(0)
    move = (torch.arange(page, device=DEV) < part[:, None])[None, :, :, None, None]
    for x in (s["kl"], s["vl"]):
        x[:, fresh] = torch.where(move, x[:, src], x[:, fresh])
    return {"table": s["table_out"].t, "len": s["len_out"].t, "k": s["k"].t, "v": s["v"].t}


def _plain_compact(s):
    src, dst, table = s["src"].t.long(), s["dst"].t.long(), s["table"].t
    for x in (s["kl"], s["vl"]):
        x[:, dst] = x[:, src]
    to = torch.arange(s["n_pages"], device=DEV, dtype=torch.int32)
    to[src] = s["dst"].t
    table.copy_(torch.where(table >= 0, to[table.long().clamp_min(0)], table))
    return {"table": table, "k": s["k"].t, "v": s["v"].t}


# ---------------------------------------------------------------- run

def _own(s):
    from sheep_amd import serving

    c, op = s["case"], s["op"]
    pages = serving.Pages(s["k"], s["v"], s["table"], s["n_pages"], c["page"], c["seqs"], s["table"].t.shape[1], c["kv"],
                          c["hd"], c["type"], page_stride=s.get("page_stride", 0))
    if op == "append":
        serving.append_axes(pages, s["qkv"], s["n"], s["slot"], s["pos"], s["axis"], s["cos"], s["sin"],
                            s["cos"].t.shape[0], c["heads"], n_axis=c["axes"], seq=s["seq"], q_out=s["q_out"])
        return {"q": s["q_out"].t, "k": s["k"].t, "v": s["v"].t}
    if op == "rows":
        plain = c["mask"] in ("tree", "causal") and not c["idle"]    # what the call takes by itself
        rows = serving.Rows(s["start"], s["len"], s["n"], s["longest"], first=None if plain else s["first"],
                            last=None if plain else s["last"], tree=s.get("tree"), tree_words=s.get("words", 0),
                            pos=s["pos"], slope=s.get("slope"), cap=c["cap"])
        serving.attention_rows(pages, rows, s["q"], c["heads"], s["part"], s["out"])
        return {"out": s["out"].t}
    layers = dict(n_layer=c["layers"], layer_stride=s["layer_stride"])
    if op == "accept":
        serving.accept(pages, s["n"], s["start"], s["len"], s["tok"], s["parent"], s["pick"], s["most"], s["n_kept"],
                       s["kept"], s["next"], s["len_out"], **layers)
        return {"n_kept": s["n_kept"].t, "kept": s["kept"].t, "next": s["next"].t, "len": s["len_out"].t,
                "k": s["k"].t, "v": s["v"].t}
    if op == "fork":
        serving.fork(pages, s["len"], c["forks"], s["parent"], s["fresh"], s["table_out"], s["len_out"], **layers)
        return {"table": s["table_out"].t, "len": s["len_out"].t, "k": s["k"].t, "v": s["v"].t}
    serving.compact(pages, s["n"], s["src"], s["dst"], table=s["table"], **layers)
    return {"table": s["table"].t, "k": s["k"].t, "v": s["v"].t}


def run(s):
    if own:
        return _own(s)
    return {"append": _plain_append, "rows": _plain_rows, "accept": _plain_accept, "fork": _plain_fork,
            "compact": _plain_compact}[s["op"]](s)


# ---------------------------------------------------------------- work

def work(case):
    op, kv, hd, page = case["op"], case["kv"], case["hd"], case["page"]
    if op == "append":
        H = case["heads"]
        n = sum(_counts(dict(case, longest=1))[0])
        # rows in, the rotated q and the rounded k and v out, each row's angles
        return {"bytes": n * (4 * (H + 2 * kv) * hd + 4 * H * hd + 4 * kv * hd + 4 * hd + 8 + 4 * case["axes"]),
                "flops": 3 * n * (H + kv) * hd}
    if op == "rows":
        H = case["heads"]
        ms, ns = _counts(case)
        bits = _bits(case) if case["mask"] == "tree" else [0] * sum(ms)
        rows = _ranges(case)
        pairs = sum(hi - lo + bin(x).count("1") for (lo, hi, _, _), x in zip(rows, bits))
        read, at = 0, 0
        for m, n in zip(ms, ns):
            mine = rows[at:at + m]
            low = min((lo for lo, hi, _, _ in mine if hi > lo), default=0)
            read += n - low if case["mask"] == "tree" or any(hi > lo for lo, hi, _, _ in mine) else 0
            at += m
        return {"bytes": read * 4 * kv * hd + len(rows) * 8 * H * hd + 8 * len(rows), "flops": 4 * pairs * H * hd}
    row = 2 * kv * hd * 2 * case["layers"]                 # a position's keys and values in all layers
    ms, ns = _counts(dict(case, rows=case.get("rows", 1)))
    if op == "accept":
        # about one row a sequence moves; the tree's tokens, parents and picks
        return {"bytes": 2 * row * case["seqs"] + 12 * sum(ms) + 16 * case["seqs"], "flops": 0}
    if op == "fork":
        return {"bytes": 2 * row * case["forks"] * sum(n % page for n in ns) / len(ns)
                + 8 * case["forks"] * (-(-max(ns) // page)), "flops": 0}
    total = sum(-(-n // page) for n in ns)
    return {"bytes": 2 * row * page * min(case["moves"], total) + 8 * total + 8 * case["moves"], "flops": 0}


# ---------------------------------------------------------------- 64 bits

def exact(case, seed):
    if case["op"] not in ("append", "rows"):
        return None                                        # copies and whole numbers
    s = prepare(case, seed)
    H, KV, hd, page, n = case["heads"], case["kv"], case["hd"], case["page"], s["n"]
    table = s["table"].t.cpu().tolist()
    if case["op"] == "append":
        slots, pos = _patches(case)
        axis = _axis(case)
        rows = s["qkv"].t.double().view(n, H + 2 * KV, 2, hd // 2)
        at = torch.tensor([pos[axis[d]] for d in range(hd // 2)], device=DEV).t()
        pair = torch.arange(hd // 2, device=DEV)
        turn = torch.complex(s["cos"].t[at, pair].double(), s["sin"].t[at, pair].double())[:, None]
        z = torch.complex(rows[:, :H + KV, 0], rows[:, :H + KV, 1]) * turn
        z = torch.cat([z.real, z.imag], -1)
        k, v = (torch.zeros(s["n_pages"] * page, KV, hd, dtype=torch.float64, device=DEV) for _ in range(2))
        where = torch.tensor([table[b][p // page] * page + p % page for b, p in slots], device=DEV)
        k[where], v[where] = z[:, H:], s["qkv"].t.double().view(n, H + 2 * KV, hd)[:, H + KV:]
        return {"q": z[:, :H].reshape(n, -1), "k": k.view(-1, page, KV, hd), "v": v.view(-1, page, KV, hd)}
    ms, ns = _counts(case)
    G, at = H // KV, 0
    out = torch.zeros(n, H, hd, dtype=torch.float64, device=DEV)
    rows = _ranges(case)
    bits = _bits(case) if case["mask"] == "tree" else [0] * n
    for b, (m, length) in enumerate(zip(ms, ns)):
        mine, trees = rows[at:at + m], bits[at:at + m]
        slot = torch.arange(length, device=DEV)
        lo, hi = (torch.tensor([r[i] for r in mine], device=DEV)[:, None] for i in (0, 1))
        see = (slot >= lo) & (slot < hi)
        if case["mask"] == "tree":
            see[:, length - m:] |= torch.tensor([[x >> j & 1 for j in range(m)] for x in trees], device=DEV).bool()
        q_at = torch.tensor([r[3] for r in mine], device=DEV)
        k_at = slot.clone()
        k_at[length - m:] = q_at
        far = (q_at[:, None] - k_at).abs().double()
        ids = torch.tensor(table[b][:-(-length // page)], device=DEV)
        for h in range(KV):
            k, v = (s[x].t[ids, :, h].double().reshape(-1, hd)[:length] for x in "kv")
            for e in range(h * G, (h + 1) * G):
                q = s["q"].t[at:at + m].double().view(m, H, hd)[:, e].contiguous()
                z = torch.mm(q, k.t().contiguous()) / math.sqrt(hd)
                if case["cap"]:
                    z = torch.tanh(z / case["cap"]) * case["cap"]
                if case["bias"]:
                    z = z - s["slope"].t[e].double() * far
                p = torch.softmax(z.masked_fill(~see, -math.inf), -1)
                out[at:at + m, e] = torch.mm(torch.nan_to_num(p), v)
        at += m
    return {"out": out.view(n, H * hd)}
