"""The operators of a step that serves many requests at once: their plain forms
beside the calls a program makes of the library (sheep_amd/serving.py).

Keys and values are appended to a paged cache with their rotation, one new
token a sequence attends over that cache, low-rank adapters are added beside a
shared projection, and logits get their penalties, biases and grammar masks
before the greedy pick. `own` chooses which of the two `run` computes.

A case is a dict of plain values; "op" says which operator it takes. Lengths
of a ragged batch follow from the case alone, values from the seed.
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
        # the new token's keys and values of 16 conversations: the smallest
        # call of a step, all latency (32 heads over 8 of 128, pages of 16)
        dict(name="append_16_tokens", op="append", heads=32, kv=8, hd=128, type="f16", page=16, rows=16, seqs=16,
             at=1024),
        # the prompts of three requests in one call, ragged, on the 12-over-2
        # head shape with a bfloat16 cache
        dict(name="append_prompts_1021", op="append", heads=12, kv=2, hd=128, type="bf16", page=64, rows=1021, seqs=3,
             at=0),
        # one conversation at the end of a 4096-position context
        dict(name="attend_1_at_4095", op="attend", heads=32, kv=8, hd=128, type="f16", page=16, seqs=1, shortest=4095,
             longest=4095, gone=0),
        # a full server: 48 conversations from a few words to 8192 positions
        dict(name="attend_48_to_8192", op="attend", heads=32, kv=8, hd=128, type="f16", page=64, seqs=48, shortest=33,
             longest=8192, gone=0),
        # one long document, bfloat16, the 28-over-4 head shape
        dict(name="attend_1_at_65537", op="attend", heads=28, kv=4, hd=128, type="bf16", page=128, seqs=1,
             shortest=65537, longest=65537, gone=0),
        # heads of 64, conversations whose first pages were given back
        dict(name="attend_13_hd64_gone", op="attend", heads=32, kv=8, hd=64, type="f16", page=32, seqs=13,
             shortest=700, longest=3001, gone=7),
        # one request's logits with penalties over its whole context
        dict(name="logits_1x128256", op="logits", rows=1, vocab=128256, past=4001, biases=0, mask=False),
        # a batch under grammars, with biases, on the larger vocabulary
        dict(name="logits_16x151936_grammar", op="logits", rows=16, vocab=151936, past=1500, biases=40, mask=True),
        # the largest batch of logits
        dict(name="logits_96x128256", op="logits", rows=96, vocab=128256, past=2047, biases=7, mask=True),
        # one request with a small adapter beside the gate projection
        dict(name="lora_1x1536x8960_r8", op="lora", n_in=1536, n_out=8960, rank=8, type="f16", rows=1, adapters=1,
             runs=False),
        # a step of 16 requests, 11 adapters among them, one without
        dict(name="lora_16x4096x4096_r16", op="lora", n_in=4096, n_out=4096, rank=16, type="f16", rows=16, adapters=11,
             runs=False),
        # a prompt chunk of four requests, adapters of rank 64 beside the up
        # projection
        dict(name="lora_509x4096x14336_r64", op="lora", n_in=4096, n_out=14336, rank=64, type="bf16", rows=509,
             adapters=4, runs=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "logits", "lora", "lora"])
    heads, kv, hd = rng.choice([(32, 8, 128), (12, 2, 128), (16, 8, 128), (8, 8, 128), (28, 4, 128), (32, 8, 64),
                                (14, 2, 64), (32, 2, 128)])
    kind, page = rng.choice(["f16", "bf16"]), rng.choice([16, 32, 64, 128])
    if op == "append":
        rows = _log(rng, 1, 2048)
        return dict(op=op, heads=heads, kv=kv, hd=hd, type=kind, page=page, rows=rows,
                    seqs=rng.randint(1, min(rows, 64)), at=rng.randint(0, 3000))
    if op == "attend":
        seqs = _log(rng, 1, 48)
        longest = _log(rng, 1, min(65537, 200000 // seqs))
        return dict(op=op, heads=heads, kv=kv, hd=hd, type=kind, page=page, seqs=seqs,
                    shortest=rng.randint(0, longest), longest=longest, gone=rng.choice([0, 0, 1, 5]))
    if op == "logits":
        return dict(op=op, rows=_log(rng, 1, 96), vocab=_log(rng, 1000, 128256), past=_log(rng, 1, 8192),
                    biases=rng.choice([0, 1, 13, 300]), mask=rng.random() < 0.5)
    rows = _log(rng, 1, 509)
    return dict(op=op, n_in=32 * _log(rng, 16, 128), n_out=_log(rng, 257, 14336), rank=8 * _log(rng, 1, 8), type=kind,
                rows=rows, adapters=rng.randint(1, min(rows, 16)), runs=rng.random() < 0.5)


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


def _spread(n, lo, hi):
    """n whole numbers from lo to hi, hi among them, even over their logarithm and in no order."""
    return [hi if i == 0 else min(hi, lo + int((hi - lo + 1) ** ((i * 0.6180339887) % 1.0)) - 1) for i in range(n)]


def _rope(half, n):
    f = 5e5 ** (-torch.arange(half, device=DEV, dtype=torch.float64) / half)
    a = torch.arange(n, device=DEV, dtype=torch.float64)[:, None] * f
    return torch.cos(a).float(), torch.sin(a).float()


def _row_places(case):
    """The sequence and the position of each appended row: each sequence's rows follow one another."""
    n, S = case["rows"], case["seqs"]
    seq = [r * S // n for r in range(n)]
    first = {}
    for r, b in enumerate(seq):
        first.setdefault(b, r)
    return seq, [case["at"] + 13 * b * (case["at"] > 0) + r - first[b] for r, b in enumerate(seq)]


def _lengths(case):
    return _spread(case["seqs"], case["shortest"], case["longest"])


def _gone(case, length):
    """Leading pages a sequence has given back: never its last one."""
    return min(case["gone"], max(0, (length - 1) // case["page"]))


def _past(case):
    return _spread(case["rows"], max(1, case["past"] // 8), case["past"])


def _row_adapters(case):
    """Each row's adapter; one row in twelve of a mixed batch has none."""
    n, A = case["rows"], case["adapters"]
    if case["runs"]:
        return [r * A // n for r in range(n)]
    return [-1 if r % 12 == 11 else r % A for r in range(n)]


def _table(g, pages_of, spare):
    """A table of scattered page ids: row b has pages_of[b] of them, -1 behind."""
    total, width = sum(pages_of), max(1, max(pages_of))
    order = torch.randperm(total + spare, generator=g, device=DEV).int()
    table = torch.full((len(pages_of), width), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(pages_of):
        table[b, :n] = order[at:at + n]
        at += n
    return table, total + spare


def prepare(case, seed):
    op = case["op"]
    g = _gen(seed, op)
    s = dict(case=case, op=op)
    if op in ("append", "attend"):
        H, KV, hd, page, dt = case["heads"], case["kv"], case["hd"], case["page"], KV_TYPES[case["type"]]
    if op == "append":
        seq, pos = _row_places(case)
        ends = [max([p for p, q in zip(pos, seq) if q == b], default=0) for b in range(case["seqs"])]
        table, n_pages = _table(g, [e // page + 1 for e in ends], 5)
        s.update(table=Buf(table), n_pages=n_pages, seq=Buf(_ints(seq)), pos=Buf(_ints(pos)))
        s["qkv"] = Buf(_randn(g, case["rows"], (H + 2 * KV) * hd))
        s["cos"], s["sin"] = (Buf(t) for t in _rope(hd // 2, max(ends) + 1))
        s["k"], s["v"] = (Buf(torch.zeros(n_pages, page, KV, hd, dtype=dt, device=DEV)) for _ in range(2))
        s["q_out"] = Buf(torch.empty(case["rows"], H * hd, device=DEV))
    elif op == "attend":
        lens = _lengths(case)
        table, n_pages = _table(g, [-(-n // page) for n in lens], 5)
        for b, n in enumerate(lens):
            table[b, :_gone(case, n)] = -1
        s.update(table=Buf(table), n_pages=n_pages, len=Buf(_ints(lens)), longest=max(1, max(lens)))
        s["k"], s["v"] = (Buf(_randn(g, n_pages, page, KV, hd).to(dt)) for _ in range(2))
        s["q"] = Buf(1.5 * _randn(g, case["seqs"], H * hd))
        s["out"] = Buf(torch.empty(case["seqs"], H * hd, device=DEV))
        # the workspace, as the header sizes it
        splits = min(256, -(-s["longest"] // 64))
        s["part"] = Buf(torch.empty(case["seqs"] * H * splits * (hd + 2), device=DEV))
    elif op == "logits":
        n, V, past = case["rows"], case["vocab"], _past(case)
        s["logits"] = Buf(3.0 * _randn(g, n, V))
        # ids of a text: few common ones, many rare ones
        u = torch.rand(sum(past), generator=g, device=DEV, dtype=torch.float64)
        s["hist"] = Buf((torch.exp(u * math.log(V)) - 1).long().clamp(0, V - 1).int())
        s["n_hist"] = sum(past)
        starts = [0]
        for m in past:
            starts.append(starts[-1] + m)
        s["start"], s["n_prompt"] = Buf(_ints(starts)), Buf(_ints([m // 2 for m in past]))
        s["past"] = past
        s["rep"] = Buf(1.0 + 0.3 * torch.rand(n, generator=g, device=DEV))
        s["pres"], s["freq"] = (Buf(0.5 * torch.rand(n, generator=g, device=DEV)) for _ in range(2))
        nb = case["biases"]
        if nb:
            ids = torch.rand(n, V, generator=g, device=DEV).topk(nb, dim=1).indices
            s["bias_id"], s["bias"] = Buf(ids.reshape(-1).int()), Buf(2.0 * _randn(g, n * nb))
            s["bias_start"] = Buf(_ints([nb * b for b in range(n + 1)]))
        if case["mask"]:
            # a few grammars' states; one row in five goes without
            states = max(1, n // 3)
            bits = torch.randint(-(1 << 31), 1 << 31, (states, -(-V // 32)), generator=g, device=DEV)
            s["mask"], s["n_mask"] = Buf(bits.int()), states
            s["mask_row"] = Buf(_ints([-1 if b % 5 == 4 else b % states for b in range(n)]))
        s["out"], s["tok"] = Buf(torch.empty(n, V, device=DEV)), Buf(torch.empty(n, dtype=torch.int32, device=DEV))
        s["part"] = Buf(torch.empty(n * -(-V // 2048) * 4, dtype=torch.int32, device=DEV))
    else:
        n, ni, no, r, A = case["rows"], case["n_in"], case["n_out"], case["rank"], case["adapters"]
        dt = KV_TYPES[case["type"]]
        s["x"], s["base"] = Buf(_randn(g, n, ni)), Buf(_randn(g, n, no))
        s["a"] = Buf((_randn(g, A, r, ni) / math.sqrt(ni)).to(dt))
        s["b"] = Buf((0.5 * _randn(g, A, no, r) / math.sqrt(r)).to(dt))
        s["scale"] = Buf(0.5 + torch.rand(A, generator=g, device=DEV))
        # some adapters have a lower rank than the pool's rows
        s["ranks"] = Buf(_ints([r if i % 3 else max(1, r - 3 * (i // 3)) for i in range(A)]))
        s["adapter"] = Buf(_ints(_row_adapters(case)))
        s["y"] = Buf(torch.empty(n, no, device=DEV))
        s["work"] = Buf(torch.empty(r * max(n, min(32 * n, 8192)), device=DEV))
    return s


# ---------------------------------------------------------------- plain forms

def _rotate(x, c, sn):
    h = x.shape[-1] // 2
    a, b = x[..., :h], x[..., h:]
    return torch.cat([a * c - b * sn, b * c + a * sn], -1)


def _plain_append(s):
    c = s["case"]
    H, KV, hd, page = c["heads"], c["kv"], c["hd"], c["page"]
    pos, seq = s["pos"].t.long(), s["seq"].t.long()
    rows = s["qkv"].t.view(c["rows"], H + 2 * KV, hd)
    cos, sin = s["cos"].t[pos][:, None], s["sin"].t[pos][:, None]
    s["q_out"].t.copy_(_rotate(rows[:, :H], cos, sin).view(c["rows"], H * hd))
    at = s["table"].t[seq, pos // page].long()
    k, v = s["k"].t, s["v"].t
    k[at, pos % page] = _rotate(rows[:, H:H + KV], cos, sin).to(k.dtype)
    v[at, pos % page] = rows[:, H + KV:].to(v.dtype)
    return {"q": s["q_out"].t, "k": k, "v": v}


def _plain_attend(s):
    c = s["case"]
    B, H, KV, hd, page = c["seqs"], c["heads"], c["kv"], c["hd"], c["page"]
    table = s["table"].t
    L = table.shape[1] * page
    pages = table.long().clamp_min(0)
    k = s["k"].t[pages].view(B, L, KV, hd).permute(0, 2, 3, 1).float()
    v = s["v"].t[pages].view(B, L, KV, hd).permute(0, 2, 1, 3).float()
    there = (table >= 0).repeat_interleave(page, 1) & (torch.arange(L, device=DEV) < s["len"].t[:, None])
    score = torch.matmul(s["q"].t.view(B, KV, H // KV, hd), k) / math.sqrt(hd)
    score = score.masked_fill(~there[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - top.masked_fill(top == -math.inf, 0.0))
    den = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v) / den.masked_fill(den == 0, 1.0)
    return {"out": out.view(B, H * hd)}


def _plain_logits(s):
    c = s["case"]
    n, V = c["rows"], c["vocab"]
    l = s["logits"].t
    at = torch.arange(s["n_hist"], device=DEV, dtype=torch.int32)
    row = torch.searchsorted(s["start"].t, at, right=True) - 1
    gen = (at - s["start"].t[row] >= s["n_prompt"].t[row]).float()
    place = row * V + s["hist"].t
    made = torch.zeros(n * V, device=DEV).index_add_(0, place, gen).view(n, V)
    seen = torch.zeros(n * V, device=DEV).index_fill_(0, place, 1.0).view(n, V) > 0
    rep = s["rep"].t[:, None]
    l = torch.where(seen, torch.where(l > 0, l / rep, l * rep), l)
    l = l - s["freq"].t[:, None] * made
    l = l - s["pres"].t[:, None] * (made > 0)
    if c["biases"]:
        owner = torch.arange(n, device=DEV)[:, None]
        ids = s["bias_id"].t.long().view(n, -1)
        l[owner, ids] = l[owner, ids] + s["bias"].t.view(n, -1)
    if c["mask"]:
        bits = (s["mask"].t[:, :, None] >> torch.arange(32, device=DEV, dtype=torch.int32)) & 1
        bits = bits.view(s["n_mask"], -1)[:, :V] == 0
        which = s["mask_row"].t.long()
        l = l.masked_fill(bits[which.clamp_min(0)] & (which >= 0)[:, None], -math.inf)
    return {"out": l, "tok": l.argmax(1).int()}


def _plain_lora(s):
    c = s["case"]
    A, r, n = c["adapters"], c["rank"], c["rows"]
    which = torch.arange(A, device=DEV)
    mine = (s["adapter"].t[:, None] == which) * s["scale"].t
    live = torch.arange(r, device=DEV) < s["ranks"].t[:, None]
    t = torch.matmul(s["x"].t, s["a"].t.float().view(A * r, -1).t()).view(n, A, r)
    t = t * (mine[:, :, None] * live)
    up = s["b"].t.float().permute(0, 2, 1).reshape(A * r, -1)
    return {"y": s["base"].t + torch.matmul(t.view(n, A * r), up)}


# ---------------------------------------------------------------- run

def _own(s):
    from sheep_amd import serving

    c, op = s["case"], s["op"]
    if op in ("append", "attend"):
        pages = serving.Pages(s["k"], s["v"], s["table"], s["n_pages"], c["page"], c["seqs"], s["table"].t.shape[1],
                              c["kv"], c["hd"], c["type"])
    if op == "append":
        serving.append(pages, s["qkv"], c["rows"], s["pos"], s["cos"], s["sin"], s["cos"].t.shape[0], c["heads"],
                       seq=s["seq"], q_out=s["q_out"])
        return {"q": s["q_out"].t, "k": s["k"].t, "v": s["v"].t}
    if op == "attend":
        serving.attention(pages, s["q"], s["len"], s["longest"], c["heads"], s["part"], s["out"])
        return {"out": s["out"].t}
    if op == "logits":
        serving.adjust_logits(s["logits"], c["rows"], c["vocab"], out=s["out"], tok=s["tok"], part=s["part"],
                              hist=s["hist"], n_hist=s["n_hist"], hist_start=s["start"], n_prompt=s["n_prompt"],
                              rep=s["rep"], presence=s["pres"], frequency=s["freq"], bias_id=s.get("bias_id"),
                              bias=s.get("bias"), n_bias=c["rows"] * c["biases"], bias_start=s.get("bias_start"),
                              mask=s.get("mask"), n_mask=s.get("n_mask", 0), mask_row=s.get("mask_row"))
        return {"out": s["out"].t, "tok": s["tok"].t}
    adapters = serving.Adapters(s["a"], s["b"], c["adapters"], c["rank"], c["n_in"], c["n_out"], c["type"],
                                scale=s["scale"], ranks=s["ranks"])
    serving.lora(adapters, s["x"], c["rows"], s["adapter"], s["y"], s["work"], base=s["base"])
    return {"y": s["y"].t}


def run(s):
    if own:
        return _own(s)
    return {"append": _plain_append, "attend": _plain_attend, "logits": _plain_logits, "lora": _plain_lora}[s["op"]](s)


# ---------------------------------------------------------------- work

def work(case):
    op = case["op"]
    if op == "append":
        n, H, KV, hd = case["rows"], case["heads"], case["kv"], case["hd"]
        # rows in, the rotated q and the rounded k and v out, each position's angles
        return {"bytes": n * (4 * (H + 2 * KV) * hd + 4 * H * hd + 4 * KV * hd + 4 * hd + 12),
                "flops": 3 * n * (H + KV) * hd}
    if op == "attend":
        H, KV, hd = case["heads"], case["kv"], case["hd"]
        live = sum(n - min(n, _gone(case, n) * case["page"]) for n in _lengths(case))
        return {"bytes": live * 4 * KV * hd + case["seqs"] * (8 * H * hd + 4) + live // case["page"] * 4,
                "flops": 4 * live * H * hd}
    if op == "logits":
        n, V = case["rows"], case["vocab"]
        masks = max(1, n // 3) * -(-V // 32) * 4 if case["mask"] else 0
        return {"bytes": 8 * n * V + 4 * sum(_past(case)) + 8 * n * case["biases"] + masks + 40 * n, "flops": 3 * n * V}
    n, ni, no, r = case["rows"], case["n_in"], case["n_out"], case["rank"]
    mine = [a for a in _row_adapters(case) if a >= 0]
    return {"bytes": len(set(mine)) * 2 * r * (ni + no) + 4 * n * ni + 8 * n * no, "flops": 2 * len(mine) * r * (ni + no)}


# ---------------------------------------------------------------- 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "append":
        H, KV, hd, page = case["heads"], case["kv"], case["hd"], case["page"]
        seq, pos = _row_places(case)
        rows = s["qkv"].t.double().view(len(pos), H + 2 * KV, 2, hd // 2)
        p = torch.tensor(pos, device=DEV)
        turn = torch.complex(s["cos"].t[p].double(), s["sin"].t[p].double())[:, None]
        z = torch.complex(rows[:, :H + KV, 0], rows[:, :H + KV, 1]) * turn
        z = torch.cat([z.real, z.imag], -1)
        k, v = (torch.zeros(s["n_pages"] * page, KV, hd, dtype=torch.float64, device=DEV) for _ in range(2))
        table = s["table"].t.cpu().tolist()
        at = torch.tensor([table[b][q // page] * page + q % page for b, q in zip(seq, pos)], device=DEV)
        k[at], v[at] = z[:, H:], s["qkv"].t.double().view(len(pos), H + 2 * KV, hd)[:, H + KV:]
        return {"q": z[:, :H].reshape(len(pos), -1), "k": k.view(-1, page, KV, hd), "v": v.view(-1, page, KV, hd)}
    if op == "attend":
        H, KV, hd, page = case["heads"], case["kv"], case["hd"], case["page"]
        out = torch.zeros(case["seqs"], H, hd, dtype=torch.float64, device=DEV)
        table = s["table"].t.cpu().tolist()
        for b, n in enumerate(_lengths(case)):
            live = [i for i in range(-(-n // page)) if table[b][i] >= 0]
            if not n or not live:
                continue
            ids = torch.tensor([table[b][i] for i in live], device=DEV)
            tail = len(live) * page - ((live[-1] + 1) * page - n)
            for h in range(KV):
                k = s["k"].t[ids, :, h].double().reshape(-1, hd)[:tail]
                v = s["v"].t[ids, :, h].double().reshape(-1, hd)[:tail]
                q = s["q"].t[b].double().view(KV, H // KV, hd)[h]
                w = torch.softmax(torch.mm(q, k.t()) * hd ** -0.5, -1)
                out[b, h * (H // KV):(h + 1) * (H // KV)] = torch.mm(w, v)
        return {"out": out.view(case["seqs"], H * hd)}
    if op == "logits":
        out = s["logits"].t.double().clone()
        hist, nb = s["hist"].t.long(), case["biases"]
        at = 0
        for b, m in enumerate(s["past"]):
            ids, made = torch.unique(hist[at + m // 2:at + m], return_counts=True)
            both = torch.unique(hist[at:at + m])
            at += m
            rep = float(s["rep"].t[b])
            x = out[b, both]
            out[b, both] = torch.maximum(x, x * 0) / rep + torch.minimum(x, x * 0) * rep
            out[b, ids] -= float(s["freq"].t[b]) * made + float(s["pres"].t[b])
            if nb:
                out[b, s["bias_id"].t[b * nb:(b + 1) * nb].long()] += s["bias"].t[b * nb:(b + 1) * nb].double()
            state = b % s["n_mask"] if case["mask"] and b % 5 != 4 else -1
            if state >= 0:
                words = s["mask"].t[state].long()
                v = torch.arange(case["vocab"], device=DEV)
                out[b, (words[v // 32] >> (v % 32)) % 2 == 0] = -math.inf
        return {"out": out, "tok": None}
    y = s["base"].t.double().clone()
    ranks = s["ranks"].t.cpu().tolist()
    rows = _row_adapters(case)
    for a in sorted(set(rows) - {-1}):
        mine = torch.tensor([i for i, w in enumerate(rows) if w == a], device=DEV)
        down = s["a"].t[a, :ranks[a]].double()
        up = s["b"].t[a, :, :ranks[a]].double()
        y[mine] += float(s["scale"].t[a]) * torch.mm(torch.mm(s["x"].t[mine].double(), down.t()), up.t())
    return {"y": y}
