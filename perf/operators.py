"""Operators of batched serving over a paged key-value cache: attention of one new token per
sequence, the preparation and store of new tokens, page upkeep (extend, fork, free, compact) and
the logits' penalties, biases and grammar masks.

Shapes follow the library's benchmark configuration (64 query / 4 KV heads of 128, vocabulary
151,936, positions to 131,072) and generic ones around it.  With `own` false every case runs in
elementary torch operations; with `own` true through mnemocuda_amd.ops.

Page layout: K [page][kv head][position][dim], V [page][kv head][dim][position], int8 scales
[page][kv head][position]; a table row lists a sequence's pages (-1: none).
"""
import math
import random

import torch

own = False

DEV = "cuda"
EPS, THETA = 1e-6, 1e6
WS_BYTES = 64 << 20  # one workspace for every call, as a server keeps it


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # a single conversation's next token: latency of a call
        {"name": "attend_one_short", "kind": "attend", "seqs": 1, "lo": 300, "hi": 300, "heads": 64, "kv": 4,
         "hd": 128, "page": 64, "int8": False},
        # a small server: 16 conversations of mixed lengths, one finished, one just begun
        {"name": "attend_batch16", "kind": "attend", "seqs": 16, "lo": 200, "hi": 4096, "heads": 64, "kv": 4,
         "hd": 128, "page": 64, "int8": False},
        # a few very long documents in an 8-bit cache
        {"name": "attend_long_int8", "kind": "attend", "seqs": 3, "lo": 30000, "hi": 131072, "heads": 64, "kv": 4,
         "hd": 128, "page": 64, "int8": True},
        # a full server with small pages
        {"name": "attend_batch96_page16", "kind": "attend", "seqs": 96, "lo": 500, "hi": 8192, "heads": 64, "kv": 8,
         "hd": 128, "page": 16, "int8": False},
        # a model without shared heads and with a small head size
        {"name": "attend_mha_hd64", "kind": "attend", "seqs": 25, "lo": 2, "hi": 1500, "heads": 12, "kv": 12,
         "hd": 64, "page": 32, "int8": False},
        # the new tokens of 33 decoding sequences
        {"name": "prep_step33", "kind": "prep", "seqs": 33, "tokens": 1, "start": 9000, "heads": 64, "kv": 4,
         "hd": 128, "page": 64, "int8": False},
        # prompt chunks of three sequences into an 8-bit cache
        {"name": "prep_prompt_int8", "kind": "prep", "seqs": 3, "tokens": 633, "start": 1000, "heads": 64, "kv": 4,
         "hd": 128, "page": 64, "int8": True},
        # a beam step: 24 losing beams are freed, 24 forks of 8 parents take their rows
        {"name": "refork_beams", "kind": "refork", "parents": 8, "beams": 3, "lo": 100, "hi": 2000, "layers": 16,
         "kv": 4, "hd": 128, "page": 64, "int8": False},
        # sequences come and go, and the pool is compacted behind them
        {"name": "compact_pool", "kind": "compact", "rows": 30, "lo": 50, "hi": 1500, "layers": 12, "kv": 4,
         "hd": 128, "page": 32, "int8": True},
        # one constrained row
        {"name": "logits_one", "kind": "logits", "rows": 1, "vocab": 151936, "history": 700, "bias": 16, "mask": True},
        # a small model's batch without a grammar
        {"name": "logits_7_small", "kind": "logits", "rows": 7, "vocab": 32003, "history": 2000, "bias": 0,
         "mask": False},
        # a full server's batch with long histories
        {"name": "logits_61", "kind": "logits", "rows": 61, "vocab": 151936, "history": 8000, "bias": 100,
         "mask": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend"] * 5 + ["prep"] * 2 + ["refork"] * 2 + ["compact"] * 2 + ["logits"] * 3)
    while True:
        int8 = rng.random() < 0.4
        page = rng.choice([16, 32, 64, 128])
        kv = rng.choice([1, 2, 3, 4, 8])
        hd = rng.choice([64, 128, 128, 256])
        if kind == "attend":
            hi = _log(rng, 8, 131072)
            c = {"kind": kind, "seqs": _log(rng, 1, 160), "lo": rng.randint(1, hi), "hi": hi,
                 "heads": kv * rng.randint(1, 16), "kv": kv, "hd": hd, "page": page, "int8": int8}
        elif kind == "prep":
            c = {"kind": kind, "seqs": _log(rng, 1, 64), "tokens": rng.choice([1, 1, _log(rng, 2, 1000)]),
                 "start": _log(rng, 1, 8000), "heads": kv * rng.randint(1, 16), "kv": kv, "hd": hd, "page": page,
                 "int8": int8}
        elif kind == "refork":
            c = {"kind": kind, "parents": _log(rng, 1, 24), "beams": rng.randint(1, 6), "lo": rng.randint(1, 100),
                 "hi": _log(rng, 101, 4000), "layers": _log(rng, 1, 24), "kv": kv, "hd": hd, "page": page, "int8": int8}
        elif kind == "compact":
            c = {"kind": kind, "rows": _log(rng, 2, 100), "lo": rng.randint(1, 50), "hi": _log(rng, 51, 4000),
                 "layers": _log(rng, 1, 24), "kv": kv, "hd": hd, "page": page, "int8": int8}
        else:
            c = {"kind": kind, "rows": _log(rng, 1, 64), "vocab": _log(rng, 1000, 151936),
                 "history": _log(rng, 1, 16000), "bias": rng.choice([0, _log(rng, 1, 300)]),
                 "mask": rng.random() < 0.6}
        # no dearer than the largest listed case, in traffic or in the pool that it needs
        if work(c)["bytes"] <= 900e6 and _pool_bytes(c) <= 4e9:
            return c


def _lens(c, n, what=""):
    """The lengths of a case's sequences, the same for every seed: spread evenly over their logarithm between
    lo and hi, the longest first; a batch of 8 or more holds a row of one token and an empty one."""
    r = random.Random("%s %d %d %d" % (what, n, c["lo"], c["hi"]))
    x = [c["hi"]] + [_log(r, c["lo"], c["hi"]) for _ in range(n - 1)]
    if n >= 8 and not what:
        x[3], x[5] = 1, 0
    return x


def _pages(lens, page):
    return [-(-x // page) for x in lens]


def _pool_bytes(c):
    if c["kind"] == "logits":
        return 0
    positions = {"attend": c.get("seqs", 0) * c.get("hi", 0), "prep": c.get("seqs", 0) * (c.get("start", 0) + c.get("tokens", 0)),
                 "refork": c.get("parents", 0) * (c.get("hi", 0) + c.get("beams", 0) * c["page"]),
                 "compact": 2 * c.get("rows", 0) * c.get("hi", 0)}[c["kind"]]
    return positions * c.get("layers", 1) * c["kv"] * c["hd"] * (2 if c["int8"] else 4)


# ------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _pool(g, c, layers, n):
    """Cache pages with every position filled: normalised keys, values a little wider spread."""
    kv, ps, hd = c["kv"], c["page"], c["hd"]
    s = {}
    if c["int8"]:
        s["k"] = torch.randint(-127, 128, (layers, n, kv, ps, hd), dtype=torch.int8, device=DEV, generator=g)
        s["v"] = torch.randint(-127, 128, (layers, n, kv, hd, ps), dtype=torch.int8, device=DEV, generator=g)
        s["ks"] = (0.5 + torch.rand((layers, n, kv, ps), device=DEV, generator=g)) * 0.02
        s["vs"] = (0.5 + torch.rand((layers, n, kv, ps), device=DEV, generator=g)) * 0.02
    else:
        s["k"] = torch.randn((layers, n, kv, ps, hd), dtype=torch.float16, device=DEV, generator=g)
        s["v"] = torch.randn((layers, n, kv, hd, ps), dtype=torch.float16, device=DEV, generator=g)
        s["ks"] = s["vs"] = None
    return s


def _table(g, need, width, n_pages):
    """A table whose rows hold need[i] pages each, drawn without replacement from the pool."""
    ids = torch.randperm(n_pages, device=DEV, generator=g).to(torch.int32)
    t = torch.full((len(need), width), -1, dtype=torch.int32, device=DEV)
    at = 0
    for i, n in enumerate(need):
        t[i, :n] = ids[at:at + n]
        at += n
    return t


def prepare(case, seed):
    c, g = case, _gen(seed)
    s = {"c": c, "kind": c["kind"]}
    if c["kind"] == "attend":
        lens = _lens(c, c["seqs"])
        need = _pages(lens, c["page"])
        n = sum(need) + max(4, sum(need) // 16)
        s |= {t: x if x is None else x[0] for t, x in _pool(g, c, 1, n).items()}
        s["table"], s["lens"] = _table(g, need, max(need), n), _ints(lens)
        # normalised query heads of several sharpnesses
        s["q"] = torch.randn((c["seqs"], c["heads"], c["hd"]), device=DEV, generator=g) * \
            (0.5 + 1.5 * torch.rand((c["seqs"], c["heads"], 1), device=DEV, generator=g))
        s["out"] = torch.empty_like(s["q"])
        s["ws"] = torch.empty(WS_BYTES, dtype=torch.uint8, device=DEV)
    elif c["kind"] == "prep":
        n_seq, t = c["seqs"], c["tokens"]
        r = random.Random(c["start"])
        start = [max(0, c["start"] - r.randint(0, c["page"]) * (i > 0)) for i in range(n_seq)]
        lens = [x + t for x in start]
        need = _pages(lens, c["page"])
        n = sum(need) + 3
        s |= {k: x if x is None else x[0] for k, x in _pool(g, c, 1, n).items()}
        s["table"], s["lens"] = _table(g, need, max(need), n), _ints(lens)
        s["seq"] = _ints([i for i in range(n_seq) for _ in range(t)])
        s["pos"] = _ints([x + j for x in start for j in range(t)])
        T = n_seq * t
        s["q"] = 2 * torch.randn((T, c["heads"], c["hd"]), device=DEV, generator=g)
        s["kn"] = 2 * torch.randn((T, c["kv"], c["hd"]), device=DEV, generator=g)
        s["vn"] = torch.randn((T, c["kv"], c["hd"]), device=DEV, generator=g)
        s["qw"] = 1 + 0.1 * torch.randn(c["hd"], device=DEV, generator=g)
        s["kw"] = 1 + 0.1 * torch.randn(c["hd"], device=DEV, generator=g)
        s["q_out"] = torch.empty_like(s["q"])
        if c["int8"]:  # the values that the 8-bit pages stand for
            s["kf"] = torch.empty(s["k"].shape, dtype=torch.float16, device=DEV)
            s["vf"] = torch.empty(s["v"].shape, dtype=torch.float16, device=DEV)
    elif c["kind"] == "refork":
        P, B = c["parents"], c["beams"]
        lens = _lens(c, P, "parents")
        need = _pages(lens, c["page"])
        n = sum(need) + P * B + 5
        s |= _pool(g, c, c["layers"], n)
        table = _table(g, need, max(need) + 1, n)
        s["table"] = torch.cat([table, torch.full((P * B, max(need) + 1), -1, dtype=torch.int32, device=DEV)])
        s["lens"] = _ints(lens + [0] * (P * B))
        s["refs"] = torch.zeros(n, dtype=torch.int32, device=DEV)
        s["refs"][table[table >= 0].long()] = 1
        order = torch.randperm(P * B, device=DEV, generator=g) % P  # which parent each beam continues
        s["parents"] = torch.cat([torch.full((P,), -1, device=DEV), order]).to(torch.int32)
        s["gone"] = _ints([0] * P + [1] * (P * B))
        s["ws"], s["status"] = torch.empty(WS_BYTES, dtype=torch.uint8, device=DEV), _ints([0])
    elif c["kind"] == "compact":
        R = c["rows"]
        la, lb = _lens(c, R, "a"), _lens(c, R, "b")
        na, nb = _pages(la, c["page"]), _pages(lb, c["page"])
        n = sum(na) + sum(nb) + 3
        s |= _pool(g, c, c["layers"], n)
        width = max(na + nb)
        s["table"] = torch.cat([torch.full((R, width), -1, dtype=torch.int32, device=DEV),
                                _table(g, nb, width, sum(nb))])
        s["refs"] = torch.zeros(n, dtype=torch.int32, device=DEV)
        s["refs"][:sum(nb)] = 1
        s["lens"] = _ints([0] * R + lb)
        s["to_a"], s["to_b"] = _ints(la + [0] * R), _ints([0] * R + lb)
        s["is_a"], s["is_b"] = _ints([1] * R + [0] * R), _ints([0] * R + [1] * R)
        s["ws"] = torch.empty(WS_BYTES, dtype=torch.uint8, device=DEV)
        s["status"], s["live"] = _ints([0]), _ints([0])
    else:
        n, V = c["rows"], c["vocab"]
        s["z"] = 3 * torch.randn((n, V), device=DEV, generator=g)
        # text repeats itself: low ids are common
        u = torch.rand((n, c["history"]), device=DEV, generator=g)
        s["hist"] = (V * u ** 4).to(torch.int32).clamp_(max=V - 1)
        h = c["history"]
        r = random.Random(h)
        hl = [h] + [r.randint(0, h) for _ in range(n - 1)]
        s["hist_len"], s["prompt_len"] = _ints(hl), _ints([x // 2 for x in hl])
        s["rep"] = 1 + 0.3 * torch.rand(n, device=DEV, generator=g)
        s["freq"], s["pres"] = (torch.rand(n, device=DEV, generator=g) for _ in range(2))
        s["bias_ids"] = s["bias"] = s["mask"] = None
        if c["bias"]:
            ids = torch.rand((n, V), device=DEV, generator=g).topk(min(V, c["bias"]), dim=1).indices
            s["bias_ids"] = ids.to(torch.int32)
            s["bias"] = 5 * torch.randn(ids.shape, device=DEV, generator=g)
        if c["mask"]:  # a grammar state: about a quarter of the words of 32 tokens allow some of theirs
            w = torch.randint(-2 ** 31, 2 ** 31, (n, -(-V // 32)), device=DEV, generator=g)
            w = w * (torch.rand(w.shape, device=DEV, generator=g) < 0.25)
            s["mask"] = w.to(torch.int32)
        s["out"] = torch.empty_like(s["z"])
    return s


# ------------------------------------------------------------------ plain forms
def _attend(s):
    c = s["c"]
    n, kv, hd, ps = c["seqs"], c["kv"], c["hd"], c["page"]
    ids = s["table"].clamp(min=0).long()
    S = ids.shape[1] * ps
    k, v = s["k"][ids].float(), s["v"][ids].float()  # [n][P][kv][ps][hd], [n][P][kv][hd][ps]
    if c["int8"]:
        k = k * s["ks"][ids][..., None]
        v = v * s["vs"][ids][:, :, :, None, :]
    k = k.permute(0, 2, 4, 1, 3).reshape(n, kv, hd, S)
    v = v.permute(0, 2, 1, 4, 3).reshape(n, kv, S, hd)
    z = torch.matmul(s["q"].view(n, kv, -1, hd), k) / math.sqrt(hd)
    dead = torch.arange(S, device=DEV) >= s["lens"][:, None]
    z = z.masked_fill(dead[:, None, None], -math.inf)
    m = z.amax(-1, keepdim=True)
    e = torch.exp(z - m.masked_fill(m == -math.inf, 0))
    o = torch.matmul(e, v) / e.sum(-1, keepdim=True).clamp(min=1e-30)
    return o.reshape(n, -1, hd)


def _rotated(x, w, pos):
    """RMS norm with w over each head, then the pairs (j, j + hd/2) turned by pos theta^(-2j/hd)."""
    hd = x.shape[-1]
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    j = torch.arange(hd // 2, device=DEV, dtype=torch.float64)
    a = pos.double()[:, None] * THETA ** (-2 * j / hd)
    cs, sn = torch.cos(a).float()[:, None], torch.sin(a).float()[:, None]
    x0, x1 = x[..., :hd // 2], x[..., hd // 2:]
    return torch.cat([x0 * cs - x1 * sn, x1 * cs + x0 * sn], -1)


def _prep(s):
    ps, pos = s["c"]["page"], s["pos"].long()
    q = _rotated(s["q"], s["qw"], pos)
    k, v = _rotated(s["kn"], s["kw"], pos), s["vn"]
    page, off = s["table"][s["seq"].long(), pos // ps].long(), pos % ps
    if s["c"]["int8"]:
        ka, va = k.abs().amax(-1, keepdim=True), v.abs().amax(-1, keepdim=True)
        s["ks"][page, :, off], s["vs"][page, :, off] = ka[..., 0] / 127, va[..., 0] / 127
        k = torch.round(k * (127 / ka)).clamp(-127, 127)
        v = torch.round(v * (127 / va)).clamp(-127, 127)
    s["k"][page, :, off] = k.to(s["k"].dtype)
    s["v"][page, :, :, off] = v.to(s["v"].dtype)
    return q


def _held(s):
    """[rows][width]: whether a table entry names a page of its row."""
    ps = s["c"]["page"]
    return torch.arange(s["table"].shape[1], device=DEV) < ((s["lens"] + ps - 1) // ps)[:, None]


def _refer(s, which, by):
    s["refs"].index_add_(0, s["table"].clamp(min=0).flatten().long(), by * which.flatten().to(torch.int32))


def _free(s, gone):
    gone = gone[:, None] != 0
    _refer(s, _held(s) & gone, -1)
    s["table"].masked_fill_(gone, -1)
    s["lens"].masked_fill_(gone[:, 0], 0)


def _lowest_free(s, need, asked):
    """The free pages in rising order, each row's first place among them, and whether there is enough for it."""
    order = torch.argsort((s["refs"] > 0).to(torch.int32), stable=True).to(torch.int32)
    total = torch.cumsum(need, 0)
    return order, total - need, asked & (total <= (s["refs"] == 0).sum())


def _extend(s, to):
    ps = s["c"]["page"]
    have, want = (s["lens"] + ps - 1) // ps, (to + ps - 1) // ps
    asked = to > s["lens"]
    need = torch.where(asked, want - have, 0)
    order, at, served = _lowest_free(s, need, asked)
    slot = torch.arange(s["table"].shape[1], device=DEV) - have[:, None]
    take = served[:, None] & (slot >= 0) & (slot < need[:, None])
    s["table"].copy_(torch.where(take, order[(at[:, None] + slot).clamp(0, len(order) - 1).long()], s["table"]))
    _refer(s, take, 1)
    s["lens"].copy_(torch.where(served, to, s["lens"]))
    s["status"].copy_((asked & ~served).sum()[None])


def _copy_pages(s, src):
    """Page p of every layer becomes the old page src[p]."""
    for t in ("k", "v", "ks", "vs"):
        if s[t] is not None:
            s[t].copy_(s[t][:, src])


def _fork(s, parents):
    ps, N = s["c"]["page"], len(s["refs"])
    p = parents.clamp(min=0).long()
    asked = (parents >= 0) & (s["lens"] == 0) & (s["lens"][p] > 0)
    full = s["lens"][p] // ps
    need = (asked & (s["lens"][p] % ps > 0)).to(torch.int32)
    order, at, served = _lowest_free(s, need, asked)
    new = order[at.clamp(0, N - 1).long()]
    slot = torch.arange(s["table"].shape[1], device=DEV)
    rows = torch.where(slot < full[:, None], s["table"][p], -1)
    tail = (slot == full[:, None]) & (need > 0)[:, None]
    old = s["table"][p].gather(1, full[:, None].clamp(max=s["table"].shape[1] - 1).long())[:, 0]
    rows = torch.where(tail, new[:, None], rows)
    s["table"].copy_(torch.where(served[:, None], rows, s["table"]))
    _refer(s, served[:, None] & (rows >= 0), 1)
    s["lens"].copy_(torch.where(served, s["lens"][p], s["lens"]))
    s["status"].copy_(((parents >= 0) & ~served).sum()[None])
    src = torch.arange(N + 1, device=DEV)
    src.scatter_(0, torch.where(served & (need > 0), new, N).long(), old.long())
    _copy_pages(s, src[:N])


def _compact(s):
    N = len(s["refs"])
    ids = torch.arange(N, device=DEV)
    used = s["refs"] > 0
    live = used.sum()
    holes, movers = ~used & (ids < live), used & (ids >= live)
    to = torch.argsort((~holes).to(torch.int32), stable=True)[(torch.cumsum(movers, 0) - 1).clamp(min=0)]
    to = torch.where(movers, to, ids)
    s["table"].copy_(torch.where(s["table"] >= 0, to[s["table"].clamp(min=0).long()].to(torch.int32), s["table"]))
    s["refs"].copy_(torch.zeros_like(s["refs"]).index_add_(0, to, s["refs"]))
    src = torch.arange(N + 1, device=DEV)
    src.scatter_(0, torch.where(movers, to, N), ids)
    _copy_pages(s, src[:N])
    s["live"].copy_(live[None])


def _logits(s):
    n, V = s["z"].shape
    at = torch.arange(s["hist"].shape[1], device=DEV)
    said = at < s["hist_len"][:, None]
    made = said & (at >= s["prompt_len"][:, None])
    h = s["hist"].long()
    seen = torch.zeros((n, V), dtype=torch.int32, device=DEV).scatter_add_(1, h, said.to(torch.int32)) > 0
    count = torch.zeros((n, V), dtype=torch.int32, device=DEV).scatter_add_(1, h, made.to(torch.int32))
    z, r = s["z"], s["rep"][:, None]
    z = torch.where(seen, torch.where(z > 0, z / r, z * r), z)
    z = z - count * s["freq"][:, None] - (count > 0) * s["pres"][:, None]
    if s["bias"] is not None:
        z = z.scatter_add(1, s["bias_ids"].long(), s["bias"])
    if s["mask"] is not None:
        t = torch.arange(V, device=DEV)
        z = torch.where((s["mask"][:, t // 32] >> (t % 32).to(torch.int32)) & 1 != 0, z, -math.inf)
    return z


def _pool_out(s):
    return [s["k"], s["v"]] + ([s["ks"], s["vs"]] if s["ks"] is not None else [])


def _values(s):
    """The cache as the values that it stands for."""
    if not s["c"]["int8"]:
        return [s["k"], s["v"]]
    torch.mul(s["k"], s["ks"][..., None], out=s["kf"])
    torch.mul(s["v"], s["vs"][:, :, None], out=s["vf"])
    return [s["kf"], s["vf"], s["ks"], s["vs"]]


def _run_plain(s):
    if s["kind"] == "attend":
        return _attend(s)
    if s["kind"] == "prep":
        return [_prep(s)] + _values(s)
    if s["kind"] == "refork":
        _free(s, s["gone"])
        _fork(s, s["parents"])
        return [s["table"], s["lens"], s["refs"], s["status"]] + _pool_out(s)
    if s["kind"] == "compact":
        _extend(s, s["to_a"])
        _free(s, s["is_b"])
        _compact(s)
        _extend(s, s["to_b"])
        _free(s, s["is_a"])
        _compact(s)
        return [s["table"], s["lens"], s["refs"], s["status"], s["live"]] + _pool_out(s)
    return _logits(s)


# ------------------------------------------------------------------ the framework's operators
def _run_own(s):
    from mnemocuda_amd import ops
    c = s["c"]
    if s["kind"] == "attend":
        ops.paged_attention_decode(s["q"], s["k"], s["v"], s["table"], s["lens"], s["out"], 1 / math.sqrt(c["hd"]),
                                   s["ws"], s["ks"], s["vs"])
        return s["out"]
    if s["kind"] == "prep":
        ops.paged_attn_prep(s["q"], s["kn"], s["vn"], s["qw"], s["kw"], EPS, THETA, s["k"], s["v"], s["table"],
                            s["q_out"], s["pos"], s["seq"], s["ks"], s["vs"])
        return [s["q_out"]] + _values(s)
    if s["kind"] == "refork":
        ops.kv_pages_free(s["table"], s["lens"], s["refs"], s["gone"], c["page"])
        ops.kv_pages_fork(s["table"], s["lens"], s["refs"], s["parents"], s["k"], s["v"], s["status"], s["ws"],
                          s["ks"], s["vs"])
        return [s["table"], s["lens"], s["refs"], s["status"]] + _pool_out(s)
    if s["kind"] == "compact":
        for to, gone in ((s["to_a"], s["is_b"]), (s["to_b"], s["is_a"])):
            ops.kv_pages_extend(s["table"], s["lens"], s["refs"], to, c["page"], s["status"])
            ops.kv_pages_free(s["table"], s["lens"], s["refs"], gone, c["page"])
            ops.kv_pages_compact(s["table"], s["refs"], s["k"], s["v"], s["live"], s["ws"], s["ks"], s["vs"])
        return [s["table"], s["lens"], s["refs"], s["status"], s["live"]] + _pool_out(s)
    ops.logits_process(s["z"], s["out"], s["hist"], s["hist_len"], s["prompt_len"], s["rep"], s["freq"], s["pres"],
                       s["bias_ids"], s["bias"], s["mask"])
    return s["out"]


def run(state):
    if own:
        return _run_own(state)
    return _run_plain(state)


# ------------------------------------------------------------------ work
def _page_bytes(c):
    return c["layers"] * c["kv"] * c["page"] * ((c["hd"] + 4) * 2 if c["int8"] else c["hd"] * 4)


def work(case):
    c = case
    if c["kind"] == "attend":
        lens = _lens(c, c["seqs"])
        per = c["kv"] * ((c["hd"] + 4) * 2 if c["int8"] else c["hd"] * 4)
        return {"bytes": sum(lens) * per + 8 * c["seqs"] * c["heads"] * c["hd"] + 4 * sum(_pages(lens, c["page"])),
                "flops": 4 * sum(lens) * c["heads"] * c["hd"]}
    if c["kind"] == "prep":
        T = c["seqs"] * c["tokens"]
        kv = c["kv"] * (8 * c["hd"] + ((c["hd"] + 4) * 2 if c["int8"] else c["hd"] * 4))
        return {"bytes": T * (8 * c["heads"] * c["hd"] + kv + 8), "flops": 9 * T * (c["heads"] + c["kv"]) * c["hd"]}
    if c["kind"] == "refork":
        lens = _lens(c, c["parents"], "parents")
        part = sum(x % c["page"] > 0 for x in lens) * (1 + c["beams"])  # read once, written for each beam
        held = sum(_pages(lens, c["page"])) * c["beams"]
        refs = sum(_pages(lens, c["page"])) + c["parents"] * c["beams"]
        return {"bytes": part * _page_bytes(c) + 12 * held + 8 * refs, "flops": 0}
    if c["kind"] == "compact":
        na, nb = (sum(_pages(_lens(c, c["rows"], w), c["page"])) for w in "ab")
        # each half of the pass moves the smaller group's pages down over the other's
        return {"bytes": 2 * (2 * min(na, nb) * _page_bytes(c) + 16 * (na + nb)), "flops": 0}
    n, V = c["rows"], c["vocab"]
    r = random.Random(c["history"])
    said = c["history"] + sum(r.randint(0, c["history"]) for _ in range(n - 1))
    return {"bytes": n * V * 8 + (n * (-(-V // 32)) * 4 if c["mask"] else 0) + 4 * said + 8 * n * c["bias"],
            "flops": 6 * n * V}


# ------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    """What run returns, from the definitions in 64 bits, one sequence or row at a time.  Page upkeep moves values and
    whole numbers only: nothing there has a rounding."""
    c, s = case, prepare(case, seed)
    if c["kind"] == "attend":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
        G = c["heads"] // c["kv"]
        for i, L in enumerate(_lens(c, c["seqs"])):
            if L == 0:
                continue
            pages = s["table"][i, :-(-L // c["page"])].long()
            for h in range(c["kv"]):
                K = s["k"][pages, h].double()
                V = s["v"][pages, h].double().transpose(1, 2)
                if c["int8"]:
                    K = K * s["ks"][pages, h].double()[..., None]
                    V = V * s["vs"][pages, h].double()[..., None]
                K, V = K.reshape(-1, c["hd"])[:L], V.reshape(-1, c["hd"])[:L].contiguous()
                w = torch.softmax(s["q"][i, h * G:(h + 1) * G].double() @ K.T.contiguous() * c["hd"] ** -0.5, -1)
                out[i, h * G:(h + 1) * G] = w @ V
        return out
    if c["kind"] == "prep":
        hd = c["hd"]
        freq = torch.exp(torch.arange(0, hd, 2, device=DEV, dtype=torch.float64) * (-math.log(THETA) / hd))
        turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV), s["pos"].double()[:, None] * freq)[:, None]

        def turned(x, w):
            x = x.double()
            x = w.double() * x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt()
            y = torch.complex(x[..., :hd // 2].contiguous(), x[..., hd // 2:].contiguous()) * turn
            return torch.cat([y.real, y.imag], -1)

        rows = [turned(s["kn"], s["kw"]), s["vn"].double()]
        pools = [s["k"].double(), s["v"].double().transpose(2, 3).contiguous()]
        scales = [s["ks"].double(), s["vs"].double()] if c["int8"] else []
        page = s["table"][s["seq"].long(), (s["pos"] // c["page"]).long()].long()
        off = (s["pos"] % c["page"]).long()
        for i in range(2):
            x = rows[i]
            if c["int8"]:
                step = x.abs().amax(-1) / 127
                scales[i][page, :, off] = step
                pools[i] = pools[i] * (s["ks"], s["vs"])[i].double()[..., None]
                x = torch.round(x / step[..., None]) * step[..., None]
            pools[i][page, :, off] = x
        return [turned(s["q"], s["qw"]), pools[0], pools[1].transpose(2, 3).contiguous()] + scales
    if c["kind"] in ("refork", "compact"):
        return None
    out = torch.empty(s["z"].shape, dtype=torch.float64, device=DEV)
    hist_len, prompt_len = s["hist_len"].tolist(), s["prompt_len"].tolist()
    for i in range(c["rows"]):
        z, h, V = s["z"][i].double(), s["hist"][i].long(), c["vocab"]
        seen = torch.bincount(h[:hist_len[i]], minlength=V) > 0
        count = torch.bincount(h[prompt_len[i]:hist_len[i]], minlength=V)
        r = s["rep"][i].double()
        z[seen] = torch.minimum(z[seen] * r, z[seen] / r)  # r >= 1: toward minus infinity either way
        z -= count * s["freq"][i].double() + (count > 0) * s["pres"][i].double()
        if s["bias"] is not None:
            z[s["bias_ids"][i].long()] += s["bias"][i].double()
        if s["mask"] is not None:
            bits = (s["mask"][i].long()[:, None] >> torch.arange(32, device=DEV)) & 1
            z[bits.flatten()[:V] == 0] = -math.inf
        out[i] = z
    return out
