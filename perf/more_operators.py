"""Operators of batches that hold prompts: attention of many new tokens per sequence over the paged cache,
low-rank adapters of several requests beside a shared projection, routing of all tokens to their experts, and
log probabilities of given tokens.

Shapes follow the library's benchmark configuration (hidden 4096, 64 query / 4 KV heads of 128, 128 experts of
which 8 are taken, vocabulary 151,936) and generic ones around it.  With `own` false every case runs in elementary
torch operations; with `own` true through mnemocuda_amd.ops.

Page layout: K [page][kv head][position][dim], V [page][kv head][dim][position], int8 scales
[page][kv head][position]; a table row lists a sequence's pages (-1: none).  Adapters: A [adapter][rank][in],
B [adapter][out][rank].
"""
import math
import random

import torch

own = False

DEV = "cuda"


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # drafted tokens of five conversations are verified: latency of a call with few rows
        {"name": "attend_draft", "kind": "attend", "seqs": 5, "new_lo": 3, "new_hi": 6, "lo": 400, "hi": 5000,
         "heads": 64, "kv": 4, "hd": 128, "page": 64, "int8": False},
        # a fresh prompt of one request
        {"name": "attend_prompt", "kind": "attend", "seqs": 1, "new_lo": 2000, "new_hi": 2000, "lo": 0, "hi": 0,
         "heads": 64, "kv": 4, "hd": 128, "page": 64, "int8": False},
        # chunks of three long documents, over an 8-bit cache
        {"name": "attend_chunks_int8", "kind": "attend", "seqs": 3, "new_lo": 300, "new_hi": 512, "lo": 6000, "hi": 30000,
         "heads": 64, "kv": 8, "hd": 128, "page": 32, "int8": True},
        # a mixed step of a small model: some prompts, some single tokens, one row idle; no shared heads
        {"name": "attend_mixed_hd64", "kind": "attend", "seqs": 25, "new_lo": 1, "new_hi": 700, "lo": 0, "hi": 1500,
         "heads": 12, "kv": 12, "hd": 64, "page": 16, "int8": False},
        # a decode step's batch with 128 experts
        {"name": "route_decode", "kind": "route", "tokens": 33, "experts": 128, "k": 8, "sigmoid": False, "bias": False,
         "groups": 1, "top_groups": 1, "best": 1, "renorm": True},
        # prompts, scores balanced by a bias, experts in groups
        {"name": "route_groups", "kind": "route", "tokens": 8191, "experts": 256, "k": 8, "sigmoid": True, "bias": True,
         "groups": 8, "top_groups": 4, "best": 2, "renorm": True},
        # a single conversation with its adapter: latency of a call
        {"name": "lora_one", "kind": "lora", "tokens": 1, "runs": 1, "adapters": 4, "rank": 16, "max_rank": 16, "in": 4096,
         "out": 4096, "bf16": False},
        # decoding requests, an adapter for most of them, ranks of their own
        {"name": "lora_decode", "kind": "lora", "tokens": 61, "runs": 61, "adapters": 40, "rank": 8, "max_rank": 64,
         "in": 4096, "out": 8192, "bf16": False},
        # prompts of seven requests
        {"name": "lora_prompts", "kind": "lora", "tokens": 3001, "runs": 7, "adapters": 5, "rank": 16, "max_rank": 32,
         "in": 4096, "out": 8192, "bf16": True},
        # the token just drawn, with its alternatives
        {"name": "logprobs_one", "kind": "logprobs", "rows": 1, "vocab": 151936, "top": 20, "masked": 0.0},
        # a small model's batch under a grammar
        {"name": "logprobs_31_small", "kind": "logprobs", "rows": 31, "vocab": 32003, "top": 5, "masked": 0.7},
        # a prompt is scored
        {"name": "logprobs_prompt", "kind": "logprobs", "rows": 1201, "vocab": 151936, "top": 5, "masked": 0.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend"] * 5 + ["lora"] * 3 + ["route"] * 2 + ["logprobs"] * 2)
    while True:
        if kind == "attend":
            kv = rng.choice([1, 2, 3, 4, 8])
            new, ctx = _log(rng, 1, 4000), rng.choice([0, _log(rng, 1, 60000)])
            c = {"kind": kind, "seqs": _log(rng, 1, 64), "new_lo": rng.randint(1, new), "new_hi": new,
                 "lo": rng.randint(0, ctx), "hi": ctx, "heads": kv * rng.randint(1, 16), "kv": kv,
                 "hd": rng.choice([64, 128, 128, 256]), "page": rng.choice([16, 32, 64, 128]), "int8": rng.random() < 0.4}
            # the plain form's scores of one sequence and the cache have to fit as well
            if c["heads"] * new * (new + ctx) > 1 << 30 or c["seqs"] * (new + ctx) * kv * c["hd"] > 1 << 30:
                continue
        elif kind == "route":
            groups = rng.choice([1, 1, 2, 4, 8])
            experts = groups * _log(rng, 4, 512 // groups)
            top_groups = rng.randint(1, groups)
            k = rng.randint(1, min(16, experts // groups * top_groups))
            c = {"kind": kind, "tokens": _log(rng, 1, 8191), "experts": experts, "k": k, "sigmoid": rng.random() < 0.5,
                 "bias": rng.random() < 0.5, "groups": groups, "top_groups": top_groups, "best": rng.randint(1, 2),
                 "renorm": rng.random() < 0.7}
        elif kind == "lora":
            tokens = _log(rng, 1, 3001)
            top = rng.choice([8, 16, 32, 64, 128, 256])
            c = {"kind": kind, "tokens": tokens, "runs": rng.choice([tokens, rng.randint(1, min(tokens, 64))]),
                 "adapters": _log(rng, 1, 40), "rank": rng.randint(1, top), "max_rank": top, "in": 8 * _log(rng, 16, 1024),
                 "out": _log(rng, 32, 12000), "bf16": rng.random() < 0.5}
        else:
            c = {"kind": kind, "rows": _log(rng, 1, 1201), "vocab": _log(rng, 100, 151936), "top": rng.choice([0, 1, rng.randint(2, 32)]),
                 "masked": rng.choice([0.0, 0.0, rng.random()])}
        w = work(c)
        if w["bytes"] <= 7e8 and w["flops"] <= 9e11:
            return c


def _spread(n, lo, hi, what):
    """n lengths of a case, the same for every seed, spread over their logarithm, the longest first."""
    r = random.Random("%s %d %d %d" % (what, n, lo, hi))
    return [hi] + [min(hi, max(lo, _log(r, lo + 1, hi + 1) - 1)) for _ in range(n - 1)]


def _lens(c):
    """(new tokens, positions after them) of each sequence; of 8 sequences or more one takes no token, one is empty."""
    new, before = _spread(c["seqs"], c["new_lo"], c["new_hi"], "new"), _spread(c["seqs"], c["lo"], c["hi"], "before")
    random.Random(c["seqs"]).shuffle(before)
    if c["seqs"] >= 8:
        new[3], new[6], before[6] = 0, 0, 0
    return new, [a + b for a, b in zip(new, before)]


def _ids(c):
    """The adapter of each token, the same for every seed: runs of tokens of one request, some requests without."""
    r = random.Random("%d %d %d" % (c["tokens"], c["runs"], c["adapters"]))
    cuts = sorted(r.sample(range(1, c["tokens"]), c["runs"] - 1)) + [c["tokens"]]
    ids, at = [], 0
    for i, to in enumerate(cuts):
        a = r.randrange(c["adapters"]) if i == 0 or r.random() < 0.9 else -1
        ids += [a] * (to - at)
        at = to
    return ids


def _ranks(c):
    r = random.Random("%d %d %d" % (c["adapters"], c["rank"], c["max_rank"]))
    return [c["rank"]] + [r.choice([c["rank"], r.randint(c["rank"], c["max_rank"]), c["max_rank"]])
                          for _ in range(c["adapters"] - 1)]


def _pages(lens, page):
    return [-(-x // page) for x in lens]


# ------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _randn(g, *shape):
    return torch.randn(shape, device=DEV, generator=g)


def prepare(case, seed):
    c, g = case, _gen(seed)
    s = {"c": c, "kind": c["kind"]}
    if own:
        from mnemocuda_amd import ops
    if c["kind"] == "attend":
        kv, ps, hd = c["kv"], c["page"], c["hd"]
        s["new"], s["len"] = _lens(c)
        need = _pages(s["len"], ps)
        n = sum(need) + 2
        if c["int8"]:
            s["k"] = torch.randint(-127, 128, (n, kv, ps, hd), dtype=torch.int8, device=DEV, generator=g)
            s["v"] = torch.randint(-127, 128, (n, kv, hd, ps), dtype=torch.int8, device=DEV, generator=g)
            s["ks"], s["vs"] = ((0.5 + torch.rand((n, kv, ps), device=DEV, generator=g)) * 0.02 for _ in range(2))
        else:
            s["k"] = torch.randn((n, kv, ps, hd), dtype=torch.float16, device=DEV, generator=g)
            s["v"] = torch.randn((n, kv, hd, ps), dtype=torch.float16, device=DEV, generator=g)
            s["ks"] = s["vs"] = None
        ids = torch.randperm(n, device=DEV, generator=g).to(torch.int32)
        s["table"] = torch.full((c["seqs"], max(need)), -1, dtype=torch.int32, device=DEV)
        at, starts = 0, [0]
        for i, m in enumerate(need):
            s["table"][i, :m] = ids[at:at + m]
            at += m
            starts.append(starts[-1] + s["new"][i])
        s["starts"], s["lens"] = _ints(starts), _ints(s["len"])
        # normalised query heads of several sharpnesses
        s["q"] = _randn(g, starts[-1], c["heads"], hd) * \
            (0.5 + 1.5 * torch.rand((1, c["heads"], 1), device=DEV, generator=g))
        if own:
            s["out"] = torch.empty_like(s["q"])
            s["ws"] = torch.empty(ops.paged_attention_prompt_workspace_bytes(c["heads"], kv, hd), dtype=torch.uint8,
                                  device=DEV)
    elif c["kind"] == "route":
        n, e, k = c["tokens"], c["experts"], c["k"]
        s["z"] = 1.5 * _randn(g, n, e)
        # what balances the load over training: of the size of the scores' own differences
        s["bias"] = _randn(g, e) * (0.1 if c["sigmoid"] else 0.3 / e) if c["bias"] else None
        if own:
            s["idx"], s["w"] = torch.empty((n, k), dtype=torch.int32, device=DEV), torch.empty((n, k), device=DEV)
    elif c["kind"] == "lora":
        t = torch.bfloat16 if c["bf16"] else torch.float16
        s["x"], s["base"] = _randn(g, c["tokens"], c["in"]), _randn(g, c["tokens"], c["out"])
        s["a"] = (_randn(g, c["adapters"], c["max_rank"], c["in"]) * c["in"] ** -0.5).to(t)
        s["b"] = (_randn(g, c["adapters"], c["out"], c["max_rank"]) * c["max_rank"] ** -0.5).to(t)
        ids, s["rank"] = _ids(c), _ranks(c)
        s["ids"], s["ranks"] = _ints(ids), _ints(s["rank"])
        s["scales"] = 0.5 + torch.rand(c["adapters"], device=DEV, generator=g)
        # which tokens each adapter has
        s["of"] = {a: torch.tensor([i for i, b in enumerate(ids) if b == a], device=DEV) for a in sorted(set(ids)) if a >= 0}
        if own:
            s["out"] = torch.empty_like(s["base"])
            s["ws"] = torch.empty(ops.lora_workspace_bytes(c["tokens"], c["in"], c["max_rank"]), dtype=torch.uint8,
                                  device=DEV)
    else:
        n, V = c["rows"], c["vocab"]
        s["z"] = 3 * _randn(g, n, V)
        s["t"] = torch.randint(0, V, (n,), dtype=torch.int32, device=DEV, generator=g)
        # half the rows ask for a likely token
        s["t"][::2] = s["z"][::2].argmax(1).to(torch.int32)
        if c["masked"]:
            keep = s["z"].gather(1, s["t"].long()[:, None])
            s["z"].masked_fill_(torch.rand((n, V), device=DEV, generator=g) < c["masked"], -math.inf)
            s["z"].scatter_(1, s["t"].long()[:, None], keep)
        if own:
            k = c["top"]
            s["logp"], s["ent"] = torch.empty(n, device=DEV), torch.empty(n, device=DEV)
            s["rank"] = torch.empty(n, dtype=torch.int32, device=DEV)
            s["ids"] = torch.empty((n, k), dtype=torch.int32, device=DEV) if k else None
            s["tops"] = torch.empty((n, k), device=DEV) if k else None
            s["ws"] = torch.empty(ops.logprobs_workspace_bytes(n, V, k), dtype=torch.uint8, device=DEV)
    return s


# ------------------------------------------------------------------ plain forms
def _cache(s, i):
    """K [kv][L][hd] and V [kv][L][hd] of sequence i in 32 bits."""
    c, L = s["c"], s["len"][i]
    pages = s["table"][i, :-(-L // c["page"])].long()
    k, v = s["k"][pages].float(), s["v"][pages].float()
    if c["int8"]:
        k = k * s["ks"][pages][..., None]
        v = v * s["vs"][pages][:, :, None]
    k = k.permute(1, 0, 2, 3).reshape(c["kv"], -1, c["hd"])[:, :L]
    v = v.permute(1, 0, 3, 2).reshape(c["kv"], -1, c["hd"])[:, :L]
    return k, v


def _attend(s):
    c, out, at = s["c"], torch.empty_like(s["q"]), 0
    kv, hd = c["kv"], c["hd"]
    for i, n in enumerate(s["new"]):
        if n == 0:
            continue
        L = s["len"][i]
        k, v = _cache(s, i)
        q = s["q"][at:at + n].view(n, kv, -1, hd).permute(1, 2, 0, 3).reshape(kv, -1, hd)  # [kv][head][token]
        z = torch.matmul(q, k.transpose(1, 2).contiguous()).view(kv, -1, n, L) / math.sqrt(hd)
        ahead = torch.arange(L, device=DEV) > (L - n + torch.arange(n, device=DEV))[:, None]
        z = z.masked_fill_(ahead, -math.inf)
        e = torch.exp_(z.sub_(z.amax(-1, keepdim=True)))
        o = torch.matmul(e.view(kv, -1, L), v).view(kv, -1, n, hd) / e.sum(-1, keepdim=True)
        out[at:at + n] = o.permute(2, 0, 1, 3).reshape(n, -1, hd)
        at += n
    return out


def _route(s):
    """The choice is made among scores in 64 bits, where two that differ are told apart."""
    c, z = s["c"], s["z"].double()
    n, E, k, G = c["tokens"], c["experts"], c["k"], c["groups"]
    if c["sigmoid"]:
        p = 1 / (1 + torch.exp(-z))
    else:
        p = torch.exp(z - z.amax(1, keepdim=True))
        p = p / p.sum(1, keepdim=True)
    t = p if s["bias"] is None else p + s["bias"].double()
    if c["top_groups"] < G:
        by_group = torch.sort(t.view(n, G, -1), 2, descending=True).values
        score = by_group[:, :, 0] + by_group[:, :, 1] if c["best"] == 2 and E > G else by_group[:, :, 0]
        kept = torch.sort(score, dim=1, descending=True, stable=True).indices[:, :c["top_groups"]]
        on = torch.zeros((n, G), dtype=torch.bool, device=DEV).scatter_(1, kept, True)
        t = t.masked_fill(~on.repeat_interleave(E // G, 1), -math.inf)
    idx = torch.sort(t, dim=1, descending=True, stable=True).indices[:, :k]
    w = p.gather(1, idx)
    if c["renorm"]:
        w = w / w.sum(1, keepdim=True)
    return [idx.to(torch.int32), (w * 2.5).float()]


def _lora(s):
    out = s["base"].clone()
    for a, rows in s["of"].items():
        r = s["rank"][a]
        v = torch.matmul(s["x"][rows], s["a"][a, :r].float().t().contiguous())
        out[rows] += s["scales"][a] * torch.matmul(v, s["b"][a, :, :r].float().t().contiguous())
    return out


def _logprobs(s):
    z, k = s["z"], s["c"]["top"]
    t = s["t"].long()[:, None]
    zt = z.gather(1, t)
    m = z.amax(1, keepdim=True)
    d = z - m
    e = torch.exp(d)
    S = e.sum(1, keepdim=True)
    lse = torch.log(S)
    d.masked_fill_(d == -math.inf, 0)
    ent = (lse - (e.mul_(d)).sum(1, keepdim=True) / S)[:, 0]
    ids = torch.arange(z.shape[1], device=DEV)
    rank = ((z > zt) | ((z == zt) & (ids < t))).sum(1) + 1
    out = [(zt - m - lse)[:, 0], rank.to(torch.int32), ent]
    if k:
        # one whole number per token, larger for a larger logit, and for the lower id among equal ones
        bits = (z + 0.0).view(torch.int32).long()
        key = (torch.where(bits < 0, -(bits & 0x7fffffff), bits) << 32) | (0x7fffffff - ids)
        top = torch.topk(key, min(k, z.shape[1]), 1).values
        at = 0x7fffffff - (top & 0x7fffffff)
        val = z.gather(1, at)
        none = torch.isinf(val)
        out += [at.masked_fill(none, -1).to(torch.int32), (val - m - lse).masked_fill(none, -math.inf)]
        if k > z.shape[1]:
            more = (0, k - z.shape[1])
            out[3:] = [torch.nn.functional.pad(out[3], more, value=-1), torch.nn.functional.pad(out[4], more, value=-math.inf)]
    return out


# ------------------------------------------------------------------ the framework's operators
def _run_own(s):
    from mnemocuda_amd import ops
    c = s["c"]
    if s["kind"] == "attend":
        ops.paged_attention_prompt(s["q"], s["k"], s["v"], s["table"], s["starts"], s["lens"], s["out"],
                                   1 / math.sqrt(c["hd"]), s["ws"], s["ks"], s["vs"])
        return s["out"]
    if s["kind"] == "route":
        ops.moe_route(s["z"], s["idx"], s["w"], sigmoid=c["sigmoid"], bias=s["bias"], n_groups=c["groups"],
                      top_groups=c["top_groups"], group_best=c["best"], renormalise=c["renorm"], scale=2.5)
        return [s["idx"], s["w"]]
    if s["kind"] == "lora":
        ops.lora_add(s["x"], s["a"], s["b"], s["ids"], s["ranks"], s["scales"], s["base"], s["out"], s["ws"])
        return s["out"]
    ops.logprobs(s["z"], s["t"], s["logp"], s["rank"], s["ent"], s["ids"], s["tops"], s["ws"])
    return [s["logp"], s["rank"], s["ent"]] + ([s["ids"], s["tops"]] if c["top"] else [])


def run(state):
    if own:
        return _run_own(state)
    return {"attend": _attend, "route": _route, "lora": _lora, "logprobs": _logprobs}[state["kind"]](state)


# ------------------------------------------------------------------ work
def work(case):
    c = case
    if c["kind"] == "attend":
        new, lens = _lens(c)
        per = c["kv"] * ((c["hd"] + 4) * 2 if c["int8"] else c["hd"] * 4)
        pairs = sum(n * (L - n) + n * (n + 1) // 2 for n, L in zip(new, lens))
        held = sum(L for n, L in zip(new, lens) if n)
        return {"bytes": held * per + 8 * sum(new) * c["heads"] * c["hd"] + 4 * sum(_pages(lens, c["page"])),
                "flops": 4 * pairs * c["heads"] * c["hd"]}
    if c["kind"] == "route":
        return {"bytes": c["tokens"] * (4 * c["experts"] + 8 * c["k"]) + (4 * c["experts"] if c["bias"] else 0),
                "flops": 8 * c["tokens"] * c["experts"]}
    if c["kind"] == "lora":
        ids, ranks = _ids(c), _ranks(c)
        io = c["in"] + c["out"]
        return {"bytes": c["tokens"] * (4 * c["in"] + 8 * c["out"] + 4) + sum(2 * ranks[a] * io for a in set(ids) if a >= 0),
                "flops": 2 * io * sum(ranks[a] for a in ids if a >= 0)}
    return {"bytes": c["rows"] * (4 * c["vocab"] + 16 + 8 * c["top"]), "flops": 6 * c["rows"] * c["vocab"]}


# ------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    """What run returns, from the definitions in 64 bits, one head, adapter or row at a time."""
    c, s = case, prepare(case, seed)
    if c["kind"] == "attend":
        out, at = torch.empty(s["q"].shape, dtype=torch.float64, device=DEV), 0
        G = c["heads"] // c["kv"]
        for i, n in enumerate(s["new"]):
            L = s["len"][i]
            pages = s["table"][i, :-(-L // c["page"])].long()
            seen = torch.ones((n, L), dtype=torch.bool, device=DEV).tril(L - n)
            for h in range(c["heads"] if n else 0):
                K = s["k"][pages, h // G].double()
                V = s["v"][pages, h // G].double().transpose(1, 2)
                if c["int8"]:
                    K = K * s["ks"][pages, h // G].double()[..., None]
                    V = V * s["vs"][pages, h // G].double()[..., None]
                K, V = K.reshape(-1, c["hd"])[:L], V.reshape(-1, c["hd"])[:L].contiguous()
                z = s["q"][at:at + n, h].double() @ K.T.contiguous() * c["hd"] ** -0.5
                out[at:at + n, h] = torch.softmax(torch.where(seen, z, -math.inf), -1) @ V
            at += n
        return out
    if c["kind"] == "route":
        E, G, k = c["experts"], c["groups"], c["k"]
        z = s["z"].double()
        p = torch.sigmoid(z) if c["sigmoid"] else torch.softmax(z, 1)
        t = p + (0 if s["bias"] is None else s["bias"].double())
        idx = torch.empty((c["tokens"], k), dtype=torch.int32, device=DEV)
        per = E // G
        if c["top_groups"] < G:
            score = t.view(-1, G, per).topk(min(c["best"], per), 2).values.sum(2)
            worst = score.topk(c["top_groups"], 1).values[:, -1:]
            t = torch.where((score >= worst).repeat_interleave(per, 1), t, -math.inf)
        for j in range(k):
            best = t.argmax(1)
            idx[:, j] = best.to(torch.int32)
            t[torch.arange(len(t), device=DEV), best] = -math.inf
        w = p.gather(1, idx.long())
        return [idx, 2.5 * (w / w.sum(1, keepdim=True) if c["renorm"] else w)]
    if c["kind"] == "lora":
        out = s["base"].double()
        for a, rows in s["of"].items():
            r = s["rank"][a]
            W = s["b"][a, :, :r].double() @ s["a"][a, :r].double()
            out[rows] += s["scales"][a].double() * (s["x"][rows].double() @ W.T.contiguous())
        return out
    n, V, k = c["rows"], c["vocab"], c["top"]
    logp, ent = (torch.empty(n, dtype=torch.float64, device=DEV) for _ in range(2))
    rank = torch.empty(n, dtype=torch.int32, device=DEV)
    ids = torch.full((n, k), -1, dtype=torch.int32, device=DEV)
    tops = torch.full((n, k), -math.inf, dtype=torch.float64, device=DEV)
    for i in range(n):
        z = s["z"][i].double()
        y = z - torch.logsumexp(z, 0)
        p = y.exp()
        logp[i] = y[s["t"][i].long()]
        ent[i] = -(p * torch.where(p > 0, y, 0)).sum()
        order = torch.sort(z, descending=True, stable=True).indices
        rank[i] = (order == s["t"][i]).nonzero()[0, 0] + 1
        m = min(k, int((z > -math.inf).sum()))
        ids[i, :m], tops[i, :m] = order[:m].to(torch.int32), y[order[:m]]
    return [logp, rank, ent] + ([ids, tops] if k else [])
