"""Several sequences decoded together: page upkeep, preparation, attention, logits and sampling as a server strings
them together, eagerly and as one captured step, against a plain model in 64 bits that keeps each sequence's keys
and values in a list.

Bar of a step's attention, 1e-3 relative L2: the reference rounds the same values to f16 (2^-11 each) and may round a
few of them the other way, where fp32 and fp64 fall on different sides of a tie."""
import math

import numpy as np
import pytest
import torch

from tests.conftest import rel_l2
from tests.gpu_util import case, dev, host
from tests.test_gpu_paged_attn import rotated

pytestmark = pytest.mark.gpu

LAYERS, NH, NKV, HD, PS, VOCAB = 2, 8, 2, 64, 16, 500
ROWS, WIDTH, PAGES, MAX_HIST = 6, 10, 40, 160
THETA, EPS, SCALE = 1e4, 1e-6, 1 / math.sqrt(HD)
WQ, WK = NH * HD, NKV * HD
ROW = LAYERS * (WQ + 2 * WK)  # a token's q, k and v of every layer


class Server:
    """The batch on the device.  A token's queries, keys and values are rows of a table (the model has no mixing
    between layers), its logits a projection of the last layer's attention."""

    def __init__(self, gpu, table, head, graph):
        self.o, self.graph = gpu.ops, None
        self.table_w, self.head = dev(table), dev(head)
        z = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
        self.table, self.lens, self.refs = z(ROWS, WIDTH) - 1, z(ROWS), z(PAGES)
        self.new, self.active, self.status, self.live = z(ROWS), z(ROWS), z(1), z(1)
        self.k = torch.full((LAYERS, PAGES, NKV, PS, HD), float("nan"), dtype=torch.float16, device="cuda")
        self.v = torch.full((LAYERS, PAGES, NKV, HD, PS), float("nan"), dtype=torch.float16, device="cuda")
        self.tok, self.hist, self.prompt = z(ROWS), z(ROWS, MAX_HIST), z(ROWS)
        self.emb = torch.zeros((ROWS, ROW), device="cuda")
        self.q = [torch.zeros((ROWS, NH, HD), device="cuda") for _ in range(LAYERS)]
        self.kn = [torch.zeros((ROWS, NKV, HD), device="cuda") for _ in range(LAYERS)]
        self.vn = [torch.zeros((ROWS, NKV, HD), device="cuda") for _ in range(LAYERS)]
        self.out = [torch.zeros((ROWS, NH, HD), device="cuda") for _ in range(LAYERS)]
        self.logits = torch.zeros((ROWS, VOCAB), device="cuda")
        self.rep, self.freq, self.pres = (torch.full((ROWS,), x, device="cuda") for x in (1.2, 0.3, 0.1))
        self.bias_ids = torch.zeros((ROWS, 1), dtype=torch.int32, device="cuda") - 1
        self.bias = torch.zeros((ROWS, 1), device="cuda")
        self.mask = torch.full((ROWS, -(-VOCAB // 32)), -1, dtype=torch.int32, device="cuda")
        self.ws = torch.empty(self.o.paged_attention_workspace_bytes(NH, NKV, HD), dtype=torch.uint8, device="cuda")
        self.pws = torch.empty(self.o.kv_pages_workspace_bytes(ROWS, PAGES), dtype=torch.uint8, device="cuda")
        self.sws = torch.zeros(self.o.sample_workspace_bytes(), dtype=torch.uint8, device="cuda")
        self.want_graph = graph

    def _step(self):
        o = self.o
        torch.add(self.lens, self.active, out=self.new)
        o.kv_pages_extend(self.table, self.lens, self.refs, self.new, PS, self.status)
        # the token goes into the history at its position, its q, k and v come from the table
        self.hist.scatter_(1, (self.lens - 1).clamp(min=0).long()[:, None], self.tok[:, None])
        for r in range(ROWS):
            o.embedding_lookup(self.table_w, 0, self.tok[r:r + 1], VOCAB, self.emb[r], ROW)
        at = 0
        for i in range(LAYERS):
            for t, n in ((self.q[i], WQ), (self.kn[i], WK), (self.vn[i], WK)):
                t.view(ROWS, n).copy_(self.emb[:, at:at + n])
                at += n
            o.paged_attn_prep(self.q[i], self.kn[i], self.vn[i], None, None, EPS, THETA, self.k[i], self.v[i], self.table,
                              self.q[i], seq_lens=self.lens)
            o.paged_attention_decode(self.q[i], self.k[i], self.v[i], self.table, self.lens, self.out[i], SCALE, self.ws)
        for r in range(ROWS):
            o.matvec_f32(self.head, self.out[-1][r], self.logits[r], VOCAB, WQ)
        o.logits_process(self.logits, self.logits, self.hist, self.lens, self.prompt, self.rep, self.freq, self.pres,
                         self.bias_ids, self.bias, self.mask)
        for r in range(ROWS):
            o.sample_token_ws(self.logits[r], VOCAB, 0.0, 1.0, 7, self.sws, self.tok[r:r + 1])

    def step(self):
        if not self.want_graph:
            return self._step()
        if self.graph is None:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                self.graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(self.graph, stream=side):
                    self._step()
            torch.cuda.current_stream().wait_stream(side)
        self.graph.replay()

    def prompt_in(self, row, tokens):
        """A prompt's keys and values in one call per layer; the last token is left for the next step."""
        n = len(tokens) - 1
        to = torch.zeros(ROWS, dtype=torch.int32, device="cuda")
        to[row] = n
        self.o.kv_pages_extend(self.table, self.lens, self.refs, to, PS, self.status)
        assert int(host(self.status)[0]) == 0
        t = torch.tensor(tokens, device="cuda")
        self.hist[row] = 0
        self.hist[row, :n] = t[:n].int()
        self.prompt[row], self.tok[row], self.active[row] = len(tokens), tokens[-1], 1
        rows, pos = self.table_w[t[:n]], torch.arange(n, dtype=torch.int32, device="cuda")
        seq = torch.full((n,), row, dtype=torch.int32, device="cuda")
        at = 0
        for i in range(LAYERS):
            q, k, v = (rows[:, at + a:at + b].contiguous().view(n, -1, HD) for a, b in
                       ((0, WQ), (WQ, WQ + WK), (WQ + WK, WQ + 2 * WK)))
            at += WQ + 2 * WK
            self.o.paged_attn_prep(q, k, v, None, None, EPS, THETA, self.k[i], self.v[i], self.table, q, pos, seq)

    def fork(self, parents):
        p = torch.full((ROWS,), -1, dtype=torch.int32, device="cuda")
        for row, parent in parents.items():
            p[row] = parent
            for t in (self.tok, self.hist, self.prompt, self.active):
                t[row] = t[parent]
        self.o.kv_pages_fork(self.table, self.lens, self.refs, p, self.k, self.v, self.status, self.pws)
        assert int(host(self.status)[0]) == 0

    def free(self, rows):
        gone = torch.zeros(ROWS, dtype=torch.int32, device="cuda")
        gone[rows] = 1
        self.active[rows] = 0
        self.o.kv_pages_free(self.table, self.lens, self.refs, gone, PS)

    def compact(self):
        self.o.kv_pages_compact(self.table, self.refs, self.k, self.v, self.live, self.pws)
        return int(host(self.live)[0])


def kv_of(table, token, pos, layer):
    at = layer * (WQ + 2 * WK)
    row = table[token, at:at + WQ + 2 * WK]
    q = rotated(row[None, :WQ].reshape(1, NH, HD), None, np.array([pos]), THETA, EPS)[0]
    k = rotated(row[None, WQ:WQ + WK].reshape(1, NKV, HD), None, np.array([pos]), THETA, EPS)[0]
    return q, k.astype(np.float16), row[WQ + WK:].reshape(NKV, HD).astype(np.float16)


def attention_of(table, tokens, layer):
    rows = [kv_of(table, t, p, layer) for p, t in enumerate(tokens)]
    K, V = (np.stack([r[i] for r in rows]).astype(np.float64) for i in (1, 2))
    out = np.empty((NH, HD))
    for h in range(NH):
        s = K[:, h * NKV // NH] @ rows[-1][0][h] * SCALE
        e = np.exp(s - s.max())
        out[h] = e @ V[:, h * NKV // NH] / e.sum()
    return out


def play(gpu, graph):
    """The run: two prompts, forks, freed rows, compaction, a third prompt; returns what every step drew."""
    rng = np.random.default_rng(77)
    table = (1.5 * rng.standard_normal((VOCAB, ROW))).astype(np.float32)
    head = rng.standard_normal((VOCAB, WQ)).astype(np.float32)
    prompts = {0: list(rng.integers(0, VOCAB, 37)), 1: list(rng.integers(0, VOCAB, 20)), 4: list(rng.integers(0, VOCAB, 49))}
    s = Server(gpu, table, head, graph)
    seqs, drawn = {}, []
    for r in (0, 1):
        s.prompt_in(r, prompts[r])
        seqs[r] = list(prompts[r])
    for step in range(30):
        case(f"batch decode graph={graph} step {step}")
        if step == 6:  # two continuations of row 0, one of row 1; biases part them
            s.fork({2: 0, 3: 0, 5: 1})
            for row, parent in ((2, 0), (3, 0), (5, 1)):
                seqs[row] = list(seqs[parent])
                s.bias_ids[row, 0], s.bias[row, 0] = 10 * row, 100.0
        if step == 7:
            s.bias_ids.fill_(-1)
        if step == 12:
            s.free([0])
            del seqs[0]
        if step == 14:
            assert s.compact() == len({(p) for p in host(s.table).flatten() if p >= 0}) == int((host(s.refs) > 0).sum())
        if step == 15:
            s.prompt_in(4, prompts[4])
            seqs[4] = list(prompts[4])
            s.mask[4] = 0
            s.mask[4, 3] = 0b1010  # tokens 97 and 99 alone
        s.step()
        torch.cuda.synchronize()
        assert int(host(s.status)[0]) == 0
        tok, lens = host(s.tok).copy(), host(s.lens)
        outs, logits = [host(o).copy() for o in s.out], host(s.logits)
        for r in range(ROWS):
            if r not in seqs:
                assert lens[r] == 0 and not outs[0][r].any() and not outs[1][r].any()
                continue
            assert lens[r] == len(seqs[r]), (step, r)
            if step in (0, 5, 6, 7, 13, 14, 15, 16, 29):
                for i in range(LAYERS):
                    assert rel_l2(outs[i][r], attention_of(table, seqs[r], i)) <= 1e-3, (step, r, i)
            if step >= 15 and r == 4:
                assert tok[r] in (97, 99)
            assert tok[r] == int(np.argmax(logits[r]))
            seqs[r].append(int(tok[r]))
        if step == 6:
            assert tok[2] == 20 and tok[3] == 30 and tok[5] == 50
        drawn.append((tok, outs))
    refs = np.zeros(PAGES, np.int32)
    t, lens = host(s.table), host(s.lens)
    for r in range(ROWS):
        np.add.at(refs, t[r, :-(-int(lens[r]) // PS)], 1)
    assert np.array_equal(refs, host(s.refs)) and refs.max() > 1
    return drawn


def test_batch_decode(gpu):
    eager = play(gpu, False)
    graph = play(gpu, True)
    for (a, oa), (b, ob) in zip(eager, graph):
        assert np.array_equal(a, b)
        for x, y in zip(oa, ob):
            assert np.array_equal(x, y)
