"""A batch that holds prompts, taken through a layer as a server strings the calls together: shared projections with
each request's adapter beside them, preparation and store, attention over the paged cache, routing and grouped
experts, log probabilities of the prompts' own tokens; then a step of single tokens over the same cache.  Each
operator's result is held against the formula in 64 bits on what it was given; the batch as one captured graph
against the eager calls bit for bit.

Bar of the attention: what these projections give makes scores of hundreds.  A score of size s is off by s sqrt(10) 2^-24
(about ten roundings), one standard deviation, and so is a weight; five of them, s 1e-6, are the 5e-6 that scores of 5
are allowed elsewhere."""
import numpy as np
import pytest
import torch

from mnemocuda_amd import synth
from tests import torch_ref
from tests.conftest import rel_l2
from tests.gpu_util import case, dev, host
from tests.test_gpu_lora import reference as lora_reference
from tests.test_gpu_logprobs import reference as logprobs_reference
from tests.test_gpu_paged_prompt import check as check_attention
from tests.test_gpu_paged_prompt import reference as attention_reference
from tests.test_gpu_route import check as check_route
from tests.test_gpu_route import reference as route_reference

pytestmark = pytest.mark.gpu

H, NH, NKV, HD, PS = 256, 8, 2, 64, 16
EFF, E, K, VOCAB, RANK, ADAPTERS = 256, 12, 3, 1000, 16, 3
NEW = [23, 1, 0, 40]  # a fresh prompt, a decoding row, an idle one, a chunk behind 70 positions
BEFORE = [0, 33, 12, 70]
T, ROWS, PAGES, WIDTH = sum(NEW), len(NEW), 24, 8
EPS, THETA, SCALE = 1e-6, 1e4, HD ** -0.5


class Layer:
    def __init__(self, gpu, int8, seed=5):
        self.o, self.int8 = gpu.ops, int8
        rng, g = np.random.default_rng(seed), torch.Generator().manual_seed(seed)
        rn = lambda *s: torch.randn(s, generator=g).cuda()  # noqa: E731
        z = lambda *s: torch.zeros(s, device="cuda")  # noqa: E731
        i = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
        self.w = {n: dev(synth.weights(rng, 12, rows, H)) for n, rows in (("q", NH * HD), ("k", NKV * HD), ("v", NKV * HD), ("head", VOCAB))}
        self.experts, self.layout = dev(synth.expert_table(rng, E, H, EFF, 14)), synth.expert_layout(H, EFF, 14)
        self.a, self.b = (rn(ADAPTERS, RANK, H) * H ** -0.5).half(), (rn(ADAPTERS, NH * HD, RANK) * 0.25).half()
        self.ranks, self.scales = torch.tensor([16, 5, 8], dtype=torch.int32, device="cuda"), 0.5 + torch.rand(ADAPTERS, generator=g).cuda()
        self.router, self.bias = rn(E, H) * H ** -0.5, 0.1 * rn(E)
        self.x = rn(T, H)
        ids = np.concatenate([np.full(n, a) for n, a in zip(NEW, (1, 0, 2, -1))]).astype(np.int32)
        self.ids, self.targets = dev(ids), dev(rng.integers(0, VOCAB, T).astype(np.int32))
        kind = torch.int8 if int8 else torch.float16
        self.kp, self.vp = torch.zeros((PAGES, NKV, PS, HD), dtype=kind, device="cuda"), torch.zeros((PAGES, NKV, HD, PS), dtype=kind, device="cuda")
        self.ks, self.vs = (z(PAGES, NKV, PS), z(PAGES, NKV, PS)) if int8 else (None, None)
        self.table, self.lens, self.refs, self.status = i(ROWS, WIDTH) - 1, i(ROWS), i(PAGES), i(1)
        self.new_lens = torch.tensor([a + b for a, b in zip(NEW, BEFORE)], dtype=torch.int32, device="cuda")
        self.starts = torch.tensor(np.concatenate([[0], np.cumsum(NEW)]), dtype=torch.int32, device="cuda")
        self.seq = dev(np.repeat(np.arange(ROWS), NEW).astype(np.int32))
        self.pos = dev(np.concatenate([b + np.arange(n) for n, b in zip(NEW, BEFORE)]).astype(np.int32))
        self.xq = torch.zeros(T * (H // 128) * 144, dtype=torch.uint8, device="cuda")
        self.q0, self.q, self.k, self.v = z(T, NH * HD), z(T, NH * HD), z(T, NKV * HD), z(T, NKV * HD)
        self.qr, self.att = z(T, NH, HD), z(T, NH, HD)
        self.z, self.idx, self.wt, self.moe = z(T, E), i(T, K), z(T, K), z(T, H)
        self.ones, self.normed = torch.ones(H, device="cuda"), z(T, H)
        self.logits, self.logp, self.rank, self.ent = z(T, VOCAB), z(T), i(T), z(T)
        self.tops, self.top_ids = z(T, 5), i(T, 5)
        b = lambda n: torch.empty(n, dtype=torch.uint8, device="cuda")  # noqa: E731
        self.ws = [b(self.o.lora_workspace_bytes(T, H, RANK)), b(self.o.paged_attention_prompt_workspace_bytes(NH, NKV, HD)),
                   b(self.o.moe_prefill_workspace_bytes(T, H, EFF, E, K)), b(self.o.logprobs_workspace_bytes(T, VOCAB, 5))]
        # what earlier steps have stored: the rows hold their first positions
        self.o.kv_pages_extend(self.table, self.lens, self.refs, torch.tensor(BEFORE, dtype=torch.int32, device="cuda"), PS, self.status)
        n = sum(BEFORE)
        self.o.paged_attn_prep(rn(n, NH, HD), rn(n, NKV, HD), rn(n, NKV, HD), None, None, EPS, THETA, self.kp, self.vp, self.table,
                               z(n, NH, HD), dev(np.concatenate([np.arange(b) for b in BEFORE]).astype(np.int32)),
                               dev(np.repeat(np.arange(ROWS), BEFORE).astype(np.int32)), self.ks, self.vs)

    def step(self):
        o = self.o
        o.kv_pages_extend(self.table, self.lens, self.refs, self.new_lens, PS, self.status)
        o.quantize_q8_1(self.x, self.xq, H, T)
        o.gemm(self.w["q"], 12, self.xq, self.q0, NH * HD, H, T)
        o.gemm(self.w["k"], 12, self.xq, self.k, NKV * HD, H, T)
        o.gemm(self.w["v"], 12, self.xq, self.v, NKV * HD, H, T)
        o.lora_add(self.x, self.a, self.b, self.ids, self.ranks, self.scales, self.q0, self.q, self.ws[0])
        o.paged_attn_prep(self.q.view(T, NH, HD), self.k.view(T, NKV, HD), self.v.view(T, NKV, HD), None, None, EPS, THETA, self.kp,
                          self.vp, self.table, self.qr, self.pos, self.seq, self.ks, self.vs, seq_lens=self.lens)
        o.paged_attention_prompt(self.qr, self.kp, self.vp, self.table, self.starts, self.lens, self.att, SCALE, self.ws[1], self.ks, self.vs)
        for t in range(T):
            o.matvec_f32(self.router, self.x[t], self.z[t], E, H)
        o.moe_route(self.z, self.idx, self.wt, sigmoid=True, bias=self.bias, n_groups=4, top_groups=2, group_best=2, scale=1.5)
        self.moe.zero_()
        stride, g, u, d = self.layout
        o.moe_prefill(self.experts, stride, g, u, d, 14, self.x, self.idx, self.wt, T, H, EFF, E, K, self.ws[2], self.moe)
        o.rms_norm_batched(self.moe, self.ones, self.normed, H, EPS)
        o.quantize_q8_1(self.normed, self.xq, H, T)
        o.gemm(self.w["head"], 12, self.xq, self.logits, VOCAB, H, T)
        o.logprobs(self.logits, self.targets, self.logp, self.rank, self.ent, self.top_ids, self.tops, self.ws[3])

    def results(self):
        torch.cuda.synchronize()
        return [host(t).copy() for t in (self.q, self.att, self.idx, self.wt, self.moe, self.logp, self.rank, self.ent, self.top_ids, self.tops)]


def score_sizes(q, k, ks, table, lens):
    """The largest score, by size, of each token."""
    out, at = [], 0
    for r, n in enumerate(NEW):
        pos = np.arange(lens[r])
        K = k[table[r, pos // PS], :, pos % PS].astype(np.float64)
        if ks is not None:
            K = K * ks[table[r, pos // PS], :, pos % PS][..., None]
        for t in range(at, at + n):
            seen = int(lens[r]) - at - n + t + 1
            out.append(max(np.abs(K[:seen, h * NKV // NH] @ q[t, h]).max() * SCALE for h in range(NH)))
        at += n
    return np.array(out)


@pytest.mark.parametrize("int8", [False, True])
def test_a_layer(gpu, int8):
    s = Layer(gpu, int8)
    case(f"prompt batch int8={int8}")
    s.step()
    q, att, idx, wt, moe, logp, rank, ent, top_ids, tops = s.results()
    assert int(host(s.status)[0]) == 0 and host(s.lens).tolist() == [a + b for a, b in zip(NEW, BEFORE)]
    want, bound = lora_reference({"x": s.x.cpu(), "a": s.a.cpu(), "b": s.b.cpu(), "base": s.q0.cpu(), "ids": s.ids.cpu(),
                                  "ranks": s.ranks.cpu(), "scales": s.scales.cpu()})
    assert (np.abs(q - want) <= bound).all()
    cache = [host(s.kp), host(s.vp)] + ([host(s.ks), host(s.vs)] if int8 else [None, None])
    size = score_sizes(host(s.qr), cache[0], cache[2], host(s.table), host(s.lens))
    check_attention(att, attention_reference(host(s.qr), *cache, host(s.table), host(s.starts), host(s.lens), SCALE), 1e-6 * np.maximum(size, 5))
    check_route((idx, wt), route_reference(host(s.z), K, True, host(s.bias), 4, 2, 2, True, 1.5))
    stride, g, u, d = s.layout
    expert = torch_ref.moe_prefill(s.experts, stride, g, u, d, 14, s.x, idx, wt, H, EFF)
    assert rel_l2(moe, host(expert)) <= 1e-3  # values on a border of a requantisation may go to either side
    want = logprobs_reference(host(s.logits), host(s.targets), 5)
    assert np.array_equal(rank, want["rank"]) and np.array_equal(top_ids, want["ids"])
    for got, name, bound in ((logp, "logp", want["e"]), (ent, "ent", want["e_ent"]), (tops, "tops", want["e"][:, None])):
        assert (np.abs(got - want[name]) <= bound + 2.0 ** -24 * np.abs(want[name])).all(), name
    # the next step: one token a row, over what the prompts have stored
    n = ROWS
    to = s.lens + torch.tensor([1, 1, 0, 1], dtype=torch.int32, device="cuda")
    s.o.kv_pages_extend(s.table, s.lens, s.refs, to, PS, s.status)
    x = torch.randn((n, NH, HD), generator=torch.Generator().manual_seed(9)).cuda()
    kv = torch.randn((2, n, NKV, HD), generator=torch.Generator().manual_seed(10)).cuda()
    s.o.paged_attn_prep(x, kv[0], kv[1], None, None, EPS, THETA, s.kp, s.vp, s.table, x, dev(np.array([23, 34, -1, 110], np.int32)),
                        dev(np.arange(n, dtype=np.int32)), s.ks, s.vs, seq_lens=s.lens)
    one, many = torch.empty_like(x), torch.zeros_like(x)
    ws = torch.empty(s.o.paged_attention_workspace_bytes(NH, NKV, HD), dtype=torch.uint8, device="cuda")
    s.o.paged_attention_decode(x, s.kp, s.vp, s.table, s.lens, one, SCALE, ws, s.ks, s.vs)
    rows = torch.tensor([0, 1, 3], device="cuda")
    part = torch.empty((3, NH, HD), device="cuda")
    s.o.paged_attention_prompt(x[rows], s.kp, s.vp, s.table, dev(np.array([0, 1, 2, 2, 3], np.int32)), s.lens, part, SCALE, s.ws[1], s.ks, s.vs)
    many[rows] = part
    for r in (0, 1, 3):  # 5e-6 each
        assert rel_l2(host(many)[r], host(one)[r]) <= 1e-5


@pytest.mark.parametrize("int8", [False, True])
def test_the_layer_as_a_graph(gpu, int8):
    """Captured, replayed from the same state with other tokens, requests and adapters, against eager calls."""
    eager, s = Layer(gpu, int8), Layer(gpu, int8)
    side = torch.cuda.Stream()
    case(f"prompt batch graph int8={int8}")
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            s.step()
    for i in range(3):
        g = torch.Generator().manual_seed(100 + i)
        x, ids = torch.randn((T, H), generator=g), torch.randint(-1, ADAPTERS, (T,), generator=g).to(torch.int32)
        for y in (eager, s):
            y.x.copy_(x)
            y.ids.copy_(ids)
            y.lens.copy_(torch.tensor(BEFORE, dtype=torch.int32) if i == 0 else y.lens)  # later ones write their positions again
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        eager.step()
        for a, b in zip(eager.results(), s.results()):
            assert np.array_equal(a, b)
