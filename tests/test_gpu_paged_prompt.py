"""Attention of several new tokens per sequence over the paged cache against the formula in 64 bits.

Bar, relative L2 of a token's output 5e-6, as for one token a sequence: a score is a sum of products of an fp32 query
(held as two f16 parts, 22 bits or more of it) and an exact cache value, rounded to fp32 (2^-24) about ten times on
the way, so with scores of up to ~5 in size it is off by ~5 * sqrt(10) * 2^-24 ~ 1e-6; that is the relative error of a
weight, and of the output, which weighs independent values.  5e-6 leaves room for larger scores."""
import math

import numpy as np
import pytest
import torch

from tests.conftest import rel_l2
from tests.gpu_util import case, dev, host
from tests.test_gpu_paged_attn import attend as attend_one
from tests.test_gpu_paged_attn import block_table, opt, pool

pytestmark = pytest.mark.gpu
BAR = 5e-6


def reference(q, k, v, ks, vs, table, starts, lens, scale):
    """What a token does not see is left out, whatever it holds."""
    nkv, ps = k.shape[1], k.shape[2]
    G = q.shape[1] // nkv
    out = np.full(q.shape, np.nan)  # rows of no sequence
    for s in range(len(lens)):
        n, L = int(starts[s + 1] - starts[s]), min(max(int(lens[s]), 0), table.shape[1] * ps)
        pos = np.arange(L)
        page, off = table[s, pos // ps], pos % ps
        ok = (page >= 0) & (page < k.shape[0])
        pos, page, off = pos[ok], page[ok], off[ok]
        at = L - n + np.arange(n)
        rows = slice(int(starts[s]), int(starts[s + 1]))
        if not len(page):
            out[rows] = 0
            continue
        seen = pos[None] <= at[:, None]
        for h in range(nkv):
            K, V = k[page, h, off].astype(np.float64), v[page, h, :, off].astype(np.float64)
            if ks is not None:
                K, V = K * ks[page, h, off][:, None].astype(np.float64), V * vs[page, h, off][:, None].astype(np.float64)
            odd = ~(np.isfinite(K).all(1) & np.isfinite(V).all(1))
            for g in range(h * G, (h + 1) * G):
                x = q[rows, g].astype(np.float64) @ np.where(odd[:, None], 0, K).T * scale
                x = np.where(seen, x, -np.inf)
                m = x.max(1, keepdims=True)
                e = np.exp(x - np.where(np.isfinite(m), m, 0))
                o = e @ np.where(odd[:, None], 0, V) / np.maximum(e.sum(1, keepdims=True), 1e-300)
                o[(seen & odd[None]).any(1)] = np.nan
                out[rows, g] = o
    return out


def attend(gpu, q, k, v, ks, vs, table, starts, lens, scale, out=None, ws=None, wide=False):
    """wide: with rows of no sequence behind the last, so many that the rows are not few."""
    if wide:
        more = 128 * len(lens) + 1
        got = attend(gpu, np.concatenate([q, np.ones((more, *q.shape[1:]), np.float32)]), k, v, ks, vs, table, starts, lens, scale)
        assert torch.isnan(got[len(q):]).all()
        return got[:len(q)]
    T, nh, hd = q.shape
    if ws is None:
        ws = torch.full((gpu.ops.paged_attention_prompt_workspace_bytes(nh, k.shape[1], hd),), 255, dtype=torch.uint8, device="cuda")
    if out is None:
        out = torch.full(q.shape, float("nan"), device="cuda")
    as_dev = lambda x: x if isinstance(x, torch.Tensor) else opt(x)  # noqa: E731
    gpu.ops.paged_attention_prompt(as_dev(q), as_dev(k), as_dev(v), as_dev(table), as_dev(starts), as_dev(lens), out, scale,
                                   ws, as_dev(ks), as_dev(vs))
    return out


def make(seed, new, before, nkv, G, hd, ps, int8, extra=3):
    """Sequences that take new[s] tokens behind before[s] positions."""
    rng = np.random.default_rng(seed)
    lens = np.array([a + b for a, b in zip(new, before)], np.int32)
    starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    n_pages = int(sum(-(-np.maximum(lens, 0) // ps))) + extra
    k, v, ks, vs = pool(rng, n_pages, nkv, ps, hd, int8)
    table = block_table(rng, lens, ps, int(max(-(-np.max(lens) // ps), 1)) + 1, n_pages)
    q = (rng.standard_normal((int(starts[-1]), nkv * G, hd)) * rng.uniform(0.3, 1.5, (1, nkv * G, 1))).astype(np.float32)
    return q, k, v, ks, vs, table, starts, lens


def check(got, want, bar=BAR):
    """bar: of all tokens, or of each."""
    bar = np.broadcast_to(bar, len(want))
    for t in range(len(want)):
        if not want[t].any():
            assert not got[t].any(), t
        else:
            assert rel_l2(got[t], want[t]) <= bar[t], (t, rel_l2(got[t], want[t]), bar[t])


SHAPES = [(128, 64, 4, 16, False), (128, 64, 2, 16, True), (128, 16, 2, 5, False), (128, 16, 2, 5, True), (128, 32, 1, 1, False),
          (128, 128, 3, 8, True), (64, 16, 2, 7, False), (64, 64, 12, 1, False), (64, 32, 2, 16, True), (256, 16, 1, 16, False),
          (256, 64, 2, 3, False), (256, 128, 1, 4, True), (256, 32, 2, 1, True)]
EDGE_NEW = [1, 0, 2, 7, 8, 9, 1, 63, 64, 65, 1, 130, 3, 17, 40]
EDGE_BEFORE = [0, 30, 0, 0, 1, 63, 64, 0, 0, 64, 127, 65, 600, 15, 0]


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("hd,ps,nkv,G,int8", SHAPES)
def test_at_the_edges(gpu, hd, ps, nkv, G, int8, wide):
    a = make(hd + ps + G, EDGE_NEW, EDGE_BEFORE, nkv, G, hd, ps, int8)
    case(f"paged prompt hd={hd} ps={ps} nkv={nkv} gqa={G} int8={int8} edges")
    got = attend(gpu, *a, hd ** -0.5, wide=wide)
    assert torch.equal(got, attend(gpu, *a, hd ** -0.5, wide=wide))
    check(host(got), reference(*a, hd ** -0.5))


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("new,before,nkv,G,hd,ps", [
    ([1], [0], 1, 1, 64, 16), ([1], [5000], 4, 16, 128, 64), ([2000], [0], 1, 4, 128, 64), ([5, 3, 4], [4000, 700, 90], 4, 8, 128, 32),
    ([4], [70000], 1, 4, 128, 16), ([300, 411], [3000, 20], 2, 3, 64, 128), ([257], [999], 2, 2, 256, 64), ([700], [300], 3, 1, 64, 16),
    ([33] * 70, list(range(0, 350, 5)), 2, 4, 64, 16), ([1] * 300, [i % 97 for i in range(300)], 1, 16, 128, 16),
    ([1] * 4096, [i % 7 for i in range(4096)], 1, 1, 64, 16), ([1500], [0], 1, 1, 256, 128)])
def test_split_over_the_workgroups(gpu, new, before, nkv, G, hd, ps, int8):
    """Few long tiles, whose shares cut them, and many short ones; more sequences than a wave has lanes."""
    a = make(sum(new) + hd, new, before, nkv, G, hd, ps, int8)
    case(f"paged prompt new={new[:4]} before={before[:4]} ({len(new)}) nkv={nkv} gqa={G} hd={hd} ps={ps} int8={int8}")
    got = attend(gpu, *a, hd ** -0.5)
    assert torch.equal(got, attend(gpu, *a, hd ** -0.5))
    check(host(got), reference(*a, hd ** -0.5))


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("hd,ps", [(64, 16), (128, 64), (256, 32)])
def test_single_tokens_as_in_decoding(gpu, hd, ps, int8):
    """A token a sequence is what the decode entry point computes."""
    lens = [1, 17, 300, 64, 2000, 0]
    a = make(hd, [1, 1, 1, 1, 1, 0], [n - 1 if n else 0 for n in lens], 2, 4, hd, ps, int8)
    q, k, v, ks, vs, table, starts, ln = a
    case(f"paged prompt as decode hd={hd} int8={int8}")
    got = host(attend(gpu, *a, 0.1))
    one = host(attend_one(gpu, np.concatenate([q, q[:1]]), k, v, ks, vs, table, ln, 0.1))
    for t in range(5):
        assert rel_l2(got[t], one[t]) <= 2 * BAR


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("hd,ps", [(64, 64), (128, 16), (256, 32)])
def test_nothing_of_what_a_token_does_not_see(gpu, hd, ps, int8, wide):
    """NaN and infinities in later tokens' keys and values, past the end, in pages that nothing names and in the
    table's rest; tokens that see them get no numbers in the heads concerned."""
    q, k, v, ks, vs, table, starts, lens = make(7, [90, 5, 20], [10, 200, 0], 2, 3, hd, ps, int8, extra=6)
    clean = reference(q, k, v, ks, vs, table, starts, lens, 0.1)
    rng = np.random.default_rng(5)
    n_pages = len(k)
    used = np.zeros((n_pages, ps), bool)
    for s, L in enumerate(lens):
        p = np.arange(L)
        used[table[s, p // ps], p % ps] = True
    for p, o in np.argwhere(~used):
        b = rng.choice(np.array([np.nan, np.inf, -np.inf], np.float32))
        if int8:
            ks[p, :, o] = vs[p, :, o] = b
        else:
            k[p, :, o] = v[p, :, :, o] = b
    for s, L in enumerate(lens):
        rest = table[s, -(-int(L) // ps):]
        rest[:] = rng.choice(np.array([-1, n_pages, 2 ** 31 - 1, -2 ** 31, n_pages - 1], np.int64), len(rest)).astype(np.int32)
    # (sequence, position, KV head, key or value): late ones, so that earlier tokens of the tile do not see them
    odd = [(0, 97, 0, "v", np.nan), (0, 70, 1, "v", np.inf), (0, 45, 0, "k", np.nan), (1, 203, 1, "v", -np.inf), (2, 19, 0, "k", np.nan),
           (2, 18, 1, "v", np.nan)]
    for s, p, h, what, x in odd:
        page, off = table[s, p // ps], p % ps
        if int8:
            (ks if what == "k" else vs)[page, h, off] = x
        elif what == "k":
            k[page, h, off, 3] = x
        else:
            v[page, h, 5, off] = x
    case(f"paged prompt, NaN ahead, hd={hd} ps={ps} int8={int8}")
    got = host(attend(gpu, q, k, v, ks, vs, table, starts, lens, 0.1, wide=wide))
    for t in range(len(q)):
        s = int(np.searchsorted(starts, t, "right")) - 1
        p = int(lens[s] - starts[s + 1] + t)
        for h in range(2):
            hit = [o for o in odd if o[0] == s and o[2] == h and o[1] <= p]
            mine, want = got[t, 3 * h:3 * h + 3], clean[t, 3 * h:3 * h + 3]
            if not hit:
                assert rel_l2(mine, want) <= BAR, (t, h)
            elif any(o[3] == "k" for o in hit) or int8:
                assert np.isnan(mine).all() or not np.isfinite(mine).any(), (t, h)
            else:  # one dim of the values
                assert not np.isfinite(mine[:, 5]).any() and rel_l2(np.delete(mine, 5, 1), np.delete(want, 5, 1)) <= BAR, (t, h)


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("int8", [False, True])
def test_pages_that_are_not_there(gpu, int8, wide):
    """Entries outside the pool are absent positions, a row of them gives zeros, a length past the table is cut."""
    rng = np.random.default_rng(3)
    lens = np.array([300, 64, 200, 100000], np.int32)
    starts = np.array([0, 40, 50, 57, 90], np.int32)
    k, v, ks, vs = pool(rng, 40, 2, 16, 128, int8)
    table = block_table(rng, [320, 64, 208, 20 * 16], 16, 20, 60) % 40
    table[0, 3], table[0, 7], table[0, 18] = -1, 40, 2 ** 31 - 1
    table[1, :4] = [-1, -5, 40, -2 ** 31]
    q = rng.standard_normal((90, 6, 128)).astype(np.float32)
    case(f"paged prompt, invalid pages, int8={int8}")
    got = host(attend(gpu, q, k, v, ks, vs, table, starts, lens, 0.09, wide=wide))
    check(got, reference(q, k, v, ks, vs, table, starts, lens, 0.09))
    assert not got[40:50].any()


def test_tokens_before_the_first_position_and_rows_of_no_sequence(gpu):
    """More tokens than positions: the first ones get zeros.  Rows before the first start and behind the last stay."""
    rng = np.random.default_rng(4)
    k, v, _, _ = pool(rng, 30, 2, 16, 64, False)
    lens = np.array([5, 0, 70, -4, 3], np.int32)
    starts = np.array([3, 20, 30, 100, 110, 250], np.int32)
    table = block_table(rng, [16, 0, 80, 0, 16], 16, 6, 30)
    q = rng.standard_normal((260, 8, 64)).astype(np.float32)
    out = torch.full(q.shape, 3.0, device="cuda")
    case("paged prompt, tokens before the first position")
    got = host(attend(gpu, q, k, v, None, None, table, starts, lens, 0.2, out=out))
    assert (got[:3] == 3).all() and (got[250:] == 3).all()
    want = reference(q, k, v, None, None, table, starts, lens, 0.2)
    assert not want[3:15].any() and not want[20:30].any() and not want[100:247].any()
    check(got[3:250], want[3:250])


def test_starts_that_leave_the_rows(gpu):
    """Starts outside 0..n_tokens are cut to it, a falling one gives a sequence without tokens: nothing outside is
    read or written."""
    rng = np.random.default_rng(6)
    k, v, _, _ = pool(rng, 30, 1, 16, 64, False)
    lens = np.array([40, 40, 40, 40], np.int32)
    table = block_table(rng, [48] * 4, 16, 3, 30)
    q = rng.standard_normal((50, 2, 64)).astype(np.float32)
    starts = np.array([-5, 10, 7, 30, 2 ** 31 - 1], np.int32)
    buf = torch.full((52, 2, 64), 3.0, device="cuda")
    case("paged prompt, starts out of range")
    attend(gpu, q, k, v, None, None, table, starts, lens, 0.2, out=buf[1:51])
    got = host(buf)
    assert (got[0] == 3).all() and (got[51] == 3).all()
    # (sequence, its rows, those that it alone claims)
    for s, a, b, lo, hi in ((0, 0, 10, 0, 7), (2, 7, 30, 10, 30), (3, 30, 50, 30, 50)):
        want = reference(q[a:b], k, v, None, None, table[s:s + 1], np.array([0, b - a]), lens[s:s + 1], 0.2)
        check(got[1 + lo:1 + hi], want[lo - a:hi - a])


@pytest.mark.parametrize("int8", [False, True])
def test_size_of_the_query(gpu, int8):
    """A query 2^20 times larger under a scale 2^20 times smaller (and the other way round) gives the same bits."""
    a = make(8, [70, 3], [40, 900], 2, 5, 128, 16, int8)
    case(f"paged prompt, scaled queries, int8={int8}")
    base = attend(gpu, *a, 0.08)
    check(host(base), reference(*a, 0.08))
    for f in (2.0 ** 20, 2.0 ** -20):
        assert torch.equal(attend(gpu, a[0] * np.float32(f), *a[1:], float(np.float32(0.08)) / f), base), f


@pytest.mark.parametrize("wide", [False, True])
def test_value_scales_of_any_size(gpu, wide):
    """int8 value scales from 1e-20 to 1e20, within a sequence too: what has weight keeps its bits."""
    q, k, v, ks, vs, table, starts, lens = make(9, [40] * 5, [110] * 5, 2, 2, 128, 16, True)
    for i, f in enumerate([1e-20, 1e-3, 1.0, 1e8, 1e20]):
        vs[table[i, :10]] *= np.float32(f)
    vs[table[2, 3], :, 7] *= np.float32(1e6)
    case("paged prompt, value scales")
    got = host(attend(gpu, q, k, v, ks, vs, table, starts, lens, 0.09, wide=wide))
    check(got, reference(q, k, v, ks, vs, table, starts, lens, 0.09))


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("rise", [1, -1])
def test_scores_that_rise_and_fall(gpu, rise, int8, wide):
    """Scores that climb (or fall) by 400 along the sequence: the reference of the softmax moves many times."""
    q, k, v, ks, vs, table, starts, lens = make(10, [100], [900], 1, 4, 64, 32, int8)
    q[:] = 1.0
    pos = np.arange(1000)
    page, off = table[0, pos // 32], pos % 32
    level = (pos if rise > 0 else 999 - pos) / 1000 * 400 / 64
    if int8:
        k[page, 0, off] = 100
        ks[page, 0, off] = level / 100
    else:
        k[page, 0, off] = (level[:, None] + 0 * k[page, 0, off]).astype(np.float16)
    case(f"paged prompt, scores rise={rise} int8={int8}")
    got = host(attend(gpu, q, k, v, ks, vs, table, starts, lens, 1.0, wide=wide))
    # scores of 400 round at 400 * 2^-24 some ten times: ~1e-4 of a weight
    check(got, reference(q, k, v, ks, vs, table, starts, lens, 1.0), 1e-4)


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("int8", [False, True])
def test_queries_that_are_no_number(gpu, int8, wide):
    """NaN or an infinity in a head of a token gives no numbers there and leaves all others as they are, in tiles
    that are cut, too."""
    a = make(11, [60, 2], [100, 9000], 2, 3, 128, 64, int8)
    case(f"paged prompt, NaN queries int8={int8}")
    base = host(attend(gpu, *a, 0.1, wide=wide)).copy()
    q = a[0].copy()
    for t, h, x in ((0, 1, np.nan), (30, 5, np.inf), (59, 0, np.nan), (61, 4, -np.inf), (60, 2, np.nan)):
        q[t, h, 17] = x
    got = host(attend(gpu, q, *a[1:], 0.1, wide=wide))
    for t in range(62):
        for h in range(6):
            if (t, h) in ((0, 1), (30, 5), (59, 0), (61, 4), (60, 2)):
                assert np.isnan(got[t, h]).all(), (t, h)
            else:
                assert np.array_equal(got[t, h], base[t, h]), (t, h)


def test_pages_past_4_gib(gpu):
    """Pages whose byte offset passes 32 bits (a pool of ~6.5 GB each for K and V)."""
    nkv, ps, hd, n_pages = 8, 128, 256, 12500
    k = torch.zeros((n_pages, nkv, ps, hd), dtype=torch.float16, device="cuda")
    v = torch.zeros((n_pages, nkv, hd, ps), dtype=torch.float16, device="cuda")
    ids = np.array([12499, 0, 8192, 12000], np.int32)
    rng = np.random.default_rng(1)
    kk, vv, _, _ = pool(rng, 4, nkv, ps, hd, False)
    at = torch.from_numpy(ids.astype(np.int64)).cuda()
    k[at], v[at] = dev(kk), dev(vv)
    q = rng.standard_normal((21, nkv * 2, hd)).astype(np.float32)
    lens, starts = np.array([4 * ps - 5], np.int32), np.array([0, 21], np.int32)
    case("paged prompt past 4 GiB")
    got = host(attend(gpu, q, k, v, None, None, ids[None], starts, lens, 0.06))
    check(got, reference(q, kk, vv, None, None, np.arange(4, dtype=np.int32)[None], starts, lens, 0.06))


def test_in_a_graph(gpu):
    """One captured call serves other starts, lengths, tables and queries; replays between eager calls on the same
    workspace."""
    rng = np.random.default_rng(11)
    k, v, _, _ = pool(rng, 200, 4, 32, 128, False)
    kd, vd = dev(k), dev(v)
    table, lens = torch.full((3, 60), -1, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    starts = torch.zeros(4, dtype=torch.int32, device="cuda")
    q = torch.zeros((150, 32, 128), device="cuda")
    out = torch.empty_like(q)
    ws = torch.empty(gpu.ops.paged_attention_prompt_workspace_bytes(32, 4, 128), dtype=torch.uint8, device="cuda")
    call = lambda: gpu.ops.paged_attention_prompt(q, kd, vd, table, starts, lens, out, 0.09, ws)  # noqa: E731
    case("paged prompt graph capture")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            call()
    for new, ln in (([5, 0, 140], [5, 0, 1900]), ([1, 2, 3], [1, 700, 33]), ([0, 0, 0], [0, 9, 0]), ([50, 50, 50], [1900, 1900, 50])):
        t, st = block_table(rng, ln, 32, 60, 200), np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        x = rng.standard_normal((150, 32, 128)).astype(np.float32)
        for d, h in ((table, t), (lens, np.array(ln, np.int32)), (starts, st), (q, x)):
            d.copy_(dev(h))
        out.fill_(3.0)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        torch.cuda.synchronize()
        got = host(out).copy()
        n = int(st[-1])
        assert (got[n:] == 3).all()
        check(got[:n], reference(x[:n], k, v, None, None, t, st, np.array(ln, np.int32), 0.09))
        call()
        assert np.array_equal(host(out), got)


def test_on_two_streams(gpu):
    """Two calls at once, each with a workspace of its own."""
    a, b = make(20, [200], [3000], 2, 4, 128, 64, False), make(21, [150, 9], [10, 2000], 2, 4, 64, 16, True)
    want = [host(attend(gpu, *x, 0.1)).copy() for x in (a, b)]
    d = [[opt(t) for t in x] for x in (a, b)]
    outs = [torch.empty(x[0].shape, device="cuda") for x in (a, b)]
    wss = [torch.empty(gpu.ops.paged_attention_prompt_workspace_bytes(8, 2, x[0].shape[2]), dtype=torch.uint8, device="cuda") for x in (a, b)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    case("paged prompt on two streams")
    for _ in range(5):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                attend(gpu, *d[i], 0.1, out=outs[i], ws=wss[i])
    torch.cuda.synchronize()
    for i in range(2):
        assert np.array_equal(host(outs[i]), want[i])


@pytest.mark.parametrize("int8", [False, True])
def test_long_rows_keep_their_bits(gpu, int8):
    """40,000 positions added up by one lane group after another: the sum of the weights is compensated, and the output is
    rounded four times a step, 2,500 times with one standard deviation of 2^-24 / sqrt(12) * 2 each at most, 1.7e-6; with
    the scores' share (see above) below 2.5e-6."""
    a = make(12, [40], [40000], 1, 3, 128, 64, int8)
    case(f"paged prompt, long rows int8={int8}")
    got = host(attend(gpu, *a, 128 ** -0.5))
    assert rel_l2(got, reference(*a, 128 ** -0.5)) <= 2.5e-6


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("scale", [0.0, -0.1])
def test_scales_of_the_scores(gpu, scale, int8):
    """A scale of 0 (all weights equal) and one below 0."""
    a = make(14, [70, 3], [20, 300], 2, 3, 128, 32, int8)
    case(f"paged prompt, scale {scale} int8={int8}")
    check(host(attend(gpu, *a, scale)), reference(*a, scale))


@pytest.mark.parametrize("wide", [False, True])
def test_value_scales_of_zero(gpu, wide):
    """Rows of zeros (scale 0) whose scores are the largest by far: their weights count in the sum.  Behind them, before
    them and alone; and scales of 2^-75 beside them."""
    q, k, v, ks, vs, table, starts, lens = make(15, [30, 30, 30, 30], [170] * 4, 1, 2, 64, 16, True)
    q[:] = np.abs(q) + 0.5
    for s, zero in enumerate([range(0, 100), range(150, 200), range(0, 200), range(0, 200, 2)]):
        pos = np.array(list(zero))
        page, off = table[s, pos // 16], pos % 16
        vs[page, :, off] = 0.0
        k[page, :, off] = 100  # scores of 20 and more above the others'
        rest = np.setdiff1d(np.arange(200), pos)
        if s == 3:
            vs[table[s, rest // 16], :, rest % 16] *= np.float32(2.0 ** -75)
    case("paged prompt, value scales of zero")
    got = host(attend(gpu, q, k, v, ks, vs, table, starts, lens, 0.05, wide=wide))
    want = reference(q, k, v, ks, vs, table, starts, lens, 0.05)
    assert np.isfinite(got).all() and not got[60:90].any()
    check(got, want)


def test_starts_that_fall(gpu):
    """Starts that give all rows to many sequences: whatever comes out, nothing outside the rows is read or written."""
    rng = np.random.default_rng(16)
    k, v, _, _ = pool(rng, 4, 1, 16, 64, False)
    n = 400
    q = dev(rng.standard_normal((64, 2, 64)).astype(np.float32))
    table = np.zeros((n, 1), np.int32)
    buf = torch.full((66, 2, 64), 3.0, device="cuda")
    case("paged prompt, falling starts")
    for far in (64, 2 ** 31 - 1):
        starts = np.array([0, far] * (n // 2) + [0], np.int64).astype(np.int32)
        attend(gpu, q, k, v, None, None, table, starts, np.full(n, 16, np.int32), 0.2, out=buf[1:65])
        got = host(buf)
        assert (got[0] == 3).all() and (got[65] == 3).all()


@pytest.mark.parametrize("wide", [False, True])
def test_value_scales_of_the_ends(gpu, wide):
    """Values of up to 2^97, and below 2^-99."""
    for e in (90, -106):
        q, k, v, ks, vs, table, starts, lens = make(17, [40, 1], [300, 900], 1, 2, 64, 16, True)
        vs[:] = np.float32(2.0 ** e)
        case(f"paged prompt, value scales 2^{e}")
        a = (q, k, v, ks, vs, table, starts, lens, 0.1)
        want = reference(*a)
        check(host(attend(gpu, *a, wide=wide)) * 2.0 ** -e, want * 2.0 ** -e)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("n,before,nkv,G,hd,ps", [(1700, 0, 4, 16, 128, 64), (1305, 0, 4, 16, 64, 16), (2003, 0, 2, 16, 256, 128), (2048, 777, 4, 16, 128, 16),
                                                  (2300, 0, 9, 5, 64, 64), (4099, 0, 4, 8, 128, 32), (3500, 10, 16, 3, 128, 64)])
def test_one_long_prompt(gpu, n, before, nkv, G, hd, ps, int8):
    """Prompts whose tiles are dealt out whole, and next to them others; with rows that take nothing beside them.  Some heads
    of the first and the last KV head are looked at."""
    a = make(n + hd, [0, n, 0], [50, before, 0], nkv, G, hd, ps, int8)
    q, k, v, ks, vs, table, starts, lens = a
    case(f"paged prompt, one of {n} behind {before}, nkv={nkv} gqa={G} hd={hd} ps={ps} int8={int8}")
    got = attend(gpu, *a, hd ** -0.5)
    assert torch.equal(got, attend(gpu, *a, hd ** -0.5))
    got = host(got)
    assert np.isfinite(got).all()
    for h in (0, nkv - 1):
        some = [h * G, h * G + G - 1]
        of = lambda x: None if x is None else x[:, h:h + 1]  # noqa: E731
        check(got[:, some], reference(q[:, some], of(k), of(v), of(ks), of(vs), table, starts, lens, hd ** -0.5))


def test_one_long_prompt_that_ends_early(gpu):
    """More tokens than positions; values that are no numbers ahead of most tokens; a page that is not there."""
    q, k, v, _, _, table, starts, lens = make(77, [1800], [0], 4, 16, 128, 64, False)
    v[table[0, 1700 // 64], 1, 7, 1700 % 64] = np.nan
    table[0, 5] = -1
    case("paged prompt, one long, NaN ahead")
    got = host(attend(gpu, q, k, v, None, None, table, starts, lens, 0.09))
    assert np.isnan(got[1700:, 16:32, 7]).all()
    got[1700:, 16:32, 7] = 0
    assert np.isfinite(got).all()
    for h in (0, 1):
        some = [16 * h, 16 * h + 15]
        want = reference(q[:, some], k[:, h:h + 1], np.nan_to_num(v[:, h:h + 1]), None, None, table, starts, lens, 0.09)
        if h == 1:
            want[1700:, :, 7] = 0
        check(got[:, some], want)
    lens[0] = 1500
    case("paged prompt, one long, 300 tokens before the first position")
    got = host(attend(gpu, q, k, v, None, None, table, starts, lens, 0.09))
    assert not got[:300].any()
    check(got[300:, [0, 15]], reference(q[300:, [0, 15]], k[:, :1], v[:, :1], None, None, table, starts - np.array([0, 300], np.int32), lens, 0.09))
