"""Paged attention and the store of new tokens against the formulas in 64 bits.

Attention bar, relative L2 5e-6: a score is a sum of products of an fp32 query (held as two f16
parts, 22 bits or more of it) and an exact cache value, rounded to fp32 (2^-24) about ten times on
the way, so with scores of up to ~5 in size it is off by ~5 * sqrt(10) * 2^-24 ~ 1e-6 (one standard
deviation); that is the relative error of each weight exp(score), and of the output, which weighs
independent values.  5e-6 leaves room for heads with larger scores.
"""
import math

import numpy as np
import pytest
import torch

from tests.conftest import rel_l2
from tests.gpu_util import case, dev, host

pytestmark = pytest.mark.gpu

BAR = 5e-6


def pool(rng, n_pages, nkv, ps, hd, int8):
    """Random pages (k, v, ks, vs) as numpy arrays in the cache's types (ks, vs None for f16)."""
    if int8:
        k = rng.integers(-127, 128, (n_pages, nkv, ps, hd)).astype(np.int8)
        v = rng.integers(-127, 128, (n_pages, nkv, hd, ps)).astype(np.int8)
        ks, vs = ((rng.uniform(0.5, 1.5, (n_pages, nkv, ps)) * 0.02).astype(np.float32) for _ in range(2))
        return k, v, ks, vs
    return (rng.standard_normal((n_pages, nkv, ps, hd)).astype(np.float16),
            rng.standard_normal((n_pages, nkv, hd, ps)).astype(np.float16), None, None)


def block_table(rng, lens, ps, width, n_pages):
    ids = rng.permutation(n_pages).astype(np.int32)
    t, at = np.full((len(lens), width), -1, np.int32), 0
    for i, n in enumerate(lens):
        p = min(max(-(-n // ps), 0), width)
        t[i, :p] = ids[at:at + p]
        at += p
    return t


def reference(q, k, v, ks, vs, table, lens, scale):
    n, nh, hd = q.shape
    nkv, ps = k.shape[1], k.shape[2]
    G = nh // nkv
    out = np.zeros(q.shape)
    for i in range(n):
        L = min(max(int(lens[i]), 0), table.shape[1] * ps)
        pos = np.arange(L)
        page, off = table[i, pos // ps], pos % ps
        ok = (page >= 0) & (page < k.shape[0])
        page, off = page[ok], off[ok]
        if not len(page):
            continue
        for h in range(nkv):
            K, V = k[page, h, off].astype(np.float64), v[page, h, :, off].astype(np.float64)
            if ks is not None:
                K, V = K * ks[page, h, off][:, None].astype(np.float64), V * vs[page, h, off][:, None].astype(np.float64)
            s = q[i, h * G:(h + 1) * G].astype(np.float64) @ K.T * scale
            e = np.exp(s - s.max(1, keepdims=True))
            out[i, h * G:(h + 1) * G] = e @ V / e.sum(1, keepdims=True)
    return out


def opt(x):
    return None if x is None else dev(x)


def attend(gpu, q, k, v, ks, vs, table, lens, scale, out=None, ws=None):
    n, nh, hd = q.shape
    if ws is None:
        ws = torch.empty(gpu.ops.paged_attention_workspace_bytes(nh, k.shape[1], hd), dtype=torch.uint8, device="cuda")
    if out is None:
        out = torch.full(q.shape, float("nan"), device="cuda")
    as_dev = lambda x: x if isinstance(x, torch.Tensor) else opt(x)  # noqa: E731
    gpu.ops.paged_attention_decode(as_dev(q), as_dev(k), as_dev(v), as_dev(table), as_dev(lens), out, scale, ws,
                                   as_dev(ks), as_dev(vs))
    return out


EDGES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 600, -3]


@pytest.mark.parametrize("hd,ps,nkv,G,int8", [
    (128, 64, 4, 16, False), (128, 64, 4, 16, True), (128, 16, 2, 5, False), (128, 16, 2, 5, True),
    (128, 32, 1, 1, False), (128, 128, 3, 8, True), (64, 16, 2, 7, False), (64, 64, 12, 1, False),
    (64, 32, 2, 16, True), (256, 16, 1, 16, False), (256, 64, 2, 3, False), (256, 128, 1, 4, True)])
@pytest.mark.parametrize("wide", [False, True])  # tables far wider than the lengths: the kernels of long ones
def test_attention_at_the_edges(gpu, hd, ps, nkv, G, int8, wide):
    rng = np.random.default_rng(hd + ps + G)
    lens = np.array(EDGES, np.int32)
    width = -(-max(EDGES) // ps) + (32768 // ps if wide else 0)
    n_pages = sum(-(-max(n, 0) // ps) for n in EDGES) + 5
    k, v, ks, vs = pool(rng, n_pages, nkv, ps, hd, int8)
    table = block_table(rng, EDGES, ps, width, n_pages)
    q = (rng.standard_normal((len(EDGES), nkv * G, hd)) * rng.uniform(0.3, 1.5, (len(EDGES), nkv * G, 1))).astype(np.float32)
    scale = 1 / math.sqrt(hd)
    case(f"paged attention hd={hd} ps={ps} nkv={nkv} gqa={G} int8={int8} lens={EDGES}")
    got = host(attend(gpu, q, k, v, ks, vs, table, lens, scale))
    want = reference(q, k, v, ks, vs, table, lens, scale)
    for i in range(len(EDGES)):
        if lens[i] <= 0:
            assert not got[i].any(), i
        else:
            assert rel_l2(got[i], want[i]) <= BAR, (i, lens[i])


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("seqs,hi,nkv,hd,ps", [(70, 112, 2, 128, 16), (400, 128, 4, 128, 64), (90, 100, 12, 64, 32),
                                               (130, 128, 3, 256, 128), (4096, 30, 1, 64, 16), (1, 1, 1, 128, 16)])
def test_short_tables(gpu, seqs, hi, nkv, hd, ps, int8):
    """Tables of a few steps, which no workgroup shares with another; more sequences than a wave has lanes."""
    rng = np.random.default_rng(seqs)
    lens = rng.integers(0, hi + 1, seqs).astype(np.int32)
    lens[-1] = hi
    n_pages = int(sum(-(-lens // ps))) + 1
    k, v, ks, vs = pool(rng, n_pages, nkv, ps, hd, int8)
    table = block_table(rng, lens, ps, -(-hi // ps), n_pages)
    q = rng.standard_normal((seqs, nkv * 3, hd)).astype(np.float32)
    case(f"paged attention, short tables seqs={seqs} hi={hi} nkv={nkv} hd={hd} ps={ps} int8={int8}")
    got = host(attend(gpu, q, k, v, ks, vs, table, lens, hd ** -0.5))
    want = reference(q, k, v, ks, vs, table, lens, hd ** -0.5)
    assert not got[lens == 0].any()
    for i in np.flatnonzero(lens):
        assert rel_l2(got[i], want[i]) <= BAR, (i, lens[i])


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("seqs,hi,nkv,G,ps", [(1000, 300, 1, 2, 16), (1, 5000, 4, 16, 64), (1, 70001, 1, 4, 16), (9, 3000, 2, 6, 32),
                                              (70, 400, 4, 8, 64), (3, 40000, 8, 2, 128)])
def test_attention_split_over_the_length(gpu, seqs, hi, nkv, G, ps, int8):
    rng = np.random.default_rng(hi + seqs)
    lens = np.exp(rng.uniform(0, math.log(hi), seqs)).astype(np.int32)
    lens[0] = hi
    n_pages = int(sum(-(-lens // ps))) + 3
    k, v, ks, vs = pool(rng, n_pages, nkv, ps, 128, int8)
    table = block_table(rng, lens, ps, -(-hi // ps) + 3, n_pages)
    q = rng.standard_normal((seqs, nkv * G, 128)).astype(np.float32)
    case(f"paged attention seqs={seqs} hi={hi} nkv={nkv} gqa={G} ps={ps} int8={int8}")
    got = attend(gpu, q, k, v, ks, vs, table, lens, 128 ** -0.5)
    again = attend(gpu, q, k, v, ks, vs, table, lens, 128 ** -0.5)
    assert torch.equal(got, again)
    want = reference(q, k, v, ks, vs, table, lens, 128 ** -0.5)
    for i in range(seqs):
        assert rel_l2(host(got)[i], want[i]) <= BAR, (i, lens[i])


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("seqs,hi,nkv,hd,G,ps", [(90, 700, 3, 64, 2, 16), (300, 260, 1, 256, 3, 32), (40, 900, 8, 128, 4, 128),
                                                 (30, 400, 12, 64, 1, 64), (2, 20000, 2, 256, 16, 64), (5, 9000, 3, 64, 9, 128)])
def test_many_and_few_sequences_of_every_head_size(gpu, seqs, hi, nkv, hd, G, ps, int8):
    """More (sequence, KV head)s than workgroups, and far fewer, with shares that cut them."""
    rng = np.random.default_rng(seqs + hd)
    lens = rng.integers(0, hi + 1, seqs).astype(np.int32)
    lens[seqs // 2] = hi
    n_pages = int(sum(-(-lens // ps))) + 1
    k, v, ks, vs = pool(rng, n_pages, nkv, ps, hd, int8)
    table = block_table(rng, lens, ps, -(-hi // ps) + 1, n_pages)
    q = rng.standard_normal((seqs, nkv * G, hd)).astype(np.float32)
    case(f"paged attention seqs={seqs} hi={hi} nkv={nkv} hd={hd} gqa={G} ps={ps} int8={int8}")
    got = attend(gpu, q, k, v, ks, vs, table, lens, hd ** -0.5)
    assert torch.equal(got, attend(gpu, q, k, v, ks, vs, table, lens, hd ** -0.5))
    want = reference(q, k, v, ks, vs, table, lens, hd ** -0.5)
    for i in range(seqs):
        if lens[i] == 0:
            assert not host(got)[i].any()
        else:
            assert rel_l2(host(got)[i], want[i]) <= BAR, (i, lens[i])


def test_rows_behind_the_last_are_left(gpu):
    """The C entry points write n_seqs, n_tokens and n_rows rows and nothing behind them."""
    import ctypes as C
    lib = gpu.load_library()
    rng = np.random.default_rng(21)
    p = lambda t: C.c_void_p(t.data_ptr())  # noqa: E731
    stream = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    k, v, _, _ = pool(rng, 40, 2, 16, 64, False)
    kd, vd = dev(k), dev(v)
    lens = np.array([100, 0, 33, 5], np.int32)
    table, ld = dev(block_table(rng, lens, 16, 8, 40)), dev(lens)
    q, out = dev(rng.standard_normal((4, 6, 64)).astype(np.float32)), torch.full((4, 6, 64), 3.0, device="cuda")
    n = gpu.ops.paged_attention_workspace_bytes(6, 2, 64)
    ws = torch.full((n + 256,), 0x5A, dtype=torch.uint8, device="cuda")
    case("rows behind the last")
    assert lib.mnemo_paged_attention_decode(p(q), p(kd), p(vd), None, None, 0, p(out), 3, 6, 64, 2, 40, 16, p(table), 8, p(ld),
                                            0.1, p(ws), n, stream) == 0
    o = host(out)
    assert (o[3] == 3.0).all() and not o[1].any() and (o[0] != 3.0).all()
    assert (host(ws)[n:] == 0x5A).all()
    kn = dev(rng.standard_normal((4, 2, 64)).astype(np.float32))
    before = [x.clone() for x in (kd, vd)]
    out.fill_(3.0)
    assert lib.mnemo_paged_attn_prep(p(q), p(kn), p(kn), None, None, 1e-6, 1e4, 3, 6, 64, 2, None, None, p(table), p(ld), 4, 8,
                                     p(kd), p(vd), None, None, 0, 40, 16, p(out), stream) == 0
    o, t = host(out), host(table)
    assert (o[3] == 3.0).all() and (o[1] == 3.0).all() and (o[0] != 3.0).all() and (o[2] != 3.0).all()
    changed = (kd != before[0]).any(-1).nonzero().tolist()
    assert sorted(set((a, c) for a, _, c in changed)) == sorted([(t[0, 6], 3), (t[2, 2], 0)])
    z, zo = torch.randn((3, 77), device="cuda"), torch.full((3, 77), 3.0, device="cuda")
    assert lib.mnemo_logits_process(p(z), p(zo), 2, 77, None, None, None, 0, None, None, None, None, None, 0, None, stream) == 0
    assert torch.equal(zo[:2], z[:2]) and (host(zo)[2] == 3.0).all()
    lib.mnemo_last_error()


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("ps", [16, 64])
def test_positions_past_the_end_are_not_looked_at(gpu, ps, int8):
    """NaN and infinities in the unused rest of a last page, in pages that nothing names, and in the table's rest."""
    rng = np.random.default_rng(ps)
    lens = np.array([1, 9, ps + 3, 3 * ps - 1, 200], np.int32)
    width = 200 // ps + 4
    n_pages = int(sum(-(-lens // ps))) + 6
    k, v, ks, vs = pool(rng, n_pages, 2, ps, 128, int8)
    table = block_table(rng, lens, ps, width, n_pages)
    q = rng.standard_normal((5, 8, 128)).astype(np.float32)
    want = reference(q, k, v, ks, vs, table, lens, 0.1)
    used = np.zeros((n_pages, ps), bool)
    for i, n in enumerate(lens):
        pos = np.arange(n)
        used[table[i, pos // ps], pos % ps] = True
    dead = np.argwhere(~used)
    bad = rng.choice(np.array([np.nan, np.inf, -np.inf], np.float32), len(dead))
    for (p, o), b in zip(dead, bad):
        if int8:
            ks[p, :, o] = vs[p, :, o] = b
        else:
            k[p, :, o] = v[p, :, :, o] = b
    for i, n in enumerate(lens):  # the table's rest names pages that hold no number at all, or none
        rest = table[i, -(-n // ps):]
        rest[:] = rng.choice(np.array([-1, n_pages, 2 ** 31 - 1, -2 ** 31, n_pages - 1], np.int64), len(rest)).astype(np.int32)
    case(f"paged attention, NaN past the end, ps={ps} int8={int8}")
    got = host(attend(gpu, q, k, v, ks, vs, table, lens, 0.1))
    assert rel_l2(got, want) <= BAR


@pytest.mark.parametrize("int8", [False, True])
def test_pages_that_are_not_there(gpu, int8):
    """Table entries outside the pool count as absent positions; a row of them gives zeros; a length past the table
    is cut to it."""
    rng = np.random.default_rng(3)
    lens = np.array([300, 64, 200, 100000], np.int32)
    k, v, ks, vs = pool(rng, 40, 2, 16, 128, int8)
    table = block_table(rng, [320, 64, 208, 20 * 16], 16, 20, 60) % 40
    table[0, 3], table[0, 7], table[0, 18] = -1, 40, 2 ** 31 - 1
    table[1, :4] = [-1, -5, 40, -2 ** 31]
    q = rng.standard_normal((4, 6, 128)).astype(np.float32)
    case(f"paged attention, invalid pages, int8={int8}")
    got = host(attend(gpu, q, k, v, ks, vs, table, lens, 0.09))
    want = reference(q, k, v, ks, vs, table, lens, 0.09)
    assert not got[1].any()
    for i in (0, 2, 3):
        assert rel_l2(got[i], want[i]) <= BAR, i


@pytest.mark.parametrize("int8", [False, True])
def test_size_of_the_query(gpu, int8):
    """A query 2^20 times larger under a scale 2^20 times smaller (and the other way round) gives the same result bit
    for bit: powers of two round nothing."""
    rng = np.random.default_rng(8)
    lens = np.array([700, 33], np.int32)
    k, v, ks, vs = pool(rng, 60, 2, 16, 128, int8)
    table = block_table(rng, lens, 16, 44, 60)
    q = rng.standard_normal((2, 10, 128)).astype(np.float32)
    case(f"paged attention, scaled queries, int8={int8}")
    base = attend(gpu, q, k, v, ks, vs, table, lens, 0.08)
    assert rel_l2(host(base), reference(q, k, v, ks, vs, table, lens, 0.08)) <= BAR
    for f in (2.0 ** 20, 2.0 ** -20):
        got = attend(gpu, (q * np.float32(f)), k, v, ks, vs, table, lens, float(np.float32(0.08)) / f)
        assert torch.equal(got, base), f


def test_value_scales_of_any_size(gpu):
    """int8 value scales from 1e-8 to 1e8: each sequence's relative error is held (weights times scales do not leave
    the range of the matrix instructions' operands)."""
    rng = np.random.default_rng(9)
    sizes = [1e-8, 1e-3, 1.0, 1e4, 1e8]
    lens = np.full(len(sizes), 150, np.int32)
    k, v, ks, vs = pool(rng, 60, 2, 16, 128, True)
    table = block_table(rng, lens, 16, 10, 60)
    for i, f in enumerate(sizes):
        vs[table[i]] *= np.float32(f)
    q = rng.standard_normal((len(sizes), 4, 128)).astype(np.float32)
    case("paged attention, value scales")
    got = host(attend(gpu, q, k, v, ks, vs, table, lens, 0.09))
    want = reference(q, k, v, ks, vs, table, lens, 0.09)
    for i in range(len(sizes)):
        assert rel_l2(got[i], want[i]) <= BAR, sizes[i]


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
    q = rng.standard_normal((1, nkv * 2, hd)).astype(np.float32)
    lens = np.array([4 * ps - 5], np.int32)
    case("paged attention past 4 GiB")
    got = host(attend(gpu, q, k, v, None, None, ids[None], lens, 0.06))
    want = reference(q, kk, vv, None, None, np.arange(4, dtype=np.int32)[None], lens, 0.06)
    assert rel_l2(got, want) <= BAR


def test_attention_in_a_graph(gpu):
    """One captured call serves other lengths, tables and queries; replays between eager calls on the same workspace."""
    rng = np.random.default_rng(11)
    k, v, _, _ = pool(rng, 200, 4, 32, 128, False)
    kd, vd = dev(k), dev(v)
    table, lens = torch.full((3, 60), -1, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    q = torch.zeros((3, 32, 128), device="cuda")
    out = torch.empty_like(q)
    ws = torch.empty(gpu.ops.paged_attention_workspace_bytes(32, 4, 128), dtype=torch.uint8, device="cuda")
    call = lambda: gpu.ops.paged_attention_decode(q, kd, vd, table, lens, out, 0.09, ws)  # noqa: E731
    case("paged attention graph capture")
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        call()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            call()
    for ln in ([5, 0, 1900], [1, 700, 33], [0, 0, 0], [1900, 1900, 1900]):
        t = block_table(rng, ln, 32, 60, 200)
        qq = rng.standard_normal((3, 32, 128)).astype(np.float32)
        table.copy_(dev(t)), lens.copy_(dev(np.array(ln, np.int32))), q.copy_(dev(qq))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        out.zero_()
        call()
        assert torch.equal(out, got)
        want = reference(qq, k, v, None, None, t, ln, 0.09)
        assert rel_l2(host(got), want) <= BAR, ln


def test_attention_on_two_streams(gpu):
    rng = np.random.default_rng(12)
    k, v, _, _ = pool(rng, 600, 4, 64, 128, False)
    kd, vd = dev(k), dev(v)
    jobs = []
    for i in range(2):
        lens = np.array([15000 - 333 * i, 100, 7], np.int32)
        table = block_table(rng, lens, 64, 240, 600)
        q = rng.standard_normal((3, 64, 128)).astype(np.float32)
        ws = torch.empty(gpu.ops.paged_attention_workspace_bytes(64, 4, 128), dtype=torch.uint8, device="cuda")
        jobs.append((q, table, lens, torch.cuda.Stream(), dev(q), dev(table), dev(lens), torch.empty(q.shape, device="cuda"), ws))
    torch.cuda.synchronize()
    case("paged attention on two streams")
    for _ in range(5):
        for q, table, lens, st, qd, td, ld, out, ws in jobs:
            with torch.cuda.stream(st):
                gpu.ops.paged_attention_decode(qd, kd, vd, td, ld, out, 0.09, ws)
    torch.cuda.synchronize()
    for q, table, lens, st, qd, td, ld, out, ws in jobs:
        assert rel_l2(host(out), reference(q, k, v, None, None, table, lens, 0.09)) <= BAR


# ------------------------------------------------------------------ preparation and store
def rotated(x, w, pos, theta, eps):
    """RMS norm (w None: none) and RoPE of x [T][heads][hd] in 64 bits."""
    x = x.astype(np.float64)
    hd = x.shape[-1]
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w.astype(np.float64)
    a = pos.astype(np.float64)[:, None] * theta ** (-2.0 * np.arange(hd // 2) / hd)
    a = np.fmod(a, 2 * np.pi)
    c, s = np.cos(a)[:, None], np.sin(a)[:, None]
    x0, x1 = x[..., :hd // 2], x[..., hd // 2:]
    return np.concatenate([x0 * c - x1 * s, x1 * c + x0 * s], -1)


# An element of a rotated head: norm factor, weight, two products with a sine and a cosine (each off by ~2^-23 of 1,
# the angle's own rounding included) and their sum: below 16 roundings of 2^-24 of the head's largest element times
# sqrt 2.
ROT = 16 * math.sqrt(2) * 2.0 ** -24


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("hd,ps,nkv,nh,norm", [(128, 64, 4, 64, True), (64, 16, 3, 9, True), (256, 32, 1, 5, False),
                                               (128, 128, 2, 2, False), (128, 16, 8, 40, True)])
def test_prep(gpu, hd, ps, nkv, nh, norm, int8):
    """Tokens of several sequences in one call: runs that start and end inside pages, single tokens, padding, a far
    position, a position past the table, a row that is not there, a page that is not there."""
    rng = np.random.default_rng(hd + ps + nh)
    theta, eps, n_seqs, width = 1e6, 1e-6, 5, 14
    n_pages = n_seqs * width + 4
    table = rng.permutation(n_pages)[:n_seqs * width].astype(np.int32).reshape(n_seqs, width)
    table[3, 5] = n_pages
    runs = [(0, 0, 41), (1, ps - 3, ps + 9), (2, 5 * ps + 7, 1), (3, 5 * ps - 1, 3), (4, width * ps - 2, 4), (1, -2, 1),
            (0, 60, 3), (-1, 3, 1), (n_seqs, 3, 1)]
    seq = np.concatenate([np.full(n, s) for s, p, n in runs]).astype(np.int32)
    pos = np.concatenate([np.arange(p, p + n) for s, p, n in runs]).astype(np.int32)
    T = len(seq)
    q, k, v = (rng.standard_normal((T, h, hd)).astype(np.float32) * 3 for h in (nh, nkv, nkv))
    qw, kw = ((1 + 0.2 * rng.standard_normal(hd)).astype(np.float32) for _ in range(2))
    kp, vp, ks, vs = pool(rng, n_pages, nkv, ps, hd, int8)
    kpd, vpd, ksd, vsd = opt(kp), opt(vp), opt(ks), opt(vs)
    q_out = torch.full((T, nh, hd), 7.0, device="cuda")
    kd, vd = dev(k), dev(v)
    case(f"paged prep hd={hd} ps={ps} nkv={nkv} nh={nh} norm={norm} int8={int8}")
    gpu.ops.paged_attn_prep(dev(q), kd, vd, dev(qw) if norm else None, dev(kw) if norm else None, eps, theta, kpd, vpd,
                            dev(table), q_out, dev(pos), dev(seq), ksd, vsd)
    assert np.array_equal(host(kd), k) and np.array_equal(host(vd), v)
    live = pos >= 0
    want_q = rotated(q, qw if norm else None, np.maximum(pos, 0), theta, eps)
    got_q = host(q_out)
    assert (got_q[~live] == 7.0).all()
    err = np.abs(got_q - want_q)[live]
    assert (err <= ROT * np.abs(want_q[live]).max(-1, keepdims=True)).all(), err.max()
    want_k = rotated(k, kw if norm else None, np.maximum(pos, 0), theta, eps)
    # the pages: what was not written stays, bit for bit
    touched = np.zeros((n_pages, ps), bool)
    got = [host(kpd), host(vpd)] + ([host(ksd), host(vsd)] if int8 else [])
    stored = 0
    for t in range(T):
        if pos[t] < 0 or not 0 <= seq[t] < n_seqs or pos[t] // ps >= width or table[seq[t], pos[t] // ps] >= n_pages:
            continue
        p, o = table[seq[t], pos[t] // ps], pos[t] % ps
        assert not touched[p, o]
        touched[p, o] = True
        stored += 1
        for x, row, sc in ((want_k[t], got[0][p, :, o], 2), (v[t].astype(np.float64), got[1][p, :, :, o], 3)):
            size = np.abs(x).max(-1, keepdims=True)
            rounding = ROT * size if sc == 2 else 0.0
            if int8:
                step = got[sc][p, :, o][:, None].astype(np.float64)
                np.testing.assert_allclose(step, size / 127, rtol=ROT + 2.0 ** -23)
                # half a step, plus what the value, its quotient and the scale are off by
                assert (np.abs(row * step - x) <= 0.5 * step + rounding + 127 * step * 2.0 ** -22).all()
                assert np.abs(row).max() == 127
            else:
                assert (np.abs(row.astype(np.float64) - x) <= np.abs(x) * 2.0 ** -11 + 2.0 ** -25 + rounding).all()
    assert stored == 41 + (ps + 9) + 1 + 1 + 2 + 3  # two of row 3 fall on a page that is not there, two of row 4 past the table
    for new, old in zip(got, (kp, vp, ks, vs)):
        hit = touched[:, None, None, :] if new is got[1] else touched[:, None, :, None] if new is got[0] else touched[:, None]
        hit = np.broadcast_to(hit, new.shape)
        assert np.array_equal(new[~hit].view(np.uint8), old[~hit].view(np.uint8))


@pytest.mark.parametrize("hd,ps,nkv,nh", [(128, 64, 4, 8), (64, 16, 12, 12), (256, 32, 3, 3), (128, 128, 8, 16)])
@pytest.mark.parametrize("int8", [False, True])
def test_prep_of_many_tokens(gpu, hd, ps, nkv, nh, int8):
    """A call of many tokens equals calls of few, bit for bit: runs that begin anywhere in a page, runs of under
    eight, two sequences' tokens in turn, a run backwards, padding and absent pages within a run."""
    rng = np.random.default_rng(hd + ps + nkv)
    n_seqs, width = 6, 1200 // ps + 2
    n_pages = n_seqs * width
    table = rng.permutation(n_pages).astype(np.int32).reshape(n_seqs, width)
    table[2, 1] = -1
    seq, pos = [], []
    for s, p in [(0, range(3, 503)), (1, range(8, 13)), (1, range(16, 24)), (2, range(0, 300)), (3, range(400, 200, -1)),
                 (4, [x for i in range(100) for x in (i, -1)]), (1, range(100, 101)), (5, range(64, 1000))]:
        seq += [s] * len(p)
        pos += list(p)
    a = np.arange(200)  # two sequences in turn
    seq += list(np.where(a % 2, 0, 3))
    pos += list(600 + a // 2)
    seq, pos = np.array(seq, np.int32), np.array(pos, np.int32)
    pos[1100:1103] = -1
    T = len(seq)
    assert T * nkv >= 2048
    q, k, v = (rng.standard_normal((T, h, hd)).astype(np.float32) for h in (nh, nkv, nkv))
    w = dev(np.ones(hd, np.float32))
    start = pool(rng, n_pages, nkv, ps, hd, int8)
    qd, kd, vd, td, sd, pd = dev(q), dev(k), dev(v), dev(table), dev(seq), dev(pos)
    got = []
    for step in (T, 100):
        p = [opt(x) for x in start]
        qo = torch.zeros((T, nh, hd), device="cuda")
        case(f"paged prep of {T} tokens by {step}, hd={hd} ps={ps} nkv={nkv} int8={int8}")
        for t in range(0, T, step):
            at = slice(t, t + step)
            gpu.ops.paged_attn_prep(qd[at], kd[at], vd[at], w, w, 1e-6, 1e6, p[0], p[1], td, qo[at], pd[at], sd[at], p[2], p[3])
        got.append([qo] + [x for x in p if x is not None])
    for x, y in zip(*got):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    assert not torch.equal(got[0][1].view(torch.uint8), opt(start[0]).view(torch.uint8))


@pytest.mark.parametrize("theta", [1e6, 1e4, 1.0])
def test_prep_far_positions(gpu, theta):
    """Positions to 2^31 - 1: the angle loses nothing."""
    pos = np.array([0, 1, 4095, 131071, 10 ** 6, 10 ** 7 + 1, 2 ** 30 + 1, 2 ** 31 - 1], np.int32)
    T, nh, hd = len(pos), 3, 128
    rng = np.random.default_rng(5)
    q = rng.standard_normal((T, nh, hd)).astype(np.float32)
    kv = torch.zeros((T, 1, hd), device="cuda")
    kp = torch.zeros((1, 1, 16, hd), dtype=torch.float16, device="cuda")
    vp = torch.zeros((1, 1, hd, 16), dtype=torch.float16, device="cuda")
    qd = dev(q)
    case(f"paged prep, far positions, theta={theta}")
    gpu.ops.paged_attn_prep(qd, kv, kv, None, None, 1e-6, theta, kp, vp, torch.full((1, 1), -1, dtype=torch.int32, device="cuda"),
                            qd, dev(pos), torch.zeros(T, dtype=torch.int32, device="cuda"))  # in place
    # the angle in extended precision: position times the frequency, reduced
    f = np.longdouble(theta) ** (-2 * np.arange(hd // 2, dtype=np.longdouble) / hd)
    a = np.fmod(pos.astype(np.longdouble)[:, None] * f, 2 * np.arccos(np.longdouble(-1)))
    c, s = np.cos(a)[:, None].astype(np.float64), np.sin(a)[:, None].astype(np.float64)
    x0, x1 = q[..., :64].astype(np.float64), q[..., 64:].astype(np.float64)
    want = np.concatenate([x0 * c - x1 * s, x1 * c + x0 * s], -1)
    # frequencies in 64 bits: pi, the power and the quotient are off by 2^-53 each, of the angle
    bound = (ROT + pos.astype(np.float64) * 2.0 ** -51)[:, None, None] * np.abs(want).max(-1, keepdims=True)
    assert (np.abs(host(qd) - want) <= bound).all()


def test_prep_by_lengths(gpu):
    """Without positions, token t is the last position of row t; empty rows are padding."""
    rng = np.random.default_rng(6)
    lens = np.array([5, 0, 17, 32], np.int32)
    table = np.arange(8, dtype=np.int32).reshape(4, 2)
    q, k, v = (rng.standard_normal((4, h, 64)).astype(np.float32) for h in (4, 2, 2))
    outs = []
    for by_lens in (True, False):
        kp = torch.zeros((8, 2, 16, 64), dtype=torch.float16, device="cuda")
        vp = torch.zeros((8, 2, 64, 16), dtype=torch.float16, device="cuda")
        qo = torch.zeros((4, 4, 64), device="cuda")
        where = dict(seq_lens=dev(lens)) if by_lens else dict(positions=dev(lens - 1), seq_ids=dev(np.arange(4, dtype=np.int32)))
        case(f"paged prep by lengths={by_lens}")
        gpu.ops.paged_attn_prep(dev(q), dev(k), dev(v), None, None, 1e-6, 1e4, kp, vp, dev(table), qo, **where)
        outs.append((qo, kp, vp))
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    assert not host(outs[0][0])[1].any() and host(outs[0][0])[0].any()


def test_int8_rows_of_zeros_and_of_tiny_values(gpu):
    """A row of zeros and one below the smallest usable scale are stored as zeros, not as rounding noise."""
    x = np.zeros((3, 1, 64), np.float32)
    x[1] = 1e-39
    x[2] = np.linspace(-1e-30, 1e-30, 64)
    kp = torch.full((1, 1, 16, 64), 9, dtype=torch.int8, device="cuda")
    vp = torch.full((1, 1, 64, 16), 9, dtype=torch.int8, device="cuda")
    ks, vs = torch.full((1, 1, 16), 9.0, device="cuda"), torch.full((1, 1, 16), 9.0, device="cuda")
    case("paged prep, int8 zeros")
    gpu.ops.paged_attn_prep(dev(x), dev(x), dev(x), None, None, 1e-6, 1e4, kp, vp, torch.zeros((1, 1), dtype=torch.int32, device="cuda"),
                            torch.empty((3, 1, 64), device="cuda"), torch.arange(3, dtype=torch.int32, device="cuda"),
                            torch.zeros(3, dtype=torch.int32, device="cuda"), ks, vs)
    for p, s in ((host(kp)[0, 0, :3], host(ks)), (host(vp)[0, 0, :, :3].T, host(vs))):
        assert not p[:2].any() and not s[0, 0, :2].any()
        assert np.abs(p[2]).max() == 127



@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("lens,nkv,hd,ps", [([10, 5000, 300, 64, 20000], 2, 128, 64), ([7, 900, 4000], 1, 256, 32),
                                            (list(range(1, 1400, 14)), 3, 64, 16)])
def test_queries_that_are_no_number(gpu, lens, nkv, hd, ps, int8):
    """A query head that holds a NaN or an infinity gives NaN, whether its sequence lies in one workgroup's share or in
    several (few and many sequences: both kinds of merge); the other heads are not touched."""
    rng = np.random.default_rng(hd)
    lens = np.array(lens, np.int32)
    n_pages = int(sum(-(-lens // ps))) + 1
    k, v, ks, vs = pool(rng, n_pages, nkv, ps, hd, int8)
    table = block_table(rng, lens, ps, -(-int(lens.max()) // ps) + 2, n_pages)
    nh = 3 * nkv
    q = rng.standard_normal((len(lens), nh, hd)).astype(np.float32)
    want = reference(q, k, v, ks, vs, table, lens, hd ** -0.5)
    bad = np.zeros((len(lens), nh), bool)
    for i in range(len(lens)):
        bad[i, [i % nh, (i + 4) % nh]] = True
        q[i, i % nh, (5 * i) % hd] = np.nan
        q[i, (i + 4) % nh, (7 * i) % hd] = (np.inf, np.nan)[i % 2]
    case(f"paged attention, NaN queries, {len(lens)} sequences nkv={nkv} hd={hd} int8={int8}")
    got = host(attend(gpu, q, k, v, ks, vs, table, lens, hd ** -0.5))
    for i in range(len(lens)):
        for h in range(nh):
            if bad[i, h]:
                assert np.isnan(got[i, h]).all(), (i, h, lens[i])
            else:
                assert rel_l2(got[i, h], want[i, h]) <= 2 * BAR, (i, h, lens[i])  # one head: two deviations



# Scores of these tests: K rows and queries of equal signs, so that a head's products are one power of two and their sum is
# exact; scale, log2(e) and the key's scale are four roundings of the score S, its difference to the maximum another
# (2^-24 each, of S at most), exp2 and the weight's three products and its sum 16 at most of the weight itself.  So a
# weight is off by (6 S + 16) 2^-24 of itself, numerator and denominator both; a sum over n positions by n 2^-24 of the
# sizes that it adds; and the two f16 parts of a weight times scale by 2^-33 of the largest of them per position.
@pytest.mark.parametrize("order", ["random", "scores rise", "scores fall", "one large", "one large at last"])
@pytest.mark.parametrize("n,nkv,hd,ps", [(64, 1, 128, 16), (150, 2, 64, 32), (3000, 2, 128, 64), (900, 1, 256, 128)])
def test_value_scales_within_a_sequence(gpu, n, nkv, hd, ps, order):
    """int8 value scales that differ by many orders of magnitude within one sequence, also where the largest of them has
    next to no weight."""
    rng = np.random.default_rng(n + len(order))
    width = -(-n // ps)
    u = rng.choice(np.array([-1, 1], np.int8), hd)
    k = np.broadcast_to(u, (width, nkv, ps, hd)).copy()
    v = rng.integers(-127, 128, (width, nkv, hd, ps)).astype(np.int8)
    a = np.array([1.0, 0.5, 0.25, 1.0])
    q = np.tile((a[:, None] * u).astype(np.float32), (nkv, 1))[None]
    for trial in range(4):
        if order.startswith("one"):  # the other scales 1e-6, 1e-8, 1e-12 and 1e-20 of it
            s = rng.uniform(0, 3, (nkv, width * ps))
            vs = rng.uniform(0.5, 1.5, s.shape) * (1e-6, 1e-8, 1e-12, 1e-20)[trial]
            at = n - 1 if order.endswith("last") else n // 2
            s[:, at], vs[:, at] = -50.0, 1.0
        else:
            s = rng.uniform(-30, 30, (nkv, width * ps))
            if order != "random":
                s[:, :n] = np.sort(s[:, :n], -1)[:, ::1 if order == "scores rise" else -1]
            vs = 10 ** rng.uniform(-15, 15, s.shape)
            if trial % 2:  # large scales on small scores
                vs = np.exp(-s * (0.5 + 0.5 * trial)) * rng.uniform(0.5, 1.5, s.shape)
        ks = np.ascontiguousarray(s.astype(np.float32).reshape(nkv, width, ps).transpose(1, 0, 2))
        vs = np.ascontiguousarray(vs.astype(np.float32).reshape(nkv, width, ps).transpose(1, 0, 2))
        table, lens = np.arange(width, dtype=np.int32)[None], np.array([n], np.int32)
        case(f"paged attention, value scales within a sequence n={n} nkv={nkv} hd={hd} {order} {trial}")
        got = host(attend(gpu, q, k, v, ks, vs, table, lens, 1.0 / hd))[0]
        for h in range(4 * nkv):
            g = h // 4
            sc = a[h % 4] * ks[:, g].astype(np.float64).flatten()[:n]
            w = np.exp(sc - sc.max())
            sizes = w * vs[:, g].astype(np.float64).flatten()[:n]
            V = v[:, g].transpose(0, 2, 1).reshape(-1, hd)[:n].astype(np.float64)
            want = sizes @ V / w.sum()
            eps = 2 * (6 * np.abs(sc).max() + 16 + n) * 2.0 ** -24
            bound = (eps * (sizes @ np.abs(V)) + n * 2.0 ** -33 * 127 * sizes.max()) / w.sum()
            assert (np.abs(got[h] - want) <= bound).all(), (trial, h, np.abs(got[h] - want).max(), bound.max())



def test_prep_stores_nothing_past_the_lengths(gpu):
    """With positions and lengths, a token at or past its row's length (a row that could not be extended) is prepared
    but not stored."""
    rng = np.random.default_rng(17)
    lens = np.array([5, 0, 20, 33], np.int32)
    table = np.arange(16, dtype=np.int32).reshape(4, 4)
    seq = np.array([0, 0, 1, 2, 2, 2, 3, 3, -1, 4], np.int32)
    pos = np.array([4, 5, 0, 18, 20, 63, 31, 33, 2, 2], np.int32)
    q, k, v = (rng.standard_normal((10, h, 64)).astype(np.float32) for h in (4, 2, 2))
    for int8 in (False, True):
        p = [opt(x) for x in pool(rng, 16, 2, 16, 64, int8)]
        before = [None if x is None else x.clone() for x in p]
        alone = [None if x is None else x.clone() for x in p]
        qo, qa = torch.zeros((10, 4, 64), device="cuda"), torch.zeros((10, 4, 64), device="cuda")
        case(f"paged prep past the lengths int8={int8}")
        gpu.ops.paged_attn_prep(dev(q), dev(k), dev(v), None, None, 1e-6, 1e4, p[0], p[1], dev(table), qo, dev(pos), dev(seq),
                                p[2], p[3], seq_lens=dev(lens))
        keep = [0, 3, 6]
        gpu.ops.paged_attn_prep(dev(q), dev(k), dev(v), None, None, 1e-6, 1e4, alone[0], alone[1], dev(table), qa, dev(pos),
                                dev(np.where(np.isin(np.arange(10), keep), seq, -1).astype(np.int32)), alone[2], alone[3])
        assert torch.equal(qo, qa)
        for x, y, b in zip(p, alone, before):
            if x is not None:
                assert torch.equal(x.view(torch.uint8), y.view(torch.uint8)) and not torch.equal(x, b)



@pytest.mark.parametrize("hd,T", [(64, 40), (128, 40), (256, 40), (64, 2100), (128, 2100), (256, 2100)])
def test_int8_rows_that_hold_no_number(gpu, hd, T):
    """A row with a NaN or an infinity reads back as NaN throughout, as its definition says (the scale is the largest
    absolute value / 127); its neighbours are as without it."""
    rng = np.random.default_rng(hd)
    x = rng.standard_normal((T, 1, hd)).astype(np.float32)
    ps, width = 64, -(-T // 64)
    outs = []
    bad = np.zeros(T, bool)
    bad[[0, 7, 18, 33, T - 1]] = True
    y = x.copy()
    y[bad, 0, rng.integers(0, hd, 5)] = [np.nan, np.inf, -np.inf, np.nan, -np.inf]
    y[18, 0, :3] = np.nan
    for z in (x, y):
        kp = torch.full((width, 1, ps, hd), 9, dtype=torch.int8, device="cuda")
        vp = torch.full((width, 1, hd, ps), 9, dtype=torch.int8, device="cuda")
        ks, vs = torch.full((width, 1, ps), 9.0, device="cuda"), torch.full((width, 1, ps), 9.0, device="cuda")
        case(f"paged prep, int8 rows with NaN hd={hd} T={T}")
        gpu.ops.paged_attn_prep(dev(z), dev(z), dev(z), None, None, 1e-6, 1e4, kp, vp, torch.arange(width, dtype=torch.int32, device="cuda")[None],
                                torch.empty((T, 1, hd), device="cuda"), torch.arange(T, dtype=torch.int32, device="cuda"),
                                torch.zeros(T, dtype=torch.int32, device="cuda"), ks, vs)
        with np.errstate(invalid="ignore"):
            outs.append((host(kp)[:, 0].reshape(-1, hd)[:T] * host(ks).flatten()[:T, None],
                         host(vp)[:, 0].transpose(0, 2, 1).reshape(-1, hd)[:T] * host(vs).flatten()[:T, None]))
    for a, b in zip(*outs):
        assert np.isnan(b[bad]).all()
        assert np.array_equal(a[~bad], b[~bad])
    # attention over such a cache says so
    q = torch.ones((1, 2, hd), device="cuda")
    table, n = torch.arange(width, dtype=torch.int32, device="cuda")[None], torch.tensor([T], dtype=torch.int32, device="cuda")
    for scales in ((ks, torch.nan_to_num(vs)), (torch.nan_to_num(ks), vs)):
        assert np.isnan(host(attend(gpu, q, kp, vp, *scales, table, n, 0.1))).all()



@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("theta", [1.0 + 2.0 ** -23, 1.00009, 1.0104, 1e3, 3e38])
def test_prep_far_positions_of_every_head_size(gpu, hd, theta):
    """Bases next to 1, where the frequencies' factors are next to 1 as well, and the largest one."""
    theta = float(np.float32(theta))
    pos = np.array([3, 131071, 10 ** 7 + 1, 2 ** 30 + 1, 2 ** 31 - 1], np.int32)
    rng = np.random.default_rng(15)
    q = rng.standard_normal((len(pos), 2, hd)).astype(np.float32)
    kv = torch.zeros((len(pos), 1, hd), device="cuda")
    kp = torch.zeros((1, 1, 16, hd), dtype=torch.float16, device="cuda")
    vp = torch.zeros((1, 1, hd, 16), dtype=torch.float16, device="cuda")
    qd = dev(q)
    case(f"paged prep, far positions, hd={hd} theta={theta}")
    gpu.ops.paged_attn_prep(qd, kv, kv, None, None, 1e-6, theta, kp, vp, torch.full((1, 1), -1, dtype=torch.int32, device="cuda"),
                            qd, dev(pos), torch.zeros(len(pos), dtype=torch.int32, device="cuda"))
    # the angle in extended precision, whose frequencies are off by 2^-63 of themselves (4 roundings), products by as much
    f = np.longdouble(theta) ** (-2 * np.arange(hd // 2, dtype=np.longdouble) / hd)
    a = np.fmod(pos.astype(np.longdouble)[:, None] * f, 2 * np.arccos(np.longdouble(-1)))
    c, s = np.cos(a)[:, None].astype(np.float64), np.sin(a)[:, None].astype(np.float64)
    x0, x1 = q[..., :hd // 2].astype(np.float64), q[..., hd // 2:].astype(np.float64)
    want = np.concatenate([x0 * c - x1 * s, x1 * c + x0 * s], -1)
    # the kernel's angle: 10 p 2^-64 and, cut off when it is reduced, 2^-32 of a turn
    off = (pos.astype(np.float64) * (2.0 ** -64 * 10 * 2 * math.pi + 2.0 ** -60) + 2.0 ** -32 * 2 * math.pi)[:, None, None]
    assert (np.abs(host(qd) - want) <= (ROT + off) * np.abs(want).max(-1, keepdims=True)).all()


@pytest.mark.parametrize("int8", [False, True])
def test_tokens_of_chunks_as_rows(gpu, int8):
    """Chunks of prompts: stored in one call, then attended with a table that has a row for every token, a copy of its
    sequence's, and the length up to it: causal, over the pages that the rows share."""
    rng = np.random.default_rng(31)
    ps, nkv, G, hd = 32, 2, 4, 128
    begin, n = np.array([0, 70, 31, 5]), np.array([130, 33, 2, 1])
    lens = (begin + n).astype(np.int32)
    n_pages = int(sum(-(-lens // ps))) + 2
    pages = pool(rng, n_pages, nkv, ps, hd, int8)
    table = block_table(rng, lens, ps, 6, n_pages)
    seq = np.repeat(np.arange(4), n).astype(np.int32)
    pos = np.concatenate([np.arange(b, b + m) for b, m in zip(begin, n)]).astype(np.int32)
    T = len(seq)
    q, k, v = (rng.standard_normal((T, h, hd)).astype(np.float32) for h in (nkv * G, nkv, nkv))
    p = [opt(x) for x in pages]
    qo = torch.empty((T, nkv * G, hd), device="cuda")
    case(f"chunks as rows int8={int8}")
    gpu.ops.paged_attn_prep(dev(q), dev(k), dev(v), None, None, 1e-6, 1e4, p[0], p[1], dev(table), qo, dev(pos), dev(seq), p[2],
                            p[3], seq_lens=dev(lens))
    got = host(attend(gpu, qo, *p, table[seq], pos + 1, hd ** -0.5))
    stored = [None if x is None else host(x) for x in p]
    want = reference(host(qo), *stored, table[seq], pos + 1, hd ** -0.5)
    for t in range(T):
        assert rel_l2(got[t], want[t]) <= BAR, (t, seq[t], pos[t])
