"""Page upkeep against a plain model of the state in Python (whole numbers and copied bytes: exact)."""
import numpy as np
import pytest
import torch

from tests.gpu_util import case, dev, host

pytestmark = pytest.mark.gpu


class Model:
    """The state as the entry points define it, one row and page at a time."""

    def __init__(self, rows, width, n_pages, ps, layers=2, nkv=2, hd=64, int8=False, seed=0):
        rng = np.random.default_rng(seed)
        self.ps, self.n = ps, n_pages
        self.table = np.full((rows, width), -1, np.int32)
        self.lens = np.zeros(rows, np.int32)
        self.refs = np.zeros(n_pages, np.int32)
        shape = (layers, n_pages, nkv)
        if int8:
            self.arr = [rng.integers(-128, 128, (*shape, ps, hd)).astype(np.int8),
                        rng.integers(-128, 128, (*shape, hd, ps)).astype(np.int8),
                        rng.standard_normal((*shape, ps)).astype(np.float32),
                        rng.standard_normal((*shape, ps)).astype(np.float32)]
        else:
            self.arr = [rng.standard_normal((*shape, ps, hd)).astype(np.float16),
                        rng.standard_normal((*shape, hd, ps)).astype(np.float16)]

    def pages(self, n):
        return -(-int(n) // self.ps)

    def free_pages(self):
        return [p for p in range(self.n) if self.refs[p] == 0]

    def extend(self, to):
        free, need_so_far, refused = self.free_pages(), 0, 0
        for r in range(len(self.lens)):
            if to[r] <= self.lens[r]:
                continue
            have, want = self.pages(self.lens[r]), self.pages(to[r])
            if want > self.table.shape[1]:
                refused += 1
                continue
            at, need_so_far = need_so_far, need_so_far + want - have
            if need_so_far > len(free):
                refused += 1
                continue
            for i, p in enumerate(free[at:need_so_far]):
                self.table[r, have + i] = p
                self.refs[p] = 1
            self.lens[r] = to[r]
        return refused

    def free(self, gone):
        for r in np.flatnonzero(gone):
            for p in self.table[r, :self.pages(self.lens[r])]:
                self.refs[p] -= 1
            self.table[r] = -1
            self.lens[r] = 0

    def fork(self, parents):
        before, table = self.lens.copy(), self.table.copy()
        free, need, refused = self.free_pages(), 0, 0
        for r, p in enumerate(parents):
            if p < 0:
                continue
            if p >= len(before) or before[r] > 0 or before[p] == 0:
                refused += 1
                continue
            part = before[p] % self.ps > 0
            need += part
            if need > len(free):
                refused += 1
                continue
            held = self.pages(before[p])
            self.table[r] = -1
            self.table[r, :held] = table[p, :held]
            if part:
                new, old = free[need - 1], table[p, held - 1]
                self.table[r, held - 1] = new
                for a in self.arr:
                    a[:, new] = a[:, old]
            for q in self.table[r, :held]:
                self.refs[q] += 1
            self.lens[r] = before[p]
        return refused

    def compact(self):
        used = [p for p in range(self.n) if self.refs[p] > 0]
        n = len(used)
        moves = dict(zip([p for p in used if p >= n], [p for p in range(n) if self.refs[p] == 0]))
        for a, b in moves.items():
            for x in self.arr:
                x[:, b] = x[:, a]
            self.refs[b], self.refs[a] = self.refs[a], 0
        for i, p in np.ndenumerate(self.table):
            self.table[i] = moves.get(int(p), p)
        return n


class Device:
    def __init__(self, gpu, m):
        self.o, self.ps = gpu.ops, m.ps
        self.table, self.lens, self.refs = dev(m.table), dev(m.lens), dev(m.refs)
        self.arr = [dev(a) for a in m.arr]
        self.scales = dict(ks=self.arr[2], vs=self.arr[3]) if len(self.arr) == 4 else {}
        n = self.o.kv_pages_workspace_bytes(len(m.lens), m.n)
        self.ws = torch.full((n + 64,), 0xA5, dtype=torch.uint8, device="cuda")  # nothing relies on what it holds
        self.st = torch.full((2,), -77, dtype=torch.int32, device="cuda")

    def state(self):
        return self.table, self.lens, self.refs

    def extend(self, to):
        self.o.kv_pages_extend(*self.state(), dev(to), self.ps, self.st)
        return int(host(self.st)[0])

    def free(self, gone):
        self.o.kv_pages_free(*self.state(), dev(gone), self.ps)

    def fork(self, parents):
        self.o.kv_pages_fork(*self.state(), dev(parents), *self.arr[:2], self.st, self.ws, **self.scales)
        return int(host(self.st)[0])

    def compact(self):
        self.o.kv_pages_compact(self.table, self.refs, *self.arr[:2], self.st, self.ws, **self.scales)
        return int(host(self.st)[0])


def same(d, m, what):
    for name in ("table", "lens", "refs"):
        assert np.array_equal(host(getattr(d, name)), getattr(m, name)), (what, name)
    for i, (a, b) in enumerate(zip(d.arr, m.arr)):
        assert np.array_equal(host(a).view(np.uint8), b.view(np.uint8)), (what, i)
    assert host(d.st)[1] == -77
    assert (host(d.ws)[-64:] == 0xA5).all()


def i32(x):
    return np.asarray(x, np.int32)


@pytest.mark.parametrize("ps,rows,width,n_pages,int8", [(16, 7, 9, 30, False), (32, 40, 6, 100, True),
                                                        (64, 1, 4, 5, False), (128, 13, 3, 20, True)])
def test_random_upkeep(gpu, ps, rows, width, n_pages, int8):
    """Forty random calls in a row: lengths that grow, repeat, shrink (ignored) and pass the table, pools that run
    out, forks of forks, of empty rows, of rows out of range and onto live rows, rows freed twice."""
    rng = np.random.default_rng(ps + rows)
    m = Model(rows, width, n_pages, ps, int8=int8, seed=rows)
    d = Device(gpu, m)
    for step in range(40):
        kind = rng.choice(["extend", "extend", "free", "fork", "fork", "compact"])
        case(f"kv pages ps={ps} rows={rows} step {step}: {kind}")
        if kind == "extend":
            to = i32(rng.integers(-3, int(width * ps * 1.1), rows) * (rng.random(rows) < 0.4))
            a = (d.extend(to), m.extend(to))
        elif kind == "fork":
            parents = i32(np.where(rng.random(rows) < 0.5, rng.integers(-2, rows + 2, rows), -1))
            a = (d.fork(parents), m.fork(parents))
        elif kind == "free":
            gone = i32((rng.random(rows) < 0.4) * rng.integers(-2, 3, rows))
            a = (d.free(gone), m.free(gone))
        else:
            a = (d.compact(), m.compact())
        assert a[0] == a[1], (step, kind)
        same(d, m, (step, kind))


@pytest.mark.parametrize("rows,width,n_pages", [(4096, 4, 20011), (1025, 9, 8193), (3, 5000, 16400)])
def test_large_tables(gpu, rows, width, n_pages):
    rng = np.random.default_rng(rows)
    m = Model(rows, width, n_pages, 16, layers=1, nkv=1)
    d = Device(gpu, m)
    case(f"kv pages rows={rows} width={width} n_pages={n_pages}")
    to = i32(rng.integers(0, width * 16 + 1, rows))
    for step in range(3):
        assert d.extend(to) == m.extend(to)
        same(d, m, ("extend", step))
        gone = i32(rng.random(rows) < 0.5)
        d.free(gone), m.free(gone)
        same(d, m, ("free", step))
        parents = i32(np.where(gone, rng.integers(0, rows, rows), -1))
        assert d.fork(parents) == m.fork(parents)
        same(d, m, ("fork", step))
        gone = i32(rng.random(rows) < 0.3)
        d.free(gone), m.free(gone)
        assert d.compact() == m.compact()
        same(d, m, ("compact", step))
        to = i32(rng.integers(0, width * 16 + 1, rows))


def test_forks_share_until_the_last_is_freed(gpu):
    m = Model(6, 4, 16, 16)
    d = Device(gpu, m)
    case("kv pages, shared pages")
    for to in ([40, 32, 0, 0, 0, 0],):
        assert d.extend(i32(to)) == m.extend(to) == 0
    parents = i32([-1, -1, 0, 0, 1, 1])
    assert d.fork(parents) == m.fork(parents) == 0
    assert list(m.refs[:8]) == [3, 3, 1, 3, 3, 1, 1, 0]  # two full pages each, three and one tail pages
    same(d, m, "fork")
    for gone in ([1, 0, 0, 0, 0, 0], [0, 1, 0, 0, 1, 0], [0, 0, 1, 1, 0, 1]):
        d.free(i32(gone)), m.free(gone)
        same(d, m, gone)
    assert not m.refs.any()


def test_copy(gpu):
    m = Model(1, 1, 50, 32, layers=3, nkv=3, hd=128, int8=True)
    d = Device(gpu, m)
    src, dst = i32([3, 3, 49, 0, 7, -1, 5, 50, 9]), i32([10, 11, 12, 48, 7, 13, 50, 14, -2])
    case("kv pages copy")
    gpu.ops.kv_pages_copy(dev(src), dev(dst), *d.arr[:2], **d.scales)
    for a in m.arr:
        for s, t in zip(src, dst):
            if 0 <= s < 50 and 0 <= t < 50:
                a[:, t] = a[:, s]
    same(d, m, "copy")
    gpu.ops.kv_pages_copy(dev(src)[:0], dev(dst)[:0], *d.arr[:2], **d.scales)
    same(d, m, "nothing")


def test_copies_past_4_gib(gpu):
    """Pages whose byte offset within a layer passes 32 bits."""
    k = torch.zeros((1, 12500, 8, 128, 256), dtype=torch.float16, device="cuda")
    v = torch.zeros((1, 12500, 8, 256, 128), dtype=torch.float16, device="cuda")
    k[0, 2], v[0, 2] = 1.5, 2.5
    case("kv pages copy past 4 GiB")
    gpu.ops.kv_pages_copy(dev(i32([2])), dev(i32([12499])), k, v)
    for t, x in ((k, 1.5), (v, 2.5)):
        at = torch.nonzero(t[0].flatten(1).amax(1)).flatten().tolist()
        assert at == [2, 12499] and (t[0, 12499] == x).all()


def test_upkeep_in_a_graph(gpu):
    """A captured fork + compact, replayed from restored states, against the model."""
    m = Model(8, 5, 40, 16, seed=3)
    d = Device(gpu, m)
    parents, to, gone = i32([-1, -1, 0, 1, 0, -1, -1, 1]), i32([50, 33, 0, 0, 0, 20, 70, 0]), i32([0, 0, 0, 0, 0, 1, 0, 0])
    pd, td, gd = dev(parents), dev(to), dev(gone)
    start = [t.clone() for t in (*d.state(), *d.arr)]

    def step():
        d.o.kv_pages_extend(*d.state(), td, d.ps, d.st)
        d.o.kv_pages_free(*d.state(), gd, d.ps)
        d.o.kv_pages_fork(*d.state(), pd, *d.arr[:2], d.st, d.ws)
        d.o.kv_pages_compact(d.table, d.refs, *d.arr[:2], None, d.ws)

    def restore():
        for t, x in zip((*d.state(), *d.arr), start):
            t.copy_(x)

    case("kv pages graph capture")
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
    m.extend(to), m.free(gone), m.fork(parents), m.compact()
    for _ in range(3):
        restore()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        same(d, m, "replay")
        restore()
        step()
        same(d, m, "eager")



@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("graph", [False, True])
def test_step_of_a_pool_that_runs_out(gpu, int8, graph):
    """Extend and prep as a server's step calls them, the tokens named by their positions (-1: a row that takes none) and
    the lengths: a row that could not be extended, its sibling on the same full pages and a paused row keep their pages
    bit for bit."""
    ps, nkv, hd, S = 16, 2, 64, 6
    m = Model(S, 4, 9, ps, layers=1, nkv=nkv, hd=hd, int8=int8, seed=5)
    d = Device(gpu, m)
    # row 0: two full pages, row 1 its fork; rows 2 (paused), 3 and 5 partly filled; row 4 empty
    for call, arg in (("extend", [32, 0, 20, 21, 0, 3]), ("fork", [-1, 0, -1, -1, -1, -1])):
        assert getattr(d, call)(i32(arg)) == getattr(m, call)(i32(arg)) == 0
    same(d, m, "begin")
    assert len(m.free_pages()) == 2 and m.table[0, 1] == m.table[1, 1]
    rng = np.random.default_rng(1)
    new, pos, seq = dev(np.zeros(S, np.int32)), dev(np.zeros(S, np.int32)), dev(np.arange(S, dtype=np.int32))
    active = dev(i32([1, 1, 0, 1, 0, 1]))
    q = dev(rng.standard_normal((S, 4, hd)).astype(np.float32))
    k, v = (dev(rng.standard_normal((S, nkv, hd)).astype(np.float32)) for _ in range(2))
    q_out = torch.zeros_like(q)

    def step():
        torch.add(d.lens, active, out=new)
        torch.mul(new, active, out=pos)
        pos.sub_(1)
        d.o.kv_pages_extend(*d.state(), new, ps, d.st)
        d.o.paged_attn_prep(q, k, v, None, None, 1e-6, 1e4, d.arr[0][0], d.arr[1][0], d.table, q_out, pos, seq,
                            d.arr[2][0] if int8 else None, d.arr[3][0] if int8 else None, seq_lens=d.lens)

    case(f"a step of a pool that runs out int8={int8} graph={graph}")
    run = step
    if graph:
        start = [t.clone() for t in (*d.state(), *d.arr)]
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            step()
            side.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                step()
        for t, x in zip((*d.state(), *d.arr), start):
            t.copy_(x)
        torch.cuda.synchronize()
        run = g.replay
    on = np.array([1, 1, 0, 1, 0, 1])
    refused = []
    for i in range(14):  # rows 0 and 1 take the two pages that are left; row 3 is stopped at its page's end, with it row 5
        before, old = [host(a).copy() for a in d.arr], m.lens.copy()
        n = m.extend(i32(m.lens + on))
        run()
        torch.cuda.synchronize()
        assert int(host(d.st)[0]) == n
        assert np.array_equal(host(d.lens), m.lens) and np.array_equal(host(d.table), m.table) and np.array_equal(host(d.refs), m.refs)
        wrote = {(int(m.table[r, (m.lens[r] - 1) // ps]), int((m.lens[r] - 1) % ps)) for r in range(S) if m.lens[r] > old[r]}
        refused.append(n)
        for t, (a, b) in enumerate(zip(d.arr, before)):
            x = host(a)[0] != b[0]
            x = x.any(1) if t > 1 else x.any((1, 2)) if t == 1 else x.any((1, 3))  # [page][position]
            assert {(int(p), int(o)) for p, o in np.argwhere(x)} <= wrote, (i, t)
            if t < 2:
                assert {(int(p), int(o)) for p, o in np.argwhere(x)} == wrote, (i, t)
    assert refused[0] == 0 and max(refused) == 2
