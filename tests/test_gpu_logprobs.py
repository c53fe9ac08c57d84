"""Log probabilities, ranks, entropies and alternatives against the formula in 64 bits.

Bounds, with u = 2^-24 and d = z - max: an exponential is off by 2u, and by 2u|d| for its argument; a thread adds at most
vocab / 256 + 16 of them one after the other, and a step in which the maximum rises costs two roundings more.  So S is off by
e = (2 + 2 E|d| + n) u relative, n = vocab / 128 + 48, with E|d| = sum p|d|, and log S by as much.  What is returned is
rounded once more.  T adds the same, of terms p d that round once more: T / S is off by (2 + n) u E|d| + 2u E d^2 + e E|d|."""
import numpy as np
import pytest
import torch

from tests.gpu_util import case, dev, host

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def reference(z, t, k):
    n, V = z.shape
    r = {"logp": np.zeros(n), "rank": np.zeros(n, np.int32), "ent": np.zeros(n), "ids": np.full((n, k), -1, np.int32),
         "tops": np.full((n, k), -np.inf), "e": np.zeros(n), "e_ent": np.zeros(n)}
    for i in range(n):
        x = z[i].astype(np.float64)
        in_range = 0 <= t[i] < V
        if np.isnan(x).any() or (x == np.inf).any():
            r["logp"][i] = np.nan if in_range else 0.0
            r["ent"][i], r["tops"][i] = np.nan, np.nan
            continue
        if in_range:
            r["rank"][i] = 1 + (x > x[t[i]]).sum() + (x[:t[i]] == x[t[i]]).sum()
        m = x.max()
        if m == -np.inf:
            r["logp"][i] = -np.inf if in_range else 0.0
            continue
        d = x - m
        p = np.exp(d)
        S = p.sum()
        y = d - np.log(S)
        p /= S
        w = np.where(p > 0, np.abs(np.where(p > 0, d, 0)), 0)
        Ed, Ed2 = (p * w).sum(), (p * w * w).sum()
        steps = V / 128 + 48
        r["e"][i] = (2 + 2 * Ed + steps) * U
        r["e_ent"][i] = r["e"][i] * (1 + Ed) + (2 + steps) * U * Ed + 2 * U * Ed2
        if in_range:
            r["logp"][i] = y[t[i]]
        r["ent"][i] = -(p * np.where(p > 0, y, 0)).sum()
        order = np.lexsort((np.arange(V), -x))[:k]
        order = order[x[order] > -np.inf]
        r["ids"][i, :len(order)], r["tops"][i, :len(order)] = order, y[order]
    return r


def run(gpu, z, t, k, off=0):
    n, V = z.shape
    zd = torch.empty(n * V + off, device="cuda")[off:].view(n, V)
    zd.copy_(dev(z))
    f = lambda *s: torch.full(s, 77.0, device="cuda")  # noqa: E731
    i = lambda *s: torch.full(s, 77, dtype=torch.int32, device="cuda")  # noqa: E731
    logp, rank, ent, ids, tops = f(n + 1), i(n + 1), f(n + 1), i(n + 1, k), f(n + 1, k)
    ws = torch.full((gpu.ops.logprobs_workspace_bytes(n, V, k),), 255, dtype=torch.uint8, device="cuda")
    gpu.ops.logprobs(zd, dev(t), logp[:n], rank[:n], ent[:n], ids[:n] if k else None, tops[:n] if k else None, ws)
    got = {"logp": host(logp), "rank": host(rank), "ent": host(ent), "ids": host(ids), "tops": host(tops)}
    for x in got.values():
        assert (x[n] == 77).all()
    return {name: x[:n] for name, x in got.items()}


def near(got, want, bound):
    fine = np.isfinite(want)
    assert np.array_equal(got[~fine], want[~fine].astype(np.float32), equal_nan=True)
    assert (np.abs(got[fine] - want[fine]) <= bound[fine] + U * np.abs(want[fine])).all()


def check(got, want):
    for name in ("rank", "ids"):
        assert np.array_equal(got[name], want[name]), name
    near(got["logp"], want["logp"], want["e"])
    near(got["tops"], want["tops"], np.repeat(want["e"][:, None], want["tops"].shape[1], 1))
    near(got["ent"], want["ent"], want["e_ent"])


def inputs(seed, n, V, masked=0.0):
    rng = np.random.default_rng(seed)
    z = (3 * rng.standard_normal((n, V))).astype(np.float32)
    if masked:
        z[rng.random((n, V)) < masked] = -np.inf
    t = rng.integers(0, V, n).astype(np.int32)
    t[::3] = z[::3].argmax(1)
    return z, t


@pytest.mark.parametrize("n,V,k,masked", [
    (1, 1, 1, 0), (2, 2, 5, 0), (3, 63, 64, 0), (4, 100, 7, 0.9), (1, 151936, 20, 0), (2, 151937, 64, 0), (31, 32003, 5, 0.7), (5, 4096, 1, 0),
    (5, 4097, 33, 0), (7, 8191, 0, 0), (1100, 5000, 3, 0), (600, 40001, 10, 0.2), (1030, 4099, 0, 0), (2000, 130, 16, 0.5),
    (1, 600000, 12, 0), (70, 70000, 2, 0)])
def test_against_the_formula(gpu, n, V, k, masked):
    z, t = inputs(n + V, n, V, masked)
    case(f"logprobs n={n} V={V} k={k} masked={masked}")
    check(run(gpu, z, t, k), reference(z, t, k))


@pytest.mark.parametrize("n", [3, 1500])
def test_ties_go_to_the_lower_id(gpu, n):
    """Logits of a few values, all equal ones, rising and falling rows."""
    rng = np.random.default_rng(n)
    V = 9001
    z = rng.integers(0, 40, (n, V)).astype(np.float32)
    z[0] = 1.5
    z[1] = np.arange(V)
    z[2] = -np.arange(V)
    z[2, 4000:] = 0.0
    z[2, 5000:6000] = -0.0
    t = rng.integers(0, V, n).astype(np.int32)
    case(f"logprobs ties n={n}")
    check(run(gpu, z, t, 40), reference(z, t, 40))


@pytest.mark.parametrize("n,V", [(10, 3000), (10, 40000), (1200, 5001)])
def test_rows_that_are_no_distribution(gpu, n, V):
    """Rows of -inf, rows with a NaN or +inf, one number alone, the type's largest and lowest values; targets
    outside the vocabulary."""
    z, t = inputs(n, n, V)
    z[0] = -np.inf
    z[1, 77] = np.nan
    z[2, 1234] = np.inf
    z[3] = -np.inf
    z[3, 2999] = -5.0
    z[4] = np.finfo(np.float32).min
    z[5, ::2] = np.finfo(np.float32).max
    z[6, :2000] = np.finfo(np.float32).min
    z[7, 5] = np.nan
    z[7, 9] = np.inf
    t[3] = 2999
    t[6], t[7], t[8], t[9] = -1, V, 2 ** 31 - 1, -2 ** 31
    case(f"logprobs none n={n} V={V}")
    want = reference(z, t, 12)
    check(run(gpu, z, t, 12), want)
    assert want["rank"][0] == t[0] + 1 and want["ids"][3].tolist() == [2999] + [-1] * 11


def test_certain_rows(gpu):
    """A logit far above the rest: the entropy is small, and never below zero by more than a rounding."""
    z, t = inputs(4, 6, 50000)
    z[:, 40000] = [20.0, 30.0, 50.0, 100.0, 1e4, 1e30]
    t[:] = 40000
    case("logprobs certain")
    got = run(gpu, z, t, 3)
    check(got, reference(z, t, 3))
    assert (got["ids"][:, 0] == 40000).all() and (got["rank"] == 1).all()


@pytest.mark.parametrize("off", [1, 2, 3])
def test_unaligned_rows(gpu, off):
    z, t = inputs(off, 9, 9002 + off)
    case(f"logprobs unaligned {off}")
    check(run(gpu, z, t, 6, off), reference(z, t, 6))


def test_parts_of_the_answer(gpu):
    """Each of the three on its own gives what all together give."""
    z, t = inputs(12, 5, 20000)
    all_ = run(gpu, z, t, 6)
    zd, td = dev(z), dev(t)
    ws = torch.empty(gpu.ops.logprobs_workspace_bytes(5, 20000, 6), dtype=torch.uint8, device="cuda")
    f = lambda *s: torch.full(s, 5.0, device="cuda")  # noqa: E731
    logp, ent, tops, ids = f(5), f(5), f(5, 6), torch.zeros((5, 6), dtype=torch.int32, device="cuda")
    case("logprobs parts")
    gpu.ops.logprobs(zd, td, logp, None, None, None, None, ws)
    gpu.ops.logprobs(zd, None, None, None, ent, None, None, ws)
    gpu.ops.logprobs(zd, None, None, None, None, ids, tops, ws)
    for got, name in ((logp, "logp"), (ent, "ent"), (ids, "ids"), (tops, "tops")):
        assert np.array_equal(host(got), all_[name]), name


def test_in_a_graph(gpu):
    """Captured with the logits' processing before it, replayed with other logits."""
    n, V, k = 3, 32003, 8
    z, mask = torch.zeros((n, V), device="cuda"), torch.zeros((n, -(-V // 32)), dtype=torch.int32, device="cuda")
    t = torch.zeros(n, dtype=torch.int32, device="cuda")
    logp, rank, ent = torch.zeros(n, device="cuda"), torch.zeros(n, dtype=torch.int32, device="cuda"), torch.zeros(n, device="cuda")
    ids, tops = torch.zeros((n, k), dtype=torch.int32, device="cuda"), torch.zeros((n, k), device="cuda")
    ws = torch.empty(gpu.ops.logprobs_workspace_bytes(n, V, k), dtype=torch.uint8, device="cuda")
    out = torch.empty_like(z)

    def step():
        gpu.ops.logits_process(z, out, allowed=mask)
        gpu.ops.logprobs(out, t, logp, rank, ent, ids, tops, ws)

    side = torch.cuda.Stream()
    case("logprobs graph")
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
    for i in range(4):
        x, ti = inputs(40 + i, n, V)
        bits = np.random.default_rng(i).integers(-2 ** 31, 2 ** 31, (n, -(-V // 32))).astype(np.int32)
        z.copy_(dev(x))
        t.copy_(dev(ti))
        mask.copy_(dev(bits))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        torch.cuda.synchronize()
        on = ((bits.astype(np.int64)[:, :, None] >> np.arange(32)) & 1).reshape(n, -1)[:, :V]
        x[on == 0] = -np.inf
        got = {"logp": host(logp), "rank": host(rank), "ent": host(ent), "ids": host(ids), "tops": host(tops)}
        got = {a: b.copy() for a, b in got.items()}
        check(got, reference(x, ti, k))
        step()
        for a, b in (("logp", logp), ("rank", rank), ("ent", ent), ("ids", ids), ("tops", tops)):
            assert np.array_equal(host(b), got[a])
