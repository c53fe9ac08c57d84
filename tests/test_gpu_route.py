"""Routing of many tokens against the formula in 64 bits."""
import numpy as np
import pytest
import torch

from tests.gpu_util import case, dev, host

pytestmark = pytest.mark.gpu


def reference(z, k, sigmoid=False, bias=None, groups=1, top_groups=1, best=1, renorm=True, scale=1.0):
    """(ids, weights, bound of the weights' error)."""
    T, E = z.shape
    z64 = z.astype(np.float64)
    idx, w = np.full((T, k), -1, np.int32), np.zeros((T, k))
    bound = np.zeros((T, 1))
    with np.errstate(all="ignore"):
        m = z64.max(1, keepdims=True)
        e = np.exp(z64 - m)
        p = 1 / (1 + np.exp(-z64)) if sigmoid else e / e.sum(1, keepdims=True)
        c = p if bias is None else p + bias.astype(np.float64)
        if not sigmoid:  # the sum of fp32 exponentials: 2^-23 of each, and the argument's rounding, 2^-24 of it
            d = np.where(np.isfinite(z64 - m), np.abs(z64 - m), 0.0)
            bound = 2.0 ** -22 + 2.0 ** -24 * (np.where(p > 0, p, 0.0) * d).sum(1, keepdims=True)
    for t in range(T):
        out = (z[t] == -np.inf) | ((bias == -np.inf) if bias is not None else False)
        if np.isnan(c[t][~(z[t] == -np.inf)]).any() or (not sigmoid and (z[t] == np.inf).any()):
            w[t] = np.nan
            continue
        ct = np.where(out, -np.inf, c[t])
        order = z64[t] if bias is None and (best == 1 or top_groups == groups) else ct
        order = np.where(out, -np.inf, order)
        score = []
        for g in order.reshape(groups, -1):
            g = np.sort(g)[::-1]
            score.append(g[0] + g[1] if best == 2 and len(g) > 1 and g[1] > -np.inf else g[0])
        kept = np.argsort(-np.array(score), kind="stable")[:top_groups]
        on = np.isin(np.arange(E) // (E // groups), kept)
        order = np.where(on, order, -np.inf)
        at = [i for i in np.argsort(-order, kind="stable")[:k] if order[i] > -np.inf]
        idx[t, :len(at)], w[t, :len(at)] = at, p[t, at]
        if renorm and w[t].sum() > 0:
            w[t] /= w[t].sum()
    return idx, w * scale, (bound + 2.0 ** -23) * np.abs(w * scale) + 1e-38


def run(gpu, z, k, sigmoid=False, bias=None, groups=1, top_groups=1, best=1, renorm=True, scale=1.0):
    T = z.shape[0]
    z = dev(z) if isinstance(z, np.ndarray) else z
    idx = torch.full((T + 1, k), 77, dtype=torch.int32, device="cuda")  # one row behind the last
    w = torch.full((T + 1, k), 77.0, device="cuda")
    gpu.ops.moe_route(z, idx[:T], w[:T], sigmoid, None if bias is None else dev(bias), groups, top_groups, best, renorm, scale)
    i, w = host(idx), host(w)
    assert (i[T] == 77).all() and (w[T] == 77).all()
    return i[:T], w[:T]


def check(got, want):
    assert np.array_equal(got[0], want[0])
    none = np.isnan(want[1])
    assert np.array_equal(np.isnan(got[1]), none)
    assert (np.abs(got[1] - want[1]) <= want[2])[~none].all()


@pytest.mark.parametrize("T,E,k,sigmoid,bias,groups,top_groups,best,renorm", [
    (1, 1, 1, False, False, 1, 1, 1, True), (1, 128, 8, False, False, 1, 1, 1, True), (3, 128, 8, False, False, 1, 1, 1, False),
    (37, 60, 4, False, False, 1, 1, 1, False), (5, 7, 7, True, True, 1, 1, 1, True), (33, 256, 8, True, True, 8, 4, 2, True),
    (33, 256, 8, True, False, 8, 4, 2, False), (9, 160, 6, False, False, 8, 3, 1, False), (9, 160, 6, False, True, 8, 3, 1, True),
    (5, 1024, 16, False, False, 1, 1, 1, True), (5, 1024, 16, True, True, 64, 10, 2, True), (4, 1023, 9, True, True, 33, 5, 2, True),
    (4, 1020, 9, False, True, 17, 5, 2, False), (6, 64, 2, True, True, 64, 2, 2, True), (11, 51, 5, True, False, 17, 3, 1, True),
    (2048, 128, 8, False, False, 1, 1, 1, True), (2051, 256, 8, True, True, 8, 4, 2, True), (2049, 512, 16, True, True, 16, 1, 1, True),
    (2050, 510, 3, False, True, 1, 1, 1, False), (2053, 174, 15, True, True, 2, 1, 1, True), (2048, 520, 5, True, False, 4, 2, 2, True),
    (2055, 9, 3, False, False, 3, 2, 2, True), (16391, 256, 8, True, True, 8, 4, 2, True), (2060, 1024, 7, True, True, 1, 1, 1, True),
    (2061, 768, 4, False, True, 24, 3, 2, True), (16385, 340, 5, True, True, 17, 4, 2, False), (16384, 40, 6, False, False, 1, 1, 1, False)])
def test_against_the_formula(gpu, T, E, k, sigmoid, bias, groups, top_groups, best, renorm):
    rng = np.random.default_rng(T + E)
    z = (2 * rng.standard_normal((T, E))).astype(np.float32)
    b = (0.1 * rng.standard_normal(E)).astype(np.float32) if bias else None
    a = (k, sigmoid, b, groups, top_groups, best, renorm, 2.5)
    case(f"route T={T} E={E} k={k} sigmoid={sigmoid} bias={bias} groups={groups}/{top_groups} best={best} renorm={renorm}")
    check(run(gpu, z, *a), reference(z, *a))


@pytest.mark.parametrize("T", [6, 2100])
@pytest.mark.parametrize("sigmoid,bias,best", [(False, False, 1), (True, True, 2), (False, True, 2)])
def test_ties_go_to_the_lower_index(gpu, T, sigmoid, bias, best):
    """Logits of three values; groups tie as well."""
    rng = np.random.default_rng(T)
    z = rng.integers(-1, 2, (T, 96)).astype(np.float32)
    z[0] = 0.0
    z[1, ::2] = -0.0
    z[1, 1::2] = 0.0
    b = np.full(96, 0.25, np.float32) if bias else None
    a = (9, sigmoid, b, 6, 3, best, True, 1.0)
    case(f"route ties T={T} sigmoid={sigmoid} bias={bias}")
    got = run(gpu, z, *a)
    check(got, reference(z, *a))
    assert got[0][0].tolist() == list(range(9)) and got[0][1].tolist() == list(range(9))


@pytest.mark.parametrize("T", [9, 2100])
@pytest.mark.parametrize("sigmoid,bias", [(False, False), (True, True), (False, True), (True, False)])
def test_scores_that_are_none(gpu, T, sigmoid, bias):
    """Masked experts, rows that they fill, NaN and infinities; the rows beside them are untouched."""
    rng = np.random.default_rng(T + 1)
    z = rng.standard_normal((T, 40)).astype(np.float32)
    z[0] = -np.inf
    z[1, 3:] = -np.inf
    z[2, 7] = np.nan
    z[3, 8] = np.inf
    z[5, :20] = -np.inf  # a whole group
    z[6] = -200.0  # scores of 1e-87
    z[7] = 3e38
    b = (0.1 * rng.standard_normal(40)).astype(np.float32) if bias else None
    if bias:
        b[11] = -np.inf
    a = (6, sigmoid, b, 2, 2, 1, True, 1.5)
    case(f"route none T={T} sigmoid={sigmoid} bias={bias}")
    check(run(gpu, z, *a), reference(z, *a))
    a = (6, sigmoid, b, 4, 1, 2, False, 1.0)
    check(run(gpu, z, *a), reference(z, *a))


def test_a_bias_that_is_none(gpu):
    z = np.random.default_rng(3).standard_normal((3, 16)).astype(np.float32)
    b = np.zeros(16, np.float32)
    b[4] = np.nan
    case("route NaN bias")
    i, w = run(gpu, z, 2, True, b)
    assert (i == -1).all() and np.isnan(w).all()


def test_near_ties_are_told_apart(gpu):
    """Scores whose difference fp32 does not hold: sigmoids of logits near 12 with the bias that makes them equal but
    for 2^-30."""
    z = np.full((2, 8), -5.0, np.float32)
    z[:, 2], z[:, 5] = 12.0, 12.0 + 2.0 ** -12
    case("route near ties")
    i, _ = run(gpu, z, 2, True, np.zeros(8, np.float32))
    assert i.tolist() == [[5, 2], [5, 2]]


def test_unaligned_rows(gpu):
    rng = np.random.default_rng(5)
    z = rng.standard_normal((2100, 64)).astype(np.float32)
    buf = torch.empty(2100 * 64 + 1, device="cuda")[1:].view(2100, 64)
    buf.copy_(dev(z))
    case("route unaligned")
    check(run(gpu, buf, 4, True), reference(z, 4, True))


def test_in_a_graph_on_two_streams(gpu):
    """Captured once, replayed with other logits, next to eager calls on another stream."""
    rng = np.random.default_rng(6)
    T, E, k = 300, 256, 8
    bias = (0.1 * rng.standard_normal(E)).astype(np.float32)
    z, idx, w = torch.empty((T, E), device="cuda"), torch.empty((T, k), dtype=torch.int32, device="cuda"), torch.empty((T, k), device="cuda")
    b = dev(bias)
    z.zero_()
    side = torch.cuda.Stream()
    case("route graph")
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            gpu.ops.moe_route(z, idx, w, True, b, 8, 4, 2)
    for _ in range(3):
        x = rng.standard_normal((T, E)).astype(np.float32)
        z.copy_(dev(x))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        got = run(gpu, x, k, True, bias, 8, 4, 2)
        torch.cuda.synchronize()
        assert np.array_equal(host(idx), got[0]) and np.array_equal(host(w), got[1])
        check(got, reference(x, k, True, bias, 8, 4, 2))
