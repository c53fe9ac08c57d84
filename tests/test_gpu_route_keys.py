"""Routing of many tokens where scores of both signs are chosen, against the formula in 64 bits.

Logits are whole numbers or eighths, and biases eighths where they alone decide, so that two scores are equal or far apart:
the order has no rounding in it.
A weight is a quotient in 64 bits rounded to fp32 once: off by 2^-24 of it, and by 2^-150 where it has no normal number;
the bound is twice that."""
import numpy as np
import pytest
import torch

from tests.gpu_util import case, dev, host

pytestmark = pytest.mark.gpu


def reference(z, k, sigmoid=False, bias=None, groups=1, top_groups=1, best=1):
    """(ids, renormalised weights).  Without a bias the order is that of the logits, but with groups that are left out by
    the sum of two experts that of the scores."""
    T, E = z.shape
    z64 = z.astype(np.float64)
    with np.errstate(over="ignore", invalid="ignore"):  # (a row without experts has no scores)
        p = 1 / (1 + np.exp(-z64)) if sigmoid else np.exp(z64 - z64.max(1, keepdims=True))
        if not sigmoid:
            p /= p.sum(1, keepdims=True)
    if bias is not None:
        c = p + bias.astype(np.float64)
    else:
        c = p.copy() if best == 2 and top_groups < groups < E else z64.copy()
    c[z64 == -np.inf] = -np.inf
    if bias is not None:
        c[:, bias == -np.inf] = -np.inf
    if top_groups < groups:
        by = -np.sort(-c.reshape(T, groups, -1), axis=2)[:, :, :best]
        score = np.where((by == -np.inf).any(2), -np.inf, by.sum(2, where=by > -np.inf))  # (an infinite bias and a masked one)
        place = np.empty((T, groups), int)
        np.put_along_axis(place, np.argsort(-score, axis=1, kind="stable"), np.arange(groups)[None], 1)
        c = np.where(np.repeat(place < top_groups, E // groups, axis=1), c, -np.inf)
    idx = np.argsort(-c, axis=1, kind="stable")[:, :k].astype(np.int32)
    there = np.take_along_axis(c, idx, 1) > -np.inf
    w = np.where(there, np.take_along_axis(p, idx, 1), 0.0)
    total = w.sum(1, keepdims=True)
    return np.where(there, idx, -1), np.divide(w, total, out=np.zeros_like(w), where=total > 0)


def check(gpu, z, k, **how):
    T = z.shape[0]
    idx, w = torch.empty((T, k), dtype=torch.int32, device="cuda"), torch.empty((T, k), device="cuda")
    bias = how.get("bias")
    gpu.ops.moe_route(dev(z), idx, w, how.get("sigmoid", False), None if bias is None else dev(bias), how.get("groups", 1),
                      how.get("top_groups", 1), how.get("best", 1))
    want, weights = reference(z, k, **how)
    got = host(idx)
    wrong = np.flatnonzero((got != want).any(1))
    assert wrong.size == 0, f"{wrong.size} of {T} tokens, the first: {got[wrong[0]]} for {want[wrong[0]]}"
    assert (np.abs(host(w) - weights) <= 2.0 ** -23 * weights + 2.0 ** -149).all()


def live(rng, T, E):
    """Some 20 experts a row: ten with, where there are such, the one whose index has the complement of their bits, and others."""
    on = rng.random((T, E)) < 6 / E
    e = rng.integers(max(0, min(1023 - (E - 1), E - 1)), E, (T, 10))
    np.put_along_axis(on, e, True, 1)
    np.put_along_axis(on, np.clip(1023 - e, 0, E - 1), True, 1)
    return on


SIZES = [(T, E) for T in (7, 2050, 16387) for E in (512, 513, 520, 768, 1023, 1024)]


@pytest.mark.parametrize("T,E", SIZES)
def test_a_choice_leaves_the_others(gpu, T, E):
    """The best expert of a row, e, is above 0, the second, 1023 - e, below 0: their indices' bits are each other's complement."""
    rng = np.random.default_rng(T + E)
    z = np.full((T, E), -10.0, np.float32)
    lo = max(0, 1023 - (E - 1))
    for t in range(T):
        e = int(rng.integers(min(lo, E - 1), E))
        z[t, (e * 3 + 1) % E] = -2.0
        z[t, min(max(1023 - e, 0), E - 1)] = -1.0
        z[t, e] = 1.0
    z[0, [0, E - 1]] = [1.0, -1.0]
    case(f"route pair T={T} E={E}")
    check(gpu, z, 3)
    check(gpu, z, 3, sigmoid=True)


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("T,E", SIZES)
def test_choices_of_both_signs(gpu, T, E, sigmoid):
    """A few logits above 0 and the rest below, of whole numbers, many of them equal; rows of which a mask leaves some 20."""
    rng = np.random.default_rng(T + E + sigmoid)
    z = np.rint(rng.normal(-3.5, 1.5, (T, E))).astype(np.float32)
    z[::3][~live(rng, len(z[::3]), E)] = -np.inf
    case(f"route signs T={T} E={E} sigmoid={sigmoid}")
    check(gpu, z, 16, sigmoid=sigmoid)
    check(gpu, z, 8, sigmoid=sigmoid)


@pytest.mark.parametrize("groups,top_groups", [(1, 1), (4, 2)])
@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("T,E", [(T, E) for T in (7, 2050, 16387) for E in (512, 520, 768, 1024)])
def test_biases_beside_which_scores_vanish(gpu, T, E, sigmoid, groups, top_groups):
    """Scores of 1e-87 or less beside biases of eighths of both signs, few of them above 0: the bias alone orders the experts."""
    rng = np.random.default_rng(T + E + groups)
    z = np.full((T, E), -200.0, np.float32)
    z[::2][~live(rng, len(z[::2]), E)] = -np.inf
    if not sigmoid:
        z[np.arange(T), rng.integers(0, E, T)] = 100.0
    bias = (np.rint(8 * rng.normal(-2.5, 1.2, E)) / 8).astype(np.float32)
    bias[bias == 0] = 0.125  # (a score beside no bias is one)
    case(f"route biases T={T} E={E} sigmoid={sigmoid} groups={groups}/{top_groups}")
    check(gpu, z, 9, sigmoid=sigmoid, bias=bias, groups=groups, top_groups=top_groups)


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("E,groups,top_groups", [(40, 8, 3), (256, 8, 4), (24, 24, 5), (1024, 64, 9), (520, 4, 1)])
@pytest.mark.parametrize("T", [7, 2050, 16387])
def test_groups_of_which_a_mask_leaves_less_than_two(gpu, T, E, groups, top_groups, sigmoid, bias):
    """The sum of a group's two largest scores is -inf where it has one: any other group comes first, and of such groups
    the first ones."""
    rng = np.random.default_rng(T + E + 2 * sigmoid + bias)
    # (all below 0, where no two pairs of sigmoids have one sum)
    z = (rng.permuted(np.tile(np.arange(E), (T, 1)), axis=1) % 61 / 8.0 - 7.75).astype(np.float32)
    left = rng.integers(0, 4, (T, groups, 1))  # of each group
    order = rng.permuted(np.tile(np.arange(E // groups), (T, groups, 1)), axis=2)
    z[(order >= left).reshape(T, E)] = -np.inf
    z[0] = -np.inf
    z[0, E // groups * (groups - 1)] = 3.0  # one expert in all, of the last group
    z[1] = -np.inf
    z[1, :E // groups] = 1.0
    b = None
    if bias:
        b = (2 * rng.standard_normal(E)).astype(np.float32)
        b[E // 2] = np.inf
        b[E - 1] = -np.inf
    case(f"route groups T={T} E={E} groups={groups}/{top_groups} sigmoid={sigmoid} bias={bias}")
    check(gpu, z, 6, sigmoid=sigmoid, bias=b, groups=groups, top_groups=top_groups, best=2)


@pytest.mark.parametrize("T", [5, 2050, 16387])
@pytest.mark.parametrize("bias,groups,top_groups,best,want", [
    (False, 1, 1, 1, [5, 2, 6]), (False, 4, 3, 1, [5, 2, 6]), (False, 4, 4, 2, [5, 2, 6]), (False, 8, 5, 2, [5, 2, 6]),
    (True, 1, 1, 1, [0, 2, 5]), (True, 4, 3, 1, [0, 2, 5]), (False, 4, 3, 2, [0, 5, 6])])
def test_sigmoids_that_are_one(gpu, T, bias, groups, top_groups, best, want):
    """exp(-38) is below 2^-54, so sigmoids of 38 and more are 1 in 64 bits: the logits tell them apart where they are the
    order, and the index where c is."""
    z = np.full((T, 8), -3.0, np.float32)
    z[:, 0], z[:, 2], z[:, 5], z[:, 6] = 38.0, 40.0, 41.0, 39.0
    z[:, 4] = 2.0
    z[:, 7] = 1.0
    case(f"route ones T={T} bias={bias} groups={groups}/{top_groups} best={best}")
    b = np.zeros(8, np.float32) if bias else None
    assert reference(z, 3, True, b, groups, top_groups, best)[0][0].tolist() == want
    check(gpu, z, 3, sigmoid=True, bias=b, groups=groups, top_groups=top_groups, best=best)


@pytest.mark.parametrize("sigmoid", [True, False])
@pytest.mark.parametrize("seed", range(3))
def test_scores_hold_49_bits(gpu, seed, sigmoid):
    """A score s (a sigmoid, or the softmax of it and 0) less its fp32 value, which is exact, lies between fp32 biases just
    below and above: exp is off by 2^-50 of it and what follows it by five roundings of 2^-53 or less, together less
    than 2^-49 of s, and the biases are further away."""
    rng = np.random.default_rng(seed)
    T, E = 340, 1023
    zt = rng.uniform(-30.0, 0.0 if not sigmoid else 12.0, T).astype(np.float32)
    e = np.exp(-np.abs(zt.astype(np.longdouble)))
    s = np.where(zt >= 0, np.longdouble(1), e) / (1 + e)
    rest = s - s.astype(np.float32).astype(np.longdouble)
    up, down = np.float32(np.inf), np.float32(-np.inf)
    hi = np.nextafter((rest + s * 2.0 ** -49).astype(np.float32), up)
    lo = np.nextafter((rest - s * 2.0 ** -49).astype(np.float32), down)
    z, bias = np.full((T, E), -np.inf, np.float32), np.zeros(E, np.float32)
    at = rng.permutation(E - 3)[:3 * T].reshape(T, 3)  # of each token: below, s, above
    np.put_along_axis(z, at, np.stack([np.full(T, -200.0), zt, np.full(T, -200.0)], 1).astype(np.float32), 1)
    bias[at] = np.stack([lo, -s.astype(np.float32), hi], 1)
    if not sigmoid:
        z[:, E - 1] = 0.0  # in the sum, and never chosen
        bias[E - 1] = -np.inf
    case(f"route 49 bits seed={seed} sigmoid={sigmoid}")
    idx, w = torch.empty((T, 4), dtype=torch.int32, device="cuda"), torch.empty((T, 4), device="cuda")
    gpu.ops.moe_route(dev(z), idx, w, sigmoid, dev(bias))
    assert np.array_equal(host(idx), np.concatenate([at[:, ::-1], np.full((T, 1), -1)], 1))
