"""Logits processing against the formula in 64 bits, one token at a time."""
import numpy as np
import pytest
import torch

from tests.gpu_util import case, dev, host

pytestmark = pytest.mark.gpu


def reference(z, hist=None, hl=None, pl=None, rep=None, freq=None, pres=None, ids=None, bias=None, allowed=None):
    """(result, bound): the bound counts the roundings, 2^-24 each, of the sizes that occur on the way."""
    n, V = z.shape
    out, size = z.astype(np.float64).copy(), np.abs(z.astype(np.float64))
    for r in range(n):
        if hist is not None:
            h = hist[r, :min(max(int(hl[r]), 0), hist.shape[1])]
            ok = (h >= 0) & (h < V)
            prompt = np.arange(len(h)) < pl[r]
            count = np.bincount(h[ok & ~prompt], minlength=V)
            seen = np.bincount(h[ok], minlength=V) > 0
            x = out[r]
            with np.errstate(invalid="ignore"):
                y = np.where(x > 0, x / np.float64(rep[r]), x * np.float64(rep[r]))
            x = np.where(seen, y, x)
            out[r] = np.where(count > 0, x - count * np.float64(freq[r]) - np.float64(pres[r]), x)
            size[r] = np.abs(x) + count * abs(float(freq[r])) + (count > 0) * abs(float(pres[r])) + size[r] * ~seen
        if ids is not None:
            last = {int(t): float(b) for t, b in zip(ids[r], bias[r]) if 0 <= t < V}
            for t, b in last.items():
                out[r, t] += b
                size[r, t] += abs(b)
        if allowed is not None:
            bits = (allowed[r].astype(np.int64)[:, None] >> np.arange(32)) & 1
            out[r, bits.flatten()[:V] == 0] = -np.inf
    return out, 5 * 2.0 ** -24 * size


def check(got, want, bound):
    fine = np.isfinite(want)
    assert np.array_equal(got[~fine], want[~fine].astype(np.float32), equal_nan=True)
    assert (np.abs(got[fine] - want[fine]) <= bound[fine]).all()


def inputs(rng, n, V, H, B, mask):
    a = {"z": (3 * rng.standard_normal((n, V))).astype(np.float32)}
    if H is not None:
        a["hist"] = (V * rng.random((n, H)) ** 4).astype(np.int32)
        a["hl"] = rng.integers(0, H + 1, n).astype(np.int32)
        a["hl"][0] = H
        a["pl"] = (a["hl"] * rng.random(n)).astype(np.int32)
        a["rep"] = rng.uniform(0.7, 1.5, n).astype(np.float32)
        a["freq"], a["pres"] = (rng.uniform(-1, 1, n).astype(np.float32) for _ in range(2))
    if B:
        a["ids"] = rng.integers(0, V, (n, B)).astype(np.int32)  # tokens named twice among them
        a["bias"] = (5 * rng.standard_normal((n, B))).astype(np.float32)
    if mask:
        a["allowed"] = rng.integers(-2 ** 31, 2 ** 31, (n, -(-V // 32))).astype(np.int32)
    return a


NAMES = dict(hist="history", hl="history_lens", pl="prompt_lens", rep="repetition", freq="frequency", pres="presence",
             ids="bias_ids", bias="bias", allowed="allowed")


def run(gpu, a, out=None):
    d = {NAMES[k]: dev(x) for k, x in a.items() if k != "z"}
    z = dev(a["z"])
    out = torch.full(a["z"].shape, 55.0, device="cuda") if out is None else z
    gpu.ops.logits_process(z, out, **d)
    return host(out), host(z)


@pytest.mark.parametrize("n,V,H,B,mask", [
    (1, 1, 4, 1, True), (3, 31, 10, 5, True), (2, 33, 1, 0, True), (2, 4095, 300, 9, True), (2, 4096, 300, 9, False),
    (3, 4097, 300, 9, True), (5, 10007, 0, 3, True), (4, 8195, None, 40, True), (4, 20001, 5000, 0, False),
    (1, 151936, 131072, 300, True), (9, 151937, 900, 2000, True), (700, 50, 77, 3, True), (2, 262144, 10, 1, True),
    (20, 151937, 3000, 90, True), (41, 151935, 9000, 40, True), (2100, 2001, 33, 2, False)])  # larger slices
def test_against_the_formula(gpu, n, V, H, B, mask):
    rng = np.random.default_rng(n + V)
    a = inputs(rng, n, V, H, B, mask)
    want, bound = reference(**a)
    case(f"logits n={n} V={V} history={H} bias={B} mask={mask}")
    got, z = run(gpu, a)
    assert np.array_equal(z, a["z"])
    check(got, want, bound)
    inplace, _ = run(gpu, a, out="z")
    assert np.array_equal(inplace, got)


def test_ids_and_lengths_out_of_range(gpu):
    """Ids outside the vocabulary are ignored, lengths outside 0..max_history cut, prompts longer than the history
    and below zero taken as they are."""
    rng = np.random.default_rng(2)
    a = inputs(rng, 6, 5000, 64, 8, False)
    a["hist"][:, ::5] = rng.choice(np.array([-1, 5000, 2 ** 31 - 1, -2 ** 31, 5001, 9192], np.int64), (6, 13)).astype(np.int32)
    a["ids"][:, ::3] = rng.choice(np.array([-1, 5000, 2 ** 31 - 1, -2 ** 31], np.int64), (6, 3)).astype(np.int32)
    a["hl"][:] = [64, 1000, -4, 0, 30, 2 ** 31 - 1]
    a["pl"][:] = [100, 10, 5, 0, -3, 64]
    want, bound = reference(**a)
    case("logits, ids and lengths out of range")
    check(run(gpu, a)[0], want, bound)


def test_numbers_that_are_none(gpu):
    """NaN and infinities: masked ones give -inf, the others follow the formula; a mask that allows nothing."""
    rng = np.random.default_rng(4)
    a = inputs(rng, 4, 3000, 50, 3, True)
    a["z"][:, ::7] = rng.choice(np.array([np.nan, np.inf, -np.inf], np.float32), (4, 429))
    a["z"][3, :40] = [0.0, -0.0] * 20
    a["allowed"][1] = 0
    a["allowed"][2] = -1
    with np.errstate(invalid="ignore"):
        want, bound = reference(**a)
    case("logits, NaN and infinities")
    got = run(gpu, a)[0]
    assert (got[1] == -np.inf).all()
    check(got, want, bound)


def test_many_times_the_same_token(gpu):
    """A count past 2^16, in one counter."""
    a = {"z": np.zeros((1, 100), np.float32), "hist": np.full((1, 100000), 42, np.int32),
         "hl": np.array([100000], np.int32), "pl": np.array([1], np.int32), "rep": np.array([1.5], np.float32),
         "freq": np.array([0.5], np.float32), "pres": np.array([2.0], np.float32)}
    case("logits, one token 99,999 times")
    got = run(gpu, a)[0]
    assert got[0, 42] == -99999 * 0.5 - 2.0 and not np.delete(got[0], 42).any()


def test_rows_that_are_not_aligned(gpu):
    """Rows that start at odd multiples of 4 bytes (vocabulary of 1 mod 4, and a view that is offset by one)."""
    rng = np.random.default_rng(6)
    a = inputs(rng, 3, 9001, 40, 4, True)
    want, bound = reference(**a)
    z = torch.empty(3 * 9001 + 1, device="cuda")[1:].view(3, 9001)
    z.copy_(dev(a["z"]))
    out = torch.empty(3 * 9001 + 3, device="cuda")[3:].view(3, 9001)
    case("logits, unaligned rows")
    gpu.ops.logits_process(z, out, **{NAMES[k]: dev(x) for k, x in a.items() if k != "z"})
    check(host(out), want, bound)


def test_in_a_graph_then_sampled(gpu):
    """A captured call followed by the sampler, replayed with other logits and histories: the mask's only token is
    drawn, and the eager result is met bit for bit."""
    rng = np.random.default_rng(7)
    V = 32003
    a = inputs(rng, 1, V, 60, 5, True)
    d = {NAMES[k]: dev(x) for k, x in a.items() if k != "z"}
    z, out = dev(a["z"]), torch.empty((1, V), device="cuda")
    tok = torch.full((1,), -1, dtype=torch.int32, device="cuda")
    ws = torch.zeros(gpu.ops.sample_workspace_bytes(), dtype=torch.uint8, device="cuda")

    def step():
        gpu.ops.logits_process(z, out, **d)
        gpu.ops.sample_token_ws(out[0], V, 0.0, 1.0, 1, ws, tok)

    case("logits graph capture")
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
    for i in range(4):
        b = inputs(rng, 1, V, 60, 5, True)
        only = int(rng.integers(0, V))
        if i % 2:
            b["allowed"][:] = 0
            b["allowed"][0, only // 32] = np.int32(np.uint32(1 << (only % 32)).astype(np.int64) - (1 << 32 if only % 32 == 31 else 0))
        z.copy_(dev(b["z"]))
        for k, t in d.items():
            t.copy_(dev(b[{v: n for n, v in NAMES.items()}[k]]))
        graph.replay()
        torch.cuda.synchronize()
        got, drawn = host(out).copy(), int(host(tok)[0])
        check(got, *reference(**b))
        assert drawn == (only if i % 2 else int(np.argmax(got)))
        step()
        assert np.array_equal(host(out), got) and int(host(tok)[0]) == drawn
