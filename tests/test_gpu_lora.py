"""Adapters of many requests against the formula in 64 bits.

Bound of an output: the sums over n_in and the rank are fp32, at most one rounding per term, so with u = 2^-24 and
S = |base| + |scale| sum_r |B| sum_k |A| |x| an output is off by less than (n_in + rank + 64) u S.  That is the worst case;
the relative L2 of an output whose roundings are independent is that of some 256 of them, 2^-20, and is held below
2^-19."""
import numpy as np
import pytest
import torch

from tests.conftest import rel_l2
from tests.gpu_util import case, dev, host

pytestmark = pytest.mark.gpu
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def inputs(seed, T, K, M, N, R, typ, ids="mixed", rank=None):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    t = TYPES[typ]
    a = {"x": rn(T, K), "a": (rn(N, R, K) * K ** -0.5).to(t), "b": (rn(N, M, R) * R ** -0.5).to(t), "base": rn(T, M),
         "scales": 0.5 + torch.rand(N, generator=g)}
    a["ranks"] = (torch.randint(1, R + 1, (N,), generator=g) if rank is None else torch.full((N,), rank)).to(torch.int32)
    if ids == "mixed":
        i = torch.randint(-1, N, (T,), generator=g)
    elif ids == "runs":
        i = torch.arange(T) * N // T
    else:
        i = torch.full((T,), ids)
    a["ids"] = i.to(torch.int32)
    # what lies behind the rank counts for nothing
    for n in range(N):
        a["a"][n, max(int(a["ranks"][n]), 0):] = float("nan")
        a["b"][n, :, max(int(a["ranks"][n]), 0):] = float("inf")
    return a


def reference(a):
    out = a["base"].double().numpy().copy()
    size = np.abs(out)
    x = a["x"].double().numpy()
    for t, i in enumerate(a["ids"].tolist()):
        if not 0 <= i < len(a["ranks"]) or a["ranks"][i] <= 0:
            continue
        r, s = int(a["ranks"][i]), float(a["scales"][i])
        A, B = a["a"][i, :r].double().numpy(), a["b"][i, :, :r].double().numpy()
        out[t] += s * (B @ (A @ x[t]))
        size[t] += abs(s) * (np.abs(B) @ (np.abs(A) @ np.abs(x[t])))
    return out, (a["x"].shape[1] + a["a"].shape[1] + 64) * 2.0 ** -24 * size


def run(gpu, a, inplace=False):
    T, K = a["x"].shape
    d = {k: t.cuda() for k, t in a.items()}
    M = a["base"].shape[1]
    buf = torch.full((T + 1, M), 55.0, device="cuda")
    out = buf[:T]
    base = d["base"]
    if inplace:
        out.copy_(base)
        base = out
    ws = torch.full((gpu.ops.lora_workspace_bytes(T, K, a["a"].shape[1]),), 255, dtype=torch.uint8, device="cuda")  # NaN
    gpu.ops.lora_add(d["x"], d["a"], d["b"], d["ids"], d["ranks"], d["scales"], base, out, ws)
    got = host(buf)
    assert (got[T] == 55).all()
    if not inplace:
        assert torch.equal(base.cpu(), a["base"])
    return got[:T]


def check(got, want, bound):
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= bound).all()


@pytest.mark.parametrize("typ", ["f16", "bf16"])
@pytest.mark.parametrize("T,K,M,N,R,ids", [
    (1, 8, 1, 1, 8, 0), (1, 4096, 4096, 4, 16, 2), (3, 264, 37, 2, 8, "mixed"), (16, 1024, 64, 16, 16, "runs"), (17, 1032, 257, 3, 24, "mixed"),
    (61, 512, 1000, 40, 64, "mixed"), (33, 4096, 260, 5, 32, "mixed"), (40, 520, 1030, 7, 128, "mixed"), (18, 256, 515, 3, 256, "mixed"),
    (5, 9000, 40, 2, 40, "mixed"), (700, 256, 512, 6, 16, "runs"), (1100, 128, 130, 9, 32, "mixed"), (64, 64, 64, 2, 8, -1)])
def test_against_the_formula(gpu, typ, T, K, M, N, R, ids):
    a = inputs(T + K, T, K, M, N, R, typ, ids)
    want, bound = reference(a)
    case(f"lora {typ} T={T} K={K} M={M} N={N} R={R} ids={ids}")
    got = run(gpu, a)
    check(got, want, bound)
    assert rel_l2(got, want) <= 2.0 ** -19
    assert np.array_equal(run(gpu, a, inplace=True), got)


@pytest.mark.parametrize("typ", ["f16", "bf16"])
def test_ids_and_ranks_out_of_range(gpu, typ):
    """Ids outside the table and ranks of 0 and less leave the base, ranks past max_rank are cut."""
    a = inputs(3, 20, 128, 70, 5, 16, typ)
    a["a"] = torch.randn(a["a"].shape).to(a["a"].dtype)
    a["b"] = torch.randn(a["b"].shape).to(a["b"].dtype)
    a["ids"][:8] = torch.tensor([-1, 5, 2 ** 31 - 1, -2 ** 31, 0, 1, 2, 3], dtype=torch.int32)
    a["ranks"] = torch.tensor([16, 0, -3, 16, 7], dtype=torch.int32)
    want, bound = reference(a)
    case("lora ids out of range")
    got = run(gpu, a)
    check(got, want, bound)
    for t in (0, 1, 2, 3, 5, 6):
        assert np.array_equal(got[t], a["base"][t].numpy())
    b = {k: t.clone() for k, t in a.items()}
    b["ranks"][0] = 1000
    assert np.array_equal(run(gpu, b), got)


@pytest.mark.parametrize("typ", ["f16", "bf16"])
def test_rows_do_not_meet(gpu, typ):
    """NaN and infinities of one token or adapter stay with the tokens that have them."""
    a = inputs(5, 32, 512, 90, 4, 16, typ)
    a["ids"] = (torch.arange(32) % 5 - 1).to(torch.int32)
    clean, bound = reference(a)
    a["x"][3, 17], a["x"][9, 400], a["x"][20, 0] = float("nan"), float("inf"), -float("inf")
    a["a"][2, 0, 5] = float("nan")
    a["b"][3, 7, 0] = float("inf")
    case("lora NaN")
    got = run(gpu, a)
    ids = a["ids"].numpy()
    for t in range(32):
        if t in (3, 9) or ids[t] == 2:
            assert np.isnan(got[t]).all(), t
        elif ids[t] == 3:
            assert not np.isfinite(got[t, 7]) and np.isfinite(np.delete(got[t], 7)).all()
        else:  # token 20 has no adapter
            assert (np.abs(got[t] - clean[t]) <= bound[t]).all(), t
    assert ids[20] == -1 and ids[3] >= 0 and ids[9] >= 0


@pytest.mark.parametrize("typ", ["f16", "bf16"])
def test_sizes_far_apart(gpu, typ):
    """Tokens of 2^-100 to 2^100, and one whose values rise along the row: a later chunk's scale exceeds an
    earlier one's."""
    a = inputs(6, 20, 2304, 40, 2, 16, typ, 1, rank=16)
    for t in range(18):
        a["x"][t] *= 2.0 ** (12 * t - 100)
        a["base"][t] *= 2.0 ** (12 * t - 100)
    a["x"][18] *= 2.0 ** (torch.arange(2304) // 64 - 10.0)
    a["x"][19] *= 2.0 ** (20.0 - torch.arange(2304) // 64)
    want, bound = reference(a)
    case("lora sizes")
    got = run(gpu, a)
    check(got, want, bound)
    for t in range(20):
        assert rel_l2(got[t], want[t]) <= 2.0 ** -19, t


def test_in_a_graph_with_other_adapters(gpu):
    """Captured once; ids, ranks and inputs change between replays."""
    T, K, M, N, R = 37, 1024, 300, 6, 32
    a = inputs(7, T, K, M, N, R, "bf16")
    d = {k: t.cuda() for k, t in a.items()}
    out = torch.empty((T, M), device="cuda")
    ws = torch.empty(gpu.ops.lora_workspace_bytes(T, K, R), dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    case("lora graph")
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            gpu.ops.lora_add(d["x"], d["a"], d["b"], d["ids"], d["ranks"], d["scales"], d["base"], out, ws)
    for i in range(4):
        b = inputs(70 + i, T, K, M, N, R, "bf16", "runs" if i == 2 else "mixed")
        for k, t in d.items():
            t.copy_(b[k])
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        torch.cuda.synchronize()
        got = host(out).copy()
        check(got, *reference(b))
        assert np.array_equal(run(gpu, b), got)


def test_unaligned_rows(gpu):
    """x, base and out at odd multiples of 4 bytes."""
    a = inputs(8, 19, 264, 131, 3, 16, "f16")
    want, bound = reference(a)
    d = {k: t.cuda() for k, t in a.items()}
    off = lambda t: torch.empty(t.numel() + 1, device="cuda")[1:].view(t.shape).copy_(t)  # noqa: E731
    x, base, out = off(d["x"]), off(d["base"]), off(d["base"])
    ws = torch.empty(gpu.ops.lora_workspace_bytes(19, 264, 16), dtype=torch.uint8, device="cuda")
    case("lora unaligned")
    gpu.ops.lora_add(x, d["a"], d["b"], d["ids"], d["ranks"], d["scales"], base, out, ws)
    check(host(out), want, bound)


@pytest.mark.parametrize("typ", ["f16", "bf16"])
@pytest.mark.parametrize("T,K,M,N,R,ids", [(1030, 264, 520, 5, 128, "mixed"), (1041, 136, 300, 3, 256, "runs"), (1030, 1500 * 8, 24, 2, 8, "runs"),
                                           (16401, 2056, 24, 4, 8, "runs")])
def test_many_tokens(gpu, typ, T, K, M, N, R, ids):
    """High ranks; and parts of K that are more than one pass of a workgroup."""
    a = inputs(T + K, T, K, M, N, R, typ, ids)
    want, bound = reference(a)
    case(f"lora {typ} T={T} K={K} M={M} N={N} R={R} ids={ids}")
    got = run(gpu, a)
    check(got, want, bound)
    assert rel_l2(got, want) <= 2.0 ** -19


def test_two_streams_with_their_own_workspaces(gpu):
    """Calls of two streams at once, each as if alone."""
    a, b = inputs(30, 900, 1032, 260, 6, 16, "f16"), inputs(31, 40, 4096, 1000, 40, 64, "bf16")
    want = [run(gpu, a), run(gpu, b)]
    todo = []
    for c in (a, b):
        d = {k: t.cuda() for k, t in c.items()}
        ws = torch.empty(gpu.ops.lora_workspace_bytes(*d["x"].shape, d["a"].shape[1]), dtype=torch.uint8, device="cuda")
        todo.append((torch.cuda.Stream(), d, torch.empty_like(d["base"]), ws))
    torch.cuda.synchronize()
    case("lora, two streams")
    for _ in range(5):
        for stream, d, out, ws in todo:
            with torch.cuda.stream(stream):
                gpu.ops.lora_add(d["x"], d["a"], d["b"], d["ids"], d["ranks"], d["scales"], d["base"], out, ws)
    torch.cuda.synchronize()
    for (_, _, out, _), w in zip(todo, want):
        assert np.array_equal(host(out), w)
