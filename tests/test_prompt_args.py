"""Refusals of the entry points for batches that hold prompts: every call below is rejected on the host, before any
launch (no GPU)."""
import pytest

from mnemocuda_amd import lib as mlib

A = 4096  # a non-null, aligned address that no call below reaches


@pytest.fixture(scope="module")
def L():
    return mlib.load_library()


def refused(L, rc, what, capfd):
    assert rc == 1
    assert what in capfd.readouterr().err
    assert L.mnemo_last_error() == 1


def prompt(L, *, q=A, kp=A, vp=A, ks=None, vs=None, kv_type=0, out=A, T=20, nh=8, hd=128, nkv=2, n_pages=8, ps=64, table=A, n_seqs=4,
           max_pages=4, starts=A, lens=A, ws=A, wsb=1 << 30):
    return L.mnemo_paged_attention_prompt(q, kp, vp, ks, vs, kv_type, out, T, nh, hd, nkv, n_pages, ps, table, n_seqs, max_pages,
                                          starts, lens, 0.1, ws, wsb, None)


@pytest.mark.parametrize("bad", [
    dict(kp=None), dict(vp=None), dict(kp=A + 8), dict(kv_type=2), dict(kv_type=1), dict(kv_type=1, ks=A, vs=A + 4), dict(hd=96),
    dict(ps=48), dict(nkv=0), dict(n_pages=0), dict(n_pages=(1 << 30) + 1), dict(q=None), dict(out=None), dict(table=None),
    dict(starts=None), dict(lens=None), dict(ws=None), dict(ws=A + 4), dict(wsb=8), dict(wsb=1 << 20), dict(nh=7), dict(nh=34),
    dict(nh=0), dict(n_seqs=0), dict(n_seqs=4097), dict(max_pages=0), dict(max_pages=1 << 25), dict(T=-1), dict(T=(1 << 22) + 1),
    dict(n_seqs=4096, max_pages=1 << 19, ps=16), dict(T=1 << 22, max_pages=1 << 14, nh=32), dict(T=1 << 20, max_pages=1 << 20)])
def test_prompt_attention_refuses(L, bad, capfd):
    refused(L, prompt(L, **bad), "paged_attention_prompt", capfd)


def route(L, *, z=A, T=4, E=64, score=0, bias=A, groups=4, top=2, best=2, k=6, idx=A, w=A):
    return L.mnemo_moe_route(z, T, E, score, bias, groups, top, best, k, 1, 1.0, idx, w, None)


@pytest.mark.parametrize("bad", [
    dict(z=None), dict(idx=None), dict(w=None), dict(T=-1), dict(T=4194304, k=2), dict(E=0), dict(E=1025, groups=1, top=1), dict(E=4, k=6),
    dict(k=0), dict(k=17), dict(groups=0), dict(groups=3), dict(groups=128, E=128), dict(top=0), dict(top=5), dict(best=0),
    dict(best=3), dict(score=2), dict(score=-1)])
def test_route_refuses(L, bad, capfd):
    refused(L, route(L, **bad), "moe_route", capfd)


def lora(L, *, x=A, a=A, b=A, typ=0, ids=A, ranks=A, scales=A, base=A, out=A, T=4, K=64, M=32, N=2, R=16, ws=A, wsb=1 << 30):
    return L.mnemo_lora_add(x, a, b, typ, ids, ranks, scales, base, out, T, K, M, N, R, ws, wsb, None)


@pytest.mark.parametrize("bad", [
    dict(x=None), dict(a=None), dict(b=None), dict(ids=None), dict(ranks=None), dict(scales=None), dict(base=None),
    dict(out=None), dict(ws=None), dict(ws=A + 4), dict(wsb=16), dict(a=A + 8), dict(b=A + 2), dict(typ=2), dict(typ=-1),
    dict(T=-1), dict(T=524289), dict(K=0), dict(K=60), dict(K=(1 << 20) + 8), dict(M=0), dict(M=(1 << 24) + 1), dict(N=0),
    dict(N=65537), dict(R=0), dict(R=12), dict(R=264)])
def test_lora_refuses(L, bad, capfd):
    refused(L, lora(L, **bad), "lora_add", capfd)


def logprobs(L, *, z=A, t=A, n=2, V=100, lp=A, rank=A, ent=A, k=4, ids=A, tops=A, ws=A, wsb=1 << 30):
    return L.mnemo_logprobs(z, t, n, V, lp, rank, ent, k, ids, tops, ws, wsb, None)


@pytest.mark.parametrize("bad", [
    dict(z=None), dict(lp=None), dict(ids=None), dict(tops=None), dict(n=-1), dict(n=65536), dict(V=0), dict(V=(1 << 30) + 1),
    dict(k=-1), dict(k=65), dict(ws=None), dict(ws=A + 8), dict(V=100000, wsb=16)])
def test_logprobs_refuses(L, bad, capfd):
    refused(L, logprobs(L, **bad), "logprobs", capfd)


def test_nothing_of_no_rows(L):
    assert prompt(L, T=0, q=None, out=None, ws=None) == 0
    assert route(L, T=0, z=None, idx=None, w=None) == 0
    assert lora(L, T=0, x=None, out=None, ws=None) == 0
    assert logprobs(L, n=0, z=None, ws=None) == 0


def test_workspaces(L):
    """What suffices for a call suffices for every smaller one."""
    lora, lp, at = L.mnemo_lora_workspace_bytes, L.mnemo_logprobs_workspace_bytes, L.mnemo_paged_attention_prompt_workspace_bytes
    assert lora(100, 4096, 16) == 4 * 100 * 16 * 4  # four parts
    assert lora(524288, 1 << 20, 256) > 524288 * 256 * 4  # past 32 bits
    sizes = [1, 2, 15, 16, 17, 100, 1000, 1023, 1024, 1025, 3000, 5000, 8192, 16384, 16385, 60000]
    for k in (8, 1000, 4096, 9000, 1 << 20):
        need = [lora(n, k, 64) for n in sizes]
        assert need == sorted(need) and need[0] > 0
    for v in (1, 5000, 151936, 1 << 30):
        need = [lp(n, v, 20) for n in sizes]
        assert need == sorted(need) and need[0] > 0
        assert lp(7, v, 0) <= lp(7, v, 1) <= lp(7, v, 64)
    assert lora(10, 60, 16) == lora(10, 64, 260) == lora(-1, 64, 16) == 0
    assert lp(0, 100, 4) == lp(1, 100, 65) == 0
    assert at(8, 2, 128) == at(64, 4, 128) > 0 and at(8, 2, 96) == at(0, 2, 128) == 0


def test_wrappers_refuse_host_tensors_and_shapes(L):
    """The Python wrappers check tensors before anything is launched (CPU tensors reach no kernel)."""
    import torch

    from mnemocuda_amd import MnemoError, ops
    z = lambda *s, t=torch.float32: torch.zeros(s, dtype=t)  # noqa: E731
    i = lambda *s: z(*s, t=torch.int32)  # noqa: E731
    h = lambda *s: z(*s, t=torch.float16)  # noqa: E731
    k, v = h(8, 2, 16, 64), h(8, 2, 64, 16)
    with pytest.raises(MnemoError, match="do not fit"):  # v laid out as k is
        ops.paged_attention_prompt(z(5, 4, 64), k, h(8, 2, 16, 64), i(2, 3), i(3), i(2), z(5, 4, 64), 0.1, z(64))
    with pytest.raises(MnemoError, match="GPU tensor"):
        ops.paged_attention_prompt(z(5, 4, 64), k, v, i(2, 3), i(3), i(2), z(5, 4, 64), 0.1, z(64))
    with pytest.raises(MnemoError, match="moe_route: logits must be"):
        ops.moe_route(z(4, 8), i(3, 2), z(3, 2))
    with pytest.raises(MnemoError, match="GPU tensor"):
        ops.moe_route(z(4, 8), i(4, 2), z(4, 2))
    with pytest.raises(MnemoError, match="a_w must be"):
        ops.lora_add(z(4, 64), h(2, 8, 64), h(2, 8, 32), i(4), i(2), z(2), z(4, 32), z(4, 32), z(64))
    with pytest.raises(MnemoError, match="2 dimensions"):
        ops.lora_add(z(4, 64), h(2, 8, 64), h(2, 32, 8), i(4), i(2), z(2), z(4, 32), z(4, 33), z(64))
    with pytest.raises(MnemoError, match="float16 or bfloat16"):
        ops.lora_add(z(4, 64), z(2, 8, 64), z(2, 32, 8), i(4), i(2), z(2), z(4, 32), z(4, 32), z(64))
    with pytest.raises(MnemoError, match="GPU tensor"):
        ops.lora_add(z(4, 64), h(2, 8, 64), h(2, 32, 8), i(4), i(2), z(2), z(4, 32), z(4, 32), z(64))
    with pytest.raises(MnemoError, match="logprobs: logits must be"):
        ops.logprobs(z(4, 64), i(4), z(4), i(4), z(4), i(4, 3), z(4, 2), z(64))
    with pytest.raises(MnemoError, match="GPU tensor"):
        ops.logprobs(z(4, 64), i(4), z(4), i(4), z(4), None, None, z(64))
