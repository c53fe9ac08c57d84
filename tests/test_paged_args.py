"""Refusals of the paged-cache and logits entry points: every call below is rejected on the host,
before any launch (no GPU)."""
import pytest

from mnemocuda_amd import lib as mlib

A = 4096  # a non-null, aligned address that no call below reaches


@pytest.fixture(scope="module")
def L():
    return mlib.load_library()


def prep(L, *, q=A, k=A, v=A, qw=A, kw=A, theta=1e6, T=2, nh=8, hd=128, nkv=2, pos=A, seq=A, table=A, lens=None,
         n_seqs=4, max_pages=4, kp=A, vp=A, ks=None, vs=None, kv_type=0, n_pages=8, ps=64, out=A):
    return L.mnemo_paged_attn_prep(q, k, v, qw, kw, 1e-6, theta, T, nh, hd, nkv, pos, seq, table, lens, n_seqs,
                                   max_pages, kp, vp, ks, vs, kv_type, n_pages, ps, out, None)


def attend(L, *, q=A, kp=A, vp=A, ks=None, vs=None, kv_type=0, out=A, n_seqs=4, nh=8, hd=128, nkv=2, n_pages=8, ps=64,
           table=A, max_pages=4, lens=A, ws=A, wsb=1 << 30):
    return L.mnemo_paged_attention_decode(q, kp, vp, ks, vs, kv_type, out, n_seqs, nh, hd, nkv, n_pages, ps, table,
                                          max_pages, lens, 0.1, ws, wsb, None)


CACHE = [dict(kp=None), dict(vp=None), dict(kp=A + 8), dict(kv_type=2), dict(kv_type=1), dict(kv_type=1, ks=A, vs=A + 4),
         dict(hd=96), dict(ps=48), dict(ps=8), dict(nkv=0), dict(n_pages=0), dict(n_pages=(1 << 30) + 1)]


@pytest.mark.parametrize("bad", CACHE + [
    dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(table=None), dict(qw=None), dict(kw=None),
    dict(pos=None), dict(seq=None), dict(pos=None, seq=None), dict(pos=None, seq=None, lens=A, T=5), dict(T=-1),
    dict(T=(1 << 22) + 1), dict(n_seqs=0), dict(n_seqs=4097), dict(max_pages=0), dict(max_pages=1 << 25, ps=64),
    dict(nh=0), dict(theta=0.0), dict(theta=0.9), dict(theta=float("inf")), dict(theta=float("nan"))])
def test_prep_refuses(L, bad, capfd):
    assert prep(L, **bad) == 1
    assert "paged_attn_prep" in capfd.readouterr().err
    assert L.mnemo_last_error() == 1


def test_prep_of_no_tokens_is_nothing(L):
    assert prep(L, T=0, q=None, k=None, v=None, out=None, pos=None, seq=None) == 0


@pytest.mark.parametrize("bad", CACHE + [
    dict(q=None), dict(out=None), dict(table=None), dict(lens=None), dict(ws=None), dict(ws=A + 4), dict(wsb=8),
    dict(nh=7), dict(nh=34), dict(nh=0), dict(n_seqs=0), dict(n_seqs=4097), dict(max_pages=0),
    dict(max_pages=1 << 25, ps=64), dict(n_seqs=4096, max_pages=1 << 20, ps=16)])
def test_attention_refuses(L, bad, capfd):
    assert attend(L, **bad) == 1
    assert "paged_attention_decode" in capfd.readouterr().err
    assert L.mnemo_last_error() == 1


def extend(L, *, table=A, lens=A, refs=A, new=A, n_seqs=4, max_pages=4, n_pages=8, ps=64):
    return L.mnemo_kv_pages_extend(table, lens, refs, new, n_seqs, max_pages, n_pages, ps, None, None)


def free(L, *, table=A, lens=A, refs=A, new=A, n_seqs=4, max_pages=4, n_pages=8, ps=64):
    return L.mnemo_kv_pages_free(table, lens, refs, new, n_seqs, max_pages, n_pages, ps, None)


def fork(L, *, table=A, lens=A, refs=A, new=A, n_seqs=4, max_pages=4, n_pages=8, ps=64, kp=A, vp=A, ks=None, vs=None,
         kv_type=0, layers=2, nkv=2, hd=128, ws=A, wsb=1 << 30):
    return L.mnemo_kv_pages_fork(table, lens, refs, new, n_seqs, max_pages, kp, vp, ks, vs, kv_type, layers, n_pages,
                                 ps, nkv, hd, None, ws, wsb, None)


def compact(L, *, table=A, refs=A, n_seqs=4, max_pages=4, n_pages=8, ps=64, kp=A, vp=A, ks=None, vs=None, kv_type=0,
            layers=2, nkv=2, hd=128, ws=A, wsb=1 << 30):
    return L.mnemo_kv_pages_compact(table, refs, n_seqs, max_pages, kp, vp, ks, vs, kv_type, layers, n_pages, ps, nkv,
                                    hd, None, ws, wsb, None)


def copy(L, *, src=A, dst=A, n=2, n_pages=8, ps=64, kp=A, vp=A, ks=None, vs=None, kv_type=0, layers=2, nkv=2, hd=128):
    return L.mnemo_kv_pages_copy(src, dst, n, kp, vp, ks, vs, kv_type, layers, n_pages, ps, nkv, hd, None)


STATE = [dict(table=None), dict(refs=None), dict(n_seqs=0), dict(n_seqs=4097), dict(max_pages=0), dict(n_pages=0), dict(n_pages=(1 << 30) + 1),
         dict(ps=24), dict(max_pages=1 << 25), dict(n_seqs=4096, max_pages=1 << 19, ps=16)]
ROWS = STATE + [dict(lens=None), dict(new=None)]
MOVING = CACHE + [dict(layers=0), dict(layers=4097)]
WS = [dict(ws=None), dict(ws=A + 4), dict(wsb=16)]


@pytest.mark.parametrize("call,bad", [(extend, b) for b in ROWS] + [(free, b) for b in ROWS] +
                         [(fork, b) for b in ROWS + MOVING + WS] + [(compact, b) for b in STATE + MOVING + WS] +
                         [(copy, b) for b in MOVING + [dict(src=None), dict(dst=None), dict(n=-1), dict(n=(1 << 30) + 1)]])
def test_page_upkeep_refuses(L, call, bad, capfd):
    assert call(L, **bad) == 1
    assert f"kv_pages_{call.__name__}" in capfd.readouterr().err
    assert L.mnemo_last_error() == 1


def test_copy_of_no_pages_is_nothing(L):
    assert copy(L, n=0, src=None, dst=None) == 0


def logits(L, *, z=A, out=A, n=2, vocab=100, hist=A, hl=A, pl=A, max_hist=8, rep=A, freq=A, pres=A, ids=A, bias=A, nb=4,
           allowed=A):
    return L.mnemo_logits_process(z, out, n, vocab, hist, hl, pl, max_hist, rep, freq, pres, ids, bias, nb, allowed,
                                  None)


@pytest.mark.parametrize("bad", [dict(z=None), dict(out=None), dict(n=-1), dict(n=65536), dict(vocab=0), dict(vocab=(1 << 30) + 1), dict(hl=None),
                                 dict(pl=None), dict(rep=None), dict(freq=None), dict(pres=None), dict(max_hist=-1),
                                 dict(bias=None), dict(nb=-1)])
def test_logits_refuses(L, bad, capfd):
    assert logits(L, **bad) == 1
    assert "logits_process" in capfd.readouterr().err
    assert L.mnemo_last_error() == 1


def test_logits_of_no_rows_is_nothing(L):
    assert logits(L, n=0, z=None, out=None) == 0


def test_cache_bytes(L):
    assert L.mnemo_paged_cache_bytes(10, 64, 4, 128, 0) == 10 * 64 * 4 * 128 * 2
    assert L.mnemo_paged_cache_bytes(10, 64, 4, 128, 1) == 10 * 64 * 4 * 128
    assert L.mnemo_paged_cache_bytes(1 << 20, 128, 16, 256, 0) == (1 << 20) * 128 * 16 * 256 * 2  # past 32 bits
    assert L.mnemo_paged_cache_bytes(0, 64, 4, 128, 0) == 0


def test_wrappers_refuse_host_tensors_and_shapes(L):
    """The Python wrappers check tensors before anything is launched (CPU tensors reach no kernel)."""
    import torch

    from mnemocuda_amd import MnemoError, ops
    z = lambda *s, t=torch.float32: torch.zeros(s, dtype=t)  # noqa: E731
    i = lambda *s: z(*s, t=torch.int32)  # noqa: E731
    q, k, v, table, lens = z(2, 4, 64), z(8, 2, 16, 64, t=torch.float16), z(8, 2, 64, 16, t=torch.float16), i(2, 3), i(2)
    with pytest.raises(MnemoError, match="GPU tensor"):
        ops.paged_attention_decode(q, k, v, table, lens, z(2, 4, 64), 0.1, z(64))
    with pytest.raises(MnemoError, match="do not fit"):  # v laid out as k is
        ops.paged_attention_decode(q, k, z(8, 2, 16, 64, t=torch.float16), table, lens, z(2, 4, 64), 0.1, z(64))
    with pytest.raises(MnemoError, match="do not fit"):  # no layers
        ops.kv_pages_fork(table, lens, i(8), i(2), k, v, i(1), z(64))
    with pytest.raises(MnemoError, match="float16 or int8"):
        ops.paged_attention_decode(q, k.float(), v.float(), table, lens, z(2, 4, 64), 0.1, z(64))
    with pytest.raises(MnemoError, match="need scales"):
        ops.paged_attention_decode(q, k.to(torch.int8), v.to(torch.int8), table, lens, z(2, 4, 64), 0.1, z(64))
    with pytest.raises(MnemoError, match="GPU tensor"):
        ops.paged_attn_prep(q, z(2, 2, 64), z(2, 2, 64), None, None, 1e-6, 1e4, k, v, table, q, seq_lens=lens)
    with pytest.raises(MnemoError, match="2 dimensions"):
        ops.kv_pages_free(lens, lens, i(8), lens, 16)
    with pytest.raises(MnemoError, match="GPU tensor"):
        ops.kv_pages_extend(table, lens, i(8), lens, 16)
    with pytest.raises(MnemoError, match="differ in length"):
        ops.kv_pages_copy(i(2), i(3), z(1, 8, 2, 16, 64, t=torch.float16), z(1, 8, 2, 64, 16, t=torch.float16))
    with pytest.raises(MnemoError, match="must be .n, vocab"):
        ops.logits_process(z(2, 50), z(2, 51))
    with pytest.raises(MnemoError, match="history must be"):
        ops.logits_process(z(2, 50), z(2, 50), i(3, 4))
    with pytest.raises(MnemoError, match="GPU tensor"):
        ops.logits_process(z(2, 50), z(2, 50))



@pytest.mark.parametrize("bad", [dict(max_hist=(1 << 30) + 1), dict(max_hist=(1 << 31) - 1), dict(nb=(1 << 30) + 1),
                                 dict(nb=(1 << 31) - 1)])
def test_logits_refuses_lengths_that_its_steps_would_leave_the_range_with(L, bad, capfd):
    """The kernel walks the history 4096 entries and the biases 256 at a time in 32-bit counters."""
    assert logits(L, z=None, out=None, n=0, **{k: v for k, v in bad.items()}) == 1
    assert "logits_process" in capfd.readouterr().err
