"""Torch-tensor wrappers over the C ABI (one call = one C entry point).

Tensors must be CUDA (HIP) tensors on the current device; weights are uint8 tensors that
hold raw GGUF blocks.  Calls are enqueued on torch's current stream.  Nothing here
computes on the host: a missing library or a CPU tensor raises MnemoError.
"""
from __future__ import annotations

import torch

from .lib import MnemoError, check, load_library

TYPE_F32, TYPE_Q4K, TYPE_Q6K = 0, 12, 14
BLOCK_BYTES = {TYPE_Q4K: 144, TYPE_Q6K: 210}


def _dev(t: torch.Tensor, name: str, dtype: torch.dtype | None = None) -> int:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise MnemoError(f"{name} must be a GPU tensor")
    if dtype is not None and t.dtype != dtype:
        raise MnemoError(f"{name} must be {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise MnemoError(f"{name} must be contiguous")
    return t.data_ptr()


def _stream() -> int:
    # torch.cuda.current_stream().cuda_stream without the Stream object (2.8 us a call)
    return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())


def row_bytes(type_id: int, n_cols: int) -> int:
    if type_id == TYPE_F32:
        return 4 * n_cols
    return (n_cols + 255) // 256 * BLOCK_BYTES[type_id]


def _check_w(w: torch.Tensor, type_id: int, rows: int, cols: int, name: str = "W") -> int:
    p = _dev(w, name)
    need = rows * row_bytes(type_id, cols)
    if w.numel() * w.element_size() < need:
        raise MnemoError(f"{name}: {w.numel() * w.element_size()} bytes < {need} needed for "
                         f"{rows}x{cols} type {type_id}")
    return p


def _check_rc(lib, rc: int, what: str) -> None:
    """Raise for a non-zero return code; also consumes the library's per-thread error slot
    so that a later call does not report this error again."""
    lib.mnemo_last_error()
    if rc:
        raise MnemoError(f"{what}: error {rc}: {lib.mnemo_last_error_string().decode()}")


def init() -> None:
    lib = load_library()
    lib.cuda_kernels_init()
    check(lib, "cuda_kernels_init")


def matvec(w, x, y, rows, cols, type_id):
    """Reference dispatcher matvec() (forward.c:160-173) via mnemo_matvec."""
    lib = load_library()
    _check_w(w, type_id, rows, cols)
    e = lib.mnemo_matvec(w.data_ptr(), _dev(x, "x", torch.float32), _dev(y, "y", torch.float32),
                         rows, cols, type_id, _stream())
    _check_rc(lib, e, "mnemo_matvec")


def matvec_q4k(w, x, y, rows, cols):
    lib = load_library()
    lib.cuda_matvec_q4k(_check_w(w, TYPE_Q4K, rows, cols), _dev(x, "x", torch.float32),
                        _dev(y, "y", torch.float32), rows, cols, _stream())
    check(lib, "cuda_matvec_q4k")


def matvec_q6k(w, x, y, rows, cols):
    lib = load_library()
    lib.cuda_matvec_q6k(_check_w(w, TYPE_Q6K, rows, cols), _dev(x, "x", torch.float32),
                        _dev(y, "y", torch.float32), rows, cols, _stream())
    check(lib, "cuda_matvec_q6k")


def matvec_q4k_add(w, x, residual, y, rows, cols):
    lib = load_library()
    lib.cuda_matvec_q4k_add(_check_w(w, TYPE_Q4K, rows, cols), _dev(x, "x", torch.float32),
                            _dev(residual, "residual", torch.float32), _dev(y, "y", torch.float32),
                            rows, cols, _stream())
    check(lib, "cuda_matvec_q4k_add")


def matvec_q4k_qkv(wq, wk, wv, x, q, k, v, q_rows, kv_rows, cols):
    lib = load_library()
    lib.cuda_matvec_q4k_qkv(_check_w(wq, TYPE_Q4K, q_rows, cols, "wq"),
                            _check_w(wk, TYPE_Q4K, kv_rows, cols, "wk"),
                            _check_w(wv, TYPE_Q4K, kv_rows, cols, "wv"), _dev(x, "x", torch.float32),
                            _dev(q, "q", torch.float32), _dev(k, "k", torch.float32),
                            _dev(v, "v", torch.float32), q_rows, kv_rows, cols, _stream())
    check(lib, "cuda_matvec_q4k_qkv")


def matvec_q4k_dual(wa, wb, x, ya, yb, rows, cols):
    lib = load_library()
    lib.cuda_matvec_q4k_dual(_check_w(wa, TYPE_Q4K, rows, cols, "wa"), _check_w(wb, TYPE_Q4K, rows, cols, "wb"),
                             _dev(x, "x", torch.float32), _dev(ya, "ya", torch.float32),
                             _dev(yb, "yb", torch.float32), rows, cols, _stream())
    check(lib, "cuda_matvec_q4k_dual")


def matvec_dual(wa, ta, wb, tb, x, ya, yb, rows, cols):
    lib = load_library()
    lib.mnemo_matvec_dual(_check_w(wa, ta, rows, cols, "wa"), ta, _check_w(wb, tb, rows, cols, "wb"), tb,
                          _dev(x, "x", torch.float32), _dev(ya, "ya", torch.float32),
                          _dev(yb, "yb", torch.float32), rows, cols, _stream())
    check(lib, "mnemo_matvec_dual")


def matvec_qkv(wq, tq, wk, tk, wv, tv, x, oq, ok, ov, q_rows, kv_rows, cols):
    lib = load_library()
    lib.mnemo_matvec_qkv(_check_w(wq, tq, q_rows, cols, "wq"), tq, _check_w(wk, tk, kv_rows, cols, "wk"), tk,
                         _check_w(wv, tv, kv_rows, cols, "wv"), tv, _dev(x, "x", torch.float32),
                         _dev(oq, "oq", torch.float32), _dev(ok, "ok", torch.float32),
                         _dev(ov, "ov", torch.float32), q_rows, kv_rows, cols, _stream())
    check(lib, "mnemo_matvec_qkv")


def matvec_qkv_rmsnorm(wq, tq, wk, tk, wv, tv, x, norm_w, eps, oq, ok, ov, q_rows, kv_rows, cols):
    """matvec_qkv of rms_norm(x) * norm_w, the norm computed inside the projection launch."""
    lib = load_library()
    if x.numel() < cols or norm_w.numel() < cols:
        raise MnemoError("matvec_qkv_rmsnorm: x or norm_w too small")
    lib.mnemo_matvec_qkv_rmsnorm(_check_w(wq, tq, q_rows, cols, "wq"), tq, _check_w(wk, tk, kv_rows, cols, "wk"), tk,
                                 _check_w(wv, tv, kv_rows, cols, "wv"), tv, _dev(x, "x", torch.float32),
                                 _dev(norm_w, "norm_w", torch.float32), float(eps), _dev(oq, "oq", torch.float32),
                                 _dev(ok, "ok", torch.float32), _dev(ov, "ov", torch.float32), q_rows, kv_rows, cols,
                                 _stream())
    check(lib, "mnemo_matvec_qkv_rmsnorm")


def matvec_q4k_scaled_add(w, x, y, rows, cols, scale):
    lib = load_library()
    lib.cuda_matvec_q4k_scaled_add(_check_w(w, TYPE_Q4K, rows, cols), _dev(x, "x", torch.float32),
                                   _dev(y, "y", torch.float32), rows, cols, float(scale), _stream())
    check(lib, "cuda_matvec_q4k_scaled_add")


def matvec_q6k_scaled_add(w, x, y, rows, cols, scale):
    lib = load_library()
    lib.mnemo_matvec_q6k_scaled_add(_check_w(w, TYPE_Q6K, rows, cols), _dev(x, "x", torch.float32),
                                    _dev(y, "y", torch.float32), rows, cols, float(scale), _stream())
    check(lib, "mnemo_matvec_q6k_scaled_add")


def matvec_swiglu_scaled_add(w, type_id, gate, up, y, rows, cols, scale):
    lib = load_library()
    lib.mnemo_matvec_swiglu_scaled_add(_check_w(w, type_id, rows, cols), type_id,
                                       _dev(gate, "gate", torch.float32), _dev(up, "up", torch.float32),
                                       _dev(y, "y", torch.float32), rows, cols, float(scale), _stream())
    check(lib, "mnemo_matvec_swiglu_scaled_add")


def matvec_f32(w, x, y, rows, cols):
    lib = load_library()
    lib.cuda_matvec_f32(_dev(w, "W", torch.float32), _dev(x, "x", torch.float32), _dev(y, "y", torch.float32),
                        rows, cols, _stream())
    check(lib, "cuda_matvec_f32")


def topk_softmax(scores, idx, w, n_experts, k):
    lib = load_library()
    lib.cuda_topk_softmax(_dev(scores, "scores", torch.float32), _dev(idx, "idx", torch.int32),
                          _dev(w, "w", torch.float32), n_experts, k, _stream())
    check(lib, "cuda_topk_softmax")


def swiglu(g, u, out, n):
    lib = load_library()
    lib.cuda_swiglu(_dev(g, "g", torch.float32), _dev(u, "u", torch.float32), _dev(out, "out", torch.float32),
                    n, _stream())
    check(lib, "cuda_swiglu")


def scaled_add(out, x, scale, n):
    lib = load_library()
    lib.cuda_scaled_add(_dev(out, "out", torch.float32), _dev(x, "x", torch.float32), float(scale), n, _stream())
    check(lib, "cuda_scaled_add")


def quantize_q8_1(src, dst, K, N):
    lib = load_library()
    if dst.numel() * dst.element_size() < N * (K // 128) * 144:
        raise MnemoError("quantize_q8_1: dst too small")
    lib.cuda_quantize_mmq_q8_1(_dev(src, "src", torch.float32), _dev(dst, "dst"), K, N, _stream())
    check(lib, "cuda_quantize_mmq_q8_1")


def gemm(w, type_id, act, out, M, K, N):
    lib = load_library()
    _check_w(w, type_id, M, K)
    if act.numel() * act.element_size() < N * (K // 128) * 144:
        raise MnemoError("gemm: activation buffer too small")
    if out.numel() < M * N:
        raise MnemoError("gemm: output too small")
    fn = lib.cuda_gemm_q4k if type_id == TYPE_Q4K else lib.mnemo_gemm_q6k
    fn(w.data_ptr(), _dev(act, "act"), _dev(out, "out", torch.float32), M, K, N, _stream())
    check(lib, "gemm")


def expert_fwd(expert, gate_sz, up_sz, H, EFF, down_type, weight, x, gate_buf, up_buf, moe_out):
    lib = load_library()
    e = lib.mnemo_expert_fwd(_dev(expert, "expert"), gate_sz, up_sz, H, EFF, down_type, float(weight),
                             _dev(x, "x", torch.float32), _dev(gate_buf, "gate_buf", torch.float32),
                             _dev(up_buf, "up_buf", torch.float32), _dev(moe_out, "moe_out", torch.float32),
                             _stream())
    _check_rc(lib, e, "mnemo_expert_fwd")


def moe_prefill_workspace_bytes(T, hidden, eff, n_experts, k) -> int:
    return int(load_library().mnemo_moe_prefill_workspace_bytes(T, hidden, eff, n_experts, k))


def moe_prefill(experts, expert_stride, gate_off, up_off, down_off, down_type, x, topk_idx, topk_w,
                T, hidden, eff, n_experts, k, workspace, out):
    """Grouped-expert prefill: out[t] += sum_slot w * down(silu(gate x_t) * up x_t)."""
    lib = load_library()
    need = expert_stride * (n_experts - 1) + down_off + row_bytes(down_type, eff) * hidden \
        if down_type in BLOCK_BYTES else 0  # an unknown type is reported by the library
    if experts.numel() * experts.element_size() < need:
        raise MnemoError("moe_prefill: expert table too small")
    if topk_idx.numel() < T * k or topk_w.numel() < T * k or x.numel() < T * hidden or out.numel() < T * hidden:
        raise MnemoError("moe_prefill: routing, x or out too small")
    e = lib.mnemo_moe_prefill(_dev(experts, "experts"), expert_stride, gate_off, up_off, down_off, down_type,
                              _dev(x, "x", torch.float32), _dev(topk_idx, "topk_idx", torch.int32),
                              _dev(topk_w, "topk_w", torch.float32), T, hidden, eff, n_experts, k,
                              _dev(workspace, "workspace"), workspace.numel() * workspace.element_size(),
                              _dev(out, "out", torch.float32), _stream())
    _check_rc(lib, e, "mnemo_moe_prefill")


def moe_decode_workspace_bytes(hidden, eff, n_experts, k) -> int:
    return int(load_library().mnemo_moe_decode_workspace_bytes(hidden, eff, n_experts, k))


def moe_decode(router_w, experts, expert_stride, gate_off, up_off, down_off, down_type, x, hidden, eff,
               n_experts, k, workspace, out, topk_idx=None, topk_w=None):
    """One token's MoE block with device-side dispatch: out += sum_slot w * expert(x)."""
    lib = load_library()
    need = expert_stride * (n_experts - 1) + down_off + row_bytes(down_type, eff) * hidden \
        if down_type in BLOCK_BYTES else 0
    if experts.numel() * experts.element_size() < need:
        raise MnemoError("moe_decode: expert table too small")
    if router_w.numel() < n_experts * hidden or x.numel() < hidden or out.numel() < hidden:
        raise MnemoError("moe_decode: router, x or out too small")
    e = lib.mnemo_moe_decode(_dev(router_w, "router_w", torch.float32), _dev(experts, "experts"), expert_stride,
                             gate_off, up_off, down_off, down_type, _dev(x, "x", torch.float32), hidden, eff,
                             n_experts, k, _dev(workspace, "workspace"),
                             workspace.numel() * workspace.element_size(), _dev(out, "out", torch.float32),
                             None if topk_idx is None else _dev(topk_idx, "topk_idx", torch.int32),
                             None if topk_w is None else _dev(topk_w, "topk_w", torch.float32), _stream())
    _check_rc(lib, e, "mnemo_moe_decode")


def moe_decode_rmsnorm(router_w, experts, expert_stride, gate_off, up_off, down_off, down_type, x, norm_w, eps,
                       hidden, eff, n_experts, k, workspace, out, topk_idx=None, topk_w=None):
    """moe_decode of rms_norm(x) * norm_w with the norm computed by the router and gate/up
    launches; x is the raw hidden state and may be out itself."""
    lib = load_library()
    need = expert_stride * (n_experts - 1) + down_off + row_bytes(down_type, eff) * hidden \
        if down_type in BLOCK_BYTES else 0
    if experts.numel() * experts.element_size() < need:
        raise MnemoError("moe_decode_rmsnorm: expert table too small")
    if router_w.numel() < n_experts * hidden or x.numel() < hidden or out.numel() < hidden \
            or norm_w.numel() < hidden:
        raise MnemoError("moe_decode_rmsnorm: router, x, norm_w or out too small")
    e = lib.mnemo_moe_decode_rmsnorm(
        _dev(router_w, "router_w", torch.float32), _dev(experts, "experts"), expert_stride, gate_off, up_off,
        down_off, down_type, _dev(x, "x", torch.float32), _dev(norm_w, "norm_w", torch.float32), float(eps), hidden,
        eff, n_experts, k, _dev(workspace, "workspace"), workspace.numel() * workspace.element_size(),
        _dev(out, "out", torch.float32), None if topk_idx is None else _dev(topk_idx, "topk_idx", torch.int32),
        None if topk_w is None else _dev(topk_w, "topk_w", torch.float32), _stream())
    _check_rc(lib, e, "mnemo_moe_decode_rmsnorm")


def sample_token(logits, vocab, temperature, top_p, seed, out):
    """Next token from logits[vocab] (greedy for temperature <= 0, else top-p) into out[0]."""
    lib = load_library()
    if logits.numel() < vocab or out.numel() < 1:
        raise MnemoError("sample_token: logits or out too small")
    lib.cuda_sample_token(_dev(logits, "logits", torch.float32), vocab, float(temperature), float(top_p),
                          int(seed) & 0xFFFFFFFFFFFFFFFF, _dev(out, "out", torch.int32), _stream())
    check(lib, "cuda_sample_token")


def sample_workspace_bytes() -> int:
    return int(load_library().mnemo_sample_workspace_bytes())


def sample_token_ws(logits, vocab, temperature, top_p, seed, workspace, out):
    """sample_token with the vocabulary scan over 64 workgroups (workspace of
    sample_workspace_bytes() bytes)."""
    lib = load_library()
    if logits.numel() < vocab or out.numel() < 1:
        raise MnemoError("sample_token_ws: logits or out too small")
    rc = lib.mnemo_sample_token_ws(_dev(logits, "logits", torch.float32), vocab, float(temperature), float(top_p),
                                   int(seed) & 0xFFFFFFFFFFFFFFFF, _dev(workspace, "workspace"),
                                   workspace.numel() * workspace.element_size(), _dev(out, "out", torch.int32),
                                   _stream())
    _check_rc(lib, rc, "mnemo_sample_token_ws")


# ---------------------------------------------------------------- attention chain
F32 = torch.float32


def _opt(t, name, dtype=None) -> int | None:
    return None if t is None else _dev(t, name, dtype)


def rms_norm(x, w, out, eps: float, residual=None):
    """out = x * rsqrt(mean(x^2) + eps) * w (cuda_rms_norm); with residual, also residual = x
    (cuda_rms_norm_residual)."""
    lib = load_library()
    n = x.numel()
    if w.numel() < n or out.numel() < n or (residual is not None and residual.numel() < n):
        raise MnemoError("rms_norm: buffers too small")
    if residual is None:
        lib.cuda_rms_norm(_dev(x, "x", F32), _dev(w, "w", F32), _dev(out, "out", F32), n, float(eps), _stream())
        check(lib, "cuda_rms_norm")
    else:
        lib.cuda_rms_norm_residual(_dev(x, "x", F32), _dev(w, "w", F32), _dev(out, "out", F32),
                                   _dev(residual, "residual", F32), n, float(eps), _stream())
        check(lib, "cuda_rms_norm_residual")


def rms_norm_batched(x, w, out, head_dim: int, eps: float):
    lib = load_library()
    lib.cuda_rms_norm_batched(_dev(x, "x", F32), _dev(w, "w", F32), _dev(out, "out", F32), head_dim,
                              x.numel() // head_dim, float(eps), _stream())
    check(lib, "cuda_rms_norm_batched")


def rms_norm_qk(q, k, qw, kw, head_dim: int, eps: float):
    lib = load_library()
    lib.cuda_rms_norm_qk(_dev(q, "q", F32), _dev(k, "k", F32), _dev(qw, "qw", F32), _dev(kw, "kw", F32), head_dim,
                         q.numel() // head_dim, k.numel() // head_dim, float(eps), _stream())
    check(lib, "cuda_rms_norm_qk")


def residual_add(a, b, out):
    lib = load_library()
    lib.cuda_residual_add(_dev(a, "a", F32), _dev(b, "b", F32), _dev(out, "out", F32), a.numel(), _stream())
    check(lib, "cuda_residual_add")


def rope(q, k, head_dim: int, pos: int, theta: float):
    lib = load_library()
    lib.cuda_rope(_dev(q, "q", F32), _dev(k, "k", F32), head_dim, int(pos), float(theta), q.numel() // head_dim,
                  k.numel() // head_dim, _stream())
    check(lib, "cuda_rope")


def f32_to_f16_dual(a, b, oa, ob):
    lib = load_library()
    lib.cuda_f32_to_f16_dual(_dev(a, "a", F32), _dev(b, "b", F32), _dev(oa, "oa", torch.float16),
                             _dev(ob, "ob", torch.float16), a.numel(), _stream())
    check(lib, "cuda_f32_to_f16_dual")


def f32_to_int8_kv_dual(k, v, ok, ov, ks, vs, head_dim: int):
    lib = load_library()
    lib.cuda_f32_to_int8_kv_dual(_dev(k, "k", F32), _dev(v, "v", F32), _dev(ok, "ok", torch.int8),
                                 _dev(ov, "ov", torch.int8), _dev(ks, "ks", F32), _dev(vs, "vs", F32), head_dim,
                                 k.numel() // head_dim, _stream())
    check(lib, "cuda_f32_to_int8_kv_dual")


def attention(q, kc, vc, out, n_heads: int, head_dim: int, n_kv_heads: int, seq_len: int, scale: float,
              ks=None, vs=None):
    """cuda_attention_f16kv (kc/vc float16) or cuda_attention_int8kv (int8 with scales)."""
    lib = load_library()
    gqa = n_heads // n_kv_heads
    if kc.dtype == torch.float16:
        lib.cuda_attention_f16kv(_dev(q, "q", F32), _dev(kc, "kc"), _dev(vc, "vc"), _dev(out, "out", F32), n_heads,
                                 head_dim, n_kv_heads, int(seq_len), gqa, float(scale), _stream())
        check(lib, "cuda_attention_f16kv")
    else:
        lib.cuda_attention_int8kv(_dev(q, "q", F32), _dev(kc, "kc", torch.int8), _dev(vc, "vc", torch.int8),
                                  _dev(ks, "ks", F32), _dev(vs, "vs", F32), _dev(out, "out", F32), n_heads, head_dim,
                                  n_kv_heads, int(seq_len), gqa, float(scale), _stream())
        check(lib, "cuda_attention_int8kv")


def attention_reserve(n_slots: int) -> None:
    """mnemo_attention_reserve: at least n_slots free workspace slots for captured
    cuda_attention_* calls on the current GPU (allocates; not under capture)."""
    lib = load_library()
    _check_rc(lib, lib.mnemo_attention_reserve(int(n_slots)), "mnemo_attention_reserve")


def attn_prep(q, k, v, qw, kw, head_dim: int, eps: float, theta: float, pos_dev, kc, vc, ks=None, vs=None,
              v_layout: int = 0):
    """QK norm (when qw/kw are given) + RoPE + KV store at cache row pos_dev[0], one launch
    (v_layout 1: V in the blocked layout of attention_decode)."""
    lib = load_library()
    kv_type = 0 if kc.dtype == torch.float16 else 1
    rc = lib.mnemo_attn_prep(_dev(q, "q", F32), _dev(k, "k", F32), _dev(v, "v", F32), _opt(qw, "qw", F32),
                             _opt(kw, "kw", F32), head_dim, q.numel() // head_dim, k.numel() // head_dim, float(eps),
                             float(theta), _dev(pos_dev, "pos_dev", torch.int32), _dev(kc, "kc"), _dev(vc, "vc"),
                             _opt(ks, "ks", F32), _opt(vs, "vs", F32), kv_type, int(v_layout), _stream())
    _check_rc(lib, rc, "mnemo_attn_prep")


def attention_dev(q, kc, vc, out, n_heads: int, head_dim: int, n_kv_heads: int, pos_dev, scale: float,
                  ks=None, vs=None):
    """attention over positions 0..pos_dev[0] (length read on the device)."""
    lib = load_library()
    kv_type = 0 if kc.dtype == torch.float16 else 1
    rc = lib.mnemo_attention(_dev(q, "q", F32), _dev(kc, "kc"), _dev(vc, "vc"), _opt(ks, "ks", F32),
                             _opt(vs, "vs", F32), kv_type, _dev(out, "out", F32), n_heads, head_dim, n_kv_heads,
                             _dev(pos_dev, "pos_dev", torch.int32), float(scale), _stream())
    _check_rc(lib, rc, "mnemo_attention")


def attention_decode_workspace_bytes(n_kv_heads: int, max_ctx: int) -> int:
    return int(load_library().mnemo_attention_decode_workspace_bytes(n_kv_heads, max_ctx))


def v_cache_bytes(n_kv_heads: int, head_dim: int, max_ctx: int, kv_type: int, v_layout: int) -> int:
    return int(load_library().mnemo_v_cache_bytes(n_kv_heads, head_dim, max_ctx, kv_type, v_layout))


def attention_decode(q, kc, vc, out, n_heads: int, head_dim: int, n_kv_heads: int, max_ctx: int, pos_dev,
                     scale: float, ws, ks=None, vs=None, v_layout: int = 0):
    """GQA-batched split-position attention over positions 0..pos_dev[0] (matrix cores)."""
    lib = load_library()
    kv_type = 0 if kc.dtype == torch.float16 else 1
    rc = lib.mnemo_attention_decode(_dev(q, "q", F32), _dev(kc, "kc"), _dev(vc, "vc"), _opt(ks, "ks", F32),
                                    _opt(vs, "vs", F32), kv_type, int(v_layout), _dev(out, "out", F32), n_heads,
                                    head_dim,
                                    n_kv_heads, int(max_ctx), _dev(pos_dev, "pos_dev", torch.int32), float(scale),
                                    _dev(ws, "ws"), ws.numel() * ws.element_size(), _stream())
    _check_rc(lib, rc, "mnemo_attention_decode")


def attention_decode_prep(q, k, v, qw, kw, eps: float, theta: float, kc, vc, out, n_heads: int, head_dim: int,
                          n_kv_heads: int, max_ctx: int, pos_dev, scale: float, ws, ks=None, vs=None,
                          v_layout: int = 0):
    """attn_prep + attention_decode in the same two launches: q, k, v raw (left unchanged),
    the new K / V rows stored at pos_dev[0], attention over 0..pos_dev[0]."""
    lib = load_library()
    kv_type = 0 if kc.dtype == torch.float16 else 1
    if q.numel() < n_heads * head_dim or k.numel() < n_kv_heads * head_dim or v.numel() < n_kv_heads * head_dim:
        raise MnemoError("attention_decode_prep: q, k or v too small")
    rc = lib.mnemo_attention_decode_prep(
        _dev(q, "q", F32), _dev(k, "k", F32), _dev(v, "v", F32), _opt(qw, "qw", F32), _opt(kw, "kw", F32),
        float(eps), float(theta), _dev(kc, "kc"), _dev(vc, "vc"), _opt(ks, "ks", F32), _opt(vs, "vs", F32), kv_type,
        int(v_layout), _dev(out, "out", F32), n_heads, head_dim, n_kv_heads, int(max_ctx),
        _dev(pos_dev, "pos_dev", torch.int32), float(scale), _dev(ws, "ws"), ws.numel() * ws.element_size(),
        _stream())
    _check_rc(lib, rc, "mnemo_attention_decode_prep")


# ---------------------------------------------------------------- embedding
def embedding_lookup(table, type_id: int, token_dev, n_vocab: int, out, hidden: int):
    """out[:hidden] = dequantised row token_dev[0] of table (F32 / Q4_K / Q6_K).  table is a
    GPU tensor or a raw device pointer (int)."""
    lib = load_library()
    tp = table if isinstance(table, int) else _dev(table, "table")
    rc = lib.mnemo_embedding_lookup(tp, int(type_id), _dev(token_dev, "token_dev", torch.int32), int(n_vocab),
                                    _dev(out, "out", F32), int(hidden), _stream())
    _check_rc(lib, rc, "mnemo_embedding_lookup")


def embedding_lookup_q4k(table, out, token_id: int, hidden: int, row_bytes: int):
    """cuda_embedding_lookup_q4k (reference signature)."""
    lib = load_library()
    tp = table if isinstance(table, int) else _dev(table, "table")
    lib.cuda_embedding_lookup_q4k(tp, _dev(out, "out", F32), int(token_id), int(hidden), int(row_bytes), _stream())
    check(lib, "cuda_embedding_lookup_q4k")


# ---------------------------------------------------------------- several sequences in one paged cache
I32 = torch.int32


def paged_cache_bytes(n_pages: int, page_size: int, n_kv_heads: int, head_dim: int, kv_type: int) -> int:
    return int(load_library().mnemo_paged_cache_bytes(n_pages, page_size, n_kv_heads, head_dim, kv_type))


_gpus = 0  # visible GPUs, asked for once


def _arg(t, name: str, dtype: torch.dtype | None = None, n: int = 0) -> int:
    """The address of a contiguous tensor on the current GPU with at least n elements."""
    try:
        # the order of the checks is that of their use; each costs ~0.06 us, a call has up to 20 tensors
        if t.is_cuda and (dtype is None or t.dtype is dtype) and t.is_contiguous() and (not n or t.numel() >= n):
            if _gpus == 1 or t.get_device() == _current_gpu():
                return t.data_ptr()
            raise MnemoError(f"{name} must be on the current GPU")
    except AttributeError:
        pass
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise MnemoError(f"{name} must be a GPU tensor")
    if dtype is not None and t.dtype != dtype:
        raise MnemoError(f"{name} must be {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise MnemoError(f"{name} must be contiguous")
    raise MnemoError(f"{name}: {t.numel()} elements < {n}")


def _current_gpu() -> int:
    global _gpus
    _gpus = torch.cuda.device_count()
    return torch._C._cuda_getDevice()


def _opt_arg(t, name: str, dtype: torch.dtype | None = None, n: int = 0) -> int | None:
    return None if t is None else _arg(t, name, dtype, n)


def _pages(k, v, ks, vs, layers: bool):
    """The arguments (pointers, kv_type) and shape (n_layers, n_pages, n_kv_heads, page_size, head_dim) of cache
    pages k [..., n_kv_heads, page_size, head_dim] and v [..., n_kv_heads, head_dim, page_size]."""
    try:
        if layers:
            L, n, h, p, d = k.shape
            fits = v.shape == (L, n, h, d, p)
        else:
            n, h, p, d = k.shape
            L, fits = 1, v.shape == (n, h, d, p)
    except ValueError:
        fits = False
    if not fits:
        raise MnemoError(f"pages: k {tuple(k.shape)} and v {tuple(v.shape)} do not fit ({5 if layers else 4} dimensions, "
                         "v transposed)")
    if k.dtype is torch.float16:
        return (_arg(k, "k_pages"), _arg(v, "v_pages", torch.float16), None, None, 0), (L, n, h, p, d)
    if k.dtype is not torch.int8:
        raise MnemoError(f"pages must be float16 or int8, got {k.dtype}")
    if ks is None or vs is None:
        raise MnemoError("int8 pages need scales")
    rows = L * n * h * p
    return (_arg(k, "k_pages"), _arg(v, "v_pages", torch.int8), _arg(ks, "k_scales", F32, rows),
            _arg(vs, "v_scales", F32, rows), 1), (L, n, h, p, d)


def _rows(table):
    """(address, n_seqs, max_pages) of a block table."""
    shape = table.shape
    if len(shape) != 2:
        raise MnemoError(f"block_table must have 2 dimensions, got {len(shape)}")
    return _arg(table, "block_table", I32), shape[0], shape[1]


def paged_attn_prep(q, k, v, qw, kw, eps: float, theta: float, k_pages, v_pages, block_table, q_out, positions=None,
                    seq_ids=None, ks=None, vs=None, seq_lens=None):
    """QK norm (when qw/kw are given) + RoPE of the new tokens q [T, n_heads, head_dim] (into q_out, which may be q)
    and k [T, n_kv_heads, head_dim], and the store of k and v into the pages.  Token t is position positions[t] of
    row seq_ids[t] of the block table (with seq_lens: not stored unless it lies before the row's end, as in a row that
    could not be extended); without them it is the last position of row t (seq_lens[t] - 1), also if the row did not
    grow."""
    lib = load_library()
    ptrs, (_, n_pages, nkv, ps, hd) = _pages(k_pages, v_pages, ks, vs, False)
    table, n_seqs, max_pages = _rows(block_table)
    shape = q.shape
    if len(shape) != 3 or shape[2] != hd or k.shape != (shape[0], nkv, hd) or v.shape != k.shape or q_out.shape != shape:
        raise MnemoError("paged_attn_prep: q, k, v and q_out must be [T, heads, head_dim]")
    T, nh = shape[0], shape[1]
    rc = lib.mnemo_paged_attn_prep(
        _arg(q, "q", F32), _arg(k, "k", F32), _arg(v, "v", F32), _opt_arg(qw, "qw", F32, hd),
        _opt_arg(kw, "kw", F32, hd), float(eps), float(theta), T, nh, hd, nkv,
        _opt_arg(positions, "positions", I32, T), _opt_arg(seq_ids, "seq_ids", I32, T), table,
        _opt_arg(seq_lens, "seq_lens", I32, n_seqs), n_seqs, max_pages, *ptrs, n_pages, ps, _arg(q_out, "q_out", F32),
        _stream())
    _check_rc(lib, rc, "mnemo_paged_attn_prep")


def paged_attention_workspace_bytes(n_heads: int, n_kv_heads: int, head_dim: int) -> int:
    return int(load_library().mnemo_paged_attention_workspace_bytes(n_heads, n_kv_heads, head_dim))


def paged_attention_decode(q, k_pages, v_pages, block_table, seq_lens, out, scale: float, ws, ks=None, vs=None):
    """out[s] = attention of q[s] [n_heads, head_dim] over the positions 0..seq_lens[s]-1 that row s of the block
    table holds (zeros for an empty row)."""
    lib = load_library()
    ptrs, (_, n_pages, nkv, ps, hd) = _pages(k_pages, v_pages, ks, vs, False)
    table, n_seqs, max_pages = _rows(block_table)
    shape = q.shape
    if len(shape) != 3 or shape[0] != n_seqs or shape[2] != hd or out.shape != shape:
        raise MnemoError("paged_attention_decode: q and out must be [n_seqs, n_heads, head_dim]")
    rc = lib.mnemo_paged_attention_decode(
        _arg(q, "q", F32), *ptrs, _arg(out, "out", F32), n_seqs, shape[1], hd, nkv, n_pages, ps, table, max_pages,
        _arg(seq_lens, "seq_lens", I32, n_seqs), float(scale), _arg(ws, "ws"), ws.numel() * ws.element_size(),
        _stream())
    _check_rc(lib, rc, "mnemo_paged_attention_decode")


def kv_pages_extend(block_table, seq_lens, page_refs, new_lens, page_size: int, status=None):
    """Gives pages to every row with new_lens > seq_lens; status[0] = rows that could not be served."""
    lib = load_library()
    table, n_seqs, max_pages = _rows(block_table)
    rc = lib.mnemo_kv_pages_extend(table, _arg(seq_lens, "seq_lens", I32, n_seqs), _arg(page_refs, "page_refs", I32),
                                   _arg(new_lens, "new_lens", I32, n_seqs), n_seqs, max_pages, page_refs.numel(),
                                   int(page_size), _opt_arg(status, "status", I32, 1), _stream())
    _check_rc(lib, rc, "mnemo_kv_pages_extend")


def kv_pages_free(block_table, seq_lens, page_refs, gone, page_size: int):
    """Drops the pages of every row with gone != 0."""
    lib = load_library()
    table, n_seqs, max_pages = _rows(block_table)
    rc = lib.mnemo_kv_pages_free(table, _arg(seq_lens, "seq_lens", I32, n_seqs), _arg(page_refs, "page_refs", I32),
                                 _arg(gone, "gone", I32, n_seqs), n_seqs, max_pages, page_refs.numel(),
                                 int(page_size), _stream())
    _check_rc(lib, rc, "mnemo_kv_pages_free")


def kv_pages_workspace_bytes(n_seqs: int, n_pages: int) -> int:
    return int(load_library().mnemo_kv_pages_workspace_bytes(n_seqs, n_pages))


def kv_pages_fork(block_table, seq_lens, page_refs, parents, k_pages, v_pages, status, ws, ks=None, vs=None):
    """Every empty row with parents >= 0 becomes a copy of that row: full pages shared, a partly filled last page
    copied in all layers of k_pages / v_pages [n_layers, n_pages, ...]; status[0] = rows that could not be served."""
    lib = load_library()
    ptrs, (n_layers, n_pages, nkv, ps, hd) = _pages(k_pages, v_pages, ks, vs, True)
    table, n_seqs, max_pages = _rows(block_table)
    rc = lib.mnemo_kv_pages_fork(table, _arg(seq_lens, "seq_lens", I32, n_seqs),
                                 _arg(page_refs, "page_refs", I32, n_pages), _arg(parents, "parents", I32, n_seqs),
                                 n_seqs, max_pages, *ptrs, n_layers, n_pages, ps, nkv, hd,
                                 _opt_arg(status, "status", I32, 1), _arg(ws, "ws"), ws.numel() * ws.element_size(),
                                 _stream())
    _check_rc(lib, rc, "mnemo_kv_pages_fork")


def kv_pages_compact(block_table, page_refs, k_pages, v_pages, n_live, ws, ks=None, vs=None):
    """Moves the pages in use to the front of the pool, in all layers; n_live[0] = their number."""
    lib = load_library()
    ptrs, (n_layers, n_pages, nkv, ps, hd) = _pages(k_pages, v_pages, ks, vs, True)
    table, n_seqs, max_pages = _rows(block_table)
    rc = lib.mnemo_kv_pages_compact(table, _arg(page_refs, "page_refs", I32, n_pages), n_seqs, max_pages, *ptrs,
                                    n_layers, n_pages, ps, nkv, hd, _opt_arg(n_live, "n_live", I32, 1),
                                    _arg(ws, "ws"), ws.numel() * ws.element_size(), _stream())
    _check_rc(lib, rc, "mnemo_kv_pages_compact")


def kv_pages_copy(src, dst, k_pages, v_pages, ks=None, vs=None):
    """Copies page src[i] to page dst[i] in all layers (int32 device tensors; destinations distinct, no source)."""
    lib = load_library()
    if src.numel() != dst.numel():
        raise MnemoError("kv_pages_copy: src and dst differ in length")
    ptrs, (n_layers, n_pages, nkv, ps, hd) = _pages(k_pages, v_pages, ks, vs, True)
    rc = lib.mnemo_kv_pages_copy(_arg(src, "src", I32), _arg(dst, "dst", I32), src.numel(), *ptrs, n_layers, n_pages,
                                 ps, nkv, hd, _stream())
    _check_rc(lib, rc, "mnemo_kv_pages_copy")


# ---------------------------------------------------------------- logits before sampling
def logits_process(logits, out, history=None, history_lens=None, prompt_lens=None, repetition=None, frequency=None,
                   presence=None, bias_ids=None, bias=None, allowed=None):
    """Repetition, frequency and presence penalties over each row's history [n, max_history], biases of single
    tokens [n, n_bias] and a mask of allowed tokens (int32 bit words [n, ceil(vocab / 32)]) applied to
    logits [n, vocab] into out (which may be logits)."""
    lib = load_library()
    if logits.dim() != 2 or out.shape != logits.shape:
        raise MnemoError("logits_process: logits and out must be [n, vocab]")
    n, vocab = logits.shape
    h = (None, None, None, 0, None, None, None)
    if history is not None:
        if history.dim() != 2 or history.shape[0] != n:
            raise MnemoError("logits_process: history must be [n, max_history]")
        h = (_arg(history, "history", I32), _arg(history_lens, "history_lens", I32, n),
             _arg(prompt_lens, "prompt_lens", I32, n), history.shape[1], _arg(repetition, "repetition", F32, n),
             _arg(frequency, "frequency", F32, n), _arg(presence, "presence", F32, n))
    b = (None, None, 0)
    if bias_ids is not None:
        if bias is None or bias_ids.dim() != 2 or bias_ids.shape[0] != n or bias.shape != bias_ids.shape:
            raise MnemoError("logits_process: bias_ids and bias must be [n, n_bias]")
        b = (_arg(bias_ids, "bias_ids", I32), _arg(bias, "bias", F32), bias_ids.shape[1])
    rc = lib.mnemo_logits_process(
        _arg(logits, "logits", F32), _arg(out, "out", F32), n, vocab, *h, *b,
        _opt_arg(allowed, "allowed", I32, n * ((vocab + 31) // 32)), _stream())
    _check_rc(lib, rc, "mnemo_logits_process")


# ---------------------------------------------------------------- batches that hold prompts
def paged_attention_prompt_workspace_bytes(n_heads: int, n_kv_heads: int, head_dim: int) -> int:
    return int(load_library().mnemo_paged_attention_prompt_workspace_bytes(n_heads, n_kv_heads, head_dim))


def paged_attention_prompt(q, k_pages, v_pages, block_table, starts, seq_lens, out, scale: float, ws, ks=None, vs=None):
    """Causal attention of the rows starts[s] .. starts[s+1]-1 of q [T, n_heads, head_dim], the last new tokens of
    sequence s (the cache holds them already: the last of them is position seq_lens[s] - 1), into out."""
    lib = load_library()
    ptrs, (_, n_pages, nkv, ps, hd) = _pages(k_pages, v_pages, ks, vs, False)
    table, n_seqs, max_pages = _rows(block_table)
    shape = q.shape
    if len(shape) != 3 or shape[2] != hd or out.shape != shape:
        raise MnemoError("paged_attention_prompt: q and out must be [T, n_heads, head_dim]")
    rc = lib.mnemo_paged_attention_prompt(
        _arg(q, "q", F32), *ptrs, _arg(out, "out", F32), shape[0], shape[1], hd, nkv, n_pages, ps, table, n_seqs, max_pages,
        _arg(starts, "starts", I32, n_seqs + 1), _arg(seq_lens, "seq_lens", I32, n_seqs), float(scale), _arg(ws, "ws"),
        ws.numel() * ws.element_size(), _stream())
    _check_rc(lib, rc, "mnemo_paged_attention_prompt")


def moe_route(logits, topk_idx, topk_w, sigmoid: bool = False, bias=None, n_groups: int = 1, top_groups: int = 1,
              group_best: int = 1, renormalise: bool = True, scale: float = 1.0):
    """topk_idx, topk_w [T, k]: the experts of each row of logits [T, n_experts] and their weights, best first, as
    moe_prefill takes them.  Softmax or sigmoid scores; the choice goes by score + bias [n_experts], among the experts
    of the top_groups groups with the largest sum of their group_best best."""
    lib = load_library()
    shape, to = logits.shape, topk_idx.shape
    if len(shape) != 2 or len(to) != 2 or to[0] != shape[0] or topk_w.shape != to:
        raise MnemoError("moe_route: logits must be [T, n_experts], topk_idx and topk_w [T, k]")
    rc = lib.mnemo_moe_route(_arg(logits, "logits", F32), shape[0], shape[1], int(sigmoid),
                             _opt_arg(bias, "bias", F32, shape[1]), int(n_groups), int(top_groups), int(group_best), to[1],
                             int(renormalise), float(scale), _arg(topk_idx, "topk_idx", I32), _arg(topk_w, "topk_w", F32),
                             _stream())
    _check_rc(lib, rc, "mnemo_moe_route")


def lora_workspace_bytes(n_tokens: int, n_in: int, max_rank: int) -> int:
    return int(load_library().mnemo_lora_workspace_bytes(n_tokens, n_in, max_rank))


def lora_add(x, a_w, b_w, adapter_ids, ranks, scales, base, out, ws):
    """out[t] = base[t] + scales[a] * B_a (A_a x[t]) with a = adapter_ids[t] (none outside the table): x [T, n_in], base
    and out [T, n_out] (out may be base), a_w [n_adapters, max_rank, n_in] and b_w [n_adapters, n_out, max_rank] float16 or
    bfloat16, of which the first ranks[a] ranks count."""
    lib = load_library()
    if x.dim() != 2 or a_w.dim() != 3 or b_w.dim() != 3 or base.dim() != 2 or out.shape != base.shape:
        raise MnemoError("lora_add: x, base and out must have 2 dimensions, a_w and b_w 3")
    (T, K), (N, R, _), M = x.shape, a_w.shape, base.shape[1]
    if a_w.shape[2] != K or b_w.shape != (N, M, R) or base.shape[0] != T:
        raise MnemoError("lora_add: a_w must be [n_adapters, max_rank, n_in], b_w [n_adapters, n_out, max_rank], x [T, n_in], "
                         "base and out [T, n_out]")
    if a_w.dtype is not torch.float16 and a_w.dtype is not torch.bfloat16:
        raise MnemoError(f"adapters must be float16 or bfloat16, got {a_w.dtype}")
    rc = lib.mnemo_lora_add(_arg(x, "x", F32), _arg(a_w, "a_w"), _arg(b_w, "b_w", a_w.dtype),
                            int(a_w.dtype is torch.bfloat16), _arg(adapter_ids, "adapter_ids", I32, T),
                            _arg(ranks, "ranks", I32, N), _arg(scales, "scales", F32, N), _arg(base, "base", F32),
                            _arg(out, "out", F32), T, K, M, N, R, _arg(ws, "ws"), ws.numel() * ws.element_size(), _stream())
    _check_rc(lib, rc, "mnemo_lora_add")


def logprobs_workspace_bytes(n_rows: int, vocab: int, n_top: int) -> int:
    return int(load_library().mnemo_logprobs_workspace_bytes(n_rows, vocab, n_top))


def logprobs(logits, targets, logprob, rank, entropy, top_ids, top_logprobs, ws):
    """Of each row of logits [n, vocab]: the log probability and rank of targets[n], the entropy, and the ids and log
    probabilities [n, n_top] of the likeliest tokens.  Any of the three may be left out (targets with logprob and rank,
    entropy, top_ids with top_logprobs: None)."""
    lib = load_library()
    if logits.dim() != 2 or (top_ids is not None and (top_logprobs is None or top_ids.dim() != 2 or
                                                      top_ids.shape[0] != logits.shape[0] or
                                                      top_logprobs.shape != top_ids.shape)):
        raise MnemoError("logprobs: logits must be [n, vocab], top_ids and top_logprobs [n, n_top]")
    n, vocab = logits.shape
    rc = lib.mnemo_logprobs(_arg(logits, "logits", F32), _opt_arg(targets, "targets", I32, n), n, vocab,
                            _opt_arg(logprob, "logprob", F32, n), _opt_arg(rank, "rank", I32, n),
                            _opt_arg(entropy, "entropy", F32, n), 0 if top_ids is None else top_ids.shape[1],
                            _opt_arg(top_ids, "top_ids", I32), _opt_arg(top_logprobs, "top_logprobs", F32),
                            _arg(ws, "ws"), ws.numel() * ws.element_size(), _stream())
    _check_rc(lib, rc, "mnemo_logprobs")
