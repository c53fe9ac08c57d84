// paged_attn.hip -- several sequences in one pool of cache pages: the new tokens' preparation and
// store, and the attention of one new token per sequence.
//
// Pages: K [page][n_kv][ps][hd], V [page][n_kv][hd][ps] (8 consecutive positions of a dim are
// contiguous, a matrix instruction's operand), int8 scales [page][n_kv][ps].
#include <math.h>

#include "mnemo_common.hpp"
#include "mnemo_internal.hpp"

namespace mnemo {

// ------------------------------------------------------------------ attention
size_t paged_attn_workspace_bytes(int, int) { return 16; }

// One workgroup per (query head, sequence); thread d owns dim d.
__global__ void __launch_bounds__(256) paged_attn_kernel(PagedAttnArgs a) {
    __shared__ float red[256];
    const int h = blockIdx.x, s = blockIdx.y, d = threadIdx.x, hd = a.c.hd, ps = a.c.ps;
    const int kvh = h / a.gqa;
    const int len = min(max(a.lens[s], 0), a.max_pages * ps);
    const float qd = a.q[((size_t)s * a.nh + h) * hd + d];
    float m = -INFINITY;
    double l = 0.0, o = 0.0;  // tens of thousands of terms one by one
    for (int p = 0; p < len; p++) {
        const int page = a.table[(size_t)s * a.max_pages + p / ps];
        if ((unsigned)page >= (unsigned)a.c.n_pages) continue;
        const size_t row = (size_t)page * a.c.nkv + kvh;
        const size_t ki = (row * ps + p % ps) * hd + d, vi = (row * hd + d) * ps + p % ps;
        float k, v;
        if (a.c.kv_type == kKvF16) {
            k = (float)((const _Float16 *)a.c.k)[ki];
            v = (float)((const _Float16 *)a.c.v)[vi];
        } else {
            k = (float)((const int8_t *)a.c.k)[ki] * a.c.ksc[row * ps + p % ps];
            v = (float)((const int8_t *)a.c.v)[vi] * a.c.vsc[row * ps + p % ps];
        }
        red[d] = qd * k;
        __syncthreads();
        float z = 0.0f;
        for (int i = 0; i < hd; i++) z += red[i];
        __syncthreads();
        z *= a.scale;
        const float mn = fmaxf(m, z);
        const float r = expf(m - mn), e = expf(z - mn);
        l = l * r + e;
        o = o * r + (double)e * v;
        m = mn;
    }
    a.out[((size_t)s * a.nh + h) * hd + d] = l > 0.0 ? (float)(o / l) : 0.0f;
}

int launch_paged_attention(const PagedAttnArgs &a, hipStream_t s) {
    hipLaunchKernelGGL(paged_attn_kernel, dim3(a.nh, a.n_seqs), dim3(a.c.hd), 0, s, a);
    return check_launch("paged_attention_decode");
}

// ------------------------------------------------------------------ preparation of new tokens
// One workgroup per (token, group of heads): q heads, then k, then v.  HD / 8 lanes own a head,
// four rotated pairs (j, j + HD/2) each.  The angle of pair j at position p is p turn[j] in units
// of 2^-64 of a turn, formed in integers (the product keeps its low 64 bits, whole turns fall off),
// so that it is as exact at position 10^6 as at 1: fp32 angles are off by p 2^-24.
template <int KV, int HD>
__global__ void __launch_bounds__(256) paged_prep_kernel(PagedPrepArgs a) {
    constexpr int LPH = HD / 8, HALF = HD / 2;
    __shared__ float cs[HALF], sn[HALF];
    const int t = blockIdx.x, tid = threadIdx.x;
    const int seq = a.seq ? a.seq[t] : t;
    const bool row = (unsigned)seq < (unsigned)a.n_seqs;
    const int pos = a.pos ? a.pos[t] : (row ? a.lens[t] - 1 : -1);
    if (pos < 0) return;  // padding
    if (tid < HALF) {
        const int32_t frac = (int32_t)(((uint64_t)(uint32_t)pos * a.turn[tid]) >> 32);  // of a turn, in 2^-32
        sincospif((float)frac * 0x1p-31f, &sn[tid], &cs[tid]);
    }
    const int head = (int)blockIdx.y * (256 / LPH) + tid / LPH, l = tid % LPH;
    const int nkv = a.c.nkv;
    const bool is_q = head < a.nh, is_k = !is_q && head < a.nh + nkv;
    const int h = is_q ? head : is_k ? head - a.nh : head - a.nh - nkv;
    const bool live = head < a.nh + 2 * nkv;
    float x0[4] = {}, x1[4] = {};
    if (live) {
        const float *src = is_q ? a.q + ((size_t)t * a.nh + h) * HD
                                : (is_k ? a.k : a.v) + ((size_t)t * nkv + h) * HD;
        __builtin_memcpy(x0, src + 4 * l, 16);
        __builtin_memcpy(x1, src + HALF + 4 * l, 16);
    }
    __syncthreads();
    if (!live) return;
    if (is_q || is_k) {
        if (a.qw) {
            const float *w = is_q ? a.qw : a.kw;
            float ss = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; i++) ss = fmaf(x0[i], x0[i], fmaf(x1[i], x1[i], ss));
#pragma unroll
            for (int o = 1; o < LPH; o <<= 1) ss += __shfl_xor(ss, o);
            const float g = 1.0f / sqrtf(ss / (float)HD + a.eps);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                x0[i] = x0[i] * g * w[4 * l + i];
                x1[i] = x1[i] * g * w[HALF + 4 * l + i];
            }
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float c = cs[4 * l + i], s = sn[4 * l + i], v0 = x0[i], v1 = x1[i];
            x0[i] = fmaf(v0, c, -(v1 * s));
            x1[i] = fmaf(v0, s, v1 * c);
        }
    }
    if (is_q) {
        float *dst = a.q_out + ((size_t)t * a.nh + h) * HD;
        __builtin_memcpy(dst + 4 * l, x0, 16);
        __builtin_memcpy(dst + HALF + 4 * l, x1, 16);
        return;
    }
    const int pi = pos / a.c.ps, off = pos % a.c.ps;
    if (!row || pi >= a.max_pages) return;
    const int page = a.table[(size_t)seq * a.max_pages + pi];
    if ((unsigned)page >= (unsigned)a.c.n_pages) return;
    const size_t r = (size_t)page * nkv + h;
    const size_t base = is_k ? (r * a.c.ps + off) * HD : r * HD * a.c.ps + off;
    const int es = is_k ? 1 : a.c.ps;  // element stride along the head dim
    if (KV == kKvF16) {
        _Float16 *c = (_Float16 *)(is_k ? a.c.k : a.c.v) + base;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            c[(size_t)(4 * l + i) * es] = (_Float16)x0[i];
            c[(size_t)(HALF + 4 * l + i) * es] = (_Float16)x1[i];
        }
    } else {
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; i++) m = fmaxf(m, fmaxf(fabsf(x0[i]), fabsf(x1[i])));
#pragma unroll
        for (int o = 1; o < LPH; o <<= 1) m = fmaxf(m, __shfl_xor(m, o));
        // a row below 1e-36 (its 127 / m leaves the range) is stored as zeros
        const float inv = m >= 1e-36f ? 127.0f / m : 0.0f;
        int8_t *c = (int8_t *)(is_k ? a.c.k : a.c.v) + base;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            c[(size_t)(4 * l + i) * es] = (int8_t)fminf(fmaxf(rintf(x0[i] * inv), -127.0f), 127.0f);
            c[(size_t)(HALF + 4 * l + i) * es] = (int8_t)fminf(fmaxf(rintf(x1[i] * inv), -127.0f), 127.0f);
        }
        if (l == 0) (is_k ? a.c.ksc : a.c.vsc)[r * a.c.ps + off] = m >= 1e-36f ? m / 127.0f : 0.0f;
    }
}

int launch_paged_prep(PagedPrepArgs &a, double theta, hipStream_t s) {
    const int hd = a.c.hd;
    for (int j = 0; j < hd / 2; j++) {
        const double turns = pow(theta, -2.0 * j / hd) / (2.0 * M_PI);  // of position 1, below 1 for theta >= 1
        a.turn[j] = (uint64_t)ldexp(turns - floor(turns), 64);
    }
    const dim3 grid(a.n_tokens, (a.nh + 2 * a.c.nkv + 2048 / hd - 1) / (2048 / hd));
#define MNEMO_PREP(HD_)                                                                                             \
    do {                                                                                                            \
        if (a.c.kv_type == kKvF16) hipLaunchKernelGGL((paged_prep_kernel<kKvF16, HD_>), grid, dim3(256), 0, s, a);  \
        else hipLaunchKernelGGL((paged_prep_kernel<kKvInt8, HD_>), grid, dim3(256), 0, s, a);                       \
    } while (0)
    if (hd == 64) MNEMO_PREP(64);
    else if (hd == 128) MNEMO_PREP(128);
    else MNEMO_PREP(256);
#undef MNEMO_PREP
    return check_launch("paged_attn_prep");
}

}  // namespace mnemo
