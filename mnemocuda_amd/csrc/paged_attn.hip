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
// out[s][h] = sum_p P_p v_p / sum_p P_p,  P_p = exp(scale q.k_p - m), over the positions of row s.
//
// The work is cut into units of kUnit positions of one (sequence, KV head), in that order, and the
// workgroups take equal shares of the row of units, whatever the lengths are: every workgroup
// computes its share from the lengths itself.  A (sequence, KV head) that lies within one share
// is finished there; one that several shares cut leaves a partial (max, sum, O) in each, which a
// second launch merges.
//
// Within a share the four waves take STEP positions each in turn, with no exchange between them
// until the end, and no LDS: S^T = K Q^T (positions x heads) comes out of the matrix instruction
// with a lane holding four positions of one head, which is how O^T = V^T P^T (dims x heads) wants
// P^T, when the K rows of a tile are picked so: lane row m of tile t is position
// (STEP/4)(m/4) + 4t + m%4, so that a lane's rows over the tiles are STEP/4 consecutive positions.
// K fragments are 16 bytes of a K row, V fragments 16 bytes of positions of one dim.
//
// Precision: Q is scaled by a power of two into [1, 2) per head and split into two f16 parts, P
// likewise split; K and V enter exactly (f16 or int8).  P is formed relative to a reference that
// follows the maximum only when a score exceeds it by 2^kSlack, and is 2^kLift at the reference:
// its smallest f16 step, 2^-24, is then 2^-33 of the largest weight.  int8 value scales multiply
// P relative to a power of two that follows the largest of them in the same way.
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr int kPaThreads = 256, kPaWaves = 4, kPaRows = 16;
constexpr float kSlack = 5.0f, kLift = 9.0f;  // powers of two: P <= 2^14, times a scale below 2

template <int KV, int HD>
struct PaShape {
    static constexpr int kStep = KV == kKvF16 ? 32 : 64;  // positions of a wave's step
    static constexpr int kUnit = kPaWaves * kStep;
    static constexpr int kTiles = kStep / 16;
    static constexpr int kKs = HD / 32, kNd = HD / 16;  // dim steps of S, dim tiles of O
};

constexpr int kPaMaxGroups = 768;
static int part_floats(int hd) { return kPaRows * (hd + 2); }
size_t paged_attn_workspace_bytes(int, int hd) { return (size_t)2 * kPaMaxGroups * part_floats(hd) * sizeof(float); }

// Inclusive sum over the lower lanes.
__device__ __forceinline__ int wave_scan(int v) {
    const int lane = lane_id();
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(v, o);
        if (lane >= o) v += y;
    }
    return v;
}

__device__ __forceinline__ int seq_len(const PagedAttnArgs &a, int s) {
    return min(max(a.lens[s], 0), a.max_pages * a.c.ps);
}

// Where the units begin: the row of units is [sequence][KV head][unit].
struct PaPlan {
    int total;   // units
    int groups;  // workgroups that have some
    int per;     // sequences per lane of the sums
    int before;  // lane: units before its sequences
};

template <int UNIT>
__device__ __forceinline__ PaPlan pa_plan(const PagedAttnArgs &a, int groups) {
    PaPlan p;
    p.per = (a.n_seqs + 63) / 64;
    const int s0 = lane_id() * p.per;
    int sum = 0;
    for (int i = 0; i < p.per; i++)
        if (s0 + i < a.n_seqs) sum += (seq_len(a, s0 + i) + UNIT - 1) / UNIT;
    sum *= a.c.nkv;
    const int incl = wave_scan(sum);
    p.total = __builtin_amdgcn_readlane(incl, 63);
    p.before = incl - sum;
    p.groups = min(groups, p.total);
    return p;
}

// First unit of workgroup w, and the workgroup of unit u.
__device__ __forceinline__ int pa_first(const PaPlan &p, int w) { return (int)((long long)w * p.total / p.groups); }
__device__ __forceinline__ int pa_group(const PaPlan &p, int u) {
    return (int)(((long long)(u + 1) * p.groups - 1) / p.total);
}

// The sequence, KV head and unit within them of unit u; len: of the sequence.
template <int UNIT>
__device__ __forceinline__ void pa_find(const PagedAttnArgs &a, const PaPlan &p, int u, int &seq, int &kvh, int &unit,
                                        int &len) {
    const int lane = lane_id();
    const int L = __popcll(__ballot(p.before <= u)) - 1;  // the last lane that begins at or before u holds it
    const int base = __builtin_amdgcn_readlane(p.before, L);
    const int s = L * p.per + lane;
    const int ln = lane < p.per && s < a.n_seqs ? seq_len(a, s) : 0;
    const int n = (ln + UNIT - 1) / UNIT * a.c.nkv;
    const int before = base + wave_scan(n) - n;
    const int j = __popcll(__ballot(lane < p.per && before <= u)) - 1;
    seq = L * p.per + j;
    len = __builtin_amdgcn_readlane(ln, j);
    const int at = u - __builtin_amdgcn_readlane(before, j), nu = (len + UNIT - 1) / UNIT;
    kvh = at / nu;
    unit = at % nu;
}

// max over the four lanes that share a head (lane % 16), in all of them
__device__ __forceinline__ float max_heads(float v) {
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float sum_heads(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

// 1 / v of a power of two from 2^-126 to 2^126
__device__ __forceinline__ float inverse2(float v) {
    return __builtin_bit_cast(float, 0x7f000000u - __builtin_bit_cast(uint32_t, v));
}

// 8 int8 as f16: 0x64uu is 1024 + uu, so with the sign bit flipped and 1152 taken off it is the number.
__device__ __forceinline__ h4 cvt4(uint32_t w) {
    const uint32_t u = w ^ 0x80808080u;
    const uint32_t lo = __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u), hi = __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u);
    const h2 off = {(_Float16)1152.0f, (_Float16)1152.0f};
    const h2 a = __builtin_bit_cast(h2, lo) - off, b = __builtin_bit_cast(h2, hi) - off;
    return __builtin_shufflevector(a, b, 0, 1, 2, 3);
}
__device__ __forceinline__ h8 cvt8(uint32_t a, uint32_t b) {
    return __builtin_shufflevector(cvt4(a), cvt4(b), 0, 1, 2, 3, 4, 5, 6, 7);
}

template <int KV, int HD>
__global__ void __launch_bounds__(kPaThreads, HD == 256 ? 1 : 2) paged_attn_kernel(PagedAttnArgs a) {
    using S = PaShape<KV, HD>;
    constexpr int STEP = S::kStep, UNIT = S::kUnit, NT = S::kTiles, KS = S::kKs, ND = S::kNd;
    constexpr int EB = KV == kKvF16 ? 2 : 1;
    constexpr int PV = STEP / 32;  // position steps of O
    __shared__ __align__(16) float lo[kPaWaves][kPaRows][HD + 4];
    __shared__ float lm[kPaWaves][kPaRows], ll[kPaWaves][kPaRows];
    const int lane = lane_id(), r = lane & 15, kg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int ps = a.c.ps, psl = 31 - __builtin_clz(ps);

    // rows with no positions
    for (int s = blockIdx.x; s < a.n_seqs; s += gridDim.x)
        if (seq_len(a, s) == 0)
            for (int i = threadIdx.x; i < a.nh * HD; i += kPaThreads) a.out[(size_t)s * a.nh * HD + i] = 0.0f;

    const PaPlan plan = pa_plan<UNIT>(a, gridDim.x);
    if ((int)blockIdx.x >= plan.groups) return;
    int at = pa_first(plan, blockIdx.x);
    const int end = pa_first(plan, blockIdx.x + 1);
    int seq, kvh, unit, len;
    pa_find<UNIT>(a, plan, at, seq, kvh, unit, len);

    while (true) {
        const int nu = (len + UNIT - 1) / UNIT, n = min(end - at, nu - unit);
        const int p_end = min(len, (unit + n) * UNIT);
        const int *table = a.table + (size_t)seq * a.max_pages;
        const uint8_t *kc = (const uint8_t *)a.c.k, *vc = (const uint8_t *)a.c.v;

        // page entries of a step: of the lane's K rows (position group r / 4) and V positions (group kg)
        struct Pages { int k, v; };
        auto entries = [&](int p0) {
            const int last = (len - 1) >> psl;
            Pages e;
            e.k = table[min((p0 + STEP / 4 * (r >> 2)) >> psl, last)];
            e.v = table[min((p0 + STEP / 4 * kg) >> psl, last)];
            return e;
        };
        u4 kr[NT][HD * EB / 64], vr[ND];
        float ksc[KV == kKvInt8 ? 16 : 1], vsc[KV == kKvInt8 ? 16 : 1];
        auto load_k = [&](int p0, int page) {
            const int row = ((p0 + STEP / 4 * (r >> 2)) & (ps - 1)) + (r & 3);
            page = (unsigned)page < (unsigned)a.c.n_pages ? page : 0;
            const uint8_t *base = kc + ((((size_t)page * a.c.nkv + kvh) * ps + row) * HD) * EB + 16 * kg;
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int j = 0; j < HD * EB / 64; j++) __builtin_memcpy(&kr[t][j], base + 4 * t * HD * EB + 64 * j, 16);
        };
        auto load_v = [&](int p0, int page) {
            const int off = (p0 + STEP / 4 * kg) & (ps - 1);
            page = (unsigned)page < (unsigned)a.c.n_pages ? page : 0;
            const uint8_t *base = vc + ((((size_t)page * a.c.nkv + kvh) * HD + r) * ps + off) * EB;
#pragma unroll
            for (int i = 0; i < ND; i++) __builtin_memcpy(&vr[i], base + (size_t)16 * i * ps * EB, 16);
        };
        auto load_scales = [&](int p0, int page) {
            const int off = (p0 + STEP / 4 * kg) & (ps - 1);
            page = (unsigned)page < (unsigned)a.c.n_pages ? page : 0;
            const size_t base = ((size_t)page * a.c.nkv + kvh) * ps + off;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                __builtin_memcpy(&ksc[4 * i], a.c.ksc + base + 4 * i, 16);
                __builtin_memcpy(&vsc[4 * i], a.c.vsc + base + 4 * i, 16);
            }
        };

        float m = -INFINITY, l = 0.0f;  // reference (log2) of the lane's head, sum over the lane's positions
        float vref = 0x1p-126f;
        f4 o[ND] = {};
        int p0 = unit * UNIT + wave * STEP;
        if (p0 < p_end) {
            Pages cur = entries(p0);
            // ---- Q: dims of slot j of dim step st as the K fragments have them
            float q[KS][8];
            const float *qh = a.q + ((size_t)seq * a.nh + kvh * a.gqa + min(r, a.gqa - 1)) * HD;
#pragma unroll
            for (int st = 0; st < KS; st++) {
                const int d = KV == kKvF16 ? 32 * st + 8 * kg : 64 * (st >> 1) + 16 * kg + 8 * (st & 1);
                __builtin_memcpy(&q[st][0], qh + d, 16);
                __builtin_memcpy(&q[st][4], qh + d + 4, 16);
            }
            load_k(p0, cur.k);
            if (KV == kKvInt8) load_scales(p0, cur.v);
            int next = p0 + UNIT;
            Pages nxt = entries(min(next, len - 1));
            load_v(p0, cur.v);
            float qm = 0.0f;
#pragma unroll
            for (int st = 0; st < KS; st++)
#pragma unroll
                for (int j = 0; j < 8; j++) qm = fmaxf(qm, fabsf(q[st][j]));
            qm = max_heads(qm);
            const int qe = (int)((__builtin_bit_cast(uint32_t, qm) >> 23) & 255) - 127;  // exponent of the largest
            const float qs = ldexpf(1.0f, -qe);
            const float c = ldexpf(a.scale * 1.44269504088896341f, qe);
            h8 qhi[KS], qlo[KS];
#pragma unroll
            for (int st = 0; st < KS; st++)
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float x = q[st][j] * qs;
                    qhi[st][j] = (_Float16)x;
                    qlo[st][j] = (_Float16)(x - (float)qhi[st][j]);
                }
            for (;;) {
                // ---- S^T: lane: head r, positions p0 + STEP/4 kg + 4t + i
                f4 s[NT];
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    s[t] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int st = 0; st < KS; st++) {
                        h8 kf;
                        if (KV == kKvF16) kf = __builtin_bit_cast(h8, kr[t][st]);
                        else kf = cvt8(kr[t][st >> 1][2 * (st & 1)], kr[t][st >> 1][2 * (st & 1) + 1]);
                        s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qhi[st], s[t], 0, 0, 0);
                        s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qlo[st], s[t], 0, 0, 0);
                    }
                }
                const bool more = next < p_end;  // uniform
                if (more) load_k(next, nxt.k);
                // ---- weights
                const int live = min(max(len - (p0 + STEP / 4 * kg), 0), STEP / 4);  // of the lane's positions
                const bool ok = (unsigned)cur.v < (unsigned)a.c.n_pages;
                const bool full = __all(ok && live == STEP / 4);  // uniform
                float smax = -INFINITY, vmax = 0.0f;
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        float x = s[t][i] * c;
                        if (KV == kKvInt8) x *= ksc[4 * t + i];
                        if (!full) {
                            const bool in = ok && 4 * t + i < live;
                            x = in ? x : -INFINITY;
                            if (KV == kKvInt8) vsc[4 * t + i] = in ? vsc[4 * t + i] : 0.0f;
                        }
                        s[t][i] = x;
                        smax = fmaxf(smax, x);
                        if (KV == kKvInt8) vmax = fmaxf(vmax, fabsf(vsc[4 * t + i]));
                    }
                if (__any(smax > m + kSlack || (KV == kKvInt8 && vmax >= 2.0f * vref))) {
                    const float mn = fmaxf(m, max_heads(smax));
                    const float al = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
                    float f = al;
                    if (KV == kKvInt8) {
                        float vm = vmax;
#pragma unroll
                        for (int x = 1; x < 64; x <<= 1) vm = fmaxf(vm, __shfl_xor(vm, x));
                        // the power of two at or below vm (at most 2^126, so that its inverse is a float)
                        const uint32_t e = min(__builtin_bit_cast(uint32_t, vm) & 0x7f800000u, 0x7e800000u);
                        const float vn = fmaxf(vref, __builtin_bit_cast(float, e));
                        f = al * (vref * inverse2(vn));
                        vref = vn;
                    }
                    l *= al;
#pragma unroll
                    for (int i = 0; i < ND; i++) o[i] *= f;
                    m = mn;
                }
                const float ref = m == -INFINITY ? 0.0f : m - kLift;
                const float vi = inverse2(vref);
                h8 phi[PV], plo[PV];
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float p = __builtin_amdgcn_exp2f(s[t][i] - ref);
                        l += p;
                        float w = KV == kKvInt8 ? p * (vsc[4 * t + i] * vi) : p;
                        // one fp32 value for both parts: a product folded into one of the conversions
                        // would round differently there
                        asm("" : "+v"(w));
                        const _Float16 hi = (_Float16)w;
                        phi[t / 2][4 * (t & 1) + i] = hi;
                        plo[t / 2][4 * (t & 1) + i] = (_Float16)(w - (float)hi);
                    }
                if (KV == kKvInt8 && more) load_scales(next, nxt.v);
                const Pages after = entries(min(next + UNIT, len - 1));
                // ---- O^T
                if (KV == kKvF16 && !full) {
                    // what lies past the end may be no number, which a weight of 0 does not hide
#pragma unroll
                    for (int i = 0; i < ND; i++)
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            uint32_t w = vr[i][j];
                            if (!ok || live <= 2 * j) w = 0;
                            else if (live == 2 * j + 1) w &= 0xffffu;
                            vr[i][j] = w;
                        }
                }
#pragma unroll
                for (int i = 0; i < ND; i++)
#pragma unroll
                    for (int k = 0; k < PV; k++) {
                        h8 vf;
                        if (KV == kKvF16) vf = __builtin_bit_cast(h8, vr[i]);
                        else vf = cvt8(vr[i][2 * k], vr[i][2 * k + 1]);
                        o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, phi[k], o[i], 0, 0, 0);
                        o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, plo[k], o[i], 0, 0, 0);
                    }
                if (!more) break;
                load_v(next, nxt.v);
                p0 = next;
                next += UNIT;
                cur = nxt;
                nxt = after;
            }
        }
        // ---- the four waves' results meet in LDS
        l = sum_heads(l);
        if (kg == 0) {
            lm[wave][r] = m;
            ll[wave][r] = l;
        }
#pragma unroll
        for (int i = 0; i < ND; i++) {
            f4 x = o[i];
            if (KV == kKvInt8) x *= vref;
            __builtin_memcpy(&lo[wave][r][16 * i + 4 * kg], &x, 16);
        }
        __syncthreads();
        const bool whole = unit == 0 && n == nu;  // finished here
        // a partial goes to the first slot when the (sequence, KV head) began in an earlier workgroup
        float *part = a.ws + (size_t)(2 * blockIdx.x + (unit == 0)) * (kPaRows * (HD + 2));
        for (int e = threadIdx.x; e < a.gqa * (HD / 4); e += kPaThreads) {
            const int h = e / (HD / 4), d = 4 * (e % (HD / 4));
            float mm = lm[0][h];
#pragma unroll
            for (int w = 1; w < kPaWaves; w++) mm = fmaxf(mm, lm[w][h]);
            f4 x = {};
            float sum = 0.0f;
#pragma unroll
            for (int w = 0; w < kPaWaves; w++) {
                const float f = mm == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(lm[w][h] - mm);
                f4 y;
                __builtin_memcpy(&y, &lo[w][h][d], 16);
                x += y * f;
                sum = fmaf(ll[w][h], f, sum);
            }
            if (whole) {
                x = sum == 0.0f ? f4{0.f, 0.f, 0.f, 0.f} : x / sum;
                __builtin_memcpy(a.out + ((size_t)seq * a.nh + kvh * a.gqa + h) * HD + d, &x, 16);
            } else {
                __builtin_memcpy(part + 2 * kPaRows + h * HD + d, &x, 16);
                if (d == 0) {
                    part[h] = mm;
                    part[kPaRows + h] = sum;
                }
            }
        }
        at += n;
        if (at >= end) return;
        __syncthreads();  // the sums are read
        unit = 0;
        if (++kvh == a.c.nkv) {
            kvh = 0;
            do len = seq_len(a, ++seq);
            while (len == 0);  // a unit is left, so a sequence with positions is
        }
    }
}

// Merges the partials of the (sequence, KV head)s that several workgroups share.  Workgroup x looks
// after the one that begins in share x and goes on behind it (BY_SHARE), or after (sequence, KV head)
// x itself.  32 x 8 threads: HD / 32 dims each of every eighth partial, then over the eight.
template <int UNIT, int HD, bool BY_SHARE>
__global__ void __launch_bounds__(256) paged_merge_kernel(PagedAttnArgs a, int groups) {
    constexpr int D = HD / 32;
    __shared__ float so[8][HD], sm[8], sl[8];
    const PaPlan plan = pa_plan<UNIT>(a, groups);
    int seq, kvh, first, last, len;
    if (BY_SHARE) {
        if ((int)blockIdx.x + 1 >= plan.groups) return;
        const int u = pa_first(plan, blockIdx.x + 1) - 1;  // the last unit of the share
        int unit;
        pa_find<UNIT>(a, plan, u, seq, kvh, unit, len);
        const int nu = (len + UNIT - 1) / UNIT;
        if (unit + 1 == nu || u - unit < pa_first(plan, blockIdx.x)) return;
        first = u - unit;
        last = first + nu - 1;
    } else {
        seq = blockIdx.x / a.c.nkv;
        kvh = blockIdx.x % a.c.nkv;
        len = seq_len(a, seq);
        if (len == 0) return;
        const int nu = (len + UNIT - 1) / UNIT;
        const int L = seq / plan.per;
        int before = __builtin_amdgcn_readlane(plan.before, L);
        int mine = 0;
        const int s = L * plan.per + lane_id();
        if (s < seq) mine = (seq_len(a, s) + UNIT - 1) / UNIT * a.c.nkv;
        before += __builtin_amdgcn_readlane(wave_scan(mine), 63);
        first = before + kvh * nu;
        last = first + nu - 1;
    }
    const int w0 = pa_group(plan, first), w1 = pa_group(plan, last);
    if (w0 == w1) return;
    const int dl = threadIdx.x & 31, g = threadIdx.x >> 5;
    constexpr int PART = kPaRows * (HD + 2);
    for (int h = blockIdx.y; h < a.gqa; h += gridDim.y) {
        float m = -INFINITY, l = 0.0f, o[D] = {};
        for (int w = w0 + g; w <= w1; w += 8) {
            // the first share holds its beginning in its second slot, the others in the first
            const float *p = a.ws + (size_t)(2 * w + (w == w0)) * PART;
            const float pm = p[h], pl = p[kPaRows + h];
            float x[D];
            __builtin_memcpy(x, p + 2 * kPaRows + h * HD + D * dl, 4 * D);
            const float mn = fmaxf(m, pm);
            if (mn == -INFINITY) continue;
            const float fa = __builtin_amdgcn_exp2f(m - mn), fb = __builtin_amdgcn_exp2f(pm - mn);
            l = l * fa + pl * fb;
#pragma unroll
            for (int i = 0; i < D; i++) o[i] = o[i] * fa + x[i] * fb;
            m = mn;
        }
        __syncthreads();  // the last head's sums are read
        __builtin_memcpy(&so[g][D * dl], o, 4 * D);
        if (dl == 0) {
            sm[g] = m;
            sl[g] = l;
        }
        __syncthreads();
        if ((int)threadIdx.x < HD) {
            float mm = sm[0];
#pragma unroll
            for (int i = 1; i < 8; i++) mm = fmaxf(mm, sm[i]);
            float sum = 0.0f, x = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float f = mm == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(sm[i] - mm);
                sum = fmaf(sl[i], f, sum);
                x = fmaf(so[i][threadIdx.x], f, x);
            }
            a.out[((size_t)seq * a.nh + kvh * a.gqa + h) * HD + threadIdx.x] = sum == 0.0f ? 0.0f : x / sum;
        }
    }
}

template <int KV, int HD>
static void launch_pa(const PagedAttnArgs &a, hipStream_t s) {
    constexpr int UNIT = PaShape<KV, HD>::kUnit;
    const long long pairs = (long long)a.n_seqs * a.c.nkv;
    const long long most = pairs * (((long long)a.max_pages * a.c.ps + UNIT - 1) / UNIT);  // units, whatever the lengths
    const int groups = (int)(most < kPaMaxGroups ? most : kPaMaxGroups);
    hipLaunchKernelGGL((paged_attn_kernel<KV, HD>), dim3(groups), dim3(kPaThreads), 0, s, a);
    if (pairs < groups) {
        const int y = (int)(1024 / pairs < a.gqa ? (1024 / pairs < 1 ? 1 : 1024 / pairs) : a.gqa);
        hipLaunchKernelGGL((paged_merge_kernel<UNIT, HD, false>), dim3((int)pairs, y), dim3(256), 0, s, a, groups);
    } else if (most > pairs) {  // else no (sequence, KV head) has a second unit
        hipLaunchKernelGGL((paged_merge_kernel<UNIT, HD, true>), dim3(groups, 1), dim3(256), 0, s, a, groups);
    }
}

int launch_paged_attention(const PagedAttnArgs &a, hipStream_t s) {
#define MNEMO_PA(HD_)                                      \
    do {                                                   \
        if (a.c.kv_type == kKvF16) launch_pa<kKvF16, HD_>(a, s); \
        else launch_pa<kKvInt8, HD_>(a, s);                \
    } while (0)
    if (a.c.hd == 64) MNEMO_PA(64);
    else if (a.c.hd == 128) MNEMO_PA(128);
    else MNEMO_PA(256);
#undef MNEMO_PA
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
