// paged_attn.hip -- several sequences in one pool of cache pages: the new tokens' preparation and
// store, and the attention of one new token per sequence.
//
// Pages: K [page][n_kv][ps][hd], V [page][n_kv][hd][ps] (8 consecutive positions of a dim are
// contiguous, a matrix instruction's operand), int8 scales [page][n_kv][ps].
#include <limits.h>
#include <math.h>

#include "mfma_types.hpp"
#include "mnemo_common.hpp"
#include "mnemo_internal.hpp"

namespace mnemo {

// ------------------------------------------------------------------ attention
// out[s][h] = sum_p P_p v_p / sum_p P_p,  P_p = exp(scale q.k_p - m), over the positions of row s.
//
// The work is cut into steps of STEP positions of one (sequence, KV head), in that order, and the
// waves of the launch take equal shares of the row of steps, whatever the lengths are: every wave
// computes its share from the lengths itself.  A (sequence, KV head) that lies within one share
// is finished there; pieces of one that several shares cut meet in LDS where the shares belong to
// one workgroup, and as partials (max, sum, O) in memory, which a second launch merges, where not.
//
// A wave streams its steps with no exchange with others and no LDS: S^T = K Q^T (positions x heads)
// comes out of the matrix instruction with a lane holding four positions of one head, which is how
// O^T = V^T P^T (dims x heads) wants P^T, when the K rows of a tile are picked so: lane row m of
// tile t is position (STEP/4)(m/4) + 4t + m%4, so that a lane's rows over the tiles are STEP/4
// consecutive positions.  K fragments are 16 bytes of a K row, V fragments 16 bytes of positions of
// one dim.
//
// Bound by memory: 96 sequences to 8192 positions (957 MB) take 172 us, 5.5 TB/s, where a plain read of
// as much reaches 6.2; 3 int8 sequences to 131,072 (324 MB) 67.5 us.  A CU is given one workgroup, so
// shares are spread over the CUs first (300 positions 11.3 us on 4 CUs, 8.3 on 40); what a small call
// takes is its chain of loads: lengths, table, K, V, then the same for the merge (300 positions: 8.5 us,
// of which 3.1 are the second launch; 3.1 to 3.9 of five calls from 8.5 to 172 us).
//
// Precision: Q is scaled by a power of two into [1, 2) per head and split into two f16 parts, P
// likewise split; K and V enter exactly (f16 or int8).  P is formed relative to a reference that
// follows the maximum only when a score exceeds it by 2^kSlack, and is 2^kLift at the reference:
// its smallest f16 step, 2^-24, is then 2^-33 of the largest weight.  int8: what is split is P times
// the value's scale, relative to a power of two (wref) that follows the largest such product in the
// same way, not the largest scale: a large scale of no weight leaves the others their bits.  The
// reference of P is a whole power there, so that O and its unit are rescaled without rounding.
constexpr int kPaRows = 16;
constexpr float kSlack = 5.0f, kLift = 9.0f;  // powers of two: P <= 2^14 (int8: 2^5, P times scale below 2^15 wref)

template <int KV, int HD, int STEP>
struct PaShape {
    static constexpr int kTiles = STEP / 16;
    static constexpr int kKs = HD / 32, kNd = HD / 16;  // dim steps of S, dim tiles of O
    // one workgroup per CU, whose pieces take most of its LDS (134 KB at head_dim 128 and 256; 70 KB at 64, where
    // there is room for a second one that is not launched)
    static constexpr int kWaves = HD == 256 ? 4 : 8;
    // the parts of Q wait in LDS where registers are short
    static constexpr bool kQInLds = HD == 128 && STEP == 64;
    static constexpr int kThreads = 64 * kWaves;
};

constexpr int kPaGroups = 256;  // one per CU
// Workspace: two partials per workgroup (max [16], sum [16], O [16][hd]) and what they are: begun[g] is the
// (sequence, KV head) that begins in workgroup g's share and goes on behind it (its second partial), taken[g]
// the one that it goes on with from the workgroup before (its first), -1 for none.
__host__ __device__ constexpr int part_floats(int hd) { return kPaRows * (hd + 2); }
size_t paged_attn_workspace_bytes(int hd) {
    return (size_t)2 * kPaGroups * (part_floats(hd) * sizeof(float) + sizeof(int));
}
__device__ __forceinline__ int *pa_begun(const PagedAttnArgs &a) {
    return (int *)(a.ws + (size_t)2 * kPaGroups * part_floats(a.c.hd));
}

__device__ __forceinline__ int seq_len(const PagedAttnArgs &a, int s) {
    return min(max(a.lens[s], 0), a.max_pages * a.c.ps);
}

// The row of steps, [sequence][KV head][step], and its shares.
struct PaPlan {
    int total;   // steps
    int groups;  // workgroups that have some
    int base, more;  // steps of a workgroup; the first `more` of them have one more
    int nw;      // waves of a workgroup that take shares
    bool empty;  // lane: a sequence of its has no positions
    int per;     // sequences per lane of the sums
    int len;     // lane: length of its sequence, where per is 1
    int before;  // lane: steps before its sequences
};

// The CUs are filled before the waves of a workgroup: eight steps on one CU end ~4 us after a step alone.
template <int STEP, int NW>
__device__ __forceinline__ PaPlan pa_plan(const PagedAttnArgs &a, int groups) {
    PaPlan p;
    p.per = (a.n_seqs + 63) / 64;
    p.len = 0;
    p.empty = false;
    const int s0 = lane_id() * p.per;
    int sum = 0;
    for (int i = 0; i < p.per; i++)
        if (s0 + i < a.n_seqs) {
            p.len = seq_len(a, s0 + i);
            p.empty |= p.len == 0;
            sum += (p.len + STEP - 1) / STEP;
        }
    sum *= a.c.nkv;
    const int incl = wave_scan(sum);
    p.total = __builtin_amdgcn_readlane(incl, 63);
    p.before = incl - sum;
    p.groups = max(min(groups, p.total), 1);
    p.base = p.total / p.groups;
    p.more = p.total - p.base * p.groups;
    p.nw = min(p.base + 1, NW);
    return p;
}

// First step of workgroup g (the end of the row from g = groups on).
__device__ __forceinline__ int pa_first(const PaPlan &p, int g) {
    return g >= p.groups ? p.total : g * p.base + min(g, p.more);
}

// The sequence, its length, the KV head and the step within them of step u.
template <int STEP>
__device__ __forceinline__ void pa_find(const PagedAttnArgs &a, const PaPlan &p, int u, int &seq, int &kvh, int &step,
                                        int &len) {
    const int lane = lane_id();
    // the last lane that begins at or before u holds it (lanes without steps share their successor's beginning)
    const int L = __popcll(__ballot(p.before <= u)) - 1;
    int at = u - __builtin_amdgcn_readlane(p.before, L);
    if (p.per == 1) {
        seq = L;
        len = __builtin_amdgcn_readlane(p.len, L);
    } else {
        const int s = L * p.per + lane;
        const int ln = lane < p.per && s < a.n_seqs ? seq_len(a, s) : 0;
        const int n = (ln + STEP - 1) / STEP * a.c.nkv;
        const int before = wave_scan(n) - n;
        const int j = __popcll(__ballot(lane < p.per && before <= at)) - 1;
        seq = L * p.per + j;
        len = __builtin_amdgcn_readlane(ln, j);
        at -= __builtin_amdgcn_readlane(before, j);
    }
    const int steps = (len + STEP - 1) / STEP;
    kvh = at / steps;
    step = at % steps;
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

template <int KV, int HD, int STEP>
__global__ void __launch_bounds__((PaShape<KV, HD, STEP>::kThreads)) paged_attn_kernel(PagedAttnArgs a, int whole_pairs) {
    using S = PaShape<KV, HD, STEP>;
    constexpr int NT = S::kTiles, KS = S::kKs, ND = S::kNd, NW = S::kWaves;
    constexpr int EB = KV == kKvF16 ? 2 : 1;
    constexpr int VW = STEP / 4 * EB / 16;  // 16-byte words of a dim's positions per lane
    constexpr int PV = STEP / 32;  // position steps of O
    // pieces of cut (sequence, KV head)s: [.][0] one that began before the wave's share, [.][1] one
    // that begins in it and goes on
    __shared__ __align__(16) float lo[NW][2][kPaRows][HD + 4];
    __shared__ float lm[NW][2][kPaRows], ll[NW][2][kPaRows];
    __shared__ int pair_of[NW][2], ends[NW];  // the pieces' seq * n_kv + kvh (-1: none); whether piece 0 ends there
    const int lane = lane_id(), r = lane & 15, kg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int ps = a.c.ps, psl = 31 - __builtin_clz(ps);

    const PaPlan plan = pa_plan<STEP, NW>(a, gridDim.x);
    // the workgroup's steps, shared out to its waves in the same way
    int g0 = pa_first(plan, blockIdx.x), g1 = pa_first(plan, blockIdx.x + 1);
    int nw = plan.nw, seq = 0, kvh = 0, step = 0, len = 0;
    if (whole_pairs) {  // both ends move up to the next (sequence, KV head)'s beginning
        nw = min(NW, 4);
        auto up = [&](int u) {
            if (u >= plan.total) return plan.total;
            pa_find<STEP>(a, plan, u, seq, kvh, step, len);
            return step > 0 ? u + (len + STEP - 1) / STEP - step : u;
        };
        g0 = up(g0);
        g1 = up(g1);
    }
    const int each = (g1 - g0) / nw, odd = g1 - g0 - each * nw;
    int at = g0 + wave * each + min(wave, odd);
    const int end = wave < nw ? at + each + (wave < odd) : at;
    if (lane < 2) pair_of[wave][lane] = -1;
    if (at < end) pa_find<STEP>(a, plan, at, seq, kvh, step, len);

    while (at < end) {
        const int steps = (len + STEP - 1) / STEP, n = min(end - at, steps - step);
        const int p_end = min(len, (step + n) * STEP);
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
        u4 kr[NT][HD * EB / 64], vr[ND][VW];
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
            for (int i = 0; i < ND; i++)
#pragma unroll
                for (int j = 0; j < VW; j++) __builtin_memcpy(&vr[i][j], base + (size_t)16 * i * ps * EB + 16 * j, 16);
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
        float wref = 0x1p-126f;  // of the lane's head
        f4 o[ND] = {};
        int p0 = step * STEP;
        {
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
            int next = p0 + STEP;
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
            // in LDS they wait where the wave's last piece goes in the end
            uint8_t *ql = (uint8_t *)&lo[wave][1][0][0] + 16 * lane;
#pragma unroll
            for (int st = 0; st < KS; st++) {
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float x = q[st][j] * qs;
                    qhi[st][j] = (_Float16)x;
                    qlo[st][j] = (_Float16)(x - (float)qhi[st][j]);
                }
                if (S::kQInLds) {
                    __builtin_memcpy(ql + 2048 * st, &qhi[st], 16);
                    __builtin_memcpy(ql + 2048 * st + 1024, &qlo[st], 16);
                }
            }
            for (;;) {
                // ---- S^T: lane: head r, positions p0 + STEP/4 kg + 4t + i
                f4 s[NT] = {};
#pragma unroll
                for (int st = 0; st < KS; st++) {
                    if (S::kQInLds) {
                        asm volatile("" ::: "memory");  // read again every step
                        __builtin_memcpy(&qhi[st], ql + 2048 * st, 16);
                        __builtin_memcpy(&qlo[st], ql + 2048 * st + 1024, 16);
                    }
#pragma unroll
                    for (int t = 0; t < NT; t++) {
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
                float smax = -INFINITY;
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
                    }
                bool rescale = __any(smax > m + kSlack);  // uniform
                float f = 1.0f;
                if (rescale) {
                    float mn = max_heads(smax), al;
                    if (KV == kKvF16) {
                        mn = fmaxf(m, mn);
                        f = al = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
                    } else {
                        mn = fmaxf(m, ceilf(mn));
                        al = mn == -INFINITY ? 1.0f : ldexpf(1.0f, (int)fmaxf(m - mn, -256.0f));
                        // O stays as it is while its unit, 2^m wref, can
                        const float w = wref * al;
                        wref = fmaxf(w, 0x1p-126f);
                        f = w * inverse2(wref);
                    }
                    l *= al;
                    m = mn;
                }
                const float ref = m == -INFINITY ? 0.0f : KV == kKvF16 ? m - kLift : m;
                float wi = 1.0f;
                if (KV == kKvInt8) {
                    float wmax = 0.0f;
#pragma unroll
                    for (int t = 0; t < NT; t++)
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const float p = __builtin_amdgcn_exp2f(s[t][i] - ref);
                            l += p;
                            s[t][i] = p * vsc[4 * t + i];
                            wmax = fmaxf(wmax, fabsf(s[t][i]));
                        }
                    if (__any(wmax >= 0x1p15f * wref)) {
                        // the power of two at or below the largest (at most 2^126) becomes 2^kLift
                        const uint32_t e = min(__builtin_bit_cast(uint32_t, max_heads(wmax)) & 0x7f800000u, 0x7e800000u);
                        const float wn = fmaxf(wref, __builtin_bit_cast(float, e) * exp2f(-kLift));
                        f *= wref * inverse2(wn);
                        wref = wn;
                        rescale = true;
                    }
                    wi = inverse2(wref);
                }
                if (rescale) {
#pragma unroll
                    for (int i = 0; i < ND; i++) o[i] *= f;
                }
                h8 phi[PV], plo[PV];
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        float w;
                        if (KV == kKvF16) l += w = __builtin_amdgcn_exp2f(s[t][i] - ref);
                        else w = s[t][i] * wi;
                        // one fp32 value for both parts: a product folded into one of the conversions
                        // would round differently there
                        asm("" : "+v"(w));
                        const _Float16 hi = (_Float16)w;
                        phi[t / 2][4 * (t & 1) + i] = hi;
                        plo[t / 2][4 * (t & 1) + i] = (_Float16)(w - (float)hi);
                    }
                if (KV == kKvInt8 && more) load_scales(next, nxt.v);
                const Pages after = entries(min(next + STEP, len - 1));
                // ---- O^T
                if (KV == kKvF16 && !full) {
                    // what lies past the end may be no number, which a weight of 0 does not hide
#pragma unroll
                    for (int i = 0; i < ND; i++)
#pragma unroll
                        for (int j = 0; j < 4 * VW; j++) {
                            uint32_t w = vr[i][j / 4][j % 4];
                            if (!ok || live <= 2 * j) w = 0;
                            else if (live == 2 * j + 1) w &= 0xffffu;
                            vr[i][j / 4][j % 4] = w;
                        }
                }
#pragma unroll
                for (int i = 0; i < ND; i++)
#pragma unroll
                    for (int k = 0; k < PV; k++) {
                        h8 vf;
                        if (KV == kKvF16) vf = __builtin_bit_cast(h8, vr[i][k]);
                        else vf = cvt8(vr[i][0][2 * k], vr[i][0][2 * k + 1]);
                        o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, phi[k], o[i], 0, 0, 0);
                        o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, plo[k], o[i], 0, 0, 0);
                    }
                if (!more) break;
                load_v(next, nxt.v);
                p0 = next;
                next += STEP;
                cur = nxt;
                nxt = after;
            }
        }
        l = sum_heads(l);
        const bool begins = step == 0, finishes = step + n == steps;
        if (begins && finishes) {
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            float *out = a.out + ((size_t)seq * a.nh + kvh * a.gqa + r) * HD + 4 * kg;
            if (r < a.gqa) {
#pragma unroll
                for (int i = 0; i < ND; i++) {
                    f4 x = o[i] * inv;
                    if (KV == kKvInt8) x *= wref;
                    __builtin_memcpy(out + 16 * i, &x, 16);
                }
            }
        } else {
            if (lane == 0) {
                pair_of[wave][begins] = seq * a.c.nkv + kvh;
                if (!begins) ends[wave] = finishes;
            }
            if (kg == 0) {
                lm[wave][begins][r] = m;
                ll[wave][begins][r] = l;
            }
#pragma unroll
            for (int i = 0; i < ND; i++) {
                f4 x = o[i];
                if (KV == kKvInt8) x *= wref;
                __builtin_memcpy(&lo[wave][begins][r][16 * i + 4 * kg], &x, 16);
            }
        }
        at += n;
        step = 0;
        if (at < end && ++kvh == a.c.nkv) {
            kvh = 0;
            do len = seq_len(a, ++seq);
            while (len == 0);  // a step is left, so a sequence with positions is
        }
    }
    if (__any(plan.empty))  // sequences with no positions: zeros, a KV head's query heads by a wave
        for (int i = blockIdx.x * NW + wave; i < a.n_seqs * a.c.nkv; i += gridDim.x * NW)
            if (seq_len(a, i / a.c.nkv) == 0) {
                const f4 zero = {};
                float *out = a.out + (size_t)i * a.gqa * HD;
                for (int e = 4 * lane; e < a.gqa * HD; e += 256) __builtin_memcpy(out + e, &zero, 16);
            }

    // ---- pieces of one (sequence, KV head), from consecutive waves, are merged.  Lane i holds piece
    // (i / 2, i % 2).  A chain begins with a piece 1, or with piece 0 of the first wave, and takes in
    // the pieces 0 of the waves that follow, up to the next beginning.
    __syncthreads();
    const int pair = lane < 2 * NW ? pair_of[lane >> 1][lane & 1] : -1;
    const bool closes = lane < 2 * NW && !(lane & 1) && pair >= 0 && ends[lane >> 1];
    const uint32_t pieces = (uint32_t)__ballot(pair >= 0), closed = (uint32_t)__ballot(closes);
    const uint32_t starts = pieces & (0xaaaaaaaau | 1u);
    if (threadIdx.x == 0) {
        const int last = 31 - __builtin_clz(starts | 1u), after = ~((2u << last) - 1);
        const bool goes_on = (starts & 2 * 0x55555555u) && (last & 1) && !(closed & after);
        pa_begun(a)[blockIdx.x] = goes_on ? pair_of[last >> 1][1] : -1;
        pa_begun(a)[kPaGroups + blockIdx.x] = pair_of[0][0];
    }
    const int per = a.gqa * (HD / 4);  // elements of four dims
    for (int e = threadIdx.x; e < __popc(starts) * per; e += S::kThreads) {
        const int c = e / per, h = e % per / (HD / 4), d = 4 * (e % (HD / 4));
        uint32_t from = starts;  // from its c-th bit on
        for (int i = 0; i < c; i++) from &= from - 1;
        const int first = __ffs((int)from) - 1;
        const uint32_t rest = from & (from - 1);
        // its pieces: pieces 0 between its beginning and the next one
        const uint32_t in = pieces & 0x55555555u & ~((2u << first) - 1) & (rest ? (rest & (0u - rest)) - 1 : ~0u);
        const int w = first >> 1, k = first & 1, n = __popc(in);
        const bool whole = k == 1 && (in & closed);
        float mm = lm[w][k][h];
#pragma unroll 4
        for (int i = 1; i <= n; i++) mm = fmaxf(mm, lm[w + i][0][h]);
        f4 x = {};
        float sum = 0.0f;
#pragma unroll 4
        for (int i = 0; i <= n; i++) {
            const int ki = i ? 0 : k;
            const float f = mm == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(lm[w + i][ki][h] - mm);
            f4 y;
            __builtin_memcpy(&y, &lo[w + i][ki][h][d], 16);
            x += y * f;
            sum = fmaf(ll[w + i][ki][h], f, sum);
        }
        const int pr = pair_of[w][k];
        if (whole) {
            x *= sum == 0.0f ? 0.0f : 1.0f / sum;
            __builtin_memcpy(a.out + ((size_t)(pr / a.c.nkv) * a.nh + pr % a.c.nkv * a.gqa + h) * HD + d, &x, 16);
        } else {
            float *part = a.ws + (size_t)(2 * blockIdx.x + k) * part_floats(HD);
            __builtin_memcpy(part + 2 * kPaRows + h * HD + d, &x, 16);
            if (d == 0) {
                part[h] = mm;
                part[kPaRows + h] = sum;
            }
        }
    }
}

// Merges the partials of the (sequence, KV head)s that several workgroups share.  Workgroup x looks
// after the one that begins in workgroup x's share and goes on behind it (BY_SHARE), or after
// (sequence, KV head) x itself.  256 threads are HD / 4 lanes of four dims, times CHAIN threads that
// divide the partials among them, times heads.
template <int HD, int CHAIN, bool BY_SHARE>
__global__ void __launch_bounds__(256) paged_merge_kernel(PagedAttnArgs a, int groups) {
    constexpr int D4 = HD / 4, HEADS = 256 / (D4 * CHAIN), BATCH = 4;
    static_assert(kPaGroups == 256, "a lane reads four entries");
    __shared__ __align__(16) float so[CHAIN > 1 ? CHAIN : 1][HEADS][HD];
    __shared__ float sm[CHAIN][HEADS], sl[CHAIN][HEADS];
    const int *begun = pa_begun(a);
    int b[4], t[4], pair = blockIdx.x, w0 = blockIdx.x, n = 0;
    __builtin_memcpy(t, begun + kPaGroups + 4 * lane_id(), 16);
    if (BY_SHARE) pair = begun[blockIdx.x];
    else {
        __builtin_memcpy(b, begun + 4 * lane_id(), 16);
        w0 = -1;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint64_t at = __ballot(4 * lane_id() + i < groups && b[i] == pair);
            if (at) w0 = 4 * (__ffsll((unsigned long long)at) - 1) + i;
        }
    }
    if (pair < 0 || w0 < 0) return;  // nothing, or finished in one workgroup
#pragma unroll
    for (int i = 0; i < 4; i++) n += __popcll(__ballot(4 * lane_id() + i < groups && t[i] == pair));
    const int w1 = w0 + n, seq = pair / a.c.nkv, kvh = pair % a.c.nkv;
    const int dl = threadIdx.x % D4, g = threadIdx.x / D4 % CHAIN, hh = threadIdx.x / (D4 * CHAIN);
    constexpr int PART = part_floats(HD);
    for (int h0 = blockIdx.y * HEADS; h0 < a.gqa; h0 += gridDim.y * HEADS) {
        const int h = min(h0 + hh, a.gqa - 1);
        float m = -INFINITY, l = 0.0f;
        f4 o = {};
        for (int w = w0 + g; w <= w1; w += CHAIN * BATCH) {
            float pm[BATCH], pl[BATCH];
            f4 x[BATCH];
#pragma unroll
            for (int i = 0; i < BATCH; i++) {  // all loads of a batch go out together
                const int v = min(w + CHAIN * i, w1);
                // the first workgroup holds its beginning in its second slot, the others in the first
                const float *p = a.ws + (size_t)(2 * v + (v == w0)) * PART;
                pm[i] = w + CHAIN * i <= w1 ? p[h] : -INFINITY;
                pl[i] = p[kPaRows + h];
                __builtin_memcpy(&x[i], p + 2 * kPaRows + h * HD + 4 * dl, 16);
            }
            float mn = m;
#pragma unroll
            for (int i = 0; i < BATCH; i++) mn = fmaxf(mn, pm[i]);
            // partials without a maximum are taken in, too: their sums are 0, or NaN where every score is one
            const float ref = mn == -INFINITY ? 0.0f : mn;
            const float fa = __builtin_amdgcn_exp2f(m - ref);
            l *= fa;
            o *= fa;
#pragma unroll
            for (int i = 0; i < BATCH; i++) {
                const float f = __builtin_amdgcn_exp2f(pm[i] - ref);
                l = fmaf(pl[i], f, l);
                o += x[i] * f;
            }
            m = mn;
        }
        if (CHAIN > 1) {
            __syncthreads();  // the last heads' sums are read
            __builtin_memcpy(&so[g][hh][4 * dl], &o, 16);
            if (dl == 0) {
                sm[g][hh] = m;
                sl[g][hh] = l;
            }
            __syncthreads();
            if (g > 0) continue;
            float mm = sm[0][hh];
#pragma unroll
            for (int i = 1; i < CHAIN; i++) mm = fmaxf(mm, sm[i][hh]);
            l = 0.0f;
            o = f4{};
#pragma unroll
            for (int i = 0; i < CHAIN; i++) {
                const float f = mm == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(sm[i][hh] - mm);
                f4 y;
                __builtin_memcpy(&y, &so[i][hh][4 * dl], 16);
                l = fmaf(sl[i][hh], f, l);
                o += y * f;
            }
        }
        if (h0 + hh < a.gqa) {
            o *= l == 0.0f ? 0.0f : 1.0f / l;
            __builtin_memcpy(a.out + ((size_t)seq * a.nh + kvh * a.gqa + h) * HD + 4 * dl, &o, 16);
        }
    }
}

template <int KV, int HD, int STEP>
static void launch_pa(const PagedAttnArgs &a, hipStream_t s) {
    using S = PaShape<KV, HD, STEP>;
    constexpr int CHAIN = 1024 / HD;  // 256 threads for one head
    const long long pairs = (long long)a.n_seqs * a.c.nkv;
    const long long most = pairs * (((long long)a.max_pages * a.c.ps + STEP - 1) / STEP);  // steps
    const int groups = (int)(most < kPaGroups ? most : kPaGroups);
    // Tables of up to four steps: no (sequence, KV head) is cut between workgroups, and nothing is left to merge (100
    // sequences to 60 positions 7.0 us against 9.2 with the merge launch).  Longer ones are cut: 300 positions of one
    // sequence take 11.3 us on 4 CUs against 8.3 on 40, the merge launch included.
    const bool whole_pairs = most <= 4 * pairs;
    hipLaunchKernelGGL((paged_attn_kernel<KV, HD, STEP>), dim3(groups), dim3(S::kThreads), 0, s, a, (int)whole_pairs);
    if (whole_pairs) return;
    // few (sequence, KV head)s: long chains, a workgroup for each head; many: short ones, found by the shares' ends
    if (pairs < groups)
        hipLaunchKernelGGL((paged_merge_kernel<HD, CHAIN, false>), dim3((int)pairs, a.gqa), dim3(256),
                           0, s, a, groups);
    else
        hipLaunchKernelGGL((paged_merge_kernel<HD, 1, true>), dim3(groups - 1, 1), dim3(256), 0, s, a,
                           groups);
}

int launch_paged_attention(const PagedAttnArgs &a, hipStream_t s) {
    const bool f16 = a.c.kv_type == kKvF16;
    // Steps of 64 positions read whole lines of V where pages hold 64 or more, and halve what a step costs besides its
    // loads: 96 sequences to 8192 (8 KV heads of 128) 173.7 us against 188.0 with steps of 32, one of 32,768 20.7
    // against 23.2.  Few steps are spread thinner by 32: 300 positions 8.4 us against 9.3, 100 sequences to 60
    // positions 7.2 against 8.0; 40 to 250, 2 KV heads of 256, 11.3 against 16.2 (to 8192: 37.1 against 33.9).
    const bool few = (long long)a.n_seqs * a.c.nkv * a.max_pages * a.c.ps <= 32 * 1024;
    if (a.c.hd == 64) f16 ? launch_pa<kKvF16, 64, 64>(a, s) : launch_pa<kKvInt8, 64, 64>(a, s);
    else if (!f16) a.c.hd == 128 ? launch_pa<kKvInt8, 128, 64>(a, s) : launch_pa<kKvInt8, 256, 64>(a, s);
    else if (a.c.hd == 128) few ? launch_pa<kKvF16, 128, 32>(a, s) : launch_pa<kKvF16, 128, 64>(a, s);
    else few ? launch_pa<kKvF16, 256, 32>(a, s) : launch_pa<kKvF16, 256, 64>(a, s);
    return check_launch("paged_attention_decode");
}

// ------------------------------------------------------------------ preparation of new tokens
// HD / 8 lanes own a head, four rotated pairs (j, j + HD/2) each.  The angle of pair j at position p
// is p turn(j) in units of 2^-64 of a turn, formed in integers (the product keeps its low 64 bits,
// whole turns fall off): off by less than 10 p 2^-64 of a turn, where fp32 angles are off by p 2^-24.
// What is left of a turn is rounded to fp32 for the sine and cosine.
//
// A row that is stored (k, v) as the cache's elements, and its int8 scale.  A row whose largest
// value is below 1e-36 (127 / m leaves the range) is stored as zeros.  The largest value is found
// among the bits, where a NaN is the largest of all: a row with a NaN or an infinity has that for
// its scale and zeros for elements, so that all of it reads as NaN.
template <int KV>
struct CacheRow {
    uint32_t w0[KV == kKvF16 ? 2 : 1], w1[KV == kKvF16 ? 2 : 1];  // elements 4l .. 4l + 3, HD/2 + 4l ..
    float scale;
};
template <int KV, int LPH>
__device__ __forceinline__ CacheRow<KV> cache_row(const float (&x0)[4], const float (&x1)[4]) {
    CacheRow<KV> r;
    if (KV == kKvF16) {
        r.scale = 1.0f;
        const h4 a = {(_Float16)x0[0], (_Float16)x0[1], (_Float16)x0[2], (_Float16)x0[3]};
        const h4 b = {(_Float16)x1[0], (_Float16)x1[1], (_Float16)x1[2], (_Float16)x1[3]};
        __builtin_memcpy(r.w0, &a, 8);
        __builtin_memcpy(r.w1, &b, 8);
    } else {
        uint32_t mb = 0;
#pragma unroll
        for (int i = 0; i < 4; i++)
            mb = max(mb, max(__builtin_bit_cast(uint32_t, fabsf(x0[i])), __builtin_bit_cast(uint32_t, fabsf(x1[i]))));
#pragma unroll
        for (int o = 1; o < LPH; o <<= 1) mb = max(mb, (uint32_t)__shfl_xor((int)mb, o));
        const float m = __builtin_bit_cast(float, mb);
        const float inv = m < 1e-36f ? 0.0f : 127.0f / m;
        r.scale = m < 1e-36f ? 0.0f : m / 127.0f;
        r.w0[0] = r.w1[0] = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int a = (int)fminf(fmaxf(rintf(x0[i] * inv), -127.0f), 127.0f);
            const int b = (int)fminf(fmaxf(rintf(x1[i] * inv), -127.0f), 127.0f);
            r.w0[0] |= (uint32_t)(a & 255) << (8 * i);
            r.w1[0] |= (uint32_t)(b & 255) << (8 * i);
        }
        if (mb >= 0x7f800000u) r.w0[0] = r.w1[0] = 0;
    }
    return r;
}

// Sequence and position of token t (position -1: padding, sequence -1: not stored), and its page.  Where positions come
// with lengths, a token at its row's length or behind it is not stored: the row was not extended for it.
struct Token { int seq, pos, page; };
__device__ __forceinline__ Token token_of(const PagedPrepArgs &a, int t) {
    Token k;
    k.seq = a.seq ? a.seq[t] : t;
    k.pos = a.pos ? a.pos[t] : a.lens[t] - 1;
    const int i = k.pos / a.c.ps;
    const bool in = (unsigned)k.seq < (unsigned)a.n_seqs && k.pos >= 0 && i < a.max_pages;
    int end = INT_MAX;
    if (in && a.pos && a.lens) end = a.lens[k.seq];
    k.page = in ? a.table[(size_t)k.seq * a.max_pages + i] : -1;
    if ((unsigned)k.page >= (unsigned)a.c.n_pages || k.pos >= end) k.page = -1;
    return k;
}

// The row of V at position off of page and head r: one element in each of HD rows of positions.
template <int KV, int HD>
__device__ __forceinline__ void store_v(const PagedCache &c, const CacheRow<KV> &row, size_t r, int off, int l) {
    constexpr int EB = KV == kKvF16 ? 2 : 1;
    uint8_t *dst = (uint8_t *)c.v + (r * HD * c.ps + off) * EB;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        __builtin_memcpy(dst + (size_t)(4 * l + i) * c.ps * EB, (const uint8_t *)row.w0 + i * EB, EB);
        __builtin_memcpy(dst + (size_t)(HD / 2 + 4 * l + i) * c.ps * EB, (const uint8_t *)row.w1 + i * EB, EB);
    }
}

constexpr int kVTokens = 64;  // tokens of a tile of V, at head_dim 64 and 128; half of that at 256
constexpr int kFewBlocks = 2048;  // resident at once
typedef f4 f4a4 __attribute__((aligned(4)));

// With V_TILES the first v_blocks take kVTokens tokens of one V head through LDS: V pages hold the
// positions of a dim side by side, so eight tokens in a row that fill a group of eight positions are
// one store per dim instead of eight of one element each.  Tokens outside such groups are stored
// singly.  The other blocks take one token each and gridDim.y-th parts of its heads: q heads, then k,
// then (V_TILES false) v.
template <int KV, int HD, bool V_TILES>
__global__ void __launch_bounds__(256) paged_prep_kernel(PagedPrepArgs a, int v_blocks) {
    constexpr int LPH = HD / 8, HALF = HD / 2, EB = KV == kKvF16 ? 2 : 1;
    constexpr int PER = 256 / LPH;  // heads (or tokens) of a pass
    constexpr int VT = HD == 256 ? kVTokens / 2 : kVTokens;
    constexpr int ROW = VT * EB + 8;  // bytes of a dim in the tile
    __shared__ float cs[HALF], sn[HALF];
    __shared__ __align__(16) uint8_t tile[V_TILES ? HD * ROW : 4];
    __shared__ int tpage[V_TILES ? VT : 1], tpos[V_TILES ? VT : 1], column[V_TILES ? VT : 1];
    __shared__ int lead[V_TILES ? VT / 8 : 1], groups;
    const int tid = threadIdx.x, l = tid % LPH, nkv = a.c.nkv, ps = a.c.ps;
    if (!V_TILES || (int)blockIdx.x >= v_blocks) {
        const int t = blockIdx.x - v_blocks;
        const int heads = a.nh + nkv * (V_TILES ? 1 : 2);
        // the rows of a pass are loaded before the last pass is worked on, the first ones before the
        // token's position is known
        float x0[4], x1[4], n0[4], n1[4];
        auto load = [&](int h0, float(&u)[4], float(&v)[4]) {
            const int head = min(h0 + tid / LPH, heads - 1);
            const float *src = head < a.nh ? a.q + ((size_t)t * a.nh + head) * HD
                               : head < a.nh + nkv ? a.k + ((size_t)t * nkv + head - a.nh) * HD
                                                   : a.v + ((size_t)t * nkv + head - a.nh - nkv) * HD;
            __builtin_memcpy(u, src + 4 * l, 16);
            __builtin_memcpy(v, src + HALF + 4 * l, 16);
        };
        uint64_t turn = a.turn0;  // of pair tid
#pragma unroll
        for (int i = 0; (1 << i) < HALF; i++) {
            const uint64_t next = __umul64hi(turn, a.step[i]);
            turn = tid >> i & 1 ? next : turn;
        }
        load(blockIdx.y * PER, x0, x1);
        const Token k = token_of(a, t);
        if (k.pos < 0) return;
        if (tid < HALF) {
            const int32_t frac = (int32_t)(((uint64_t)(uint32_t)k.pos * turn) >> 32);  // of a turn, in 2^-32
            sincospif((float)frac * 0x1p-31f, &sn[tid], &cs[tid]);
        }
        lds_barrier();
        const int off = k.pos % ps, by = gridDim.y * PER;
        for (int h0 = blockIdx.y * PER; h0 < heads; h0 += by) {
            if (h0 > (int)blockIdx.y * PER) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    x0[i] = n0[i];
                    x1[i] = n1[i];
                }
            }
            if (h0 + by < heads) load(h0 + by, n0, n1);
            const int head = h0 + tid / LPH;
            const bool is_q = head < a.nh, is_k = !is_q && head < a.nh + nkv;
            const int h = is_q ? head : is_k ? head - a.nh : head - a.nh - nkv;
            if (head >= heads) continue;
            if (is_q || is_k) {
                if (a.qw) {
                    const float *w = is_q ? a.qw : a.kw;
                    float ss = 0.0f, w0[4], w1[4];
                    __builtin_memcpy(w0, w + 4 * l, 16);
                    __builtin_memcpy(w1, w + HALF + 4 * l, 16);
#pragma unroll
                    for (int i = 0; i < 4; i++) ss = fmaf(x0[i], x0[i], fmaf(x1[i], x1[i], ss));
#pragma unroll
                    for (int o = 1; o < LPH; o <<= 1) ss += __shfl_xor(ss, o);
                    const float g = __builtin_amdgcn_rsqf(ss * (1.0f / HD) + a.eps);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        x0[i] = x0[i] * g * w0[i];
                        x1[i] = x1[i] * g * w1[i];
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
                if (a.q_streams) {
                    __builtin_nontemporal_store(f4{x0[0], x0[1], x0[2], x0[3]}, (f4a4 *)(dst + 4 * l));
                    __builtin_nontemporal_store(f4{x1[0], x1[1], x1[2], x1[3]}, (f4a4 *)(dst + HALF + 4 * l));
                } else {
                    __builtin_memcpy(dst + 4 * l, x0, 16);
                    __builtin_memcpy(dst + HALF + 4 * l, x1, 16);
                }
                continue;
            }
            if (k.page < 0) continue;
            const CacheRow<KV> row = cache_row<KV, LPH>(x0, x1);
            const size_t r = (size_t)k.page * nkv + h;
            if (is_k) {
                uint8_t *dst = (uint8_t *)a.c.k + (r * ps + off) * HD * EB;
                __builtin_memcpy(dst + 4 * l * EB, row.w0, 4 * EB);
                __builtin_memcpy(dst + (HALF + 4 * l) * EB, row.w1, 4 * EB);
            } else {
                store_v<KV, HD>(a.c, row, r, off, l);
            }
            if (KV == kKvInt8 && l == 0) (is_k ? a.c.ksc : a.c.vsc)[r * ps + off] = row.scale;
        }
        return;
    }
    if (V_TILES) {
        const int b = blockIdx.x * gridDim.y + blockIdx.y;
        const int t0 = b / nkv * VT, h = b % nkv;
        if (t0 >= a.n_tokens) return;
        const int n = min(VT, a.n_tokens - t0);
        constexpr int PASSES = VT / PER;
        float x0[PASSES][4], x1[PASSES][4];
#pragma unroll
        for (int u = 0; u < PASSES; u++) {  // one round trip, together with the tokens' places
            const float *src = a.v + ((size_t)(t0 + min(u * PER + tid / LPH, n - 1)) * nkv + h) * HD;
            __builtin_memcpy(x0[u], src + 4 * l, 16);
            __builtin_memcpy(x1[u], src + HALF + 4 * l, 16);
        }
        if (tid < VT) {  // a lane of one wave per token
            static_assert(VT <= 64, "one wave");
            Token k = {-1, -1, -1};
            if (tid < n) k = token_of(a, t0 + tid);
            // groups of 8 positions that lie whole and in order in the tile, by the token that leads them (a page
            // holds whole groups); the g-th takes columns 8g .. 8g + 7
            const int page = __shfl_up(k.page, 1), pos = __shfl_up(k.pos, 1);
            const uint64_t next = __ballot(tid > 0 && k.page >= 0 && k.page == page && k.pos == pos + 1);
            const bool leads = k.page >= 0 && k.pos % 8 == 0 && tid <= VT - 8 && ((next >> tid) >> 1 & 127) == 127;
            const uint64_t leaders = __ballot(leads);
            uint64_t led = leaders | leaders << 1;
            led |= led << 2;
            led |= led << 4;  // each leader and the seven after it
            const int g = __popcll(leaders & ((2ull << tid) - 1)) - 1;
            tpage[tid] = k.page;
            tpos[tid] = k.pos;
            column[tid] = led >> tid & 1 ? 8 * g + k.pos % 8 : -1;
            if (leads) lead[g] = tid;
            if (tid == 0) groups = __popcll(leaders);
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < PASSES; u++) {
            const int i = u * PER + tid / LPH;
            const CacheRow<KV> row = cache_row<KV, LPH>(x0[u], x1[u]);
            if (i >= n || tpage[i] < 0) continue;
            const size_t r = (size_t)tpage[i] * nkv + h;
            if (column[i] >= 0) {
                uint8_t *dst = &tile[column[i] * EB];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    __builtin_memcpy(dst + (4 * l + j) * ROW, (const uint8_t *)row.w0 + j * EB, EB);
                    __builtin_memcpy(dst + (HALF + 4 * l + j) * ROW, (const uint8_t *)row.w1 + j * EB, EB);
                }
            } else store_v<KV, HD>(a.c, row, r, tpos[i] % ps, l);
            if (KV == kKvInt8 && l == 0) a.c.vsc[r * ps + tpos[i] % ps] = row.scale;
        }
        __syncthreads();
        for (int e = tid; e < groups * HD; e += 256) {
            const int d = e % HD, g = e / HD, i = lead[g];
            uint2 w[EB];  // 8 elements
            __builtin_memcpy(w, __builtin_assume_aligned(&tile[d * ROW + 8 * g * EB], 8), 8 * EB);
            __builtin_memcpy((uint8_t *)a.c.v + ((((size_t)tpage[i] * nkv + h) * HD + d) * ps + tpos[i] % ps) * EB, w,
                             8 * EB);
        }
    }
}

int launch_paged_prep(PagedPrepArgs &a, double theta, hipStream_t s) {
    const int hd = a.c.hd;
    // A turn per position is theta^(-2j/hd) / (2 pi) for pair j: the kernel forms it from theta^(-2 2^i/hd), in whole
    // numbers of 2^-64.  The largest i gives 1 / sqrt(theta), the others are its square roots, each of which halves what
    // the last is off by (squares would double it).  Seven products cut off below 1 each, their factors are off by at
    // most 1.5 (times a turn of 0.16 at most): together below 10 of 2^-64, 7.5 at most over 1000 values of theta from 1
    // to 3e38 in extended precision.  At position 2^31 that is 2^-29.7 of a turn.
    long double step = 1.0L / sqrtl(theta);  // <= 1
    a.turn0 = (uint64_t)(0x1p64L / (2.0L * 3.14159265358979323846264338327950288L));
    for (int i = hd == 64 ? 4 : hd == 128 ? 5 : 6; i >= 0; i--) {
        a.step[i] = step < 1.0L ? (uint64_t)rintl(step * 0x1p64L) : UINT64_MAX;
        step = sqrtl(step);
    }
    // V through tiles where runs of tokens can be expected (a call by lengths has one token per sequence) and
    // there are enough tiles to hide their two phases behind the other blocks: 4 KV heads of 128, f16, 256
    // tokens 5.7 us with tiles against 5.3, 400 6.5 either way, 1899 21.9 against 25.7; 12 heads of 64, 2000
    // tokens 7.2 against 15.0; 2 heads of 256, 1000 tokens 9.1 against 8.9.
    const bool tiles = a.pos && (long long)a.n_tokens * a.c.nkv >= 2048;
    // Few tokens: a workgroup for every pass of heads; many: two per token, whose passes overlap (64 + 4
    // heads of 128, 1899 tokens: 21.9 us, 23.8 with five workgroups per token, 22.8 with one).
    const int per = 2048 / hd, heads = a.nh + a.c.nkv * (tiles ? 1 : 2), parts = (heads + per - 1) / per;
    const int y = (long long)a.n_tokens * parts <= kFewBlocks ? parts : min(parts, 2);
    // queries that outgrow an XCD's L2 (4 MB) are stored past it: 1899 tokens into an int8 cache 25.6 us where the
    // stores through it take 31.6 and evict the pages, too; 800 tokens 9.7 against 11.6
    a.q_streams = (long long)a.n_tokens * a.nh * hd * 4 > 4 << 20;
    const int vt = hd == 256 ? kVTokens / 2 : kVTokens;
    const int v_blocks = tiles ? ((a.n_tokens + vt - 1) / vt * a.c.nkv + y - 1) / y : 0;
    const dim3 grid(a.n_tokens + v_blocks, y);
#define MNEMO_PREP2(KV_, HD_)                                                                                       \
    do {                                                                                                            \
        if (tiles) hipLaunchKernelGGL((paged_prep_kernel<KV_, HD_, true>), grid, dim3(256), 0, s, a, v_blocks);     \
        else hipLaunchKernelGGL((paged_prep_kernel<KV_, HD_, false>), grid, dim3(256), 0, s, a, v_blocks);          \
    } while (0)
#define MNEMO_PREP(HD_)                                        \
    do {                                                       \
        if (a.c.kv_type == kKvF16) MNEMO_PREP2(kKvF16, HD_);   \
        else MNEMO_PREP2(kKvInt8, HD_);                        \
    } while (0)
    if (hd == 64) MNEMO_PREP(64);
    else if (hd == 128) MNEMO_PREP(128);
    else MNEMO_PREP(256);
#undef MNEMO_PREP
#undef MNEMO_PREP2
    return check_launch("paged_attn_prep");
}

}  // namespace mnemo
