// paged_prompt.hip -- attention of several new tokens per sequence over a pool of cache pages: prompts, chunks of
// prompts, drafted tokens, and single ones among them.
//
// Sequence s has n tokens, rows starts[s] .. starts[s+1]-1 of q, the last of them at position L - 1 (L = lens[s]).
// Token i, at p = L - n + i:  out = sum_{j<=p} P_j v_j / sum_{j<=p} P_j,  P_j = exp(scale q.k_j - m).
//
// A tile is the query heads of one KV head for a power of two of tokens, 128 rows (64 at head_dim 256): 4 waves of
// 32 (16) rows share the K and V of 64 positions, a step, in LDS.  The steps of all tiles stand in one row,
// [sequence][KV head][tile][step], which the workgroups divide into equal shares, whatever the lengths are: the sum
// of a sequence's steps has a closed form, so every workgroup finds its share by itself.  A tile that several
// shares cut leaves partials (max, sum, O) in memory, which a second launch merges.
//
// S^T = K Q^T (positions x rows) leaves a lane with positions of one row, which is how O^T = V^T P^T (dims x rows)
// wants P^T, when the K rows of a tile are picked so: lane row m of tile t is position 16 (m/4) + 4t + m%4, so that
// a lane's positions over the tiles are 16 consecutive ones.  Words of 16 bytes in LDS are permuted within their
// row, so that the 16 lanes of an operand's column lie in different banks.
//
// Precision: as in paged_attn.hip, Q is scaled by a power of two per row and split into two f16 parts; f16 pages: P likewise,
// relative to a reference that follows the maximum only when a score exceeds it by 2^kSlack, and 2^kLift at the
// reference.  int8 pages: K enters as f16 (exact), P times the value's scale as three bf16 parts (24 bits,
// the range of fp32), V as bf16 (exact).
#include <limits.h>
#include <math.h>

#include "mfma_types.hpp"
#include "mnemo_common.hpp"
#include "mnemo_internal.hpp"

namespace mnemo {

namespace {

constexpr float kSlack = 5.0f, kLift = 9.0f;  // powers of two
constexpr int kStep = 64;                     // positions
constexpr int kWaves = 4, kThreads = 64 * kWaves;
constexpr int kGroups = 512;                  // workgroups, two per CU

template <int HD>
struct Shape {
    static constexpr int RT = HD == 256 ? 1 : 2;  // tiles of 16 rows per wave
    static constexpr int kRows = 16 * RT * kWaves;
    static constexpr int kKs = HD / 32, kNd = HD / 16;  // dim steps of S, dim tiles of O
};

// Workspace: two partials per workgroup (max [rows], sum [rows], O [rows][hd]), and what they are: begun[g] describes the
// tile that begins in workgroup g's share and goes on behind it (its second partial), taken[g] is the first step of the
// tile that it goes on with from the workgroup before (its first), -1 for none.
__host__ __device__ constexpr int rows_of(int hd) { return hd == 256 ? 64 : 128; }
__host__ __device__ constexpr int part_floats(int hd) { return rows_of(hd) * (hd + 2); }
struct Begun {
    int first;  // first step, -1 for none
    int row0, n_rows, kvh;  // first token (row of q), rows in use, KV head
};
__device__ __forceinline__ Begun *begun_of(const PagedPromptArgs &a) {
    return (Begun *)(a.ws + (size_t)2 * kGroups * part_floats(a.c.hd));
}
__device__ __forceinline__ int *taken_of(const PagedPromptArgs &a) { return (int *)(begun_of(a) + kGroups); }

// ------------------------------------------------------------------ the row of steps
struct Seq {
    int start, n, len;  // first row of q, tokens, positions
};
__device__ __forceinline__ Seq seq_of(const PagedPromptArgs &a, int s) {
    Seq q;
    q.start = min(max(a.starts[s], 0), a.n_tokens);
    q.n = min(max(a.starts[s + 1], q.start), a.n_tokens) - q.start;
    q.len = min(max(a.lens[s], 0), a.max_pages * a.c.ps);
    return q;
}

// x (x + 1) / 2 modulo 2^32
__device__ __forceinline__ uint32_t triangle(uint32_t x) { return x & 1 ? x * ((x + 1) / 2) : (x / 2) * (x + 1); }

// The steps of the first j tiles of 2^tl tokens, none of them the sequence's last: the sum over i = 1 .. j of
// ceil(max(b + i 2^tl, 0) / 64), b = len - n.
__device__ __forceinline__ int steps_before(const Seq &s, int tl, int j) {
    int b = s.len - s.n;
    if (b < 0) {  // tiles of tokens before position 0 have no steps
        const int none = min(-b >> tl, j);
        j -= none;
        b += none << tl;
        if (b <= -(1 << tl)) return 0;
    }
    if (tl > 6) return j * (j + 1) * (1 << (tl - 7)) + j * ((b + 63) >> 6);
    const int gl = 6 - tl;
    const uint32_t c = (uint32_t)(b + (1 << tl) - 1) >> tl, d = c + (uint32_t)j;  // ceil(u / 2^gl) from u = c + 1 to d
    auto sum = [&](uint32_t x) { return (triangle(x >> gl) << gl) + (x & ((1u << gl) - 1)) * ((x >> gl) + 1); };
    return (int)(sum(d) - sum(c));
}
__device__ __forceinline__ int tiles_of(const Seq &s, int tl) { return (s.n + (1 << tl) - 1) >> tl; }
// of one KV head
__device__ __forceinline__ int steps_of(const Seq &s, int tl) {
    if (s.n == 0 || s.len == 0) return 0;
    return steps_before(s, tl, tiles_of(s, tl) - 1) + (s.len + kStep - 1) / kStep;
}

struct Plan {
    int total;       // steps
    int groups;      // workgroups that have some
    int base, more;  // steps of a workgroup; the first `more` of them have one more
    bool short_;     // lane: a sequence of its has tokens before position 0
    int per;         // sequences per lane of the sums
    int before;      // lane: steps before its sequences
};
__device__ __forceinline__ Plan make_plan(const PagedPromptArgs &a) {
    Plan p;
    p.per = (a.n_seqs + 63) / 64;
    p.short_ = false;
    const int s0 = lane_id() * p.per;
    int sum = 0;
    for (int i = 0; i < p.per; i++)
        if (s0 + i < a.n_seqs) {
            const Seq s = seq_of(a, s0 + i);
            p.short_ |= s.n > s.len;
            sum += steps_of(s, a.tl);
        }
    sum *= a.c.nkv;
    const int incl = wave_scan(sum);
    p.total = __builtin_amdgcn_readlane(incl, 63);
    p.before = incl - sum;
    p.groups = max(min(kGroups, p.total), 1);
    p.base = p.total / p.groups;
    p.more = p.total - p.base * p.groups;
    return p;
}
__device__ __forceinline__ int first_of(const Plan &p, int g) {
    return g >= p.groups ? p.total : g * p.base + min(g, p.more);
}

struct Where {
    Seq s;
    int seq, kvh, tile, step, steps;
};
// The tile of step u, and the step within it.
__device__ __forceinline__ Where find(const PagedPromptArgs &a, const Plan &p, int u) {
    // the last lane that begins at or before u holds it (lanes without steps share their successor's beginning)
    const int lane = lane_id(), L = __popcll(__ballot(p.before <= u)) - 1;
    int at = u - __builtin_amdgcn_readlane(p.before, L);
    Where w;
    w.seq = L;
    if (p.per > 1) {
        const int s = L * p.per + lane;
        const bool in = lane < p.per && s < a.n_seqs;
        const int n = in ? steps_of(seq_of(a, s), a.tl) * a.c.nkv : 0;
        const int before = wave_scan(n) - n;
        const int j = __popcll(__ballot(lane < p.per && before <= at)) - 1;
        w.seq = L * p.per + j;
        at -= __builtin_amdgcn_readlane(before, j);
    }
    w.seq = __builtin_amdgcn_readfirstlane(w.seq);
    w.s = seq_of(a, w.seq);
    const int each = steps_of(w.s, a.tl);
    w.kvh = at / each;
    at -= w.kvh * each;
    int lo = 0, hi = tiles_of(w.s, a.tl) - 1;  // the last tile that begins at or before the step
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (steps_before(w.s, a.tl, mid) <= at) lo = mid;
        else hi = mid - 1;
    }
    w.tile = lo;
    w.step = at - steps_before(w.s, a.tl, lo);
    const int end = w.s.len - w.s.n + min((lo + 1) << a.tl, w.s.n);  // positions that the tile's last token sees
    w.steps = (end + kStep - 1) / kStep;
    return w;
}

// max over the four lanes that share a row (lane % 16), in all of them
__device__ __forceinline__ float max_row(float v) {
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float sum_row(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

// ------------------------------------------------------------------ LDS
// Word c of K row p (a position of the step), and of V row d (a dim): their places in 16-byte words.
template <int HD>
__device__ __forceinline__ int k_word(int p, int c) {
    const int m = ((p >> 4) & 3) * 4 + (p & 3);  // the row's lane in an operand
    return p * (HD / 8) + (c ^ (HD == 64 ? m >> 1 : m));
}
__device__ __forceinline__ int v_word(int d, int c) { return d * (kStep / 8) + (c ^ ((d >> 1) & 7)); }

// 8 int8 as bf16, exact
__device__ __forceinline__ u4 int8_bf16(uint32_t a, uint32_t b) {
    u4 w;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t x = i < 2 ? a : b;
        const float lo = (float)(int8_t)(x >> (16 * (i & 1))), hi = (float)(int8_t)(x >> (16 * (i & 1) + 8));
        w[i] = __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, hi), __builtin_bit_cast(uint32_t, lo), 0x07060302u);
    }
    return w;
}

template <int KV, int HD>
__global__ void __launch_bounds__(kThreads, 2) paged_prompt_kernel(PagedPromptArgs a) {
    using S = Shape<HD>;
    constexpr int RT = S::RT, KS = S::kKs, ND = S::kNd;
    constexpr int EB = KV == kKvF16 ? 2 : 1;
    constexpr int NL = kStep * HD * EB / 16 / kThreads;  // 16-byte loads per thread of K, and of V
    __shared__ u4 kt[kStep * HD / 8], vt[kStep * HD / 8];
    __shared__ __align__(16) float ksc[KV == kKvInt8 ? kStep : 4], vsc[KV == kKvInt8 ? kStep : 4];
    __shared__ uint32_t odd[2][2];  // by the step's parity: positions with values that are none
    const int lane = lane_id(), r = lane & 15, kg = lane >> 4, tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int ps = a.c.ps, psl = 31 - __builtin_clz(ps);
    // neighbouring shares, which read the same pages, on one XCD
    const int g = (blockIdx.x & 7) * (kGroups / 8) + (blockIdx.x >> 3);

    const Plan plan = make_plan(a);
    int at = first_of(plan, g);
    const int end = first_of(plan, g + 1);
    if (tid == 0) {
        begun_of(a)[g].first = -1;
        taken_of(a)[g] = -1;
    }
    if (tid < 4) odd[tid >> 1][tid & 1] = 0;
    int parity = 0;
    __syncthreads();

    while (at < end) {
        const Where w = find(a, plan, at);
        const Seq sq = w.s;
        const int n = min(end - at, w.steps - w.step);
        const int tok0 = w.tile << a.tl, toks = min(1 << a.tl, sq.n - tok0);
        const int *table = a.table + (size_t)w.seq * a.max_pages;
        const int pos0 = sq.len - sq.n + tok0;  // of the tile's first token
        const uint8_t *kc = (const uint8_t *)a.c.k, *vc = (const uint8_t *)a.c.v;

        // ---- the lane's rows
        int lim[RT];  // last position that the row sees
        size_t io[RT];  // of its query and output
        bool used[RT];
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            const int row = (wave * RT + rt) * 16 + r, tok = row / a.gqa, head = row - tok * a.gqa;
            used[rt] = tok < toks;
            lim[rt] = used[rt] ? pos0 + tok : INT_MAX;  // what other rows give is dropped
            io[rt] = ((size_t)(sq.start + tok0 + (used[rt] ? tok : 0)) * a.nh + w.kvh * a.gqa + (used[rt] ? head : 0)) * HD;
        }
        int lim_max = -1, lim_min = INT_MAX;
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            lim_max = max(lim_max, used[rt] ? lim[rt] : -1);
            lim_min = min(lim_min, lim[rt]);
        }
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) {
            lim_max = max(lim_max, __shfl_xor(lim_max, o));
            lim_min = min(lim_min, __shfl_xor(lim_min, o));
        }
        lim_max = __builtin_amdgcn_readfirstlane(lim_max);
        lim_min = __builtin_amdgcn_readfirstlane(lim_min);

        // ---- Q
        h8 qhi[RT][KS], qlo[RT][KS];
        float c[RT];
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            float q[KS][8], qm = 0.0f;
#pragma unroll
            for (int st = 0; st < KS; st++) {
                __builtin_memcpy(&q[st][0], a.q + io[rt] + 32 * st + 8 * kg, 16);
                __builtin_memcpy(&q[st][4], a.q + io[rt] + 32 * st + 8 * kg + 4, 16);
            }
#pragma unroll
            for (int st = 0; st < KS; st++)
#pragma unroll
                for (int j = 0; j < 8; j++) qm = fmaxf(qm, fabsf(q[st][j]));
            qm = max_row(qm);
            const int qe = (int)((__builtin_bit_cast(uint32_t, qm) >> 23) & 255) - 127;  // exponent of the largest
            const float qs = ldexpf(1.0f, -qe);
            c[rt] = ldexpf(a.scale * 1.44269504088896341f, qe);
#pragma unroll
            for (int st = 0; st < KS; st++)
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    float x = q[st][j] * qs;
                    asm("" : "+v"(x));  // one value for both parts
                    qhi[rt][st][j] = (_Float16)x;
                    qlo[rt][st][j] = (_Float16)(x - (float)qhi[rt][st][j]);
                }
        }

        // ---- a step's pages: the entry of position p0 + lane
        const int last = (sq.len - 1) >> psl;
        auto entry = [&](int p0) { return table[min((p0 + lane) >> psl, last)]; };
        auto page_of = [&](int ent, int p) {  // of position p of the step
            const int e = ps >= kStep ? __builtin_amdgcn_readfirstlane(ent) : __shfl(ent, p);
            return (unsigned)e < (unsigned)a.c.n_pages ? e : 0;
        };
        u4 kr[NL], vr[NL];
        float sc = 0.0f;
        auto load = [&](int p0, int ent) {
#pragma unroll
            for (int i = 0; i < NL; i++) {
                constexpr int KW = HD * EB / 16, VW = kStep * EB / 16;  // words of a row
                const int nn = i * kThreads + tid;
                const int row = nn / KW, kw = nn % KW;
                const int kp = page_of(ent, row);
                const uint8_t *k = kc + ((((size_t)kp * a.c.nkv + w.kvh) * ps + ((p0 + row) & (ps - 1))) * HD) * EB + 16 * kw;
                __builtin_memcpy(&kr[i], k, 16);
                const int d = nn / VW, vp0 = nn % VW * (16 / EB);
                const int vp = page_of(ent, vp0);
                const uint8_t *v = vc + ((((size_t)vp * a.c.nkv + w.kvh) * HD + d) * ps + ((p0 + vp0) & (ps - 1))) * EB;
                __builtin_memcpy(&vr[i], v, 16);
            }
            if (KV == kKvInt8 && tid < 2 * kStep) {
                const int e = (unsigned)ent < (unsigned)a.c.n_pages ? ent : 0;
                sc = (tid < kStep ? a.c.ksc : a.c.vsc)[((size_t)e * a.c.nkv + w.kvh) * ps + ((p0 + lane) & (ps - 1))];
            }
        };
        // positions of a step that are there
        auto present = [&](int p0, int ent) {
            return (uint64_t)__ballot((unsigned)ent < (unsigned)a.c.n_pages && p0 + lane < sq.len);
        };

        float m[RT], l[RT];  // reference (log2) of the lane's row, sum over the lane's positions
        f4 o[RT][ND] = {};
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            m[rt] = -INFINITY;
            l[rt] = 0.0f;
        }
        int p0 = w.step * kStep;
        const int p_end = p0 + n * kStep;
        int ent = entry(p0);
        load(p0, ent);
        int ent_next = entry(p0 + kStep);
        for (; p0 < p_end; p0 += kStep) {
            const uint64_t there = present(p0, ent);
            const bool edge = there != ~0ull || p0 + kStep - 1 > pos0;  // some row does not see all of the step
            lds_barrier();
            // ---- K and V into LDS
#pragma unroll
            for (int i = 0; i < NL; i++) {
                constexpr int KW = HD * EB / 16, VW = kStep * EB / 16;
                const int nn = i * kThreads + tid;
                const int row = nn / KW, kw = nn % KW, d = nn / VW, vw = nn % VW;
                if (KV == kKvF16) {
                    kt[k_word<HD>(row, kw)] = kr[i];
                    u4 v = vr[i];
                    if (edge) {
                        // what lies past the end, or ahead of a row, may be no number, which a weight of 0 does not hide
                        const uint32_t in = (uint32_t)(there >> (8 * vw)) & 255u;
                        uint32_t none = 0;
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            if (!(in >> (2 * j) & 1)) v[j] &= 0xffff0000u;
                            if (!(in >> (2 * j + 1) & 1)) v[j] &= 0xffffu;
                            if ((v[j] & 0x7c00u) == 0x7c00u) {
                                none |= 1u << (2 * j);
                                v[j] &= 0xffff0000u;
                            }
                            if ((v[j] & 0x7c000000u) == 0x7c000000u) {
                                none |= 2u << (2 * j);
                                v[j] &= 0xffffu;
                            }
                        }
                        if (none) atomicOr(&odd[parity][vw >> 2], none << (8 * (vw & 3)));
                    }
                    vt[v_word(d, vw)] = v;
                } else {
                    kt[k_word<HD>(row, 2 * kw)] = __builtin_bit_cast(u4, cvt8(kr[i][0], kr[i][1]));
                    kt[k_word<HD>(row, 2 * kw + 1)] = __builtin_bit_cast(u4, cvt8(kr[i][2], kr[i][3]));
                    vt[v_word(d, 2 * vw)] = int8_bf16(vr[i][0], vr[i][1]);
                    vt[v_word(d, 2 * vw + 1)] = int8_bf16(vr[i][2], vr[i][3]);
                }
            }
            if (KV == kKvInt8 && tid < 2 * kStep) (tid < kStep ? ksc : vsc)[lane] = sc;
            lds_barrier();
            const int ent_now = ent;
            if (p0 + kStep < p_end) {
                ent = ent_next;
                load(p0 + kStep, ent);
                ent_next = entry(p0 + 2 * kStep);
            }
            uint64_t none = 0;
            if (KV == kKvF16 && edge) none = (uint64_t)odd[parity][1] << 32 | odd[parity][0];
            parity ^= 1;
            if (tid < 2) odd[parity][tid] = 0;  // (last read before the step's first barrier)
            if (p0 > lim_max) continue;  // no row of the wave sees the step
            // ---- S^T: lane: row r, positions p0 + 16 kg + 4t + i
            f4 s[RT][4] = {};
#pragma unroll
            for (int st = 0; st < KS; st++)
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    const h8 kf = __builtin_bit_cast(h8, kt[k_word<HD>(16 * (r >> 2) + 4 * t + (r & 3), 4 * st + kg)]);
#pragma unroll
                    for (int rt = 0; rt < RT; rt++) {
                        s[rt][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qhi[rt][st], s[rt][t], 0, 0, 0);
                        s[rt][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qlo[rt][st], s[rt][t], 0, 0, 0);
                    }
                }
            // ---- weights
            const bool full = there == ~0ull && p0 + kStep - 1 <= lim_min;  // uniform
            const uint32_t mine = (uint32_t)(there >> (16 * kg)) & 0xffffu;
            h8 phi[RT][2], plo[RT][2];
            b8 pb[RT][2][3];
#pragma unroll
            for (int rt = 0; rt < RT; rt++) {
                float smax = -INFINITY;
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    f4 ks;
                    if (KV == kKvInt8) ks = *(const f4 *)&ksc[16 * kg + 4 * t];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        float x = s[rt][t][i] * c[rt];
                        if (KV == kKvInt8) x *= ks[i];
                        if (!full) x = (mine >> (4 * t + i) & 1) && p0 + 16 * kg + 4 * t + i <= lim[rt] ? x : -INFINITY;
                        s[rt][t][i] = x;
                        smax = fmaxf(smax, x);
                    }
                }
                if (__any(smax > m[rt] + kSlack)) {  // uniform
                    const float mn = fmaxf(m[rt], max_row(smax));
                    const float al = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m[rt] - mn);
                    l[rt] *= al;
                    m[rt] = mn;
#pragma unroll
                    for (int i = 0; i < ND; i++) o[rt][i] *= al;
                }
                const float ref = m[rt] == -INFINITY ? 0.0f : KV == kKvF16 ? m[rt] - kLift : m[rt];
                if (KV == kKvF16) {
#pragma unroll
                    for (int t = 0; t < 4; t++)
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            float p = __builtin_amdgcn_exp2f(s[rt][t][i] - ref);
                            l[rt] += p;
                            asm("" : "+v"(p));
                            const _Float16 hi = (_Float16)p;
                            phi[rt][t / 2][4 * (t & 1) + i] = hi;
                            plo[rt][t / 2][4 * (t & 1) + i] = (_Float16)(p - (float)hi);
                        }
                } else {
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        float p[8];
#pragma unroll
                        for (int j = 0; j < 8; j++) {
                            const int t = 2 * k + j / 4, i = j & 3;
                            const float x = __builtin_amdgcn_exp2f(s[rt][t][i] - ref);
                            l[rt] += x;
                            p[j] = x * vsc[16 * kg + 4 * t + i];
                            // the scale of a masked position may be no number
                            if (!full) p[j] = s[rt][t][i] == -INFINITY ? 0.0f : p[j];
                        }
                        bf16_parts(p, pb[rt][k]);
                    }
                }
            }
            // ---- O^T
#pragma unroll
            for (int i = 0; i < ND; i++)
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    const u4 vw = vt[v_word(16 * i + r, 2 * kg + k)];
#pragma unroll
                    for (int rt = 0; rt < RT; rt++) {
                        if (KV == kKvF16) {
                            o[rt][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, vw), phi[rt][k], o[rt][i], 0, 0, 0);
                            o[rt][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, vw), plo[rt][k], o[rt][i], 0, 0, 0);
                        } else {
#pragma unroll
                            for (int j = 2; j >= 0; j--)
                                o[rt][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, vw), pb[rt][k][j], o[rt][i], 0, 0, 0);
                        }
                    }
                }
            // ---- values that are no numbers, for the rows that see them
            while (KV == kKvF16 && none) {
                const int j = __ffsll((unsigned long long)none) - 1;
                none &= none - 1;
                const int page = __builtin_amdgcn_readlane(ent_now, j);
#pragma unroll
                for (int rt = 0; rt < RT; rt++) {
                    float p = 0.0f;
#pragma unroll
                    for (int x = 0; x < 16; x++)
                        if (x == (j & 15)) p = (float)phi[rt][x >> 3][x & 7] + (float)plo[rt][x >> 3][x & 7];
                    p = __shfl(p, (j & ~15) + r);
#pragma unroll
                    for (int i = 0; i < ND; i++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const int d = 16 * i + 4 * kg + e;
                            const float v = h2f(((const uint16_t *)vc)[(((size_t)page * a.c.nkv + w.kvh) * HD + d) * ps + ((p0 + j) & (ps - 1))]);
                            if (!(fabsf(v) <= 65504.0f) && p0 + j <= lim[rt]) o[rt][i][e] += p * v;
                        }
                }
            }
        }
        const bool begins = w.step == 0, finishes = w.step + n == w.steps;
        const int piece = 2 * g + begins;
        float *part = a.ws + (size_t)piece * part_floats(HD);
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            const float sum = sum_row(l[rt]);
            if (!used[rt]) continue;
            if (begins && finishes) {
                const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
                for (int i = 0; i < ND; i++) {
                    const f4 x = o[rt][i] * inv;
                    __builtin_memcpy(a.out + io[rt] + 16 * i + 4 * kg, &x, 16);
                }
            } else {
                const int row = (wave * RT + rt) * 16 + r;
                if (kg == 0) {
                    part[row] = m[rt];
                    part[S::kRows + row] = sum;
                }
#pragma unroll
                for (int i = 0; i < ND; i++)
                    __builtin_memcpy(part + 2 * S::kRows + (size_t)row * HD + 16 * i + 4 * kg, &o[rt][i], 16);
            }
        }
        if (tid == 0) {
            if (!begins) taken_of(a)[g] = at - w.step;
            else if (!finishes) begun_of(a)[g] = {at, sq.start + tok0, toks * a.gqa, w.kvh};
        }
        at += n;
    }

    if (__any(plan.short_))  // tokens before position 0: zeros
        for (int s = g; s < a.n_seqs; s += kGroups) {
            const Seq q = seq_of(a, s);
            const f4 zero = {};
            float *out = a.out + (size_t)q.start * a.nh * HD;
            for (size_t i = 4 * tid; i < (size_t)max(q.n - q.len, 0) * a.nh * HD; i += 4 * kThreads)
                __builtin_memcpy(out + i, &zero, 16);
        }
}

// Merges the partials of the tile that begins in workgroup blockIdx.x's share and goes on behind it; blockIdx.y: 16 of
// its rows.
template <int HD>
__global__ void __launch_bounds__(256) paged_prompt_merge_kernel(PagedPromptArgs a) {
    const Begun b = begun_of(a)[blockIdx.x];
    if (b.first < 0 || 16 * (int)blockIdx.y >= b.n_rows) return;
    const int *taken = taken_of(a);
    int n = 0;
    for (int g0 = blockIdx.x + 1; g0 < kGroups; g0 += 64) {  // workgroups that go on with it, one after another
        const int g = g0 + lane_id();
        const uint64_t on = __ballot(g < kGroups && taken[min(g, kGroups - 1)] == b.first);
        const int more = on == ~0ull ? 64 : __ffsll((unsigned long long)~on) - 1;
        n += more;
        if (more < 64) break;
    }
    constexpr int R = rows_of(HD);
    const float *first = a.ws + (size_t)(2 * blockIdx.x + 1) * part_floats(HD);
    const float *rest = a.ws + (size_t)(2 * blockIdx.x + 2) * part_floats(HD);  // every second one from here
    for (int e = threadIdx.x; e < 16 * (HD / 4); e += 256) {
        const int row = 16 * blockIdx.y + e / (HD / 4), d = 4 * (e % (HD / 4));
        if (row >= b.n_rows) break;
        float mm = first[row];
#pragma unroll 4
        for (int i = 0; i < n; i++) mm = fmaxf(mm, rest[(size_t)2 * i * part_floats(HD) + row]);
        f4 x = {};
        float sum = 0.0f;
#pragma unroll 4
        for (int i = -1; i < n; i++) {
            const float *p = i < 0 ? first : rest + (size_t)2 * i * part_floats(HD);
            const float f = mm == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(p[row] - mm);
            f4 y;
            __builtin_memcpy(&y, p + 2 * R + (size_t)row * HD + d, 16);
            x += y * f;
            sum = fmaf(p[R + row], f, sum);
        }
        x *= sum == 0.0f ? 0.0f : 1.0f / sum;
        const int tok = row / a.gqa, head = row - tok * a.gqa;
        __builtin_memcpy(a.out + ((size_t)(b.row0 + tok) * a.nh + b.kvh * a.gqa + head) * HD + d, &x, 16);
    }
}

template <int KV, int HD>
int launch_shape(const PagedPromptArgs &a, hipStream_t s) {
    hipLaunchKernelGGL((paged_prompt_kernel<KV, HD>), dim3(kGroups), dim3(kThreads), 0, s, a);
    if (int rc = check_launch("paged_attention_prompt")) return rc;
    hipLaunchKernelGGL(paged_prompt_merge_kernel<HD>, dim3(kGroups, rows_of(HD) / 16), dim3(256), 0, s, a);
    return check_launch("paged_attention_prompt");
}

}  // namespace

size_t paged_prompt_workspace_bytes(int hd) {
    return (size_t)2 * kGroups * part_floats(hd) * sizeof(float) + kGroups * (sizeof(Begun) + sizeof(int));
}

// Tokens of a tile: a power of two, whose rows fill the tile as far as they can.
int paged_prompt_tile_log(int hd, int gqa) {
    int tl = 0;
    while ((2 << tl) * gqa <= rows_of(hd)) tl++;
    return tl;
}

int launch_paged_prompt(PagedPromptArgs a, hipStream_t s) {
    a.tl = paged_prompt_tile_log(a.c.hd, a.gqa);
    if (a.c.kv_type == kKvF16)
        return a.c.hd == 64 ? launch_shape<kKvF16, 64>(a, s) : a.c.hd == 128 ? launch_shape<kKvF16, 128>(a, s)
                                                                              : launch_shape<kKvF16, 256>(a, s);
    return a.c.hd == 64 ? launch_shape<kKvInt8, 64>(a, s) : a.c.hd == 128 ? launch_shape<kKvInt8, 128>(a, s)
                                                                           : launch_shape<kKvInt8, 256>(a, s);
}

}  // namespace mnemo
