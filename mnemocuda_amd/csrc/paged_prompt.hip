// paged_prompt.hip -- attention of several new tokens per sequence over a pool of cache pages: prompts, chunks of
// prompts, drafted tokens, and single ones among them.
//
// Sequence s has n tokens, rows starts[s] .. starts[s+1]-1 of q, the last of them at position L - 1 (L = lens[s]).
// Token i, at p = L - n + i:  out = sum_{j<=p} P_j v_j / sum_{j<=p} P_j,  P_j = exp(scale q.k_j - m).
//
// A tile is the query heads of one KV head for a power of two of tokens, 128 rows, whose waves share the K and V of 64
// positions, a step, in LDS.  The steps of all tiles stand in one row, [sequence][KV head][tile][step], which the
// workgroups divide into equal shares, whatever the lengths are: the sum of a sequence's steps has a closed form, so
// every workgroup finds its share by itself.  A tile that several shares cut leaves partials (max, sum, O) in memory,
// which a second launch merges.  A long prompt alone is dealt out in whole tiles where they balance.
//
// S^T = K Q^T (positions x rows) leaves a lane with positions of one row, which is how O^T = V^T P^T (dims x rows)
// wants P^T, when the K rows of a tile are picked so: lane row m of tile t is position 16 (m/4) + 4t + m%4, so that
// a lane's positions over the tiles are 16 consecutive ones.  Words of 16 bytes in LDS are permuted within their
// row, so that the 16 lanes of an operand's column lie in different banks.
//
// Precision: Q is scaled by a power of two per row and split into two f16 parts, P likewise, relative to a reference
// that moves only when a weight (int8: times its value's scale, by which P is multiplied) exceeds it by 2^kSlack, and
// is 2^kLift at the reference: 22 bits or more of each.  K and V enter as f16, which is exact.  Sums are fp32, the
// weights' with what their additions lose.  So an output is off by 4e-7 of its size (int8 1e-6), fp32 products of
// the same values by 7e-7 to 3e-6.
//
// Long calls are bound by the matrix cores: two products for each.  4096 tokens of 64 heads of 128 on 4 KV heads, 275 GFLOP
// and 550 executed, take 475 us, 1160 TFLOP/s; a large f16 product of the library's runs at 1150 to 1180, what the card's
// power allows with such values (both are a third faster with zeros).  Short calls are bound by the chain of a share: plan,
// table, K and V, two dependent products and a softmax per step, partials, second launch: one token behind 500 positions
// takes 12 us, 21 tokens of 5 sequences behind 13,000 positions 23.
#include <limits.h>
#include <math.h>

#include <float.h>

#include "gemm_ops.hpp"
#include "mfma_types.hpp"
#include "mnemo_common.hpp"
#include "mnemo_internal.hpp"

namespace mnemo {

namespace {

constexpr float kSlack = 5.0f, kLift = 9.0f;  // powers of two
// int8: a reference moves when a weight times its value's scale is more than kMost, which is seen from the products themselves
// (1.87 ms for three long chunks; 1.90 with the products' logarithms looked at first).  Value scales below 2^-98 count as it for the
// reference, and the sum of eight weights is below 2^112 (in its unit: kMost / kMostSum).  The weights' sum is kept in
// units of 2^16: those of 2^30 positions stay in range, and beside scales of 2^90 weights down to 2^-29 of the largest.
constexpr float kLeastScale = -98.0f, kUnit = 0x1p-16f, kMost = 0x1p14f, kMostSum = 0x1p-82f;
constexpr int kStep = 64;                     // positions
// The shares are counted in units: a step is one, and what a tile takes beside its steps (its queries, its output) are
// a few, `cost`.  A share has kLeast or more, as far as there are any: one token behind 500 positions takes 11.3, 12.1 and
// 12.8 us with 1, 2 and 3, five behind 3000 18.0, 16.6 and 17.5.
constexpr int kLeast = 2;
// Where one sequence alone has tokens, of a table of 64 rows at most, and none of the 64 workgroups that are looked at gets more
// than kUneven units, or half, above the average, whole tiles are dealt out instead, in kRounds at most: nothing is cut,
// nothing merged.  1300 tokens of 64 heads of 128 take 81 us and 87 in
// shares, 2000 133 and 155, 4096 473 and 498; where it is less even 600 47 and 45, 1000 67 and 65.
constexpr int kUneven = 8, kRounds = 8;

// 128 rows, by 4 waves of 32 or 8 of 16 (RT tiles of 16 rows each).
constexpr int kRows = 128;
__host__ __device__ constexpr int threads_of(int rt) { return 64 * kRows / (16 * rt); }
__host__ __device__ constexpr int waves_of(int hd, int rt) { return hd == 64 && rt == 1 ? 4 : 2; }  // per SIMD
__host__ __device__ constexpr int groups_of(int hd, int rt) { return 256 * 4 * 64 * waves_of(hd, rt) / threads_of(rt); }  // as many fill the chip

// Workspace: two partials per workgroup (max [rows], sum [rows], O [rows][hd]): of the tile that its share goes on with, and
// of the one that its share begins and does not end; and what these tiles are.
__host__ __device__ constexpr int part_floats(int hd) { return kRows * (hd + 2); }
struct __align__(16) Cut {
    int n;   // workgroups that share the tile, 0 for none
    int g0;  // the first of them
    int row0, n_rows, kvh;  // first token (row of q), rows in use, KV head
    int pad[3];
};
// [workgroup][0: gone on with, 1: begun]
template <int HD, int RT>
__device__ __forceinline__ Cut *cuts_of(const PagedPromptArgs &a) {
    return (Cut *)(a.ws + (size_t)2 * groups_of(HD, RT) * part_floats(HD));
}

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

// The units of the first j tiles of 2^tl tokens, none of them the sequence's last: with b = len - n, the sum over
// i = 1 .. j of ceil(max(b + i 2^tl, 0) / 64) steps, and `cost` for each tile that has one.
__device__ __forceinline__ int units_before(const Seq &s, int tl, int cost, int j) {
    int b = s.len - s.n;
    if (b < 0) {  // tiles of tokens before position 0 have no steps
        const int none = min(-b >> tl, j);
        j -= none;
        b += none << tl;
        if (b <= -(1 << tl)) return 0;
    }
    if (tl > 6) return j * (j + 1) * (1 << (tl - 7)) + j * (((b + 63) >> 6) + cost);
    const int gl = 6 - tl;
    const uint32_t c = (uint32_t)(b + (1 << tl) - 1) >> tl, d = c + (uint32_t)j;  // ceil(u / 2^gl) from u = c + 1 to d
    auto sum = [&](uint32_t x) { return (triangle(x >> gl) << gl) + (x & ((1u << gl) - 1)) * ((x >> gl) + 1); };
    return (int)(sum(d) - sum(c)) + j * cost;
}
__device__ __forceinline__ int tiles_of(const Seq &s, int tl) { return (s.n + (1 << tl) - 1) >> tl; }
// of one KV head
__device__ __forceinline__ int units_of(const Seq &s, int tl, int cost) {
    if (s.n == 0 || s.len == 0) return 0;
    return units_before(s, tl, cost, tiles_of(s, tl) - 1) + (s.len + kStep - 1) / kStep + cost;
}

struct Plan {
    int total;       // units
    int groups;      // workgroups that have some
    int base, more;  // units of a workgroup; the first `more` of them have one more
    bool short_;     // lane: a sequence of its has tokens before position 0
    int per;         // sequences per lane of the sums
    int before;      // lane: units before its sequences
    int alone;       // the sequence whose tiles are taken whole, or -1
};
// of tile j: the positions that its last token sees
__device__ __forceinline__ int tile_steps(const Seq &s, int tl, int j) {
    return (s.len - s.n + min((j + 1) << tl, s.n) + kStep - 1) / kStep;
}
// Round r of workgroup g of as many: the tiles of all KV heads are dealt out from the longest, in turn forwards and backwards.
__device__ __forceinline__ int dealt(int r, int g, int groups) { return r * groups + (r & 1 ? groups - 1 - g : g); }

__device__ __forceinline__ Plan make_plan(const PagedPromptArgs &a, int groups) {
    Plan p;
    p.per = (a.n_seqs + 63) / 64;
    p.short_ = false;
    const int s0 = lane_id() * p.per;
    int sum = 0;
    float size = 0.0f;
    for (int i = 0; i < p.per; i++)
        if (s0 + i < a.n_seqs) {
            const Seq s = seq_of(a, s0 + i);
            p.short_ |= s.n > s.len;
            const int u = units_of(s, a.tl, a.cost);
            sum += u;
            size += (float)u;
        }
    // (starts that do not rise may give the same rows to many sequences, and more units than an int holds: no work at all)
    const bool fits = wave_sum_all(size) * (float)a.c.nkv < 0x1.fp30f;
    sum = fits ? sum : 0;
    sum *= a.c.nkv;
    const int incl = wave_scan(sum);
    p.total = __builtin_amdgcn_readlane(incl, 63);
    p.before = incl - sum;
    p.groups = max(min(groups, p.total / kLeast), 1);
    p.base = p.total / p.groups;
    p.more = p.total - p.base * p.groups;
    p.alone = -1;
    const uint64_t some = __ballot(sum > 0);
    const int mean = p.total / groups;
    if (p.per == 1 && __popcll(some) == 1 && mean >= kUneven) {  // (64 of the workgroups, the first and the last among them)
        const int seq = __ffsll((unsigned long long)some) - 1;
        const Seq s = seq_of(a, seq);
        const int each = tiles_of(s, a.tl), g = lane_id() * (groups - 1) / 63;
        if (s.n <= s.len && each * a.c.nkv <= kRounds * groups) {
            int load = 0;
            for (int r = 0; r < kRounds; r++) {
                const int i = dealt(r, g, groups);
                if (i < each * a.c.nkv) load += tile_steps(s, a.tl, each - 1 - i / a.c.nkv) + a.cost;
            }
            if (!__any(load > mean + min(kUneven, mean / 2))) p.alone = seq;
        }
    }
    return p;
}
__device__ __forceinline__ int first_of(const Plan &p, int g) {
    return g >= p.groups ? p.total : g * p.base + min(g, p.more);
}
// The workgroup that has unit u.
__device__ __forceinline__ int group_of(const Plan &p, int u) {
    const int longer = p.more * (p.base + 1);
    return u < longer ? u / (p.base + 1) : p.more + (u - longer) / p.base;
}

struct Where {
    Seq s;
    int seq, kvh, tile, unit, steps;
};
// The tile of unit u, and the unit within it.
__device__ __forceinline__ Where find(const PagedPromptArgs &a, const Plan &p, int u) {
    // the last lane that begins at or before u holds it (lanes without steps share their successor's beginning)
    const int lane = lane_id(), L = __popcll(__ballot(p.before <= u)) - 1;
    int at = u - __builtin_amdgcn_readlane(p.before, L);
    Where w;
    w.seq = L;
    if (p.per > 1) {
        const int s = L * p.per + lane;
        const bool in = lane < p.per && s < a.n_seqs;
        const int n = in ? units_of(seq_of(a, s), a.tl, a.cost) * a.c.nkv : 0;
        const int before = wave_scan(n) - n;
        const int j = __popcll(__ballot(lane < p.per && before <= at)) - 1;
        w.seq = L * p.per + j;
        at -= __builtin_amdgcn_readlane(before, j);
    }
    w.seq = __builtin_amdgcn_readfirstlane(w.seq);
    w.s = seq_of(a, w.seq);
    const int each = units_of(w.s, a.tl, a.cost);
    w.kvh = at / each;
    at -= w.kvh * each;
    int lo = 0, hi = tiles_of(w.s, a.tl) - 1;  // the last tile that begins at or before the unit
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (units_before(w.s, a.tl, a.cost, mid) <= at) lo = mid;
        else hi = mid - 1;
    }
    w.tile = lo;
    w.unit = at - units_before(w.s, a.tl, a.cost, lo);
    w.steps = tile_steps(w.s, a.tl, lo);
    return w;
}
// The tile of round r, where whole tiles are dealt out.
__device__ __forceinline__ bool deal(const PagedPromptArgs &a, Where &w, int r, int g, int groups) {
    const int each = tiles_of(w.s, a.tl), i = dealt(r, g, groups), j = i / a.c.nkv;
    if (j >= each) return false;
    w.tile = each - 1 - j;
    w.kvh = i - j * a.c.nkv;
    w.unit = 0;
    w.steps = tile_steps(w.s, a.tl, w.tile);
    return true;
}
// The tile after w, from its first unit on (there is one).
__device__ __forceinline__ void advance(const PagedPromptArgs &a, Where &w) {
    if (++w.tile == tiles_of(w.s, a.tl)) {
        if (++w.kvh == a.c.nkv) {
            w.kvh = 0;
            do w.s = seq_of(a, ++w.seq);
            while (w.s.n == 0 || w.s.len == 0);
        }
        w.tile = max(w.s.n - w.s.len, 0) >> a.tl;  // the first one with a position
    }
    w.unit = 0;
    w.steps = tile_steps(w.s, a.tl, w.tile);
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

// Steps that some row of a tile does not see all of hold its tokens' positions, 128 at most, and the rest of the
// words that the first and the last of them lie in.
constexpr int kOddWords = (kRows + 2 * kStep) / 32;

// Two f16 parts of each of two values, the first cut off, the second rounded: together 22 bits or more.
struct h2x2 {
    h2 hi, lo;
};
__device__ __forceinline__ h2x2 two_parts(float a, float b) {
    h2x2 x;
    x.hi = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_pkrtz(a, b));
    x.lo = h2{(_Float16)fmaf((float)x.hi[0], -1.0f, a), (_Float16)fmaf((float)x.hi[1], -1.0f, b)};
    return x;
}

template <int KV, int HD, int RT>
__global__ void __launch_bounds__(threads_of(RT), waves_of(HD, RT)) paged_prompt_kernel(PagedPromptArgs a) {
    constexpr int KS = HD / 32, ND = HD / 16, kThreads = threads_of(RT), kGroups = groups_of(HD, RT);  // dim steps of S, dim tiles of O
    constexpr int EB = KV == kKvF16 ? 2 : 1;
    constexpr int kWords = kStep * HD / 8;  // 16-byte words of K, and of V, of a step in LDS
    // f16: a step's words are copied straight into one buffer while the other is worked on.  int8: they are copied as
    // they are, and converted by the waves that copied them.
    constexpr int kBufs = KV == kKvF16 ? 2 : 1, kRaw = KV == kKvInt8 ? kStep * HD / 16 : 1;
    __shared__ __align__(1024) u4 kt[kBufs][kWords], vt[kBufs][kWords];  // (words are picked by bits of their addresses)
    __shared__ u4 k_raw[kRaw], v_raw[kRaw];
    // int8: scales of K and V, and log2 of the latter's size
    constexpr int kScales = KV == kKvInt8 ? kStep : 4;
    __shared__ __align__(16) float ksc[kScales], vsc[kScales], vlg[kScales], sc_raw[2][kScales];
    // f16: positions of the tile, from its first token's last step on, whose values are no numbers
    __shared__ uint32_t odd[kOddWords];
    const int lane = lane_id(), r = lane & 15, kg = lane >> 4, tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int ps = a.c.ps, psl = 31 - __builtin_clz(ps);
    // of the lane's words of K (row 16 (r/4) + r%4, word kg) and V (dim r, word 2 kg)
    const uint32_t ka0 = lds_addr(&kt[0][0]) + 16 * k_word<HD>(16 * (r >> 2) + (r & 3), kg);
    const uint32_t va0 = lds_addr(&vt[0][0]) + 16 * v_word(r, 2 * kg);
    // ---- a wave's loads: K rows i * kKRows + wave * kKWave + k_l, V dims i * kVRows + wave * kVWave + v_l, 16 bytes a lane,
    // from uniform addresses and these offsets of the lane
    constexpr int KW = HD * EB / 16, VW = kStep * EB / 16, kKWave = 64 / KW, kVWave = 64 / VW;
    constexpr int kKRows = kThreads / KW, kVRows = kThreads / VW, NL = kStep / kKRows;
    static_assert(NL * kVRows == HD && kKWave <= 16, "whole rows, of one page");
    const int k_l = lane / KW, v_l = lane / VW;
    uint32_t k_off = k_l * (HD * EB), v_off = v_l * ps * EB;
    int v_pos;  // first position of the lane's word of V
    if (KV == kKvF16) {  // the words lie in LDS in the order that k_word and v_word give them
        k_off += 16 * (lane % KW ^ (HD == 64 ? (k_l & 3) >> 1 : k_l & 3));
        v_pos = 8 * (lane % VW ^ ((wave * kVWave + v_l) >> 1 & 7));
    } else {
        k_off += 16 * (lane % KW);
        v_pos = 16 * (lane % VW);
    }
    v_off += (v_pos & (ps - 1)) * EB;

    const Plan plan = make_plan(a, kGroups);
    // neighbouring shares, which read the same pages, on one XCD; workgroups that go without one behind them
    const int per_xcd = (plan.groups + 7) / 8;
    const int g = (int)(blockIdx.x >> 3) < per_xcd ? (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3) : blockIdx.x;
    int at = first_of(plan, g);
    int end = first_of(plan, g + 1);
    if (tid < 2) cuts_of<HD, RT>(a)[2 * g + tid].n = 0;
    // of the lane's rows: the token within a tile and its head
    int tok_of[RT], head_of[RT];
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        const int row = (wave * RT + rt) * 16 + r;
        tok_of[rt] = row / a.gqa;
        head_of[rt] = row - tok_of[rt] * a.gqa;
    }
    // the wave's first and last token
    const int tok_first = __builtin_amdgcn_readfirstlane(tok_of[0]), tok_last = __builtin_amdgcn_readlane(tok_of[RT - 1], 15);

    Where w;
    int round = 0;
    if (plan.alone >= 0) {
        w.seq = plan.alone;
        w.s = seq_of(a, w.seq);
        at = 0;
        end = deal(a, w, 0, g, kGroups) ? INT_MAX : 0;
    } else if (at < end) w = find(a, plan, at);
    while (at < end) {
        const int units = min(end - at, w.steps + a.cost - w.unit);
        const int step = max(w.unit - a.cost, 0), n = max(w.unit + units - a.cost, 0) - step;
        if (n == 0) {  // none of its steps: the next workgroup begins it
            at += units;
            if (at < end) advance(a, w);
            continue;
        }
        const int tok0 = w.tile << a.tl, toks = min(1 << a.tl, w.s.n - tok0);
        const int *table = a.table + (size_t)w.seq * a.max_pages;
        const int pos0 = w.s.len - w.s.n + tok0;  // of the tile's first token
        const int last = (w.s.len - 1) >> psl;
        const int odd0 = max(pos0, 0) & ~(kStep - 1);  // what odd begins with

        // ---- a step's pages: the entry of position p0 + lane
        auto entry = [&](int p0) { return table[min((p0 + lane) >> psl, last)]; };
        auto valid = [&](int e) { return (unsigned)e < (unsigned)a.c.n_pages ? e : 0; };
        // copies K and V of the step at p0, into buffer b
        auto load = [&](int p0, int ent, int b) {
            const size_t page_bytes = (size_t)ps * HD * EB;  // of a KV head
#pragma unroll
            for (int i = 0; i < NL; i++) {
                const int row0 = i * kKRows + wave * kKWave;  // (a wave's rows lie in one page)
                const uint8_t *k = (const uint8_t *)a.c.k + ((size_t)valid(__builtin_amdgcn_readlane(ent, row0)) * a.c.nkv + w.kvh) * page_bytes +
                                   ((p0 + row0) & (ps - 1)) * (HD * EB);
                if (KV == kKvF16) {
                    const int m = ((row0 >> 4) & 3) * 4 + (row0 & 3);
                    lds_copy16(k, k_off ^ (16 * (HD == 64 ? m >> 1 : m)), lds_addr(&kt[0][0]) + 16 * (b * kWords + i * kThreads + 64 * wave));
                } else lds_copy16(k, k_off, lds_addr(k_raw) + 16 * (i * kThreads + 64 * wave));
            }
            if (ps >= kStep) {
                const uint8_t *v = (const uint8_t *)a.c.v + ((size_t)valid(__builtin_amdgcn_readfirstlane(ent)) * a.c.nkv + w.kvh) * page_bytes +
                                   (wave * kVWave * ps + (p0 & (ps - 1))) * EB;
#pragma unroll
                for (int i = 0; i < NL; i++, v += kVRows * ps * EB)
                    if (KV == kKvF16) lds_copy16(v, v_off, lds_addr(&vt[0][0]) + 16 * (b * kWords + i * kThreads + 64 * wave));
                    else lds_copy16(v, v_off, lds_addr(v_raw) + 16 * (i * kThreads + 64 * wave));
            } else {
                const uint8_t *v = (const uint8_t *)a.c.v + ((size_t)valid(__shfl(ent, v_pos)) * a.c.nkv + w.kvh) * page_bytes + v_off +
                                   wave * kVWave * ps * EB;
#pragma unroll
                for (int i = 0; i < NL; i++, v += kVRows * ps * EB)
                    if (KV == kKvF16) lds_copy16(v, lds_addr(&vt[0][0]) + 16 * (b * kWords + i * kThreads + 64 * wave));
                    else lds_copy16(v, lds_addr(v_raw) + 16 * (i * kThreads + 64 * wave));
            }
            if (KV == kKvInt8 && wave < 2)  // the first waves' copies of the scales
                lds_copy4((wave ? a.c.vsc : a.c.ksc) + ((size_t)valid(ent) * a.c.nkv + w.kvh) * ps + ((p0 + lane) & (ps - 1)),
                          lds_addr(&sc_raw[0][0]) + 4 * kStep * wave);
        };
        // int8: what the wave has copied, as f16
        auto convert = [&] {
#pragma unroll
            for (int i = 0; i < NL; i++) {
                const int row = i * kKRows + wave * kKWave + k_l, d = i * kVRows + wave * kVWave + v_l, kw = lane % KW, vw = lane % VW;
                const u4 x = k_raw[i * kThreads + tid], y = v_raw[i * kThreads + tid];
                kt[0][k_word<HD>(row, 2 * kw)] = __builtin_bit_cast(u4, cvt8(x[0], x[1]));
                kt[0][k_word<HD>(row, 2 * kw + 1)] = __builtin_bit_cast(u4, cvt8(x[2], x[3]));
                vt[0][v_word(d, 2 * vw)] = __builtin_bit_cast(u4, cvt8(y[0], y[1]));
                vt[0][v_word(d, 2 * vw + 1)] = __builtin_bit_cast(u4, cvt8(y[2], y[3]));
            }
            if (wave < 2) {
                const float x = sc_raw[wave][lane];
                (wave ? vsc : ksc)[lane] = x;
                // (a scale of 0 or next to it: its weight still counts in the sum, whose range this bounds)
                if (wave) vlg[lane] = fmaxf(__builtin_amdgcn_logf(fabsf(x)), kLeastScale);
            }
        };

        int p0 = step * kStep, b = 0;
        const int p_end = p0 + n * kStep;
        int ent = entry(p0), ent_next = entry(p0 + kStep);
        lds_barrier();  // the buffers are free
        if (KV == kKvF16 && tid < kOddWords) odd[tid] = 0;
        load(p0, ent, 0);

        // ---- the lane's rows
        int lim[RT];  // last position that the row sees; what the rows of no token (INT_MAX) give is dropped
#pragma unroll
        for (int rt = 0; rt < RT; rt++) lim[rt] = tok_of[rt] < toks ? pos0 + tok_of[rt] : INT_MAX;
        auto io = [&](int rt) {  // of the row's query and output, the tile's first for the rows of no token
            const bool used = tok_of[rt] < toks;
            return ((size_t)(w.s.start + tok0 + (used ? tok_of[rt] : 0)) * a.nh + w.kvh * a.gqa + (used ? head_of[rt] : 0)) * HD;
        };
        const int lim_min = pos0 + tok_first, lim_max = tok_first < toks ? pos0 + min(tok_last, toks - 1) : -1;

        // ---- Q
        h8 qhi[RT][KS], qlo[RT][KS];
        float c[RT];
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            const float *qp = a.q + io(rt) + 8 * kg;
            float q[KS][8], qm = 0.0f;
#pragma unroll
            for (int st = 0; st < KS; st++) {
                __builtin_memcpy(&q[st][0], qp + 32 * st, 16);
                __builtin_memcpy(&q[st][4], qp + 32 * st + 4, 16);
            }
#pragma unroll
            for (int st = 0; st < KS; st++)
#pragma unroll
                for (int j = 0; j < 8; j++) qm = fmaxf(qm, fabsf(q[st][j]));
            qm = max_row(qm);
            const int qe = (int)((__builtin_bit_cast(uint32_t, qm) >> 23) & 255) - 127;  // exponent of the largest
            const float qs = copysignf(ldexpf(1.0f, -qe), a.scale);
            // more than 0, so that the largest product has the largest score and what is masked stays below
            c[rt] = ldexpf(fabsf(a.scale) * 1.44269504088896341f, qe);
            c[rt] = c[rt] < FLT_MIN ? FLT_MIN : c[rt];
#pragma unroll
            for (int st = 0; st < KS; st++)
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                    const h2x2 x = two_parts(q[st][j] * qs, q[st][j + 1] * qs);
                    qhi[rt][st][j] = x.hi[0];
                    qhi[rt][st][j + 1] = x.hi[1];
                    qlo[rt][st][j] = x.lo[0];
                    qlo[rt][st][j + 1] = x.lo[1];
                }
        }

        // reference (log2) of the lane's row, sum over the lane's positions and what its additions have lost: of a long row
        // they are thousands
        float m[RT], l[RT], lost[RT];
        f4 o[RT][ND] = {};
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            m[rt] = -INFINITY;
            l[rt] = lost[rt] = 0.0f;
        }
        for (; p0 < p_end; p0 += kStep, b ^= KV == kKvF16) {
            // positions that are there; whether there is something that some row does not see
            const uint64_t there = __ballot((unsigned)ent < (unsigned)a.c.n_pages && p0 + lane < w.s.len);
            wait_vm<0>();  // the wave's own copies
            lds_barrier();
            if (KV == kKvInt8) {
                convert();
                lds_barrier();
            }
            if (KV == kKvF16 && (there != ~0ull || p0 + kStep - 1 > pos0)) {
                // V past the end, or ahead of a row, may be no number, which a weight of 0 does not hide: it becomes 0.
                // What is there and no number is noted, for the rows that do see it.
                const int p = v_pos, in = (int)((there >> p) & 255);
                u4 keep;
#pragma unroll
                for (int j = 0; j < 4; j++) keep[j] = (in >> (2 * j) & 1 ? 0xffffu : 0u) | (in >> (2 * j + 1) & 1 ? 0xffff0000u : 0u);
                uint32_t sum = 0;  // bit 15 of a half: an exponent of all ones is among them
#pragma unroll
                for (int i = 0; i < NL; i++) {
                    const u4 v = vt[b][i * kThreads + tid] & keep;
                    if (in != 255) vt[b][i * kThreads + tid] = v;
#pragma unroll
                    for (int j = 0; j < 4; j++) sum |= (v[j] & 0x7fff7fffu) + 0x04000400u;
                }
                if (p0 >= odd0 && (sum & 0x80008000u)) {  // (before odd0 all rows see what is there)
                    uint32_t bad = 0;
                    for (int i = 0; i < NL; i++) {
                        u4 v = vt[b][i * kThreads + tid];
#pragma unroll
                        for (int j = 0; j < 8; j++) {
                            const uint32_t inf = 0x7c00u << (16 * (j & 1));
                            if ((v[j / 2] & inf) == inf) {
                                v[j / 2] &= ~(0xffffu << (16 * (j & 1)));
                                bad |= 1u << j;
                            }
                        }
                        vt[b][i * kThreads + tid] = v;
                    }
                    atomicOr(&odd[(p0 - odd0 + p) >> 5], bad << (p & 31));
                }
                lds_barrier();
            }
            if (p0 + kStep < p_end) {
                ent = ent_next;
                ent_next = entry(p0 + 2 * kStep);
                load(p0 + kStep, ent, b ^ 1);
            }
            if (p0 > lim_max) continue;  // no row of the wave sees the step
            const bool full = there == ~0ull && p0 + kStep - 1 <= lim_min;  // uniform
            // ---- in halves: of a lane's 16 positions the first 8, then the others.  Operands are read from LDS four at a
            // time, four ahead of the products: K for the products before, V for the weights before.
            const uint32_t kb = ka0 + b * (16 * kWords), vb = va0 + b * (16 * kWords);
            constexpr int CK = KS / 2, CV = ND / 4;  // fours of K and of V
            u4 w4[2][4];
            auto read_k = [&](int k, int n, int to) {
#pragma unroll
                for (int i = 0; i < 4; i++) w4[to][i] = lds_get<u4>(kb ^ (64 * (2 * n + i / 2)), (8 * k + 4 * (i & 1)) * (HD * 2));
                __builtin_amdgcn_sched_barrier(0x7f);  // (LDS reads stay where they are)
            };
            auto read_v = [&](int k, int n, int to) {
#pragma unroll
                for (int i = 0; i < 4; i++) w4[to][i] = lds_get<u4>(vb ^ (16 * k), (4 * n + i) * (16 * kStep * 2));
                __builtin_amdgcn_sched_barrier(0x7f);
            };
            read_k(0, 0, 0);
#pragma unroll
            for (int k = 0; k < 2; k++) {
                constexpr int per_half = CK + CV;
                // S^T: lane: row r, positions p0 + first + 4t + i
                __builtin_amdgcn_s_setprio(1);  // the SIMD's other wave forms its weights meanwhile
                const int first = 16 * kg + 8 * k;
                f4 s[RT][2] = {};
#pragma unroll
                for (int n = 0; n < CK; n++) {
                    const int at = (k * per_half + n) & 1;
                    if (n + 1 < CK) read_k(k, n + 1, at ^ 1);
#pragma unroll
                    for (int st = 0; st < 2; st++) {
#pragma unroll
                        for (int t = 0; t < 2; t++)
#pragma unroll
                            for (int rt = 0; rt < RT; rt++) s[rt][t] = mfma(__builtin_bit_cast(h8, w4[at][2 * st + t]), qhi[rt][2 * n + st], s[rt][t]);
#pragma unroll
                        for (int t = 0; t < 2; t++)
#pragma unroll
                            for (int rt = 0; rt < RT; rt++) s[rt][t] = mfma(__builtin_bit_cast(h8, w4[at][2 * st + t]), qlo[rt][2 * n + st], s[rt][t]);
                    }
                }
                read_v(k, 0, (k * per_half + CK) & 1);
                __builtin_amdgcn_s_setprio(0);
                // weights
                h8 phi[RT], plo[RT];
#pragma unroll
                for (int rt = 0; rt < RT; rt++) {
                    uint32_t seen = 255;
                    if (!full) {
                        const int live = min(max(lim[rt] - (p0 + first), -1), 7) + 1;
                        seen = (uint32_t)(there >> first) & ((1u << live) - 1);
                    }
                    f4 f[2], vs[2];
                    if (KV == kKvInt8) {
#pragma unroll
                        for (int t = 0; t < 2; t++) {
                            f[t] = *(const f4 *)&ksc[first + 4 * t] * c[rt];
                            vs[t] = *(const f4 *)&vsc[first + 4 * t];
                        }
                    }
                    if (!full) {
#pragma unroll
                        for (int j = 0; j < 8; j++) {
                            const bool in = seen >> j & 1;
                            s[rt][j / 4][j & 3] = in ? s[rt][j / 4][j & 3] : -INFINITY;
                            if (KV == kKvInt8) {  // (the scales of a position that is not seen may be no numbers)
                                f[j / 4][j & 3] = in ? f[j / 4][j & 3] : 1.0f;
                                vs[j / 4][j & 3] = in ? vs[j / 4][j & 3] : 0.0f;
                            }
                        }
                    }
                    // moves the reference of rows that have need of it, which is a row's own doing, to their largest score
                    auto move = [&](float top, bool need) {
                        top = max_row(top);
                        const float mn = need ? top : m[rt];
                        const float al = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m[rt] - mn);
                        l[rt] *= al;
                        lost[rt] *= al;
                        m[rt] = mn;
#pragma unroll
                        for (int i = 0; i < ND; i++) o[rt][i] *= al;
                    };
                    float p[8], more;
                    auto weigh = [&] {
                        const float ref = m[rt] == -INFINITY ? 0.0f : m[rt] - kLift;
                        float sum[4];
#pragma unroll
                        for (int j = 0; j < 8; j++) {
                            const float x = __builtin_amdgcn_exp2f(fmaf(s[rt][j / 4][j & 3], KV == kKvF16 ? c[rt] : f[j / 4][j & 3], -ref));
                            sum[j & 3] = j < 4 ? x : sum[j & 3] + x;
                            p[j] = KV == kKvInt8 ? x * vs[j / 4][j & 3] : x;
                        }
                        more = (sum[0] + sum[1]) + (sum[2] + sum[3]);
                        if (KV == kKvInt8) more *= kUnit;
                    };
                    if (KV == kKvF16) {
                        float top = -INFINITY;  // of the lane's scores
#pragma unroll
                        for (int j = 0; j < 8; j++) top = fmaxf(top, s[rt][j / 4][j & 3]);
                        top *= c[rt];
                        if (__any(top > m[rt] + kSlack)) {  // uniform
                            top = max_row(top);
                            move(top, top > m[rt] + kSlack);
                        }
                        weigh();
                    } else {
                        weigh();
                        float most = more * kMostSum;
#pragma unroll
                        for (int j = 0; j < 8; j++) most = fmaxf(most, fabsf(p[j]));
                        const bool need = most > kMost || m[rt] == -INFINITY;
                        if (__any(need)) {  // uniform
                            float top = -INFINITY;
#pragma unroll
                            for (int t = 0; t < 2; t++) {
                                const f4 lg = *(const f4 *)&vlg[first + 4 * t];
#pragma unroll
                                for (int i = 0; i < 4; i++) top = fmaxf(top, fmaf(s[rt][t][i], f[t][i], lg[i]));
                            }
                            move(top, max_row(need ? 1.0f : 0.0f) != 0.0f);
                            weigh();
                        }
                    }
                    const float to = l[rt] + more;
                    lost[rt] += more - (to - l[rt]);  // (exact while l is the larger)
                    l[rt] = to;
#pragma unroll
                    for (int j = 0; j < 8; j += 2) {
                        const h2x2 x = two_parts(p[j], p[j + 1]);
                        phi[rt][j] = x.hi[0];
                        phi[rt][j + 1] = x.hi[1];
                        plo[rt][j] = x.lo[0];
                        plo[rt][j + 1] = x.lo[1];
                    }
                }
                __builtin_amdgcn_s_setprio(1);
                // O^T
#pragma unroll
                for (int n = 0; n < CV; n++) {
                    const int at = (k * per_half + CK + n) & 1;
                    if (n + 1 < CV) read_v(k, n + 1, at ^ 1);
                    else if (k == 0) read_k(1, 0, at ^ 1);
#pragma unroll
                    for (int i = 0; i < 4; i++)
#pragma unroll
                        for (int rt = 0; rt < RT; rt++) o[rt][4 * n + i] = mfma(__builtin_bit_cast(h8, w4[at][i]), phi[rt], o[rt][4 * n + i]);
#pragma unroll
                    for (int i = 0; i < 4; i++)
#pragma unroll
                        for (int rt = 0; rt < RT; rt++) o[rt][4 * n + i] = mfma(__builtin_bit_cast(h8, w4[at][i]), plo[rt], o[rt][4 * n + i]);
                }
            }
        }
        if (KV == kKvF16) {
            // values that are no numbers: nor is, then, their dim of the rows that see them.  (The last barrier has passed
            // since they were noted.)
            for (int i = 0; i < kOddWords; i++)
                for (uint32_t left = odd[i]; left; left &= left - 1) {
                    const int p = odd0 + 32 * i + __ffs((int)left) - 1;
                    const int page = valid(table[min(p >> psl, last)]);
                    const uint16_t *v = (const uint16_t *)a.c.v + (((size_t)page * a.c.nkv + w.kvh) * HD + 4 * kg) * ps + (p & (ps - 1));
#pragma unroll
                    for (int i = 0; i < ND; i++)
#pragma unroll
                        for (int e = 0; e < 4; e++, v += e < 4 ? ps : 13 * ps) {
                            const bool none = (*v & 0x7c00) == 0x7c00;
#pragma unroll
                            for (int rt = 0; rt < RT; rt++)
                                if (none && p <= lim[rt]) o[rt][i][e] = NAN;
                        }
                }
        }
        const bool begins = step == 0, finishes = step + n == w.steps;
        float *part = a.ws + (size_t)(2 * g + begins) * part_floats(HD);
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            const float sum = sum_row(l[rt] + (l[rt] <= FLT_MAX ? lost[rt] : 0.0f));
            if (lim[rt] == INT_MAX) continue;
            if (KV == kKvInt8)
#pragma unroll
                for (int i = 0; i < ND; i++) o[rt][i] *= kUnit;
            if (begins && finishes) {
                const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                float *out = a.out + io(rt) + 4 * kg;
#pragma unroll
                for (int i = 0; i < ND; i++) {
                    const f4 x = o[rt][i] * inv;
                    __builtin_memcpy(out + 16 * i, &x, 16);
                }
            } else {
                const int row = (wave * RT + rt) * 16 + r;
                if (kg == 0) {
                    part[row] = m[rt];
                    part[kRows + row] = sum;
                }
#pragma unroll
                for (int i = 0; i < ND; i++)
                    __builtin_memcpy(part + 2 * kRows + (size_t)row * HD + 16 * i + 4 * kg, &o[rt][i], 16);
            }
        }
        if (tid == begins && !(begins && finishes)) {  // (by the thread that cleared it)
            const int u = at - w.unit + a.cost, g0 = group_of(plan, u);  // of the tile's first step
            cuts_of<HD, RT>(a)[2 * g + begins] = {group_of(plan, u + w.steps - 1) - g0 + 1, g0, w.s.start + tok0, toks * a.gqa, w.kvh, {}};
        }
        at += units;
        if (plan.alone >= 0) {
            if (!deal(a, w, ++round, g, kGroups)) break;
        } else if (at < end) advance(a, w);
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

// Merges the partials of a tile that workgroups g0 to g0 + n - 1 had shares of: all but the last of them, here workgroups of
// the same number, divide its rows (blockIdx.y: of which 16).  256 threads are HD / 4 lanes of four dims, times threads that
// divide a row's partials among them where there are many, or rows.
template <int HD, int RT>
__global__ void __launch_bounds__(256) paged_prompt_merge_kernel(PagedPromptArgs a) {
    constexpr int D4 = HD / 4, PARTS = 256 / D4;
    __shared__ __align__(16) float so[PARTS][HD];
    __shared__ float sm[PARTS], sl[PARTS];
    const Cut *cut = cuts_of<HD, RT>(a) + 2 * blockIdx.x;
    const Cut t = cut[1].n ? cut[1] : cut[0];
    const int n = t.n, g0 = t.g0, rows16 = min(16, t.n_rows - 16 * (int)blockIdx.y);
    if (n == 0 || rows16 <= 0) return;
    const int me = (int)blockIdx.x - g0, per = (rows16 + n - 2) / (n - 1), from = me * per, rows = min(per, rows16 - from);
    if (me >= n - 1 || rows <= 0) return;
    // partial i: the second of workgroup g0, then the first of each that follows
    auto part = [&](int i) { return a.ws + (size_t)(2 * (g0 + i) + (i == 0)) * part_floats(HD); };
    int per_pass = 1;  // rows at once: a power of two, in one pass where there are so many threads
    while (per_pass < rows && per_pass < PARTS) per_pass *= 2;
    const int chain = PARTS / per_pass;  // threads per word of a row
    const int d = 4 * (threadIdx.x % D4), slot = threadIdx.x / D4, c = slot % chain, rr = slot / chain;
    for (int r0 = 0; r0 < rows; r0 += per_pass) {
        const int row = 16 * blockIdx.y + from + min(r0 + rr, rows - 1);
        float m = -INFINITY, l = 0.0f;
        f4 x = {};
        for (int i0 = c; i0 < n; i0 += 4 * chain) {  // four loads in flight
            float pm[4], pl[4];
            f4 y[4];
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const float *p = part(min(i0 + u * chain, n - 1));
                pm[u] = p[row];
                pl[u] = p[kRows + row];
                __builtin_memcpy(&y[u], p + 2 * kRows + (size_t)row * HD + d, 16);
                if (i0 + u * chain >= n) {
                    pm[u] = -INFINITY;
                    pl[u] = 0.0f;
                    y[u] = f4{0.f, 0.f, 0.f, 0.f};
                }
            }
            float mn = m;
#pragma unroll
            for (int u = 0; u < 4; u++) mn = fmaxf(mn, pm[u]);
            const float f0 = mn == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
            x *= f0;
            l *= f0;
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const float f = mn == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(pm[u] - mn);
                x += y[u] * f;  // (partials of a query that is no number are none, and stay it)
                l = fmaf(pl[u], f, l);
            }
            m = mn;
        }
        if (chain > 1) {  // (one pass)
            __builtin_memcpy(&so[slot][d], &x, 16);
            if (d == 0) {
                sm[slot] = m;
                sl[slot] = l;
            }
            __syncthreads();
            if (c > 0) continue;
            float mn = m;
            for (int i = 1; i < chain; i++) mn = fmaxf(mn, sm[slot + i]);
            x = f4{0.f, 0.f, 0.f, 0.f};
            l = 0.0f;
            for (int i = 0; i < chain; i++) {
                const float f = mn == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(sm[slot + i] - mn);
                f4 y;
                __builtin_memcpy(&y, &so[slot + i][d], 16);
                x += y * f;
                l = fmaf(sl[slot + i], f, l);
            }
        }
        if (r0 + rr < rows) {
            x *= l == 0.0f ? 0.0f : 1.0f / l;
            const int tok = row / a.gqa, head = row - tok * a.gqa;
            __builtin_memcpy(a.out + ((size_t)(t.row0 + tok) * a.nh + t.kvh * a.gqa + head) * HD + d, &x, 16);
        }
    }
}

template <int KV, int HD, int RT>
int launch_rows(const PagedPromptArgs &a, hipStream_t s) {
    hipLaunchKernelGGL((paged_prompt_kernel<KV, HD, RT>), dim3(groups_of(HD, RT)), dim3(threads_of(RT)), 0, s, a);
    if (int rc = check_launch("paged_attention_prompt")) return rc;
    hipLaunchKernelGGL((paged_prompt_merge_kernel<HD, RT>), dim3(groups_of(HD, RT), kRows / 16), dim3(256), 0, s, a);
    return check_launch("paged_attention_prompt");
}
// Waves of 16 rows are done with a step sooner, of 32 read each operand from LDS half as often: 3 to 6 tokens of 5 sequences
// take 23 us by 16 and 30 by 32, 8 behind 100,000 positions 67 and 72, 300 to 512 behind 6000 to 30,000 1.93 and 1.72 ms (int8 1.99
// and 1.88), and of prompts alone, in whole tiles, 300 tokens 26 and 31 us, 1000 51 and 67, 2000 146 and 132, 4096 531 and 465.  So
// rows of one tile a sequence, as the average is, are taken by 16; the host knows the table's rows, not how many of them have
// tokens, and many idle ones lead to 16 as well (512 tokens behind 30,000: 830 us, in a table of 64 rows 913; int8 994 and
// 1033).  At head_dim 256 the registers hold no more than 16; at 64 they hold four waves a SIMD of them, which is best for all (60
// times 3 tokens behind 2000 34 us and 43 by 32, a prompt of 4096 291 and 286), but int8 rows of 64 are too few words for 8 waves
// to copy.
template <int KV, int HD>
int launch_shape(const PagedPromptArgs &a, hipStream_t s) {
    if constexpr (HD == 256 || (HD == 64 && KV == kKvF16)) return launch_rows<KV, HD, 1>(a, s);
    else if constexpr (HD == 64) return launch_rows<KV, HD, 2>(a, s);
    else return (long long)a.n_tokens * a.gqa <= (long long)kRows * a.n_seqs ? launch_rows<KV, HD, 1>(a, s) : launch_rows<KV, HD, 2>(a, s);
}

}  // namespace

size_t paged_prompt_workspace_bytes(int hd) {
    return (size_t)groups_of(hd, hd == 256 ? 1 : 2) * 2 * (part_floats(hd) * sizeof(float) + sizeof(Cut));
}

int launch_paged_prompt(PagedPromptArgs a, hipStream_t s) {
    // Tokens of a tile: a power of two, whose rows fill the tile as far as they can.  Where gqa is no power of two rows stay
    // idle, and are multiplied all the same: 4096 tokens of 8 KV heads reach 1136 TFLOP/s (two products for each) with 8 query
    // heads for each, 993 with 6 (96 rows of 128), 834 with 5 (80), 749 with 9 (72).
    a.tl = 0;
    while ((2 << a.tl) * a.gqa <= kRows) a.tl++;
    // three prompts of 700 tokens of 32 heads of 256 take 106, 90 and 84 us with 1, 2 and 3, of 64 heads of 128 97, 87 and 85, a mixed
    // step of 12 heads of 64 29.8, 29.4 and 30.8 (one prompt in whole tiles is the same with all)
    a.cost = a.c.hd == 256 ? 3 : 2;
    if (a.c.kv_type == kKvF16)
        return a.c.hd == 64 ? launch_shape<kKvF16, 64>(a, s) : a.c.hd == 128 ? launch_shape<kKvF16, 128>(a, s)
                                                                              : launch_shape<kKvF16, 256>(a, s);
    return a.c.hd == 64 ? launch_shape<kKvInt8, 64>(a, s) : a.c.hd == 128 ? launch_shape<kKvInt8, 128>(a, s)
                                                                           : launch_shape<kKvInt8, 256>(a, s);
}

}  // namespace mnemo
