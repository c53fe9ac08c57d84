// logprobs.hip -- log probabilities of given tokens, their ranks, the entropy and the likeliest tokens of rows of
// logits.
//
// With m = max z, S = sum exp(z - m), T = sum exp(z - m) (z - m):
//   log p_t = z_t - m - log S,   entropy = -sum p log p = log S - T / S,
//   rank = 1 + the tokens before t in the order (z falling, index rising).
// One pass over the logits: a thread keeps m, S and T of what it has seen (S and T are rescaled when m rises)
// and the count of tokens before t.  A wave keeps its likeliest tokens as 64 sorted keys, one a lane: the bits of
// z as a whole number that orders as z does, over the complement of the index.  Few tokens get so far as to be
// looked at: a thread compares the largest of its 16 logits with the workgroup's n-th best so far.  Lists are
// merged as two halves of a bitonic sequence.
// Rows are cut into parts where they do not fill the chip; a second launch joins the parts.
//
// Bound by reading the logits once, which are loaded past the caches: 1201 rows of 151,936 take 122 to 129 us, 5.7 to 6.0 TB/s.  Few rows
// are bound by the two launches and what each waits for: one row takes 14 us, 31 of 32,003 12; short rows by the lists'
// beginnings: 1000 of 32,003 take 24 us without, 28 with 5 tokens each and 38 with 20.
#include <float.h>
#include <math.h>

#include "mnemo_common.hpp"
#include "mnemo_internal.hpp"

namespace mnemo {

typedef float lpf4 __attribute__((ext_vector_type(4)));
typedef lpf4 lpf4u __attribute__((aligned(4)));

constexpr int kLpThreads = 256, kLpWaves = kLpThreads / 64;
constexpr int kLpWords = 4;                           // words of four logits per thread and step
constexpr int kLpStep = 4 * kLpThreads * kLpWords;    // logits of a step
constexpr float kLpLog2e = 1.44269504088896341f;

// Rows 0 .. whole-1 are done by a workgroup each, the others in parts of per_part logits, which a second launch joins.
struct LpPlan {
    int whole, parts, per_part;
};
struct LpSums {
    float m, S, T;  // m is at least -FLT_MAX: a row without any number has S = 0
    int before;     // tokens before the target
};

template <int O>
struct Lane {
    static constexpr int value = O;
};

__device__ __forceinline__ uint32_t order32(float v) {
    const uint32_t b = __builtin_bit_cast(uint32_t, v + 0.0f);  // one zero
    return b >> 31 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unorder32(uint32_t b) {
    return __builtin_bit_cast(float, b >> 31 ? b & 0x7fffffffu : ~b);
}
__device__ __forceinline__ uint64_t lp_key(float z, int id) { return (uint64_t)order32(z) << 32 | (0xffffffffu - (uint32_t)id); }

__device__ __forceinline__ uint64_t lane64(uint64_t v, int l) {
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)v, l), hi = __builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), l);
    return (uint64_t)hi << 32 | lo;
}
// v of lane ^ O
template <int O>
__device__ __forceinline__ uint32_t xor_lanes(uint32_t v) {
    if (O == 32 || O == 16) {
        // the swap leaves the lower (even) rows' values everywhere in one register, the upper ones' in the other
        const auto p = O == 32 ? __builtin_amdgcn_permlane32_swap(v, v, false, false) : __builtin_amdgcn_permlane16_swap(v, v, false, false);
        return lane_id() & O ? p[0] : p[1];
    }
    if (O == 8) return __builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xF, 0xF, false);  // row_ror:8
    if (O == 4) {  // ^7, then ^3
        const int h = __builtin_amdgcn_update_dpp(0, (int)v, kDppRowHalfMirror, 0xF, 0xF, false);
        return __builtin_amdgcn_update_dpp(0, h, 0x1B, 0xF, 0xF, false);
    }
    return __builtin_amdgcn_update_dpp(0, (int)v, O == 2 ? kDppXor2 : kDppXor1, 0xF, 0xF, false);
}
template <int O>
__device__ __forceinline__ uint64_t xor64(uint64_t v) {
    return (uint64_t)xor_lanes<O>((uint32_t)(v >> 32)) << 32 | xor_lanes<O>((uint32_t)v);
}
template <int O>
__device__ __forceinline__ double xor_double(double v) { return __builtin_bit_cast(double, xor64<O>(__builtin_bit_cast(uint64_t, v))); }

// One step of a sorting network: lanes whose bit O is clear take the larger where `down` is set.
template <int O>
__device__ __forceinline__ uint64_t lp_exchange(uint64_t v, bool down) {
    const uint64_t w = xor64<O>(v);
    const bool larger = ((lane_id() & O) == 0) == down;
    return (v > w) == larger ? v : w;
}
// a bitonic sequence of 2 O lanes, sorted
template <int O>
__device__ __forceinline__ uint64_t lp_merge(uint64_t v, bool down) {
    v = lp_exchange<O>(v, down);
    if constexpr (O > 1) v = lp_merge<O / 2>(v, down);
    return v;
}
template <int N>
__device__ __forceinline__ uint64_t lp_sort(uint64_t v) {  // runs of N lanes, falling and rising in turn
    if constexpr (N > 2) v = lp_sort<N / 2>(v);
    return lp_merge<N / 2>(v, N == 64 || (lane_id() & N) == 0);
}
// the 64 largest of two lists, sorted
__device__ __forceinline__ uint64_t lp_join(uint64_t a, uint64_t b) {
    const uint64_t r = __shfl((unsigned long long)b, 63 - lane_id());
    return lp_merge<32>(a > r ? a : r, true);
}

// What is known of a row goes out (wave 0): list is sorted.
__device__ __forceinline__ void lp_finish(const LogprobsArgs &a, int r, float m, double S, double T, int before, float zt,
                                          int t, uint64_t list) {
    const int lane = lane_id();
    const double logS = log(S);
    const bool none = S == 0.0, bad = S != S;
    if (lane == 0) {
        if (a.targets) {
            const bool in = (unsigned)t < (unsigned)a.vocab;
            float lp = (float)((double)zt - (double)m - logS);
            if (none) lp = -INFINITY;
            if (bad) lp = NAN;
            a.logp[r] = in ? lp : 0.0f;
            if (a.rank) a.rank[r] = in && !bad ? before + 1 : 0;
        }
        if (a.entropy) a.entropy[r] = bad ? NAN : none ? 0.0f : (float)(logS - T / S);
    }
    if (lane < a.k) {
        const float z = unorder32((uint32_t)(list >> 32));
        const bool is = list != 0 && z > -INFINITY && !bad;
        a.ids[(size_t)r * a.k + lane] = is ? (int)(0xffffffffu - (uint32_t)list) : -1;
        a.tops[(size_t)r * a.k + lane] = bad ? NAN : is ? (float)((double)z - (double)m - logS) : -INFINITY;
    }
}

// The lanes' sums joined, in every lane: all relative to the largest m, then added.
__device__ __forceinline__ void lp_join_lanes(float &m, double &S, double &T, int &before) {
    float M = max16(m);
    M = fmaxf(M, __builtin_bit_cast(float, xor_lanes<16>(__builtin_bit_cast(uint32_t, M))));
    M = fmaxf(M, __builtin_bit_cast(float, xor_lanes<32>(__builtin_bit_cast(uint32_t, M))));
    if (m < M) {
        const double d = (double)m - (double)M, f = exp(d);
        T = f * (T + S * fmax(d, -1e30));
        S *= f;
    }
    m = M;
    auto add = [&](auto o) {
        constexpr int O = decltype(o)::value;
        S += xor_double<O>(S);
        T += xor_double<O>(T);
        before += (int)xor_lanes<O>((uint32_t)before);
    };
    add(Lane<1>{});
    add(Lane<2>{});
    add(Lane<4>{});
    add(Lane<8>{});
    add(Lane<16>{});
    add(Lane<32>{});
}

template <bool TOP>
__global__ void __launch_bounds__(kLpThreads) logprobs_kernel(LogprobsArgs a, LpPlan p) {
    __shared__ uint64_t lists[TOP ? kLpWaves : 1][64];
    __shared__ LpSums sums[kLpWaves];
    __shared__ uint32_t floor_;  // the best of the waves' n-th best so far (as order32)
    const int cut = (int)blockIdx.x - p.whole;  // of the rows that are cut: row and part
    const int r = cut < 0 ? (int)blockIdx.x : p.whole + cut / p.parts, part = cut < 0 ? 0 : cut % p.parts, tid = threadIdx.x, lane = lane_id(), wave = tid >> 6;
    const float *z = a.z + (size_t)r * a.vocab;
    const int from = part * p.per_part, to = cut < 0 ? a.vocab : min(a.vocab, from + p.per_part);
    if (TOP && tid == 0) floor_ = 0;

    const int t = a.targets ? a.targets[r] : -1;
    const float zt = (unsigned)t < (unsigned)a.vocab ? z[t] : INFINITY;

    lpf4 x[kLpWords];
    auto load = [&](int at) {
#pragma unroll
        for (int g = 0; g < kLpWords; g++) {
            const int i = at + 4 * (kLpThreads * g + tid);
            if (i + 3 < to) x[g] = __builtin_nontemporal_load((const lpf4u *)(z + i));
            else
                for (int j = 0; j < 4; j++) x[g][j] = i + j < to ? z[i + j] : -INFINITY;
        }
    };
    load(from);
    LpSums s = {-FLT_MAX, 0.0f, 0.0f, 0};
    uint64_t list = 0;
    float least = -INFINITY;  // the wave's n-th best so far
    if (TOP) __syncthreads();
    for (int at = from; at < to; at += kLpStep) {
        lpf4 y[kLpWords];
#pragma unroll
        for (int g = 0; g < kLpWords; g++) y[g] = x[g];
        if (at + kLpStep < to) load(at + kLpStep);
        float top = -INFINITY;
#pragma unroll
        for (int g = 0; g < kLpWords; g++)
#pragma unroll
            for (int j = 0; j < 4; j++) top = fmaxf(top, y[g][j]);
        if (top > s.m) {
            const float d = s.m - top, f = __builtin_amdgcn_exp2f(d * kLpLog2e);
            s.T = f * fmaf(s.S, fmaxf(d, -1e30f), s.T);
            s.S *= f;
            s.m = top;
        }
        float S = 0.0f, T = 0.0f;  // of the step, so that a long row's sums are not of thousands of additions
#pragma unroll
        for (int g = 0; g < kLpWords; g++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float d = y[g][j] - s.m, e = __builtin_amdgcn_exp2f(d * kLpLog2e);
                S += e;
                T = fmaf(e, fmaxf(d, -1e30f), T);
            }
        s.S += S;
        s.T += T;
        const int first = at + 4 * tid;
        if (a.rank) {
            if (at + kLpStep <= t) {
#pragma unroll
                for (int g = 0; g < kLpWords; g++)
#pragma unroll
                    for (int j = 0; j < 4; j++) s.before += y[g][j] >= zt;
            } else if (at > t) {
#pragma unroll
                for (int g = 0; g < kLpWords; g++)
#pragma unroll
                    for (int j = 0; j < 4; j++) s.before += y[g][j] > zt;
            } else {
#pragma unroll
                for (int g = 0; g < kLpWords; g++)
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        s.before += y[g][j] > zt || (y[g][j] == zt && first + 4 * kLpThreads * g + j < t);
            }
        }
        if (TOP) {
            uint64_t own = 0;
            if (at == from) {  // the lanes' best are a list to begin with
#pragma unroll
                for (int g = 0; g < kLpWords; g++)
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const uint64_t c = lp_key(y[g][j], first + 4 * kLpThreads * g + j);
                        own = c > own ? c : own;
                    }
                list = lp_sort<64>(own);
                least = unorder32((uint32_t)(lane64(list, a.k - 1) >> 32));
            }
            const uint32_t known = *(volatile uint32_t *)&floor_;
            if (known) least = fmaxf(least, unorder32(known));
            if (__any(top >= least)) {
                uint64_t last = lane64(list, a.k - 1);
#pragma unroll
                for (int g = 0; g < kLpWords; g++)
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const bool in = y[g][j] >= least;  // (looked at alone: 1000 rows of 151,936 take 112 us, 129 with all at once)
                        if (__ballot(in) == 0) continue;
                        const uint64_t c = lp_key(y[g][j], first + 4 * kLpThreads * g + j);
                        uint64_t left = __ballot(in && c > last && c != own);
                        while (left) {
                            const uint64_t one = lane64(c, __ffsll((unsigned long long)left) - 1);
                            left &= left - 1;
                            if (one <= last) continue;
                            const int place = __popcll(__ballot(list > one));
                            const uint64_t up = __shfl_up((unsigned long long)list, 1);
                            list = lane < place ? list : lane == place ? one : up;
                            last = lane64(list, a.k - 1);
                        }
                    }
                const uint32_t l = (uint32_t)(last >> 32);
                least = fmaxf(least, unorder32(l));
                if (lane == 0 && l > known) atomicMax(&floor_, l);
            }
        }
    }
    float m = s.m;
    double S = s.S, T = s.T;
    int before = s.before;
    lp_join_lanes(m, S, T, before);
    if (lane == 0) sums[wave] = {m, (float)S, (float)T, before};
    if (TOP) lists[wave][lane] = list;
    __syncthreads();
    if (wave != 0) return;
    const LpSums q = sums[lane & (kLpWaves - 1)];
    m = q.m;
    S = lane < kLpWaves ? q.S : 0.0f;
    T = lane < kLpWaves ? q.T : 0.0f;
    before = lane < kLpWaves ? q.before : 0;
    lp_join_lanes(m, S, T, before);
    if (TOP)
        for (int w = 1; w < kLpWaves; w++) list = lp_join(list, lists[w][lane]);
    if (cut < 0) lp_finish(a, r, m, S, T, before, zt, t, list);
    else {
        if (lane == 0) ((LpSums *)a.ws)[cut] = {m, (float)S, (float)T, before};
        if (TOP && lane < a.k) ((uint64_t *)((LpSums *)a.ws + (size_t)(a.n_rows - p.whole) * p.parts))[(size_t)cut * a.k + lane] = list;
    }
}

// Joins the parts (at most 64) of the cut row blockIdx.x: wave w of 16 the lists of parts w, w + 16, ...
template <bool TOP>
__global__ void __launch_bounds__(TOP ? 1024 : 64) logprobs_join_kernel(LogprobsArgs a, LpPlan p) {
    __shared__ uint64_t lists[TOP ? 16 : 1][64];
    const int cut = blockIdx.x, r = p.whole + cut, parts = p.parts, lane = lane_id(), wave = threadIdx.x >> 6;
    uint64_t list = 0;
    if (TOP) {
        const uint64_t *l = (const uint64_t *)((const LpSums *)a.ws + (size_t)(a.n_rows - p.whole) * parts) + (size_t)cut * parts * a.k;
        for (int i = wave; i < parts; i += 16) {
            const uint64_t one = lane < a.k ? l[(size_t)i * a.k + lane] : 0;
            list = i == wave ? one : lp_join(list, one);
        }
        for (int half = 8; half > 0; half >>= 1) {
            if (wave >= half) lists[wave][lane] = list;
            __syncthreads();
            if (wave < half && wave + half < parts) list = lp_join(list, lists[wave + half][lane]);
        }
    }
    if (wave != 0) return;
    const LpSums q = lane < parts ? ((const LpSums *)a.ws)[(size_t)cut * parts + lane] : LpSums{-FLT_MAX, 0.0f, 0.0f, 0};
    float m = q.m;
    double S = q.S, T = q.T;
    int before = q.before;
    lp_join_lanes(m, S, T, before);
    const int t = a.targets ? a.targets[r] : -1;
    const float zt = (unsigned)t < (unsigned)a.vocab ? a.z[(size_t)r * a.vocab + t] : 0.0f;
    lp_finish(a, r, m, S, T, before, zt, t, list);
}

// 1024 workgroups, four a CU, are at work at once: as many rows as fill them once or more are done whole, the others
// (all, where there are fewer) are cut into parts of at least a step, so that they fill them too.
static LpPlan lp_plan(int n_rows, int vocab) {
    LpPlan p;
    p.whole = n_rows / 1024 * 1024;
    const int rest = n_rows - p.whole;
    const long long steps = ((long long)vocab + kLpStep - 1) / kLpStep;
    long long parts = rest ? 1024 / rest : 1;
    if (parts > 64) parts = 64;
    if (parts > steps) parts = steps;
    const long long per = (steps + parts - 1) / parts;
    p.parts = (int)((steps + per - 1) / per);
    p.per_part = (int)(per * kLpStep < vocab ? per * kLpStep : vocab);
    if (p.parts == 1) p.whole = n_rows;
    return p;
}

// Enough for every call of no more rows: there are at most 1024 parts.
size_t logprobs_workspace_bytes(int n_rows, int vocab, int k) {
    const long long steps = ((long long)vocab + kLpStep - 1) / kLpStep, most = (steps < 64 ? steps : 64) * n_rows;
    return (size_t)(most < 1024 ? most : 1024) * (sizeof(LpSums) + (size_t)k * 8);
}

int launch_logprobs(const LogprobsArgs &a, hipStream_t s) {
    const LpPlan p = lp_plan(a.n_rows, a.vocab);
    const int rest = a.n_rows - p.whole;
    const dim3 grid(p.whole + rest * p.parts), block(kLpThreads);
    if (a.k) hipLaunchKernelGGL(logprobs_kernel<true>, grid, block, 0, s, a, p);
    else hipLaunchKernelGGL(logprobs_kernel<false>, grid, block, 0, s, a, p);
    if (int rc = check_launch("logprobs")) return rc;
    if (rest == 0) return kOk;
    if (a.k) hipLaunchKernelGGL(logprobs_join_kernel<true>, dim3(rest), dim3(1024), 0, s, a, p);
    else hipLaunchKernelGGL(logprobs_join_kernel<false>, dim3(rest), dim3(64), 0, s, a, p);
    return check_launch("logprobs");
}

}  // namespace mnemo
