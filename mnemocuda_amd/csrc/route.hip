// route.hip -- routing of many tokens to their experts.
//
// For every token, from its logits z[e]:
//   s_e = 1 / (1 + exp(-z_e))  or  exp(z_e) / sum_f exp(z_f),   c_e = s_e + bias_e
//   a group of experts scores the sum of its one or two largest c (-inf where it has too few); the best groups are kept
//   the k largest c among them are chosen, ties to the lower index
//   w = s of the chosen, / their sum where asked for, * scale
// Without a bias, and with groups that score one expert or are all kept, c grows with z: the choice is made among the logits.
//
// L lanes (16, 32 or 64) look after a token and hold its experts in registers, a group's in adjacent lanes.
// An expert's place in the order is one number, its key: c with the lowest ten bits giving way to the index.  Scores
// are formed in 64 bits, so that two that differ are told apart (2^-42 of either is what the ten bits cost); k
// rounds take the largest key out.
//
// A call of few tokens is a launch and one token's chain: 33 of 128 experts take 4.6 us.  8191 tokens of 256 experts in 8
// groups take 13 us, bound by instructions in 64 bits, of the scores first and of the rounds then: the 8.9 MB alone
// would take 2.
#include <math.h>

#include "mnemo_common.hpp"
#include "mnemo_internal.hpp"

namespace mnemo {

// An expert's key: c with its lowest ten bits replaced by what orders its index, smaller before larger.  Keys are
// compared as numbers, no two of which are equal (only 0 and -0 would be, and a c below 0, made of a fp32 number, is
// never so small that its key is -0).  kNone is below all of them.
constexpr double kNone = -0x1.fffffffffffffp1023;
__device__ __forceinline__ double make_key(double c, int e) {
    const uint64_t b = __builtin_bit_cast(uint64_t, fmin(c, -kNone));  // (an infinity has no bits to spare)
    return __builtin_bit_cast(double, (b & ~1023ull) | (uint64_t)(b >> 63 ? e : 1023 - e));
}
__device__ __forceinline__ int key_expert(double key) {
    const uint64_t b = __builtin_bit_cast(uint64_t, key);
    return (int)(b >> 63 ? b & 1023 : 1023 - (b & 1023));
}
template <int CTRL>
__device__ __forceinline__ double dpp_double(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, 0xF, 0xF, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, 0xF, 0xF, false);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// over the L lanes of a token, in all of them
template <int L>
__device__ __forceinline__ double max_token(double v) {
    v = fmax(v, dpp_double<kDppXor1>(v));
    v = fmax(v, dpp_double<kDppXor2>(v));
    v = fmax(v, dpp_double<kDppRowHalfMirror>(v));
    v = fmax(v, dpp_double<kDppRowMirror>(v));
    if (L >= 32) v = fmax(v, __shfl_xor(v, 16));
    if (L == 64) v = fmax(v, __shfl_xor(v, 32));
    return v;
}
template <int L>
__device__ __forceinline__ float max_token(float v) {
    v = max16(v);
    if (L >= 32) v = fmaxf(v, __shfl_xor(v, 16));
    if (L == 64) v = fmaxf(v, __shfl_xor(v, 32));
    return v;
}
template <int L>
__device__ __forceinline__ double sum_token(double v) {
    v += dpp_double<kDppXor1>(v);
    v += dpp_double<kDppXor2>(v);
    v += dpp_double<kDppRowHalfMirror>(v);
    v += dpp_double<kDppRowMirror>(v);
    if (L >= 32) v += __shfl_xor(v, 16);
    if (L == 64) v += __shfl_xor(v, 32);
    return v;
}

// exp(v), v <= 0, within 2^-50: 2^n times the series of exp on [-ln 2 / 2, ln 2 / 2] to its 12th power.  The first term
// left out, (ln 2 / 2)^13 / 13!, is 2^-52.4, at most 2^-51.9 of the value; the last sums' roundings and the argument's add
// less than 2^-51.8.  (The largest over 30 million v: 2^-51.3.)
// (-inf: 0; no number: none.)
__device__ __forceinline__ double exp_below(double v) {
    const double n = rint(v * 1.4426950408889634);
    double r = fma(n, -0x1.62e42fefa39efp-1, v);
    r = fma(n, -0x1.abc9e3b39803fp-56, r);
    double p = 1.0 / 479001600;
#pragma unroll
    for (int i = 11; i >= 0; i--) {
        constexpr double f[12] = {1.0, 1.0, 1.0 / 2, 1.0 / 6, 1.0 / 24, 1.0 / 120, 1.0 / 720, 1.0 / 5040, 1.0 / 40320, 1.0 / 362880, 1.0 / 3628800, 1.0 / 39916800};
        p = fma(p, r, f[i]);
    }
    p = ldexp(p, (int)n);
    return v < -745.0 ? 0.0 : p;
}
// 1 / v, 1 <= v, by two Newton steps from the instruction's estimate
__device__ __forceinline__ double inverse(double v) {
    double r = __builtin_amdgcn_rcp(v);
    r = fma(fma(-v, r, 1.0), r, r);
    return fma(fma(-v, r, 1.0), r, r);
}

__device__ __forceinline__ double sigmoid(float z) {
    const double e = exp_below(-fabs((double)z));
    return (z >= 0.0f ? 1.0 : e) * inverse(1.0 + e);  // (no number: no number)
}

// N: experts per lane.  SCORED: c is formed; else the choice is among the logits.
template <int L, int N, bool SCORED>
__global__ void __launch_bounds__(256) route_kernel(RouteArgs a) {
    const int lane = lane_id(), gl = lane % L;
    const int token = blockIdx.x * (256 / L) + threadIdx.x / L;
    const size_t row = min(token, a.n_tokens - 1);
    const float *z = a.z + row * a.n_experts;
    // lane gl: expert first + t of the group
    const int g = gl >> a.lanes_log, i0 = (gl & ((1 << a.lanes_log) - 1)) * a.per_lane;
    const int mine = g < a.n_groups ? min(max(a.per_group - i0, 0), a.per_lane) : 0;
    const int first = mine > 0 ? g * a.per_group + i0 : 0;

    // (loads without branches: what a lane has no experts for is read from where it has some, and dropped)
    float x[N], bias[SCORED ? N : 1];
    auto read = [&](const float *from, float *to) {
        if (a.vec) {  // whole words of four
#pragma unroll
            for (int t = 0; t < N; t += 4) __builtin_memcpy(&to[t], from + first + (t < mine ? t : 0), 16);
        } else {
#pragma unroll
            for (int t = 0; t < N; t++) to[t] = from[first + (t < mine ? t : 0)];
        }
    };
    read(z, x);
    if (SCORED && a.bias) read(a.bias, bias);
#pragma unroll
    for (int t = 0; t < N; t++) x[t] = t < mine ? x[t] : -INFINITY;

    // softmax: the maximum, and the sum where it is asked for
    float m = -INFINITY;
    double total = 1.0;
    if (!a.sigmoid) {
#pragma unroll
        for (int t = 0; t < N; t++) m = fmaxf(m, x[t]);
        m = max_token<L>(m);
        const float ref = m == -INFINITY ? 0.0f : m;
        if (SCORED || !a.renorm) {
            double sum = 0.0;
#pragma unroll
            for (int t = 0; t < N; t++)
                sum += SCORED ? exp_below((double)x[t] - (double)ref) : (double)expf(x[t] - ref);
            total = sum_token<L>(sum);
        }
        m = ref;
    }
    const double share = total > 0.0 || total != total ? 1.0 / total : 0.0;

    double key[N];
    if (SCORED) {
        if (a.sigmoid) {
#pragma unroll
            for (int t = 0; t < N; t++) key[t] = sigmoid(x[t]);
        } else {
#pragma unroll
            for (int t = 0; t < N; t++) key[t] = exp_below((double)x[t] - (double)m) * share;
        }
        if (a.bias) {
#pragma unroll
            for (int t = 0; t < N; t++) key[t] += (double)bias[t];
        }
    } else {
#pragma unroll
        for (int t = 0; t < N; t++) key[t] = x[t];
    }
    double b1 = -INFINITY, b2 = -INFINITY;  // largest c of the lane's experts
    bool bad = false;
#pragma unroll
    for (int t = 0; t < N; t++) {
        const double c = x[t] == -INFINITY ? -INFINITY : key[t] + 0.0;  // (one zero)
        bad |= c != c || (!a.sigmoid && x[t] == INFINITY);
        b2 = fmax(b2, fmin(b1, c));
        b1 = fmax(b1, c);
        key[t] = c > -INFINITY ? make_key(c, first + t) : kNone;
    }
    bad = (__ballot(bad) >> (lane & ~(L - 1)) & (L == 64 ? ~0ull : (1ull << (L & 63)) - 1)) != 0;

    if (a.top_groups < a.n_groups) {
        for (int o = 1; o < 1 << a.lanes_log; o <<= 1) {
            const double o1 = __shfl_xor(b1, o), o2 = __shfl_xor(b2, o);
            b2 = fmax(fmin(b1, o1), fmax(b2, o2));
            b1 = fmax(b1, o1);
        }
        // (of two experts of which one is masked: -inf, whatever the other scores)
        const double score = a.best == 1 ? b1 : b2 > -INFINITY ? b1 + b2 : -INFINITY;
        const double gkey = g < a.n_groups ? make_key(fmax(score, kNone), g) : kNone;
        int better = 0;
        for (int o = 0; o < a.n_groups; o++)
            better += __shfl(gkey, (lane & ~(L - 1)) + (o << a.lanes_log)) > gkey;
        if (better >= a.top_groups) {
#pragma unroll
            for (int t = 0; t < N; t++) key[t] = kNone;
        }
    }

    int mine_idx = -1;
    for (int j = 0; j < a.k; j++) {
        double half[N / 2];
#pragma unroll
        for (int t = 0; t < N / 2; t++) half[t] = fmax(key[t], key[t + N / 2]);
#pragma unroll
        for (int n = N / 4; n > 0; n /= 2)
#pragma unroll
            for (int t = 0; t < n; t++) half[t] = fmax(half[t], half[t + n]);
        const double best = max_token<L>(half[0]);
        if (gl == j && best > kNone) mine_idx = key_expert(best);
        // (whole keys: the index's bits alone are the same for a key of e above 0 and one of 1023 - e below it)
#pragma unroll
        for (int t = 0; t < N; t++) key[t] = key[t] == best ? kNone : key[t];
    }
    double w = 0.0;
    if (mine_idx >= 0) {
        const float zi = z[mine_idx];
        w = a.sigmoid ? sigmoid(zi) : exp_below((double)zi - (double)m);
    }
    if (a.renorm) total = sum_token<L>(w);
    if (a.renorm || !a.sigmoid) w = total > 0.0 ? w / total : 0.0;
    if (token < a.n_tokens && gl < a.k) {
        a.idx[row * a.k + gl] = bad ? -1 : mine_idx;
        a.w[row * a.k + gl] = bad ? NAN : (float)(w * (double)a.scale);
    }
}

template <int L, bool SCORED>
static void launch_lanes(const RouteArgs &a, hipStream_t s) {
    const dim3 grid((a.n_tokens + 256 / L - 1) / (256 / L)), block(256);
    if (a.per_lane <= 4) hipLaunchKernelGGL((route_kernel<L, 4, SCORED>), grid, block, 0, s, a);
    else if (a.per_lane <= 8) hipLaunchKernelGGL((route_kernel<L, 8, SCORED>), grid, block, 0, s, a);
    else if (a.per_lane <= 16) hipLaunchKernelGGL((route_kernel<L, 16, SCORED>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((route_kernel<L, 32, SCORED>), grid, block, 0, s, a);
}

int launch_route(RouteArgs a, hipStream_t s) {
    a.per_group = a.n_experts / a.n_groups;
    if (a.per_group == 1) a.best = 1;
    auto spread = [&](int lanes) {  // a power of two of lanes per group
        a.lanes_log = 0;
        while ((2 << a.lanes_log) * a.n_groups <= lanes) a.lanes_log++;
        a.per_lane = (a.per_group + (1 << a.lanes_log) - 1) >> a.lanes_log;
        if (a.per_group % 4 == 0) a.per_lane = (a.per_lane + 3) & ~3;
    };
    // Few lanes a token do least in all, many are done soonest: 256 experts in 8 groups, 1500 tokens, 64 lanes 6.8 us, 16 9.3; 2048
    // tokens, 32 lanes 7.1, 16 9.4; 8191 13.4 and 13.9; 60,000 65.5 and 62.7 (of 64 experts 28.0 and 15.5).
    int lanes = a.n_tokens < 2048 ? 64 : a.n_tokens < 16384 && a.n_experts >= 256 ? 32 : 16;
    // (a lane of 64 holds at most 32 experts: with 2^n < n_groups <= 2^(n+1) it has the 2^(n+5)th part of a group)
    for (;; lanes *= 2) {
        if (lanes < a.n_groups && lanes < 64) continue;
        spread(lanes);
        if (a.per_lane <= 32) break;
    }
    a.vec = a.per_group % 4 == 0 && ((uintptr_t)a.z | (uintptr_t)a.bias) % 16 == 0;
    const bool scored = a.bias || (a.best == 2 && a.top_groups < a.n_groups);
    if (lanes == 64) scored ? launch_lanes<64, true>(a, s) : launch_lanes<64, false>(a, s);
    else if (lanes == 32) scored ? launch_lanes<32, true>(a, s) : launch_lanes<32, false>(a, s);
    else scored ? launch_lanes<16, true>(a, s) : launch_lanes<16, false>(a, s);
    return check_launch("moe_route");
}

}  // namespace mnemo
