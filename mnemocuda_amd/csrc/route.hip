// route.hip -- routing of many tokens to their experts.
//
// For every token, from its logits z[e]:
//   s_e = 1 / (1 + exp(-z_e))  or  exp(z_e) / sum_f exp(z_f),   c_e = s_e + bias_e
//   a group of experts scores the sum of its one or two largest c; the best groups are kept
//   the k largest c among them are chosen, ties to the lower index
//   w = s of the chosen, / their sum where asked for, * scale
// Without a bias, and with groups that score one expert, c grows with z: the choice is made among the logits.
//
// L lanes (16 or 64) look after a token and hold its experts in registers, a group's in adjacent lanes.
// An expert's place in the order is one 64-bit key: the bits of c as a whole number that orders as c does, its
// lowest ten replaced by 1023 - e.  Scores are formed in 64 bits, so that two that differ are told apart
// (2^-42 of either is what the ten bits cost); k rounds take the largest key out.
#include <math.h>

#include "mnemo_common.hpp"
#include "mnemo_internal.hpp"

namespace mnemo {

// a whole number that orders as v does
__device__ __forceinline__ uint64_t order_bits(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    return b >> 63 ? ~b : b | 1ull << 63;
}
__device__ __forceinline__ uint64_t max64(uint64_t a, uint64_t b) { return a > b ? a : b; }
template <int CTRL>
__device__ __forceinline__ uint64_t dpp_u64(uint64_t v) {
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, 0xF, 0xF, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, 0xF, 0xF, false);
    return (uint64_t)hi << 32 | lo;
}
// over the L lanes of a token, in all of them
template <int L>
__device__ __forceinline__ uint64_t max_token(uint64_t v) {
    v = max64(v, dpp_u64<kDppXor1>(v));
    v = max64(v, dpp_u64<kDppXor2>(v));
    v = max64(v, dpp_u64<kDppRowHalfMirror>(v));
    v = max64(v, dpp_u64<kDppRowMirror>(v));
    if (L == 64) {
        v = max64(v, __shfl_xor((unsigned long long)v, 16));
        v = max64(v, __shfl_xor((unsigned long long)v, 32));
    }
    return v;
}
template <int L>
__device__ __forceinline__ float max_token(float v) {
    v = max16(v);
    if (L == 64) {
        v = fmaxf(v, __shfl_xor(v, 16));
        v = fmaxf(v, __shfl_xor(v, 32));
    }
    return v;
}
template <int L>
__device__ __forceinline__ double sum_token(double v) {
#pragma unroll
    for (int o = 1; o < L; o <<= 1) v += __shfl_xor(v, o);
    return v;
}

__device__ __forceinline__ double sigmoid(float z) {
    const double e = exp(-fabs((double)z));
    return (z >= 0.0f ? 1.0 : e) / (1.0 + e);  // (no number: no number)
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

    float x[N];
    if (a.vec) {  // whole words of four
#pragma unroll
        for (int t = 0; t < N; t += 4) {
#pragma unroll
            for (int j = 0; j < 4 && t + j < N; j++) x[t + j] = -INFINITY;
            if (N >= 4 && t < mine) __builtin_memcpy(&x[t], z + first + t, 16);
        }
    } else {
#pragma unroll
        for (int t = 0; t < N; t++) x[t] = t < mine ? z[first + t] : -INFINITY;
    }

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
                if (t < a.per_lane) sum += SCORED ? exp((double)x[t] - (double)ref) : (double)expf(x[t] - ref);
            total = sum_token<L>(sum);
        }
        m = ref;
    }

    uint64_t key[N];
    double b1 = -INFINITY, b2 = -INFINITY;  // largest c of the lane's experts
    bool bad = false;
#pragma unroll
    for (int t = 0; t < N; t++) {
        key[t] = 0;
        if (t < a.per_lane) {
            double c = x[t];
            if (SCORED) {
                c = a.sigmoid ? sigmoid(x[t]) : exp((double)x[t] - (double)m) / total;
                if (a.bias) c += t < mine ? (double)a.bias[first + t] : 0.0;
            }
            c += 0.0;  // one zero
            if (x[t] == -INFINITY) c = -INFINITY;
            if (t < mine) bad |= c != c || (!a.sigmoid && x[t] == INFINITY);
            if (t < mine && c > -INFINITY) key[t] = (order_bits(c) & ~1023ull) | (uint64_t)(1023 - (first + t));
            else c = -INFINITY;
            b2 = fmax(b2, fmin(b1, c));
            b1 = fmax(b1, c);
        }
    }
    bad = (__ballot(bad) >> (lane & ~(L - 1)) & (L == 64 ? ~0ull : 0xffffull)) != 0;

    if (a.top_groups < a.n_groups) {
        for (int o = 1; o < 1 << a.lanes_log; o <<= 1) {
            const double o1 = __shfl_xor(b1, o), o2 = __shfl_xor(b2, o);
            b2 = fmax(fmin(b1, o1), fmax(b2, o2));
            b1 = fmax(b1, o1);
        }
        const double score = a.best == 2 && b2 > -INFINITY ? b1 + b2 : b1;
        const uint64_t gkey = g < a.n_groups && b1 > -INFINITY ? (order_bits(score) & ~63ull) | (uint64_t)(63 - g) : 0;
        int better = 0;
        for (int o = 0; o < a.n_groups; o++)
            better += __shfl((unsigned long long)gkey, (lane & ~(L - 1)) + (o << a.lanes_log)) > gkey;
        if (better >= a.top_groups) {
#pragma unroll
            for (int t = 0; t < N; t++) key[t] = 0;
        }
    }

    int mine_idx = -1;
    for (int j = 0; j < a.k; j++) {
        uint64_t best = key[0];
#pragma unroll
        for (int t = 1; t < N; t++) best = max64(best, key[t]);
        best = max_token<L>(best);
        if (gl == j && best) mine_idx = 1023 - (int)(best & 1023);
#pragma unroll
        for (int t = 0; t < N; t++) key[t] = key[t] == best ? 0 : key[t];
    }
    double w = 0.0;
    if (mine_idx >= 0) {
        const float zi = z[mine_idx];
        w = a.sigmoid ? sigmoid(zi) : exp((double)zi - (double)m);
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
    auto spread = [&](int lanes) {  // a power of two of lanes per group
        a.lanes_log = 0;
        while ((2 << a.lanes_log) * a.n_groups <= lanes) a.lanes_log++;
        a.per_lane = (a.per_group + (1 << a.lanes_log) - 1) >> a.lanes_log;
        if (a.per_group % 4 == 0) a.per_lane = (a.per_lane + 3) & ~3;
    };
    // a lane of 64 holds at most 32 experts: with 2^n < n_groups <= 2^(n+1) it has the 2^(n+5)th part of a group
    bool wide = a.n_groups > 16 || a.n_tokens < 2048;
    if (!wide) {
        spread(16);
        wide = a.per_lane > 32;
    }
    if (wide) spread(64);
    a.vec = a.per_group % 4 == 0 && (uintptr_t)a.z % 16 == 0;
    const bool scored = a.bias || (a.best == 2 && a.top_groups < a.n_groups);
    if (wide) scored ? launch_lanes<64, true>(a, s) : launch_lanes<64, false>(a, s);
    else scored ? launch_lanes<16, true>(a, s) : launch_lanes<16, false>(a, s);
    return check_launch("moe_route");
}

}  // namespace mnemo
