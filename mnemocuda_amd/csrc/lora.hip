// lora.hip -- low-rank adapters of many requests beside a shared projection.
//
//   out_t = base_t + scale_a B_a (A_a x_t),   a = the adapter of token t, or out_t = base_t where it has none
//
// Two launches, both over tiles of 16 tokens, a matrix instruction's columns, and over the adapters that occur in a
// tile (one, in a prompt; up to 16, where 16 requests decode).  The first forms v = A_a x in parts of K, the second
// adds the parts and forms B_a v.  A tile's columns are independent: a column of another adapter's token is formed
// and dropped, so nothing of an adapter reaches another's tokens.
//
// Bound by memory: x, base and out once, each adapter once per tile.
//
// Precision: x and v, fp32, meet f16 adapters as two f16 parts, scaled by a power of two per token so that the largest
// is in [2^13, 2^14) (parts are off by 2^-38 of the largest, or 2^-23 of the value), bf16 adapters as three bf16 parts (exact).
// Sums are fp32.
#include <math.h>

#include "mfma_types.hpp"
#include "mnemo_common.hpp"
#include "mnemo_internal.hpp"

namespace mnemo {

constexpr int kLoTile = 16;     // tokens
constexpr int kLoWaves = 4, kLoThreads = 64 * kLoWaves;
constexpr int kLoChunk = 256;   // of K, per wave and pass
constexpr int kLoStep = kLoChunk * kLoWaves;
constexpr int kLoMaxParts = 8;

// The values of a token's operand (lane: token lane % 16), and what a matrix instruction makes of them.
template <bool BF>
struct LoOperand;
template <>
struct LoOperand<false> {
    h8 hi, lo;
    // scaled by 2^(13 - e), e the exponent of the token's largest
    __device__ __forceinline__ void set(const float (&v)[8], int e) {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            float x = ldexpf(v[j], 13 - e);
            asm("" : "+v"(x));  // one value for both parts
            hi[j] = (_Float16)x;
            lo[j] = (_Float16)(x - (float)hi[j]);
        }
    }
    __device__ __forceinline__ f4 mul(u4 w, f4 acc) const {
        const h8 a = __builtin_bit_cast(h8, w);
        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, hi, acc, 0, 0, 0);
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, lo, acc, 0, 0, 0);
    }
};
template <>
struct LoOperand<true> {
    b8 part[3];
    __device__ __forceinline__ void set(const float (&v)[8], int) { bf16_parts(v, part); }
    __device__ __forceinline__ f4 mul(u4 w, f4 acc) const {
        const b8 a = __builtin_bit_cast(b8, w);
#pragma unroll
        for (int p = 2; p >= 0; p--) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, part[p], acc, 0, 0, 0);
        return acc;
    }
};

// the exponent of the largest of a token's values (-127 for zeros); over the four lanes of the token
__device__ __forceinline__ int lo_exponent(float largest) {
    largest = fmaxf(largest, __shfl_xor(largest, 16));
    largest = fmaxf(largest, __shfl_xor(largest, 32));
    return (int)((__builtin_bit_cast(uint32_t, largest) >> 23) & 255) - 127;
}

// The tile's tokens' adapters: lane's own (of token lane % 16; -1: none, -2: no token) and the first token of each
// distinct one, as a mask of tokens.
__device__ __forceinline__ int lo_ids(const LoraArgs &a, int t0, uint32_t &firsts) {
    const int t = t0 + (lane_id() & 15);
    int id = -2;
    if (t < a.n_tokens) {
        id = a.ids[t];
        if ((unsigned)id >= (unsigned)a.n_adapters || a.ranks[id] <= 0) id = -1;
    }
    bool first = id > -2;
#pragma unroll
    for (int i = 0; i < kLoTile - 1; i++) first &= !((lane_id() & 15) > i && __builtin_amdgcn_readlane(id, i) == id);
    firsts = (uint32_t)__ballot(first) & 0xffffu;
    return id;
}

// parts[kb][t][r] = sum over part kb of K of A_a[r][k] x_t[k].  NR: tiles of 16 ranks.
template <bool BF, int NR>
__global__ void __launch_bounds__(kLoThreads) lora_shrink_kernel(LoraArgs a, int per_part) {
    __shared__ __align__(16) float red[kLoWaves][kLoTile][16 * NR + 4];
    const int lane = lane_id(), c = lane & 15, kg = lane >> 4, wave = threadIdx.x >> 6;
    const int t0 = blockIdx.y * kLoTile, kb = blockIdx.x;
    const int k_from = kb * per_part, k_to = min(a.K, k_from + per_part);
    uint32_t firsts;
    const int id = lo_ids(a, t0, firsts);
    const float *x = a.x + (size_t)min(t0 + c, a.n_tokens - 1) * a.K;
    int d = 0;
    for (; firsts; firsts &= firsts - 1, d++) {
        if (d % gridDim.z != blockIdx.z) continue;
        const int ad = __builtin_amdgcn_readlane(id, __ffs((int)firsts) - 1);
        if (ad < 0) continue;
        const int rank = min(a.ranks[ad], a.max_rank);
        const uint16_t *A = (const uint16_t *)a.a + (size_t)ad * a.max_rank * a.K;
        f4 acc[NR] = {};
        int e = -127;
        for (int k0 = k_from + wave * kLoChunk; k0 < k_to; k0 += kLoStep) {
            float v[8][8];
            float largest = 0.0f;
#pragma unroll
            for (int st = 0; st < 8; st++) {
                const int k = k0 + 32 * st + 8 * kg;
                if (k < k_to) {  // K is a multiple of 8
                    __builtin_memcpy(&v[st][0], x + k, 16);
                    __builtin_memcpy(&v[st][4], x + k + 4, 16);
                } else {
#pragma unroll
                    for (int j = 0; j < 8; j++) v[st][j] = 0.0f;
                }
            }
            u4 w[8];
            auto load = [&](int t) {
                const int r = 16 * t + c;
#pragma unroll
                for (int st = 0; st < 8; st++) {
                    const int k = k0 + 32 * st + 8 * kg;
                    w[st] = u4{0, 0, 0, 0};
                    if (r < rank && k < k_to) __builtin_memcpy(&w[st], A + (size_t)r * a.K + k, 16);
                }
            };
            load(0);
            if (!BF) {
#pragma unroll
                for (int st = 0; st < 8; st++)
#pragma unroll
                    for (int j = 0; j < 8; j++) largest = fmaxf(largest, fabsf(v[st][j]));
                const int en = max(e, lo_exponent(largest));
                if (__any(en != e)) {
#pragma unroll
                    for (int t = 0; t < NR; t++)
#pragma unroll
                        for (int i = 0; i < 4; i++) acc[t][i] = ldexpf(acc[t][i], e - en);
                    e = en;
                }
            }
            LoOperand<BF> o[8];
#pragma unroll
            for (int st = 0; st < 8; st++) o[st].set(v[st], e);
#pragma unroll
            for (int t = 0; t < NR; t++) {
                if (16 * t >= rank) break;
                if (t > 0) load(t);
#pragma unroll
                for (int st = 0; st < 8; st++) acc[t] = o[st].mul(w[st], acc[t]);
            }
        }
        // the waves' sums are added
        __syncthreads();
#pragma unroll
        for (int t = 0; t < NR; t++) {
            f4 y = acc[t];
            if (!BF)
#pragma unroll
                for (int i = 0; i < 4; i++) y[i] = ldexpf(y[i], e - 13);
            __builtin_memcpy(&red[wave][c][16 * t + 4 * kg], &y, 16);
        }
        __syncthreads();
        for (int i = threadIdx.x; i < kLoTile * rank; i += kLoThreads) {
            const int t = i / rank, r = i - t * rank;
            // (t is no lane's own token here)
            if (t0 + t < a.n_tokens && a.ids[t0 + t] == ad)
                a.ws[((size_t)kb * a.n_tokens + t0 + t) * a.max_rank + r] =
                    (red[0][t][r] + red[1][t][r]) + (red[2][t][r] + red[3][t][r]);
        }
    }
}

// out_t[m] = base_t[m] + scale sum_r B_a[m][r] v_t[r].  NS: steps of 32 ranks.  A wave has per_wave outputs.
template <bool BF, int NS>
__global__ void __launch_bounds__(kLoThreads) lora_expand_kernel(LoraArgs a, int parts, int per_wave) {
    constexpr int U = NS <= 2 ? 4 : 1;  // tiles of 16 outputs at once
    const int lane = lane_id(), c = lane & 15, kg = lane >> 4, wave = threadIdx.x >> 6;
    const int t0 = blockIdx.y * kLoTile;
    const int m_from = (blockIdx.x * kLoWaves + wave) * per_wave, m_to = min(a.M, m_from + per_wave);
    uint32_t firsts;
    const int id = lo_ids(a, t0, firsts);
    const size_t row = (size_t)min(t0 + c, a.n_tokens - 1);
    const float *base = a.base + row * a.M;
    float *out = a.out + row * a.M;
    int d = 0;
    for (; firsts; firsts &= firsts - 1, d++) {
        if (d % gridDim.z != blockIdx.z) continue;
        const int ad = __builtin_amdgcn_readlane(id, __ffs((int)firsts) - 1);
        const bool mine = id == ad;
        if (ad < 0) {
            if (a.out != a.base && mine)
                for (int m = m_from + 4 * kg; m < m_to; m += 16) {
                    f4 y;
                    if (m + 3 < m_to) {
                        __builtin_memcpy(&y, base + m, 16);
                        __builtin_memcpy(out + m, &y, 16);
                    } else
                        for (int i = 0; m + i < m_to; i++) out[m + i] = base[m + i];
                }
            continue;
        }
        const int rank = min(a.ranks[ad], a.max_rank);
        const float scale = a.scales[ad];
        const uint16_t *B = (const uint16_t *)a.b + (size_t)ad * a.M * a.max_rank;
        LoOperand<BF> o[NS];
        int e = -127;
        {
            float v[NS][8], largest = 0.0f;
#pragma unroll
            for (int st = 0; st < NS; st++) {
                const int r = 32 * st + 8 * kg;
#pragma unroll
                for (int j = 0; j < 8; j++) v[st][j] = 0.0f;
                if (mine && r < rank)
                    for (int p = 0; p < parts; p++) {
                        float y[8];
                        __builtin_memcpy(y, a.ws + ((size_t)p * a.n_tokens + row) * a.max_rank + r, 32);
#pragma unroll
                        for (int j = 0; j < 8; j++) v[st][j] += r + j < rank ? y[j] : 0.0f;
                    }
#pragma unroll
                for (int j = 0; j < 8; j++) largest = fmaxf(largest, fabsf(v[st][j]));
            }
            if (!BF) e = lo_exponent(largest);
#pragma unroll
            for (int st = 0; st < NS; st++) o[st].set(v[st], e);
        }
        for (int m0 = m_from; m0 < m_to; m0 += 16 * U) {
            u4 w[U][NS];
            f4 y[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int m = m0 + 16 * u + c, mo = m0 + 16 * u + 4 * kg;
#pragma unroll
                for (int st = 0; st < NS; st++) {
                    const int r = 32 * st + 8 * kg;
                    w[u][st] = u4{0, 0, 0, 0};
                    if (m < m_to && r < rank) __builtin_memcpy(&w[u][st], B + (size_t)m * a.max_rank + r, 16);
                }
                y[u] = f4{0.f, 0.f, 0.f, 0.f};
                if (mine) {
                    if (mo + 3 < m_to) __builtin_memcpy(&y[u], base + mo, 16);
                    else
                        for (int i = 0; i < 4; i++)
                            if (mo + i < m_to) y[u][i] = base[mo + i];
                }
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int mo = m0 + 16 * u + 4 * kg;
                f4 acc = {};
#pragma unroll
                for (int st = 0; st < NS; st++) {
                    if (32 * st >= rank) break;
                    if (32 * st + 32 > rank) {  // what lies behind the rank may be no number
                        const int live = rank - 32 * st - 8 * kg;
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            w[u][st][j] = live > 2 * j + 1 ? w[u][st][j] : live > 2 * j ? w[u][st][j] & 0xffffu : 0;
                    }
                    acc = o[st].mul(w[u][st], acc);
                }
                f4 z;
#pragma unroll
                for (int i = 0; i < 4; i++) z[i] = fmaf(scale, BF ? acc[i] : ldexpf(acc[i], e - 13), y[u][i]);
                if (mine) {
                    if (mo + 3 < m_to) __builtin_memcpy(out + mo, &z, 16);
                    else
                        for (int i = 0; i < 4; i++)
                            if (mo + i < m_to) out[mo + i] = z[i];
                }
            }
        }
    }
}

// Parts of K: as many as there are steps, but few enough that adding them stays cheap.
static int lo_parts(int K, int *per_part) {
    const int steps = (K + kLoStep - 1) / kLoStep;
    const int per = (steps + kLoMaxParts - 1) / kLoMaxParts;
    *per_part = per * kLoStep;
    return (steps + per - 1) / per;
}

size_t lora_workspace_bytes(int n_tokens, int K, int max_rank) {
    int per;
    return (size_t)lo_parts(K, &per) * n_tokens * max_rank * sizeof(float);
}

template <bool BF>
static int launch_typed(const LoraArgs &a, hipStream_t s) {
    int per_part;
    const int parts = lo_parts(a.K, &per_part), tiles = (a.n_tokens + kLoTile - 1) / kLoTile;
    // a tile's adapters by workgroups of their own, where tiles alone do not fill the chip
    int z = tiles >= 64 ? 1 : kLoTile;
    z = z < a.n_tokens ? z : a.n_tokens;
    z = z < a.n_adapters + 1 ? z : a.n_adapters + 1;
    const dim3 block(kLoThreads);
    const dim3 g1(parts, tiles, z);
    const int ranks = (a.max_rank + 15) / 16;
#define MNEMO_SHRINK(N) hipLaunchKernelGGL((lora_shrink_kernel<BF, N>), g1, block, 0, s, a, per_part)
    if (ranks <= 1) MNEMO_SHRINK(1);
    else if (ranks <= 2) MNEMO_SHRINK(2);
    else if (ranks <= 4) MNEMO_SHRINK(4);
    else if (ranks <= 8) MNEMO_SHRINK(8);
    else MNEMO_SHRINK(16);
#undef MNEMO_SHRINK
    if (int rc = check_launch("lora_add")) return rc;
    const int per_wave = 256;
    const dim3 g2((a.M + kLoWaves * per_wave - 1) / (kLoWaves * per_wave), tiles, z);
#define MNEMO_EXPAND(N) hipLaunchKernelGGL((lora_expand_kernel<BF, N>), g2, block, 0, s, a, parts, per_wave)
    if (ranks <= 2) MNEMO_EXPAND(1);
    else if (ranks <= 4) MNEMO_EXPAND(2);
    else if (ranks <= 8) MNEMO_EXPAND(4);
    else MNEMO_EXPAND(8);
#undef MNEMO_EXPAND
    return check_launch("lora_add");
}

int launch_lora(const LoraArgs &a, hipStream_t s) { return a.bf16 ? launch_typed<true>(a, s) : launch_typed<false>(a, s); }

}  // namespace mnemo
