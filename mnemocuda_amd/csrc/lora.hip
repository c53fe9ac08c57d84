// lora.hip -- low-rank adapters of many requests beside a shared projection.
//
//   out_t = base_t + scale_a B_a (A_a x_t),   a = the adapter of token t, or out_t = base_t where it has none
//
// Two launches, both over tiles of 16 tokens, a matrix instruction's columns, and over the adapters that occur in a
// tile (one, in a prompt; up to 16, where 16 requests decode).  The first forms v = A_a x in parts of K, the second
// adds the parts and forms B_a v.  A tile's columns are independent: a column of another adapter's token is formed
// and dropped, so nothing of an adapter reaches another's tokens.
//
// Bound by memory: x, base and out once, each adapter once per tile.  3001 tokens of ranks to 32 (bf16, 4096 to 8192 features, 248 MB)
// take 70 us with nothing in the caches, 8000 tokens 145 (4.5 TB/s; a copy reaches 5.2), of which the first launch, x, is a
// third.  Few tokens are bound by what a launch waits for in turn, ids, ranks, words and the other launch: one token 9 us,
// 61 of 40 adapters 24, where lines of B of which a low rank has a part are read whole as well.  Asking for B before v
// is known costs more in registers than it hides (24 and 23, but one token 9 and 9.5, 3001 70 and 74).  High ranks of many
// tokens are bound by A and B, which every tile reads again from the L2 caches: 3001 tokens of rank 200 take 192 us, 4.9 TB/s of
// them (the next words of B asked for ahead of the products: 193 f16, 225 bf16, for spilled registers).
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
constexpr int kLoShrinkWaves = 8, kLoExpandWaves = 4;
constexpr int kLoChunk = 128, kLoSteps = kLoChunk / 32;  // of K, per wave and pass
constexpr int kLoStep = kLoChunk * kLoShrinkWaves;
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
__global__ void __launch_bounds__(64 * kLoShrinkWaves, NR <= 4 ? 4 : 2) lora_shrink_kernel(LoraArgs a, int per_part) {
    constexpr int kThreads = 64 * kLoShrinkWaves;
    __shared__ __align__(16) float red[kLoShrinkWaves][kLoTile][16 * NR + 4];
    const int lane = lane_id(), c = lane & 15, kg = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
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
            float v[kLoSteps][8];
            float largest = 0.0f;
#pragma unroll
            for (int st = 0; st < kLoSteps; st++) {
                const int k = k0 + 32 * st + 8 * kg;  // K is a multiple of 8
#pragma unroll
                for (int j = 0; j < 8; j++) v[st][j] = 0.0f;
                if (id == ad && k < k_to) {
                    __builtin_memcpy(&v[st][0], x + k, 16);
                    __builtin_memcpy(&v[st][4], x + k + 4, 16);
                }
            }
            u4 w[2][kLoSteps];  // of a tile of ranks and of the next
            auto load = [&](int t) {
                // (no branches: rows behind the rank, whose sums are dropped, and words behind K, which meet zeros in x, are others')
                const uint16_t *row = A + (size_t)min(16 * t + c, rank - 1) * a.K;
#pragma unroll
                for (int st = 0; st < kLoSteps; st++) __builtin_memcpy(&w[t & 1][st], row + min(k0 + 32 * st + 8 * kg, a.K - 8), 16);
            };
            load(0);
            if (NR > 1) load(1);
            if (!BF) {
#pragma unroll
                for (int st = 0; st < kLoSteps; st++)
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
            LoOperand<BF> o[kLoSteps];
#pragma unroll
            for (int st = 0; st < kLoSteps; st++) o[st].set(v[st], e);
#pragma unroll
            for (int t = 0; t < NR; t++) {
                if (16 * t < rank) {
#pragma unroll
                    for (int st = 0; st < kLoSteps; st++) acc[t] = o[st].mul(w[t & 1][st], acc[t]);
                    if (t + 2 < NR) load(t + 2);
                }
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
        for (int i = threadIdx.x; i < kLoTile * rank; i += kThreads) {
            const int t = i / rank, r = i - t * rank;
            // (t is no lane's own token here)
            if (t0 + t < a.n_tokens && a.ids[t0 + t] == ad) {
                float y[kLoShrinkWaves];
#pragma unroll
                for (int w = 0; w < kLoShrinkWaves; w++) y[w] = red[w][t][r];
#pragma unroll
                for (int n = kLoShrinkWaves / 2; n > 0; n /= 2)
#pragma unroll
                    for (int w = 0; w < n; w++) y[w] += y[w + n];
                a.ws[((size_t)kb * a.n_tokens + t0 + t) * a.max_rank + r] = y[0];
            }
        }
    }
}

// out_t[m] = base_t[m] + scale sum_r B_a[m][r] v_t[r].  NS: steps of 32 ranks.  A wave has per_wave outputs.
template <bool BF, int NS>
__global__ void __launch_bounds__(64 * kLoExpandWaves, NS <= 4 ? 4 : 2) lora_expand_kernel(LoraArgs a, int parts, int per_wave) {
    __shared__ __align__(16) float vs[kLoTile][32 * NS + 4];
    __shared__ int ids[kLoTile];
    // tiles of 16 outputs at once, as many as 128 registers hold (ranks to 32: 8 spill, 91 us for 3001 tokens, 4 69, 2 70)
    constexpr int U = NS <= 1 ? 4 : NS == 2 ? 2 : 1;
    const int lane = lane_id(), c = lane & 15, kg = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int t0 = blockIdx.y * kLoTile;
    const int m_from = (blockIdx.x * kLoExpandWaves + wave) * per_wave, m_to = min(a.M, m_from + per_wave);
    uint32_t firsts;
    const int id = lo_ids(a, t0, firsts);
    const size_t row = (size_t)min(t0 + c, a.n_tokens - 1);
    const float *base = a.base + row * a.M;
    float *out = a.out + row * a.M;
    if (wave == 0 && kg == 0) ids[c] = id;
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
        const uint16_t *Bw = B + (size_t)m_from * a.max_rank;  // the wave's rows
        // of the step that the rank ends in: what lies behind it may be no number
        u4 keep;
        {
            const int r = (rank & ~31) + 8 * kg, live = rank - (r < rank ? r : 0);
#pragma unroll
            for (int j = 0; j < 4; j++) keep[j] = live > 2 * j + 1 ? ~0u : live > 2 * j ? 0xffffu : 0u;
        }
        LoOperand<BF> o[NS];
        int e = -127;
        // v: the parts are added by all threads, for all waves
        lds_barrier();
        for (int i = threadIdx.x; i < kLoTile * 8 * NS; i += 64 * kLoExpandWaves) {
            const int t = i / (8 * NS), r = i % (8 * NS) * 4;
            f4 x = {};
            if (ids[t] == ad && r < rank) {
                const float *part = a.ws + ((size_t)t0 + t) * a.max_rank + r;
#pragma unroll 2
                for (int p = 0; p < parts; p++, part += (size_t)a.n_tokens * a.max_rank) {
                    f4 one;
                    __builtin_memcpy(&one, part, 16);
                    x += one;
                }
            }
#pragma unroll
            for (int j = 0; j < 4; j++) x[j] = r + j < rank ? x[j] : 0.0f;
            __builtin_memcpy(&vs[t][r], &x, 16);
        }
        lds_barrier();
        float v[NS][8], largest = 0.0f;
#pragma unroll
        for (int st = 0; st < NS; st++) {
            __builtin_memcpy(v[st], &vs[c][32 * st + 8 * kg], 32);
#pragma unroll
            for (int j = 0; j < 8; j++) largest = fmaxf(largest, fabsf(v[st][j]));
        }
        if (!BF) e = lo_exponent(largest);
#pragma unroll
        for (int st = 0; st < NS; st++) o[st].set(v[st], e);
        for (int m0 = m_from; m0 < m_to; m0 += 16 * U) {
            u4 w[U][NS];
            f4 y[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                // (rows behind the last, and words behind the rank, which meet zeros in v, are others')
                const uint32_t m = min(m0 + 16 * u + c, m_to - 1) - m_from;
#pragma unroll
                for (int st = 0; st < NS; st++) {
                    const int r = 32 * st + 8 * kg;
                    __builtin_memcpy(&w[u][st], Bw + (m * a.max_rank + (r < rank ? r : 0)), 16);
                }
                if (mine && m0 + 16 * u + 4 * kg + 3 < m_to) __builtin_memcpy(&y[u], base + m0 + 16 * u + 4 * kg, 16);
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                f4 z = {};
#pragma unroll
                for (int st = 0; st < NS; st++) {
                    if (32 * st < rank) {
                        if (st == rank / 32) w[u][st] &= keep;
                        z = o[st].mul(w[u][st], z);
                    }
                }
                if (!BF)
#pragma unroll
                    for (int i = 0; i < 4; i++) z[i] = ldexpf(z[i], e - 13);
                const int mo = m0 + 16 * u + 4 * kg;
                if (!mine) continue;
                if (mo + 3 < m_to) {
#pragma unroll
                    for (int i = 0; i < 4; i++) z[i] = fmaf(scale, z[i], y[u][i]);
                    __builtin_memcpy(out + mo, &z, 16);
                } else
#pragma unroll
                    for (int i = 0; i < 3; i++)
                        if (mo + i < m_to) out[mo + i] = fmaf(scale, z[i], base[mo + i]);
            }
        }
    }
}

// Parts of K: as many as there are steps, but no more than it takes to fill the chip, since the second launch reads them all.
// (4096 features, 61 tokens: 24 us in four parts, 27 in two; 3001 tokens 70 either way.)
static int lo_parts(int n_tokens, int K, int *per_part) {
    const int tiles = (n_tokens + kLoTile - 1) / kLoTile, steps = (K + kLoStep - 1) / kLoStep;
    int parts = tiles >= 1024 ? 1 : (1024 + tiles - 1) / tiles;
    if (parts > kLoMaxParts) parts = kLoMaxParts;
    if (parts > steps) parts = steps;
    if (parts < 1) parts = 1;
    const int per = (steps + parts - 1) / parts;
    *per_part = per * kLoStep;
    return (steps + per - 1) / per;
}

// Enough for every call of no more tokens: parts times tokens are at most kLoMaxParts times, and at most 1024 tiles more than,
// the tokens.
size_t lora_workspace_bytes(int n_tokens, int K, int max_rank) {
    const size_t steps = ((size_t)K + kLoStep - 1) / kLoStep, n = n_tokens;
    const size_t most = (steps < kLoMaxParts ? steps : kLoMaxParts) * n, rows = n + (1024 + 1) * kLoTile;
    return (most < rows ? most : rows) * max_rank * sizeof(float);
}

template <bool BF>
static int launch_typed(const LoraArgs &a, hipStream_t s) {
    int per_part;
    const int parts = lo_parts(a.n_tokens, a.K, &per_part), tiles = (a.n_tokens + kLoTile - 1) / kLoTile;
    // Outputs of a wave: one token takes 8.9 us by 64, 9.9 by 128, 11.4 by 256; 3001 tokens of ranks to 32 73, 69 and 75, of
    // 200 of 256 192 by 256 and 221 by 64: a wave forms its operands of v once.
    const int per_wave = tiles < 64 ? 64 : a.max_rank <= 64 ? 128 : 256, m_blocks = (a.M + kLoExpandWaves * per_wave - 1) / (kLoExpandWaves * per_wave);
    // a tile's adapters by workgroups of their own, as far as the chip has room for them: 1024 workgroups of either launch are at
    // work at once (61 tokens of 40 adapters take 24 us with room for 1024 of the second, 26 for 2048, 26 for 768)
    auto apart = [&](long long groups, long long room) {
        long long z = room / groups;
        z = z < kLoTile ? z : kLoTile;
        z = z < a.n_tokens ? z : a.n_tokens;
        z = z < a.n_adapters + 1 ? z : a.n_adapters + 1;
        return (int)(z > 1 ? z : 1);
    };
    const dim3 block(64 * kLoShrinkWaves), block2(64 * kLoExpandWaves);
    const dim3 g1(parts, tiles, apart((long long)parts * tiles, 1024));
    const int ranks = (a.max_rank + 15) / 16;
#define MNEMO_SHRINK(N) hipLaunchKernelGGL((lora_shrink_kernel<BF, N>), g1, block, 0, s, a, per_part)
    if (ranks <= 1) MNEMO_SHRINK(1);
    else if (ranks <= 2) MNEMO_SHRINK(2);
    else if (ranks <= 4) MNEMO_SHRINK(4);
    else if (ranks <= 8) MNEMO_SHRINK(8);
    else MNEMO_SHRINK(16);
#undef MNEMO_SHRINK
    if (int rc = check_launch("lora_add")) return rc;
    const dim3 g2(m_blocks, tiles, apart((long long)m_blocks * tiles, 1024));
#define MNEMO_EXPAND(N) hipLaunchKernelGGL((lora_expand_kernel<BF, N>), g2, block2, 0, s, a, parts, per_wave)
    if (ranks <= 2) MNEMO_EXPAND(1);
    else if (ranks <= 4) MNEMO_EXPAND(2);
    else if (ranks <= 8) MNEMO_EXPAND(4);
    else MNEMO_EXPAND(8);
#undef MNEMO_EXPAND
    return check_launch("lora_add");
}

int launch_lora(const LoraArgs &a, hipStream_t s) { return a.bf16 ? launch_typed<true>(a, s) : launch_typed<false>(a, s); }

}  // namespace mnemo
