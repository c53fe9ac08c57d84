// logits.hip -- what is done to a batch of logits before sampling: penalties for tokens already
// said, biases, a grammar's mask.
//
// For row r and token t, with c the times t occurs in the row's history after its prompt and
// seen whether it occurs in the history at all:
//   z = seen ? (z > 0 ? z / rep[r] : z * rep[r]) : z
//   z = z - c freq[r] - (c > 0) pres[r] + bias[t],   -inf where the mask has no bit for t.
// A workgroup owns a slice of a row's tokens and counts the row's whole history into the slice's
// counters in LDS: one pass over the logits and no counters in memory.  The logits are loaded before
// the history is read.  Biases are few: they are added to what the slice has stored, once per token.
//
// Bound by memory where rows are many: 61 rows of 151,936 tokens (76 MB, histories to 8000) 19.2 us, 4.0 TB/s; the
// rest is the counting, whose loads of the history come from L2 once per slice.  One row: 3.6 us, a launch.
#include <math.h>

#include "mnemo_common.hpp"
#include "mnemo_internal.hpp"

namespace mnemo {

constexpr int kLogitsThreads = 256;

typedef float lf4 __attribute__((ext_vector_type(4)));
typedef unsigned lu4 __attribute__((ext_vector_type(4)));
typedef int li4 __attribute__((ext_vector_type(4)));

// GROUPS: groups of four tokens per thread; the slice is 1024 GROUPS tokens.
template <int GROUPS>
__global__ void __launch_bounds__(kLogitsThreads) logits_kernel(LogitsArgs a) {
    constexpr int SLICE = 4 * kLogitsThreads * GROUPS;
    __shared__ __align__(16) unsigned cnt[SLICE];  // bit 31: in the prompt; below: times in the rest
    const int r = blockIdx.y, base = (int)blockIdx.x * SLICE, tid = threadIdx.x;
    const int n = min(SLICE, a.vocab - base);
    const float *z = a.z + (size_t)r * a.vocab + base;
    float *out = a.out + (size_t)r * a.vocab + base;
    const uint32_t *allowed = a.allowed ? a.allowed + (size_t)r * (((size_t)a.vocab + 31) / 32) + base / 32 : nullptr;

    lf4 x[GROUPS];
    uint32_t bits[GROUPS];
#pragma unroll
    for (int g = 0; g < GROUPS; g++) {
        const int i = 4 * (kLogitsThreads * g + tid);
        x[g] = lf4{0.f, 0.f, 0.f, 0.f};
        bits[g] = ~0u;
        if (i + 3 < n) __builtin_memcpy(&x[g], z + i, 16);
        else
            for (int j = 0; j < 4; j++)
                if (i + j < n) x[g][j] = z[i + j];
        if (allowed && i < n) bits[g] = allowed[i / 32] >> (i % 32);
    }
    if (a.hist) {
        const lu4 zero = {0, 0, 0, 0};
#pragma unroll
        for (int g = 0; g < GROUPS; g++) *(lu4 *)&cnt[4 * (kLogitsThreads * g + tid)] = zero;
        const int len = min(max(a.hist_len[r], 0), a.max_hist), prompt = a.prompt_len[r];
        const float rep = a.rep[r], freq = a.freq[r], pres = a.pres[r];
        const int *h = a.hist + (size_t)r * a.max_hist;
        lds_barrier();  // (the logits stay in flight)
        auto count = [&](int id, int i) {
            const unsigned t = (unsigned)id - (unsigned)base;
            if (t < (unsigned)n && id >= 0) {
                if (i < prompt) atomicOr(&cnt[t], 0x80000000u);
                else atomicAdd(&cnt[t], 1u);
            }
        };
        constexpr int PER = 4;  // loads of four tokens in flight
        int at = 0;
        for (; at + 4 * PER * kLogitsThreads <= len; at += 4 * PER * kLogitsThreads) {
            li4 v[PER];
#pragma unroll
            for (int u = 0; u < PER; u++) __builtin_memcpy(&v[u], h + at + 4 * (kLogitsThreads * u + tid), 16);
#pragma unroll
            for (int u = 0; u < PER; u++)
#pragma unroll
                for (int j = 0; j < 4; j++) count(v[u][j], at + 4 * (kLogitsThreads * u + tid) + j);
        }
        for (int i0 = at; i0 < len; i0 += PER * kLogitsThreads) {
            int v[PER];
#pragma unroll
            for (int u = 0; u < PER; u++) v[u] = h[min(i0 + kLogitsThreads * u + tid, len - 1)];
#pragma unroll
            for (int u = 0; u < PER; u++)
                if (i0 + kLogitsThreads * u + tid < len) count(v[u], i0 + kLogitsThreads * u + tid);
        }
        lds_barrier();
#pragma unroll
        for (int g = 0; g < GROUPS; g++) {
            const lu4 c = *(const lu4 *)&cnt[4 * (kLogitsThreads * g + tid)];
            if (!(c.x | c.y | c.z | c.w)) continue;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (!c[j]) continue;
                float y = x[g][j];
                y = y > 0.0f ? y / rep : y * rep;
                const unsigned times = c[j] & 0x7fffffffu;
                if (times) y = y - (float)times * freq - pres;
                x[g][j] = y;
            }
        }
    }
#pragma unroll
    for (int g = 0; g < GROUPS; g++) {
        const int i = 4 * (kLogitsThreads * g + tid);
#pragma unroll
        for (int j = 0; j < 4; j++) x[g][j] = bits[g] >> j & 1 ? x[g][j] : -INFINITY;
        if (i + 3 < n) __builtin_memcpy(out + i, &x[g], 16);
        else
            for (int j = 0; j < 4; j++)
                if (i + j < n) out[i + j] = x[g][j];
    }
    if (!a.bias_ids) return;
    // the counters, free again, find the last entry of each token
    const int *ids = a.bias_ids + (size_t)r * a.n_bias;
    auto in_slice = [&](int i, unsigned &t) {
        const int id = ids[i];
        t = (unsigned)id - (unsigned)base;
        return id >= 0 && t < (unsigned)n;
    };
    unsigned t;
    __syncthreads();  // the slice is stored, its counters are read
    for (int i = tid; i < a.n_bias; i += kLogitsThreads)
        if (in_slice(i, t)) cnt[t] = 0;
    __syncthreads();
    for (int i = tid; i < a.n_bias; i += kLogitsThreads)
        if (in_slice(i, t)) atomicMax(&cnt[t], (unsigned)i + 1);
    __syncthreads();
    for (int i = tid; i < a.n_bias; i += kLogitsThreads)
        if (in_slice(i, t) && cnt[t] == (unsigned)i + 1 && (!allowed || (allowed[t / 32] >> (t % 32) & 1)))
            out[t] += a.bias[(size_t)r * a.n_bias + i];
}

int launch_logits_process(const LogitsArgs &a, hipStream_t s) {
    // Small slices spread a call over the CUs, large ones read the history less often.  14 rows of 151,936 (histories to
    // 2000): 1024 tokens 7.2 us, 2048 6.8, 4096 8.2; 64 rows (16,000): 32.2, 25.6, 23.1; 8 rows: 3.6 all three.
    const long long tokens = (long long)a.n_rows * a.vocab;
    const dim3 block(kLogitsThreads);
    if (tokens < 1 << 21) hipLaunchKernelGGL(logits_kernel<1>, dim3((a.vocab + 1023) / 1024, a.n_rows), block, 0, s, a);
    else if (tokens < 1 << 22) hipLaunchKernelGGL(logits_kernel<2>, dim3((a.vocab + 2047) / 2048, a.n_rows), block, 0, s, a);
    else hipLaunchKernelGGL(logits_kernel<4>, dim3((a.vocab + 4095) / 4096, a.n_rows), block, 0, s, a);
    return check_launch("logits_process");
}

}  // namespace mnemo
