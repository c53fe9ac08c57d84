// logits.hip -- what is done to a batch of logits before sampling: penalties for tokens already
// said, biases, a grammar's mask.
//
// For row r and token t, with c the times t occurs in the row's history after its prompt and
// seen whether it occurs in the history at all:
//   z = seen ? (z > 0 ? z / rep[r] : z * rep[r]) : z
//   z = z - c freq[r] - (c > 0) pres[r] + bias[t],   -inf where the mask has no bit for t.
// A workgroup owns a slice of a row's tokens and counts the row's whole history into the slice's
// counters in LDS: one pass over the logits and no counters in memory.
#include <math.h>

#include "mnemo_common.hpp"
#include "mnemo_internal.hpp"

namespace mnemo {

constexpr int kLogitsThreads = 256;
constexpr int kSlice = 4096;

__global__ void __launch_bounds__(kLogitsThreads) logits_kernel(LogitsArgs a) {
    __shared__ unsigned cnt[kSlice];   // bit 31: in the prompt; below: times in the rest
    __shared__ unsigned slot[kSlice];  // 1 + the last bias entry of the token
    const int r = blockIdx.y, base = (int)blockIdx.x * kSlice, tid = threadIdx.x;
    const int n = min(kSlice, a.vocab - base);
    for (int i = tid; i < kSlice; i += kLogitsThreads) cnt[i] = slot[i] = 0;
    __syncthreads();
    if (a.hist) {
        const int len = min(max(a.hist_len[r], 0), a.max_hist), prompt = a.prompt_len[r];
        const int *h = a.hist + (size_t)r * a.max_hist;
        for (int i = tid; i < len; i += kLogitsThreads) {
            const unsigned t = (unsigned)h[i] - (unsigned)base;
            if (h[i] >= 0 && t < (unsigned)n) {
                if (i < prompt) atomicOr(&cnt[t], 0x80000000u);
                else atomicAdd(&cnt[t], 1u);
            }
        }
    }
    if (a.bias_ids) {
        for (int i = tid; i < a.n_bias; i += kLogitsThreads) {
            const int id = a.bias_ids[(size_t)r * a.n_bias + i];
            const unsigned t = (unsigned)id - (unsigned)base;
            if (id >= 0 && t < (unsigned)n) atomicMax(&slot[t], (unsigned)i + 1);
        }
    }
    __syncthreads();
    const float rep = a.hist ? a.rep[r] : 1.0f, freq = a.hist ? a.freq[r] : 0.0f, pres = a.hist ? a.pres[r] : 0.0f;
    for (int i = tid; i < n; i += kLogitsThreads) {
        const int t = base + i;
        float z = a.z[(size_t)r * a.vocab + t];
        if (cnt[i]) {
            z = z > 0.0f ? z / rep : z * rep;
            const unsigned c = cnt[i] & 0x7fffffffu;
            if (c) z = z - (float)c * freq - pres;
        }
        if (slot[i]) z += a.bias[(size_t)r * a.n_bias + slot[i] - 1];
        if (a.allowed && !((a.allowed[(size_t)r * ((a.vocab + 31) / 32) + t / 32] >> (t % 32)) & 1)) z = -INFINITY;
        a.out[(size_t)r * a.vocab + t] = z;
    }
}

int launch_logits_process(const LogitsArgs &a, hipStream_t s) {
    hipLaunchKernelGGL(logits_kernel, dim3((a.vocab + kSlice - 1) / kSlice, a.n_rows), dim3(kLogitsThreads), 0, s, a);
    return check_launch("logits_process");
}

}  // namespace mnemo
