// kv_pages.hip -- upkeep of a paged cache: pages are given to growing sequences, shared by forks,
// dropped, moved together and copied.
//
// The state is three arrays and nothing else: the block table [n_seqs][max_pages], the lengths
// [n_seqs] and the page references [n_pages] (how many rows hold the page).  Row s holds its first
// ceil(len / ps) entries.  A page is free when nothing refers to it; there is no free list to fall
// out of step.  Pages are always given out lowest first, in row order, so every result is a
// function of the state alone (the atomics below only add whole numbers).
#include <limits.h>

#include "mnemo_common.hpp"
#include "mnemo_internal.hpp"

namespace mnemo {

constexpr int kPlanThreads = 1024;
constexpr int kPlanRows = kMaxSeqs / kPlanThreads;  // rows per thread
constexpr int kScanPer = 8;                         // pages per thread and step of a scan over the references

// Sum of v over the lower threads of the workgroup; total: over all.
__device__ __forceinline__ int block_scan(int v, int *waves, int &total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int x = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();  // the last scan's sums are read
    if (lane == 63) waves[wave] = x;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kPlanThreads / 64; w++) {
        const int n = waves[w];
        before += w < wave ? n : 0;
        total += n;
    }
    return before + x - v;
}

__device__ __forceinline__ int pages_of(int len, int ps) { return len > 0 ? (int)(((unsigned)len + ps - 1) / ps) : 0; }

// How many of the pages are free (the whole workgroup counts).
__device__ __forceinline__ int count_free(const int *refs, int n_pages, int *waves) {
    int n = 0, total;
    for (int i = threadIdx.x; i < n_pages; i += kPlanThreads) n += refs[i] <= 0;
    block_scan(n, waves, total);
    return total;
}

// Calls give(page, rank) for the free pages in rising order, ranks 0 .. limit - 1.
template <class F>
__device__ __forceinline__ void for_free(const int *refs, int n_pages, int limit, int *waves, F give) {
    int base = 0;
    for (int p0 = 0; p0 < n_pages && base < limit; p0 += kPlanThreads * kScanPer) {
        const int p = p0 + (int)threadIdx.x * kScanPer;
        unsigned free = 0;
#pragma unroll
        for (int i = 0; i < kScanPer; i++)
            if (p + i < n_pages && refs[p + i] <= 0) free |= 1u << i;
        int total, rank = base + block_scan(__popc(free), waves, total);
        for (; free && rank < limit; rank++) {
            const int i = __ffs((int)free) - 1;
            free &= free - 1;
            give(p + i, rank);
        }
        base += total;
    }
}

// The row whose share [start[i], start[i + 1]) of the ranks holds rank.
__device__ __forceinline__ int row_of(const int *start, int n, int rank) {
    int lo = 0, hi = n - 1;  // the last row with start <= rank
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (start[mid] <= rank) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// ------------------------------------------------------------------ extend
__global__ void __launch_bounds__(kPlanThreads) kv_extend_kernel(KvPagesArgs a, const int *__restrict__ new_lens,
                                                                 int *status) {
    __shared__ int start[kMaxSeqs], have[kMaxSeqs];
    __shared__ int waves[kPlanThreads / 64];
    const int per = (a.n_seqs + kPlanThreads - 1) / kPlanThreads, r0 = (int)threadIdx.x * per;
    int need[kPlanRows], want[kPlanRows], sum = 0, total, refused = 0;
#pragma unroll
    for (int i = 0; i < kPlanRows; i++) {
        const int r = r0 + i;
        need[i] = want[i] = 0;
        if (i < per && r < a.n_seqs) {
            const int len = max(a.lens[r], 0), to = new_lens[r];
            have[r] = pages_of(len, a.ps);
            if (to > len) {
                const int pages = pages_of(to, a.ps);
                if (pages > a.max_pages) refused++;
                else {
                    want[i] = to;
                    need[i] = pages - have[r];
                    sum += need[i];
                }
            }
        }
    }
    int at = block_scan(sum, waves, total);
    const int n_free = total > 0 ? count_free(a.refs, a.n_pages, waves) : 0;
#pragma unroll
    for (int i = 0; i < kPlanRows; i++) {
        const int r = r0 + i;
        if (i < per && r < a.n_seqs) {
            start[r] = at;
            at += need[i];
            if (want[i] > 0) {
                if (at <= n_free) a.lens[r] = want[i];
                else {
                    refused++;
                    have[r] = INT_MAX;  // not served
                }
            }
        }
    }
    block_scan(refused, waves, sum);  // its barriers publish start and have, too
    if (threadIdx.x == 0 && status) *status = sum;
    for_free(a.refs, a.n_pages, min(total, n_free), waves, [&](int page, int rank) {
        const int r = row_of(start, a.n_seqs, rank);
        if (have[r] == INT_MAX) return;
        a.table[(size_t)r * a.max_pages + have[r] + (rank - start[r])] = page;
        a.refs[page] = 1;
    });
}

int launch_kv_extend(const KvPagesArgs &a, const int *new_lens, int *status, hipStream_t s) {
    hipLaunchKernelGGL(kv_extend_kernel, dim3(1), dim3(kPlanThreads), 0, s, a, new_lens, status);
    return check_launch("kv_pages_extend");
}

// ------------------------------------------------------------------ free
__global__ void __launch_bounds__(256) kv_free_kernel(KvPagesArgs a, const int *__restrict__ gone) {
    const int r = blockIdx.x;
    if (!gone[r]) return;
    const int held = min(pages_of(a.lens[r], a.ps), a.max_pages);
    int *row = a.table + (size_t)r * a.max_pages;
    for (int j = threadIdx.x; j < a.max_pages; j += 256) {
        const int page = row[j];
        if (j < held && (unsigned)page < (unsigned)a.n_pages) atomicSub(&a.refs[page], 1);
        row[j] = -1;
    }
    __syncthreads();
    if (threadIdx.x == 0) a.lens[r] = 0;
}

int launch_kv_free(const KvPagesArgs &a, const int *gone, hipStream_t s) {
    hipLaunchKernelGGL(kv_free_kernel, dim3(a.n_seqs), dim3(256), 0, s, a, gone);
    return check_launch("kv_pages_free");
}

// ------------------------------------------------------------------ copies of pages
struct CopyPlan {
    uint4 *arr[4];      // K, V, K scales, V scales
    size_t page[4];     // 16-byte words of a page
    size_t layer[4];    // words of a layer
    int n_arr, n_layers, n_pages;
};

static CopyPlan copy_plan(const PagedCache &c, int n_layers) {
    CopyPlan p = {};
    const size_t rows = (size_t)c.nkv * c.ps;
    p.n_arr = c.kv_type == kKvInt8 ? 4 : 2;
    p.n_layers = n_layers;
    p.n_pages = c.n_pages;
    void *arr[4] = {c.k, c.v, c.ksc, c.vsc};
    for (int i = 0; i < p.n_arr; i++) {
        p.arr[i] = (uint4 *)arr[i];
        p.page[i] = rows * (i < 2 ? c.hd * (c.kv_type == kKvInt8 ? 1 : 2) : 4) / 16;
        p.layer[i] = p.page[i] * c.n_pages;
    }
    return p;
}

// Copies the n pages src[i] -> dst[i] of every layer and array; the whole grid shares them.
__device__ __forceinline__ void copy_pages(const CopyPlan &p, const int *src, const int *dst, int n) {
    const long long units = (long long)n * p.n_layers;
    for (long long u = blockIdx.x; u < units; u += gridDim.x) {
        const int m = (int)(u / p.n_layers), l = (int)(u % p.n_layers);
        const int a = src[m], b = dst[m];
        if ((unsigned)a >= (unsigned)p.n_pages || (unsigned)b >= (unsigned)p.n_pages || a == b) continue;
        for (int i = 0; i < p.n_arr; i++) {
            const uint4 *from = p.arr[i] + l * p.layer[i] + a * p.page[i];
            uint4 *to = p.arr[i] + l * p.layer[i] + b * p.page[i];
            for (size_t w = threadIdx.x; w < p.page[i]; w += 256) to[w] = from[w];
        }
    }
}

constexpr int kCopyGrid = 2048;

__global__ void __launch_bounds__(256) kv_copy_kernel(CopyPlan p, const int *__restrict__ src,
                                                      const int *__restrict__ dst, int n) {
    copy_pages(p, src, dst, n);
}

int launch_kv_copy(const PagedCache &c, int n_layers, const int *src, const int *dst, int n, hipStream_t s) {
    if (n == 0) return kOk;
    hipLaunchKernelGGL(kv_copy_kernel, dim3(kCopyGrid), dim3(256), 0, s, copy_plan(c, n_layers), src, dst, n);
    return check_launch("kv_pages_copy");
}

// ------------------------------------------------------------------ fork
// Workspace: [0] number of copies, then the rows' parents [n_seqs] (-1: not forked) and the pages
// that take the copies, then the copies' sources [n_seqs] and destinations [n_seqs].
size_t kv_pages_workspace_bytes(int n_seqs, int n_pages) {
    const size_t fork = 4 + 4 * (size_t)n_seqs, compact = 4 + 3 * (size_t)n_pages;
    return 4 * (fork > compact ? fork : compact);
}

__global__ void __launch_bounds__(kPlanThreads) kv_fork_plan_kernel(KvPagesArgs a, const int *__restrict__ parents,
                                                                    int *status, int *ws) {
    __shared__ int start[kMaxSeqs];
    __shared__ int waves[kPlanThreads / 64];
    int *parent = ws + 4, *tail = parent + a.n_seqs, *src = tail + a.n_seqs, *dst = src + a.n_seqs;
    const int per = (a.n_seqs + kPlanThreads - 1) / kPlanThreads, r0 = (int)threadIdx.x * per;
    int need[kPlanRows], from[kPlanRows], len[kPlanRows], sum = 0, total, refused = 0;
#pragma unroll
    for (int i = 0; i < kPlanRows; i++) {
        const int r = r0 + i;
        need[i] = len[i] = 0;
        from[i] = -1;
        if (i < per && r < a.n_seqs) {
            const int p = parents[r];
            if (p >= 0) {
                const int pl = p < a.n_seqs && a.lens[r] <= 0 ? a.lens[p] : 0;  // as before the call
                if (pl <= 0 || pages_of(pl, a.ps) > a.max_pages) refused++;
                else {
                    from[i] = p;
                    len[i] = pl;
                    need[i] = pl % a.ps != 0;
                    sum += need[i];
                }
            }
        }
    }
    int at = block_scan(sum, waves, total);  // its barriers come between all reads of lens and the writes
    const int n_free = total > 0 ? count_free(a.refs, a.n_pages, waves) : 0;
#pragma unroll
    for (int i = 0; i < kPlanRows; i++) {
        const int r = r0 + i;
        if (i < per && r < a.n_seqs) {
            start[r] = at;
            at += need[i];
            const bool served = from[i] >= 0 && at <= n_free;
            if (from[i] >= 0 && !served) refused++;
            parent[r] = served ? from[i] : -1;
            tail[r] = -1;
            if (served) a.lens[r] = len[i];
        }
    }
    block_scan(refused, waves, sum);
    if (threadIdx.x == 0) {
        ws[0] = min(total, n_free);
        if (status) *status = sum;
    }
    // a free page for each copy: rank k of the free pages is the k-th copy's
    for_free(a.refs, a.n_pages, min(total, n_free), waves, [&](int page, int rank) {
        const int r = row_of(start, a.n_seqs, rank);
        const int p = parents[r];
        tail[r] = page;
        src[rank] = a.table[(size_t)p * a.max_pages + pages_of(a.lens[p], a.ps) - 1];
        dst[rank] = page;
        a.refs[page] = 1;
    });
}

__global__ void __launch_bounds__(256) kv_fork_kernel(KvPagesArgs a, CopyPlan c, const int *__restrict__ ws) {
    const int *parent = ws + 4, *tail = parent + a.n_seqs, *src = tail + a.n_seqs, *dst = src + a.n_seqs;
    for (int r = blockIdx.x; r < a.n_seqs; r += gridDim.x) {
        const int p = parent[r];
        if (p < 0) continue;
        const int held = pages_of(a.lens[p], a.ps), last = tail[r];
        const int shared = held - (last >= 0);
        const int *from = a.table + (size_t)p * a.max_pages;
        int *to = a.table + (size_t)r * a.max_pages;
        for (int j = threadIdx.x; j < a.max_pages; j += 256) {
            int page = -1;
            if (j < shared) {
                page = from[j];
                if ((unsigned)page < (unsigned)a.n_pages) atomicAdd(&a.refs[page], 1);
            } else if (j < held) page = last;
            to[j] = page;
        }
    }
    copy_pages(c, src, dst, ws[0]);
}

int launch_kv_fork(const KvPagesArgs &a, const PagedCache &c, int n_layers, const int *parents, int *status, int *ws,
                   hipStream_t s) {
    hipLaunchKernelGGL(kv_fork_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, a, parents, status, ws);
    hipLaunchKernelGGL(kv_fork_kernel, dim3(kCopyGrid), dim3(256), 0, s, a, copy_plan(c, n_layers), ws);
    return check_launch("kv_pages_fork");
}

// ------------------------------------------------------------------ compact
// With n pages in use, the k-th of them that lies at n or above moves to the k-th free page below
// n.  Sources and destinations are apart, so all copies can run at once.
// Workspace: [0] number of moves, [1] n, then where pages from n on went [n_pages], the moves'
// sources [n_pages] and destinations [n_pages].
__global__ void __launch_bounds__(kPlanThreads) kv_compact_plan_kernel(KvPagesArgs a, int *n_live, int *ws) {
    __shared__ int waves[kPlanThreads / 64];
    int *to = ws + 4, *src = to + a.n_pages, *dst = src + a.n_pages;
    const int live = a.n_pages - count_free(a.refs, a.n_pages, waves);
    int holes = 0, movers = 0;
    for (int p0 = 0; p0 < a.n_pages; p0 += kPlanThreads * kScanPer) {
        const int p = p0 + (int)threadIdx.x * kScanPer;
        unsigned pick = 0;  // holes below live, movers above it
#pragma unroll
        for (int i = 0; i < kScanPer; i++)
            if (p + i < a.n_pages && (a.refs[p + i] > 0) == (p + i >= live)) pick |= 1u << i;
        const unsigned below = p >= live ? 0u : live - p >= kScanPer ? ~0u : (1u << (live - p)) - 1;
        unsigned h = pick & below, m = pick & ~below;
        int th, tm;
        int rank = holes + block_scan(__popc(h), waves, th);
        for (; h; h &= h - 1) dst[rank++] = p + __ffs((int)h) - 1;
        rank = movers + block_scan(__popc(m), waves, tm);
        for (; m; m &= m - 1) src[rank++] = p + __ffs((int)m) - 1;
        holes += th;
        movers += tm;
    }
    __syncthreads();  // the lists are whole
    for (int p = live + (int)threadIdx.x; p < a.n_pages; p += kPlanThreads) to[p] = p;
    __syncthreads();
    for (int k = threadIdx.x; k < movers; k += kPlanThreads) {
        const int from = src[k], at = dst[k];
        to[from] = at;
        a.refs[at] = a.refs[from];
        a.refs[from] = 0;
    }
    if (threadIdx.x == 0) {
        ws[0] = movers;
        ws[1] = live;
        if (n_live) *n_live = live;
    }
}

__global__ void __launch_bounds__(256) kv_compact_kernel(KvPagesArgs a, CopyPlan c, const int *__restrict__ ws) {
    const int moves = ws[0], live = ws[1];
    if (moves == 0) return;
    const int *to = ws + 4, *src = to + a.n_pages, *dst = src + a.n_pages;
    const size_t n = (size_t)a.n_seqs * a.max_pages;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) {
        const int page = a.table[i];
        if (page >= live && page < a.n_pages) a.table[i] = to[page];
    }
    copy_pages(c, src, dst, moves);
}

int launch_kv_compact(const KvPagesArgs &a, const PagedCache &c, int n_layers, int *n_live, int *ws, hipStream_t s) {
    hipLaunchKernelGGL(kv_compact_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, a, n_live, ws);
    hipLaunchKernelGGL(kv_compact_kernel, dim3(kCopyGrid), dim3(256), 0, s, a, copy_plan(c, n_layers), ws);
    return check_launch("kv_pages_compact");
}

}  // namespace mnemo
