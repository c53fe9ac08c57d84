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

// Planning is one workgroup's work: a few loads of whole numbers, whose round trips are its time.  The
// references of the first kScanPages pages are loaded with the rows and held as a bit per page.
constexpr int kPlanThreads = 1024;
constexpr int kPlanRows = kMaxSeqs / kPlanThreads;  // rows per thread
constexpr int kScanPer = 16;                        // pages per thread and step of a scan over the references
constexpr int kScanPages = kPlanThreads * kScanPer;

// Sum of v over the lower threads of the workgroup; total: over all.
__device__ __forceinline__ int block_scan(int v, int *waves, int &total) {
    const int wave = threadIdx.x >> 6, x = wave_scan(v);
    __syncthreads();  // the last scan's sums are read
    if (lane_id() == 63) waves[wave] = x;
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

// The thread's pages of the scan step at p0: a bit for each that is in use (pages past the end count
// as in use).
__device__ __forceinline__ unsigned used_pages(const int *refs, int n_pages, int p0) {
    const int p = p0 + (int)threadIdx.x * kScanPer;
    unsigned used = (1u << kScanPer) - 1;
    if (p + kScanPer <= n_pages) {
        int v[kScanPer];
        __builtin_memcpy(v, refs + p, sizeof v);
        used = 0;
#pragma unroll
        for (int i = 0; i < kScanPer; i++) used |= v[i] > 0 ? 1u << i : 0;
    } else {
        for (int i = 0; i < kScanPer && p + i < n_pages; i++)
            if (refs[p + i] <= 0) used &= ~(1u << i);
    }
    return used;
}

// The free pages: their number is known after count(), give() hands out the lowest.
struct FreePages {
    const int *refs;
    int n_pages;
    unsigned used;       // the thread's pages of the first step
    int before, total0;  // free pages of lower threads, and of all, in the first step
    int n;               // free pages
    __device__ __forceinline__ void load(const int *r, int pages) {
        refs = r;
        n_pages = pages;
        used = used_pages(r, pages, 0);
    }
    __device__ __forceinline__ void count(int *waves) {
        before = block_scan(kScanPer - __popc(used), waves, total0);
        n = total0;
        if (n_pages > kScanPages) {
            int more = 0, total;
            for (int p0 = kScanPages; p0 < n_pages; p0 += kScanPages) more += kScanPer - __popc(used_pages(refs, n_pages, p0));
            block_scan(more, waves, total);
            n += total;
        }
    }
    // calls give(page, rank) for the free pages in rising order, ranks 0 .. limit - 1; the ranks of a step are
    // dealt out to the threads through list, as free pages tend to lie side by side
    template <class F>
    __device__ __forceinline__ void give(int limit, int *waves, uint16_t *list, F give) const {
        unsigned u = used;
        int rank = before, total = total0, base = 0;
        for (int p0 = 0;;) {
            for (unsigned f = ~u & ((1u << kScanPer) - 1); f; f &= f - 1)
                list[rank++] = (uint16_t)(threadIdx.x * kScanPer + __ffs((int)f) - 1);
            __syncthreads();
            const int n_here = min(total, limit - base);
            for (int k = threadIdx.x; k < n_here; k += kPlanThreads) give(p0 + list[k], base + k);
            base += total;
            p0 += kScanPages;
            if (p0 >= n_pages || base >= limit) break;
            u = used_pages(refs, n_pages, p0);
            rank = block_scan(kScanPer - __popc(u), waves, total);  // (its barriers: list is read)
        }
    }
};

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
    __shared__ uint16_t list[kScanPages];
    __shared__ int waves[kPlanThreads / 64], n_refused;
    const int per = (a.n_seqs + kPlanThreads - 1) / kPlanThreads, r0 = (int)threadIdx.x * per;
    int need[kPlanRows], want[kPlanRows], sum = 0, total, refused = 0;
    FreePages fp;
    fp.load(a.refs, a.n_pages);
    if (threadIdx.x == 0) n_refused = 0;
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
    fp.n = 0;
    if (total > 0) fp.count(waves);
#pragma unroll
    for (int i = 0; i < kPlanRows; i++) {
        const int r = r0 + i;
        if (i < per && r < a.n_seqs) {
            start[r] = at;
            at += need[i];
            if (want[i] > 0) {
                if (at <= fp.n) a.lens[r] = want[i];
                else {
                    refused++;
                    have[r] = INT_MAX;  // not served
                }
            }
        }
    }
    if (refused) atomicAdd(&n_refused, refused);
    __syncthreads();  // start, have and the count are whole
    if (threadIdx.x == 0 && status) *status = n_refused;
    if (total > 0) fp.give(min(total, fp.n), waves, list, [&](int page, int rank) {
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
    const int r = blockIdx.x, len = a.lens[r];
    if (!gone[r]) return;
    const int held = min(pages_of(len, a.ps), a.max_pages);
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
// Bound by memory.  A page of a layer is one row of 16-byte words, [K | V | K scales | V scales], cut into
// equal pieces of at most 16 KB; a workgroup copies a piece at a time, four words per thread in
// flight.  blockIdx.y is the layer; the workgroups of a layer take the (copy, piece) pairs in turn.
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
constexpr int kPiece = 1024;  // words of a piece, at most
// Workgroups of a launch that does not know how many copies there are.  Idle ones cost: 1 MB moves in 3.3 us with
// 4096, 3.8 with 8192 and 5.5 with 16384; a pool compacted twice (793 MB) takes 166, 159 and 157.
constexpr int kForkGrid = 4096, kCompactGrid = 8192;

struct CopyPlan {
    u4 *arr[4];       // K, V, K scales, V scales
    size_t page[2];   // words of a page of K or V, and of scales
    size_t layer[2];  // words of a layer
    size_t words;     // of a page with all its arrays
    int piece, pieces;
    int n_pages;
};

static CopyPlan copy_plan(const PagedCache &c) {
    CopyPlan p = {};
    const size_t rows = (size_t)c.nkv * c.ps;
    const bool int8 = c.kv_type == kKvInt8;
    p.arr[0] = (u4 *)c.k;
    p.arr[1] = (u4 *)c.v;
    p.arr[2] = (u4 *)c.ksc;
    p.arr[3] = (u4 *)c.vsc;
    p.page[0] = rows * c.hd * (int8 ? 1 : 2) / 16;
    p.page[1] = int8 ? rows * 4 / 16 : 0;
    for (int i = 0; i < 2; i++) p.layer[i] = p.page[i] * c.n_pages;
    p.words = 2 * (p.page[0] + p.page[1]);
    p.pieces = (int)((p.words + kPiece - 1) / kPiece);
    p.piece = (int)(((p.words + p.pieces - 1) / p.pieces + 63) / 64 * 64);
    p.n_pages = c.n_pages;
    return p;
}

static dim3 copy_grid(int n_layers, int groups) { return dim3(groups / n_layers > 0 ? groups / n_layers : 1, n_layers); }

// Copies the n pages src[i] -> dst[i] of layer blockIdx.y; its workgroups share them.
__device__ __forceinline__ void copy_pages(const CopyPlan &p, const int *src, const int *dst, int n) {
    const int X = gridDim.x, dm = X / p.pieces, dp = X % p.pieces;
    const size_t kv = p.page[0], sc = p.page[1];
    int m = blockIdx.x / p.pieces, piece = blockIdx.x % p.pieces;
    while (m < n) {
        const int a = src[m], b = dst[m];
        if ((unsigned)a < (unsigned)p.n_pages && (unsigned)b < (unsigned)p.n_pages && a != b) {
            const size_t w0 = (size_t)piece * p.piece;
            // word w of page x is at[array of w] + w
            u4 *at[4];
            at[0] = p.arr[0] + blockIdx.y * p.layer[0];
            at[1] = p.arr[1] + blockIdx.y * p.layer[0] - kv;
            at[2] = p.arr[2] + blockIdx.y * p.layer[1] - 2 * kv;
            at[3] = p.arr[3] + blockIdx.y * p.layer[1] - (2 * kv + sc);
            u4 v[4], *to[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const size_t w = w0 + 256 * i + threadIdx.x;
                const bool s = w >= 2 * kv;
                u4 *base = s ? (w >= 2 * kv + sc ? at[3] : at[2]) : w >= kv ? at[1] : at[0];
                const size_t page = s ? sc : kv;
                to[i] = base + b * page + w;
                if (256 * i + (int)threadIdx.x < p.piece && w < p.words) v[i] = base[a * page + w];
            }
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (256 * i + (int)threadIdx.x < p.piece && w0 + 256 * i + threadIdx.x < p.words)
                    __builtin_nontemporal_store(v[i], to[i]);  // not read again soon: a pool compacted twice takes 165 us, not 186
        }
        m += dm;
        piece += dp;
        if (piece >= p.pieces) {
            piece -= p.pieces;
            m++;
        }
    }
}

__global__ void __launch_bounds__(256) kv_copy_kernel(CopyPlan p, const int *__restrict__ src,
                                                      const int *__restrict__ dst, int n) {
    copy_pages(p, src, dst, n);
}

int launch_kv_copy(const PagedCache &c, int n_layers, const int *src, const int *dst, int n, hipStream_t s) {
    if (n == 0) return kOk;
    const CopyPlan p = copy_plan(c);
    const long long all = (long long)n * p.pieces * n_layers;
    hipLaunchKernelGGL(kv_copy_kernel, copy_grid(n_layers, (int)(all < kCompactGrid ? all : kCompactGrid)), dim3(256), 0, s, p,
                       src, dst, n);
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
    __shared__ int copy_of[kMaxSeqs], last_page[kMaxSeqs];  // of each copy: its row, its source
    __shared__ uint16_t list[kScanPages];
    __shared__ int waves[kPlanThreads / 64], n_refused;
    int *parent = ws + 4, *tail = parent + a.n_seqs, *src = tail + a.n_seqs, *dst = src + a.n_seqs;
    const int per = (a.n_seqs + kPlanThreads - 1) / kPlanThreads, r0 = (int)threadIdx.x * per;
    int need[kPlanRows], from[kPlanRows], len[kPlanRows], page[kPlanRows], sum = 0, total, refused = 0;
    FreePages fp;
    fp.load(a.refs, a.n_pages);
    if (threadIdx.x == 0) n_refused = 0;
#pragma unroll
    for (int i = 0; i < kPlanRows; i++) {
        const int r = r0 + i;
        need[i] = len[i] = 0;
        from[i] = page[i] = -1;
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
                    if (need[i]) page[i] = a.table[(size_t)p * a.max_pages + pl / a.ps];
                }
            }
        }
    }
    int at = block_scan(sum, waves, total);  // its barriers come between all reads of lens and the writes
    fp.n = 0;
    if (total > 0) fp.count(waves);
#pragma unroll
    for (int i = 0; i < kPlanRows; i++) {
        const int r = r0 + i;
        if (i < per && r < a.n_seqs) {
            if (need[i]) {
                copy_of[at] = r;
                last_page[at] = page[i];
            }
            at += need[i];
            const bool served = from[i] >= 0 && at <= fp.n;
            if (from[i] >= 0 && !served) refused++;
            parent[r] = served ? from[i] : -1;
            tail[r] = -1;
            if (served) a.lens[r] = len[i];
        }
    }
    if (refused) atomicAdd(&n_refused, refused);
    __syncthreads();  // the copies and the count are whole
    if (threadIdx.x == 0) {
        ws[0] = min(total, fp.n);
        if (status) *status = n_refused;
    }
    // a free page for each copy: rank k of the free pages is the k-th copy's
    if (total > 0) fp.give(min(total, fp.n), waves, list, [&](int page, int rank) {
        tail[copy_of[rank]] = page;
        src[rank] = last_page[rank];
        dst[rank] = page;
        a.refs[page] = 1;
    });
}

__global__ void __launch_bounds__(256) kv_fork_kernel(KvPagesArgs a, CopyPlan c, const int *__restrict__ ws) {
    const int *parent = ws + 4, *tail = parent + a.n_seqs, *src = tail + a.n_seqs, *dst = src + a.n_seqs;
    for (int r = blockIdx.y * gridDim.x + blockIdx.x; r < a.n_seqs; r += gridDim.x * gridDim.y) {
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
    hipLaunchKernelGGL(kv_fork_kernel, copy_grid(n_layers, kForkGrid), dim3(256), 0, s, a, copy_plan(c), ws);
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
    FreePages fp;
    fp.load(a.refs, a.n_pages);
    fp.count(waves);
    const int live = a.n_pages - fp.n;
    int holes = 0, movers = 0;
    unsigned used = fp.used;
    for (int p0 = 0; p0 < a.n_pages; p0 += kScanPages) {
        if (p0 > 0) used = used_pages(a.refs, a.n_pages, p0);
        const int p = p0 + (int)threadIdx.x * kScanPer;
        // holes below live, movers at it and above (pages past the end are neither)
        const unsigned below = p >= live ? 0u : live - p >= kScanPer ? ~0u : (1u << (live - p)) - 1;
        const unsigned there = p >= a.n_pages ? 0u : a.n_pages - p >= kScanPer ? (1u << kScanPer) - 1 : (1u << (a.n_pages - p)) - 1;
        unsigned h = ~used & below & there, m = used & ~below & there;
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
    const size_t n = (size_t)a.n_seqs * a.max_pages, blocks = (size_t)gridDim.x * gridDim.y;
    for (size_t i = ((size_t)blockIdx.y * gridDim.x + blockIdx.x) * 256 + threadIdx.x; i < n; i += blocks * 256) {
        const int page = a.table[i];
        if (page >= live && page < a.n_pages) a.table[i] = to[page];
    }
    copy_pages(c, src, dst, moves);
}

int launch_kv_compact(const KvPagesArgs &a, const PagedCache &c, int n_layers, int *n_live, int *ws, hipStream_t s) {
    hipLaunchKernelGGL(kv_compact_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, a, n_live, ws);
    hipLaunchKernelGGL(kv_compact_kernel, copy_grid(n_layers, kCompactGrid), dim3(256), 0, s, a, copy_plan(c), ws);
    return check_launch("kv_pages_compact");
}

}  // namespace mnemo
