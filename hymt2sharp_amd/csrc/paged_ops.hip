// paged_ops.hip -- upkeep of the multi-sequence cache's pages, and the rows of
// a batch rotated, normed and appended to them (hymt_paged, include/hymt_hip.h).
//
// Upkeep: the plan of a call -- who gets which free page, what is copied, what
// loses a reference -- is made by one workgroup, from the reference counts
// alone (there is no free list that could disagree with them), and a second
// launch over the whole chip moves the bytes.  extend moves none and is the plan
// alone.  A plan first looks at everything it would rely on and only then writes, so a
// call that finds something wrong changes nothing but `work`.
#include <algorithm>

#include "attn_kernels.hpp"
#include "device_common.hpp"
#include "ktimer.hpp"
#include "paged.hpp"

namespace hymt {

namespace {

constexpr int kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64;

// lists in work: free pages handed out or (src, dst) pairs, and compact's map
__device__ __forceinline__ int32_t *work_src(const hymt_paged &p) { return p.work + kWorkLists; }
__device__ __forceinline__ int32_t *work_dst(const hymt_paged &p) { return p.work + kWorkLists + p.pages; }
__device__ __forceinline__ int32_t *work_map(const hymt_paged &p) { return p.work + kWorkLists + 2 * (size_t)p.pages; }

__device__ __forceinline__ int blocks_of(int len) { return (len + kPage - 1) / kPage; }

// Exclusive prefix sum over the workgroup's threads, and the total.
__device__ int block_scan(int v, int *s_wave, int &total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int x = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int y = __shfl_up(x, d);
        if (lane >= d) x += y;
    }
    __syncthreads();  // s_wave's last readers
    if (lane == 63) s_wave[wave] = x;
    __syncthreads();
    int base = 0, sum = 0;
#pragma unroll
    for (int w = 0; w < kPlanWaves; w++) {
        const int t = s_wave[w];
        if (w < wave) base += t;
        sum += t;
    }
    total = sum;
    return base + x - v;
}

// The pages [lo, hi) in ascending order, 1024 at a time: f(page, refs, valid) for
// every thread of the workgroup alike.
template <typename F> __device__ __forceinline__ void for_pages(const hymt_paged &p, int lo, int hi, F f) {
    for (int base = lo; base < hi; base += kPlanThreads) {
        const int i = base + (int)threadIdx.x;
        const bool ok = i < hi;
        f(i, ok ? p.refs[i] : 0, ok);
    }
}

// The `need` lowest free pages into list[0 .. need); false if there are fewer.
__device__ bool find_free(const hymt_paged &p, int need, int32_t *list, int *s_wave) {
    int found = 0;
    for (int base = 0; base < p.pages && found < need; base += kPlanThreads) {
        const int i = base + (int)threadIdx.x;
        const int free = i < p.pages && p.refs[i] <= 0;
        int total;
        const int at = found + block_scan(free, s_wave, total);
        if (free && at < need) list[at] = i;
        found += total;
    }
    __syncthreads();
    return found >= need;
}

// One thread ends a call: its status, and the first that was not good.
__device__ void finish(const hymt_paged &p, int status, int copies) {
    p.work[kWorkStatus] = status;
    p.work[kWorkCopies] = copies;
    if (status != HYMT_OK && p.work[kWorkFirst] == HYMT_OK) p.work[kWorkFirst] = status;
}

// Pages in use (all threads get the number).
__device__ int count_live(const hymt_paged &p, int *s_wave) {
    int mine = 0;
    for (int i = threadIdx.x; i < p.pages; i += kPlanThreads) mine += p.refs[i] > 0;
    int total;
    block_scan(mine, s_wave, total);
    return total;
}

// A slot's place in a bit per slot; true if it was set already.
__device__ __forceinline__ bool mark(uint32_t *bits, int slot) {
    const uint32_t m = 1u << (slot & 31);
    return (atomicOr(&bits[slot >> 5], m) & m) != 0;
}

struct PlanShared {
    uint32_t bits[kPagedMaxSeqs / 32];
    int wave[kPlanWaves];
    int status;
    int slot[HYMT_PAGED_BATCH], first[HYMT_PAGED_BATCH], count[HYMT_PAGED_BATCH], rank[HYMT_PAGED_BATCH];
};

__device__ __forceinline__ void plan_begin(PlanShared &sh, int seqs) {
    for (int i = threadIdx.x; i < (seqs + 31) / 32; i += kPlanThreads) sh.bits[i] = 0;
    if (threadIdx.x == 0) sh.status = HYMT_OK;
    __syncthreads();
}
// statuses by rank, so that which one a call reports does not depend on the
// order of threads: the smallest code wins
__device__ __forceinline__ void plan_fail(PlanShared &sh, int code) {
    int old = atomicCAS(&sh.status, HYMT_OK, code);
    while (old != HYMT_OK && code < old) old = atomicCAS(&sh.status, old, code);
}

__global__ __launch_bounds__(kPlanThreads) void paged_extend_kernel(hymt_paged p, const int32_t *slots,
                                                                    const int32_t *cu, int n) {
    __shared__ PlanShared sh;
    plan_begin(sh, p.seqs);
    const int i = threadIdx.x;
    int slot = -1, len = 0, add = 0, need = 0;
    if (i < n) {
        slot = slots[i];
        add = cu ? cu[i + 1] - cu[i] : 1;
        if ((unsigned)slot >= (unsigned)p.seqs || add < 0 || (cu && i == 0 && cu[0] != 0) || mark(sh.bits, slot)) {
            plan_fail(sh, HYMT_E_ARG);
        } else {
            len = p.len[slot];
            const long cap = (long)p.blocks * kPage;
            if (len < 0 || len > cap) plan_fail(sh, HYMT_E_STATE);
            else if ((long)len + add > cap) plan_fail(sh, HYMT_E_CAPACITY);
            else {
                need = blocks_of(len + add) - blocks_of(len);
                if (add > 0 && len % kPage) {  // the page that is written on is this sequence's alone
                    const int page = p.table[(size_t)slot * p.blocks + len / kPage];
                    if ((unsigned)page >= (unsigned)p.pages || p.refs[page] != 1) plan_fail(sh, HYMT_E_STATE);
                }
            }
        }
    }
    int total;
    const int rank = block_scan(need, sh.wave, total);
    int32_t *list = work_src(p);
    bool enough = true;
    if (total > p.pages) enough = false;
    else if (total > 0) enough = find_free(p, total, list, sh.wave);
    if (!enough && i == 0) plan_fail(sh, HYMT_E_CAPACITY);
    __syncthreads();
    if (sh.status != HYMT_OK) {
        if (i == 0) finish(p, sh.status, 0);
        return;
    }
    if (i < n) {
        sh.slot[i] = slot;
        sh.first[i] = blocks_of(len);
        sh.count[i] = need;
        sh.rank[i] = rank;
        p.len[slot] = len + add;
    }
    __syncthreads();
    if (total > 0)
        for (int e = threadIdx.x >> 6; e < n; e += kPlanWaves)
            for (int j = threadIdx.x & 63; j < sh.count[e]; j += 64) {
                const int page = list[sh.rank[e] + j];
                p.table[(size_t)sh.slot[e] * p.blocks + sh.first[e] + j] = page;
                p.refs[page] = 1;
            }
    __syncthreads();
    if (i == 0) finish(p, HYMT_OK, 0);
}

__global__ __launch_bounds__(kPlanThreads) void paged_fork_plan_kernel(hymt_paged p, const int32_t *parent,
                                                                       const int32_t *child, int n) {
    __shared__ PlanShared sh;
    plan_begin(sh, p.seqs);
    const int i = threadIdx.x;
    int from = 0, to = 0, len = 0, need = 0, src = 0;
    if (i < n) {
        from = parent[i];
        to = child[i];
        if ((unsigned)from >= (unsigned)p.seqs || (unsigned)to >= (unsigned)p.seqs || mark(sh.bits, to))
            plan_fail(sh, HYMT_E_ARG);
    }
    __syncthreads();
    if (i < n && (unsigned)from < (unsigned)p.seqs && (unsigned)to < (unsigned)p.seqs) {
        if (sh.bits[from >> 5] >> (from & 31) & 1) plan_fail(sh, HYMT_E_ARG);
        len = p.len[from];
        if (len < 0 || len > (long)p.blocks * kPage || p.len[to] != 0) {
            plan_fail(sh, HYMT_E_STATE);
            len = 0;
        }
        if (len % kPage) {
            need = 1;
            src = p.table[(size_t)from * p.blocks + len / kPage];
            if ((unsigned)src >= (unsigned)p.pages) plan_fail(sh, HYMT_E_STATE);
        }
        sh.slot[i] = from;
        sh.count[i] = len / kPage;
    }
    int total;
    const int rank = block_scan(need, sh.wave, total);
    int32_t *list = work_dst(p);
    const bool enough = total <= p.pages && (total == 0 || find_free(p, total, list, sh.wave));
    if (!enough && i == 0) plan_fail(sh, HYMT_E_CAPACITY);
    __syncthreads();
    // whole pages have to be in the pool before one of them is counted again
    if (sh.status == HYMT_OK)
        for (int e = threadIdx.x >> 6; e < n; e += kPlanWaves)
            for (int j = threadIdx.x & 63; j < sh.count[e]; j += 64)
                if ((unsigned)p.table[(size_t)sh.slot[e] * p.blocks + j] >= (unsigned)p.pages) plan_fail(sh, HYMT_E_STATE);
    __syncthreads();
    if (sh.status != HYMT_OK) {
        if (i == 0) finish(p, sh.status, 0);
        return;
    }
    if (i < n) {
        p.len[to] = len;
        if (need) {
            const int dst = list[rank];
            work_src(p)[rank] = src;
            p.table[(size_t)to * p.blocks + len / kPage] = dst;
            p.refs[dst] = 1;
        }
    }
    if (i == 0) finish(p, HYMT_OK, total);
}

__global__ __launch_bounds__(kPlanThreads) void paged_set_len_plan_kernel(hymt_paged p, const int32_t *slots,
                                                                          const int32_t *lens, int n) {
    __shared__ PlanShared sh;
    plan_begin(sh, p.seqs);
    const int i = threadIdx.x;
    int slot = 0, len = 0, want = 0, need = 0, src = 0;
    if (i < n) {
        slot = slots[i];
        want = lens ? lens[i] : 0;
        if ((unsigned)slot >= (unsigned)p.seqs || want < 0 || mark(sh.bits, slot)) plan_fail(sh, HYMT_E_ARG);
        else {
            len = p.len[slot];
            if (len < 0 || len > (long)p.blocks * kPage) {
                plan_fail(sh, HYMT_E_STATE);
                len = 0;
            }
            want = min(want, len);
            if (want < len && want % kPage) {
                src = p.table[(size_t)slot * p.blocks + want / kPage];
                if ((unsigned)src >= (unsigned)p.pages || p.refs[src] <= 0) plan_fail(sh, HYMT_E_STATE);
                else need = p.refs[src] > 1;
            }
            sh.slot[i] = slot;
            sh.first[i] = blocks_of(want);
            sh.count[i] = blocks_of(len) - blocks_of(want);
        }
    }
    int total;
    const int rank = block_scan(need, sh.wave, total);
    int32_t *list = work_dst(p);
    const bool enough = total <= p.pages && (total == 0 || find_free(p, total, list, sh.wave));
    if (!enough && i == 0) plan_fail(sh, HYMT_E_CAPACITY);
    __syncthreads();
    if (sh.status == HYMT_OK)
        for (int e = threadIdx.x >> 6; e < n; e += kPlanWaves)
            for (int j = threadIdx.x & 63; j < sh.count[e]; j += 64)
                if ((unsigned)p.table[(size_t)sh.slot[e] * p.blocks + sh.first[e] + j] >= (unsigned)p.pages)
                    plan_fail(sh, HYMT_E_STATE);
    __syncthreads();
    if (sh.status != HYMT_OK) {
        if (i == 0) finish(p, sh.status, 0);
        return;
    }
    if (i < n) {
        p.len[slot] = want;
        if (need) {
            const int dst = list[rank];
            work_src(p)[rank] = src;
            p.table[(size_t)slot * p.blocks + want / kPage] = dst;
            p.refs[dst] = 1;
            atomicSub(&p.refs[src], 1);
        }
    }
    for (int e = threadIdx.x >> 6; e < n; e += kPlanWaves)
        for (int j = threadIdx.x & 63; j < sh.count[e]; j += 64) {
            int32_t *at = &p.table[(size_t)sh.slot[e] * p.blocks + sh.first[e] + j];
            atomicSub(&p.refs[*at], 1);
            *at = -1;
        }
    if (i == 0) finish(p, HYMT_OK, total);
}

__global__ __launch_bounds__(kPlanThreads) void paged_compact_plan_kernel(hymt_paged p) {
    __shared__ int s_wave[kPlanWaves];
    const int live = count_live(p, s_wave);
    int holes = 0, movers = 0, total;
    for_pages(p, 0, live, [&](int i, int refs, bool ok) {
        const int free = ok && refs <= 0;
        const int at = holes + block_scan(free, s_wave, total);
        if (free) work_dst(p)[at] = i;
        holes += total;
    });
    for_pages(p, live, p.pages, [&](int i, int refs, bool ok) {
        const int used = ok && refs > 0;
        const int at = movers + block_scan(used, s_wave, total);
        if (used) work_src(p)[at] = i;
        movers += total;
    });
    __syncthreads();  // as many holes below `live` as pages in use above
    for (int i = live + (int)threadIdx.x; i < p.pages; i += kPlanThreads) work_map(p)[i] = i;
    __syncthreads();
    for (int k = threadIdx.x; k < movers; k += kPlanThreads) {
        const int src = work_src(p)[k], dst = work_dst(p)[k];
        work_map(p)[src] = dst;
        p.refs[dst] = p.refs[src];
        p.refs[src] = 0;
    }
    if (threadIdx.x == 0) {
        p.work[kWorkLive] = live;
        finish(p, HYMT_OK, movers);
    }
}

// The second launch of fork, set_len and compact: the pairs of pages that the
// plan wrote, copied in every layer, and (first) the rows of the table.
//
// A unit is the share of one kv head in one page, one layer, K or V: 64 * D
// values in one run, read by 256 threads 16 bytes at a time, all of a thread's
// loads before its stores.  Units are dealt out round the whole grid, so few
// pairs in many layers and many pairs in one fill the chip alike.
enum ApplyMode { kApplyCopy, kApplyFork, kApplyCompact };

template <int D, int MODE>
__global__ __launch_bounds__(256) void paged_apply_kernel(hymt_paged p, const int32_t *parent, const int32_t *child,
                                                          int n, int table_wgs) {
    if (p.work[kWorkStatus] != HYMT_OK) return;
    if (MODE != kApplyCopy && (int)blockIdx.x < table_wgs) {
        if (MODE == kApplyFork) {
            for (int e = blockIdx.x; e < n; e += table_wgs) {
                const int32_t *from = p.table + (size_t)parent[e] * p.blocks;
                int32_t *to = p.table + (size_t)child[e] * p.blocks;
                const int whole = p.len[child[e]] / kPage;
                for (int j = threadIdx.x; j < whole; j += 256) {
                    const int page = from[j];
                    to[j] = page;
                    atomicAdd(&p.refs[page], 1);
                }
            }
        } else {
            const int live = p.work[kWorkLive];
            const size_t all = (size_t)p.seqs * p.blocks;
            for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (size_t)table_wgs * 256) {
                const int page = p.table[i];
                if (page >= live && page < p.pages) p.table[i] = work_map(p)[page];
            }
        }
        return;
    }
    const int first = MODE == kApplyCopy ? 0 : table_wgs;
    constexpr int kVec = kPage * D * 2 / 16, kEach = kVec / 256;
    const int pairs = p.work[kWorkCopies];
    const size_t units = (size_t)pairs * p.layers * 2 * p.kv_heads;
    for (size_t u = blockIdx.x - first; u < units; u += gridDim.x - first) {
        const int h = (int)(u % p.kv_heads);
        size_t r = u / p.kv_heads;
        const bool isv = r & 1;
        r >>= 1;
        const int layer = (int)(r % p.layers), pair = (int)(r / p.layers);
        const size_t at = (size_t)layer * p.pages;
        uint4 *pool = (uint4 *)(isv ? p.v : p.k);
        const uint4 *src = pool + ((at + work_src(p)[pair]) * p.kv_heads + h) * kVec;
        uint4 *dst = pool + ((at + work_dst(p)[pair]) * p.kv_heads + h) * kVec;
        uint4 x[kEach];
#pragma unroll
        for (int e = 0; e < kEach; e++) x[e] = src[threadIdx.x + 256 * e];
#pragma unroll
        for (int e = 0; e < kEach; e++) dst[threadIdx.x + 256 * e] = x[e];
    }
}

template <int MODE>
void launch_apply(const char *name, const hymt_paged &p, const int32_t *parent, const int32_t *child, int n,
                  size_t max_pairs, int table_wgs, hipStream_t s) {
    const size_t units = max_pairs * p.layers * 2 * p.kv_heads;
    const int grid = table_wgs + (int)std::min<size_t>(std::max<size_t>(units, 1), 2048);
    KernelSpan span(name, s, true);
    if (p.head_dim == 64)
        launch(span, paged_apply_kernel<64, MODE>, dim3(grid), dim3(256), 0, s, p, parent, child, n, table_wgs);
    else
        launch(span, paged_apply_kernel<128, MODE>, dim3(grid), dim3(256), 0, s, p, parent, child, n, table_wgs);
}

}  // namespace

hipError_t launch_paged_extend(const hymt_paged &p, const int32_t *slots, const int32_t *cu, int n, hipStream_t s) {
    if (n == 0) return hipSuccess;
    KernelSpan span("paged_extend", s, true);
    launch(span, paged_extend_kernel, dim3(1), dim3(kPlanThreads), 0, s, p, slots, cu, n);
    return hipGetLastError();
}

hipError_t launch_paged_fork(const hymt_paged &p, const int32_t *parent, const int32_t *child, int n, hipStream_t s) {
    if (n == 0) return hipSuccess;
    {
        KernelSpan span("paged_plan", s, true);
        launch(span, paged_fork_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, p, parent, child, n);
    }
    if (hipError_t e = hipGetLastError()) return e;
    launch_apply<kApplyFork>("paged_copy", p, parent, child, n, n, n, s);
    return hipGetLastError();
}

hipError_t launch_paged_set_len(const hymt_paged &p, const int32_t *slots, const int32_t *lens, int n, hipStream_t s) {
    if (n == 0) return hipSuccess;
    {
        KernelSpan span("paged_plan", s, true);
        launch(span, paged_set_len_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, p, slots, lens, n);
    }
    if (hipError_t e = hipGetLastError()) return e;
    if (!lens) return hipSuccess;  // whole slots: nothing to copy
    launch_apply<kApplyCopy>("paged_copy", p, nullptr, nullptr, 0, n, 0, s);
    return hipGetLastError();
}

hipError_t launch_paged_compact(const hymt_paged &p, hipStream_t s) {
    {
        KernelSpan span("paged_plan", s, true);
        launch(span, paged_compact_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, p);
    }
    if (hipError_t e = hipGetLastError()) return e;
    const size_t entries = (size_t)p.seqs * p.blocks;
    const int table_wgs = (int)std::min<size_t>((entries + 1023) / 1024, 256);
    launch_apply<kApplyCompact>("paged_copy", p, nullptr, nullptr, 0, p.pages / 2, table_wgs, s);
    return hipGetLastError();
}

// ------------------------------------------------------------------ rotary append

namespace {

// Entry of row r: the last i with cu[i] <= r.  Lanes of a wave look at 64
// entries at a time (one load each, no chain of dependent ones).
__device__ __forceinline__ int entry_of_row(const int32_t *cu, int n, int r) {
    const int lane = threadIdx.x & 63;
    int below = 0;  // entries whose end is at or before r
    for (int base = 0; base < n; base += 64) {
        const int i = base + lane;
        below += __popcll(__ballot(i < n && cu[i + 1] <= r));
    }
    return below;
}

template <typename IO> __device__ __forceinline__ void load8(const void *base, size_t i, float *o) {
    if constexpr (IO::kBytes == 4) {
        const float4 a = *(const float4 *)((const float *)base + i), b = *(const float4 *)((const float *)base + i + 4);
        o[0] = a.x; o[1] = a.y; o[2] = a.z; o[3] = a.w;
        o[4] = b.x; o[5] = b.y; o[6] = b.z; o[7] = b.w;
    } else {
        const uint4 u = *(const uint4 *)((const uint16_t *)base + i);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int e = 0; e < 4; e++) {
            o[2 * e] = from_elem<IO>((uint16_t)w[e]);
            o[2 * e + 1] = from_elem<IO>((uint16_t)(w[e] >> 16));
        }
    }
}

// One workgroup per row: cosines and sines of the row's position once into
// LDS, then D / 8 lanes per head (8 dims each) over q, k and v heads.
template <typename T, typename IO, int D>
__global__ __launch_bounds__(256) void rope_append_kernel(hymt_paged p, hymt_batch b, RopeAppend a) {
    constexpr int L = D / 8;
    __shared__ float s_cos[64], s_sin[64];
    const int row = blockIdx.x;
    int entry = row;
    int n_rows = 1, j = 0;
    if (b.cu) {
        entry = entry_of_row(b.cu, b.n, row);
        if (entry >= b.n) return;
        n_rows = b.cu[entry + 1] - b.cu[entry];
        j = row - b.cu[entry];
    }
    if (entry >= b.n) return;
    const int slot = b.slots[entry];
    const bool known = (unsigned)slot < (unsigned)p.seqs;
    const int pos = (known ? p.len[slot] : 0) - n_rows + j;
    const int half = a.dim / 2;
    if ((int)threadIdx.x < half) {
        // revolutions in fp64, whose fraction is what counts at far positions
        const double turn = (double)pos * a.freq[threadIdx.x] * 0.15915494309189535;
        const float x = (float)(turn - rint(turn)) * 2.0f;
        float sn, cs;
        sincospif(x, &sn, &cs);
        s_cos[threadIdx.x] = cs * a.scale;
        s_sin[threadIdx.x] = sn * a.scale;
    }
    __syncthreads();
    const bool stored = known && pos >= 0 && pos < (long)p.blocks * kPage;
    int page = stored ? p.table[(size_t)slot * p.blocks + pos / kPage] : -1;
    const bool in_pool = (unsigned)page < (unsigned)p.pages;
    const int t = pos & (kPage - 1);
    const int c = threadIdx.x & (L - 1), d0 = 8 * c;
    const int units = a.heads + 2 * p.kv_heads;
    for (int base = 0; base < units; base += 256 / L) {
        const int u = base + threadIdx.x / L;
        const bool on = u < units;
        const int uc = on ? u : units - 1;
        const bool isq = uc < a.heads, isv = uc >= a.heads + p.kv_heads;
        const int h = isq ? uc : isv ? uc - a.heads - p.kv_heads : uc - a.heads;
        float x[8];
        load8<IO>(isq ? a.q : isv ? a.v : a.k, (size_t)row * (isq ? a.q_ld : a.kv_ld) + (size_t)h * D + d0, x);
        if (!isv) {
            if (a.interleaved) {
                if (d0 < a.dim)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float cs = s_cos[d0 / 2 + e], sn = s_sin[d0 / 2 + e], y0 = x[2 * e], y1 = x[2 * e + 1];
                        x[2 * e] = y0 * cs - y1 * sn;
                        x[2 * e + 1] = y1 * cs + y0 * sn;
                    }
            } else {
                const bool low = d0 < half;
                const int other = (int)(threadIdx.x & 63) + (d0 >= a.dim ? 0 : low ? half / 8 : -(half / 8));
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float y = __shfl(x[e], other);
                    if (d0 < a.dim) {
                        const int i = low ? d0 + e : d0 - half + e;
                        x[e] = low ? x[e] * s_cos[i] - y * s_sin[i] : x[e] * s_cos[i] + y * s_sin[i];
                    }
                }
            }
            const float *w = isq ? a.qnw : a.knw;
            if (w) {
                float ss = 0.f;
#pragma unroll
                for (int e = 0; e < 8; e++) ss += x[e] * x[e];
#pragma unroll
                for (int m = 1; m < L; m <<= 1) ss += __shfl_xor(ss, m);
                const float r = 1.0f / sqrtf(ss / (float)D + a.eps);
#pragma unroll
                for (int e = 0; e < 8; e++) x[e] = x[e] * r * w[d0 + e];
            }
        }
        uint16_t y[8];
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] = bits_of<T>(x[e]);
        if (!on) continue;
        if (isv) {
            if (in_pool) {
                uint16_t *vp = (uint16_t *)p.v + (((size_t)a.layer * p.pages + page) * p.kv_heads + h) * (kPage * D);
                const int pc = 4 * (t >> 5) + ((t >> 2) & 3), e0 = 4 * ((t >> 4) & 1) + (t & 3);
#pragma unroll
                for (int e = 0; e < 8; e++) vp[((size_t)pc * D + d0 + e) * 8 + e0] = y[e];
            }
            continue;
        }
        const uint4 w = make_uint4(y[0] | (uint32_t)y[1] << 16, y[2] | (uint32_t)y[3] << 16, y[4] | (uint32_t)y[5] << 16,
                                   y[6] | (uint32_t)y[7] << 16);
        if (isq) {
            *(uint4 *)((uint16_t *)a.q_out + (size_t)row * a.heads * D + (size_t)h * D + d0) = w;
        } else if (in_pool) {
            uint16_t *kp = (uint16_t *)p.k + (((size_t)a.layer * p.pages + page) * p.kv_heads + h) * (kPage * D);
            *(uint4 *)(kp + ((((size_t)(t >> 4) * L + c) * 16 + (t & 15)) << 3)) = w;
        }
    }
}

template <typename T, typename IO>
void launch_rope(const hymt_paged &p, const hymt_batch &b, const RopeAppend &a, hipStream_t s) {
    KernelSpan span("rope_append", s, true);
    if (p.head_dim == 64) launch(span, rope_append_kernel<T, IO, 64>, dim3(b.rows), dim3(256), 0, s, p, b, a);
    else launch(span, rope_append_kernel<T, IO, 128>, dim3(b.rows), dim3(256), 0, s, p, b, a);
}

}  // namespace

hipError_t launch_rope_append(const hymt_paged &p, const hymt_batch &b, const RopeAppend &a, hipStream_t s) {
    if (b.n == 0 || b.rows == 0) return hipSuccess;
    const bool f16 = p.dtype == HYMT_F16;
    switch (a.io_dtype) {
    case HYMT_F32: f16 ? launch_rope<F16, F32>(p, b, a, s) : launch_rope<BF16, F32>(p, b, a, s); break;
    case HYMT_F16: f16 ? launch_rope<F16, F16>(p, b, a, s) : launch_rope<BF16, F16>(p, b, a, s); break;
    default: f16 ? launch_rope<F16, BF16>(p, b, a, s) : launch_rope<BF16, BF16>(p, b, a, s); break;
    }
    return hipGetLastError();
}

}  // namespace hymt
