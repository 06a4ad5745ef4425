// paged_ops.hip -- upkeep of the multi-sequence cache's pages, and the rows of
// a batch rotated, normed and appended to them (hymt_paged, include/hymt_hip.h).
//
// Upkeep: the plan of a call -- who gets which free page, what is copied, what
// loses a reference -- is made by one workgroup, from the reference counts
// alone (there is no free list that could disagree with them), and a second
// launch over the whole chip moves the bytes.  extend moves none and is the plan
// alone.  A plan first looks at everything it would rely on and only then writes, so a
// call that finds something wrong changes nothing but `work`.  A plan is a chain of
// round trips (entries, lengths, table, counts) and two scans: 64 slots extended in 4.2 us,
// 16 forked in 5.0, 64 of 1000 positions released in 7.4, a pool of 512 compacted in 3.5.  Free
// pages are looked for from the first on, 1024 at a time, 0.9 us each: behind 10000 pages in use 64
// slots get one in 12.7 us, behind 60000 in 59.
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

// Exclusive prefix sums of two values over the workgroup's threads, and their totals.
struct Sums {
    int a, b, all_a, all_b;
};
__device__ __forceinline__ Sums block_scan(int va, int vb, int2 *s_wave) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int xa = wave_sums(va), xb = wave_sums(vb);
    __syncthreads();  // s_wave's last readers
    if (lane == 63) s_wave[wave] = make_int2(xa, xb);
    __syncthreads();
    Sums r{xa - va, xb - vb, 0, 0};
#pragma unroll
    for (int w = 0; w < kPlanWaves; w++) {
        const int2 t = s_wave[w];
        if (w == wave) {
            r.a += r.all_a;
            r.b += r.all_b;
        }
        r.all_a += t.x;
        r.all_b += t.y;
    }
    return r;
}

// Whether page `page` of the pool can be had; a page past the end cannot.
__device__ __forceinline__ int is_free(const hymt_paged &p, int page) { return page < p.pages && p.refs[page] <= 0; }

// One thread ends a call: its status, and the first that was not good.
__device__ void finish(const hymt_paged &p, int status, int copies) {
    p.work[kWorkStatus] = status;
    p.work[kWorkCopies] = copies;
    if (status != HYMT_OK && p.work[kWorkFirst] == HYMT_OK) p.work[kWorkFirst] = status;
}

// Pages in use (all threads get the number).
__device__ int count_live(const hymt_paged &p, int2 *s_wave) {
    int mine = 0;
    for (int i = threadIdx.x; i < p.pages; i += kPlanThreads) mine += p.refs[i] > 0;
    return block_scan(mine, 0, s_wave).all_a;
}

// A slot's place in a bit per slot; true if it was set already.
__device__ __forceinline__ bool mark(uint32_t *bits, int slot) {
    const uint32_t m = 1u << (slot & 31);
    return (atomicOr(&bits[slot >> 5], m) & m) != 0;
}

struct PlanShared {
    uint32_t bits[kPagedMaxSeqs / 32];
    int2 wave[kPlanWaves];
    int status;
    int free[kPlanThreads];  // the lowest free pages handed out
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

// Ranks of the entries' `need` free pages, lowest pages first: entry i gets
// [rank, rank + need) of list, of which the first 1024 are in sh.free too.  free0 is
// is_free of page threadIdx.x, loaded before it was known how many are needed.
// False if there are too few.
__device__ bool hand_out(const hymt_paged &p, PlanShared &sh, int need, int free0, int32_t *list, int &rank, int &total) {
    const int tid = threadIdx.x;
    Sums s = block_scan(need, free0, sh.wave);
    rank = s.a;
    total = s.all_a;
    int at = s.b, found = s.all_b, page = tid, free = free0;
    for (int base = kPlanThreads;; base += kPlanThreads) {
        if (free && at < total) {
            list[at] = page;
            if (at < kPlanThreads) sh.free[at] = page;
        }
        if (found >= total || base >= p.pages) break;
        page = base + tid;
        free = is_free(p, page);
        s = block_scan(0, free, sh.wave);
        at = found + s.b;
        found += s.all_b;
    }
    __syncthreads();
    return found >= total;
}

__global__ __launch_bounds__(kPlanThreads) void paged_extend_kernel(hymt_paged p, const int32_t *slots,
                                                                    const int32_t *cu, int n) {
    __shared__ PlanShared sh;
    const int i = threadIdx.x, free0 = is_free(p, i);
    int slot = -1, from = 0, to = 0;
    if (i < n) {
        slot = slots[i];
        from = cu ? cu[i] : i;
        to = cu ? cu[i + 1] : i + 1;
    }
    plan_begin(sh, p.seqs);
    int len = 0, add = 0, need = 0;
    if (i < n) {
        if ((unsigned)slot >= (unsigned)p.seqs || to < from || (i == 0 && from != 0) || mark(sh.bits, slot)) {
            plan_fail(sh, HYMT_E_ARG);
        } else {
            add = to - from;  // offsets that rise from 0 on: all together below 2^31
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
    int32_t *list = work_src(p);
    int rank, total;
    if (!hand_out(p, sh, need, free0, list, rank, total) && i == 0) plan_fail(sh, HYMT_E_CAPACITY);
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
    if (total > 0) {
        __syncthreads();
        for (int e = threadIdx.x >> 6; e < n; e += kPlanWaves)
            for (int j = threadIdx.x & 63; j < sh.count[e]; j += 64) {
                const int at = sh.rank[e] + j, page = at < kPlanThreads ? sh.free[at] : list[at];
                p.table[(size_t)sh.slot[e] * p.blocks + sh.first[e] + j] = page;
                p.refs[page] = 1;
            }
    }
    if (i == 0) finish(p, HYMT_OK, 0);
}

__global__ __launch_bounds__(kPlanThreads) void paged_fork_plan_kernel(hymt_paged p, const int32_t *parent,
                                                                       const int32_t *child, int n) {
    __shared__ PlanShared sh;
    const int i = threadIdx.x, free0 = is_free(p, i);
    int from = 0, to = 0, len = 0, need = 0, src = 0, held = 1;
    bool known = false, gone = false;
    if (i < n) {
        from = parent[i];
        to = child[i];
        known = (unsigned)from < (unsigned)p.seqs && (unsigned)to < (unsigned)p.seqs;
    }
    plan_begin(sh, p.seqs);
    if (i < n && (!known || mark(sh.bits, to))) plan_fail(sh, HYMT_E_ARG);
    if (i < n) sh.count[i] = 0;
    if (known) {
        len = p.len[from];
        if (len < 0 || len > (long)p.blocks * kPage || p.len[to] != 0) {
            plan_fail(sh, HYMT_E_STATE);
            len = 0;
        }
        if (len % kPage) {
            need = 1;
            src = p.table[(size_t)from * p.blocks + len / kPage];
            if ((unsigned)src >= (unsigned)p.pages) plan_fail(sh, HYMT_E_STATE);
            else held = p.refs[src];
        }
        sh.slot[i] = from;
        sh.count[i] = len / kPage;
    }
    __syncthreads();
    if (known && (sh.bits[from >> 5] >> (from & 31) & 1)) plan_fail(sh, HYMT_E_ARG);
    // whole pages have to be in the pool, and in use (a free one may be handed out
    // here), before one of them is counted again
    for (int e = threadIdx.x >> 6; e < n; e += kPlanWaves)
        for (int j = threadIdx.x & 63; j < sh.count[e]; j += 64) {
            const int page = p.table[(size_t)sh.slot[e] * p.blocks + j];
            if ((unsigned)page >= (unsigned)p.pages) plan_fail(sh, HYMT_E_STATE);
            else gone |= p.refs[page] <= 0;
        }
    int32_t *list = work_dst(p);
    int rank, total;
    if (!hand_out(p, sh, need, free0, list, rank, total) && i == 0) plan_fail(sh, HYMT_E_CAPACITY);
    // the counts, loaded while the free pages were looked up; a page that is copied is
    // its sequence's alone
    if (gone || held != 1) plan_fail(sh, HYMT_E_STATE);
    __syncthreads();
    if (sh.status != HYMT_OK) {
        if (i == 0) finish(p, sh.status, 0);
        return;
    }
    if (i < n) {
        p.len[to] = len;
        if (need) {
            const int dst = sh.free[rank];
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
    const int i = threadIdx.x, free0 = is_free(p, i);
    int slot = 0, len = 0, want = 0, need = 0, src = 0;
    bool gone = false;
    if (i < n) {
        slot = slots[i];
        want = lens ? lens[i] : 0;
    }
    plan_begin(sh, p.seqs);
    if (i < n) {
        sh.count[i] = 0;
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
    __syncthreads();
    // pages that are given up have to be in the pool and in use
    for (int e = threadIdx.x >> 6; e < n; e += kPlanWaves)
        for (int j = threadIdx.x & 63; j < sh.count[e]; j += 64) {
            const int page = p.table[(size_t)sh.slot[e] * p.blocks + sh.first[e] + j];
            if ((unsigned)page >= (unsigned)p.pages) plan_fail(sh, HYMT_E_STATE);
            else gone |= p.refs[page] <= 0;
        }
    int32_t *list = work_dst(p);
    int rank, total;
    if (!hand_out(p, sh, need, free0, list, rank, total) && i == 0) plan_fail(sh, HYMT_E_CAPACITY);
    if (gone) plan_fail(sh, HYMT_E_STATE);
    __syncthreads();
    if (sh.status != HYMT_OK) {
        if (i == 0) finish(p, sh.status, 0);
        return;
    }
    if (i < n) {
        p.len[slot] = want;
        if (need) {
            const int dst = sh.free[rank];
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
    __shared__ int2 s_wave[kPlanWaves];
    const int live = count_live(p, s_wave);
    // as many holes below `live` as pages in use from there on
    int holes = 0, movers = 0;
    for (int base = 0; base < p.pages; base += kPlanThreads) {
        const int i = base + (int)threadIdx.x, refs = i < p.pages ? p.refs[i] : 0;
        const int hole = i < live && refs <= 0, mover = i >= live && refs > 0;
        const Sums s = block_scan(hole, mover, s_wave);
        if (hole) work_dst(p)[holes + s.a] = i;
        if (mover) work_src(p)[movers + s.b] = i;
        if (i >= live && i < p.pages) work_map(p)[i] = i;
        holes += s.all_a;
        movers += s.all_b;
    }
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
// pairs in many layers and many pairs in one fill the chip alike.  Bound by HBM: 150
// pages of 8 layers, 157 MB, in 62 us, 5.0 TB/s read and written; one page of 32
// layers sixteen times, 67 MB, in 13.9.
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

// 8 values of a row as loaded (16 bytes, fp32 32), and in fp32.
template <typename IO> struct Raw8 {
    uint4 u[IO::kBytes / 2];
};
template <typename IO> __device__ __forceinline__ Raw8<IO> load8(const void *base, size_t i) {
    Raw8<IO> r;
#pragma unroll
    for (int k = 0; k < IO::kBytes / 2; k++) r.u[k] = *(const uint4 *)((const char *)base + i * IO::kBytes + 16 * k);
    return r;
}
template <typename IO> __device__ __forceinline__ void values8(const Raw8<IO> &r, float *o) {
    if constexpr (IO::kBytes == 4) {
#pragma unroll
        for (int k = 0; k < 2; k++) {
            o[4 * k] = __uint_as_float(r.u[k].x);
            o[4 * k + 1] = __uint_as_float(r.u[k].y);
            o[4 * k + 2] = __uint_as_float(r.u[k].z);
            o[4 * k + 3] = __uint_as_float(r.u[k].w);
        }
    } else {
        const uint32_t w[4] = {r.u[0].x, r.u[0].y, r.u[0].z, r.u[0].w};
#pragma unroll
        for (int e = 0; e < 4; e++) {
            o[2 * e] = from_elem<IO>((uint16_t)w[e]);
            o[2 * e + 1] = from_elem<IO>((uint16_t)(w[e] >> 16));
        }
    }
}
template <typename T> __device__ __forceinline__ uint4 pack8(const float *x) {
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; e++) w[e] = bits_of<T>(x[2 * e]) | (uint32_t)bits_of<T>(x[2 * e + 1]) << 16;
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// (cosine, sine) of position * freq, times scale.  The angle is formed in
// revolutions in fp64, where the product is good to 2^-53 of itself at any
// position, and only its fraction goes on in fp32.
__device__ __forceinline__ float2 turn_of(int pos, double freq, float scale) {
    const double turn = (double)pos * freq * 0.15915494309189535;
    float sn, cs;
    sincospif((float)(turn - rint(turn)) * 2.0f, &sn, &cs);
    return make_float2(cs * scale, sn * scale);
}

// What a lane (8 dims from d0 = 8 c of a head) needs of its row's turns: the pairs of
// its dims, interleaved the 4 it holds whole, else the 8 that it holds one half of.
struct Turns {
    float cs[8], sn[8];
};
__device__ __forceinline__ Turns turns_of(const float2 *row, int c, const RopeAppend &a) {
    const int d0 = 8 * c, half = a.dim / 2;
    Turns t;
    const float2 *at = row + (d0 >= a.dim ? 0 : a.interleaved ? d0 / 2 : d0 < half ? d0 : d0 - half);
    const int n = d0 >= a.dim ? 0 : a.interleaved ? 4 : 8;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const float2 x = e < n ? at[e] : make_float2(1.f, 0.f);
        t.cs[e] = x.x;
        // the second of a pair adds what the first takes away
        t.sn[e] = !a.interleaved && d0 < half ? -x.y : x.y;
    }
    return t;
}

// y = x of lane c +- hc (half / 8) of the head's lanes: by DPP at the usual sizes
template <int CTRL> __device__ __forceinline__ float dpp_from(float x) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xF, 0xF, false));
}
__device__ __forceinline__ void partners(const float *x, float *y, int c, int hc, int other) {
    if (hc == 8) {
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] = dpp_from<0x128>(x[e]);  // turned by 8
    } else if (hc == 4) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float up = dpp_from<0x104>(x[e]), dn = dpp_from<0x114>(x[e]);  // from lanes + 4 and - 4
            y[e] = c & 4 ? dn : up;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] = __shfl(x[e], other);
    }
}

// Sum over the L = 8 or 16 neighbouring lanes of a head.
template <int L> __device__ __forceinline__ float lanes_sum(float v) {
    if constexpr (L == 16) return dpp_sum16(v);
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0xB1, 0xF, 0xF, false));
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x4E, 0xF, 0xF, false));
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x141, 0xF, 0xF, false));
    return v;
}

// 8 dims of a head, L = D / 8 neighbouring lanes holding it whole: rotation,
// then RMSNorm with the lane's weights g where the head has one.
template <int D>
__device__ __forceinline__ void rotate_norm(float *x, int c, const Turns &t, const RopeAppend &a, bool norm, const float *g) {
    constexpr int L = D / 8;
    const int d0 = 8 * c;
    if (a.interleaved) {
        if (d0 < a.dim)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float y0 = x[2 * e], y1 = x[2 * e + 1];
                x[2 * e] = y0 * t.cs[e] - y1 * t.sn[e];
                x[2 * e + 1] = y1 * t.cs[e] + y0 * t.sn[e];
            }
    } else if (a.dim) {
        const int hc = a.dim / 16;
        const int other = (int)(threadIdx.x & 63) + (d0 >= a.dim ? 0 : c < hc ? hc : -hc);
        float y[8];
        partners(x, y, c, hc, other);
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = d0 < a.dim ? x[e] * t.cs[e] + y[e] * t.sn[e] : x[e];
    }
    if (norm) {
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 8; e++) ss += x[e] * x[e];
        const float r = __builtin_amdgcn_rsqf(lanes_sum<L>(ss) * (1.0f / D) + a.eps);
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = x[e] * r * g[e];
    }
}

// The norm's weights of a lane's dims.
__device__ __forceinline__ void weights8(const float *w, int d0, float *g) {
    if (!w) return;
    const float4 w0 = *(const float4 *)(w + d0), w1 = *(const float4 *)(w + d0 + 4);
    g[0] = w0.x; g[1] = w0.y; g[2] = w0.z; g[3] = w0.w;
    g[4] = w1.x; g[5] = w1.y; g[6] = w1.z; g[7] = w1.w;
}

__device__ __forceinline__ int slot_length(const hymt_paged &p, int slot) {
    return (unsigned)slot < (unsigned)p.seqs ? max(0, min(p.len[slot], 1 << 30)) : 0;
}

// Whether the last upkeep call went through.  If not, the lengths are those before it and
// a batch's rows would fall on positions that stand already, of other sequences too
// where the last page is whole.  Loaded beside what a row needs anyway.
__device__ __forceinline__ bool has_grown(const hymt_paged &p) { return p.work[kWorkStatus] == HYMT_OK; }

// The entry of row r (the first that ends behind it), its slot and its rows from r on.
// Lanes look at 64 runs of entries, then at the run's, in two round trips at most.
struct RowEntry {
    int slot, behind;
};
__device__ __forceinline__ bool entry_of_row(const hymt_batch &b, int r, RowEntry &out) {
    static_assert(HYMT_PAGED_BATCH <= 64 * 64, "two steps");
    const int lane = threadIdx.x & 63, run = (b.n + 63) / 64;
    int first = 0;
    if (run > 1) {
        const uint64_t hit = __ballot(lane * run < b.n && b.cu[min((lane + 1) * run, b.n)] > r);
        if (!hit) return false;
        first = (__ffsll((unsigned long long)hit) - 1) * run;
    }
    const int i = min(first + lane, b.n - 1);
    const int end = b.cu[i + 1], slot = b.slots[i];
    const uint64_t hit = __ballot(first + lane < b.n && end > r);
    if (!hit) return false;
    const int k = __ffsll((unsigned long long)hit) - 1;
    out = {__builtin_amdgcn_readlane(slot, k), __builtin_amdgcn_readlane(end, k) - r};
    return true;
}

// A workgroup a row, for batches of few rows.  q, k and v do not wait for the
// row's position, so they are loaded first.  64 rows 4.9 us in a recording: a launch
// and three round trips (entry, length, page).
template <typename T, typename IO, int D>
__global__ __launch_bounds__(256) void rope_row_kernel(hymt_paged p, hymt_batch b, RopeAppend a) {
    constexpr int L = D / 8, U = 256 / L;
    __shared__ float2 s_cs[D / 2];
    const int row = blockIdx.x;
    const int c = threadIdx.x & (L - 1), d0 = 8 * c;
    const int units = a.heads + 2 * p.kv_heads;
    auto load = [&](int u) __attribute__((always_inline)) {
        u = min(u, units - 1);
        const bool isq = u < a.heads, isv = u >= a.heads + p.kv_heads;
        const int h = isq ? u : isv ? u - a.heads - p.kv_heads : u - a.heads;
        return load8<IO>(isq ? a.q : isv ? a.v : a.k, (size_t)row * (isq ? a.q_ld : a.kv_ld) + (size_t)h * D + d0);
    };
    const int u0 = threadIdx.x / L;
    Raw8<IO> next = load(u0), after = load(u0 + U);
    const double freq = (int)threadIdx.x < a.dim / 2 ? a.freq[threadIdx.x] : 0.0;
    const bool grown = has_grown(p);
    RowEntry e{0, 1};
    if (!b.cu) e.slot = b.slots[row];
    else if (!entry_of_row(b, row, e)) return;
    const int slot = e.slot, pos = slot_length(p, slot) - e.behind;
    if ((int)threadIdx.x < a.dim / 2) s_cs[threadIdx.x] = turn_of(pos, freq, a.scale);
    const bool stored = grown && pos >= 0 && pos < (long)p.blocks * kPage;
    const int page = stored ? p.table[(size_t)slot * p.blocks + pos / kPage] : -1;
    const bool in_pool = (unsigned)page < (unsigned)p.pages;
    const int t = pos & (kPage - 1);
    float gq[8] = {}, gk[8] = {};
    weights8(a.qnw, d0, gq);
    weights8(a.knw, d0, gk);
    __syncthreads();
    const Turns turns = turns_of(s_cs, c, a);
    for (int base = 0; base < units; base += U) {
        const int u = base + u0;
        const bool isq = u < a.heads, isv = u >= a.heads + p.kv_heads;
        float x[8], y[8];
        values8<IO>(next, x);
        next = after;
        if (base + 2 * U < units) after = load(u + 2 * U);
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] = x[e];
        float g[8];
#pragma unroll
        for (int e = 0; e < 8; e++) g[e] = isq ? gq[e] : gk[e];
        rotate_norm<D>(y, c, turns, a, (isq ? a.qnw : a.knw) != nullptr, g);
        if (u >= units) continue;
        const int h = isq ? u : isv ? u - a.heads - p.kv_heads : u - a.heads;
        const size_t at = (((size_t)a.layer * p.pages + page) * p.kv_heads + h) * (size_t)(kPage * D);
        if (isq) {
            *(uint4 *)((uint16_t *)a.q_out + (size_t)row * a.heads * D + (size_t)h * D + d0) = pack8<T>(y);
        } else if (in_pool && !isv) {
            *(uint4 *)((uint16_t *)p.k + at + ((((size_t)(t >> 4) * L + c) * 16 + (t & 15)) << 3)) = pack8<T>(y);
        } else if (in_pool) {
            const int pc = 4 * (t >> 5) + ((t >> 2) & 3), e0 = 4 * ((t >> 4) & 1) + (t & 3);
            uint16_t *vp = (uint16_t *)p.v + at + ((size_t)pc * D + d0) * 8 + e0;
#pragma unroll
            for (int e = 0; e < 8; e++) vp[8 * e] = bits_of<T>(x[e]);
        }
    }
}

// Packed rows: a workgroup takes the rows of one entry that lie in one block of 32
// positions, for one kv head with its q heads.  A V chunk holds 8 of the block's
// positions, so the block writes its chunks whole, 16 bytes a thread, after a
// turn through LDS; row by row each chunk is written in 8 pieces, by
// workgroups on 8 XCDs.  19 k rows of 24 heads in 58 us, 4.0 TB/s over 118 MB read and
// 118 written, no more than it must (row by row 94 us; a plain copy would take 50).
constexpr int kRopeRows = 32;
// Row by row for batches of few rows, or of few an entry.  A row alone takes a round of
// loads less than a block, whose workgroups first look for their entry and do 32 rows
// in turn; blocks win once the chip has several rows a CU.  bf16 cache, 16 q heads,
// fp32 rows, by rows and by blocks, us: one entry of 64 rows 4.9 and 11.7, of 1024 10.8
// and 12.8, of 1536 15.0 and 13.5, of 2048 17.1 and 13.7; 256 entries of 12 25.5 and 26.3, of 16
// 34.5 and 31.7; 128 of 12 15.8 and 15.4; one of 8192 and 700 of 1 71 and 89, one of 2048 and 200 of 1
// 20.9 and 24.4.  The numbers are those of 4 kv heads: a block of a kv head with more q heads
// is a longer chain, with fewer a shorter one (8 q heads of one kv head, 1536 rows 9.3 and
// 18.1, 8192 28.5 and 19.9; 8 kv heads of one q head, bf16 rows, 1024 14.2 and 10.1, 1536 19.7 and 12.0).
constexpr int kRopeFew = 1536, kRopeFewEach = 14;

template <typename T, typename IO, int D>
__global__ __launch_bounds__(256) void rope_block_kernel(hymt_paged p, hymt_batch b, RopeAppend a) {
    constexpr int L = D / 8, RP = 256 / L, PASSES = kRopeRows / RP;
    __shared__ float2 s_cs[kRopeRows][D / 2];
    __shared__ __attribute__((aligned(16))) uint16_t s_v[kRopeRows][D + 8];
    const int tid = threadIdx.x, lane = tid & 63;
    const int h = blockIdx.x % p.kv_heads, w = blockIdx.x / p.kv_heads;
    const bool grown = has_grown(p);
    // ---- the block's entry: 64 entries at a time, one a lane
    int slot = -1, row0 = 0, n = 0, p0 = 0, index = -1;  // first row, rows, their first position, block of it
    for (int base = 0, before = 0; base < b.n; base += 64) {
        const int i = base + lane;
        int lo = 0, cnt = 0, sl = -1;
        if (i < b.n) {
            lo = max(0, min(b.cu[i], b.rows));
            cnt = max(lo, min(b.cu[i + 1], b.rows)) - lo;
            sl = b.slots[i];
        }
        const int at = slot_length(p, sl) - cnt;
        const int blocks = cnt ? ((at + cnt - 1) >> 5) - (at >> 5) + 1 : 0;
        const int x = wave_sums(blocks);
        const uint64_t hit = __ballot(w < before + x);
        if (hit) {
            const int k = __ffsll((unsigned long long)hit) - 1;
            slot = __builtin_amdgcn_readlane(sl, k);
            row0 = __builtin_amdgcn_readlane(lo, k);
            n = __builtin_amdgcn_readlane(cnt, k);
            p0 = __builtin_amdgcn_readlane(at, k);
            index = w - before - (__builtin_amdgcn_readlane(x, k) - __builtin_amdgcn_readlane(blocks, k));
            break;
        }
        before += __builtin_amdgcn_readlane(x, 63);
    }
    if (index < 0) return;
    const int pb = ((p0 >> 5) + index) * 32;  // position of the block's first row
    const int r_lo = max(0, p0 - pb), r_hi = min(kRopeRows, p0 + n - pb);
    const bool stored = grown && slot >= 0 && slot < p.seqs && pb >= 0 && pb < (long)p.blocks * kPage;
    const int page = stored ? p.table[(size_t)slot * p.blocks + pb / kPage] : -1;
    const bool in_pool = (unsigned)page < (unsigned)p.pages;
    const int c = tid & (L - 1), d0 = 8 * c, r0 = tid / L;
    const int group = a.heads / p.kv_heads, items = (group + 2) * PASSES;
    auto load = [&](int item) __attribute__((always_inline)) {
        const int u = item / PASSES, r = r0 + item % PASSES * RP;
        const size_t row = row0 + max(0, min(pb + r - p0, n - 1));  // rows outside are loaded for nothing, from inside
        const bool isq = u < group;
        return load8<IO>(isq ? a.q : u == group ? a.k : a.v,
                         row * (isq ? a.q_ld : a.kv_ld) + (size_t)(isq ? h * group + u : h) * D + d0);
    };
    Raw8<IO> next = load(0), after = load(1);
    const int half = a.dim / 2;
    for (int i = tid; i < (r_hi - r_lo) * half; i += 256) {
        const int r = r_lo + i / half, k = i % half;
        s_cs[r][k] = turn_of(pb + r, a.freq[k], a.scale);
    }
    float gq[8] = {}, gk[8] = {};
    weights8(a.qnw, d0, gq);
    weights8(a.knw, d0, gk);
    __syncthreads();
    const size_t at = (((size_t)a.layer * p.pages + page) * p.kv_heads + h) * (size_t)(kPage * D);
    Turns turns[PASSES];
#pragma unroll
    for (int k = 0; k < PASSES; k++) turns[k] = turns_of(s_cs[r0 + k * RP], c, a);
    for (int first = 0; first < items; first += PASSES)
#pragma unroll
    for (int pass = 0; pass < PASSES; pass++) {
        const int item = first + pass, u = item / PASSES, r = r0 + pass * RP, t = (pb + r) & (kPage - 1);
        float x[8];
        values8<IO>(next, x);
        next = after;
        if (item + 2 < items) after = load(item + 2);
        if (u > group) {
            *(uint4 *)&s_v[r][d0] = pack8<T>(x);
            continue;
        }
        if (u < group) rotate_norm<D>(x, c, turns[pass], a, a.qnw != nullptr, gq);
        else rotate_norm<D>(x, c, turns[pass], a, a.knw != nullptr, gk);
        if (r < r_lo || r >= r_hi) continue;
        if (u < group)
            *(uint4 *)((uint16_t *)a.q_out + (size_t)(row0 + pb + r - p0) * a.heads * D + (size_t)(h * group + u) * D + d0) =
                pack8<T>(x);
        else if (in_pool)
            *(uint4 *)((uint16_t *)p.k + at + ((((size_t)(t >> 4) * L + c) * 16 + (t & 15)) << 3)) = pack8<T>(x);
    }
    __syncthreads();
    if (!in_pool) return;
    // ---- V chunks (4 m + g, d), m the block's half of the page
    for (int i = tid; i < 4 * D; i += 256) {
        const int g = i / D, d = i - g * D;
        uint16_t *vp = (uint16_t *)p.v + at + ((size_t)(4 * ((pb >> 5) & 1) + g) * D + d) * 8;
        uint16_t y[8];
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] = s_v[v_chunk_pos(g, e)][d];
        if (v_chunk_pos(g, 0) >= r_lo && v_chunk_pos(g, 7) < r_hi) {
            *(uint4 *)vp = make_uint4(y[0] | (uint32_t)y[1] << 16, y[2] | (uint32_t)y[3] << 16, y[4] | (uint32_t)y[5] << 16,
                                      y[6] | (uint32_t)y[7] << 16);
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int r = v_chunk_pos(g, e);
                if (r >= r_lo && r < r_hi) vp[e] = y[e];
            }
        }
    }
}

template <typename T, typename IO>
void launch_rope(const hymt_paged &p, const hymt_batch &b, const RopeAppend &a, hipStream_t s) {
    KernelSpan span("rope_append", s, true);
    if (!b.cu || b.rows < kRopeFew || b.rows < kRopeFewEach * b.n) {
        if (p.head_dim == 64) launch(span, rope_row_kernel<T, IO, 64>, dim3(b.rows), dim3(256), 0, s, p, b, a);
        else launch(span, rope_row_kernel<T, IO, 128>, dim3(b.rows), dim3(256), 0, s, p, b, a);
        return;
    }
    // an entry's rows touch at most two blocks more than they fill
    const dim3 grid((unsigned)(((b.rows + kRopeRows - 1) / kRopeRows + 2 * b.n) * p.kv_heads));
    if (p.head_dim == 64) launch(span, rope_block_kernel<T, IO, 64>, grid, dim3(256), 0, s, p, b, a);
    else launch(span, rope_block_kernel<T, IO, 128>, grid, dim3(256), 0, s, p, b, a);
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
