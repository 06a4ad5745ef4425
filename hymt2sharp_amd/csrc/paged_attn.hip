// paged_attn.hip -- attention over the multi-sequence cache (hymt_paged,
// include/hymt_hip.h): a batch's packed rows, causal (hymt_attn_packed), and single
// rows behind a shared prefix (hymt_attn_shared).
//
// Rows.  The q heads of a kv head's group are rows of the same products: row r of
// an entry is its token r / G, head r % G (G q heads per kv head, any number), so
// every G fills the matrix instructions and each K/V page is read once for the
// group.
//
// tile part   (tile_part) a workgroup takes 128 rows of one kv head; each of its
//             4 waves 32 of them, two blocks of 16.  K and V pages go straight
//             into LDS (they hold their chunks in operand order), two pages deep; a
//             page's step is S^T = K Q^T, softmax in registers, O^T += V^T P^T on
//             v_mfma_f32_16x16x32: lane (grp, c) has row c's scores of positions
//             16 kb + 4 grp + [0, 4), which are its P operand as they stand.  The
//             running maximum moves only when a score passes it by 2^8.  Causal
//             for packed rows; the prefix of attn_shared is the same with the
//             rows of all entries and one kv range.
// row part    (row_part) one entry's G rows over its own pages: pages go
//             from memory straight into operand registers, a page to a wave.
// joining     where rows are few, a kv range is cut into parts whose (O, m, l) meet
//             in attn_merge, in fp32.
//
// Softmax: weights 2^(c s - m), c = scale log2 e, s the exact products' fp32 sums.
// Weights are rounded to the cache's type for the product with V and
// summed as rounded, so they sum to 1.
#include <algorithm>

#include "attn_kernels.hpp"
#include "device_common.hpp"
#include "ktimer.hpp"
#include "paged.hpp"

namespace hymt {

namespace {

typedef __bf16 pa_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 pa_f16x8 __attribute__((ext_vector_type(8)));
typedef float pa_f32x4 __attribute__((ext_vector_type(4)));

template <typename T> struct Mma;
template <> struct Mma<BF16> {
    typedef pa_bf16x8 vec;
    typedef __bf16 pair __attribute__((ext_vector_type(2)));
    static constexpr uint32_t kOnes = 0x3F803F80u, kInf = 0x7F80u;
    __device__ static __forceinline__ pa_f32x4 mma(vec a, vec b, pa_f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
    __device__ static __forceinline__ uint32_t pack(float x, float y) {
        pair r;
        r[0] = (__bf16)x;
        r[1] = (__bf16)y;
        return __builtin_bit_cast(uint32_t, r);
    }
    // acc + both halves
    __device__ static __forceinline__ float sum(uint32_t p, float acc) {
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(pair, p), __builtin_bit_cast(pair, kOnes), acc, false);
    }
};
template <> struct Mma<F16> {
    typedef pa_f16x8 vec;
    typedef _Float16 pair __attribute__((ext_vector_type(2)));
    static constexpr uint32_t kOnes = 0x3C003C00u, kInf = 0x7C00u;
    __device__ static __forceinline__ pa_f32x4 mma(vec a, vec b, pa_f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
    __device__ static __forceinline__ uint32_t pack(float x, float y) {
        pair r;
        r[0] = (_Float16)x;
        r[1] = (_Float16)y;
        return __builtin_bit_cast(uint32_t, r);
    }
    __device__ static __forceinline__ float sum(uint32_t p, float acc) {
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(pair, p), __builtin_bit_cast(pair, kOnes), acc, false);
    }
};

// The four 16-lane rows of a wave joined: every lane gets the result of its column.
__device__ __forceinline__ float rows_max(float v) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float rows_sum(float v) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ int wave_min(int v) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) v = min(v, __shfl_xor(v, m));
    return v;
}

constexpr int kRows = 128;         // rows of a tile
constexpr int kMinPages = 4;       // pages that a part of a split range has at least
constexpr int kMaxParts = 64;      // parts of a split range
constexpr float kLazyMax = 8.0f;   // weights stay below 2^8 of the running maximum's
constexpr float kNoMax = -1e30f;   // the maximum before any score: finite, so that -inf - m is -inf

struct Plan {
    hymt_paged p;
    hymt_batch b;
    const void *q;
    void *out;
    int heads, group, layer, prefix, out_f16;
    float c;          // |scale| log2 e; 0 is replaced by a number that makes every weight 1
    uint32_t flip;    // sign bits flipped in q where scale is negative
    int parts;        // parts that a kv range is cut into at most (prefix: of it)
    int own_parts;    // shared: parts of an entry's own range at most
    int direct;       // shared: no prefix and no split, the row part writes the output
    float *o, *ml;    // partials: [part][rows * heads][D], [part][rows * heads][2]
};

__device__ __forceinline__ int slot_len(const hymt_paged &p, int slot) {
    return (unsigned)slot < (unsigned)p.seqs ? max(0, min(p.len[slot], p.blocks * kPage)) : 0;
}
__device__ __forceinline__ int pages_of(int positions) { return (positions + kPage - 1) / kPage; }
// Parts that a range of `pages` is cut into, at most `most`.
__device__ __forceinline__ int parts_of(int pages, int most) { return max(1, min(most, pages / kMinPages)); }

// An entry's rows in the packed tensors, whatever cu holds: inside [0, rows).
struct Span {
    int first, n;
};
__device__ __forceinline__ Span span_of(const hymt_batch &b, int entry) {
    if (!b.cu) return {entry, 1};
    const int lo = max(0, min(b.cu[entry], b.rows));
    return {lo, max(lo, min(b.cu[entry + 1], b.rows)) - lo};
}

// What a tile's rows attend to: row r (token r / group) sees the positions below
// limit(r).
struct Rows {
    int first;   // first packed row
    int n;       // rows: tokens * group
    int seen;    // positions that the entry's first token attends to (may be negative)
};

template <typename T>
__device__ __forceinline__ void put4(const Plan &a, size_t at, float x, float y, float z, float w) {
    uint2 u;
    if (a.out_f16) u = make_uint2(Mma<F16>::pack(x, y), Mma<F16>::pack(z, w));
    else u = make_uint2(Mma<BF16>::pack(x, y), Mma<BF16>::pack(z, w));
    *(uint2 *)((uint16_t *)a.out + at) = u;
}

// LDS reads ahead of the products that use them: DEPTH in flight, then one more
// after every operand's two products.
template <int READS> __device__ __forceinline__ void read_ahead() {
    constexpr int DEPTH = 6;
    __builtin_amdgcn_sched_group_barrier(0x100, DEPTH, 0);
#pragma unroll
    for (int i = 0; i < READS - DEPTH; i++) {
        __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, 2 * DEPTH, 0);
}

template <int D> struct TileLds {
    uint16_t kv[2][2][kPage * D];  // [buffer][K, V][page]
    int flag[2];                   // a value that is not finite was seen in V, by buffer
    int low[4];                    // lowest limit of each wave's rows
};

// 128 rows of kv head h over pages [t0, t1) of `slot`.  PREFIX: row r is entry
// r / G's, its limit min(common, that entry's length), the result a partial.
template <typename T, int D, bool PREFIX>
__device__ __forceinline__ void tile_part(const Plan &a, TileLds<D> &s, int h, int slot, int slot_positions, Rows rows,
                                          int r0, int t0, int t1, int part, bool partial) {
    typedef typename Mma<T>::vec vec;
    constexpr int KS = D / 32, DB = D / 16, kPageBytes = kPage * D * 2;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int grp = lane >> 4, c = lane & 15;

    // ---- pages: lane i has the page of tile (base & ~63) + i
    const int32_t *table = a.p.table + (size_t)slot * a.p.blocks;
    int ids = -1, ids_at = -1;
    auto page_of = [&](int t) __attribute__((always_inline)) {
        if ((t & ~63) != ids_at) {  // uniform
            ids_at = t & ~63;
            ids = ids_at + lane < t1 ? table[ids_at + lane] : -1;
        }
        const int page = __builtin_amdgcn_readlane(ids, t & 63);
        return (unsigned)page < (unsigned)a.p.pages ? page : -1;
    };
    const uint32_t off = (wave * 64 + lane) * 16;
    const uint32_t lds0 = lds_addr(&s.kv[0][0][0]) + wave * 1024;
    auto fetch = [&](int page, int buf, int v) __attribute__((always_inline)) {
        const char *base = (const char *)(v ? a.p.v : a.p.k) +
                           (((size_t)a.layer * a.p.pages + page) * a.p.kv_heads + h) * (size_t)kPageBytes;
#pragma unroll
        for (int i = 0; i < kPageBytes / 4096; i++)
            lds_dma16_sv(base + i * 4096, off, lds0 + (buf * 2 + v) * kPageBytes + i * 4096);
    };

    int page = t0 < t1 ? page_of(t0) : -1;
    if (page >= 0) {
        fetch(page, 0, 0);
        fetch(page, 0, 1);
    }

    // ---- the wave's rows: q as the S^T B operand, lane (grp, c) has dims
    // 32 ks + 8 grp + [0, 8) of row c; rows past the end repeat the last one
    int limit[2];
    size_t at[2];  // element of (row, head) in q and out
    uint4 qu[2][KS];
#pragma unroll
    for (int qq = 0; qq < 2; qq++) {
        const int r = min(r0 + wave * 32 + qq * 16 + c, rows.n - 1);
        const int token = r / a.group, g = r - token * a.group;
        at[qq] = ((size_t)(rows.first + token) * a.heads + h * a.group + g) * D;
#pragma unroll
        for (int ks = 0; ks < KS; ks++) qu[qq][ks] = *(const uint4 *)((const uint16_t *)a.q + at[qq] + 32 * ks + 8 * grp);
        if constexpr (PREFIX) limit[qq] = min(slot_positions, slot_len(a.p, a.b.slots[token]));
        else limit[qq] = min(rows.seen + token, slot_positions);
    }
    vec qf[2][KS];
#pragma unroll
    for (int qq = 0; qq < 2; qq++)
#pragma unroll
        for (int ks = 0; ks < KS; ks++)
            qf[qq][ks] = __builtin_bit_cast(vec, make_uint4(qu[qq][ks].x ^ a.flip, qu[qq][ks].y ^ a.flip,
                                                            qu[qq][ks].z ^ a.flip, qu[qq][ks].w ^ a.flip));
    // lowest limits: of the wave's blocks, and of the tile
    int low[2];
#pragma unroll
    for (int qq = 0; qq < 2; qq++) low[qq] = __builtin_amdgcn_readfirstlane(wave_min(limit[qq]));
    if (lane == 0) s.low[wave] = min(low[0], low[1]);
    if (tid < 2) s.flag[tid] = 0;

    const bool live = r0 + wave * 32 < rows.n;  // the wave has a row
    pa_f32x4 o[DB][2];
#pragma unroll
    for (int db = 0; db < DB; db++)
#pragma unroll
        for (int qq = 0; qq < 2; qq++) o[db][qq] = pa_f32x4{0.f, 0.f, 0.f, 0.f};
    float m[2] = {kNoMax, kNoMax}, l[2] = {0.f, 0.f};  // m in units of c s; l this lane's share

    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    const int tile_low = min(min(s.low[0], s.low[1]), min(s.low[2], s.low[3]));

    for (int t = t0; t < t1; t++) {
        const int buf = (t - t0) & 1, base = t * kPage;
        const int next = t + 1 < t1 ? page_of(t + 1) : -1;
        const uint16_t *kt = s.kv[buf][0] + lane * 8, *vt = s.kv[buf][1] + grp * (D * 8) + c * 8;
        if (next >= 0) fetch(next, buf ^ 1, 0);
        bool odd = false;
        if (page >= 0 && base + kPage > tile_low) {
            // Some row does not see some position of this page.  Its weight is 0
            // there, and 0 times an infinity or a NaN is none: values past the
            // sequence's end (anything may stand there) become 0 in LDS, and
            // if others are not finite the products leave them out (below).
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < kPage * D / 8 / 256; i++) {
                const int ch = tid + 256 * i, pc = ch / D;
                uint4 *at_v = (uint4 *)s.kv[buf][1] + ch;
                uint4 u = *at_v;
                uint32_t w[4] = {u.x, u.y, u.z, u.w};
                if (!PREFIX && base + kPage > slot_positions) {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int p0 = base + v_chunk_pos(pc, 2 * e);
                        if (p0 + 1 >= slot_positions) w[e] &= 0xFFFFu;
                        if (p0 >= slot_positions) w[e] = 0;
                    }
                    *at_v = make_uint4(w[0], w[1], w[2], w[3]);
                }
#pragma unroll
                for (int e = 0; e < 4; e++) top = max(top, max(w[e] & 0x7FFFu, w[e] >> 16 & 0x7FFFu));
            }
            if (top >= Mma<T>::kInf) s.flag[buf] = 1;
            __syncthreads();
            odd = s.flag[buf] != 0;
        }
        if (page >= 0 && live) {
            // ---- S^T = K Q^T, 64 positions x 16 rows a block
            pa_f32x4 sc[4][2];
#pragma unroll
            for (int kb = 0; kb < 4; kb++)
#pragma unroll
                for (int qq = 0; qq < 2; qq++) sc[kb][qq] = pa_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
#pragma unroll
                for (int kb = 0; kb < 4; kb++) {
                    const vec kf = __builtin_bit_cast(vec, *(const uint4 *)(kt + kb * (16 * D) + ks * 512));
#pragma unroll
                    for (int qq = 0; qq < 2; qq++) sc[kb][qq] = Mma<T>::mma(kf, qf[qq][ks], sc[kb][qq]);
                }
            read_ahead<4 * KS>();
            if (next >= 0) fetch(next, buf ^ 1, 1);

            // ---- softmax
            float mx[2];
#pragma unroll
            for (int qq = 0; qq < 2; qq++) {
                if (base + kPage > low[qq]) {
#pragma unroll
                    for (int kb = 0; kb < 4; kb++)
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            if (base + 16 * kb + 4 * grp + i >= limit[qq]) sc[kb][qq][i] = -INFINITY;
                }
                float v = sc[0][qq][0];
#pragma unroll
                for (int kb = 0; kb < 4; kb++)
#pragma unroll
                    for (int i = 0; i < 4; i++) v = fmaxf(v, sc[kb][qq][i]);
                mx[qq] = v * a.c;
            }
            if (__any(mx[0] > m[0] + kLazyMax || mx[1] > m[1] + kLazyMax)) {
#pragma unroll
                for (int qq = 0; qq < 2; qq++) {
                    const float now = fmaxf(m[qq], rows_max(mx[qq]));
                    const float al = __builtin_amdgcn_exp2f(m[qq] - now);
                    m[qq] = now;
                    l[qq] *= al;
#pragma unroll
                    for (int db = 0; db < DB; db++) o[db][qq] *= al;
                }
            }
#pragma unroll
            for (int kb = 0; kb < 4; kb++)
#pragma unroll
                for (int qq = 0; qq < 2; qq++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        sc[kb][qq][i] = __builtin_amdgcn_exp2f(fmaf(sc[kb][qq][i], a.c, -m[qq]));

            // ---- O^T += V^T P^T
            vec pf[2][2];
#pragma unroll
            for (int k2 = 0; k2 < 2; k2++)
#pragma unroll
                for (int qq = 0; qq < 2; qq++) {
                    const pa_f32x4 x = sc[2 * k2][qq], y = sc[2 * k2 + 1][qq];
                    const uint4 u = make_uint4(Mma<T>::pack(x[0], x[1]), Mma<T>::pack(x[2], x[3]),
                                               Mma<T>::pack(y[0], y[1]), Mma<T>::pack(y[2], y[3]));
                    l[qq] = Mma<T>::sum(u.w, Mma<T>::sum(u.z, Mma<T>::sum(u.y, Mma<T>::sum(u.x, l[qq]))));
                    pf[k2][qq] = __builtin_bit_cast(vec, u);
                }
            if (!odd) {
#pragma unroll
                for (int k2 = 0; k2 < 2; k2++)
#pragma unroll
                    for (int db = 0; db < DB; db++) {
                        const vec vf = __builtin_bit_cast(vec, *(const uint4 *)(vt + k2 * (4 * D * 8) + db * 128));
#pragma unroll
                        for (int qq = 0; qq < 2; qq++) o[db][qq] = Mma<T>::mma(vf, pf[k2][qq], o[db][qq]);
                    }
                read_ahead<2 * DB>();
            } else {
                // the products without the values that are not finite ...
#pragma unroll
                for (int k2 = 0; k2 < 2; k2++)
#pragma unroll
                    for (int db = 0; db < DB; db++) {
                        const uint4 u = *(const uint4 *)(vt + k2 * (4 * D * 8) + db * 128);
                        uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            if ((w[e] & 0x7FFFu) >= Mma<T>::kInf) w[e] &= 0xFFFF0000u;
                            if ((w[e] >> 16 & 0x7FFFu) >= Mma<T>::kInf) w[e] &= 0xFFFFu;
                        }
                        const vec vf = __builtin_bit_cast(vec, make_uint4(w[0], w[1], w[2], w[3]));
#pragma unroll
                        for (int qq = 0; qq < 2; qq++) o[db][qq] = Mma<T>::mma(vf, pf[k2][qq], o[db][qq]);
                    }
                // ... and those to the rows that see them (their weight is
                // positive, so the result is the value)
                for (int pos = 0; pos < kPage; pos++) {
                    const int pc = 4 * (pos >> 5) + ((pos >> 2) & 3), e = 4 * ((pos >> 4) & 1) + (pos & 3);
                    const uint16_t *v = s.kv[buf][1] + (size_t)pc * (D * 8) + e;
#pragma unroll
                    for (int db = 0; db < DB; db++)
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const uint16_t x = v[(16 * db + 4 * grp + i) * 8];
                            if ((x & 0x7FFFu) >= Mma<T>::kInf)
#pragma unroll
                                for (int qq = 0; qq < 2; qq++)
                                    if (base + pos < limit[qq]) o[db][qq][i] += from_elem<T>(x);
                        }
                }
            }
        } else if (next >= 0) {
            fetch(next, buf ^ 1, 1);
        }
        page = next;
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
        if (odd && tid == 0) s.flag[buf] = 0;  // every wave has read it; the next that sets it does so two steps on
    }

#pragma unroll
    for (int qq = 0; qq < 2; qq++) {
        l[qq] = rows_sum(l[qq]);
        if (r0 + wave * 32 + qq * 16 + c >= rows.n) continue;
        if (partial) {
            const size_t rh = at[qq] / D + (size_t)part * a.b.rows * a.heads;
            float *po = a.o + rh * D + 4 * grp;
#pragma unroll
            for (int db = 0; db < DB; db++) *(pa_f32x4 *)(po + 16 * db) = o[db][qq];
            if (grp == 0) *(float2 *)(a.ml + rh * 2) = make_float2(m[qq], l[qq]);
        } else {
            const float inv = l[qq] == 0.f ? 0.f : 1.0f / l[qq];
#pragma unroll
            for (int db = 0; db < DB; db++) {
                const pa_f32x4 y = o[db][qq] * inv;
                put4<T>(a, at[qq] + 16 * db + 4 * grp, y[0], y[1], y[2], y[3]);
            }
        }
    }
}

// The tile that work index w is of: its entry, place and number there.  Tiles of
// an entry come last first, so that the longest kv ranges start first.
struct Tile {
    int entry, index, slot, len;
    Span span;
};
__device__ __forceinline__ bool find_tile(const Plan &a, int w, Tile &out) {
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int base = 0; base < a.b.n; base += 64) {
        const int i = base + lane;
        Span sp{0, 0};
        int slot = -1;
        if (i < a.b.n) {
            sp = span_of(a.b, i);
            slot = a.b.slots[i];
        }
        const int len = slot_len(a.p, slot);  // for every entry: one load deep, not one more after the search
        const int tiles = (sp.n * a.group + kRows - 1) / kRows;
        int x = tiles;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int y = __shfl_up(x, d);
            if (lane >= d) x += y;
        }
        const uint64_t hit = __ballot(w < before + x);
        if (hit) {
            const int at = __ffsll((unsigned long long)hit) - 1;
            out.entry = base + at;
            const int count = __builtin_amdgcn_readlane(tiles, at);
            const int first = before + __builtin_amdgcn_readlane(x, at) - count;
            out.index = count - 1 - (w - first);
            out.slot = __builtin_amdgcn_readlane(slot, at);
            out.len = __builtin_amdgcn_readlane(len, at);
            out.span = {__builtin_amdgcn_readlane(sp.first, at), __builtin_amdgcn_readlane(sp.n, at)};
            return true;
        }
        before += __builtin_amdgcn_readlane(x, 63);
    }
    return false;
}

// Pages that a tile of an entry attends to.
__device__ __forceinline__ int tile_pages(int len, Span sp, int index, int group) {
    const int last = min(sp.n - 1, (min((index + 1) * kRows, sp.n * group) - 1) / group);
    return pages_of(max(0, min(len, len - sp.n + last + 1)));
}

template <typename T, int D> __global__ __launch_bounds__(256, 2) void attn_packed_kernel(Plan a) {
    __shared__ __attribute__((aligned(256))) TileLds<D> s;
    // workgroups of one kv head on the same XCDs (workgroup b runs on XCD
    // b % 8), whose L2 then holds that head's pages
    const int h = blockIdx.x % a.p.kv_heads, rest = blockIdx.x / a.p.kv_heads;
    const int part = rest % a.parts;
    Tile t;
    if (!find_tile(a, rest / a.parts, t)) return;
    const int pages = tile_pages(t.len, t.span, t.index, a.group), parts = parts_of(pages, a.parts);
    if (part >= parts) return;
    const Rows rows{t.span.first, t.span.n * a.group, t.len - t.span.n + 1};
    const int slot = max(0, t.slot);  // an unknown slot has no pages
    tile_part<T, D, false>(a, s, h, slot, t.len, rows, t.index * kRows, (int)((long)part * pages / parts),
                           (int)((long)(part + 1) * pages / parts), part, parts > 1);
}

// ---- single rows -------------------------------------------------------------------

template <int D> struct RowLds {
    float o[4][16][D + 4];
    float m[4][16], l[4][16];
};

// Up to 16 rows (heads g0 ..) of one entry over pages [t0, t1) of its slot, a page to
// a wave: K and V go from memory into operand registers.
template <typename T, int D>
__device__ __forceinline__ void row_part(const Plan &a, RowLds<D> &s, int entry, int h, int g0, int slot, int len, int t0,
                                         int t1, int part, bool partial) {
    typedef typename Mma<T>::vec vec;
    constexpr int KS = D / 32, DB = D / 16;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int grp = lane >> 4, c = lane & 15;
    const int g = min(g0 + c, a.group - 1);
    const size_t at = ((size_t)entry * a.heads + h * a.group + g) * D;
    vec qf[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ks++) {
        const uint4 u = *(const uint4 *)((const uint16_t *)a.q + at + 32 * ks + 8 * grp);
        qf[ks] = __builtin_bit_cast(vec, make_uint4(u.x ^ a.flip, u.y ^ a.flip, u.z ^ a.flip, u.w ^ a.flip));
    }
    pa_f32x4 o[DB];
#pragma unroll
    for (int db = 0; db < DB; db++) o[db] = pa_f32x4{0.f, 0.f, 0.f, 0.f};
    float m = kNoMax, l = 0.f;
    const int32_t *table = a.p.table + (size_t)slot * a.p.blocks;
    for (int t = t0 + wave; t < t1; t += 4) {
        const int page = __builtin_amdgcn_readfirstlane(table[t]);
        if ((unsigned)page >= (unsigned)a.p.pages) continue;
        const size_t base = (((size_t)a.layer * a.p.pages + page) * a.p.kv_heads + h) * (size_t)(kPage * D);
        const uint16_t *kp = (const uint16_t *)a.p.k + base + lane * 8;
        const uint16_t *vp = (const uint16_t *)a.p.v + base + grp * (D * 8) + c * 8;
        uint4 ku[KS][4], vu[2][DB];
#pragma unroll
        for (int ks = 0; ks < KS; ks++)
#pragma unroll
            for (int kb = 0; kb < 4; kb++) ku[ks][kb] = *(const uint4 *)(kp + kb * (16 * D) + ks * 512);
#pragma unroll
        for (int k2 = 0; k2 < 2; k2++)
#pragma unroll
            for (int db = 0; db < DB; db++) vu[k2][db] = *(const uint4 *)(vp + k2 * (4 * D * 8) + db * 128);
        pa_f32x4 sc[4];
#pragma unroll
        for (int kb = 0; kb < 4; kb++) sc[kb] = pa_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ks++)
#pragma unroll
            for (int kb = 0; kb < 4; kb++) sc[kb] = Mma<T>::mma(__builtin_bit_cast(vec, ku[ks][kb]), qf[ks], sc[kb]);
        const int left = len - t * kPage;  // positions of this page
        if (left < kPage) {
#pragma unroll
            for (int kb = 0; kb < 4; kb++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (16 * kb + 4 * grp + i >= left) sc[kb][i] = -INFINITY;
            // anything may stand past the end: 0 weights have to meet 0
#pragma unroll
            for (int k2 = 0; k2 < 2; k2++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int p0 = v_chunk_pos(4 * k2 + grp, 2 * e);
                    const uint32_t keep = p0 >= left ? 0u : p0 + 1 >= left ? 0xFFFFu : 0xFFFFFFFFu;
#pragma unroll
                    for (int db = 0; db < DB; db++) ((uint32_t *)&vu[k2][db])[e] &= keep;
                }
        }
        float v = sc[0][0];
#pragma unroll
        for (int kb = 0; kb < 4; kb++)
#pragma unroll
            for (int i = 0; i < 4; i++) v = fmaxf(v, sc[kb][i]);
        const float now = fmaxf(m, rows_max(v) * a.c), al = __builtin_amdgcn_exp2f(m - now);
        m = now;
        l *= al;
#pragma unroll
        for (int db = 0; db < DB; db++) o[db] *= al;
#pragma unroll
        for (int kb = 0; kb < 4; kb++)
#pragma unroll
            for (int i = 0; i < 4; i++) sc[kb][i] = __builtin_amdgcn_exp2f(fmaf(sc[kb][i], a.c, -m));
#pragma unroll
        for (int k2 = 0; k2 < 2; k2++) {
            const pa_f32x4 x = sc[2 * k2], y = sc[2 * k2 + 1];
            const uint4 u = make_uint4(Mma<T>::pack(x[0], x[1]), Mma<T>::pack(x[2], x[3]), Mma<T>::pack(y[0], y[1]),
                                       Mma<T>::pack(y[2], y[3]));
            l = Mma<T>::sum(u.w, Mma<T>::sum(u.z, Mma<T>::sum(u.y, Mma<T>::sum(u.x, l))));
#pragma unroll
            for (int db = 0; db < DB; db++)
                o[db] = Mma<T>::mma(__builtin_bit_cast(vec, vu[k2][db]), __builtin_bit_cast(vec, u), o[db]);
        }
    }
    l = rows_sum(l);
    // ---- the four waves' results meet in LDS
#pragma unroll
    for (int db = 0; db < DB; db++) *(pa_f32x4 *)&s.o[wave][c][16 * db + 4 * grp] = o[db];
    if (grp == 0) {
        s.m[wave][c] = m;
        s.l[wave][c] = l;
    }
    __syncthreads();
    // 16 threads a row, 4 dims each at a time
    const int row = tid >> 4, d0 = 4 * (tid & 15);
    if (g0 + row >= a.group) return;
    float top = s.m[0][row], sum = 0.f, w[4];
#pragma unroll
    for (int k = 1; k < 4; k++) top = fmaxf(top, s.m[k][row]);
#pragma unroll
    for (int k = 0; k < 4; k++) {
        w[k] = __builtin_amdgcn_exp2f(s.m[k][row] - top);
        sum += w[k] * s.l[k][row];
    }
    const size_t rh = (size_t)entry * a.heads + h * a.group + g0 + row;
    const float inv = partial ? 1.0f : sum == 0.f ? 0.f : 1.0f / sum;
#pragma unroll
    for (int d = d0; d < D; d += 64) {
        pa_f32x4 y{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < 4; k++) y += *(const pa_f32x4 *)&s.o[k][row][d] * w[k];
        y *= inv;
        if (partial) *(pa_f32x4 *)(a.o + ((size_t)part * a.b.rows * a.heads + rh) * D + d) = y;
        else put4<T>(a, rh * D + d, y[0], y[1], y[2], y[3]);
    }
    if (partial && d0 == 0) *(float2 *)(a.ml + ((size_t)part * a.b.rows * a.heads + rh) * 2) = make_float2(top, sum);
}

// Positions that all entries read from slots[0]'s pages.
__device__ __forceinline__ int common_of(const Plan &a) {
    return a.prefix ? min(a.prefix, slot_len(a.p, a.b.slots[0]) / kPage * kPage) : 0;
}

// Workgroups [0, tile_wgs) the prefix, the others the entries' own positions.
template <typename T, int D> __global__ __launch_bounds__(256, 2) void attn_shared_kernel(Plan a, int tile_wgs) {
    __shared__ __attribute__((aligned(256))) union {
        TileLds<D> tile;
        RowLds<D> row;
    } s;
    const int common = common_of(a);
    if ((int)blockIdx.x < tile_wgs) {
        const int h = blockIdx.x % a.p.kv_heads, rest = blockIdx.x / a.p.kv_heads;
        const int pages = common / kPage, parts = parts_of(pages, a.parts), part = rest % a.parts;
        if (part >= parts || pages == 0) return;
        tile_part<T, D, true>(a, s.tile, h, a.b.slots[0], common, Rows{0, a.b.n * a.group, 0}, rest / a.parts * kRows,
                              (int)((long)part * pages / parts), (int)((long)(part + 1) * pages / parts), part, true);
        return;
    }
    int w = blockIdx.x - tile_wgs;
    const int h = w % a.p.kv_heads;
    w /= a.p.kv_heads;
    const int blocks16 = (a.group + 15) / 16;
    const int g0 = w % blocks16 * 16;
    w /= blocks16;
    const int part = w % a.own_parts, entry = w / a.own_parts;
    const int slot = a.b.slots[entry], len = slot_len(a.p, slot);
    const int first = common / kPage, pages = max(0, pages_of(len) - first), parts = parts_of(pages, a.own_parts);
    if (part >= parts) return;
    row_part<T, D>(a, s.row, entry, h, g0, max(0, slot), len, first + (int)((long)part * pages / parts),
                   first + (int)((long)(part + 1) * pages / parts), a.parts + part, !a.direct);
}

// ---- joining -----------------------------------------------------------------------

// A wave a row of one head: the parts' sums, weighed by their maxima.
template <typename T, int D, bool SHARED> __global__ __launch_bounds__(256) void attn_merge_kernel(Plan a) {
    const int lane = threadIdx.x & 63;
    const int rh = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row = rh / a.heads;
    if (row >= a.b.rows) return;
    int n0 = 0, n1 = 0;  // parts [0, n0) and [a.parts, a.parts + n1)
    if constexpr (SHARED) {
        const int common = common_of(a), len = slot_len(a.p, a.b.slots[row]);
        if (common) n0 = parts_of(common / kPage, a.parts);
        n1 = parts_of(max(0, pages_of(len) - common / kPage), a.own_parts);
    } else {
        int below = 0;
        if (a.b.cu) {
            for (int base = 0; base < a.b.n; base += 64) {
                const int i = base + lane;
                below += __popcll(__ballot(i < a.b.n && a.b.cu[i + 1] <= row));
            }
        } else {
            below = row;
        }
        if (below >= a.b.n) return;
        const Span sp = a.b.cu ? span_of(a.b, below) : Span{row, 1};
        if (row < sp.first || row >= sp.first + sp.n) return;
        const int index = ((row - sp.first) * a.group + rh % a.heads % a.group) / kRows;
        n0 = parts_of(tile_pages(slot_len(a.p, a.b.slots[below]), sp, index, a.group), a.parts);
        if (n0 == 1) return;  // written by its tile
    }
    const size_t stride = (size_t)a.b.rows * a.heads;
    const int total = n0 + n1;
    float top = kNoMax, sum = 0.f;
    auto index_of = [&](int k) { return (size_t)(k < n0 ? k : a.parts + k - n0) * stride + rh; };
    for (int base = 0; base < total; base += 64) {
        float2 x = make_float2(kNoMax, 0.f);
        if (base + lane < total) x = *(const float2 *)(a.ml + index_of(base + lane) * 2);
        float mx = x.x;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) mx = fmaxf(mx, __shfl_xor(mx, d));
        const float now = fmaxf(top, mx);
        float w = x.y * __builtin_amdgcn_exp2f(x.x - now);
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) w += __shfl_xor(w, d);
        sum = sum * __builtin_amdgcn_exp2f(top - now) + w;
        top = now;
    }
    // 4 dims a lane, D / 4 lanes a part, several parts at a time
    constexpr int L = D / 4, S = 64 / L;
    pa_f32x4 acc{0.f, 0.f, 0.f, 0.f};
    for (int k = lane / L; k < total; k += S) {
        const size_t i = index_of(k);
        const float w = __builtin_amdgcn_exp2f(a.ml[i * 2] - top);
        acc += *(const pa_f32x4 *)(a.o + i * D + 4 * (lane % L)) * w;
    }
#pragma unroll
    for (int d = L; d < 64; d <<= 1)
#pragma unroll
        for (int e = 0; e < 4; e++) acc[e] += __shfl_xor(acc[e], d);
    const float inv = sum == 0.f ? 0.f : 1.0f / sum;
    if (lane < L) put4<T>(a, (size_t)rh * D + 4 * lane, acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
}

// ---- host --------------------------------------------------------------------------

constexpr int kSlots = 512;  // tile workgroups that the chip holds at once, two a CU

struct Shape {
    int tiles, parts, own, blocks16;
};
int ceil_div(long a, long b) { return (int)((a + b - 1) / b); }

Shape shape_of(const hymt_paged &p, const hymt_batch &b, const PagedAttn &a, bool shared) {
    const int group = a.heads / p.kv_heads;
    const int longest = b.max_len > 0 ? std::min<long>(b.max_len, (long)p.blocks * kPage) : p.blocks * kPage;
    Shape s{0, 1, 1, (group + 15) / 16};
    auto cut = [&](int wgs, int pages) {  // parts that fill the chip
        return std::max(1, std::min({kSlots / std::max(wgs, 1), pages / kMinPages, kMaxParts}));
    };
    if (shared) {
        const int common = std::min(a.prefix, longest) / kPage;
        s.tiles = a.prefix ? ceil_div((long)b.n * group, kRows) : 0;
        if (s.tiles) s.parts = cut(s.tiles * p.kv_heads, common);
        s.own = cut(b.n * p.kv_heads * s.blocks16, ceil_div(longest, kPage) - common);
    } else {
        const long rows = b.cu ? (long)b.rows * group / kRows + b.n : (long)b.n * ceil_div(group, kRows);
        s.tiles = (int)rows;
        s.parts = cut(s.tiles * p.kv_heads, ceil_div(longest, kPage));
    }
    return s;
}

Plan plan_of(const hymt_paged &p, const hymt_batch &b, const PagedAttn &a, const Shape &s, float *ws) {
    Plan r{};
    r.p = p;
    r.b = b;
    r.q = a.q;
    r.out = a.out;
    r.heads = a.heads;
    r.group = a.heads / p.kv_heads;
    r.layer = a.layer;
    r.prefix = a.prefix;
    r.out_f16 = a.out_dtype == HYMT_F16;
    r.c = std::max(std::abs(a.scale) * 1.4426950408889634f, 1e-30f);
    r.flip = a.scale < 0 ? 0x80008000u : 0u;
    r.parts = s.parts;
    r.own_parts = s.own;
    const size_t rh = (size_t)b.rows * a.heads;
    r.o = ws;
    r.ml = ws + (size_t)(s.parts + s.own) * rh * p.head_dim;
    return r;
}

template <typename K> void launch_merge(K k, const Plan &a, hipStream_t s) {
    KernelSpan span("attn_merge", s, true);
    launch(span, k, dim3((unsigned)(((size_t)a.b.rows * a.heads + 3) / 4)), dim3(256), 0, s, a);
}

template <typename T, int D> void packed(const Plan &a, const Shape &s, hipStream_t st) {
    {
        KernelSpan span("attn_packed", st, true);
        launch(span, attn_packed_kernel<T, D>, dim3(s.tiles * s.parts * a.p.kv_heads), dim3(256), 0, st, a);
    }
    if (s.parts > 1) launch_merge(attn_merge_kernel<T, D, false>, a, st);
}

template <typename T, int D> void shared(Plan a, const Shape &s, hipStream_t st) {
    const int tile_wgs = s.tiles * s.parts * a.p.kv_heads, row_wgs = a.b.n * a.p.kv_heads * s.blocks16 * s.own;
    a.direct = s.tiles == 0 && s.own == 1;
    if (s.tiles == 0) a.parts = 0;
    {
        KernelSpan span("attn_shared", st, true);
        launch(span, attn_shared_kernel<T, D>, dim3(tile_wgs + row_wgs), dim3(256), 0, st, a, tile_wgs);
    }
    if (!a.direct) launch_merge(attn_merge_kernel<T, D, true>, a, st);
}

}  // namespace

size_t paged_attn_workspace(const hymt_paged &p, const hymt_batch &b, const PagedAttn &a, bool shared) {
    if (b.n == 0 || b.rows == 0) return 0;
    const Shape s = shape_of(p, b, a, shared);
    if (shared ? s.tiles == 0 && s.own == 1 : s.parts == 1) return 0;
    return (size_t)(s.parts + s.own) * b.rows * a.heads * (p.head_dim + 2);
}

hipError_t launch_attn_packed(const hymt_paged &p, const hymt_batch &b, const PagedAttn &a, float *ws, hipStream_t st) {
    if (b.n == 0 || b.rows == 0) return hipSuccess;
    const Shape s = shape_of(p, b, a, false);
    const Plan r = plan_of(p, b, a, s, ws);
    if (p.dtype == HYMT_F16) p.head_dim == 64 ? packed<F16, 64>(r, s, st) : packed<F16, 128>(r, s, st);
    else p.head_dim == 64 ? packed<BF16, 64>(r, s, st) : packed<BF16, 128>(r, s, st);
    return hipGetLastError();
}

hipError_t launch_attn_shared(const hymt_paged &p, const hymt_batch &b, const PagedAttn &a, float *ws, hipStream_t st) {
    if (b.n == 0) return hipSuccess;
    const Shape s = shape_of(p, b, a, true);
    const Plan r = plan_of(p, b, a, s, ws);
    if (p.dtype == HYMT_F16) p.head_dim == 64 ? shared<F16, 64>(r, s, st) : shared<F16, 128>(r, s, st);
    else p.head_dim == 64 ? shared<BF16, 64>(r, s, st) : shared<BF16, 128>(r, s, st);
    return hipGetLastError();
}

}  // namespace hymt
