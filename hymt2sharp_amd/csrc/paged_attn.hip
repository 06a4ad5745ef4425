// paged_attn.hip -- attention over the multi-sequence cache (hymt_paged,
// include/hymt_hip.h): a batch's packed rows, causal (hymt_attn_packed), and single
// rows behind a shared prefix (hymt_attn_shared).
//
// Rows.  The q heads of a kv head's group are rows of the same products: row r of
// an entry is its token r / G, head r % G (G q heads per kv head, any number), so
// every G fills the matrix instructions and each K/V page is read once for the
// group.
//
// tile part   (tile_part) a workgroup takes 64 or 128 rows of one kv head; each of its
//             4 waves one or two blocks of 16.  K and V pages go straight
//             into LDS (they hold their chunks in operand order), two pages deep; a
//             page's step is S^T = K Q^T, softmax in registers, O^T += V^T P^T on
//             v_mfma_f32_16x16x32: lane (grp, c) has row c's scores of positions
//             16 kb + 4 grp + [0, 4), which are its P operand as they stand.  The
//             running maximum moves only when a score passes it by 2^8.  Causal
//             for packed rows; the prefix of attn_shared is the same with the
//             rows of all entries and one kv range.  With two groups of four waves
//             the groups take every other page and meet in LDS.
//               A step of two tiles of 128 rows on a CU takes 2 us: 0.9 of products, as
//             much of exponentials and other vector work, which hardly run beside the
//             products (a wave of 4 fmas to a product took 10.1 ns a product, products
//             alone 6.8, fmas alone 4.4), and LDS reads of 32 KB a wave.  One prompt of
//             8192: 235-243 us, 1.13-1.17 PFLOP/s; four of 4096 to 8192: 495, 1.10.  Not
//             kept: the next page's S beside this one's weights (48 -> 49-56 us at
//             2048), tiles of 192 rows, one to a CU (495 -> 840).
// row part    (row_part) one entry's G rows over its own pages, and those of the prefix
//             where sequences are short: pages go from memory straight into operand
//             registers, a page to a wave, the next page's as soon as the products have
//             read these.  Bound by memory:
//             64 rows over 2048 positions each 48-49 us, 5.5 TB/s.
// joining     where rows are few, a kv range is cut into parts whose (O, m, l) meet
//             in a second launch, in fp32: 4 to 7 us, most of it the launch (64 rows behind 4096
//             10 MB of partials in 5.1 us).
//
// Softmax: weights 2^(c s - m), c = scale log2 e, s the exact products' fp32 sums.
// Weights are rounded to the cache's type for the product with V and
// summed as rounded, so they sum to 1.
#include <algorithm>
#include <limits>

#include "attn_kernels.hpp"
#include "device_common.hpp"
#include "ktimer.hpp"
#include "paged.hpp"
#include "paged_split.hpp"

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
constexpr float kLazyMax = 8.0f;   // weights stay below 2^8 of the running maximum's
constexpr float kNoMax = -3.4028234e38f;  // the maximum before any score: finite, so that -inf - m is -inf
// c s - m in one fma has the rounding of m = c max s left over, |m| 2^-25 of a power of
// 2: from here on (2^-13) the product is rounded first, so that it is 0 where s is the
// maximum, in every part of a range
constexpr float kFarMax = 4096.f;
__device__ __forceinline__ float product_less(float x, float y, float z) {
#pragma clang fp contract(off)
    return x * y - z;
}

struct Plan {
    hymt_paged p;
    hymt_batch b;
    const void *q;
    void *out;
    int heads, group, layer, prefix, out_f16;
    float c;          // |scale| log2 e; 0 is replaced by a number that makes every weight 1
    uint32_t flip;    // sign bits flipped in q where scale is negative
    int parts, span;  // a kv range (shared: the prefix) is cut into parts of about `span` pages, `parts` at most
    int own_parts, own_span;  // shared: the same of an entry's own range
    int tiles;        // tiles of one kv head, at most
    int tile_rows;    // 64 or 128
    int direct;       // shared: no tiles and no split, the row part writes the output
    float *o, *ml;    // partials: [part][rows * heads][D], [part][rows * heads][2]
};

__device__ __forceinline__ int slot_len(const hymt_paged &p, int slot) {
    return (unsigned)slot < (unsigned)p.seqs ? max(0, min(p.len[slot], p.blocks * kPage)) : 0;
}
__device__ __forceinline__ int pages_of(int positions) { return (positions + kPage - 1) / kPage; }
// Parts of about `span` pages that a range of `pages` is cut into, at most `most`.
__device__ __forceinline__ int parts_of(int pages, int span, int most) {
    return max(1, min(most, (pages + span - 1) / span));
}

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
// after every operand's products.
template <int READS, int EACH> __device__ __forceinline__ void read_ahead() {
    constexpr int DEPTH = 6;
    __builtin_amdgcn_sched_group_barrier(0x100, DEPTH, 0);
#pragma unroll
    for (int i = 0; i < READS - DEPTH; i++) {
        __builtin_amdgcn_sched_group_barrier(0x008, EACH, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, EACH * DEPTH, 0);
}

// Pages of a slot's table: lane i holds that of tile at + i.  The first 64 are loaded by
// whoever knows the slot, beside the length that the tiles hang on, and others as
// they come up.
struct Ids {
    const int32_t *table;  // the slot's row, null for a slot outside the cache
    int blocks, at, v;
    __device__ __forceinline__ void load(int first) {
        const int i = first + (int)(threadIdx.x & 63);
        at = first;
        v = table && i < blocks ? table[i] : -1;
    }
    // -1: absent.  t is the same in all lanes and below `blocks`.
    __device__ __forceinline__ int page(const hymt_paged &p, int t) {
        if ((unsigned)(t - at) >= 64u) load(t);
        const int x = __builtin_amdgcn_readlane(v, t - at);
        return (unsigned)x < (unsigned)p.pages ? x : -1;
    }
};
__device__ __forceinline__ Ids ids_of(const hymt_paged &p, int slot, int first) {
    Ids r;
    r.table = (unsigned)slot < (unsigned)p.seqs ? p.table + (size_t)slot * p.blocks : nullptr;
    r.blocks = p.blocks;
    r.load(first);
    return r;
}

// KS: groups of four waves that take the rows' pages in turn.
template <int D, int KS> struct TileLds {
    uint16_t kv[KS][2][2][kPage * D];  // [group][buffer][K, V][page]; later what the groups hand over
    int flag[2];                       // a value that is not finite was seen in V, by buffer
    int low[4];                        // lowest limit of each wave's rows
};

// 64 QB rows of kv head h over pages [t0, t1) of a slot.  PREFIX: row r is entry
// r / G's, its limit min(common, that entry's length), the result a partial.
template <typename T, int D, int KS, int QB, bool PREFIX>
__device__ __forceinline__ void tile_part(const Plan &a, TileLds<D, KS> &s, int h, Ids ids, int slot_positions, Rows rows,
                                          int r0, int t0, int t1, int part, bool partial) {
    typedef typename Mma<T>::vec vec;
    constexpr int DS = D / 32, DB = D / 16, kPageBytes = kPage * D * 2;
    const int tid = threadIdx.x & 255, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int half = KS == 1 ? 0 : __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 8);
    const int grp = lane >> 4, c = lane & 15;

    const uint32_t off = (wave * 64 + lane) * 16;
    const uint32_t lds0 = lds_addr(&s.kv[half][0][0][0]) + wave * 1024;
    auto fetch = [&](int page, int buf, int v) __attribute__((always_inline)) {
        const char *base = (const char *)(v ? a.p.v : a.p.k) +
                           (((size_t)a.layer * a.p.pages + page) * a.p.kv_heads + h) * (size_t)kPageBytes;
#pragma unroll
        for (int i = 0; i < kPageBytes / 4096; i++)
            lds_dma16_sv(base + i * 4096, off, lds0 + (buf * 2 + v) * kPageBytes + i * 4096);
    };

    // ---- the wave's rows: q as the S^T B operand, lane (grp, c) has dims
    // 32 ks + 8 grp + [0, 8) of row c; rows past the end repeat the last one
    int limit[QB];
    size_t at[QB];  // element of (row, head) in q and out
    uint4 qu[QB][DS];
#pragma unroll
    for (int qq = 0; qq < QB; qq++) {
        const int r = min(r0 + wave * (16 * QB) + qq * 16 + c, rows.n - 1);
        const int token = r / a.group, g = r - token * a.group;
        at[qq] = ((size_t)(rows.first + token) * a.heads + h * a.group + g) * D;
#pragma unroll
        for (int ks = 0; ks < DS; ks++) qu[qq][ks] = *(const uint4 *)((const uint16_t *)a.q + at[qq] + 32 * ks + 8 * grp);
        if constexpr (PREFIX) limit[qq] = min(slot_positions, slot_len(a.p, a.b.slots[token]));
        else limit[qq] = min(rows.seen + token, slot_positions);
    }
    int page = t0 + half < t1 ? ids.page(a.p, t0 + half) : -1;
    if (page >= 0) {
        fetch(page, 0, 0);
        fetch(page, 0, 1);
    }

    vec qf[QB][DS];
#pragma unroll
    for (int qq = 0; qq < QB; qq++)
#pragma unroll
        for (int ks = 0; ks < DS; ks++)
            qf[qq][ks] = __builtin_bit_cast(vec, make_uint4(qu[qq][ks].x ^ a.flip, qu[qq][ks].y ^ a.flip,
                                                            qu[qq][ks].z ^ a.flip, qu[qq][ks].w ^ a.flip));
    // lowest limits: of the wave's blocks, and of the tile
    int low[QB];
#pragma unroll
    for (int qq = 0; qq < QB; qq++) low[qq] = wave_min(limit[qq]);
    if (lane == 0) s.low[wave] = min(low[0], low[QB - 1]);  // the groups have the same rows
    if (tid < 2) s.flag[tid] = 0;

    const bool live = r0 + wave * (16 * QB) < rows.n;  // the wave has a row
    pa_f32x4 o[DB][QB];
#pragma unroll
    for (int db = 0; db < DB; db++)
#pragma unroll
        for (int qq = 0; qq < QB; qq++) o[db][qq] = pa_f32x4{0.f, 0.f, 0.f, 0.f};
    float m[QB], l[QB];  // m in units of c s; l this lane's share
    bool far = false;    // some |m| of the wave is beyond kFarMax
#pragma unroll
    for (int qq = 0; qq < QB; qq++) {
        m[qq] = kNoMax;
        l[qq] = 0.f;
    }

    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    const int tile_low = min(min(s.low[0], s.low[1]), min(s.low[2], s.low[3]));

    for (int step = t0; step < t1; step += KS) {
        const int t = step + half, buf = KS == 1 ? (step - t0) & 1 : (step - t0) >> 1 & 1, base = t * kPage;
        const int next = t + KS < t1 ? ids.page(a.p, t + KS) : -1;
        const uint16_t *kt = s.kv[half][buf][0] + lane * 8, *vt = s.kv[half][buf][1] + grp * (D * 8) + c * 8;
        if (next >= 0) {
            fetch(next, buf ^ 1, 0);
            fetch(next, buf ^ 1, 1);
        }
        bool odd = false;
        if (min(step + KS, t1) * kPage > tile_low) {  // the same for both groups
            // Some row does not see some position of this page.  Its weight is 0
            // there, and 0 times an infinity or a NaN is none: values past the
            // sequence's end (anything may stand there) become 0 in LDS, and
            // if others are not finite the products leave them out (below).
            uint32_t top = 0;
            if (page >= 0)
#pragma unroll
            for (int i = 0; i < kPage * D / 8 / 256; i++) {
                const int ch = tid + 256 * i, pc = ch / D;
                uint4 *at_v = (uint4 *)s.kv[half][buf][1] + ch;
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
        const bool on = page >= 0 && live;
        pa_f32x4 sc[4][QB];
        if (on) {
            // ---- S^T = K Q^T, 64 positions x 16 rows a block.  Of two workgroups on
            // a CU the one at its products goes first (four prompts of 8192 512 -> 497 us)
            if constexpr (KS == 1) __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int kb = 0; kb < 4; kb++)
#pragma unroll
                for (int qq = 0; qq < QB; qq++) sc[kb][qq] = pa_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < DS; ks++)
#pragma unroll
                for (int kb = 0; kb < 4; kb++) {
                    const vec kf = __builtin_bit_cast(vec, *(const uint4 *)(kt + kb * (16 * D) + ks * 512));
#pragma unroll
                    for (int qq = 0; qq < QB; qq++) sc[kb][qq] = Mma<T>::mma(kf, qf[qq][ks], sc[kb][qq]);
                }
            read_ahead<4 * DS, QB>();
            if constexpr (KS == 1) __builtin_amdgcn_s_setprio(0);

            // ---- softmax
            float mx[QB];
#pragma unroll
            for (int qq = 0; qq < QB; qq++) {
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
            if (__any(mx[0] > m[0] + kLazyMax || mx[QB - 1] > m[QB - 1] + kLazyMax)) {
#pragma unroll
                for (int qq = 0; qq < QB; qq++) {
                    const float now = fmaxf(m[qq], rows_max(mx[qq]));
                    const float al = __builtin_amdgcn_exp2f(m[qq] - now);
                    m[qq] = now;
                    l[qq] *= al;
#pragma unroll
                    for (int db = 0; db < DB; db++) o[db][qq] *= al;
                }
                far = false;
#pragma unroll
                for (int qq = 0; qq < QB; qq++) far |= __any(m[qq] != kNoMax && fabsf(m[qq]) > kFarMax) != 0;
            }
            if (far)
#pragma unroll
                for (int qq = 0; qq < QB; qq++)
#pragma unroll
                    for (int kb = 0; kb < 4; kb++)
#pragma unroll
                        for (int i = 0; i < 4; i++) sc[kb][qq][i] = product_less(sc[kb][qq][i], a.c, m[qq]);
        }
        if (odd) {
            // Rare: the values that are not finite go to the rows that see them by
            // themselves (their weight is positive, so the result is the value)
            // and are then 0 for the products.
            if (on)
                for (int pos = 0; pos < kPage; pos++) {
                    const int pc = 4 * (pos >> 5) + ((pos >> 2) & 3), e = 4 * ((pos >> 4) & 1) + (pos & 3);
                    const uint16_t *v = s.kv[half][buf][1] + (size_t)pc * (D * 8) + e;
#pragma unroll
                    for (int db = 0; db < DB; db++)
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const uint16_t x = v[(16 * db + 4 * grp + i) * 8];
                            const float y = (x & 0x7FFFu) >= Mma<T>::kInf ? from_elem<T>(x) : 0.f;
#pragma unroll
                            for (int qq = 0; qq < QB; qq++) o[db][qq][i] += base + pos < limit[qq] ? y : 0.f;
                        }
                }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kPage * D / 8 / 256; i++) {
                uint32_t *w = (uint32_t *)((uint4 *)s.kv[half][buf][1] + tid + 256 * i);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    uint32_t x = w[e];
                    if ((x & 0x7FFFu) >= Mma<T>::kInf) x &= 0xFFFF0000u;
                    if ((x >> 16 & 0x7FFFu) >= Mma<T>::kInf) x &= 0xFFFFu;
                    w[e] = x;
                }
            }
            __syncthreads();
        }
        if (on) {
            // ---- weights, and O^T += V^T P^T: the second half's weights between the
            // first half's products
            vec pf[QB], vf[DB], vg[DB];
            const float by = far ? 1.0f : a.c;
            auto weights = [&](int k2) __attribute__((always_inline)) {
#pragma unroll
                for (int qq = 0; qq < QB; qq++) {
                    pa_f32x4 x = sc[2 * k2][qq], y = sc[2 * k2 + 1][qq];
                    const float less = far ? 0.f : -m[qq];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        x[i] = __builtin_amdgcn_exp2f(fmaf(x[i], by, less));
                        y[i] = __builtin_amdgcn_exp2f(fmaf(y[i], by, less));
                    }
                    const uint4 u = make_uint4(Mma<T>::pack(x[0], x[1]), Mma<T>::pack(x[2], x[3]),
                                               Mma<T>::pack(y[0], y[1]), Mma<T>::pack(y[2], y[3]));
                    l[qq] = Mma<T>::sum(u.w, Mma<T>::sum(u.z, Mma<T>::sum(u.y, Mma<T>::sum(u.x, l[qq]))));
                    pf[qq] = __builtin_bit_cast(vec, u);
                }
            };
#pragma unroll
            for (int db = 0; db < DB; db++) vf[db] = __builtin_bit_cast(vec, *(const uint4 *)(vt + db * 128));
            weights(0);
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (KS == 1) __builtin_amdgcn_s_setprio(1);
            vec first[QB];
#pragma unroll
            for (int qq = 0; qq < QB; qq++) first[qq] = pf[qq];
#pragma unroll
            for (int db = 0; db < DB; db++) {
#pragma unroll
                for (int qq = 0; qq < QB; qq++) o[db][qq] = Mma<T>::mma(vf[db], first[qq], o[db][qq]);
                vg[db] = __builtin_bit_cast(vec, *(const uint4 *)(vt + 4 * D * 8 + db * 128));
            }
            weights(1);
#pragma unroll
            for (int i = 0; i < DB; i++) {
                __builtin_amdgcn_sched_group_barrier(0x008, QB, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x002, 28 * QB / DB, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int db = 0; db < DB; db++)
#pragma unroll
                for (int qq = 0; qq < QB; qq++) o[db][qq] = Mma<T>::mma(vg[db], pf[qq], o[db][qq]);
            if constexpr (KS == 1) __builtin_amdgcn_s_setprio(0);
        }
        page = next;
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
        if (odd && tid == 0) s.flag[buf] = 0;  // every wave has read it; the next that sets it does so two steps on
    }

    if constexpr (KS == 2) {
        // the second group hands its (m, l, O) to the first (the last barrier is
        // behind every read of the pages)
        pa_f32x4 *x = (pa_f32x4 *)&s.kv[0][0][0][0] + (wave * (QB * DB + 1)) * 64 + lane;
        static_assert(4 * (QB * DB + 1) * 64 * 16 <= (int)sizeof(s.kv), "hand-over");
        if (half) {
#pragma unroll
            for (int db = 0; db < DB; db++)
#pragma unroll
                for (int qq = 0; qq < QB; qq++) x[(QB * db + qq) * 64] = o[db][qq];
            x[QB * DB * 64] = pa_f32x4{m[0], m[QB - 1], l[0], l[QB - 1]};
        }
        __syncthreads();
        if (half) return;
        const pa_f32x4 ml = x[QB * DB * 64];
#pragma unroll
        for (int qq = 0; qq < QB; qq++) {
            const float now = fmaxf(m[qq], ml[qq]);
            const float w0 = __builtin_amdgcn_exp2f(m[qq] - now), w1 = __builtin_amdgcn_exp2f(ml[qq] - now);
            m[qq] = now;
            l[qq] = l[qq] * w0 + ml[2 + qq] * w1;
#pragma unroll
            for (int db = 0; db < DB; db++) o[db][qq] = o[db][qq] * w0 + x[(QB * db + qq) * 64] * w1;
        }
    }

#pragma unroll
    for (int qq = 0; qq < QB; qq++) {
        l[qq] = rows_sum(l[qq]);
        if (r0 + wave * (16 * QB) + qq * 16 + c >= rows.n) continue;
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

// Pages that a tile of an entry attends to.
__device__ __forceinline__ int tile_pages(const Plan &a, int len, Span sp, int index) {
    const int last = min(sp.n - 1, (min((index + 1) * a.tile_rows, sp.n * a.group) - 1) / a.group);
    return pages_of(max(0, min(len, len - sp.n + last + 1)));
}

// The tile that work index w is of.  Tiles of an entry come last first, so that the
// longest kv ranges start first; SPLIT: only those that are cut into parts count (the
// last ones of an entry).
struct Tile {
    int index, slot, len;
    Span span;
};
template <bool SPLIT> __device__ __forceinline__ bool find_tile(const Plan &a, int w, Tile &out) {
    const int lane = threadIdx.x & 63;
    int before = 0;
    if (!SPLIT && !a.b.cu) {  // a tile an entry
        if (w >= a.b.n) return false;
        const int slot = a.b.slots[w];
        out = {0, slot, slot_len(a.p, slot), {w, 1}};
        return true;
    }
    if (!SPLIT && a.b.n > 64) {
        // 256 entries in a round trip, and the length after the search (256 prompts of 30
        // rows 33.2 -> 30-32 us, 1024 of 8 rows 121 -> 85-88)
        constexpr int C = 4;
        for (int base = 0; base < a.b.n; base += 64 * C) {
            Span sp[C];
            int slot[C];
#pragma unroll
            for (int j = 0; j < C; j++) {
                const int i = min(base + 64 * j + lane, a.b.n);  // past the end: no rows
                const int lo = max(0, min(a.b.cu[i], a.b.rows)), hi = min(a.b.cu[min(i + 1, a.b.n)], a.b.rows);
                sp[j] = {lo, max(lo, hi) - lo};
                slot[j] = a.b.slots[min(i, a.b.n - 1)];
            }
#pragma unroll
            for (int j = 0; j < C; j++) {
                const int tiles = (sp[j].n * a.group + a.tile_rows - 1) / a.tile_rows, x = wave_sums(tiles);
                const uint64_t hit = __ballot(w < before + x);
                if (hit) {
                    const int at = __ffsll((unsigned long long)hit) - 1;
                    out.index = before + __builtin_amdgcn_readlane(x, at) - 1 - w;
                    out.slot = __builtin_amdgcn_readlane(slot[j], at);
                    out.len = slot_len(a.p, out.slot);
                    out.span = {__builtin_amdgcn_readlane(sp[j].first, at), __builtin_amdgcn_readlane(sp[j].n, at)};
                    return true;
                }
                before += __builtin_amdgcn_readlane(x, 63);
            }
        }
        return false;
    }
    for (int base = 0; base < a.b.n; base += 64) {
        const int i = base + lane;
        Span sp{0, 0};
        int slot = -1;
        if (i < a.b.n) {
            sp = span_of(a.b, i);
            slot = a.b.slots[i];
        }
        const int len = slot_len(a.p, slot);  // for every entry: one load deep, not one more after the search
        const int tiles = (sp.n * a.group + a.tile_rows - 1) / a.tile_rows;
        int count = tiles;
        if constexpr (SPLIT) {
            // tile_pages(index) > span from the token on that sees span * 64 + 1 positions
            const long token = max(0L, (long)a.span * kPage - (len - sp.n));
            // the first tile whose last token is that one or a later one
            count = len > a.span * kPage && token < sp.n ? tiles - (int)(token * a.group / a.tile_rows) : 0;
        }
        const int x = wave_sums(count);
        const uint64_t hit = __ballot(w < before + x);
        if (hit) {
            const int at = __ffsll((unsigned long long)hit) - 1;
            const int first = before + __builtin_amdgcn_readlane(x, at) - __builtin_amdgcn_readlane(count, at);
            out.index = __builtin_amdgcn_readlane(tiles, at) - 1 - (w - first);
            out.slot = __builtin_amdgcn_readlane(slot, at);
            out.len = __builtin_amdgcn_readlane(len, at);
            out.span = {__builtin_amdgcn_readlane(sp.first, at), __builtin_amdgcn_readlane(sp.n, at)};
            return true;
        }
        before += __builtin_amdgcn_readlane(x, 63);
    }
    return false;
}

template <typename T, int D, int KS, int QB> __global__ __launch_bounds__(256 * KS, 2) void attn_packed_kernel(Plan a) {
    __shared__ __attribute__((aligned(256))) TileLds<D, KS> s;
    // workgroups of one kv head on the same XCDs (workgroup b runs on XCD
    // b % 8), whose L2 then holds that head's pages
    const int h = blockIdx.x % a.p.kv_heads, rest = blockIdx.x / a.p.kv_heads;
    const int part = rest / a.tiles;  // second parts, which not every tile has, come after all first ones
    Tile t;
    if (!find_tile<false>(a, rest - part * a.tiles, t)) return;
    const Ids ids = ids_of(a.p, t.slot, 0);
    const int pages = tile_pages(a, t.len, t.span, t.index), parts = parts_of(pages, a.span, a.parts);
    if (part >= parts) return;
    const Rows rows{t.span.first, t.span.n * a.group, t.len - t.span.n + 1};
    tile_part<T, D, KS, QB, false>(a, s, h, ids, t.len, rows, t.index * (64 * QB), (int)((long)part * pages / parts),
                           (int)((long)(part + 1) * pages / parts), part, parts > 1);
}

// ---- single rows -------------------------------------------------------------------

template <int D> struct RowLds {
    float o[4][16][D + 4];
    float m[4][16], l[4][16];
};

// Page t of an entry that reads the first `common` of them from another slot's table.
struct RowPages {
    Ids first, own;
    int common;
    __device__ __forceinline__ int page(const hymt_paged &p, int t) { return t < common ? first.page(p, t) : own.page(p, t); }
};

// Up to 16 rows (heads g0 ..) of one entry over pages [t0, t1) of its slot, a page to
// a wave: K and V go from memory into operand registers, those of the wave's next
// page as soon as the products have read these.
template <typename T, int D>
__device__ __forceinline__ void row_part(const Plan &a, RowLds<D> &s, int entry, int h, int g0, RowPages ids, int len, int t0,
                                         int t1, int part, bool partial) {
    typedef typename Mma<T>::vec vec;
    constexpr int DS = D / 32, DB = D / 16;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int grp = lane >> 4, c = lane & 15;
    const int g = min(g0 + c, a.group - 1);
    const size_t at = ((size_t)entry * a.heads + h * a.group + g) * D;
    uint4 qu[DS], ku[DS][4], vu[2][DB];
#pragma unroll
    for (int ks = 0; ks < DS; ks++) qu[ks] = *(const uint4 *)((const uint16_t *)a.q + at + 32 * ks + 8 * grp);
    // an absent page is read as page 0 and masked whole
    auto base_of = [&](int page) {
        return (((size_t)a.layer * a.p.pages + max(page, 0)) * a.p.kv_heads + h) * (size_t)(kPage * D);
    };
    auto load_k = [&](int page) __attribute__((always_inline)) {
        const uint16_t *kp = (const uint16_t *)a.p.k + base_of(page) + lane * 8;
#pragma unroll
        for (int ks = 0; ks < DS; ks++)
#pragma unroll
            for (int kb = 0; kb < 4; kb++) ku[ks][kb] = *(const uint4 *)(kp + kb * (16 * D) + ks * 512);
    };
    auto load_v = [&](int page) __attribute__((always_inline)) {
        const uint16_t *vp = (const uint16_t *)a.p.v + base_of(page) + grp * (D * 8) + c * 8;
#pragma unroll
        for (int k2 = 0; k2 < 2; k2++)
#pragma unroll
            for (int db = 0; db < DB; db++) vu[k2][db] = *(const uint4 *)(vp + k2 * (4 * D * 8) + db * 128);
    };
    int t = t0 + wave, page = -1;
    if (t < t1) {
        page = ids.page(a.p, t);
        load_k(page);
        load_v(page);
    }
    vec qf[DS];
#pragma unroll
    for (int ks = 0; ks < DS; ks++)
        qf[ks] = __builtin_bit_cast(vec, make_uint4(qu[ks].x ^ a.flip, qu[ks].y ^ a.flip, qu[ks].z ^ a.flip,
                                                    qu[ks].w ^ a.flip));
    pa_f32x4 o[DB];
#pragma unroll
    for (int db = 0; db < DB; db++) o[db] = pa_f32x4{0.f, 0.f, 0.f, 0.f};
    float m = kNoMax, l = 0.f;
    while (t < t1) {
        pa_f32x4 sc[4];
#pragma unroll
        for (int kb = 0; kb < 4; kb++) sc[kb] = pa_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < DS; ks++)
#pragma unroll
            for (int kb = 0; kb < 4; kb++) sc[kb] = Mma<T>::mma(__builtin_bit_cast(vec, ku[ks][kb]), qf[ks], sc[kb]);
        const int left = page < 0 ? 0 : len - t * kPage;  // positions of this page
        const int next = t + 4 < t1 ? ids.page(a.p, t + 4) : -1;
        if (t + 4 < t1) load_k(next);
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
            for (int i = 0; i < 4; i++) sc[kb][i] = __builtin_amdgcn_exp2f(product_less(sc[kb][i], a.c, m));
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
        if (t + 4 < t1) load_v(next);
        page = next;
        t += 4;
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

// Workgroups [0, tile_wgs) the prefix, the others the entries' own positions (tile_wgs
// 0: all of them).
template <typename T, int D, int QB> __global__ __launch_bounds__(256, 2) void attn_shared_kernel(Plan a, int tile_wgs) {
    __shared__ __attribute__((aligned(256))) union {
        TileLds<D, 1> tile;
        RowLds<D> row;
    } s;
    // the table's part is loaded where the range begins if slots[0] is as long as the
    // prefix, as it should be, beside the length that decides
    const int pages_expected = min(a.prefix / kPage, a.p.blocks), slot0 = a.b.slots[0];
    if ((int)blockIdx.x < tile_wgs) {
        const int h = blockIdx.x % a.p.kv_heads, rest = blockIdx.x / a.p.kv_heads, part = rest % a.parts;
        const Ids ids = ids_of(a.p, slot0, (int)((long)part * pages_expected / parts_of(pages_expected, a.span, a.parts)));
        const int common = common_of(a), pages = common / kPage, parts = parts_of(pages, a.span, a.parts);
        if (part >= parts || pages == 0) return;
        tile_part<T, D, 1, QB, true>(a, s.tile, h, ids, common, Rows{0, a.b.n * a.group, 0}, rest / a.parts * (64 * QB),
                                 (int)((long)part * pages / parts), (int)((long)(part + 1) * pages / parts), part, true);
        return;
    }
    int w = blockIdx.x - tile_wgs;
    const int h = w % a.p.kv_heads;
    w /= a.p.kv_heads;
    const int blocks16 = (a.group + 15) / 16;
    const int g0 = w % blocks16 * 16;
    w /= blocks16;
    const int part = w % a.own_parts, entry = w / a.own_parts, slot = a.b.slots[entry];
    RowPages ids{ids_of(a.p, slot0, 0), ids_of(a.p, slot, pages_expected), 0};
    const int common = common_of(a), len = slot_len(a.p, slot);
    ids.common = common / kPage;
    // without tiles the rows see to the prefix too
    const int first = tile_wgs ? ids.common : 0, pages = max(0, pages_of(len) - first),
              parts = parts_of(pages, a.own_span, a.own_parts);
    if (part >= parts) return;
    row_part<T, D>(a, s.row, entry, h, g0, ids, len, first + (int)((long)part * pages / parts),
                   first + (int)((long)(part + 1) * pages / parts), a.parts + part, !a.direct);
}

// ---- joining: out = sum_k 2^(m_k - m) O_k / sum_k 2^(m_k - m) l_k -------------------

// The split tiles of attn_packed: a group of D / 4 lanes a row of one head.  The grid
// walks over them, as their number is only known here.
constexpr int kJoinGrid = 1024;
template <typename T, int D> __global__ __launch_bounds__(256) void attn_join_tiles_kernel(Plan a) {
    constexpr int L = D / 4, G = 256 / L, K = kMaxParts / L;
    __shared__ float s_w[G][kMaxParts];
    const int g = threadIdx.x / L, lane = threadIdx.x % L;
    const size_t stride = (size_t)a.b.rows * a.heads;
    for (int u = blockIdx.x;; u += gridDim.x) {
        const int h = u % a.p.kv_heads, rest = u / a.p.kv_heads;
        Tile t;
        const int chunks = a.tile_rows / G;
        if (!find_tile<true>(a, rest / chunks, t)) return;
        const int n = parts_of(tile_pages(a, t.len, t.span, t.index), a.span, a.parts);
        const int r = t.index * a.tile_rows + rest % chunks * G + g;
        const bool on = r < t.span.n * a.group;
        const int token = min(r, t.span.n * a.group - 1) / a.group;
        const size_t at = (size_t)(t.span.first + token) * a.heads + h * a.group + (on ? r - token * a.group : 0);
        float2 ml[K];
        float top = kNoMax, sum = 0.f;
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int i = lane + L * k;
            ml[k] = i < n ? *(const float2 *)(a.ml + (i * stride + at) * 2) : make_float2(kNoMax, 0.f);
            top = fmaxf(top, ml[k].x);
        }
#pragma unroll
        for (int x = 1; x < L; x <<= 1) top = fmaxf(top, __shfl_xor(top, x));
#pragma unroll
        for (int k = 0; k < K; k++) {
            const float w = __builtin_amdgcn_exp2f(ml[k].x - top);
            sum += w * ml[k].y;
            s_w[g][lane + L * k] = w;
        }
#pragma unroll
        for (int x = 1; x < L; x <<= 1) sum += __shfl_xor(sum, x);
        __syncthreads();
        pa_f32x4 acc{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int k = 0; k < n; k++) acc += *(const pa_f32x4 *)(a.o + (k * stride + at) * D + 4 * lane) * s_w[g][k];
        const float inv = sum == 0.f ? 0.f : 1.0f / sum;
        if (on) put4<T>(a, at * D + 4 * lane, acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
        __syncthreads();
    }
}

// attn_shared: the first n0 parts of the prefix, then n1 of the entry's own.  WHOLE: a
// workgroup takes one row of one head, its groups of D / 4 lanes the parts in
// turn; else a group takes a row by itself (up to D / 4 parts).  The (m, l) are
// read before it is known how many parts the row has (what lies past them is left
// out): one round trip less between the lengths and the sums.
template <typename T, int D, bool WHOLE> __global__ __launch_bounds__(256) void attn_join_rows_kernel(Plan a) {
    constexpr int L = D / 4, G = 256 / L, K = WHOLE ? 2 : 1;
    __shared__ __attribute__((aligned(16))) float s_o[WHOLE ? G : 1][D];
    __shared__ float s_w[WHOLE ? 1 : G][WHOLE ? 2 * kMaxParts : L];
    const int tid = threadIdx.x, g = tid / L, lane = tid % L, d = 4 * lane;
    const size_t stride = (size_t)a.b.rows * a.heads;
    const size_t rh = WHOLE ? blockIdx.x : (size_t)blockIdx.x * G + g, at = min(rh, stride - 1);
    const int row = (int)(at / a.heads), most = a.parts + a.own_parts;
    constexpr int W = WHOLE ? 64 : L;  // lanes that hold a row's weights, K parts each
    const int mine = WHOLE ? tid & 63 : lane;
    float2 ml[K];
#pragma unroll
    for (int k = 0; k < K; k++) ml[k] = *(const float2 *)(a.ml + (min(mine + W * k, most - 1) * stride + at) * 2);
    const int common = common_of(a), len = slot_len(a.p, a.b.slots[row]);
    const int n0 = common ? parts_of(common / kPage, a.span, a.parts) : 0;
    const int n1 = parts_of(max(0, pages_of(len) - common / kPage), a.own_span, a.own_parts);
    float top = kNoMax, sum = 0.f;
#pragma unroll
    for (int k = 0; k < K; k++) {
        const int i = mine + W * k;
        if (i >= most || !(i < n0 || (i >= a.parts && i < a.parts + n1))) ml[k] = make_float2(kNoMax, 0.f);
        top = fmaxf(top, ml[k].x);
    }
#pragma unroll
    for (int x = 1; x < W; x <<= 1) top = fmaxf(top, __shfl_xor(top, x));
#pragma unroll
    for (int k = 0; k < K; k++) {
        const float w = __builtin_amdgcn_exp2f(ml[k].x - top);
        sum += w * ml[k].y;
        if (!WHOLE || tid < 64) s_w[WHOLE ? 0 : g][mine + W * k] = w;
    }
#pragma unroll
    for (int x = 1; x < W; x <<= 1) sum += __shfl_xor(sum, x);
    __syncthreads();
    const int total = n0 + n1;
    pa_f32x4 acc{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int k = WHOLE ? g : 0; k < total; k += WHOLE ? G : 1) {
        const int part = k < n0 ? k : a.parts + k - n0;
        acc += *(const pa_f32x4 *)(a.o + (part * stride + at) * D + d) * s_w[WHOLE ? 0 : g][part];
    }
    if constexpr (WHOLE) {
        *(pa_f32x4 *)&s_o[g][d] = acc;
        __syncthreads();
        if (tid >= L) return;
        for (int k = 1; k < G; k++) acc += *(const pa_f32x4 *)&s_o[k][d];
    }
    if (rh >= stride) return;
    const float inv = sum == 0.f ? 0.f : 1.0f / sum;
    put4<T>(a, at * D + d, acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
}

// ---- host --------------------------------------------------------------------------

Plan plan_of(const hymt_paged &p, const hymt_batch &b, const PagedAttn &a, const PagedSplit &s, float *ws) {
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
    r.c = std::max(std::abs(paged_log2_scale(a.scale)), std::numeric_limits<float>::denorm_min());
    r.flip = a.scale < 0 ? 0x80008000u : 0u;
    r.parts = s.parts;
    r.span = s.span;
    r.own_parts = s.own;
    r.own_span = s.own_span;
    r.tiles = s.tiles;
    r.tile_rows = s.rows;
    const size_t rh = (size_t)b.rows * a.heads;
    r.o = ws;
    r.ml = ws + (size_t)(s.parts + s.own) * rh * p.head_dim;
    return r;
}

template <typename T, int D> void packed(const Plan &a, const PagedSplit &s, hipStream_t st) {
    {
        KernelSpan span("attn_packed", st, true);
        const dim3 grid(s.tiles * s.parts * a.p.kv_heads);
        if (s.rows == 64) {
            if (s.groups == 2) launch(span, attn_packed_kernel<T, D, 2, 1>, grid, dim3(512), 0, st, a);
            else launch(span, attn_packed_kernel<T, D, 1, 1>, grid, dim3(256), 0, st, a);
        } else {
            if (s.groups == 2) launch(span, attn_packed_kernel<T, D, 2, 2>, grid, dim3(512), 0, st, a);
            else launch(span, attn_packed_kernel<T, D, 1, 2>, grid, dim3(256), 0, st, a);
        }
    }
    if (s.parts == 1) return;
    KernelSpan span("attn_merge", st, true);
    launch(span, attn_join_tiles_kernel<T, D>, dim3(std::min<long>((long)s.tiles * (s.rows * D / 1024) * a.p.kv_heads, kJoinGrid)), dim3(256), 0, st, a);
}

template <typename T, int D> void shared(Plan a, const PagedSplit &s, hipStream_t st) {
    const int tile_wgs = s.tiles * s.parts * a.p.kv_heads, row_wgs = a.b.n * a.p.kv_heads * s.blocks16 * s.own;
    a.direct = s.tiles == 0 && s.own == 1;
    if (s.tiles == 0) a.parts = 0;
    {
        KernelSpan span("attn_shared", st, true);
        if (s.rows == 64) launch(span, attn_shared_kernel<T, D, 1>, dim3(tile_wgs + row_wgs), dim3(256), 0, st, a, tile_wgs);
        else launch(span, attn_shared_kernel<T, D, 2>, dim3(tile_wgs + row_wgs), dim3(256), 0, st, a, tile_wgs);
    }
    if (a.direct) return;
    constexpr int L = D / 4, G = 256 / L;
    const long rows = (long)a.b.rows * a.heads;
    KernelSpan span("attn_merge", st, true);
    // many parts of few rows: a workgroup a row
    if (a.parts + a.own_parts > L || (rows < 2048 && a.parts + a.own_parts >= G))
        launch(span, attn_join_rows_kernel<T, D, true>, dim3((unsigned)rows), dim3(256), 0, st, a);
    else
        launch(span, attn_join_rows_kernel<T, D, false>, dim3((unsigned)ceil_div(rows, G)), dim3(256), 0, st, a);
}

}  // namespace

size_t paged_attn_workspace(const hymt_paged &p, const hymt_batch &b, const PagedAttn &a, bool shared) {
    if (b.n == 0 || b.rows == 0) return 0;
    const PagedSplit s = paged_split(p, b, a.heads, a.prefix, shared);
    if (shared ? s.tiles == 0 && s.own == 1 : s.parts == 1) return 0;
    return (size_t)(s.parts + s.own) * b.rows * a.heads * (p.head_dim + 2);
}

hipError_t launch_attn_packed(const hymt_paged &p, const hymt_batch &b, const PagedAttn &a, float *ws, hipStream_t st) {
    if (b.n == 0 || b.rows == 0) return hipSuccess;
    const PagedSplit s = paged_split(p, b, a.heads, 0, false);
    const Plan r = plan_of(p, b, a, s, ws);
    if (p.dtype == HYMT_F16) p.head_dim == 64 ? packed<F16, 64>(r, s, st) : packed<F16, 128>(r, s, st);
    else p.head_dim == 64 ? packed<BF16, 64>(r, s, st) : packed<BF16, 128>(r, s, st);
    return hipGetLastError();
}

hipError_t launch_attn_shared(const hymt_paged &p, const hymt_batch &b, const PagedAttn &a, float *ws, hipStream_t st) {
    if (b.n == 0) return hipSuccess;
    const PagedSplit s = paged_split(p, b, a.heads, a.prefix, true);
    const Plan r = plan_of(p, b, a, s, ws);
    if (p.dtype == HYMT_F16) p.head_dim == 64 ? shared<F16, 64>(r, s, st) : shared<F16, 128>(r, s, st);
    else p.head_dim == 64 ? shared<BF16, 64>(r, s, st) : shared<BF16, 128>(r, s, st);
    return hipGetLastError();
}

}  // namespace hymt
