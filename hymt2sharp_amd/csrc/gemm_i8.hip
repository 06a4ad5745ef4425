// gemm_i8.hip -- products of int8 codes (gfx950): y[t][f] = ws[f] xs[t] sum_k
// x[t][k] w[f][k] on v_mfma_i32_16x16x64_i8, the sum exact in int32, then fp32
// products with the two scales; fp32, added to fp32, bf16, or (SwiGLU) the bf16
// silu(g) u of two such products.
//
// The sum is exact, so its order is free: every kernel and tile below gives the
// same bits, and which one runs is a matter of time alone.
//
// What it takes (us, in a recording, over the cards seen).  here: three sets of
// operands in turn, whose weights stay in the 256 MB last-level cache but for the
// 120818 channels; cold: enough sets to exceed it.  ref: the bytes at 5.05 TB/s or the
// operations at 2058 TOP/s, what a large copy and a large int8 product of the
// library reach, and 1.8 for a launch; no bound, since a stream that is only read
// passes 6.3 TB/s and the SwiGLU beats that product.
//   tokens x channels x k      output        ref    here        cold
//   1 x 2048 x 2048            fp32          2.6    2.9-3.0     4.0
//   1 x 120818 x 2048          fp32         50.8    39.1-39.7   39.4-39.6
//   61 x 2048 x 6144           fp32 +=       4.6    6.3-6.5     9.0
//   300 x 2048 x 6144          bf16          5.5   11.7        16.2
//   700 x 2048 x 6144          bf16         10.4   15.1-16.2   20.4
//   2048 x 2048 x 2048         bf16         10.1   11.9-13.2   14.3
//   2048 x 2048 x 6144         fp32         26.8   27.4-30.4   34.9
//   61 x 2 6144 x 2048         SwiGLU        6.9    7.2-7.6    10.6
//   2048 x 2 6144 x 2048       SwiGLU       51.9   47.6-51.5   57.5
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <cstdlib>
#include <cstring>
#include <type_traits>

#include "device_common.hpp"
#include "int8.hpp"
#include "ktimer.hpp"

namespace hymt {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

enum Out { kF32, kAcc, kBf16, kGlu };

constexpr int kBK = kI8StepK;  // k (bytes of a row) per stage
constexpr int kFrag = 1024;    // bytes of one 16 x 64 operand fragment
constexpr int kPair = 2048;    // one row block's 16 rows x 128 k of a stage
constexpr int kGroupF = 4;     // feature tiles walked together (L2 reuse)

struct Args {
    I8Gemm g;
    int tiles, tiles_f, tiles_t;
    int per_xcd;  // workgroups per XCD: ceil(tiles / 8)
    bool vec;     // the output takes 16-byte stores of whole chunks
};

// s_waitcnt with vmcnt n (<= 63) alone, with lgkmcnt 0 too, and lgkmcnt 0 alone
// (gfx9 encoding: vmcnt in bits 3:0 and 15:14, expcnt 6:4, lgkmcnt 11:8)
template <int N, bool LGKM = false> __device__ __forceinline__ void wait_vm() {
    static_assert(N >= 0 && N <= 63, "vmcnt");
    __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (LGKM ? 0 : 15 << 8));
    asm volatile("" ::: "memory");
}
__device__ __forceinline__ void wait_lgkm() {
    __builtin_amdgcn_s_waitcnt(15 | (3 << 14) | (7 << 4));
    asm volatile("" ::: "memory");
}

// lds_dma16_sv past the caches.
__device__ __forceinline__ void lds_dma16_sv_nt(const void *sbase, uint32_t voff, uint32_t lds_base) {
    asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, %2 nt"
                 :
                 : "s"(__builtin_amdgcn_readfirstlane(lds_base)), "v"(voff), "s"(sbase)
                 : "memory", "m0");
}

// The one arithmetic of an output: the channel's scale first, then the token's,
// fused with the addition where there is one.
__device__ __forceinline__ float scaled(int s, float ws) { return (float)s * ws; }
__device__ __forceinline__ float glu(int g, int u, float ws, float us, float xs) {
    return silu_fast(scaled(g, ws) * xs) * (scaled(u, us) * xs);
}
// bf16, rounded to nearest even by v_cvt_pk_bf16_f32; a NaN stays one whatever its
// bits (a token's scale may be any NaN)
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf16x2));
}

// Features f .. f + 3 of token t from the sums, where f + e < n.
template <int OUT>
__device__ __forceinline__ void store4(const Args &a, int t, int f, i32x4 s, i32x4 up, const float (&ws)[4],
                                       const float (&us)[4], float xs) {
    const I8Gemm &g = a.g;
    const size_t at = (size_t)t * g.ldy + f;
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; e++)
        v[e] = OUT == kGlu ? glu(s[e], up[e], ws[e], us[e], xs) : OUT == kAcc ? scaled(s[e], ws[e]) : scaled(s[e], ws[e]) * xs;
    if constexpr (OUT == kGlu || OUT == kBf16) {
        uint16_t *y = (uint16_t *)g.y + at;
        if (a.vec && f + 4 <= g.n) {
            *(uint2 *)y = make_uint2(pack2(v[0], v[1]), pack2(v[2], v[3]));
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (f + e < g.n) y[e] = (uint16_t)pack2(v[e], 0.f);
        }
    } else {
        float *y = (float *)g.y + at;
        if (a.vec && f + 4 <= g.n) {
            if constexpr (OUT == kAcc) {
                const float4 o = *(const float4 *)y;
                *(float4 *)y = make_float4(fmaf(v[0], xs, o.x), fmaf(v[1], xs, o.y), fmaf(v[2], xs, o.z), fmaf(v[3], xs, o.w));
            } else {
                *(float4 *)y = make_float4(v[0], v[1], v[2], v[3]);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (f + e < g.n) y[e] = OUT == kAcc ? fmaf(v[e], xs, y[e]) : v[e];
        }
    }
}

// ---- tiles ---------------------------------------------------------------------
//
// Workgroup tile: TF = 32 IF features x TT = 32 JT tokens by 2 x WT waves, wave
// (wf, wt) the tile's feature half wf and token part wt, IF x BJ blocks of 16 x 16.
//
// k advances in stages of 128: a stage is (TF + TT) / 16 row blocks of 2 KiB (16
// rows x 128 k; the W blocks first, then the x blocks), copied from global
// memory straight into an LDS ring of S stages, each copy instruction 8 whole
// 128-byte lines; the rows' order and an XOR order of each row's 16-byte pieces
// leave the operand reads free of bank conflicts.  A step of 64 k is IF x BJ
// MFMAs per wave, with the operand reads of the next step and a share of a later
// stage's copies between them.  The bytes moved, the LDS reads and the MFMA cycles
// of a stage are those of a bf16 stage of 64 k, for twice the k.
//
// KG = 2: two groups of waves take every other stage, each through a ring of its
// own, two waves a SIMD: one wave's copies, which hold its issue for about 50
// cycles each, run under the other's MFMAs.  Their sums meet in LDS at the end.
// Taken for the tiles whose two rings fit (us, one group / two, bf16: 128 x 64 over
// 1024 x 2048 x 6144 18.6 / 17.4; few-token kernel / two groups: 64 x 64 over 300 x
// 2048 x 2048 6.4 / 5.2, 96 x 64 over 700 x 2048 x 6144 16.3 / 15.1; 128 x 128, whose
// rings then hold two stages each, 12.0 / 13.7 over 2048 x 2048 x 2048).
//
// SwiGLU: the tile holds TF / 2 outputs, of a wave's IF row blocks the first half
// gate rows and the others the same rows of up, so that g and u of an output
// meet in one lane's registers.
//
// Rows past n or m repeat the last one; their outputs are not written.

// Workgroup b runs on XCD b % 8 (dispatch is round-robin over the 8 XCDs): each
// XCD takes one contiguous run of tiles.  The order: groups of 4 feature tiles,
// walked token tile by token tile, so that the workgroups an XCD holds at a
// time share their W and x rows in that XCD's L2.
__device__ __forceinline__ bool tile_of(const Args &a, int &tf, int &tt) {
    const int L = (blockIdx.x & 7) * a.per_xcd + (blockIdx.x >> 3);
    if (L >= a.tiles) return false;
    const int per_group = kGroupF * a.tiles_t;
    const int g = L / per_group, r = L - g * per_group;
    const int width = min(kGroupF, a.tiles_f - g * kGroupF);
    tt = r / width;
    tf = g * kGroupF + (r - tt * width);
    return true;
}

// The schedule of a step, row by row: row i's BJ MFMAs, then its reads (W
// fragment i and the x fragments the row loads).
template <int IF, int BJ, int I> __device__ __forceinline__ void sched_rows() {
    if constexpr (I < IF) {
        __builtin_amdgcn_sched_group_barrier(0x008, BJ, 0);                                   // MFMA
        __builtin_amdgcn_sched_group_barrier(0x100, 1 + (I + 1) * BJ / IF - I * BJ / IF, 0);  // DS read
        sched_rows<IF, BJ, I + 1>();
    }
}

// One 64-k step of a wave: the MFMAs of the operands in (w, cx), row by row, with
// the operand reads of the next step (LDS at nsb + noff) interleaved: W fragment
// i of the next step replaces w[i] once row i's MFMAs have issued, the x
// fragments go to nx.  after_row(i) runs after row i's reads.
template <int IF, int BJ, typename F>
__device__ __forceinline__ void substep(i32x4 (&w)[IF], const i32x4 (&cx)[BJ], const uint8_t *nsb, uint32_t noff,
                                        int wf, int wt, i32x4 (&nx)[BJ], i32x4 (&acc)[IF][BJ], F &&after_row) {
#pragma unroll
    for (int i = 0; i < IF; i++) {
#pragma unroll
        for (int j = 0; j < BJ; j++) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[i], cx[j], acc[i][j], 0, 0, 0);
        w[i] = *(const i32x4 *)(nsb + noff + (IF * wf + i) * kPair);
#pragma unroll
        for (int j = i * BJ / IF; j < (i + 1) * BJ / IF; j++)
            nx[j] = *(const i32x4 *)(nsb + noff + (2 * IF + BJ * wt + j) * kPair);
        after_row(i);
    }
    sched_rows<IF, BJ, 0>();
}

// S stages in the ring; LGKM: a stage's slot is refilled at the barrier right
// after its last operand reads (each wave first waits for its own reads), so
// S - 1 stages are ahead of the one being read; else one barrier later, with
// S - 2 ahead and no wait on the reads.
template <int IF, int JT, int WT, int S, bool LGKM, int KG, int OUT>
__global__ __launch_bounds__(128 * WT * KG, 1) void tile_kernel(Args a) {
    constexpr bool GLU = OUT == kGlu;
    constexpr int TF = 32 * IF, TT = 32 * JT;
    constexpr int NW = 2 * WT, NT = 64 * NW * KG, BJ = TT / (16 * WT);  // waves of a k group, threads, token blocks per wave
    constexpr int BE = BJ / KG;                                          // ... that a wave writes
    constexpr int NBF = TF / 16, NB = (TF + TT) / 16;               // row blocks: W, all
    constexpr int C = 2 * NB / NW;                                   // copy instructions per wave per stage
    constexpr int kStageBytes = NB * kPair;
    constexpr int AHEAD = LGKM ? S : S - 1;  // stages issued ahead of the one being read, plus one
    constexpr int OF = GLU ? TF / 2 : TF;    // output features of the tile
    constexpr int OI = GLU ? IF / 2 : IF;    // ... and their row blocks per wave
    static_assert((2 * NB) % NW == 0 && BJ >= 1 && AHEAD >= 2 && C * (AHEAD - 1) <= 63, "tile shape");
    static_assert(!GLU || IF % 2 == 0, "gate and up row blocks");
    // after the loop: the scales, then each wave's bf16 rows (16 bytes of
    // padding each), all its token blocks at once where they fit
    constexpr int NS = TF + TT, kStageAt = NS * 4, RS = 16 * OI + 8;
    constexpr int kRing = S * kStageBytes, kLds = KG * kRing;
    constexpr int JB = kStageAt + NW * KG * BE * 16 * RS * 2 <= kLds ? BE : BE / 2;
    static_assert(kStageAt % 16 == 0 && kStageAt + NW * KG * JB * 16 * RS * 2 <= kLds && BE % JB == 0, "epilogue");
    static_assert(kLds <= 160 * 1024 && BJ % KG == 0 && (KG == 1 || KG * NW * IF * BE * 1024 <= kLds), "LDS");
    __shared__ __attribute__((aligned(1024))) uint8_t lds[kLds];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kg = KG == 1 ? 0 : wave / NW, wg = KG == 1 ? wave : wave % NW;  // k group, wave of it
    const int grp = lane >> 4, c = lane & 15;
    const I8Gemm &g = a.g;
    int tf, tt;
    if (!tile_of(a, tf, tt)) return;
    const int f0 = tf * OF, t0 = tt * TT, stages = g.k / kBK;
    // a group's stages: kg, kg + KG, ..., of which the last may lie past the end
    const int kt = (stages + KG - 1) / KG;
    const bool last = KG == 1 || KG * (kt - 1) + kg < stages;

    // The scales of the tile's features (gate, then up) and tokens, one or two a
    // thread, loaded here and handed over through LDS once the ring is idle.
    constexpr int PS = (NS + NT - 1) / NT;
    float sc[PS];
#pragma unroll
    for (int p = 0; p < PS; p++) {
        const int q = tid + NT * p;
        if (q < OF) sc[p] = g.ws[min(f0 + q, g.n - 1)];
        else if (GLU && q < TF) sc[p] = g.us[min(f0 + q - OF, g.n - 1)];
        else sc[p] = g.xs[min(t0 + min(q - TF, TT - 1), g.m - 1)];
    }

    // Staging: wave w issues loads g = C w + [0, C) of a stage, load g the half
    // h = g & 1 of row block gb = g >> 1.  The block's 16 slot groups of 128 bytes
    // hold its rows in the order 0, 8, 1, 9, ..., 7, 15: group ga = 8 h + (l >> 3)
    // holds row (ga >> 1) + 8 (ga & 1), lane l taking that row's 16-byte piece
    // (l & 7) ^ (ga >> 1), so that row c (i = c >> 3, r = c & 7) keeps piece p in
    // slot 16 r + 8 i + (p ^ r).
    uint32_t voff[C];
    const int8_t *sbase[C];
    const int8_t *wt0 = g.w + (size_t)f0 * g.k, *ut0 = GLU ? g.up + (size_t)f0 * g.k : nullptr;
    const int8_t *xt0 = g.x + (size_t)t0 * g.k;
#pragma unroll
    for (int j = 0; j < C; j++) {
        const int l = wg * C + j, gb = l >> 1, h = l & 1;
        const int ga = 8 * h + (lane >> 3);
        const int rl = (ga >> 1) + 8 * (ga & 1);
        const int piece = (lane & 7) ^ (ga >> 1);
        const bool isw = gb < NBF;
        // a wave's blocks: gate and up of the same OI output blocks
        const int i = gb % IF, ob = GLU ? gb / IF * OI + i % OI : gb;
        const int row = isw ? min(16 * ob + rl, g.n - 1 - f0) : min(16 * (gb - NBF) + rl, g.m - 1 - t0);
        voff[j] = (uint32_t)row * (uint32_t)g.k + 16 * piece;
        sbase[j] = !isw ? xt0 : GLU && i >= OI ? ut0 : wt0;
    }
    uint8_t *const ring = lds + kg * kRing;
    const uint32_t lds0 = lds_addr(lds) + kg * kRing + wg * C * kFrag;
    // copy j of stage t into its ring slot t % S.  Stages past the last copy the
    // last stage's rows again: their slots are never read, every iteration issues
    // C copies, and the waits and the loop have no branch.
    auto copy = [&](int t, int j) __attribute__((always_inline)) {
        lds_dma16_sv(sbase[j] + min(KG * t + kg, stages - 1) * kBK, voff[j], lds0 + (t % S) * kStageBytes + j * kFrag);
    };
    // A stage's copies are spread over the MFMA rows of two steps: [0, CB) in
    // the step after the barrier that frees its slot, [CB, C) in the next one
    // (all in the first with two stages ahead, where the next wait lands them).
    constexpr int CB = AHEAD > 2 ? (C + 1) / 2 : C;
    auto first_half = [&](int t) __attribute__((always_inline)) {
        return [&, t](int i) __attribute__((always_inline)) {
#pragma unroll
            for (int j = i * CB / IF; j < (i + 1) * CB / IF; j++) copy(t, j);
        };
    };
    auto second_half = [&](int t) __attribute__((always_inline)) {
        return [&, t](int i) __attribute__((always_inline)) {
#pragma unroll
            for (int j = CB + i * (C - CB) / IF; j < CB + (i + 1) * (C - CB) / IF; j++) copy(t, j);
        };
    };
    // Operand reads: lane (grp, c) takes row c, k 16 grp + [0, 16) of step ks,
    // i.e. piece 4 ks + grp, at byte off[ks] of each row block.
    uint32_t off[2];
#pragma unroll
    for (int ks = 0; ks < 2; ks++) {
        const int i = c >> 3, r = c & 7;
        off[ks] = 16 * (16 * r + 8 * i + ((4 * ks + grp) ^ r));
    }

    const int wf = wg & 1, wt = wg >> 1;
    i32x4 acc[IF][BJ];
#pragma unroll
    for (int i = 0; i < IF; i++)
#pragma unroll
        for (int j = 0; j < BJ; j++) acc[i][j] = i32x4{0, 0, 0, 0};

    // A wave's copies (C a stage) retire in order, so a wait for at most C n
    // outstanding copies lands all but the last n stages issued.
#pragma unroll
    for (int t = 0; t < AHEAD - 1; t++)
#pragma unroll
        for (int j = 0; j < C; j++) copy(t, j);
#pragma unroll
    for (int j = 0; j < CB; j++) copy(AHEAD - 1, j);
    wait_vm<C * (AHEAD - 2) + CB>();
    asm volatile("s_barrier" ::: "memory");
    i32x4 w[IF], ax[BJ], bx[BJ];
#pragma unroll
    for (int i = 0; i < IF; i++) w[i] = *(const i32x4 *)(ring + off[0] + (IF * wf + i) * kPair);
#pragma unroll
    for (int j = 0; j < BJ; j++) ax[j] = *(const i32x4 *)(ring + off[0] + (NBF + BJ * wt + j) * kPair);

    // The last stage is peeled, so that the accumulators meet no branch.
    for (int s = 0; s < kt - 1; s++) {
        // step (s, 0): its operands in (w, ax); read step (s, 1) into (w, bx);
        // the second half of stage s - 1 + AHEAD
        substep<IF, BJ>(w, ax, ring + (s % S) * kStageBytes, off[1], wf, wt, bx, acc, second_half(s - 1 + AHEAD));
        // stage s + 1 landed: AHEAD - 2 later ones may stay in flight
        wait_vm<C * (AHEAD - 2), LGKM>();
        asm volatile("s_barrier" ::: "memory");
        // step (s, 1): operands in (w, bx); read step (s + 1, 0) into (w, ax);
        // the first half of stage s + AHEAD
        substep<IF, BJ>(w, bx, ring + ((s + 1) % S) * kStageBytes, off[0], wf, wt, ax, acc, first_half(s + AHEAD));
    }
    if (last) {
        substep<IF, BJ>(w, ax, ring + ((kt - 1) % S) * kStageBytes, off[1], wf, wt, bx, acc, [](int) {});
#pragma unroll
        for (int i = 0; i < IF; i++)
#pragma unroll
            for (int j = 0; j < BJ; j++) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[i], bx[j], acc[i][j], 0, 0, 0);
    }
    wait_vm<0>();     // the copies past the last stage have landed before the ring is reused or freed
    __syncthreads();  // every wave's operand reads are done

    // The groups' sums meet: of the token blocks of a wave and the wave of the
    // other group over the same ones each hands the other half over and writes
    // its own.
    i32x4 sum[IF][BE];
    if constexpr (KG == 1) {
#pragma unroll
        for (int i = 0; i < IF; i++)
#pragma unroll
            for (int j = 0; j < BE; j++) sum[i][j] = acc[i][j];
    } else {
        static_assert(KG == 2, "two groups");
        i32x4 *mine = (i32x4 *)lds + (size_t)wave * IF * BE * 64 + lane;
        const i32x4 *others = (const i32x4 *)lds + (size_t)(wave ^ NW) * IF * BE * 64 + lane;
#pragma unroll
        for (int i = 0; i < IF; i++)
#pragma unroll
            for (int j = 0; j < BE; j++) {
                mine[(i * BE + j) * 64] = kg ? acc[i][j] : acc[i][BE + j];
                sum[i][j] = kg ? acc[i][BE + j] : acc[i][j];
            }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < IF; i++)
#pragma unroll
            for (int j = 0; j < BE; j++) sum[i][j] += others[(i * BE + j) * 64];
        __syncthreads();
    }
    float *scales = (float *)lds;
#pragma unroll
    for (int p = 0; p < PS; p++)
        if (tid + NT * p < NS) scales[tid + NT * p] = sc[p];
    __syncthreads();

    // Each wave writes its own part of the tile, a block of 16 tokens at a time.
    // chunks: the output's rows are whole 16-byte chunks, which are inside it or
    // not; whole: the part lies inside the output (its writes have no branch).
    const int fw = f0 + (OF / 2) * wf, tl = (TT / WT) * wt + 16 * BE * kg, tw = t0 + tl;
    const bool chunks = a.vec && g.n % (OUT == kBf16 || GLU ? 8 : 4) == 0;
    const bool whole = a.vec && fw + OF / 2 <= g.n && tw + 16 * BE <= g.m;
    float4 ws[OI], us[GLU ? OI : 1];
#pragma unroll
    for (int i = 0; i < OI; i++) {
        ws[i] = *(const float4 *)(scales + (OF / 2) * wf + 16 * i + 4 * grp);
        if constexpr (GLU) us[i] = *(const float4 *)(scales + OF + (OF / 2) * wf + 16 * i + 4 * grp);
    }
    if constexpr (OUT == kBf16 || GLU) {
        // through LDS as [token][feature] rows, then whole rows, 16 bytes a
        // lane (the wave's own rows: no barrier)
        constexpr int CPR = 2 * OI, NQ = JB * 16 * CPR;  // 16-byte chunks of a row, of a batch
        uint16_t *st = (uint16_t *)(lds + kStageAt) + wave * JB * 16 * RS;
#pragma unroll
        for (int j0 = 0; j0 < BE; j0 += JB) {
            asm volatile("" ::: "memory");  // the rows change hands between the wave's lanes
#pragma unroll
            for (int j = j0; j < j0 + JB; j++) {
                const float xs = scales[TF + tl + 16 * j + c];
#pragma unroll
                for (int i = 0; i < OI; i++) {
                    const i32x4 v = sum[i][j];
                    float o[4];
                    if constexpr (GLU) {
                        const i32x4 u = sum[i + OI][j];
                        o[0] = glu(v[0], u[0], ws[i].x, us[i].x, xs);
                        o[1] = glu(v[1], u[1], ws[i].y, us[i].y, xs);
                        o[2] = glu(v[2], u[2], ws[i].z, us[i].z, xs);
                        o[3] = glu(v[3], u[3], ws[i].w, us[i].w, xs);
                    } else {
                        o[0] = scaled(v[0], ws[i].x) * xs;
                        o[1] = scaled(v[1], ws[i].y) * xs;
                        o[2] = scaled(v[2], ws[i].z) * xs;
                        o[3] = scaled(v[3], ws[i].w) * xs;
                    }
                    *(uint2 *)(st + (16 * (j - j0) + c) * RS + 16 * i + 4 * grp) = make_uint2(pack2(o[0], o[1]), pack2(o[2], o[3]));
                }
            }
            asm volatile("" ::: "memory");
#pragma unroll
            for (int q0 = 0; q0 < NQ; q0 += 64) {
                const int q = q0 + lane, row = q / CPR, col = q - row * CPR;
                if (NQ % 64 != 0 && q >= NQ) continue;
                const int t = tw + 16 * j0 + row, f = fw + 8 * col;
                const uint16_t *from = st + row * RS + 8 * col;
                uint16_t *y = (uint16_t *)g.y + (size_t)t * g.ldy + f;
                if (whole) {
                    *(uint4 *)y = *(const uint4 *)from;
                } else if (chunks) {
                    if (t < g.m && f < g.n) *(uint4 *)y = *(const uint4 *)from;
                } else if (t < g.m) {
                    for (int e = 0; e < 8; e++)
                        if (f + e < g.n) y[e] = from[e];
                }
            }
        }
    } else if (whole || chunks) {
        float *y = (float *)g.y + (size_t)(tw + c) * g.ldy + fw + 4 * grp;
        const size_t step = (size_t)16 * g.ldy;
        auto write = [&](auto all) __attribute__((always_inline)) {
            auto inside = [&](int i, int j) __attribute__((always_inline)) {
                return decltype(all)::value || (tw + 16 * j + c < g.m && fw + 16 * i + 4 * grp < g.n);
            };
#pragma unroll
            for (int j = 0; j < BE; j++) {
                const float xs = scales[TF + tl + 16 * j + c];
                float4 old[OUT == kAcc ? IF : 1];
                if constexpr (OUT == kAcc)
#pragma unroll
                    for (int i = 0; i < IF; i++)
                        if (inside(i, j)) old[i] = *(const float4 *)(y + j * step + 16 * i);
#pragma unroll
                for (int i = 0; i < IF; i++) {
                    const i32x4 v = sum[i][j];
                    const float o[4] = {scaled(v[0], ws[i].x), scaled(v[1], ws[i].y), scaled(v[2], ws[i].z),
                                        scaled(v[3], ws[i].w)};
                    float4 r = make_float4(o[0] * xs, o[1] * xs, o[2] * xs, o[3] * xs);
                    if constexpr (OUT == kAcc)
                        r = make_float4(fmaf(o[0], xs, old[i].x), fmaf(o[1], xs, old[i].y), fmaf(o[2], xs, old[i].z),
                                        fmaf(o[3], xs, old[i].w));
                    if (inside(i, j)) *(float4 *)(y + j * step + 16 * i) = r;
                }
            }
        };
        if (whole) write(std::true_type{});
        else write(std::false_type{});
    } else {
#pragma unroll
        for (int j = 0; j < BE; j++) {
            const int t = tw + 16 * j + c;
            if (t >= g.m) continue;
            const float xs = scales[TF + tl + 16 * j + c];
#pragma unroll
            for (int i = 0; i < OI; i++) {
                const float w4[4] = {ws[i].x, ws[i].y, ws[i].z, ws[i].w};
                store4<OUT>(a, t, fw + 16 * i + 4 * grp, sum[i][j], sum[i][j], w4, w4, xs);
            }
        }
    }
}

// ---- few tokens ----------------------------------------------------------------
//
// A workgroup owns 16 A features x 16 B tokens and its four waves split k: each
// streams its own quarter of the tile's W and x rows through an LDS ring of its
// own, so there is no barrier before the end and four load streams run per
// workgroup.  The four partial tiles meet in LDS.  Bound by the stream of W (one
// token, 120818 channels: 39 us, 6.3 TB/s) or, where that is short, by a launch, the
// way of the operands and that of the scales, which are loaded after the last
// stage (one token, 2048 x 2048: 2.9 us in a recording, 4.0 with W cold).  Deeper
// rings and eight waves a workgroup were no faster at 1-700 tokens, nor was W
// straight into registers.  SwiGLU: the first A / 2 row
// blocks are gate rows, the others the same rows of up.
// ONCE: W goes past the caches (nt), where each of its rows is read by one
// workgroup alone and it is too large to be found in the L2s by the next call
// anyway (reads_once).
template <int A, int B, int S, bool ONCE, int OUT>
__global__ __launch_bounds__(256) void skinny_kernel(Args a) {
    constexpr bool GLU = OUT == kGlu;
    constexpr int C = 2 * (A + B);  // copies (1 KiB each) of a stage
    constexpr int kStage = C * 1024, kRing = S * kStage;
    constexpr int AO = GLU ? A / 2 : A;                         // output row blocks
    constexpr int Q = AO * B * 64, NQ = (Q + 255) / 256;        // 4-feature outputs, per thread
    static_assert(4 * kRing <= 160 * 1024 && C * (S - 1) <= 63, "ring");
    static_assert(A * B * 1024 <= kRing, "a wave's partial tile is handed over in its ring");
    static_assert(!GLU || A % 2 == 0, "gate and up row blocks");
    __shared__ __attribute__((aligned(1024))) uint8_t lds[4 * kRing];
    const I8Gemm &g = a.g;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int grp = lane >> 4, c = lane & 15;
    // each XCD takes a contiguous run of tiles, the token tiles of one W slab
    // next to each other: a slab is read from HBM into one L2
    const int L = (blockIdx.x & 7) * a.per_xcd + (blockIdx.x >> 3);
    if (L >= a.tiles) return;
    const int tf = L / a.tiles_t, tt = L - tf * a.tiles_t;
    const int f0 = tf * 16 * AO, t0 = tt * 16 * B;

    uint32_t voff[C];
#pragma unroll
    for (int l = 0; l < C; l++) {
        const int gb = l >> 1, ga = 8 * (l & 1) + (lane >> 3);
        const int rl = (ga >> 1) + 8 * (ga & 1), piece = (lane & 7) ^ (ga >> 1);
        const int row = gb < A ? min(16 * (GLU && gb >= AO ? gb - AO : gb) + rl, g.n - 1 - f0)
                               : min(16 * (gb - A) + rl, g.m - 1 - t0);
        voff[l] = (uint32_t)row * (uint32_t)g.k + 16 * piece;
    }
    // this wave's stages: a quarter of them, one more or less
    const int kt = g.k / kBK, s0 = kt * wave / 4, n = kt * (wave + 1) / 4 - s0;
    const int8_t *wb = g.w + (size_t)f0 * g.k + s0 * kBK;
    const int8_t *ub = GLU ? g.up + (size_t)f0 * g.k + s0 * kBK : nullptr;
    const int8_t *xb = g.x + (size_t)t0 * g.k + s0 * kBK;
    const uint32_t ring = lds_addr(lds) + wave * kRing;
    auto copy = [&](int t, int slot) __attribute__((always_inline)) {
#pragma unroll
        for (int l = 0; l < C; l++) {
            const int gb = l >> 1;
            const int8_t *from = (gb >= A ? xb : GLU && gb >= AO ? ub : wb) + t * kBK;
            const uint32_t to = ring + slot * kStage + l * 1024;
            if (ONCE && gb < A) lds_dma16_sv_nt(from, voff[l], to);
            else lds_dma16_sv(from, voff[l], to);
        }
    };
    uint32_t off[2];
#pragma unroll
    for (int ks = 0; ks < 2; ks++) off[ks] = 16 * (16 * (c & 7) + 8 * (c >> 3) + ((4 * ks + grp) ^ (c & 7)));

    i32x4 acc[A][B];
#pragma unroll
    for (int i = 0; i < A; i++)
#pragma unroll
        for (int j = 0; j < B; j++) acc[i][j] = i32x4{0, 0, 0, 0};
    const uint8_t *my = lds + wave * kRing;
    i32x4 w[2][A], x[2][B];
    int slot = 0;
    auto read = [&]() __attribute__((always_inline)) {
        const uint8_t *p = my + slot * kStage;
#pragma unroll
        for (int ks = 0; ks < 2; ks++) {
#pragma unroll
            for (int i = 0; i < A; i++) w[ks][i] = *(const i32x4 *)(p + off[ks] + i * kPair);
#pragma unroll
            for (int j = 0; j < B; j++) x[ks][j] = *(const i32x4 *)(p + off[ks] + (A + j) * kPair);
        }
    };
    auto mma = [&](int ks) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < A; i++)
#pragma unroll
            for (int j = 0; j < B; j++)
                acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[ks][i], x[ks][j], acc[i][j], 0, 0, 0);
    };
    // A wave's copies retire in order: a stage has landed once at most S - 1
    // younger stages are outstanding.  Its slot is refilled as soon as this wave
    // has its operands in registers; no other wave touches the ring.
#pragma unroll
    for (int t = 0; t < S; t++)
        if (t < n) copy(t, t);
    for (int t = S; t < n; t++) {
        wait_vm<(S - 1) * C>();
        read();
        mma(0);
        __builtin_amdgcn_sched_barrier(0);
        wait_lgkm();
        copy(t, slot);
        __builtin_amdgcn_sched_barrier(0);
        mma(1);
        slot = slot + 1 == S ? 0 : slot + 1;
    }
    // the last S stages (or all, where there are fewer), nothing left to issue
    const int left = min(S, n);
#pragma unroll
    for (int l = S; l > 0; l--)
        if (l <= left) {
            if (l == 4) wait_vm<(S > 3 ? 3 : 0) * C>();
            else if (l == 3) wait_vm<(S > 2 ? 2 : 0) * C>();
            else if (l == 2) wait_vm<(S > 1 ? 1 : 0) * C>();
            else wait_vm<0>();
            read();
            mma(0);
            mma(1);
            slot = slot + 1 == S ? 0 : slot + 1;
        }
    wait_lgkm();

#pragma unroll
    for (int i = 0; i < A; i++)
#pragma unroll
        for (int j = 0; j < B; j++) *(i32x4 *)(lds + wave * kRing + (64 * (i * B + j) + lane) * 16) = acc[i][j];
    __syncthreads();
    auto sum = [&](int q) __attribute__((always_inline)) {
        i32x4 s = *(const i32x4 *)(lds + q * 16);
#pragma unroll
        for (int p = 1; p < 4; p++) s += *(const i32x4 *)(lds + p * kRing + q * 16);
        return s;
    };
#pragma unroll
    for (int u = 0; u < NQ; u++) {
        const int q = tid + 256 * u, fr = q >> 6, i = fr / B, j = fr - i * B;
        const int f = f0 + 16 * i + 4 * grp, t = t0 + 16 * j + c;
        if (q >= Q || t >= g.m || f >= g.n) continue;
        float ws[4], us[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            ws[e] = g.ws[min(f + e, g.n - 1)];
            us[e] = GLU ? g.us[min(f + e, g.n - 1)] : 0.f;
        }
        const i32x4 s = sum(q);
        store4<OUT>(a, t, f, s, GLU ? sum(q + Q) : s, ws, us, g.xs[t]);
    }
}

// ---- which kernel --------------------------------------------------------------

// The tiles: features x tokens (SwiGLU: half as many outputs) and what a launch
// of `tiles` of them takes, us =
//   launch + R (round + stage kt) + F (fill + fill_stage kt),
// R = ceil(tiles / 256) rounds of the chip, F = tiles / 256 (what grows with the traffic of
// all CUs together), kt = k / 128.  Fitted to 1558 measurements: 1-4096 tokens, 64-120818
// channels, k 256-8192, every output; the tile of the least estimate takes 0.5 %
// longer on average than the fastest one (worst 21 %: SwiGLU, 178 x 3606 x 768).  E.g.,
// us estimated / measured: 2048 x 2048 x 2048 bf16 128 x 128 13.8 / 12.0, 128 x 64 18.4 /
// 15.2; 700 x 2048 x 6144 bf16 96 x 64 17.0 / 15.4, 128 x 64 18.3 / 16.5.  (It knows nothing
// of HBM: one token of 120818 channels takes 39 us, not 20; the order of the tiles
// holds.)
struct Shape {
    const char *name;
    int f, t, threads;
    int glu;  // 0: any output, 1: SwiGLU only, 2: the others only
    float launch, round, stage, fill, fill_stage;
};
constexpr Shape kShapes[] = {
    {"16x16", 16, 16, 256, 2, 2.43f, 0.21f, 0.028f, 0.14f, 0.018f},
    {"32x16", 32, 16, 256, 0, 2.57f, 0.13f, 0.044f, 0.28f, 0.022f},
    {"48x16", 48, 16, 256, 2, 2.75f, 0.00f, 0.059f, 0.45f, 0.028f},
    {"64x16", 64, 16, 256, 0, 2.84f, 0.00f, 0.077f, 0.49f, 0.029f},
    {"32x32", 32, 32, 256, 0, 2.63f, 0.17f, 0.058f, 0.33f, 0.034f},
    {"64x32", 64, 32, 256, 0, 2.22f, 0.98f, 0.096f, 0.60f, 0.058f},
    {"64x64", 64, 64, 512, 0, 2.44f, 1.12f, 0.124f, 1.16f, 0.070f},
    {"96x64", 96, 64, 256, 1, 2.50f, 1.79f, 0.206f, 1.12f, 0.068f},
    {"96x64", 96, 64, 512, 2, 2.49f, 1.44f, 0.168f, 1.66f, 0.076f},
    {"128x64", 128, 64, 512, 0, 3.10f, 0.79f, 0.227f, 2.29f, 0.058f},
    {"128x96", 128, 96, 256, 0, 3.02f, 0.94f, 0.308f, 2.04f, 0.052f},
    {"128x128", 128, 128, 256, 0, 3.36f, 1.23f, 0.375f, 2.32f, 0.053f},
    {"192x128", 192, 128, 512, 0, 3.78f, 1.51f, 0.452f, 3.22f, 0.123f},
    {"256x128", 256, 128, 256, 0, 4.78f, 1.92f, 0.641f, 3.87f, 0.089f},
    {"192x256", 192, 256, 512, 0, 4.50f, 2.00f, 0.896f, 4.99f, 0.140f},
    {"256x256", 256, 256, 512, 0, 6.93f, 0.87f, 0.994f, 6.18f, 0.299f},
};
constexpr int kNumShapes = sizeof(kShapes) / sizeof(kShapes[0]);
constexpr size_t kMaxTiles = 1u << 22;  // of a launch: a grid holds less than 2^32 threads

size_t tiles_of(const Shape &p, const I8Gemm &g, bool glu) {
    const int of = glu ? p.f / 2 : p.f;
    return (size_t)((g.n + of - 1) / of) * ((g.m + p.t - 1) / p.t);
}

// The tile of the least estimated time; HYMT_HIP_I8_TILE=<tile> forces one (a
// tuning knob) on the outputs that it serves: SwiGLU takes the tiles whose row
// blocks split into gate and up.
int plan(const I8Gemm &g, bool glu) {
    const char *forced = std::getenv("HYMT_HIP_I8_TILE");
    if (forced && !gemm_i8_tile_known()) return -1;
    const float kt = (float)(g.k / kBK);
    int best = -1;
    float least = 0.f;
    for (int i = 0; i < kNumShapes; i++) {
        const Shape &p = kShapes[i];
        const size_t tiles = tiles_of(p, g, glu);
        if (tiles > kMaxTiles || p.glu == (glu ? 2 : 1)) continue;
        if (forced && !std::strcmp(forced, p.name)) return i;
        const float rounds = (float)((tiles + 255) / 256), fill = (float)tiles / 256.f;
        const float us = p.launch + rounds * (p.round + p.stage * kt) + fill * (p.fill + p.fill_stage * kt);
        if (best < 0 || us < least) {
            best = i;
            least = us;
        }
    }
    return best;
}

template <int OUT>
void launch_shape(int i, const Args &a, const KernelSpan &span, hipStream_t s) {
    const dim3 grid(8 * a.per_xcd), block(kShapes[i].threads);
    constexpr bool GLU = OUT == kGlu;
    switch (i) {
    case 0:
        if constexpr (!GLU) launch(span, skinny_kernel<1, 1, 4, false, OUT>, grid, block, 0, s, a);
        break;
    case 1: launch(span, skinny_kernel<2, 1, 3, false, OUT>, grid, block, 0, s, a); break;
    case 2:
        if constexpr (!GLU) launch(span, skinny_kernel<3, 1, 2, false, OUT>, grid, block, 0, s, a);
        break;
    case 3: launch(span, skinny_kernel<4, 1, 2, false, OUT>, grid, block, 0, s, a); break;
    case 4: launch(span, skinny_kernel<2, 2, 2, false, OUT>, grid, block, 0, s, a); break;
    case 5: launch(span, skinny_kernel<4, 2, 2, false, OUT>, grid, block, 0, s, a); break;
    case 6: launch(span, tile_kernel<2, 2, 2, 4, true, 2, OUT>, grid, block, 0, s, a); break;
    case 7:
        if constexpr (GLU) launch(span, skinny_kernel<6, 4, 2, false, OUT>, grid, block, 0, s, a);
        break;
    case 8:
        if constexpr (!GLU) launch(span, tile_kernel<3, 2, 2, 4, true, 2, OUT>, grid, block, 0, s, a);
        break;
    case 9: launch(span, tile_kernel<4, 2, 2, 3, true, 2, OUT>, grid, block, 0, s, a); break;
    case 10: launch(span, tile_kernel<4, 3, 2, 4, false, 1, OUT>, grid, block, 0, s, a); break;
    case 11: launch(span, tile_kernel<4, 4, 2, 4, false, 1, OUT>, grid, block, 0, s, a); break;
    case 12: launch(span, tile_kernel<6, 4, 4, 4, true, 1, OUT>, grid, block, 0, s, a); break;
    case 13: launch(span, tile_kernel<8, 4, 2, 3, true, 1, OUT>, grid, block, 0, s, a); break;
    case 14: launch(span, tile_kernel<6, 8, 4, 2, true, 1, OUT>, grid, block, 0, s, a); break;
    default: launch(span, tile_kernel<8, 8, 4, 2, true, 1, OUT>, grid, block, 0, s, a); break;
    }
}

// Whether the few-token kernel's W copies pass the caches: one token tile, so that
// a row of W is read once, and 8 MiB of W or more.  us through the caches / past
// them, over sets of weights of 0.6 GB (cold) and over three sets: 1 x 2048 x 6144
// cold 5.55 / 4.79, three 4.60 / 4.27; 16 x 2048 x 6144 cold 6.85 / 6.49, three 5.01 / 5.43;
// 1 x 6144 x 2048 5.36 / 4.46, 4.75 / 3.90; 1 x 12288 x 2048 7.37 / 6.29, 6.24 / 5.71; 1 x
// 120818 x 2048 44.4 / 39.2; SwiGLU 1 x 6144 x 2048 7.51 / 6.50, 6.38 / 5.88.  Below 8 MiB three
// sets stay in the L2s and take the same either way.
bool reads_once(int i, const Args &a, bool glu) {
    return i < 4 && a.tiles_t == 1 && (size_t)a.g.n * a.g.k * (glu ? 2 : 1) >= (8u << 20);
}

template <int OUT>
void launch_once(int i, const Args &a, const KernelSpan &span, hipStream_t s) {
    const dim3 grid(8 * a.per_xcd), block(kShapes[i].threads);
    constexpr bool GLU = OUT == kGlu;
    switch (i) {
    case 0:
        if constexpr (!GLU) launch(span, skinny_kernel<1, 1, 4, true, OUT>, grid, block, 0, s, a);
        break;
    case 1: launch(span, skinny_kernel<2, 1, 3, true, OUT>, grid, block, 0, s, a); break;
    case 2:
        if constexpr (!GLU) launch(span, skinny_kernel<3, 1, 2, true, OUT>, grid, block, 0, s, a);
        break;
    default: launch(span, skinny_kernel<4, 1, 2, true, OUT>, grid, block, 0, s, a); break;
    }
}

bool fits(const I8Gemm &g) {
    auto a16 = [](const void *p) { return ((uintptr_t)p & 15u) == 0; };
    return g.n > 0 && g.m >= 0 && g.n <= kI8MaxRows && g.m <= kI8MaxRows && g.k >= 2 * kI8StepK && g.k <= kI8MaxK &&
           g.k % kI8StepK == 0 && g.ldy >= g.n && a16(g.w) && a16(g.x) && a16(g.up);
}

template <int OUT>
hipError_t run(const I8Gemm &g, const char *name, hipStream_t s) {
    if (!fits(g)) return hipErrorInvalidValue;
    if (g.m == 0) return hipSuccess;
    const int i = plan(g, OUT == kGlu);
    if (i < 0) return hipErrorInvalidValue;  // more tiles than a launch holds, or no such tile
    const int of = OUT == kGlu ? kShapes[i].f / 2 : kShapes[i].f;
    Args a{};
    a.g = g;
    a.tiles_f = (g.n + of - 1) / of;
    a.tiles_t = (g.m + kShapes[i].t - 1) / kShapes[i].t;
    a.tiles = a.tiles_f * a.tiles_t;
    a.per_xcd = (a.tiles + 7) / 8;
    constexpr int es = OUT == kBf16 || OUT == kGlu ? 2 : 4;
    a.vec = ((uintptr_t)g.y & 15u) == 0 && g.ldy % (16 / es) == 0;
    KernelSpan span(name, s, true);
    if (reads_once(i, a, OUT == kGlu)) launch_once<OUT>(i, a, span, s);
    else launch_shape<OUT>(i, a, span, s);
    return hipGetLastError();
}

}  // namespace

bool gemm_i8_launches(const I8Gemm &g) {
    // no tile makes fewer than the last, the largest
    return tiles_of(kShapes[kNumShapes - 1], g, g.up != nullptr) <= kMaxTiles;
}

bool gemm_i8_tile_known() {
    const char *forced = std::getenv("HYMT_HIP_I8_TILE");
    if (!forced) return true;
    for (const Shape &p : kShapes)
        if (!std::strcmp(forced, p.name)) return true;
    return false;
}

hipError_t launch_gemm_i8(const I8Gemm &g, I8Out out, hipStream_t s) {
    if (out == kI8Bf16) return run<kBf16>(g, "gemm_i8_out_bf16", s);
    if (out == kI8Acc) return run<kAcc>(g, "gemm_i8_out_f32", s);
    return run<kF32>(g, "gemm_i8_out_f32", s);
}

hipError_t launch_gemm_i8_swiglu(const I8Gemm &g, hipStream_t s) {
    if (!g.up) return hipErrorInvalidValue;
    return run<kGlu>(g, "gemm_i8_swiglu", s);
}

}  // namespace hymt
