// paged_attn.hip -- attention over the multi-sequence cache (hymt_paged,
// include/hymt_hip.h): a batch's packed rows, causal, and single rows behind a
// shared prefix.
#include <algorithm>

#include "attn_kernels.hpp"
#include "device_common.hpp"
#include "ktimer.hpp"
#include "paged.hpp"

namespace hymt {

namespace {

// 8 values of a 16-byte chunk in fp32.
template <typename T> __device__ __forceinline__ void chunk8(uint4 u, float *o) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int e = 0; e < 4; e++) {
        o[2 * e] = from_elem<T>((uint16_t)w[e]);
        o[2 * e + 1] = from_elem<T>((uint16_t)(w[e] >> 16));
    }
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) v = fmaxf(v, __shfl_xor(v, m));
    return v;
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m);
    return v;
}

// One wave per (row, q head): lane t takes the score of a page's position t,
// then the lanes take the dims and walk the positions.
template <typename T, int D>
__global__ __launch_bounds__(256) void attn_row_kernel(hymt_paged p, hymt_batch b, PagedAttn a) {
    __shared__ float s_q[4][D], s_w[4][kPage];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int row = blockIdx.x, head = blockIdx.y * 4 + wave;
    int entry = row, n_rows = 1, j = 0;
    if (b.cu) {
        entry = 0;
        while (entry < b.n && b.cu[entry + 1] <= row) entry++;
        if (entry < b.n) {
            n_rows = b.cu[entry + 1] - b.cu[entry];
            j = row - b.cu[entry];
        }
    }
    if (entry >= b.n || head >= a.heads) return;
    const int h = head / (a.heads / p.kv_heads);
    const int cap = p.blocks * kPage;
    auto length = [&](int slot) { return (unsigned)slot < (unsigned)p.seqs ? max(0, min(p.len[slot], cap)) : 0; };
    const int slot = b.slots[entry], slot0 = b.slots[0];
    const int len = length(slot), limit = min(len - n_rows + j + 1, len);  // positions that the row attends to
    const int common = min(a.prefix, length(slot0) / kPage * kPage) / kPage;
    const size_t row_at = (size_t)row * a.heads * D + (size_t)head * D;
    for (int d = lane; d < D; d += 64) s_q[wave][d] = from_elem<T>(((const uint16_t *)a.q)[row_at + d]);
    float m = -INFINITY, l = 0.f, acc[D / 64];
#pragma unroll
    for (int i = 0; i < D / 64; i++) acc[i] = 0.f;
    for (int blk = 0; blk * kPage < limit; blk++) {
        const int page = p.table[(size_t)(blk < common ? slot0 : slot) * p.blocks + blk];
        if ((unsigned)page >= (unsigned)p.pages) continue;
        const size_t at = (((size_t)a.layer * p.pages + page) * p.kv_heads + h) * (size_t)(kPage * D);
        const uint4 *k = (const uint4 *)((const uint16_t *)p.k + at);
        const uint4 *v = (const uint4 *)((const uint16_t *)p.v + at);
        float sc = 0.f;
        for (int c = 0; c < D / 8; c++) {
            float x[8];
            chunk8<T>(k[((lane >> 4) * (D / 8) + c) * 16 + (lane & 15)], x);
#pragma unroll
            for (int e = 0; e < 8; e++) sc += x[e] * s_q[wave][8 * c + e];
        }
        const bool on = blk * kPage + lane < limit;
        sc = on ? sc * a.scale : -INFINITY;
        const float mn = fmaxf(m, wave_max(sc));
        const float w = on ? expf(sc - mn) : 0.f;
        const float al = m == -INFINITY ? 0.f : expf(m - mn);
        l = l * al + wave_sum(w);
        m = mn;
        s_w[wave][lane] = w;
#pragma unroll
        for (int i = 0; i < D / 64; i++) acc[i] *= al;
        for (int pc = 0; pc < 8; pc++) {
#pragma unroll
            for (int i = 0; i < D / 64; i++) {
                float x[8];
                chunk8<T>(v[pc * D + lane + 64 * i], x);
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int t = v_chunk_pos(pc, e);
                    if (blk * kPage + t < limit) acc[i] += s_w[wave][t] * x[e];
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < D / 64; i++) {
        const float y = l == 0.f ? 0.f : acc[i] / l;
        ((uint16_t *)a.out)[row_at + lane + 64 * i] = a.out_dtype == HYMT_F16 ? bits_of<F16>(y) : bits_of<BF16>(y);
    }
}

template <typename T> void launch_rows_of(const hymt_paged &p, const hymt_batch &b, const PagedAttn &a, hipStream_t s) {
    const dim3 grid(b.cu ? b.rows : b.n, (a.heads + 3) / 4);
    KernelSpan span(b.cu ? "attn_packed" : "attn_shared", s, true);
    if (p.head_dim == 64) launch(span, attn_row_kernel<T, 64>, grid, dim3(256), 0, s, p, b, a);
    else launch(span, attn_row_kernel<T, 128>, grid, dim3(256), 0, s, p, b, a);
}

}  // namespace

size_t paged_attn_workspace(const hymt_paged &, const hymt_batch &, const PagedAttn &, bool) { return 0; }

hipError_t launch_attn_packed(const hymt_paged &p, const hymt_batch &b, const PagedAttn &a, float *, hipStream_t s) {
    if (b.n == 0 || (b.cu && b.rows == 0)) return hipSuccess;
    if (p.dtype == HYMT_F16) launch_rows_of<F16>(p, b, a, s);
    else launch_rows_of<BF16>(p, b, a, s);
    return hipGetLastError();
}

hipError_t launch_attn_shared(const hymt_paged &p, const hymt_batch &b, const PagedAttn &a, float *ws, hipStream_t s) {
    return launch_attn_packed(p, b, a, ws, s);
}

}  // namespace hymt
