// rows_i8.hip -- rows as int8 codes with a scale each (gfx950): of fp32 or bf16
// values, and of the RMSNorm of the residual rows after an addition.
//
// The codes of a row v: with a = max|v|, q = rint(127 v / a), ties to even, and
// scale = a / 127.  Of a norm v = x w / sqrt(mean(x^2) + eps) the root is common to
// v and a, so q = rint(127 x w / max|x w|) needs no statistics, and only the
// scale has the root: a / (127 sqrt(mean(x^2) + eps)).
//
// The codes are those of exact arithmetic: x w is formed in fp64 (exact: 48
// bits) and so are the maximum and the quotient.  In fp32 a value within a few
// ulps of a border would take the one code or the other by the order of the
// roundings.  A quotient is a product with 127 / a, and only where that lands
// within 1e-9 of a border (ties of bf16 rows: a half of the maximum is 63.5) a
// division.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "device_common.hpp"
#include "int8.hpp"
#include "ktimer.hpp"

namespace hymt {
namespace {

enum Kind { kF32, kBf16, kNorm, kNormAddBf16, kNormAddF32 };

struct RowsArgs {
    const void *x;     // fp32 (kNormAdd*: written too) or bf16
    const void *add;   // kNormAdd*
    const float *w;    // kNorm*
    float eps;
    int m, n;
    int8_t *out;
    float *scale;
};

__device__ __forceinline__ int code_of(double v, double a, double r) {
    const double s = v * r;
    double q = rint(s);
    if (fabs(fabs(s - q) - 0.5) < 1e-9) q = rint(v * 127.0 / a);
    return (int)q;
}

__device__ __forceinline__ float4 load4_bf16(const uint16_t *p) {
    const uint2 b = *(const uint2 *)p;
    return make_float4(bf16_to_f32(b.x & 0xFFFF), bf16_to_f32(b.x >> 16), bf16_to_f32(b.y & 0xFFFF),
                       bf16_to_f32(b.y >> 16));
}

// WPR waves of a workgroup of 4 take a row of n <= 256 WPR NJ values, 4 values
// of a lane at a time, held in registers between the two passes.
template <int KIND, int WPR, int NJ>
__global__ __launch_bounds__(256) void rows_i8_kernel(RowsArgs a) {
    constexpr bool NORM = KIND >= kNorm, ADD = KIND >= kNormAddBf16;
    const int tid = threadIdx.x, wave = tid >> 6;
    const int row = blockIdx.x * (4 / WPR) + (WPR == 1 ? wave : 0);
    const int i0 = WPR == 1 ? (tid & 63) : tid, n4 = a.n / 4;
    const bool live = row < a.m;
    const size_t base = (size_t)(live ? row : a.m - 1) * a.n;
    float4 v[NJ], g[NJ];
#pragma unroll
    for (int j = 0; j < NJ; j++) {
        const size_t e = base + 4 * min(i0 + 64 * WPR * j, n4 - 1);
        if constexpr (KIND == kBf16) v[j] = load4_bf16((const uint16_t *)a.x + e);
        else v[j] = *(const float4 *)((const float *)a.x + e);
        if constexpr (ADD) {
            const float4 d = KIND == kNormAddBf16 ? load4_bf16((const uint16_t *)a.add + e)
                                                  : *(const float4 *)((const float *)a.add + e);
            v[j] = make_float4(v[j].x + d.x, v[j].y + d.y, v[j].z + d.z, v[j].w + d.w);
        }
        if constexpr (NORM) g[j] = ((const float4 *)a.w)[min(i0 + 64 * WPR * j, n4 - 1)];
        // past the row's end: zeros, whatever was loaded there (the row's last
        // values, which another wave may already have written with the addition)
        if (i0 + 64 * WPR * j >= n4) v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    double top = 0.0, ss = 0.0;
    bool bad = false;
    auto val = [&](int j, int e) __attribute__((always_inline)) {
        const float x = e == 0 ? v[j].x : e == 1 ? v[j].y : e == 2 ? v[j].z : v[j].w;
        if constexpr (NORM) {
            const float w = e == 0 ? g[j].x : e == 1 ? g[j].y : e == 2 ? g[j].z : g[j].w;
            return (double)x * (double)w;
        }
        return (double)x;
    };
#pragma unroll
    for (int j = 0; j < NJ; j++) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const double t = fabs(val(j, e));
            bad |= !(t < __builtin_inf());
            top = t > top ? t : top;
            if constexpr (NORM) {
                const double x = e == 0 ? v[j].x : e == 1 ? v[j].y : e == 2 ? v[j].z : v[j].w;
                ss += x * x;
            }
        }
        if constexpr (ADD)
            if (live && i0 + 64 * WPR * j < n4) *(float4 *)((float *)a.x + base + 4 * (i0 + 64 * WPR * j)) = v[j];
    }
    if (bad) top = __builtin_inf();
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        const double t = __shfl_xor(top, o);
        top = t > top ? t : top;
        if constexpr (NORM) ss += __shfl_xor(ss, o);
    }
    if constexpr (WPR > 1) {
        __shared__ double red[2][4];
        if ((tid & 63) == 0) {
            red[0][wave] = top;
            red[1][wave] = ss;
        }
        __syncthreads();
        top = fmax(fmax(red[0][0], red[0][1]), fmax(red[0][2], red[0][3]));
        ss = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
    }
    if (!live) return;
    const bool none = !(top > 0.0) || top == __builtin_inf();
    const double r = 127.0 / top;
#pragma unroll
    for (int j = 0; j < NJ; j++) {
        const int i = i0 + 64 * WPR * j;
        if (i < n4) {
            uint32_t c = 0;
            if (!none)
#pragma unroll
                for (int e = 0; e < 4; e++) c |= (uint32_t)(uint8_t)code_of(val(j, e), top, r) << (8 * e);
            *(uint32_t *)(a.out + base + 4 * i) = c;
        }
    }
    if (i0 == 0) {
        double sc = top / 127.0;
        if constexpr (NORM) sc = sc / sqrt(ss / (double)a.n + (double)a.eps);
        a.scale[row] = top == __builtin_inf() ? __builtin_nanf("") : none ? 0.f : (float)sc;
    }
}

template <int KIND>
void launch_kind(const RowsArgs &a, const char *name, hipStream_t s) {
    KernelSpan span(name, s, true);
    const dim3 block(256);
    const dim3 rows4((unsigned)(((size_t)a.m + 3) / 4)), rows1((unsigned)a.m);
    if (a.n <= 512) launch(span, rows_i8_kernel<KIND, 1, 2>, rows4, block, 0, s, a);
    else if (a.n <= 2048) launch(span, rows_i8_kernel<KIND, 1, 8>, rows4, block, 0, s, a);
    else launch(span, rows_i8_kernel<KIND, 4, 8>, rows1, block, 0, s, a);
}

}  // namespace

hipError_t launch_to_i8(const void *x, bool x_bf16, int m, int n, int8_t *out, float *scale, hipStream_t s) {
    if (n % 4 != 0 || n < 4 || n > 8192 || m < 0) return hipErrorInvalidValue;
    if (m == 0) return hipSuccess;
    const RowsArgs a{x, nullptr, nullptr, 0.f, m, n, out, scale};
    if (x_bf16) launch_kind<kBf16>(a, "to_i8", s);
    else launch_kind<kF32>(a, "to_i8", s);
    return hipGetLastError();
}

hipError_t launch_rows_rmsnorm_i8(float *x, const void *add, bool add_bf16, int m, int n, const float *w, float eps,
                                  int8_t *out, float *scale, hipStream_t s) {
    if (n % 4 != 0 || n < 4 || n > 8192 || m < 0) return hipErrorInvalidValue;
    if (m == 0) return hipSuccess;
    const RowsArgs a{x, add, w, eps, m, n, out, scale};
    if (!add) launch_kind<kNorm>(a, "rows_rmsnorm_i8", s);
    else if (add_bf16) launch_kind<kNormAddBf16>(a, "rows_rmsnorm_i8", s);
    else launch_kind<kNormAddF32>(a, "rows_rmsnorm_i8", s);
    return hipGetLastError();
}

}  // namespace hymt
