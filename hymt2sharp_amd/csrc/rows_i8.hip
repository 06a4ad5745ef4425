// rows_i8.hip -- rows as int8 codes with a scale each (gfx950): of fp32 or bf16
// values, and of the RMSNorm of the residual rows after an addition.
//
// The codes of a row v: with a = max|v|, q = rint(127 v / a), ties to even, and
// scale = a / 127.  Of a norm v = x w / sqrt(mean(x^2) + eps) the root is common to
// v and a, so q = rint(127 x w / max|x w|) needs no statistics, and only the
// scale has the root: a / (127 sqrt(mean(x^2) + eps)).
//
// The codes are those of exact arithmetic; in fp32 alone a value within a few
// ulps of a border would take the one code or the other by the order of the
// roundings.  a is exact: fp32 for plain rows, the fp64 product (48 bits) for x w.
// A code is first rounded from the fp32 product with fp32(127 / a), which is off
// by at most 127 (2^-24 + 2^-24 + 2^-24) < 2.4e-5 (the reciprocal's rounding, x w's, and as
// much for values that x w flushes); where that lands within 6e-5 of a border,
// one value in ten thousand, the code is taken from the fp64 quotient.  Rows
// whose maximum is outside [2^-90, 2^100], where fp32 could flush or overflow, take
// the quotient throughout.  (All in fp64, 2048 x 6144 bf16 rows took 15.0 us.)
// Of plain rows the quotient decides: 127 v is exact, and the quotient of two
// 24-bit values is 1/2 + a whole number or 2^-33 away, more than fp64's 2^-46.
// Of x w, whose 127-fold has 55 bits and whose quotient may be 2^-49 away, the exact
// remainder does where the quotient is within 2^-40 of a border (2048 x 2048 after an
// addition: 9.7 us, as with the quotients alone; taken for every value near a border
// in fp32 10.0).
//
// HBM-bound: each value is read once, held in registers between the passes, and
// its code written once.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

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

constexpr float kMagic = 12582912.f;  // 1.5 2^23: an addition rounds to whole numbers, in the low bits
constexpr float kNear = 0.5f - 6e-5f;

// The maximum and the sum over a wave, in every lane: rows of 16 lanes by DPP
// (quad_perm xor 1, xor 2, half-row and row mirrors), the four rows from lanes 0,
// 16, 32 and 48.
template <int CTRL> __device__ __forceinline__ float dpp(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, false));
}
template <int CTRL> __device__ __forceinline__ double dpp(double v) {
    const int2 b = __builtin_bit_cast(int2, v);
    return __builtin_bit_cast(double, make_int2(__builtin_amdgcn_update_dpp(0, b.x, CTRL, 0xF, 0xF, false),
                                                __builtin_amdgcn_update_dpp(0, b.y, CTRL, 0xF, 0xF, false)));
}
__device__ __forceinline__ float lane_of(float v, int l) {
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), l));
}
__device__ __forceinline__ double lane_of(double v, int l) {
    const int2 b = __builtin_bit_cast(int2, v);
    return __builtin_bit_cast(double, make_int2(__builtin_amdgcn_readlane(b.x, l), __builtin_amdgcn_readlane(b.y, l)));
}
template <typename T, typename F> __device__ __forceinline__ T wave_reduce(T v, F f) {
    v = f(v, dpp<0xB1>(v));
    v = f(v, dpp<0x4E>(v));
    v = f(v, dpp<0x141>(v));
    v = f(v, dpp<0x140>(v));
    return f(f(lane_of(v, 0), lane_of(v, 16)), f(lane_of(v, 32), lane_of(v, 48)));
}

// V values of a row from element e on
template <int V> struct Vals {
    float v[V];
};
template <int V> __device__ __forceinline__ Vals<V> load_f32(const float *p) {
    Vals<V> r;
#pragma unroll
    for (int q = 0; q < V / 4; q++) {
        const float4 f = ((const float4 *)p)[q];
        r.v[4 * q] = f.x, r.v[4 * q + 1] = f.y, r.v[4 * q + 2] = f.z, r.v[4 * q + 3] = f.w;
    }
    return r;
}
template <int V> __device__ __forceinline__ Vals<V> load_bf16(const uint16_t *p) {
    uint32_t b[V / 2];
    if constexpr (V == 8) {
        const uint4 u = *(const uint4 *)p;
        b[0] = u.x, b[1] = u.y, b[2] = u.z, b[3] = u.w;
    } else {
        const uint2 u = *(const uint2 *)p;
        b[0] = u.x, b[1] = u.y;
    }
    Vals<V> r;
#pragma unroll
    for (int q = 0; q < V / 2; q++) {
        r.v[2 * q] = bf16_to_f32(b[q] & 0xFFFF);
        r.v[2 * q + 1] = bf16_to_f32(b[q] >> 16);
    }
    return r;
}

// WPR waves of a workgroup of 4 take a row of n <= 64 V WPR NJ values, V values of
// a lane at a time (n a multiple of V).
template <int KIND, int WPR, int NJ, int V>
__global__ __launch_bounds__(256) void rows_i8_kernel(RowsArgs a) {
    constexpr bool NORM = KIND >= kNorm, ADD = KIND >= kNormAddBf16;
    using A = std::conditional_t<NORM, double, float>;  // exact products x w; exact values
    const int tid = threadIdx.x, wave = tid >> 6;
    const int row = blockIdx.x * (4 / WPR) + (WPR == 1 ? wave : 0);
    const int i0 = WPR == 1 ? (tid & 63) : tid, nv = a.n / V;
    const bool live = row < a.m;
    const size_t base = (size_t)(live ? row : a.m - 1) * a.n;
    Vals<V> v[NJ], g[NJ], d[NJ];
#pragma unroll
    for (int j = 0; j < NJ; j++) {
        const int i = V * min(i0 + 64 * WPR * j, nv - 1);
        if constexpr (KIND == kBf16) v[j] = load_bf16<V>((const uint16_t *)a.x + base + i);
        else v[j] = load_f32<V>((const float *)a.x + base + i);
        if constexpr (KIND == kNormAddBf16) d[j] = load_bf16<V>((const uint16_t *)a.add + base + i);
        if constexpr (KIND == kNormAddF32) d[j] = load_f32<V>((const float *)a.add + base + i);
        if constexpr (NORM) g[j] = load_f32<V>(a.w + i);
    }
    A top = 0;
    double ss = 0.0;
    float nan = 0.f;  // stays 0 while every value (norm: weight) is finite
#pragma unroll
    for (int j = 0; j < NJ; j++) {
        const bool in = i0 + 64 * WPR * j < nv;
#pragma unroll
        for (int e = 0; e < V; e++) {
            // past the row's end: zeros, whatever was loaded there (the row's
            // last values, which another wave may already have written with
            // the addition)
            float x = v[j].v[e];
            if constexpr (ADD) x += d[j].v[e];
            x = in ? x : 0.f;
            v[j].v[e] = x;
            if constexpr (NORM) {
                const double xd = x;
                top = fmax(top, fabs(xd * (double)g[j].v[e]));
                ss = fma(xd, xd, ss);
                nan = fmaf(g[j].v[e], 0.f, nan);
            } else {
                top = fmaxf(top, fabsf(x));
                nan = fmaf(x, 0.f, nan);
            }
        }
        if constexpr (ADD)
            if (live && in)
#pragma unroll
                for (int q = 0; q < V / 4; q++)
                    *(float4 *)((float *)a.x + base + V * (i0 + 64 * WPR * j) + 4 * q) =
                        make_float4(v[j].v[4 * q], v[j].v[4 * q + 1], v[j].v[4 * q + 2], v[j].v[4 * q + 3]);
    }
    if (!(nan == 0.f)) top = __builtin_inf();
    auto larger = [](A p, A q) { return p > q ? p : q; };
    auto plus = [](double p, double q) { return p + q; };
    top = wave_reduce(top, larger);
    if constexpr (NORM) ss = wave_reduce(ss, plus);
    if constexpr (WPR > 1) {
        __shared__ double red[2][4];
        if ((tid & 63) == 0) {
            red[0][wave] = top;
            red[1][wave] = ss;
        }
        __syncthreads();
        top = larger(larger((A)red[0][0], (A)red[0][1]), larger((A)red[0][2], (A)red[0][3]));
        ss = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
    }
    if (!live) return;
    // a value that is not finite: the norm's sum of squares shows those of x
    const bool bad = !(top < (A)__builtin_inf()) || !(ss < __builtin_inf());
    const bool none = bad || !(top > 0);
    const bool mid = top >= (A)0x1p-90 && top <= (A)0x1p100;
    const float r = 127.f / (float)top;
    // The codes of four values from their fp64 quotients.
    auto exact = [&](int j, int e0, uint32_t(&k)[4]) __attribute__((always_inline)) {
        double hi[4], q[4], near = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            hi[e] = (double)v[j].v[e0 + e] * (NORM ? (double)g[j].v[e0 + e] : 1.0) * 127.0;
            const double f = hi[e] / (double)top;
            q[e] = rint(f);
            near = fmax(near, fabs(f - q[e]));
        }
        // 127 x w = hi + lo; q is the code or, beside a border, its neighbour.  r = hi - q
        // top is hi, for q = 0, or of at most top's power of two and a whole number of
        // 2^-52 of that, so the fma has it exactly; so is |r| - top / 2 where lo matters.
        if (NORM && near > 0.5 - 0x1p-40)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const double t = (double)v[j].v[e0 + e] * (double)g[j].v[e0 + e];
                const double lo = fma(t, 127.0, -hi[e]), r = fma(-q[e], (double)top, hi[e]), to = r < 0 ? -1.0 : 1.0;
                const double past = (fabs(r) - 0.5 * (double)top) + to * lo;
                if (past > 0 || (past == 0 && ((int)q[e] & 1))) q[e] += to;
            }
#pragma unroll
        for (int e = 0; e < 4; e++) k[e] = (uint32_t)(uint8_t)(int)q[e];
    };
#pragma unroll
    for (int j = 0; j < NJ; j++) {
        const int i = i0 + 64 * WPR * j;
        uint32_t c[V / 4];
#pragma unroll
        for (int q = 0; q < V / 4; q++) {
            uint32_t k[4];
            float off = 0.f;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float t = NORM ? v[j].v[4 * q + e] * g[j].v[4 * q + e] : v[j].v[4 * q + e];
                const float s = fmaf(t, r, kMagic);
                k[e] = __float_as_uint(s);
                off = fmaxf(off, fabsf(fmaf(t, r, -(s - kMagic))));
            }
            if (!none && (!mid || off > kNear)) exact(j, 4 * q, k);
            c[q] = none ? 0 : (k[0] & 0xFF) | (k[1] & 0xFF) << 8 | (k[2] & 0xFF) << 16 | k[3] << 24;
        }
        if (i < nv) {
            if constexpr (V == 8) *(uint2 *)(a.out + base + 8 * i) = make_uint2(c[0], c[1]);
            else *(uint32_t *)(a.out + base + 4 * i) = c[0];
        }
    }
    if (i0 == 0) {
        double sc = (double)top / 127.0;
        if constexpr (NORM) sc = sc / sqrt(ss / (double)a.n + (double)a.eps);
        a.scale[row] = bad ? __builtin_nanf("") : none ? 0.f : (float)sc;
    }
}

// A wave a row up to 1024 values, a workgroup a row beyond: us a wave / a workgroup,
// rows after an addition in bf16: 2048 x 1024 6.7 / 7.2, 2048 x 512 4.1 / 5.3, 2048 x
// 2048 10.2 / 9.6, 256 x 2048 4.8 / 3.4.
template <int KIND, int V>
void launch_kind(const RowsArgs &a, const char *name, hipStream_t s) {
    KernelSpan span(name, s, true);
    const int nv = a.n / V;
    if (a.n <= 1024) {
        const dim3 grid((unsigned)(((size_t)a.m + 3) / 4));
        if (nv <= 64) launch(span, rows_i8_kernel<KIND, 1, 1, V>, grid, dim3(256), 0, s, a);
        else if (nv <= 128) launch(span, rows_i8_kernel<KIND, 1, 2, V>, grid, dim3(256), 0, s, a);
        else if constexpr (V == 4) launch(span, rows_i8_kernel<KIND, 1, 4, V>, grid, dim3(256), 0, s, a);
        return;
    }
    const dim3 grid((unsigned)a.m);
    const int nj = (nv + 255) / 256;  // a lane's loads: at most 4 of 8 values, 8 of 4
    if (nj <= 1) launch(span, rows_i8_kernel<KIND, 4, 1, V>, grid, dim3(256), 0, s, a);
    else if (nj <= 2) launch(span, rows_i8_kernel<KIND, 4, 2, V>, grid, dim3(256), 0, s, a);
    else if (nj <= 3) launch(span, rows_i8_kernel<KIND, 4, 3, V>, grid, dim3(256), 0, s, a);
    else if (nj <= 4) launch(span, rows_i8_kernel<KIND, 4, 4, V>, grid, dim3(256), 0, s, a);
    else if constexpr (V == 4) {
        if (nj <= 6) launch(span, rows_i8_kernel<KIND, 4, 6, V>, grid, dim3(256), 0, s, a);
        else launch(span, rows_i8_kernel<KIND, 4, 8, V>, grid, dim3(256), 0, s, a);
    }
}

// rows of one launch: a grid holds less than 2^32 threads (kMaxRows is a
// multiple of 4, so later parts are aligned as the first)
constexpr int kMaxRows = 1 << 23;

bool aligned(const void *p, size_t to) { return ((uintptr_t)p & (to - 1)) == 0; }

}  // namespace

hipError_t launch_to_i8(const void *x, bool x_bf16, int m, int n, int8_t *out, float *scale, hipStream_t s) {
    if (n % 4 != 0 || n < 4 || n > 8192 || m < 0) return hipErrorInvalidValue;
    hipError_t e = hipSuccess;
    for (int r = 0; m - r > 0 && e == hipSuccess; r += std::min(m - r, kMaxRows)) {
        const char *xr = (const char *)x + (size_t)r * n * (x_bf16 ? 2 : 4);
        const RowsArgs a{(void *)xr, nullptr, nullptr, 0.f, std::min(m - r, kMaxRows), n, out + (size_t)r * n, scale + r};
        if (!x_bf16) launch_kind<kF32, 4>(a, "to_i8", s);
        else if (n % 8 == 0 && aligned(x, 16) && aligned(out, 8)) launch_kind<kBf16, 8>(a, "to_i8", s);
        else launch_kind<kBf16, 4>(a, "to_i8", s);
        e = hipGetLastError();
    }
    return e;
}

hipError_t launch_rows_rmsnorm_i8(float *x, const void *add, bool add_bf16, int m, int n, const float *w, float eps,
                                  int8_t *out, float *scale, hipStream_t s) {
    if (n % 4 != 0 || n < 4 || n > 8192 || m < 0) return hipErrorInvalidValue;
    hipError_t e = hipSuccess;
    for (int r = 0; m - r > 0 && e == hipSuccess; r += std::min(m - r, kMaxRows)) {
        const size_t at = (size_t)r * n;
        const RowsArgs a{x + at, add ? (const char *)add + at * (add_bf16 ? 2 : 4) : nullptr, w, eps,
                         std::min(m - r, kMaxRows), n, out + at, scale + r};
        if (!add) launch_kind<kNorm, 4>(a, "rows_rmsnorm_i8", s);
        else if (add_bf16) launch_kind<kNormAddBf16, 4>(a, "rows_rmsnorm_i8", s);
        else launch_kind<kNormAddF32, 4>(a, "rows_rmsnorm_i8", s);
        e = hipGetLastError();
    }
    return e;
}

}  // namespace hymt
