// gemm_i8.hip -- products of int8 codes (gfx950): y[t][f] = ws[f] xs[t] sum_k
// x[t][k] w[f][k] on v_mfma_i32_16x16x64_i8, the sum exact in int32.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "device_common.hpp"
#include "int8.hpp"
#include "ktimer.hpp"

namespace hymt {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));

enum Out { kF32, kAcc, kBf16, kGlu };

// 4 features f .. f + 3 of token t
template <int OUT>
__device__ __forceinline__ void store4(const I8Gemm &g, int t, int f, i32x4 acc, i32x4 up) {
    const float xs = g.xs[t];
#pragma unroll
    for (int e = 0; e < 4; e++) {
        if (f + e >= g.n) break;
        const size_t at = (size_t)t * g.ldy + f + e;
        const float a = (float)acc[e] * g.ws[f + e], v = a * xs;
        if constexpr (OUT == kGlu)
            ((uint16_t *)g.y)[at] = f32_to_bf16(silu_fast(v) * ((float)up[e] * g.us[f + e] * xs));
        else if constexpr (OUT == kBf16)
            ((uint16_t *)g.y)[at] = f32_to_bf16(v);
        else if constexpr (OUT == kAcc)
            ((float *)g.y)[at] = fmaf(a, xs, ((float *)g.y)[at]);
        else
            ((float *)g.y)[at] = v;
    }
}

// 64 features x 64 tokens by 4 waves of 32 x 32, operands straight from memory
template <int OUT>
__global__ __launch_bounds__(256) void simple_kernel(I8Gemm g) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, grp = lane >> 4, c = lane & 15;
    const int tiles_f = (g.n + 63) / 64;
    const int f0 = (blockIdx.x % tiles_f) * 64 + 32 * (wave & 1), t0 = (blockIdx.x / tiles_f) * 64 + 32 * (wave >> 1);
    i32x4 acc[2][2] = {}, up[2][2] = {};
    size_t wo[2], xo[2];
    for (int i = 0; i < 2; i++) {
        wo[i] = (size_t)min(f0 + 16 * i + c, g.n - 1) * g.k + 16 * grp;
        xo[i] = (size_t)min(t0 + 16 * i + c, g.m - 1) * g.k + 16 * grp;
    }
    for (int k0 = 0; k0 < g.k; k0 += 64)
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const i32x4 x = *(const i32x4 *)(g.x + xo[j] + k0);
                acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(*(const i32x4 *)(g.w + wo[i] + k0), x, acc[i][j], 0, 0, 0);
                if constexpr (OUT == kGlu)
                    up[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(*(const i32x4 *)(g.up + wo[i] + k0), x, up[i][j], 0, 0, 0);
            }
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const int t = t0 + 16 * j + c;
            if (t < g.m) store4<OUT>(g, t, f0 + 16 * i + 4 * grp, acc[i][j], up[i][j]);
        }
}

bool fits(const I8Gemm &g) {
    auto a16 = [](const void *p) { return ((uintptr_t)p & 15u) == 0; };
    return g.n > 0 && g.m >= 0 && g.k >= 2 * kI8StepK && g.k <= kI8MaxK && g.k % kI8StepK == 0 && g.ldy >= g.n &&
           a16(g.w) && a16(g.x) && a16(g.up);
}

template <int OUT>
hipError_t run(const I8Gemm &g, const char *name, hipStream_t s) {
    if (!fits(g)) return hipErrorInvalidValue;
    if (g.m == 0) return hipSuccess;
    const size_t grid = (size_t)((g.n + 63) / 64) * ((g.m + 63) / 64);
    if (grid > 0x7fffffffu) return hipErrorInvalidValue;
    KernelSpan span(name, s, true);
    launch(span, simple_kernel<OUT>, dim3((unsigned)grid), dim3(256), 0, s, g);
    return hipGetLastError();
}

}  // namespace

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
