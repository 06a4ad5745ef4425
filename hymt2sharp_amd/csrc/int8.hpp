// int8.hpp -- the 8-bit integer operators: rows as int8 codes with a scale
// each (rows_i8.hip), and products of such rows with int8 weights that have a
// scale per channel (gemm_i8.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

namespace hymt {

// The largest row of codes that a product sums: 128 * 128 * 65536 = 2^30 fits
// an int32 with room.
constexpr int kI8MaxK = 65536;
constexpr int kI8MaxRows = 1 << 30;  // of tokens and of channels: indexes a tile past the end fit an int
constexpr int kI8StepK = 128;  // k is a multiple of this, two of them at least

// out[r] = rint(127 v / max|v|) (ties to even) and scale[r] = max|v| / 127 of
// the rows v of x, fp32 or (x_bf16) bf16; a row of zeros: zeros and 0, a row with
// a NaN or an infinity: zeros and NaN.  n a multiple of 4 up to 8192; x
// 16-byte aligned (8 for bf16), out 4.
hipError_t launch_to_i8(const void *x, bool x_bf16, int m, int n, int8_t *out, float *scale, hipStream_t s);

// The same of v = x / sqrt(mean(x^2) + eps) * w, after x = fp32(x + add) where
// add (fp32, or bf16 with add_bf16) is given.
hipError_t launch_rows_rmsnorm_i8(float *x, const void *add, bool add_bf16, int m, int n, const float *w, float eps,
                                  int8_t *out, float *scale, hipStream_t s);

// y[m][n] (rows ldy apart) = ws[f] xs[t] sum_k x[t][k] w[f][k]: the sum exact in
// int32, then one fp32 product with each scale.
enum I8Out { kI8F32 = 0, kI8Acc = 1, kI8Bf16 = 2 };
struct I8Gemm {
    const int8_t *w;   // [n][k], 16-byte aligned
    const float *ws;   // [n]
    const int8_t *up;  // SwiGLU: the up rows [n][k] beside the gate rows w, else null
    const float *us;   // SwiGLU: [n]
    const int8_t *x;   // [m][k], 16-byte aligned
    const float *xs;   // [m]
    void *y;           // [m][ldy]: fp32, or bf16 (kI8Bf16, SwiGLU)
    int n, k, m, ldy;
};
hipError_t launch_gemm_i8(const I8Gemm &g, I8Out out, hipStream_t s);
// Whether some tile covers g (up: SwiGLU) in as many workgroups as a launch holds.
bool gemm_i8_launches(const I8Gemm &g);
// Whether HYMT_HIP_I8_TILE is unset or the name of a tile; the launches refuse
// another.
bool gemm_i8_tile_known();
// act[m][n] = bf16(silu(gate) up) of the two products in fp32
hipError_t launch_gemm_i8_swiglu(const I8Gemm &g, hipStream_t s);

}  // namespace hymt
