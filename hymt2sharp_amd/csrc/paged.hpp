// paged.hpp -- the multi-sequence cache's operators: upkeep of its pages and
// the rotary append (paged_ops.hip), attention over it (paged_attn.hip).  The
// structs are the C ABI's own (include/hymt_hip.h); what stands in device memory
// is checked by the kernels, everything else by the callers of these launchers.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/hymt_hip.h"
#include "device_common.hpp"

namespace hymt {

constexpr int kPagedMaxGroup = 64;      // q heads per kv head
constexpr int kPagedMaxSeqs = 65536;    // slots (one bit each in the plan kernels' LDS)
constexpr int kPagedMaxBlocks = 1 << 24;  // positions stay below 2^30

// fp32 to an element of the cache, nearest even by the hardware's conversion (a
// NaN stays one)
template <typename T> __device__ __forceinline__ uint16_t bits_of(float x);
template <> __device__ __forceinline__ uint16_t bits_of<F16>(float x) { return f32_to_f16(x); }
template <> __device__ __forceinline__ uint16_t bits_of<BF16>(float x) {
    return __builtin_bit_cast(uint16_t, (__bf16)x);
}

// Wave-wide steps by DPP: within rows of 16 lanes, then row 15 -> the next row and lane
// 31 -> the upper half.  Lane 63 has seen all 64 lanes.
template <typename F> __device__ __forceinline__ int dpp_scan(int x, int none, F f) {
    x = f(x, __builtin_amdgcn_update_dpp(none, x, 0x111, 0xF, 0xF, false));  // row_shr:1, 2, 4, 8
    x = f(x, __builtin_amdgcn_update_dpp(none, x, 0x112, 0xF, 0xF, false));
    x = f(x, __builtin_amdgcn_update_dpp(none, x, 0x114, 0xF, 0xF, false));
    x = f(x, __builtin_amdgcn_update_dpp(none, x, 0x118, 0xF, 0xF, false));
    x = f(x, __builtin_amdgcn_update_dpp(none, x, 0x142, 0xA, 0xF, false));  // row_bcast:15 into rows 1 and 3
    x = f(x, __builtin_amdgcn_update_dpp(none, x, 0x143, 0xC, 0xF, false));  // row_bcast:31 into rows 2 and 3
    return x;
}
__device__ __forceinline__ int wave_sums(int x) {  // of the lanes up to each
    return dpp_scan(x, 0, [](int a, int b) { return a + b; });
}
__device__ __forceinline__ int wave_min(int x) {  // in a scalar register
    return __builtin_amdgcn_readlane(dpp_scan(x, 0x7FFFFFFF, [](int a, int b) { return min(a, b); }), 63);
}

// words of hymt_paged::work
enum { kWorkFirst = 0, kWorkCopies = 1, kWorkLive = 2, kWorkStatus = 3, kWorkLists = 4 };

struct RopeAppend {
    const void *q, *k, *v;
    int q_ld, kv_ld, io_dtype, heads, layer;
    const double *freq;
    int dim, interleaved;
    float scale;
    const float *qnw, *knw;
    float eps;
    void *q_out;
};

// Scores are multiplied by this before the powers of 2; the entry points see to it
// that it is finite (the product with a score of 0 would not be one otherwise).
inline float paged_log2_scale(float scale) { return scale * 1.4426950408889634f; }

struct PagedAttn {
    const void *q;
    int heads, layer, prefix;
    float scale;
    void *out;
    int out_dtype;
};

hipError_t launch_paged_extend(const hymt_paged &p, const int32_t *slots, const int32_t *cu, int n, hipStream_t s);
hipError_t launch_paged_fork(const hymt_paged &p, const int32_t *parent, const int32_t *child, int n, hipStream_t s);
hipError_t launch_paged_set_len(const hymt_paged &p, const int32_t *slots, const int32_t *lens, int n, hipStream_t s);
hipError_t launch_paged_compact(const hymt_paged &p, hipStream_t s);
hipError_t launch_rope_append(const hymt_paged &p, const hymt_batch &b, const RopeAppend &a, hipStream_t s);
// fp32 values of workspace that the two launches below need at most
size_t paged_attn_workspace(const hymt_paged &p, const hymt_batch &b, const PagedAttn &a, bool shared);
hipError_t launch_attn_packed(const hymt_paged &p, const hymt_batch &b, const PagedAttn &a, float *ws, hipStream_t s);
hipError_t launch_attn_shared(const hymt_paged &p, const hymt_batch &b, const PagedAttn &a, float *ws, hipStream_t s);

}  // namespace hymt
