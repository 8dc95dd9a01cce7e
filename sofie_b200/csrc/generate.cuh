// What the three generation operators share on the host side and in their kernels.
#pragma once
#include "common.cuh"
#include "paged.cuh"

namespace sb200 {

// Writes a code to the context's status word unless one is there already.
__device__ __forceinline__ void report(int *status, int code) { atomicCAS(status, 0, code); }

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void from_f32(float *p, float x) { *p = x; }
__device__ __forceinline__ void from_f32(__nv_bfloat16 *p, float x) { *p = __float2bfloat16_rn(x); }

// Checks a caller's paged cache and fills in its defaults.
int make_paged_view(const char *who, const sofie_b200_paged_kv *kv, int32_t kv_heads, int32_t head_dim, PagedView *out);
// Head counts, head size, type and scale of an attention plan.
int check_attention(const char *who, int32_t heads, int32_t kv_heads, int32_t head_dim, int32_t dtype, float scale);

}  // namespace sb200
