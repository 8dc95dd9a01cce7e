// What the three generation operators share on the host side and in their kernels.
#pragma once
#include "common.cuh"
#include "paged.cuh"

namespace sb200 {

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void from_f32(float *p, float x) { *p = x; }
__device__ __forceinline__ void from_f32(__nv_bfloat16 *p, float x) { *p = __float2bfloat16_rn(x); }

// 2^x by the special-function unit: relative error 2^-22, results below 2^-126 flushed to 0
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void cp_async_16(uint32_t dst, const void *src, bool there) {   // zeros where there is nothing
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Checks a caller's paged cache and fills in its defaults.
int make_paged_view(const char *who, const sofie_b200_paged_kv *kv, int32_t kv_heads, int32_t head_dim, PagedView *out);
// Head counts, head size, type and scale of an attention plan.
int check_attention(const char *who, int32_t heads, int32_t kv_heads, int32_t head_dim, int32_t dtype, float scale);

}  // namespace sb200
