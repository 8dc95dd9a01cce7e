// Attention of one new token per sequence over a paged key-value cache.
#include <math.h>
#include <new>

#include "generate.cuh"

namespace sb200 {

struct PagedAttnParams {
  PagedView kv;
  const void *q, *cache_k, *cache_v;
  void *y;
  long long ldq, ldy;
  int heads, kv_heads, dim;
  float scale_log2e;
  int *status;
};

// One warp per (sequence, head); lane l holds dimensions l, l + 32, ...
template <class T>
__global__ void __launch_bounds__(128) paged_rows_kernel(const PagedAttnParams p) {
  const long long w = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (w >= (long long)p.kv.batch * p.heads) return;
  const int b = (int)(w / p.heads), h = (int)(w % p.heads);
  bool bad = false;
  const int n = paged_len(p.kv, b, &bad);
  const int kh = h / (p.heads / p.kv_heads);
  const T *q = static_cast<const T *>(p.q) + b * p.ldq + h * p.dim;
  float qr[8], acc[8];
  for (int i = 0; i < 8; ++i) {
    const int d = lane + 32 * i;
    qr[i] = d < p.dim ? to_f32(q[d]) * p.scale_log2e : 0.f;
    acc[i] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  bool any = false;
  for (int j = 0; j < n; ++j) {
    const long long row = paged_row(p.kv, b, j);
    if (row < 0) {
      bad = true;
      continue;
    }
    any = true;
    const T *k = static_cast<const T *>(p.cache_k) + row + kh * p.kv.head_stride;
    const T *v = static_cast<const T *>(p.cache_v) + row + kh * p.kv.head_stride;
    float s = 0.f;
    for (int i = 0; i < 8; ++i) {
      const int d = lane + 32 * i;
      if (d < p.dim) s = fmaf(qr[i], to_f32(k[d]), s);
    }
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    const float m1 = fmaxf(m, s), base = m1 == -INFINITY ? 0.f : m1;
    const float f = exp2f(m - base), e = exp2f(s - base);
    m = m1;
    l = l * f + e;
    for (int i = 0; i < 8; ++i) {
      const int d = lane + 32 * i;
      if (d < p.dim) acc[i] = acc[i] * f + e * to_f32(v[d]);
    }
  }
  if (bad && lane == 0) report(p.status, DEV_BAD_INDEX);
  T *y = static_cast<T *>(p.y) + b * p.ldy + h * p.dim;
  const float inv = any ? 1.f / l : 0.f;
  for (int i = 0; i < 8; ++i) {
    const int d = lane + 32 * i;
    if (d < p.dim) from_f32(y + d, acc[i] * inv);
  }
}

}  // namespace sb200

using namespace sb200;

struct sofie_b200_paged_attention_plan {
  sofie_b200_ctx *ctx = nullptr;
  sofie_b200_paged_attention_desc d{};
  int64_t bytes = 0;
};

extern "C" {

int sofie_b200_paged_attention_plan_create(sofie_b200_ctx *ctx, const sofie_b200_paged_attention_desc *desc,
                                           sofie_b200_paged_attention_plan **out) {
  if (!desc || !out) return fail(SOFIE_B200_ERR_INVALID, "paged_attention_plan_create: NULL argument");
  *out = nullptr;
  sofie_b200_paged_attention_desc d = *desc;
  int rc = check_attention("paged_attention_plan_create", d.heads, d.kv_heads, d.head_dim, d.dtype, d.scale);
  if (rc) return rc;
  const int64_t qw = (int64_t)d.heads * d.head_dim;
  if (!d.ldq) d.ldq = qw;
  if (!d.ldy) d.ldy = qw;
  if (d.ldq < qw || d.ldy < qw) return fail(SOFIE_B200_ERR_INVALID, "paged_attention_plan_create: a row pitch is smaller than heads * head size");
  if (d.ldq % 8 || d.ldy % 8) return fail(SOFIE_B200_ERR_INVALID, "paged_attention_plan_create: row pitches must be multiples of 8 elements");
  if (d.scale == 0.f) d.scale = 1.f / sqrtf((float)d.head_dim);
  if (!ctx) return fail(SOFIE_B200_ERR_INVALID, "paged_attention_plan_create: ctx is NULL");
  auto *p = new (std::nothrow) sofie_b200_paged_attention_plan();
  if (!p) return fail(SOFIE_B200_ERR_INVALID, "paged_attention_plan_create: out of host memory");
  p->ctx = ctx;
  p->d = d;
  *out = p;
  return 0;
}

int sofie_b200_paged_attention_plan_destroy(sofie_b200_paged_attention_plan *plan) {
  delete plan;
  return 0;
}

const char *sofie_b200_paged_attention_plan_kernel(const sofie_b200_paged_attention_plan *plan) { return plan ? "rows" : ""; }

int64_t sofie_b200_paged_attention_workspace_bytes(const sofie_b200_paged_attention_plan *plan) { return plan ? plan->bytes : 0; }

int sofie_b200_paged_attention_enqueue(sofie_b200_paged_attention_plan *plan, const void *q, const sofie_b200_paged_kv *kv, void *y,
                                       void *workspace) {
  if (!plan) return fail(SOFIE_B200_ERR_INVALID, "paged_attention_enqueue: plan is NULL");
  const sofie_b200_paged_attention_desc &d = plan->d;
  PagedAttnParams p{};
  int rc = make_paged_view("paged_attention_enqueue", kv, d.kv_heads, d.head_dim, &p.kv);
  if (rc) return rc;
  if (p.kv.batch == 0) return 0;
  if (!q || !y) return fail(SOFIE_B200_ERR_INVALID, "paged_attention_enqueue: NULL tensor pointer");
  if (((uintptr_t)q % 16) || ((uintptr_t)y % 16) || ((uintptr_t)kv->k % 16) || ((uintptr_t)kv->v % 16))
    return fail(SOFIE_B200_ERR_INVALID, "paged_attention_enqueue: tensors must be 16-byte aligned");
  if (p.kv.page_stride % 8 || p.kv.token_stride % 8 || p.kv.head_stride % 8)
    return fail(SOFIE_B200_ERR_INVALID, "paged_attention_enqueue: the cache's strides must be multiples of 8 elements");
  if (plan->bytes && (!workspace || ((uintptr_t)workspace % 256)))
    return fail(SOFIE_B200_ERR_INVALID, "paged_attention_enqueue: this plan needs a 256-byte aligned workspace");
  sofie_b200_ctx *ctx = plan->ctx;
  SB_CUDA(cudaSetDevice(ctx->device));
  p.q = q; p.cache_k = kv->k; p.cache_v = kv->v; p.y = y;
  p.ldq = d.ldq; p.ldy = d.ldy;
  p.heads = d.heads; p.kv_heads = d.kv_heads; p.dim = d.head_dim;
  p.scale_log2e = d.scale * 1.4426950408889634f;
  p.status = ctx->d_status;
  const int64_t blocks = ((int64_t)p.kv.batch * d.heads + 3) / 4;
  if (blocks > 0x7fffffffLL) return fail(SOFIE_B200_ERR_TOO_LARGE, "paged_attention_enqueue: batch %d of %d heads", p.kv.batch, d.heads);
  if (d.dtype == SOFIE_B200_F32) paged_rows_kernel<float><<<(unsigned)blocks, 128, 0, ctx->stream>>>(p);
  else paged_rows_kernel<__nv_bfloat16><<<(unsigned)blocks, 128, 0, ctx->stream>>>(p);
  SB_CUDA(cudaGetLastError());
  ctx->launches++;
  return 0;
}

}  // extern "C"
