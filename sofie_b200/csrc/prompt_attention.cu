// Attention over packed prompts of different lengths: causal or full, grouped heads.
#include <math.h>
#include <new>

#include "generate.cuh"

namespace sb200 {

struct PromptParams {
  const void *q, *k, *v;
  void *y;
  const int32_t *cu_q, *cu_k;
  long long ldq, ldk, ldv, ldy;
  long long q_rows, k_rows;
  int batch, heads, kv_heads, dim, causal;
  float scale_log2e;
  int *status;
};

// One warp per (query, head); lane l holds dimensions l, l + 32, ... of q, of the running sum and of the current key and value.
// Softmax in one pass with a running maximum: a larger maximum scales the sum and the weighted values so far.
template <class T>
__global__ void __launch_bounds__(128) prompt_rows_kernel(const PromptParams p) {
  const long long w = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const long long t = w / p.heads;
  const int h = (int)(w % p.heads);
  if (t >= p.q_rows) return;
  const int b = packed_find(p.cu_q, p.batch, (int)t);
  if (b < 0) return;
  int q0, q1, k0, k1;
  bool bad = false;
  packed_range(p.cu_q, b, p.q_rows, &q0, &q1, &bad);
  packed_range(p.cu_k, b, p.k_rows, &k0, &k1, &bad);
  if (bad) {
    report(p.status, DEV_BAD_INDEX);
    return;
  }
  int n = k1 - k0;
  if (p.causal) n = min(n, max(0, (int)(t - q0) + 1 + n - (q1 - q0)));
  const int kh = h / (p.heads / p.kv_heads);
  const T *q = static_cast<const T *>(p.q) + t * p.ldq + h * p.dim;
  float qr[8], acc[8];
  for (int i = 0; i < 8; ++i) {
    const int d = lane + 32 * i;
    qr[i] = d < p.dim ? to_f32(q[d]) * p.scale_log2e : 0.f;
    acc[i] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (int j = 0; j < n; ++j) {
    const T *k = static_cast<const T *>(p.k) + (k0 + j) * p.ldk + kh * p.dim;
    const T *v = static_cast<const T *>(p.v) + (k0 + j) * p.ldv + kh * p.dim;
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
  T *y = static_cast<T *>(p.y) + t * p.ldy + h * p.dim;
  const float inv = n > 0 ? 1.f / l : 0.f;
  for (int i = 0; i < 8; ++i) {
    const int d = lane + 32 * i;
    if (d < p.dim) from_f32(y + d, acc[i] * inv);
  }
}

}  // namespace sb200

using namespace sb200;

struct sofie_b200_prompt_attention_plan {
  sofie_b200_ctx *ctx = nullptr;
  sofie_b200_prompt_attention_desc d{};
};

extern "C" {

int sofie_b200_prompt_attention_plan_create(sofie_b200_ctx *ctx, const sofie_b200_prompt_attention_desc *desc,
                                            sofie_b200_prompt_attention_plan **out) {
  if (!desc || !out) return fail(SOFIE_B200_ERR_INVALID, "prompt_attention_plan_create: NULL argument");
  *out = nullptr;
  sofie_b200_prompt_attention_desc d = *desc;
  int rc = check_attention("prompt_attention_plan_create", d.heads, d.kv_heads, d.head_dim, d.dtype, d.scale);
  if (rc) return rc;
  const int64_t qw = (int64_t)d.heads * d.head_dim, kw = (int64_t)d.kv_heads * d.head_dim;
  if (!d.ldq) d.ldq = qw;
  if (!d.ldk) d.ldk = kw;
  if (!d.ldv) d.ldv = kw;
  if (!d.ldy) d.ldy = qw;
  if (d.ldq < qw || d.ldk < kw || d.ldv < kw || d.ldy < qw)
    return fail(SOFIE_B200_ERR_INVALID, "prompt_attention_plan_create: a token pitch is smaller than heads * head size");
  if (d.ldq % 8 || d.ldk % 8 || d.ldv % 8 || d.ldy % 8)
    return fail(SOFIE_B200_ERR_INVALID, "prompt_attention_plan_create: token pitches must be multiples of 8 elements");
  if (d.ldq > (1LL << 32) || d.ldk > (1LL << 32) || d.ldv > (1LL << 32) || d.ldy > (1LL << 32))
    return fail(SOFIE_B200_ERR_INVALID, "prompt_attention_plan_create: a token pitch is too large");
  if (d.scale == 0.f) d.scale = 1.f / sqrtf((float)d.head_dim);
  if (!ctx) return fail(SOFIE_B200_ERR_INVALID, "prompt_attention_plan_create: ctx is NULL");
  auto *p = new (std::nothrow) sofie_b200_prompt_attention_plan();
  if (!p) return fail(SOFIE_B200_ERR_INVALID, "prompt_attention_plan_create: out of host memory");
  p->ctx = ctx;
  p->d = d;
  *out = p;
  return 0;
}

int sofie_b200_prompt_attention_plan_destroy(sofie_b200_prompt_attention_plan *plan) {
  delete plan;
  return 0;
}

const char *sofie_b200_prompt_attention_plan_kernel(const sofie_b200_prompt_attention_plan *plan) { return plan ? "rows" : ""; }

int sofie_b200_prompt_attention_enqueue(sofie_b200_prompt_attention_plan *plan, const void *q, const void *k, const void *v, void *y,
                                        const int32_t *cu_seqlens_q, const int32_t *cu_seqlens_k, int64_t batch, int64_t q_tokens,
                                        int64_t k_tokens) {
  if (!plan) return fail(SOFIE_B200_ERR_INVALID, "prompt_attention_enqueue: plan is NULL");
  const sofie_b200_prompt_attention_desc &d = plan->d;
  if (batch < 0 || batch > 0x3fffffff || q_tokens < 0 || q_tokens > 0x3fffffff || k_tokens < 0 || k_tokens > 0x3fffffff)
    return fail(SOFIE_B200_ERR_INVALID, "prompt_attention_enqueue: bad extent (batch %lld, %lld and %lld tokens)", (long long)batch,
                (long long)q_tokens, (long long)k_tokens);
  if (batch == 0 || q_tokens == 0) return 0;
  if (!q || !y || !cu_seqlens_q || (k_tokens > 0 && (!k || !v))) return fail(SOFIE_B200_ERR_INVALID, "prompt_attention_enqueue: NULL tensor pointer");
  if (((uintptr_t)q % 16) || ((uintptr_t)k % 16) || ((uintptr_t)v % 16) || ((uintptr_t)y % 16))
    return fail(SOFIE_B200_ERR_INVALID, "prompt_attention_enqueue: tensors must be 16-byte aligned");
  sofie_b200_ctx *ctx = plan->ctx;
  SB_CUDA(cudaSetDevice(ctx->device));
  PromptParams p{};
  p.q = q; p.k = k; p.v = v; p.y = y;
  p.cu_q = cu_seqlens_q; p.cu_k = cu_seqlens_k ? cu_seqlens_k : cu_seqlens_q;
  p.ldq = d.ldq; p.ldk = d.ldk; p.ldv = d.ldv; p.ldy = d.ldy;
  p.q_rows = q_tokens; p.k_rows = k_tokens;
  p.batch = (int)batch; p.heads = d.heads; p.kv_heads = d.kv_heads; p.dim = d.head_dim; p.causal = d.causal != 0;
  p.scale_log2e = d.scale * 1.4426950408889634f;
  p.status = ctx->d_status;
  const int64_t blocks = (q_tokens * d.heads + 3) / 4;
  if (blocks > 0x7fffffffLL) return fail(SOFIE_B200_ERR_TOO_LARGE, "prompt_attention_enqueue: %lld queries of %d heads", (long long)q_tokens, d.heads);
  if (d.dtype == SOFIE_B200_F32) prompt_rows_kernel<float><<<(unsigned)blocks, 128, 0, ctx->stream>>>(p);
  else prompt_rows_kernel<__nv_bfloat16><<<(unsigned)blocks, 128, 0, ctx->stream>>>(p);
  SB_CUDA(cudaGetLastError());
  ctx->launches++;
  return 0;
}

}  // extern "C"
