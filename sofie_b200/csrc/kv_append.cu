// Appends the keys and values of new tokens to a paged cache, rotating keys (and queries) by their positions on the way.
#include <math.h>

#include "generate.cuh"

namespace sb200 {

int make_paged_view(const char *who, const sofie_b200_paged_kv *kv, int32_t kv_heads, int32_t head_dim, PagedView *out) {
  if (!kv) return fail(SOFIE_B200_ERR_INVALID, "%s: the cache is NULL", who);
  if (kv->batch < 0 || kv->batch > 0x3fffffff) return fail(SOFIE_B200_ERR_INVALID, "%s: batch %lld out of range", who, (long long)kv->batch);
  if (kv->page_size < 1) return fail(SOFIE_B200_ERR_INVALID, "%s: page size %d (at least 1)", who, kv->page_size);
  if (kv->num_pages < 0 || kv->num_pages > 0x7fffffffLL) return fail(SOFIE_B200_ERR_INVALID, "%s: %lld pages", who, (long long)kv->num_pages);
  if (kv->table_width < 0 || kv->table_width > 0x7fffffffLL / kv->page_size)
    return fail(SOFIE_B200_ERR_INVALID, "%s: a table of %lld pages of %d tokens (at most 2^31 - 1 tokens)", who, (long long)kv->table_width, kv->page_size);
  const int64_t pitch = kv->table_pitch ? kv->table_pitch : kv->table_width;
  if (pitch < kv->table_width) return fail(SOFIE_B200_ERR_INVALID, "%s: the table's pitch is smaller than its width", who);
  int64_t ps = kv->page_stride, ts = kv->token_stride, hs = kv->head_stride;
  if (!ps && !ts && !hs) {
    hs = head_dim;
    ts = (int64_t)kv_heads * head_dim;
    ps = ts * kv->page_size;
  }
  if (ps < 0 || ts < 0 || hs < 0) return fail(SOFIE_B200_ERR_INVALID, "%s: negative strides of the cache", who);
  // no two elements share a place: the innermost extent and every stride's own step fit into the next larger stride
  struct { int64_t n, s; } ax[3] = {{kv_heads, hs}, {kv->page_size, ts}, {kv->num_pages, ps}};
  for (int i = 0; i < 3; ++i)
    for (int j = i + 1; j < 3; ++j)
      if (ax[j].s < ax[i].s) { const auto t = ax[i]; ax[i] = ax[j]; ax[j] = t; }
  int64_t room = head_dim;
  for (int i = 0; i < 3; ++i) {
    if (ax[i].n <= 1) continue;
    if (ax[i].s < room) return fail(SOFIE_B200_ERR_INVALID, "%s: the cache's strides let elements overlap", who);
    if (ax[i].s > (INT64_MAX - room) / ax[i].n) return fail(SOFIE_B200_ERR_INVALID, "%s: the cache's strides are too large", who);
    room += ax[i].s * (ax[i].n - 1);
  }
  if (kv->batch > 0) {
    if (!kv->seq_lens || (!kv->block_table && kv->table_width > 0)) return fail(SOFIE_B200_ERR_INVALID, "%s: NULL block table or lengths", who);
    if (kv->num_pages > 0 && (!kv->k || !kv->v)) return fail(SOFIE_B200_ERR_INVALID, "%s: NULL cache", who);
  }
  out->table = kv->block_table;
  out->lens = kv->seq_lens;
  out->table_pitch = pitch;
  out->page_stride = ps;
  out->token_stride = ts;
  out->head_stride = hs;
  out->batch = (int)kv->batch;
  out->num_pages = (int)kv->num_pages;
  out->table_width = (int)kv->table_width;
  out->page_size = kv->page_size;
  return 0;
}

int check_attention(const char *who, int32_t heads, int32_t kv_heads, int32_t head_dim, int32_t dtype, float scale) {
  if (dtype != SOFIE_B200_F32 && dtype != SOFIE_B200_BF16) return fail(SOFIE_B200_ERR_INVALID, "%s: type %d not supported (F32, BF16)", who, dtype);
  if (kv_heads < 1 || heads < 1 || heads % kv_heads != 0 || heads / kv_heads > 64)
    return fail(SOFIE_B200_ERR_INVALID, "%s: %d query heads over %d key heads (a multiple, up to 64 each)", who, heads, kv_heads);
  if (head_dim < 8 || head_dim > 256 || head_dim % 8 != 0)
    return fail(SOFIE_B200_ERR_INVALID, "%s: head size %d not supported (a multiple of 8 up to 256)", who, head_dim);
  if ((int64_t)heads * head_dim > (1 << 24)) return fail(SOFIE_B200_ERR_INVALID, "%s: rows of %lld elements", who, (long long)heads * head_dim);
  if (!(scale >= 0.f) || isinf(scale)) return fail(SOFIE_B200_ERR_INVALID, "%s: scale %g (positive, or 0 for 1 / sqrt(head_dim))", who, scale);
  return 0;
}

struct AppendParams {
  PagedView kv;
  const int32_t *cu;       // NULL: token t is the only new one of sequence t
  const void *q, *k, *v;
  void *q_out, *k_out, *cache_k, *cache_v;
  const float *cos, *sin;
  long long ldq, ldk, ldv, ldqo, ldko;
  int tokens, heads, kv_heads, dim, half, interleaved;   // half = rotary_dim / 2
  long long max_position;
  int *status;
};

// One block per token.  An element pair (first, second) that turns together is one thread's work, so q_out may be q.
template <class T>
__global__ void __launch_bounds__(256) kv_append_kernel(const AppendParams p) {
  const int t = blockIdx.x;
  __shared__ int s_pos;
  __shared__ long long s_row;
  if (threadIdx.x == 0) {
    int pos = -1;
    long long row = -1;
    const int b = p.cu ? packed_find(p.cu, p.kv.batch, t) : t;
    if (b >= 0) {
      const int len = p.kv.lens[b];
      if (p.cu) {
        int begin, end;
        bool bad = false;
        packed_range(p.cu, b, p.tokens, &begin, &end, &bad);
        pos = bad ? -1 : len - (end - t);
      } else {
        pos = len - 1;
      }
      if (pos >= 0 && (p.half == 0 || pos < p.max_position)) row = paged_row(p.kv, b, pos);
      if (row < 0 && !(p.cu == nullptr && len == 0)) report(p.status, DEV_BAD_INDEX);
    }
    s_pos = pos;
    s_row = row;
  }
  __syncthreads();
  const int pos = s_pos;
  const long long row = s_row;
  if (row < 0) return;
  const T *q = static_cast<const T *>(p.q) + t * p.ldq;
  const T *k = static_cast<const T *>(p.k) + t * p.ldk;
  const T *v = static_cast<const T *>(p.v) + t * p.ldv;
  T *qo = static_cast<T *>(p.q_out) + t * p.ldqo;
  T *ko = p.k_out ? static_cast<T *>(p.k_out) + t * p.ldko : nullptr;
  T *ck = static_cast<T *>(p.cache_k) + row, *cv = static_cast<T *>(p.cache_v) + row;
  const float *cs = p.cos + (long long)pos * p.half, *sn = p.sin + (long long)pos * p.half;
  const int units = p.dim - p.half;   // per head: the pairs, then the dimensions that stay
  const int turned = (p.heads + p.kv_heads) * units;
  for (int i = threadIdx.x; i < turned; i += blockDim.x) {
    const int h = i / units, u = i % units;
    const bool key = h >= p.heads;
    const int kh = h - p.heads;
    const T *src = key ? k + kh * p.dim : q + h * p.dim;
    T *dst = key ? ck + kh * p.kv.head_stride : qo + h * p.dim;
    T *dst2 = key && ko ? ko + kh * p.dim : nullptr;
    if (u < p.half) {
      const int a = p.interleaved ? 2 * u : u, b = p.interleaved ? 2 * u + 1 : u + p.half;
      const float x = to_f32(src[a]), y = to_f32(src[b]);
      const float c = cs[u], s = sn[u];
      const float x1 = x * c - y * s, y1 = y * c + x * s;
      from_f32(dst + a, x1);
      from_f32(dst + b, y1);
      if (dst2) { from_f32(dst2 + a, x1); from_f32(dst2 + b, y1); }
    } else {
      const int a = u + p.half;
      const T x = src[a];
      dst[a] = x;
      if (dst2) dst2[a] = x;
    }
  }
  for (int i = threadIdx.x; i < p.kv_heads * p.dim; i += blockDim.x) {
    const int h = i / p.dim, d = i % p.dim;
    cv[h * p.kv.head_stride + d] = v[i];
  }
}

}  // namespace sb200

using namespace sb200;

extern "C" int sofie_b200_kv_append_enqueue(sofie_b200_ctx *ctx, const sofie_b200_kv_append_desc *desc, const sofie_b200_paged_kv *kv,
                                            const int32_t *cu_seqlens, const void *q, const void *k, const void *v, const float *cos,
                                            const float *sin, void *q_out, void *k_out) {
  if (!desc) return fail(SOFIE_B200_ERR_INVALID, "kv_append_enqueue: desc is NULL");
  const sofie_b200_kv_append_desc &d = *desc;
  if (d.dtype != SOFIE_B200_F32 && d.dtype != SOFIE_B200_BF16)
    return fail(SOFIE_B200_ERR_INVALID, "kv_append_enqueue: type %d not supported (F32, BF16)", d.dtype);
  if (d.tokens < 0 || d.tokens > 0x7fffffffLL || d.heads < 0 || d.kv_heads < 1 || d.head_dim < 1 ||
      ((int64_t)d.heads + d.kv_heads) * d.head_dim > (1 << 24))
    return fail(SOFIE_B200_ERR_INVALID, "kv_append_enqueue: bad extent");
  if (d.rotary_dim < 0 || d.rotary_dim > d.head_dim || d.rotary_dim % 2 != 0)
    return fail(SOFIE_B200_ERR_INVALID, "kv_append_enqueue: %d rotated dimensions of %d (an even number)", d.rotary_dim, d.head_dim);
  AppendParams p{};
  int rc = make_paged_view("kv_append_enqueue", kv, d.kv_heads, d.head_dim, &p.kv);
  if (rc) return rc;
  const int64_t qw = (int64_t)d.heads * d.head_dim, kw = (int64_t)d.kv_heads * d.head_dim;
  p.ldq = d.ldq ? d.ldq : qw;
  p.ldqo = d.ldqo ? d.ldqo : qw;
  p.ldk = d.ldk ? d.ldk : kw;
  p.ldv = d.ldv ? d.ldv : kw;
  p.ldko = d.ldko ? d.ldko : kw;
  if (p.ldq < qw || p.ldqo < qw || p.ldk < kw || p.ldv < kw || p.ldko < kw)
    return fail(SOFIE_B200_ERR_INVALID, "kv_append_enqueue: a token pitch is smaller than heads * head size");
  if (!cu_seqlens && d.tokens != kv->batch)
    return fail(SOFIE_B200_ERR_INVALID, "kv_append_enqueue: without cu_seqlens every sequence has one token (%lld tokens, batch %lld)",
                (long long)d.tokens, (long long)kv->batch);
  if (d.tokens > 0 && kv->batch > 0) {
    if (!k || !v || (d.heads > 0 && (!q || !q_out))) return fail(SOFIE_B200_ERR_INVALID, "kv_append_enqueue: NULL tensor pointer");
    if (d.rotary_dim > 0 && (!cos || !sin || d.max_position < 1)) return fail(SOFIE_B200_ERR_INVALID, "kv_append_enqueue: a rotation needs cos and sin");
    if ((q_out == q && q && p.ldqo != p.ldq) || (k_out == k && p.ldko != p.ldk))
      return fail(SOFIE_B200_ERR_INVALID, "kv_append_enqueue: a rotation in place keeps the pitch");
  }
  if (!ctx) return fail(SOFIE_B200_ERR_INVALID, "kv_append_enqueue: ctx is NULL");
  if (d.tokens == 0 || kv->batch == 0) return 0;
  SB_CUDA(cudaSetDevice(ctx->device));
  p.cu = cu_seqlens;
  p.q = q; p.k = k; p.v = v;
  p.q_out = q_out; p.k_out = k_out;
  p.cache_k = kv->k; p.cache_v = kv->v;
  p.cos = cos; p.sin = sin;
  p.tokens = (int)d.tokens; p.heads = d.heads; p.kv_heads = d.kv_heads; p.dim = d.head_dim;
  p.half = d.rotary_dim / 2; p.interleaved = d.interleaved != 0;
  p.max_position = d.max_position;
  p.status = ctx->d_status;
  if (d.dtype == SOFIE_B200_F32) kv_append_kernel<float><<<(unsigned)d.tokens, 256, 0, ctx->stream>>>(p);
  else kv_append_kernel<__nv_bfloat16><<<(unsigned)d.tokens, 256, 0, ctx->stream>>>(p);
  SB_CUDA(cudaGetLastError());
  ctx->launches++;
  return 0;
}
