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

// Position of token t and the element offset of its place in the cache (negative: no place, the token is left out), found by a warp:
// 32 offsets of cu_seqlens at a time, so two rounds of loads for a thousand sequences.
__device__ __forceinline__ long long find_place(const AppendParams &p, int t, int *pos_out) {
  const int lane = threadIdx.x & 31;
  int b = t;
  if (p.cu) {
    int lo = 0, hi = p.kv.batch;
    while (hi - lo > 1) {
      const int at = search_probe(lo, hi, lane);
      const uint32_t below = __ballot_sync(0xffffffffu, at < hi && p.cu[at] <= t);
      search_narrow(lo, hi, below ? 31 - __clz(below) : 0);
    }
    b = p.cu[lo] <= t && t < p.cu[lo + 1] ? lo : -1;
  }
  if (b < 0) return -1;
  const int len = p.kv.lens[b];
  int pos = len - 1;
  if (p.cu) {
    int begin, end;
    bool bad = false;
    packed_range(p.cu, b, p.tokens, &begin, &end, &bad);
    pos = bad ? -1 : len - (end - t);
  }
  long long row = -1;
  if (pos >= 0 && (p.half == 0 || pos < p.max_position)) row = paged_row(p.kv, b, pos);
  if (row < 0 && !(p.cu == nullptr && len == 0) && lane == 0) report(p.status, DEV_BAD_INDEX);
  *pos_out = pos;
  return row;
}

// A piece of V elements as they lie in memory (V * sizeof(T) = 16, 8, 4 or 2 bytes).
template <class T, int V>
struct alignas(sizeof(T) * V) Piece {
  T x[V];
};

// One block per token, a thread per unit: V elements of the first half of the rotated dimensions of a head with the V of the second
// half that turn with them (or V / 2 neighbouring pairs), so q_out may be q; or V elements that are only copied.  Bound by HBM where
// tokens are many: every element is read once and written once, 16 bytes at a time where the layout allows it.  What a token's place
// is takes a chain of dependent loads, so the first two units of every thread are on their way before it is known.
template <class T, int V>
__global__ void __launch_bounds__(256) kv_append_kernel(const AppendParams p) {
  constexpr int AHEAD = 2;
  const int t = blockIdx.x;
  __shared__ int s_pos;
  __shared__ long long s_row;
  const T *q = static_cast<const T *>(p.q) + t * p.ldq;
  const T *k = static_cast<const T *>(p.k) + t * p.ldk;
  const T *v = static_cast<const T *>(p.v) + t * p.ldv;
  const bool single = V == 1 && p.interleaved;                    // neighbours in pieces of their own
  const int gap = single ? 1 : p.half;                            // from a piece to the one that turns with it
  const int pairs = p.interleaved && !single ? 0 : p.half / V;    // units of a head that hold two pieces
  const int units = p.dim / V - pairs, plain = p.dim / V;         // units of a head of q or k; of v
  const int turned = (p.heads + p.kv_heads) * units, all = turned + p.kv_heads * plain;
  struct Unit {
    int head, at;        // head: queries, then keys, then values; first element inside the head
    bool two;
  };
  auto unit = [&](int i) {
    Unit u;
    if (i < turned) {
      u.head = i / units;
      const int w = i - u.head * units;
      u.two = w < pairs;
      u.at = u.two ? w * (single ? 2 : V) : (w + pairs) * V;
    } else {
      i -= turned;
      u.head = i / plain;
      u.at = (i - u.head * plain) * V;
      u.head += p.heads + p.kv_heads;
      u.two = false;
    }
    return u;
  };
  auto source = [&](const Unit &u) {
    const int h = u.head;
    return h < p.heads ? q + h * p.dim : h < p.heads + p.kv_heads ? k + (h - p.heads) * p.dim : v + (h - p.heads - p.kv_heads) * p.dim;
  };
  Piece<T, V> a[AHEAD], b[AHEAD];
#pragma unroll
  for (int j = 0; j < AHEAD; ++j) {
    const int i = threadIdx.x + j * 256;
    if (i < all) {
      const Unit u = unit(i);
      const T *src = source(u) + u.at;
      a[j] = *reinterpret_cast<const Piece<T, V> *>(src);
      if (u.two) b[j] = *reinterpret_cast<const Piece<T, V> *>(src + gap);
    }
  }
  if (threadIdx.x < 32) {
    int pos = -1;
    const long long row = find_place(p, t, &pos);
    if (threadIdx.x == 0) {
      s_pos = pos;
      s_row = row;
    }
  }
  __syncthreads();
  const int pos = s_pos;
  const long long row = s_row;
  if (row < 0) return;
  T *qo = static_cast<T *>(p.q_out) + t * p.ldqo;
  T *ko = p.k_out ? static_cast<T *>(p.k_out) + t * p.ldko : nullptr;
  T *ck = static_cast<T *>(p.cache_k) + row, *cv = static_cast<T *>(p.cache_v) + row;
  const float *cs = p.cos + (long long)pos * p.half, *sn = p.sin + (long long)pos * p.half;
  auto finish = [&](const Unit &u, Piece<T, V> x, Piece<T, V> y) {
    const int kh = u.head - p.heads, vh = kh - p.kv_heads;
    T *dst = kh < 0 ? qo + u.head * p.dim : vh < 0 ? ck + kh * p.kv.head_stride : cv + vh * p.kv.head_stride;
    T *dst2 = kh >= 0 && vh < 0 && ko ? ko + kh * p.dim : nullptr;
    if (u.two) {
      const int angle = single ? u.at / 2 : u.at;
      const Piece<float, V> c = *reinterpret_cast<const Piece<float, V> *>(cs + angle), s = *reinterpret_cast<const Piece<float, V> *>(sn + angle);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float f = to_f32(x.x[e]), g = to_f32(y.x[e]);
        from_f32(&x.x[e], f * c.x[e] - g * s.x[e]);
        from_f32(&y.x[e], g * c.x[e] + f * s.x[e]);
      }
      *reinterpret_cast<Piece<T, V> *>(dst + u.at + gap) = y;
      if (dst2) *reinterpret_cast<Piece<T, V> *>(dst2 + u.at + gap) = y;
    } else if constexpr (V >= 2) {   // pairs of neighbours inside the piece
      if (p.interleaved && vh < 0 && u.at < 2 * p.half) {
        constexpr int W = V / 2;
        const Piece<float, W> c = *reinterpret_cast<const Piece<float, W> *>(cs + u.at / 2), s = *reinterpret_cast<const Piece<float, W> *>(sn + u.at / 2);
#pragma unroll
        for (int e = 0; e < W; ++e) {
          const float f = to_f32(x.x[2 * e]), g = to_f32(x.x[2 * e + 1]);
          from_f32(&x.x[2 * e], f * c.x[e] - g * s.x[e]);
          from_f32(&x.x[2 * e + 1], g * c.x[e] + f * s.x[e]);
        }
      }
    }
    *reinterpret_cast<Piece<T, V> *>(dst + u.at) = x;
    if (dst2) *reinterpret_cast<Piece<T, V> *>(dst2 + u.at) = x;
  };
#pragma unroll
  for (int j = 0; j < AHEAD; ++j) {
    const int i = threadIdx.x + j * 256;
    if (i < all) finish(unit(i), a[j], b[j]);
  }
  for (int i = threadIdx.x + AHEAD * 256; i < all; i += 256) {
    const Unit u = unit(i);
    const T *src = source(u) + u.at;
    Piece<T, V> x = *reinterpret_cast<const Piece<T, V> *>(src), y;
    if (u.two) y = *reinterpret_cast<const Piece<T, V> *>(src + gap);
    finish(u, x, y);
  }
}

// The widest piece that divides every extent and stride and to which every tensor is aligned.  10,832 tokens of 32 + 2 x 8 heads of 128
// in bf16: 16-byte pieces MEASURED_VEC, single elements 131 us.
static int widest_piece(const AppendParams &p, int es) {
  uint64_t bits = (uint64_t)p.dim | (uint64_t)p.ldq | (uint64_t)p.ldk | (uint64_t)p.ldv | (uint64_t)p.ldqo | (uint64_t)p.ldko | (uint64_t)p.kv.page_stride |
                  (uint64_t)p.kv.token_stride | (uint64_t)p.kv.head_stride | (uint64_t)(p.interleaved ? 2 * p.half : p.half);
  uint64_t address = (uint64_t)(uintptr_t)p.q | (uint64_t)(uintptr_t)p.k | (uint64_t)(uintptr_t)p.v | (uint64_t)(uintptr_t)p.q_out | (uint64_t)(uintptr_t)p.k_out |
                     (uint64_t)(uintptr_t)p.cache_k | (uint64_t)(uintptr_t)p.cache_v;
  // angles come V (halves) or V / 2 (pairs) at a time, as fp32 and at most 16 bytes a load
  const uint64_t angles = (uint64_t)(uintptr_t)p.cos | (uint64_t)(uintptr_t)p.sin;
  for (int v = 16 / es; v > 1; v /= 2)
    if (bits % v == 0 && address % (v * es) == 0 && angles % (p.interleaved ? v * 2 : v * 4) == 0) return v;
  return 1;
}

template <class T>
static void launch_append(cudaStream_t stream, const AppendParams &p, int v) {
  const unsigned grid = (unsigned)p.tokens;
  if (v == 8) {
    if constexpr (sizeof(T) == 2) kv_append_kernel<T, 8><<<grid, 256, 0, stream>>>(p);
  } else if (v == 4) {
    kv_append_kernel<T, 4><<<grid, 256, 0, stream>>>(p);
  } else if (v == 2) {
    kv_append_kernel<T, 2><<<grid, 256, 0, stream>>>(p);
  } else {
    kv_append_kernel<T, 1><<<grid, 256, 0, stream>>>(p);
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
  const int piece = widest_piece(p, dtype_size(d.dtype));
  if (d.dtype == SOFIE_B200_F32) launch_append<float>(ctx->stream, p, piece);
  else launch_append<__nv_bfloat16>(ctx->stream, p, piece);
  SB_CUDA(cudaGetLastError());
  ctx->launches++;
  return 0;
}
