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

// Position of token t in its sequence (and which that is), found by a warp: 32 sequences at a time, their offsets and lengths side by
// side, so that one round of loads does for up to 32 sequences and two for a thousand.  Negative: the token has no place, and `bad` says
// whether that is an error (a row behind the last sequence and a padding row are none).
__device__ __forceinline__ int find_position(const AppendParams &p, int t, int *seq, bool *bad) {
  const int lane = threadIdx.x & 31;
  *bad = false;
  *seq = t;
  if (!p.cu) {
    const int len = p.kv.lens[t];
    *bad = len < 0;
    return len - 1;
  }
  int lo = 0, hi = p.kv.batch;
  while (hi - lo > 32) {
    const int at = search_probe(lo, hi, lane);
    const uint32_t below = __ballot_sync(0xffffffffu, at < hi && p.cu[at] <= t);
    search_narrow(lo, hi, below ? 31 - __clz(below) : 0);
  }
  int begin = 0, end = 0, len = 0;
  if (lo + lane < hi) {
    begin = p.cu[lo + lane];
    end = p.cu[lo + lane + 1];
    len = p.kv.lens[lo + lane];
  }
  const uint32_t here = __ballot_sync(0xffffffffu, begin <= t && t < end);
  if (!here) return -1;
  const int src = __ffs(here) - 1;
  begin = __shfl_sync(0xffffffffu, begin, src);
  end = __shfl_sync(0xffffffffu, end, src);
  len = __shfl_sync(0xffffffffu, len, src);
  *seq = lo + src;
  *bad = begin < 0 || end > p.tokens || len < end - t;
  return *bad ? -1 : len - (end - t);
}

// A piece of V elements as they lie in memory (V * sizeof(T) = 16, 8, 4 or 2 bytes).
template <class T, int V>
struct alignas(sizeof(T) * V) Piece {
  T x[V];
};

// GROUP threads per token (a block or two warps).  A unit of a query or key head is V elements of the first half of its rotated dimensions
// with the V of the second half that turn with them (or V / 2 neighbouring pairs), so q_out may be q; or V elements that are only
// copied.  A thread has the same unit of several heads, so its angles are loaded once.  Bound by HBM where tokens are many: every element
// is read once and written once, 16 bytes at a time where the layout allows it; what keeps it from the copy rate is that a thread
// waits for its loads, two heads at a time (more take registers, and with them warps: 4 heads 79 us, 2 heads 62 us at 10,832 tokens of
// 32 + 2 x 8 heads of 128 in bf16 = 4.4 TB/s).  Even so that form, <bf16, 8, 64>, spills at its 64 registers: 150 bytes of stores and 200 of
// loads a thread, as the pieces of values and the angles are held across the look-up of the token's place.  The first heads are on their way before the token's place is known, which takes two or
// three rounds of dependent loads.
template <class T, int V, int GROUP>
__global__ void __launch_bounds__(256, GROUP < 256 ? 4 : 1) kv_append_kernel(const __grid_constant__ AppendParams p) {
  constexpr int AHEAD = 2;   // heads under way, and pieces of values
  typedef Piece<T, V> P;
  const int t = blockIdx.x * (256 / GROUP) + threadIdx.x / GROUP, me = threadIdx.x % GROUP;
  if (GROUP < 256 && t >= p.tokens) return;
  const bool single = V == 1 && p.interleaved;                    // neighbours in pieces of their own
  const int gap = single ? 1 : p.half;                            // from a piece to the one that turns with it
  const int pairs = p.interleaved && !single ? 0 : p.half / V;    // units of a head that hold two pieces
  const int units = p.dim / V - pairs, heads = p.heads + p.kv_heads;
  const int side = units < GROUP ? GROUP / units : 1;             // heads side by side
  const int first = units < GROUP ? me / units : 0;               // this thread's first head
  int u = units < GROUP ? me - first * units : me;                // its unit; with more units than threads also u + GROUP, ...
  const bool works = first < side && u < units;
  const T *q = static_cast<const T *>(p.q) + t * p.ldq;
  const T *k = static_cast<const T *>(p.k) + t * p.ldk - p.heads * p.dim;   // heads counted on from the queries'
  const T *v = static_cast<const T *>(p.v) + t * p.ldv;
  const int pieces = p.dim / V, values = p.kv_heads * pieces;
  P x[AHEAD], y[AHEAD], w[AHEAD];
  Piece<float, V> c, sn;
  bool two, inside;
  int at;
  auto choose = [&]() {
    two = u < pairs;
    at = two ? u * (single ? 2 : V) : (u + pairs) * V;
    inside = V > 1 && p.interleaved && at < 2 * p.half;   // pairs of neighbours inside the piece
  };
  auto angles = [&](int pos) {
    const float *cs = p.cos + (long long)pos * p.half, *ss = p.sin + (long long)pos * p.half;
    if (two) {
      c = *reinterpret_cast<const Piece<float, V> *>(cs + (single ? at / 2 : at));
      sn = *reinterpret_cast<const Piece<float, V> *>(ss + (single ? at / 2 : at));
    } else if (inside) {
      constexpr int W = V > 1 ? V / 2 : 1;
      const Piece<float, W> cw = *reinterpret_cast<const Piece<float, W> *>(cs + at / 2), sw = *reinterpret_cast<const Piece<float, W> *>(ss + at / 2);
#pragma unroll
      for (int e = 0; e < W; ++e) c.x[e] = cw.x[e], sn.x[e] = sw.x[e];
    }
  };
  auto take = [&](int h) {   // heads h, h + side, ...
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const int hh = h + j * side;
      if (hh < heads) {
        const T *src = (hh < p.heads ? q : k) + hh * p.dim + at;
        x[j] = *reinterpret_cast<const P *>(src);
        if (two) y[j] = *reinterpret_cast<const P *>(src + gap);
      }
    }
  };
  auto take_values = [&](int i0) {
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
      if (i0 + j * GROUP < values) w[j] = *reinterpret_cast<const P *>(v + (i0 + j * GROUP) * V);
  };
  choose();
  if (works) take(first);
  take_values(me);

  int pos, seq;
  bool bad;
  if (GROUP < 256) {   // every warp for itself
    pos = find_position(p, t, &seq, &bad);
  } else {
    __shared__ int s_pos, s_seq;
    __shared__ bool s_bad;
    if (threadIdx.x < 32) {
      pos = find_position(p, t, &seq, &bad);
      if (threadIdx.x == 0) s_pos = pos, s_seq = seq, s_bad = bad;
    }
    __syncthreads();
    pos = s_pos, seq = s_seq, bad = s_bad;
  }
  long long row = -1;
  if (pos >= 0) {
    if (p.half && pos >= p.max_position) {
      bad = true;
    } else {
      if (works) angles(pos);
      row = paged_row(p.kv, seq, pos);
      bad = row < 0;
    }
  }
  if (row < 0) {
    if (bad && me == 0) report(p.status, DEV_BAD_INDEX);
    return;
  }
  if (works) {
    T *qo = static_cast<T *>(p.q_out) + t * p.ldqo;
    T *ko = p.k_out ? static_cast<T *>(p.k_out) + t * p.ldko - p.heads * p.dim : nullptr;
    T *ck = static_cast<T *>(p.cache_k) + row - p.heads * p.kv.head_stride;
    for (bool begun = true;; begun = false) {
      for (int h = first; h < heads; h += AHEAD * side) {
        if (!begun || h != first) take(h);
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
          const int hh = h + j * side;
          if (hh < heads) {
            T *dst = hh < p.heads ? qo + hh * p.dim : ck + hh * p.kv.head_stride;
            T *dst2 = hh >= p.heads && ko ? ko + hh * p.dim : nullptr;
            if (two) {
#pragma unroll
              for (int e = 0; e < V; ++e) {
                const float f = to_f32(x[j].x[e]), g = to_f32(y[j].x[e]);
                from_f32(&x[j].x[e], f * c.x[e] - g * sn.x[e]);
                from_f32(&y[j].x[e], g * c.x[e] + f * sn.x[e]);
              }
              *reinterpret_cast<P *>(dst + at + gap) = y[j];
              if (dst2) *reinterpret_cast<P *>(dst2 + at + gap) = y[j];
            } else if (inside) {
#pragma unroll
              for (int e = 0; e + 1 < V; e += 2) {
                const float f = to_f32(x[j].x[e]), g = to_f32(x[j].x[e + 1]);
                from_f32(&x[j].x[e], f * c.x[e / 2] - g * sn.x[e / 2]);
                from_f32(&x[j].x[e + 1], g * c.x[e / 2] + f * sn.x[e / 2]);
              }
            }
            *reinterpret_cast<P *>(dst + at) = x[j];
            if (dst2) *reinterpret_cast<P *>(dst2 + at) = x[j];
          }
        }
      }
      u += GROUP;
      if (u >= units || units < GROUP) break;
      choose();
      angles(pos);
    }
  }
  // the values, as they are
  T *cv = static_cast<T *>(p.cache_v) + row;
  for (int i0 = me; i0 < values; i0 += AHEAD * GROUP) {
    if (i0 != me) take_values(i0);
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const int i = i0 + j * GROUP;
      if (i < values) {
        const int h = i / pieces;
        *reinterpret_cast<P *>(cv + h * p.kv.head_stride + (i - h * pieces) * V) = w[j];
      }
    }
  }
}

// The widest piece that divides every extent and stride and to which every tensor is aligned.  10,832 tokens of 32 + 2 x 8 heads of 128
// in bf16: 16-byte pieces 63 us, single elements 131 us.
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

template <class T, int V>
static void launch_append(sofie_b200_ctx *ctx, const AppendParams &p) {
  // Few tokens: a block each, for the shortest way (120 tokens of 32 + 2 x 8 heads of 128: as long as an empty launch either way).  From
  // four for every SM on: two warps each, four tokens to a block; of 10,832 tokens a block takes 101 us, four warps 70, two 63, one 68.
  if (p.tokens < ctx->sm_count * 4) kv_append_kernel<T, V, 256><<<(unsigned)p.tokens, 256, 0, ctx->stream>>>(p);
  else kv_append_kernel<T, V, 64><<<(unsigned)p.tokens / 4 + (p.tokens % 4 != 0), 256, 0, ctx->stream>>>(p);
}
template <class T>
static void launch_append(sofie_b200_ctx *ctx, const AppendParams &p, int v) {
  if (v == 8) {
    if constexpr (sizeof(T) == 2) launch_append<T, 8>(ctx, p);
  } else if (v == 4) {
    launch_append<T, 4>(ctx, p);
  } else if (v == 2) {
    launch_append<T, 2>(ctx, p);
  } else {
    launch_append<T, 1>(ctx, p);
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
  if (d.dtype == SOFIE_B200_F32) launch_append<float>(ctx, p, piece);
  else launch_append<__nv_bfloat16>(ctx, p, piece);
  SB_CUDA(cudaGetLastError());
  ctx->launches++;
  return 0;
}
