// Attention over packed prompts of different lengths:
//     y[i, h] = sum_j softmax_j(scale q[i, h] . k[j, h / g]) v[j, h / g],   g = heads / kv_heads,
// over the keys of query i's own sequence, all of them or (causal) those with j <= i + lk - lq.
//
// Tiles.  The rows of a tile are (query, head of the group) pairs, 128 / g queries with their g heads side by side, so the heads
// that share a key head share its tiles from memory, short sequences fill a tile better, and the causal diagonal crosses only
// 128 / g keys of a tile.  A row of the packed tensor is g * head_dim consecutive elements per query: one TMA box.
#include <cudaTypedefs.h>
#include <math.h>
#include <mutex>
#include <new>

#include "generate.cuh"
#include "ptx.cuh"

namespace sb200 {
using namespace ptx;

struct PromptParams {
  const void *q, *k, *v;
  void *y;
  const int32_t *cu_q, *cu_k;
  long long ldq, ldk, ldv, ldy;
  long long q_rows, k_rows;
  int batch, heads, kv_heads, dim, causal;
  int group, tokens;          // heads / kv_heads; queries of a tile
  float scale_log2e;
  int *status;
};

// One tile of queries: its sequence's rows, its first query and how many of them there are.
struct PromptTile {
  int q0, k0, k_len;      // first query row of the tile and first key row of the sequence in the packed tensors; keys of the sequence
  int queries;            // 0: nothing to do
  int past;               // keys that the tile's first query sees, before clamping to [0, k_len] (causal)
};

// Tiles are counted sequence by sequence; within a sequence the last one, which sees most keys, comes first.  All threads call
// it (THREADS of them); each sums up a few neighbouring sequences.
template <int THREADS>
__device__ __forceinline__ PromptTile find_tile(const PromptParams &p, int index) {
  __shared__ long long warp_sum[THREADS / 32];
  __shared__ PromptTile s_tile;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (p.batch + THREADS - 1) / THREADS;
  const int b0 = min(p.batch, tid * per), b1 = min(p.batch, b0 + per);
  auto tiles_of = [&](int b, PromptTile &t, int &q_len) -> int {
    int x0, x1, y0, y1;
    bool bad = false;
    packed_range(p.cu_q, b, p.q_rows, &x0, &x1, &bad);
    packed_range(p.cu_k, b, p.k_rows, &y0, &y1, &bad);
    if (bad) report(p.status, DEV_BAD_INDEX);
    t.q0 = x0; t.k0 = y0; t.k_len = y1 - y0;
    q_len = bad ? 0 : x1 - x0;
    return (q_len + p.tokens - 1) / p.tokens;
  };
  PromptTile t;
  int q_len;
  long long mine = 0;   // offsets that claim rows twice can make more tiles than the grid has; the rest is left out
  for (int b = b0; b < b1; ++b) mine += tiles_of(b, t, q_len);
  long long incl = mine;
  for (int o = 1; o < 32; o <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += x;
  }
  if (lane == 31) warp_sum[warp] = incl;
  if (tid == 0) s_tile.queries = 0;
  __syncthreads();
  long long before = incl - mine;
  for (int w = 0; w < warp; ++w) before += warp_sum[w];
  if (index >= before && index < before + mine) {
    long long at = before;
    for (int b = b0; b < b1; ++b) {
      const int n = tiles_of(b, t, q_len);
      if (index < at + n) {
        const int first = (n - 1 - (int)(index - at)) * p.tokens;
        t.past = first + 1 + t.k_len - q_len;
        t.q0 += first;
        t.queries = min(p.tokens, q_len - first);
        s_tile = t;
        break;
      }
      at += n;
    }
  }
  __syncthreads();
  return s_tile;
}

// Keys that query i of the tile sees.
__device__ __forceinline__ int seen(const PromptParams &p, const PromptTile &t, int i) {
  return p.causal ? min(t.k_len, max(0, t.past + i)) : t.k_len;
}

// ---- fp32 (and the first form of every type): one warp per (query, head), lane l holds dimensions l, l + 32, ... ----------------
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

// ---- bf16 on the tensor cores --------------------------------------------------------------------------------------------------
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// D (tensor memory) += A (tensor memory: 128 rows, two bf16 per 32-bit column) * B (shared memory)
__device__ __forceinline__ void umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tmem_st_x32(uint32_t taddr, const uint32_t *r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
      "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]),
      "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

constexpr int PU_THREADS = 192;   // warps 0-3: a row of the tile per thread; warp 4: TMA; warp 5: MMA
constexpr int PU_KEYS = 128;      // keys of a tile

template <int DP>
struct UmmaCfg {
  static constexpr int PANELS = DP / 64;                   // a panel: 128 rows x 64 elements, 128-byte swizzle
  static constexpr int TILE = PANELS * 16384;              // Q, or one tile of K or V
  static constexpr int STAGES = DP == 64 ? 2 : 1;          // tiles of K (and of V) in flight
  static constexpr int SMEM = (1 + 2 * STAGES) * TILE + 1024 /*barriers*/ + 1024 /*alignment*/;
  static constexpr int O_COL = 128;                        // tensor memory: scores in columns 0 .. 127, the result from here
  static constexpr int COLS = DP <= 128 ? 256 : 512;
  static constexpr bool EARLY = DP == 64;                  // the weights have columns of their own: scores of the next tile meanwhile
  static constexpr int P_COL = EARLY ? 192 : 0;
};

// The plain sum for one row, from global memory.  Taken when values that some rows of a tile do not see hold NaN or infinities: the
// tensor cores multiply every value by every row's weight, and 0 * NaN would reach rows it must not reach.
__device__ __noinline__ void plain_row(const PromptParams &p, long long q_row, int head, int k0, int n) {
  typedef __nv_bfloat16 T;
  const T *q = static_cast<const T *>(p.q) + q_row * p.ldq + (long long)head * p.dim;
  T *y = static_cast<T *>(p.y) + q_row * p.ldy + (long long)head * p.dim;
  const int kh = head / p.group;
  auto score = [&](int j) {
    const T *k = static_cast<const T *>(p.k) + (long long)(k0 + j) * p.ldk + (long long)kh * p.dim;
    float s = 0.f;
    for (int d = 0; d < p.dim; ++d) s = fmaf(to_f32(q[d]), to_f32(k[d]), s);
    return s * p.scale_log2e;
  };
  float m = -INFINITY, l = 0.f;
  for (int j = 0; j < n; ++j) m = fmaxf(m, score(j));
  if (m == -INFINITY) m = 0.f;
  for (int d0 = 0; d0 < p.dim; d0 += 8) {
    float acc[8] = {};
    l = 0.f;
    for (int j = 0; j < n; ++j) {
      const float e = ex2(score(j) - m);
      const T *v = static_cast<const T *>(p.v) + (long long)(k0 + j) * p.ldv + (long long)kh * p.dim + d0;
      l += e;
      for (int d = 0; d < 8; ++d) acc[d] = fmaf(e, to_f32(v[d]), acc[d]);
    }
    for (int d = 0; d < 8; ++d) from_f32(y + d0 + d, n > 0 ? acc[d] / l : 0.f);
  }
}

// A block computes one tile of 128 rows; two blocks share an SM (head sizes up to 128), so that one's softmax runs beside the other's
// tensor-core work, and its beginning and end beside the other's middle.
//   warp 4, lane 0   TMA: the queries once, then per tile of 128 keys K and V, from the last tile to the first
//   warp 5, lane 0   MMA: S = Q K^T (operands in shared memory), O += P V (P in tensor memory, V MN-major in shared memory)
//   warps 0-3        a thread per row: maximum, exponentials, row sum; P as bf16 back to tensor memory, over S's columns
// The reference maximum of a row moves only when a tile's maximum is 2^8 above it (weights stay below 2^8, exact in effect
// since numerator and denominator use the same); then O is rescaled in tensor memory, which after the first tiles is rare.
// Only tiles that the sequence's end or the diagonal cross pay for masks.
template <int DP>
__global__ void __launch_bounds__(PU_THREADS, DP <= 128 ? 2 : 1)
prompt_umma_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                   const __grid_constant__ PromptParams p) {
  using Cfg = UmmaCfg<DP>;
  constexpr int ST = Cfg::STAGES;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw), pad = (1024u - (raw & 1023u)) & 1023u;
  const uint32_t sm_q = raw + pad, sm_kv = sm_q + Cfg::TILE;   // [stage][K | V]
  uint8_t *gen = smem_raw + pad;
  uint8_t *tail = gen + (1 + 2 * ST) * Cfg::TILE;
  const uint32_t bar_q = smem_u32(tail);             // queries landed
  const uint32_t bar_kf = bar_q + 8;                 // [ST] keys landed
  const uint32_t bar_ke = bar_kf + 8 * ST;           // [ST] keys read
  const uint32_t bar_vf = bar_ke + 8 * ST;           // [ST] values landed
  const uint32_t bar_ve = bar_vf + 8 * ST;           // [ST] values read (the product of the tile is complete)
  const uint32_t bar_s = bar_ve + 8 * ST;            // scores complete in tensor memory
  const uint32_t bar_se = bar_s + 8;                 // scores read (EARLY)
  const uint32_t bar_p = bar_se + 8;                 // weights written to tensor memory
  const uint32_t bar_o = bar_p + 8;                  // result complete
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(tail + 256);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tail + 260);
  volatile int *unclean = reinterpret_cast<volatile int *>(tail + 264);   // non-finite values where the mask hides some of them
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  const int kh = blockIdx.x % p.kv_heads;
  const PromptTile t = find_tile<PU_THREADS>(p, blockIdx.x / p.kv_heads);
  if (t.queries == 0) return;
  const int lim_lo = seen(p, t, 0), lim_hi = seen(p, t, t.queries - 1);   // keys that the first and the last query see
  const int n = (lim_hi + PU_KEYS - 1) / PU_KEYS;                          // tiles of keys

  if (tid == 0) {
    mbar_init(bar_q, 1);
    for (int s = 0; s < ST; ++s) {
      mbar_init(bar_kf + 8 * s, 1);
      mbar_init(bar_ke + 8 * s, 1);
      mbar_init(bar_vf + 8 * s, 1);
      mbar_init(bar_ve + 8 * s, 1);
    }
    mbar_init(bar_s, 1);
    mbar_init(bar_se, 4);
    mbar_init(bar_p, 4);
    mbar_init(bar_o, 1);
    *abort_flag = 0;
    *unclean = 0;
    fence_barrier_init();
  }
  if (warp == 5) {
    tmem_alloc(smem_u32(tmem_slot), Cfg::COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 4) {
    if (lane == 0 && n > 0) {
      bool ok = true;
      mbar_arrive_expect_tx(bar_q, Cfg::PANELS * 128 * p.group * p.tokens);
      for (int c = 0; c < Cfg::PANELS; ++c) tma_load_3d(sm_q + c * 16384, &tm_q, bar_q, 64 * c, kh * p.group, t.q0);
      for (int it = 0; it < n && ok; ++it) {
        const uint32_t st = it % ST, ph = (it / ST) & 1;
        const int row = t.k0 + (n - 1 - it) * PU_KEYS;
        const uint32_t dk = sm_kv + st * 2 * Cfg::TILE, dv = dk + Cfg::TILE;
        if (!(ok = mbar_wait(bar_ke + 8 * st, ph ^ 1u, abort_flag))) break;
        mbar_arrive_expect_tx(bar_kf + 8 * st, Cfg::TILE);
        for (int c = 0; c < Cfg::PANELS; ++c) tma_load_3d(dk + c * 16384, &tm_k, bar_kf + 8 * st, 64 * c, kh, row);
        if (!(ok = mbar_wait(bar_ve + 8 * st, ph ^ 1u, abort_flag))) break;
        mbar_arrive_expect_tx(bar_vf + 8 * st, Cfg::TILE);
        for (int c = 0; c < Cfg::PANELS; ++c) tma_load_3d(dv + c * 16384, &tm_v, bar_vf + 8 * st, 64 * c, kh, row);
      }
      if (!ok) {
        *abort_flag = 1;
        report(p.status, DEV_WAIT_SMEM_EMPTY);
        const uint64_t t0 = globaltimer();   // copies in flight land before the block ends
        while (globaltimer() - t0 < 200000ull) {}
      }
    }
  } else if (warp == 5) {
    if (lane == 0 && n > 0) {
      // descriptors: 128-byte swizzle, 1024 bytes between groups of 8 rows, version 1
      const uint64_t desc_hi = (uint64_t)((1024u >> 4) | (1u << 14) | (2u << 29)) << 32;
      const uint32_t kmajor = 1u << 16, mnmajor = (16384u >> 4) << 16;   // MN-major: leading offset = one panel
      const uint32_t idesc_s = (1u << 4) | (1u << 7) | (1u << 10) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
      const uint32_t idesc_o = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | (((uint32_t)DP >> 3) << 17) | ((128u >> 4) << 24);
      bool ok = true;
      auto scores = [&](int it) -> bool {
        const uint32_t st = it % ST, ph = (it / ST) & 1;
        if (!mbar_wait(bar_kf + 8 * st, ph, abort_flag)) return false;
        tc_fence_after();
        const uint32_t k = sm_kv + st * 2 * Cfg::TILE;
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk) {
          const uint32_t off = (kk >> 2) * 16384 + (kk & 3) * 32;
          umma<KIND_F16>(tmem, desc_hi | (uint64_t)(kmajor | (((sm_q + off) >> 4) & 0x3fffu)), desc_hi | (uint64_t)(kmajor | (((k + off) >> 4) & 0x3fffu)),
                         idesc_s, kk != 0);
        }
        tc_commit(bar_s);
        tc_commit(bar_ke + 8 * st);
        return true;
      };
      ok = mbar_wait(bar_q, 0, abort_flag) && scores(0);
      for (int it = 0; it < n && ok; ++it) {
        const uint32_t st = it % ST, ph = (it / ST) & 1;
        if (Cfg::EARLY && it + 1 < n && !(ok = mbar_wait(bar_se, it & 1, abort_flag) && scores(it + 1))) break;
        if (!(ok = mbar_wait(bar_p, it & 1, abort_flag) && mbar_wait(bar_vf + 8 * st, ph, abort_flag))) break;
        tc_fence_after();
        const uint32_t v = sm_kv + st * 2 * Cfg::TILE + Cfg::TILE;
#pragma unroll
        for (int kk = 0; kk < PU_KEYS / 16; ++kk)   // 16 keys: 8 columns of P, 16 rows of V
          umma_ts(tmem + Cfg::O_COL, tmem + Cfg::P_COL + 8 * kk, desc_hi | (uint64_t)(mnmajor | (((v + 2048 * kk) >> 4) & 0x3fffu)), idesc_o,
                  it != 0 || kk != 0);
        tc_commit(bar_ve + 8 * st);
        if (it + 1 == n) tc_commit(bar_o);
        // without columns of their own the weights lie where the next scores go: that product follows this one in the pipe
        if (!Cfg::EARLY && it + 1 < n && !(ok = scores(it + 1))) break;
      }
      if (!ok) {
        *abort_flag = 1;
        report(p.status, DEV_WAIT_SMEM_FULL);
      }
    }
  } else {
    const int row = warp * 32 + lane;
    const int query = row / p.group, head = row - query * p.group;
    const bool mine = query < t.queries;          // rows past the tile's last query (and past tokens * group) hold anything
    const int lim = mine ? seen(p, t, query) : lim_hi;
    const uint32_t lanes = (uint32_t)(warp * 32) << 16;
    const uint32_t t_s = tmem + lanes, t_p = t_s + Cfg::P_COL, t_o = t_s + Cfg::O_COL;
    const float c = p.scale_log2e;
    float m = -INFINITY, l = 0.f;   // reference maximum of the unscaled scores; sum of the weights
    bool ok = true;
    for (int it = 0; it < n; ++it) {
      const int base = (n - 1 - it) * PU_KEYS;
      const uint32_t st = it % ST, ph = (it / ST) & 1;
      if (!(ok = mbar_wait(bar_s, it & 1, abort_flag))) break;
      tc_fence_after();
      uint32_t r[PU_KEYS];
      float *s = reinterpret_cast<float *>(r);
      tmem_ld_x32(t_s, r);
      tmem_ld_x32(t_s + 32, r + 32);
      tmem_ld_x32(t_s + 64, r + 64);
      tmem_ld_x32(t_s + 96, r + 96);
      tmem_ld_wait();
      if (Cfg::EARLY) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_se);
      }
      const bool masked = base + PU_KEYS > lim_lo;
      if (masked) {
        const int have = lim - base;
#pragma unroll
        for (int i = 0; i < PU_KEYS; ++i) s[i] = i < have ? s[i] : -INFINITY;
      }
      float x0 = s[0], x1 = s[1], x2 = s[2], x3 = s[3];
#pragma unroll
      for (int i = 4; i < PU_KEYS; i += 4) {
        x0 = fmaxf(x0, s[i]);
        x1 = fmaxf(x1, s[i + 1]);
        x2 = fmaxf(x2, s[i + 2]);
        x3 = fmaxf(x3, s[i + 3]);
      }
      const float top = fmaxf(fmaxf(x0, x1), fmaxf(x2, x3));
      if (Cfg::EARLY && it > 0) {   // O and P are free
        if (!(ok = mbar_wait(bar_ve + 8 * ((it - 1) % ST), ((it - 1) / ST) & 1, abort_flag))) break;
        tc_fence_after();
      }
      if (it == 0) {
        m = top;
      } else {
        const bool up = (top - m) * c > 8.f;
        if (__any_sync(0xffffffffu, up)) {
          tc_fence_after();
          const float f = up ? ex2((m - top) * c) : 1.f;
          if (up) m = top;
          l *= f;
#pragma unroll
          for (int d = 0; d < DP; d += 32) {
            uint32_t o[32];
            tmem_ld_x32(t_o + d, o);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
            tmem_st_x32(t_o + d, o);
          }
        }
      }
      const float off = m == -INFINITY ? 0.f : -m * c;
      const float2 c2 = make_float2(c, c), off2 = make_float2(off, off);
      float2 sum0 = make_float2(0.f, 0.f), sum1 = make_float2(0.f, 0.f);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t w[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          float2 e = __ffma2_rn(make_float2(s[half * 64 + 2 * i], s[half * 64 + 2 * i + 1]), c2, off2);
          e.x = ex2(e.x);
          e.y = ex2(e.y);
          if (i & 1) sum1 = __fadd2_rn(sum1, e);
          else sum0 = __fadd2_rn(sum0, e);
          const __nv_bfloat162 h = __floats2bfloat162_rn(e.x, e.y);
          w[i] = *reinterpret_cast<const uint32_t *>(&h);
        }
        tmem_st_x32(t_p + 32 * half, w);
      }
      l += (sum0.x + sum0.y) + (sum1.x + sum1.y);
      if (masked) {
        // Values past the tile's last key belong to others and may hold anything: zeros in their place.  Values on the diagonal
        // are hidden from some rows: if one is not finite, the rows are computed the plain way at the end.
        if (!(ok = mbar_wait(bar_vf + 8 * st, ph, abort_flag))) break;
        uint8_t *v = gen + (sm_kv - sm_q) + st * 2 * Cfg::TILE + Cfg::TILE;
        const int none = max(0, min(PU_KEYS, lim_hi - base)), some = max(0, min(none, lim_lo - base));
        for (int i = none * 8 * Cfg::PANELS + tid; i < PU_KEYS * 8 * Cfg::PANELS; i += 128) {
          const int key = i / (8 * Cfg::PANELS), piece = i % (8 * Cfg::PANELS);
          *reinterpret_cast<uint4 *>(v + (piece >> 3) * 16384 + key * 128 + (piece & 7) * 16) = make_uint4(0, 0, 0, 0);
        }
        bool bad = false;
        for (int i = some * 8 * Cfg::PANELS + tid; i < none * 8 * Cfg::PANELS; i += 128) {
          const int key = i / (8 * Cfg::PANELS), piece = i % (8 * Cfg::PANELS);
          const uint4 x = *reinterpret_cast<const uint4 *>(v + (piece >> 3) * 16384 + key * 128 + (piece & 7) * 16);
          for (uint32_t u : {x.x, x.y, x.z, x.w}) bad |= (u & 0x7f80u) == 0x7f80u || (u & 0x7f800000u) == 0x7f800000u;
        }
        if (bad) *unclean = 1;
        fence_proxy_async();
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_p);
    }
    if (ok && n > 0) ok = mbar_wait(bar_o, 0, abort_flag);
    if (!ok) {
      *abort_flag = 1;
      report(p.status, DEV_WAIT_TMEM_FULL);
    } else {
      tc_fence_after();
      const long long q_row = (long long)t.q0 + query;
      if (n > 0 && *unclean) {
        if (mine) plain_row(p, q_row, kh * p.group + head, t.k0, lim);
      } else {
        // through shared memory (the queries are read), so that a row leaves in whole lines
        const float inv = 1.f / l;
        const bool none = lim <= 0;
        constexpr int PIECES = DP / 8;
        uint8_t *out = gen + warp * 32 * (DP * 2);
#pragma unroll
        for (int d = 0; d < DP; d += 32) {
          uint32_t o[32];
          if (n > 0) {
            tmem_ld_x32(t_o + d, o);
            tmem_ld_wait();
          }
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const __nv_bfloat162 h = n > 0 && !none ? __floats2bfloat162_rn(__uint_as_float(o[i + 2 * k]) * inv, __uint_as_float(o[i + 2 * k + 1]) * inv)
                                                      : __floats2bfloat162_rn(0.f, 0.f);
              w[k] = *reinterpret_cast<const uint32_t *>(&h);
            }
            const int piece = (d + i) / 8;
            *reinterpret_cast<uint4 *>(out + lane * (DP * 2) + ((piece ^ (lane & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
        __syncwarp();
        __nv_bfloat16 *y = static_cast<__nv_bfloat16 *>(p.y) + (long long)t.q0 * p.ldy + (long long)kh * p.group * p.dim;
#pragma unroll 4
        for (int i = lane; i < 32 * PIECES; i += 32) {
          const int r = i / PIECES, piece = i % PIECES, at = warp * 32 + r;
          const int qi = at / p.group, hi = at - qi * p.group;
          if (qi < t.queries && piece * 8 < p.dim)
            *reinterpret_cast<uint4 *>(y + qi * p.ldy + hi * p.dim + piece * 8) = *reinterpret_cast<const uint4 *>(out + r * (DP * 2) + ((piece ^ (r & 7)) << 4));
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 5) {
    tc_fence_after();
    tmem_dealloc(tmem, Cfg::COLS);
  }
}

static PFN_cuTensorMapEncodeTiled_v12000 get_encode_prompt() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void *sym = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(sym);
  });
  return fn;
}

// [rows, heads, dim] bf16 with a pitch; box: 64 elements x box_heads x box_rows, 128-byte swizzle
static int encode_rows(CUtensorMap *tm, const void *base, int dim, int heads, long long rows, long long pitch, int box_heads, int box_rows) {
  auto enc = get_encode_prompt();
  if (!enc) return fail(SOFIE_B200_ERR_NO_DEVICE, "cuTensorMapEncodeTiled entry point not available");
  cuuint64_t dims[3] = {(cuuint64_t)dim, (cuuint64_t)heads, (cuuint64_t)rows};
  cuuint64_t strides[2] = {(cuuint64_t)dim * 2, (cuuint64_t)pitch * 2};
  cuuint32_t box[3] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_rows};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = enc(tm, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void *>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(SOFIE_B200_ERR_CUDA, "prompt_attention: cuTensorMapEncodeTiled failed (%d)", (int)r);
  return 0;
}

template <int DP>
static int launch_umma(sofie_b200_ctx *ctx, const PromptParams &p, unsigned grid) {
  CUtensorMap tm_q, tm_k, tm_v;
  const void *k = p.k_rows ? p.k : p.q, *v = p.k_rows ? p.v : p.q;   // no keys: nothing is loaded, but a map has to describe something
  const long long k_rows = p.k_rows ? p.k_rows : 1;
  int rc;
  if ((rc = encode_rows(&tm_q, p.q, p.dim, p.heads, p.q_rows, p.ldq, p.group, p.tokens))) return rc;
  if ((rc = encode_rows(&tm_k, k, p.dim, p.kv_heads, k_rows, p.ldk, 1, PU_KEYS))) return rc;
  if ((rc = encode_rows(&tm_v, v, p.dim, p.kv_heads, k_rows, p.ldv, 1, PU_KEYS))) return rc;
  SB_CUDA(cudaFuncSetAttribute(prompt_umma_kernel<DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, UmmaCfg<DP>::SMEM));   // per device
  prompt_umma_kernel<DP><<<grid, PU_THREADS, UmmaCfg<DP>::SMEM, ctx->stream>>>(tm_q, tm_k, tm_v, p);
  SB_CUDA(cudaGetLastError());
  ctx->launches++;
  return 0;
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

const char *sofie_b200_prompt_attention_plan_kernel(const sofie_b200_prompt_attention_plan *plan) {
  return !plan ? "" : plan->d.dtype == SOFIE_B200_F32 ? "rows" : "umma";
}

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
  p.group = d.heads / d.kv_heads;
  p.scale_log2e = d.scale * 1.4426950408889634f;
  p.status = ctx->d_status;
  if (d.dtype == SOFIE_B200_BF16) {
    p.tokens = 128 / p.group;
    const int64_t blocks = (q_tokens / p.tokens + batch) * d.kv_heads;   // every sequence may end inside a tile
    if (blocks > 0x7fffffffLL) return fail(SOFIE_B200_ERR_TOO_LARGE, "prompt_attention_enqueue: %lld queries of %d heads", (long long)q_tokens, d.heads);
    if (d.head_dim <= 64) return launch_umma<64>(ctx, p, (unsigned)blocks);
    if (d.head_dim <= 128) return launch_umma<128>(ctx, p, (unsigned)blocks);
    return launch_umma<256>(ctx, p, (unsigned)blocks);
  }
  const int64_t blocks = (q_tokens * d.heads + 3) / 4;
  if (blocks > 0x7fffffffLL) return fail(SOFIE_B200_ERR_TOO_LARGE, "prompt_attention_enqueue: %lld queries of %d heads", (long long)q_tokens, d.heads);
  prompt_rows_kernel<float><<<(unsigned)blocks, 128, 0, ctx->stream>>>(p);
  SB_CUDA(cudaGetLastError());
  ctx->launches++;
  return 0;
}

}  // extern "C"
