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
#include <type_traits>

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

// A wait of a whole warp.  The lanes leave together: one that lagged behind could find the barrier a phase further on, with the parity
// that means "not yet", and wait for good; and all of them agree on a wait that ran out.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int *abort_flag) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag));
}

// ---- bf16 on the tensor cores --------------------------------------------------------------------------------------------------
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// max(a, b, c), NaN if one of them is
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float y;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
// 2^x for x <= 2^7 on the FMA pipes: the special-function unit does 16 exponentials a cycle and SM, as long for a tile's scores as the
// tensor cores need for both products, so some of them go another way.  x = n + r with n the nearest integer (x + 1.5 * 2^23
// leaves n in the low bits), 2^r on [-1/2, 1/2] by the polynomial of degree 4 with p(0) = 1 whose largest relative error is
// least (2.9e-6, fitted to 2^r by linear programming), n added to the exponent.  Below -127 the result is 0, as ex2 flushes.
__device__ __forceinline__ float2 exp2_pair(float2 x) {
  x.x = fmaxf(x.x, -127.f);
  x.y = fmaxf(x.y, -127.f);
  const float2 t = __fadd2_rn(x, make_float2(12582912.f, 12582912.f));
  const float2 n = __fadd2_rn(t, make_float2(-12582912.f, -12582912.f));
  const float2 r = __ffma2_rn(n, make_float2(-1.f, -1.f), x);
  float2 p = __ffma2_rn(r, make_float2(0.0095828529f, 0.0095828529f), make_float2(0.0559064262f, 0.0559064262f));
  p = __ffma2_rn(p, r, make_float2(0.2402409911f, 0.2402409911f));
  p = __ffma2_rn(p, r, make_float2(0.6931241751f, 0.6931241751f));
  p = __ffma2_rn(p, r, make_float2(1.f, 1.f));
  return make_float2(__int_as_float(__float_as_int(p.x) + (__float_as_int(t.x) << 23)), __int_as_float(__float_as_int(p.y) + (__float_as_int(t.y) << 23)));
}
#ifndef SB_POLY
#define SB_POLY 0x8888u
#endif
constexpr uint32_t POLY = SB_POLY;   // of 16 pairs, those that exp2_pair takes
// The issuing warp stays together and one lane's predicate does the rest: the operands are then the same in every lane, which
// lets the compiler keep them in uniform registers.  With a branch to one lane around the products every operand was moved there
// one by one, and issuing a tile's 16 products took longer than computing them.
// D (tensor memory) = or += A (shared memory) * B (shared memory)
__device__ __forceinline__ void umma_ss(uint32_t leader, uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n.reg .pred p, q;\nsetp.ne.b32 p, %4, 0;\nsetp.ne.b32 q, %5, 0;\n"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(leader)
      : "memory");
}
// the same with A in tensor memory (128 rows, two bf16 per 32-bit column)
__device__ __forceinline__ void umma_ts(uint32_t leader, uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n.reg .pred p, q;\nsetp.ne.b32 p, %4, 0;\nsetp.ne.b32 q, %5, 0;\n"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void commit_if(uint32_t leader, uint32_t bar) {
  asm volatile(
      "{\n.reg .pred q;\nsetp.ne.b32 q, %1, 0;\n"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(bar),
      "r"(leader)
      : "memory");
}
// A value that all lanes hold, as one.
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __shfl_sync(0xffffffffu, x, 0); }
__device__ __forceinline__ void tmem_st_x16(uint32_t taddr, const uint32_t *r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
      "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// A block computes TILES tiles of 128 rows against the same keys and values.  What sets the sizes is the way from L2: a tile of keys
// and values takes about 3000 cycles from request to arrival and an SM sustains about 48 bytes per cycle, while the tensor cores
// would finish 128 rows x 128 keys of head size 128 (64 KB of keys and values) in 1024 cycles.  So at that head size two tiles of rows
// share every load (32 bytes per cycle at full rate) and five tiles of keys or values are in flight; at head size 64 half the bytes
// are needed per score, and two blocks of one tile share an SM instead, one's beginning and end beside the other's middle.
template <int DP>
struct UmmaCfg;
template <>
struct UmmaCfg<64> {
  static constexpr int TILES = 1, KEYS = 128, BLOCKS = 2, STAGES = 5, COLS = 256;
  static constexpr int S_COL = 0, O_COL = 128, P_COL = 192, STEP = 0;
  static constexpr bool EARLY = true;    // the weights have columns of their own: the next scores are computed meanwhile
  static constexpr bool HOLD = false;    // a thread holds its whole row of scores in registers
};
template <>
struct UmmaCfg<128> {
  static constexpr int TILES = 2, KEYS = 128, BLOCKS = 1, STAGES = 5, COLS = 512;
  static constexpr int S_COL = 0, O_COL = 128, P_COL = 0, STEP = 256;
  static constexpr bool EARLY = false, HOLD = true;
};
template <>
struct UmmaCfg<256> {
  static constexpr int TILES = 1, KEYS = 64, BLOCKS = 1, STAGES = 5, COLS = 512;
  static constexpr int S_COL = 0, O_COL = 256, P_COL = 64, STEP = 0;
  static constexpr bool EARLY = true, HOLD = true;
};
template <int DP>
struct UmmaSize : UmmaCfg<DP> {
  using C = UmmaCfg<DP>;
  static constexpr int PANELS = DP / 64;                    // a panel: rows x 64 elements, 128-byte swizzle
  static constexpr int Q = C::TILES * PANELS * 16384;
  static constexpr int TILE = C::KEYS * DP * 2;             // keys or values
  static constexpr int PANEL = C::KEYS * 128;
  // Warps of rows; then TMA, MMA.  Where a thread holds a row of 128 scores, 168 registers (12 warps' share) make it spill: the block
  // is launched with a whole third group of warps, which hands registers over, 384 x 168 = 256 x 216 + 128 x 72.
  static constexpr bool MOVE = C::TILES == 2;
  static constexpr int THREADS = C::TILES * 128 + (MOVE ? 128 : 64);
  static constexpr int SMEM = Q + C::STAGES * TILE + 1024 /*barriers*/ + 1024 /*alignment*/;
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

// Roles:
//   a warp, lane 0   TMA: the queries once, then per tile of keys K and V, from the last tile to the first, into a ring
//   a warp           MMA: S = Q K^T (operands in shared memory), O += P V (P in tensor memory, V MN-major in shared memory)
//   4 warps a tile   a thread per row: maximum, exponentials, row sum; P as bf16 back to tensor memory
// The reference maximum of a row moves only when a tile's maximum is 2^8 above it (weights stay below 2^8, exact in effect
// since numerator and denominator use the same); then O is rescaled in tensor memory, which after the first tiles is rare.
// Only tiles that the sequence's end or the diagonal cross pay for masks.
template <int DP>
__global__ void __launch_bounds__(UmmaSize<DP>::THREADS, UmmaSize<DP>::BLOCKS)
prompt_umma_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                   const __grid_constant__ PromptParams p) {
  using Cfg = UmmaSize<DP>;
  constexpr int ST = Cfg::STAGES, KEYS = Cfg::KEYS, TILES = Cfg::TILES;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw), pad = (1024u - (raw & 1023u)) & 1023u;
  const uint32_t sm_q = raw + pad, sm_ring = sm_q + Cfg::Q;
  uint8_t *gen = smem_raw + pad;
  uint8_t *tail = gen + Cfg::Q + ST * Cfg::TILE;
  const uint32_t bar_q = smem_u32(tail);             // queries landed
  const uint32_t bar_full = bar_q + 8;               // [ST] ring: keys or values landed
  const uint32_t bar_empty = bar_full + 8 * ST;      // [ST] the products that read them are complete
  const uint32_t bar_s = bar_empty + 8 * ST;         // [TILES] scores complete in tensor memory
  const uint32_t bar_se = bar_s + 8 * TILES;         // [TILES] scores read (EARLY)
  const uint32_t bar_p = bar_se + 8 * TILES;         // [TILES] weights written to tensor memory
  const uint32_t bar_o = bar_p + 8 * TILES;          // [TILES] result complete
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(tail + 512);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tail + 516);
  volatile int *unclean = reinterpret_cast<volatile int *>(tail + 520);   // non-finite values where the mask hides some of them
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  const int kh = blockIdx.x % p.kv_heads;
  const PromptTile t = find_tile<Cfg::THREADS>(p, blockIdx.x / p.kv_heads);
  if (t.queries == 0) return;
  const int per = 128 / p.group;                                           // queries of a tile of rows
  const int lim_lo = seen(p, t, 0), lim_hi = seen(p, t, t.queries - 1);   // keys that the first and the last query see
  const int n = (lim_hi + KEYS - 1) / KEYS;                                // tiles of keys; they are taken from the last to the first
  // a tile of rows whose last query sees fewer keys starts later; one without queries has no turn
  auto first_turn = [&](int x) {
    const int have = min(per, t.queries - x * per);
    return have <= 0 ? n : n - (seen(p, t, x * per + have - 1) + KEYS - 1) / KEYS;
  };

  if (tid == 0) {
    mbar_init(bar_q, 1);
    for (int s = 0; s < ST; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, 1);
    }
    for (int x = 0; x < TILES; ++x) {
      mbar_init(bar_s + 8 * x, 1);
      mbar_init(bar_se + 8 * x, 4);
      mbar_init(bar_p + 8 * x, 4);
      mbar_init(bar_o + 8 * x, 2);   // the product, and the issuer's word on `unclean`
    }
    *abort_flag = 0;
    *unclean = 0;
    fence_barrier_init();
  }
  if (warp == 4 * TILES + 1) {
    tmem_alloc(smem_u32(tmem_slot), Cfg::COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp < 4 * TILES) {
    if constexpr (Cfg::MOVE) asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const int x = warp >> 2;                      // tile of rows
    const int row = (warp & 3) * 32 + lane;
    const int in_tile = row / p.group, head = row - in_tile * p.group, query = x * per + in_tile;
    const bool mine = in_tile < per && query < t.queries;   // rows past the last query (and past per * group) hold anything
    const int lim = mine ? seen(p, t, query) : lim_hi;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + lanes + Cfg::S_COL + x * Cfg::STEP, t_p = tmem + lanes + Cfg::P_COL + x * Cfg::STEP;
    const uint32_t t_o = tmem + lanes + Cfg::O_COL + x * Cfg::STEP;
    const float c = p.scale_log2e;
    float m = -INFINITY, l = 0.f;   // reference maximum of the unscaled scores; sum of the weights
    const int begin = first_turn(x);
    // a tile's maximum: moves the reference maximum if it has to, and with it the sum and O
    auto raise = [&](float top, int turn) {
      if (turn == 0) {
        m = top;
        return;
      }
      const bool up = (top - m) * c > 8.f;
      if (!__any_sync(0xffffffffu, up)) return;
      const float f = up ? ex2((m - top) * c) : 1.f;
      if (up) m = top;
      l *= f;
#pragma unroll
      for (int d = 0; d < DP; d += 16) {
        uint32_t o[16];
        tmem_ld_x16(t_o + d, o);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
        tmem_st_x16(t_o + d, o);
      }
    };
    bool ok = true;
    for (int it = begin; it < n; ++it) {
      const int base = (n - 1 - it) * KEYS, turn = it - begin;
      if (!(ok = warp_wait(bar_s + 8 * x, turn & 1, abort_flag))) break;
      tc_fence_after();
      const int have = lim - base;   // keys of this tile that the row sees
      const bool masked = base + KEYS > lim_lo;
      const float2 c2 = make_float2(c, c);
      bool careful = masked || turn == 0;
      if constexpr (Cfg::HOLD) {
        uint32_t r[KEYS];
        float *s = reinterpret_cast<float *>(r);
#pragma unroll
        for (int i = 0; i < KEYS; i += 32) tmem_ld_x32(t_s + i, r + i);
        tmem_ld_wait();
        if (Cfg::EARLY) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar_se + 8 * x);
          if (turn > 0) {   // the previous product has left P and O
            const int i = 2 * it - 1;
            if (!(ok = warp_wait(bar_empty + 8 * (i % ST), (i / ST) & 1, abort_flag))) break;
            tc_fence_after();
          }
        }
        // 32 scores -> 16 columns of P.  MIX: the pairs of each 16 whose exponentials are a polynomial (see exp2_pair).
        auto weigh = [&](int at, float2 off2, float2 &sum, auto mix) {
          constexpr uint32_t MIX = decltype(mix)::value;
          uint32_t w[16];
          float2 other = make_float2(0.f, 0.f);
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float2 e = __ffma2_rn(make_float2(s[at + 2 * i], s[at + 2 * i + 1]), c2, off2);
            if ((MIX >> i) & 1) {
              e = exp2_pair(e);
            } else {
              e.x = ex2(e.x);
              e.y = ex2(e.y);
            }
            if (i & 1) other = __fadd2_rn(other, e);
            else sum = __fadd2_rn(sum, e);
            const __nv_bfloat162 h = __floats2bfloat162_rn(e.x, e.y);
            w[i] = *reinterpret_cast<const uint32_t *>(&h);
          }
          sum = __fadd2_rn(sum, other);
          tmem_st_x16(t_p + at / 2, w);
        };
        if (!careful) {
          // The weights by the reference maximum that is there, without waiting for this tile's own; that one is found beside
          // them and, if it is more than 2^8 above (or a score is NaN or +inf), the tile is done over.
          const float off = -m * c;
          float2 sum = make_float2(0.f, 0.f);
          float x0 = s[0], x1 = s[1];
#pragma unroll
          for (int i = 0; i < KEYS; i += 32) {
            weigh(i, make_float2(off, off), sum, std::integral_constant<uint32_t, POLY>());
#pragma unroll
            for (int k = i; k < i + 32; k += 4) {
              x0 = max3_nan(x0, s[k], s[k + 1]);
              x1 = max3_nan(x1, s[k + 2], s[k + 3]);
            }
          }
          const float top = max3_nan(x0, x1, x1);
          careful = __any_sync(0xffffffffu, mine && !((top - m) * c <= 8.f));
          if (!careful) l += sum.x + sum.y;
        }
        if (careful) {
          tmem_st_wait();   // what the first attempt wrote is written again
          if (masked)
#pragma unroll
            for (int i = 0; i < KEYS; ++i) s[i] = i < have ? s[i] : -INFINITY;
          float x0 = s[0], x1 = s[1];
#pragma unroll
          for (int i = 2; i < KEYS; i += 2) {
            x0 = fmaxf(x0, s[i]);
            x1 = fmaxf(x1, s[i + 1]);
          }
          raise(fmaxf(x0, x1), turn);
          const float off = m == -INFINITY ? 0.f : -m * c;
          float2 sum = make_float2(0.f, 0.f);
#pragma unroll
          for (int i = 0; i < KEYS; i += 32) weigh(i, make_float2(off, off), sum, std::integral_constant<uint32_t, 0>());
          l += sum.x + sum.y;
        }
      } else {
        // twice from tensor memory, 32 columns at a time: once for the maximum, once for the weights
        uint32_t r[32], other[32];
        float top = -INFINITY;
        auto take = [&](uint32_t *w, int at) {
          float *s = reinterpret_cast<float *>(w);
          if (masked)
#pragma unroll
            for (int i = 0; i < 32; ++i) s[i] = at + i < have ? s[i] : -INFINITY;
          float x0 = s[0], x1 = s[1];
#pragma unroll
          for (int i = 2; i < 32; i += 2) {
            x0 = fmaxf(x0, s[i]);
            x1 = fmaxf(x1, s[i + 1]);
          }
          top = fmaxf(top, fmaxf(x0, x1));
        };
#pragma unroll
        for (int i = 0; i < KEYS; i += 64) {
          if (i == 0) tmem_ld_x32(t_s, r);
          tmem_ld_wait();
          tmem_ld_x32(t_s + i + 32, other);
          take(r, i);
          tmem_ld_wait();
          if (i + 64 < KEYS) tmem_ld_x32(t_s + i + 64, r);
          take(other, i + 32);
        }
        if (Cfg::EARLY && turn > 0) {
          const int i = 2 * it - 1;
          if (!(ok = warp_wait(bar_empty + 8 * (i % ST), (i / ST) & 1, abort_flag))) break;
          tc_fence_after();
        }
        raise(top, turn);
        tmem_ld_x32(t_s, r);
        const float off = m == -INFINITY ? 0.f : -m * c;
        const float2 off2 = make_float2(off, off);
        float2 sum0 = make_float2(0.f, 0.f), sum1 = make_float2(0.f, 0.f);
        auto weigh = [&](const uint32_t *from, int at) {
          const float *s = reinterpret_cast<const float *>(from);
          uint32_t w[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float2 e = make_float2(s[2 * i], s[2 * i + 1]);
            if (masked) {
              e.x = at + 2 * i < have ? e.x : -INFINITY;
              e.y = at + 2 * i + 1 < have ? e.y : -INFINITY;
            }
            e = __ffma2_rn(e, c2, off2);
            e.x = ex2(e.x);
            e.y = ex2(e.y);
            if (i & 1) sum1 = __fadd2_rn(sum1, e);
            else sum0 = __fadd2_rn(sum0, e);
            const __nv_bfloat162 h = __floats2bfloat162_rn(e.x, e.y);
            w[i] = *reinterpret_cast<const uint32_t *>(&h);
          }
          tmem_st_x16(t_p + at / 2, w);
        };
#pragma unroll
        for (int i = 0; i < KEYS; i += 64) {
          tmem_ld_wait();
          tmem_ld_x32(t_s + i + 32, other);
          weigh(r, i);
          tmem_ld_wait();
          if (i + 64 < KEYS) tmem_ld_x32(t_s + i + 64, r);
          weigh(other, i + 32);
        }
        l += (sum0.x + sum0.y) + (sum1.x + sum1.y);
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (Cfg::EARLY && !Cfg::HOLD) mbar_arrive(bar_se + 8 * x);
        mbar_arrive(bar_p + 8 * x);
      }
    }
    if (ok && begin < n) ok = warp_wait(bar_o + 8 * x, 0, abort_flag);
    if (!ok) {
      *abort_flag = 1;
      report(p.status, DEV_WAIT_TMEM_FULL);
    } else if (x * per < t.queries) {
      tc_fence_after();
      const long long q_row = (long long)t.q0 + query;
      if (n > 0 && *unclean) {
        if (mine) plain_row(p, q_row, kh * p.group + head, t.k0, lim);
      } else {
        // through shared memory (the queries are read), so that a row leaves in whole lines
        const float inv = 1.f / l;
        const bool none = begin == n || lim <= 0;
        constexpr int PIECES = DP / 8;
        uint8_t *out = gen + x * Cfg::PANELS * 16384 + (warp & 3) * 32 * (DP * 2);
#pragma unroll
        for (int d = 0; d < DP; d += 32) {
          uint32_t o[32];
          if (begin < n) {
            tmem_ld_x32(t_o + d, o);
            tmem_ld_wait();
          }
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const __nv_bfloat162 h = none ? __floats2bfloat162_rn(0.f, 0.f)
                                            : __floats2bfloat162_rn(__uint_as_float(o[i + 2 * k]) * inv, __uint_as_float(o[i + 2 * k + 1]) * inv);
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
          const int rr = i / PIECES, piece = i % PIECES, at = (warp & 3) * 32 + rr;
          const int qi = at / p.group, hi = at - qi * p.group, qq = x * per + qi;
          if (qi < per && qq < t.queries && piece * 8 < p.dim)
            *reinterpret_cast<uint4 *>(y + qq * p.ldy + hi * p.dim + piece * 8) = *reinterpret_cast<const uint4 *>(out + rr * (DP * 2) + ((piece ^ (rr & 7)) << 4));
        }
      }
    }
  } else {
    if constexpr (Cfg::MOVE) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");   // the whole group of warps, the idle ones too
    if (warp == 4 * TILES) {
      if (lane == 0 && n > 0) {
        bool ok = true;
        const int tiles = first_turn(TILES - 1) < n ? TILES : 1;
        mbar_arrive_expect_tx(bar_q, tiles * Cfg::PANELS * 128 * p.group * per);
        for (int x = 0; x < tiles; ++x)
          for (int c = 0; c < Cfg::PANELS; ++c)
            tma_load_3d(sm_q + (x * Cfg::PANELS + c) * 16384, &tm_q, bar_q, 64 * c, kh * p.group, t.q0 + x * per);
        for (int i = 0; i < 2 * n; ++i) {   // K and V in turn
          const uint32_t st = i % ST, ph = (i / ST) & 1;
          const int row = t.k0 + (n - 1 - (i >> 1)) * KEYS;
          if (!(ok = mbar_wait_relaxed(bar_empty + 8 * st, ph ^ 1u, abort_flag))) break;
          mbar_arrive_expect_tx(bar_full + 8 * st, Cfg::TILE);
          for (int c = 0; c < Cfg::PANELS; ++c)
            tma_load_3d(sm_ring + st * Cfg::TILE + c * Cfg::PANEL, i & 1 ? &tm_v : &tm_k, bar_full + 8 * st, 64 * c, kh, row);
        }
        if (!ok) {
          *abort_flag = 1;
          report(p.status, DEV_WAIT_SMEM_EMPTY);
          const uint64_t t0 = globaltimer();   // copies in flight land before the block ends
          while (globaltimer() - t0 < 200000ull) {}
        }
      }
    } else if (warp == 4 * TILES + 1) {
      // descriptors: 128-byte swizzle, 1024 bytes between groups of 8 rows, version 1
      const uint64_t desc_hi = (uint64_t)((1024u >> 4) | (1u << 14) | (2u << 29)) << 32;
      const uint32_t kmajor = 1u << 16, mnmajor = ((uint32_t)Cfg::PANEL >> 4) << 16;   // MN-major: leading offset = one panel
      const uint32_t idesc_s = (1u << 4) | (1u << 7) | (1u << 10) | (((uint32_t)KEYS >> 3) << 17) | ((128u >> 4) << 24);
      const uint32_t idesc_o = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | (((uint32_t)DP >> 3) << 17) | ((128u >> 4) << 24);
      const uint32_t leader = lane == 0;
      const uint32_t q_lo = kmajor | uniform(sm_q >> 4), ring = uniform(sm_ring >> 4), tm = uniform(tmem);   // below 2^14: no carry into the next field
      const int turns = (int)uniform((uint32_t)n), visible = (int)uniform((uint32_t)lim_lo);
      int begin[TILES];
#pragma unroll
      for (int x = 0; x < TILES; ++x) begin[x] = (int)uniform((uint32_t)first_turn(x));
      bool ok = true;
      auto scores = [&](int x, int it) -> bool {
        const uint32_t st = (uint32_t)(2 * it) % ST, ph = ((uint32_t)(2 * it) / ST) & 1;
        if (it >= begin[x]) {
          if (!warp_wait(bar_full + 8 * st, ph, abort_flag)) return false;
          tc_fence_after();
          const uint32_t k_lo = kmajor | (ring + st * (Cfg::TILE >> 4));
#pragma unroll
          for (int kk = 0; kk < DP / 16; ++kk)
            umma_ss(leader, tm + Cfg::S_COL + x * Cfg::STEP, desc_hi | (q_lo + (x * Cfg::PANELS + (kk >> 2)) * 1024 + (kk & 3) * 2),
                    desc_hi | (k_lo + (kk >> 2) * (Cfg::PANEL >> 4) + (kk & 3) * 2), idesc_s, kk != 0);
          commit_if(leader, bar_s + 8 * x);
        }
        if (x == TILES - 1) commit_if(leader, bar_empty + 8 * st);   // both tiles' products with these keys are on their way
        return true;
      };
      if (turns > 0) ok = warp_wait(bar_q, 0, abort_flag);
#pragma unroll
      for (int x = 0; x < TILES; ++x)
        if (turns > 0 && ok) ok = scores(x, 0);
      for (int it = 0; it < turns && ok; ++it) {
        const int base = (turns - 1 - it) * KEYS;
        const uint32_t st = (uint32_t)(2 * it + 1) % ST, ph = ((uint32_t)(2 * it + 1) / ST) & 1;
        if (Cfg::EARLY && it + 1 < turns && !(ok = warp_wait(bar_se, it & 1, abort_flag) && scores(0, it + 1))) break;
        if (!(ok = warp_wait(bar_full + 8 * st, ph, abort_flag))) break;
        if (base + KEYS > visible) {
          // Values past the last key that anybody here sees belong to others and may hold anything: zeros in their place, since
          // the tensor cores multiply every value by every row's weight and 0 * NaN is NaN.  Values on the diagonal are hidden
          // from some rows only: if one is not finite, the rows are summed up the plain way at the end.
          uint8_t *v = gen + Cfg::Q + st * Cfg::TILE;
          constexpr int PIECES = 8 * Cfg::PANELS;   // 16-byte pieces of a key's values
          const int none = max(0, min(KEYS, lim_hi - base)), some = max(0, min(none, lim_lo - base));
          for (int i = none * PIECES + lane; i < KEYS * PIECES; i += 32) {
            const int key = i / PIECES, piece = i % PIECES;
            *reinterpret_cast<uint4 *>(v + (piece >> 3) * Cfg::PANEL + key * 128 + (piece & 7) * 16) = make_uint4(0, 0, 0, 0);
          }
          bool bad = false;
          for (int i = some * PIECES + lane; i < none * PIECES; i += 32) {
            const int key = i / PIECES, piece = i % PIECES;
            const uint4 w = *reinterpret_cast<const uint4 *>(v + (piece >> 3) * Cfg::PANEL + key * 128 + (piece & 7) * 16);
            for (uint32_t u : {w.x, w.y, w.z, w.w}) bad |= (u & 0x7f80u) == 0x7f80u || (u & 0x7f800000u) == 0x7f800000u;
          }
          if (bad) *unclean = 1;
          fence_proxy_async();
          __syncwarp();
        }
        const uint32_t v_lo = mnmajor | (ring + st * (Cfg::TILE >> 4));
#pragma unroll
        for (int x = 0; x < TILES; ++x) {
          if (it >= begin[x]) {
            if (!(ok = warp_wait(bar_p + 8 * x, (it - begin[x]) & 1, abort_flag))) break;
            tc_fence_after();
            const uint32_t more = it != begin[x];
#pragma unroll
            for (int kk = 0; kk < KEYS / 16; ++kk)   // 16 keys: 8 columns of P, 16 rows of V
              umma_ts(leader, tm + Cfg::O_COL + x * Cfg::STEP, tm + Cfg::P_COL + x * Cfg::STEP + 8 * kk, desc_hi | (v_lo + 128 * kk), idesc_o,
                      kk != 0 ? 1u : more);
          }
          if (x == TILES - 1) commit_if(leader, bar_empty + 8 * st);
          if (it + 1 == turns && begin[x] < turns) {
            commit_if(leader, bar_o + 8 * x);
            if (lane == 0) mbar_arrive(bar_o + 8 * x);
          }
          // Without columns of their own the weights lie where the next scores go.  Both products are this thread's, and the
          // tensor cores take them in order.
          if (!Cfg::EARLY && it + 1 < turns && !(ok = scores(x, it + 1))) break;
        }
      }
      if (!ok && lane == 0) {
        *abort_flag = 1;
        report(p.status, DEV_WAIT_SMEM_FULL);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 4 * TILES + 1) {
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
static int launch_umma(sofie_b200_ctx *ctx, PromptParams p) {
  using Cfg = UmmaSize<DP>;
  const int per = 128 / p.group;
  p.tokens = Cfg::TILES * per;
  const long long grid = (p.q_rows / p.tokens + p.batch) * p.kv_heads;   // every sequence may end inside a tile
  if (grid > 0x7fffffffLL) return fail(SOFIE_B200_ERR_TOO_LARGE, "prompt_attention_enqueue: %lld queries of %d heads", p.q_rows, p.heads);
  CUtensorMap tm_q, tm_k, tm_v;
  const void *k = p.k_rows ? p.k : p.q, *v = p.k_rows ? p.v : p.q;   // no keys: nothing is loaded, but a map has to describe something
  const long long k_rows = p.k_rows ? p.k_rows : 1;
  int rc;
  if ((rc = encode_rows(&tm_q, p.q, p.dim, p.heads, p.q_rows, p.ldq, p.group, per))) return rc;
  if ((rc = encode_rows(&tm_k, k, p.dim, p.kv_heads, k_rows, p.ldk, 1, Cfg::KEYS))) return rc;
  if ((rc = encode_rows(&tm_v, v, p.dim, p.kv_heads, k_rows, p.ldv, 1, Cfg::KEYS))) return rc;
  SB_CUDA(cudaFuncSetAttribute(prompt_umma_kernel<DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM));   // per device
  prompt_umma_kernel<DP><<<(unsigned)grid, Cfg::THREADS, Cfg::SMEM, ctx->stream>>>(tm_q, tm_k, tm_v, p);
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
    if (d.head_dim <= 64) return launch_umma<64>(ctx, p);
    if (d.head_dim <= 128) return launch_umma<128>(ctx, p);
    return launch_umma<256>(ctx, p);
  }
  const int64_t blocks = (q_tokens * d.heads + 3) / 4;
  if (blocks > 0x7fffffffLL) return fail(SOFIE_B200_ERR_TOO_LARGE, "prompt_attention_enqueue: %lld queries of %d heads", (long long)q_tokens, d.heads);
  prompt_rows_kernel<float><<<(unsigned)blocks, 128, 0, ctx->stream>>>(p);
  SB_CUDA(cudaGetLastError());
  ctx->launches++;
  return 0;
}

}  // extern "C"
