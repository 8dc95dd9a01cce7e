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
  int most_keys;              // of a sequence
  float scale_log2e;
  int *status;
};

// Keys of a sequence at most.  bf16: the tensor cores cut what they add to a sum below its last bits, so that values of one sign under
// equal weights lose n 2^-28 of it over n keys (measured 0.0039 at 2^20, half a step of the result's type; 0.023 at 2^22; half of
// it at 2^27); and no wait may be as long as its limit of a second, though the warps of a tile of rows without a turn wait for all turns of
// the block's other one: 1.71 us for 128 keys, 14 ms for 2^20 (and 1.79 s for 2^27).  fp32: sums in order, in which equal values count
// exactly up to 2^24 (measured 1e-5 there, values of one sign).
constexpr int MOST_KEYS_BF16 = 1 << 20, MOST_KEYS_F32 = 1 << 24;
// Blocks of the bf16 kernel at most.  One without a tile takes 2.1 ns of the whole GPU's time, and the other warps wait for all of them: 0.28 s.
constexpr long long MOST_BLOCKS = 1LL << 27;

// One tile of queries: its sequence's rows, its first query and how many of them there are.
struct PromptTile {
  int q0, k0, k_len;      // first query row of the tile and first key row of the sequence in the packed tensors; keys of the sequence
  int queries;            // 0: no such tile; -1 (in a block's mail): no more tiles
  int past;               // keys that the tile's first query sees, before clamping to [0, k_len] (causal)
  int kh;                 // key head
};

// Sequence b: tiles of `tokens` queries; fills in the parts of t that are the sequence's.
__device__ __forceinline__ int sequence_tiles(const PromptParams &p, int b, PromptTile &t, int &q_len) {
  int x0, x1, y0, y1;
  bool bad = false;
  packed_range(p.cu_q, b, p.q_rows, &x0, &x1, &bad);
  packed_range(p.cu_k, b, p.k_rows, &y0, &y1, &bad);
  bad |= x1 > x0 && y1 - y0 > p.most_keys;
  if (bad) report(p.status, DEV_BAD_INDEX);
  t.q0 = x0; t.k0 = y0; t.k_len = y1 - y0;
  q_len = bad ? 0 : x1 - x0;
  return (q_len + p.tokens - 1) / p.tokens;
}

// Tiles are counted sequence by sequence; within a sequence the last one, which sees most keys, comes first.  The table of a block
// has the tiles before each of RUNS equal runs of sequences.  All threads call this, at least RUNS of them.
constexpr int RUNS = 128;
__device__ __forceinline__ void count_tiles(const PromptParams &p, int *table) {   // [RUNS + 1]
  __shared__ long long warp_sum[RUNS / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (p.batch + RUNS - 1) / RUNS;
  const int b0 = tid < RUNS ? min(p.batch, tid * per) : p.batch, b1 = min(p.batch, b0 + per);
  PromptTile t;
  int q_len;
  long long mine = 0;   // offsets that claim rows twice can make more tiles than the grid has; the rest is left out
  for (int b = b0; b < b1; ++b) mine += sequence_tiles(p, b, t, q_len);
  long long incl = mine;
  for (int o = 1; o < 32; o <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += x;
  }
  if (lane == 31 && tid < RUNS) warp_sum[warp] = incl;
  __syncthreads();
  if (tid < RUNS) {
    for (int w = 0; w < warp; ++w) incl += warp_sum[w];
    if (tid == 0) table[0] = 0;
    table[tid + 1] = (int)min(incl, 0x7fffffffLL);
  }
  __syncthreads();
}

// Tile `index` for all lanes of a warp; queries = 0 when there is none.
__device__ __forceinline__ PromptTile find_tile(const PromptParams &p, const int *table, int index) {
  const int lane = threadIdx.x & 31;
  PromptTile t{};
  if (index >= table[RUNS]) return t;
  int run = 0;   // runs that end at or before the index
#pragma unroll
  for (int i = 0; i < RUNS; i += 32) run += __popc(__ballot_sync(0xffffffffu, table[i + lane + 1] <= index));
  const int per = (p.batch + RUNS - 1) / RUNS;
  const int b1 = min(p.batch, (run + 1) * per);
  int at = table[run];
  for (int b = run * per; b < b1; b += 32) {
    int q_len = 0;
    const int n = b + lane < b1 ? sequence_tiles(p, b + lane, t, q_len) : 0;
    int incl = n;
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += x;
    }
    const bool here = index >= at + incl - n && index < at + incl;
    const uint32_t who = __ballot_sync(0xffffffffu, here);
    if (who) {
      const int first = (n - 1 - (index - (at + incl - n))) * p.tokens;
      t.past = first + 1 + t.k_len - q_len;
      t.q0 += first;
      t.queries = min(p.tokens, q_len - first);
      const int src = __ffs(who) - 1;
      t.q0 = __shfl_sync(0xffffffffu, t.q0, src);
      t.k0 = __shfl_sync(0xffffffffu, t.k0, src);
      t.k_len = __shfl_sync(0xffffffffu, t.k_len, src);
      t.queries = __shfl_sync(0xffffffffu, t.queries, src);
      t.past = __shfl_sync(0xffffffffu, t.past, src);
      return t;
    }
    at += __shfl_sync(0xffffffffu, incl, 31);
  }
  return PromptTile{};
}

// Keys that query i of the tile sees.
__device__ __forceinline__ int seen(const PromptParams &p, const PromptTile &t, int i) {
  return p.causal ? min(t.k_len, max(0, t.past + i)) : t.k_len;
}

// ---- fp32 on the CUDA cores --------------------------------------------------------------------------------------------------------
// A block computes 32 rows; each of its teams of four warps takes every TEAMS-th tile of 64 keys, and the teams' sums are joined at the end
// (where blocks are few, those of a cluster of them too, through distributed shared memory).
// (Few blocks are long chains of tiles on few warps otherwise: 770 queries of 8 heads over 1770 keys take 80 us with one team, 71 with
// two, 61 with two blocks of two; prompts of 2048 tokens 31 TFLOP/s, 0.42 of the FMA pipes, with any.  Above head size 128 a second
// team's tiles do not fit.)
// A thread has 4 rows x 4 keys of the scores and 4 rows x DP / 16 dimensions of the result, so that a 16-byte read from shared memory
// feeds 16 FMAs and the FMA pipes are what bounds it.  The next keys arrive while this tile's values are weighed, the next values while
// the next scores are computed (cp.async, one place each).
constexpr int PF_ROWS = 32, PF_KEYS = 64, PF_TEAM = 128;
template <int DP>
struct FmaCfg {
  static constexpr int TEAMS = DP <= 128 ? 2 : 1, THREADS = TEAMS * PF_TEAM, BLOCKS = DP == 64 ? 2 : 1;   // BLOCKS: that fit an SM
  static constexpr int Q = PF_ROWS * DP * 4, TILE = PF_KEYS * DP * 4, P = PF_KEYS * PF_ROWS * 4;
  static constexpr int SMEM = Q + TEAMS * (2 * TILE + P) + 4 * (RUNS + 1);
};

template <int DP>
__global__ void __launch_bounds__(FmaCfg<DP>::THREADS) prompt_fma_kernel(const __grid_constant__ PromptParams p, int parts, int share) {
  using Cfg = FmaCfg<DP>;
  constexpr int CH = DP / 4, PIECES = DP / 64;   // 16-byte pieces of a row; of the result per thread and row
  extern __shared__ __align__(128) uint8_t smem[];
  const int team = threadIdx.x / PF_TEAM, tid = threadIdx.x % PF_TEAM, warp = tid >> 5, lane = tid & 31;
  float4 *sq = reinterpret_cast<float4 *>(smem), *sk = sq + (Cfg::Q + team * (2 * Cfg::TILE + Cfg::P)) / 16, *sv = sk + Cfg::TILE / 16, *sp = sv + Cfg::TILE / 16;
  int *table = reinterpret_cast<int *>(smem + Cfg::Q + Cfg::TEAMS * (2 * Cfg::TILE + Cfg::P));
  auto meet = [&]() { asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "n"(PF_TEAM) : "memory"); };   // the team
  count_tiles(p, table);
  const int block = blockIdx.x / share, rank = blockIdx.x % share;
  const int work = block / parts, part = block % parts, kh = work % p.kv_heads;   // a group of more than 32 heads is several parts
  const PromptTile t = find_tile(p, table, work / p.kv_heads);
  if (t.queries == 0) return;
  const int head0 = part * PF_ROWS, heads = min(PF_ROWS, p.group - head0);   // heads of the group in this block
  const int lim_lo = seen(p, t, 0), lim_hi = seen(p, t, t.queries - 1);
  const int n = (lim_hi + PF_KEYS - 1) / PF_KEYS;
  const float *q = static_cast<const float *>(p.q) + t.q0 * p.ldq + (long long)(kh * p.group + head0) * p.dim;
  const float *k = static_cast<const float *>(p.k) + t.k0 * p.ldk + (long long)kh * p.dim;
  const float *v = static_cast<const float *>(p.v) + t.k0 * p.ldv + (long long)kh * p.dim;
  const uint32_t a_q = smem_u32(sq), a_k = smem_u32(sk), a_v = smem_u32(sv);

  auto load_tile = [&](uint32_t dst, const float *src, long long pitch, int base, bool swizzle) {
#pragma unroll 4
    for (int i = tid; i < PF_KEYS * CH; i += PF_TEAM) {
      const int r = i / CH, c = i % CH;
      const bool there = base + r < lim_hi && c * 4 < p.dim;
      cp_async_16(dst + (r * CH + (swizzle ? c ^ (r & 7) : c)) * 16, src + (there ? (base + r) * pitch + c * 4 : 0), there);
    }
  };
  const int stride = Cfg::TEAMS * share, begin = n - 1 - (rank * Cfg::TEAMS + team);   // this team's tiles: begin, begin - stride, ...
  for (int i = threadIdx.x; i < PF_ROWS * CH; i += Cfg::THREADS) {
    const int r = i / CH, c = i % CH, query = r / heads, h = r - query * heads;
    const bool there = query < t.queries && c * 4 < p.dim;
    cp_async_16(a_q + i * 16, q + (there ? query * p.ldq + (long long)h * p.dim + c * 4 : 0), there);
  }
  cp_async_commit();
  if (begin >= 0) load_tile(a_k, k, p.ldk, begin * PF_KEYS, true);
  cp_async_commit();
  if (begin >= 0) load_tile(a_v, v, p.ldv, begin * PF_KEYS, false);
  cp_async_commit();
  cp_async_wait<2>();
  __syncthreads();   // the queries, which both teams brought

  const int rg = warp * 2 + (lane >> 4), g = lane & 15;   // rows 4 rg .. 4 rg + 3; keys g + 16 j; pieces g + 16 j of the result
  int lim[4];
  float m[4], l[4];
  float4 acc[4][PIECES];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int query = (4 * rg + r) / heads;
    lim[r] = query < t.queries ? seen(p, t, query) : 0;
    m[r] = -INFINITY;   // in units of log2; -inf: no key yet
    l[r] = 0.f;         // this thread's keys only
#pragma unroll
    for (int j = 0; j < PIECES; ++j) acc[r][j] = make_float4(0.f, 0.f, 0.f, 0.f);
  }

  for (int it = begin; it >= 0; it -= stride) {
    const int base = it * PF_KEYS;
    const bool masked = base + PF_KEYS > lim_lo;
    cp_async_wait<1>();   // the keys
    meet();
    float s[4][4] = {};
#pragma unroll 2
    for (int c = 0; c < CH; ++c) {
      float4 a[4], b[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) a[r] = sq[(4 * rg + r) * CH + c];
#pragma unroll
      for (int j = 0; j < 4; ++j) b[j] = sk[(g + 16 * j) * CH + (c ^ (g & 7))];
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[r][j] = fmaf(a[r].x, b[j].x, fmaf(a[r].y, b[j].y, fmaf(a[r].z, b[j].z, fmaf(a[r].w, b[j].w, s[r][j]))));
    }
    meet();   // the keys are read
    if (it >= stride) load_tile(a_k, k, p.ldk, base - stride * PF_KEYS, true);
    cp_async_commit();
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      float top = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[r][j] = base + g + 16 * j < lim[r] ? s[r][j] * p.scale_log2e : -INFINITY;
        top = fmaxf(top, s[r][j]);
      }
#pragma unroll
      for (int o = 1; o < 16; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      if (base < lim[r]) top = fmaxf(top, -3.0e38f);   // a key is there: the maximum is a number
      if (top > m[r]) {
        const float f = ex2(m[r] - top);
        m[r] = top;
        l[r] *= f;
#pragma unroll
        for (int j = 0; j < PIECES; ++j) { acc[r][j].x *= f; acc[r][j].y *= f; acc[r][j].z *= f; acc[r][j].w *= f; }
      }
      const float off = m[r] == -INFINITY ? 0.f : m[r];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[r][j] = ex2(s[r][j] - off);
        l[r] += s[r][j];
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int key = g + 16 * j;
      sp[key * (PF_ROWS / 4) + (rg ^ (key & 7))] = make_float4(s[0][j], s[1][j], s[2][j], s[3][j]);
    }
    cp_async_wait<1>();   // the values
    meet();
    if (!masked) {
#pragma unroll 4
      for (int key = 0; key < PF_KEYS; ++key) {
        const float4 w = sp[key * (PF_ROWS / 4) + (rg ^ (key & 7))];
#pragma unroll
        for (int j = 0; j < PIECES; ++j) {
          const float4 x = sv[key * CH + g + 16 * j];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float e = r == 0 ? w.x : r == 1 ? w.y : r == 2 ? w.z : w.w;
            acc[r][j].x = fmaf(e, x.x, acc[r][j].x);
            acc[r][j].y = fmaf(e, x.y, acc[r][j].y);
            acc[r][j].z = fmaf(e, x.z, acc[r][j].z);
            acc[r][j].w = fmaf(e, x.w, acc[r][j].w);
          }
        }
      }
    } else {   // a hidden value may be NaN or infinite: it is left out, not multiplied by 0
      for (int key = 0; key < PF_KEYS; ++key) {
        const float4 w = sp[key * (PF_ROWS / 4) + (rg ^ (key & 7))];
#pragma unroll
        for (int j = 0; j < PIECES; ++j) {
          const float4 x = sv[key * CH + g + 16 * j];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float e = r == 0 ? w.x : r == 1 ? w.y : r == 2 ? w.z : w.w;
            if (base + key < lim[r]) {
              acc[r][j].x = fmaf(e, x.x, acc[r][j].x);
              acc[r][j].y = fmaf(e, x.y, acc[r][j].y);
              acc[r][j].z = fmaf(e, x.z, acc[r][j].z);
              acc[r][j].w = fmaf(e, x.w, acc[r][j].w);
            }
          }
        }
      }
    }
    meet();   // values and weights are read
    if (it >= stride) load_tile(a_v, v, p.ldv, base - stride * PF_KEYS, false);
    cp_async_commit();
  }
  cp_async_wait<0>();
  // Sums meet thread by thread: a thread's rows and dimensions are the same in every team and block.  They lie where the last team's
  // keys were, which are read.
  constexpr int PLACE = Cfg::Q + (Cfg::TEAMS - 1) * (2 * Cfg::TILE + Cfg::P);
  float4 *sum = reinterpret_cast<float4 *>(smem + PLACE) + tid;
  auto leave = [&]() {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      sum[r * (PIECES + 1) * PF_TEAM] = make_float4(m[r], l[r], 0.f, 0.f);
#pragma unroll
      for (int j = 0; j < PIECES; ++j) sum[(r * (PIECES + 1) + 1 + j) * PF_TEAM] = acc[r][j];
    }
  };
  auto join = [&](auto fetch) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float4 ml = fetch(r * (PIECES + 1) * PF_TEAM);
      const float top = fmaxf(m[r], ml.x), off = top == -INFINITY ? 0.f : top, f = ex2(m[r] - off), g2 = ex2(ml.x - off);
      m[r] = top;
      l[r] = l[r] * f + ml.y * g2;
#pragma unroll
      for (int j = 0; j < PIECES; ++j) {
        const float4 x = fetch((r * (PIECES + 1) + 1 + j) * PF_TEAM);
        acc[r][j] = make_float4(acc[r][j].x * f + x.x * g2, acc[r][j].y * f + x.y * g2, acc[r][j].z * f + x.z * g2, acc[r][j].w * f + x.w * g2);
      }
    }
  };
  if constexpr (Cfg::TEAMS == 2) {
    if (team == 1) {
      meet();
      leave();
    }
    __syncthreads();
    if (team == 1) return;
    join([&](int i) { return sum[i]; });
  }
  if (share > 1) {   // the cluster's blocks: the first one takes the others' sums, in order
    meet();          // with one team: its keys are read; with two: so are the second one's sums, by their own threads
    if (rank > 0) leave();
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (rank == 0) {
      for (int other = 1; other < share; ++other) {
        uint32_t at;
        asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(sum)), "r"(other));
        join([&](int i) {
          float4 x;
          asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w) : "r"(at + i * 16) : "memory");
          return x;
        });
      }
    }
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");   // and they stay until it has
    if (rank > 0) return;
  }

#pragma unroll
  for (int r = 0; r < 4; ++r) {
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], o);
    const int at = 4 * rg + r, query = at / heads, h = at - query * heads;
    if (query >= t.queries) continue;
    const float inv = m[r] == -INFINITY ? 0.f : 1.f / l[r];
    float *y = static_cast<float *>(p.y) + (t.q0 + query) * p.ldy + (long long)(kh * p.group + head0 + h) * p.dim;
#pragma unroll
    for (int j = 0; j < PIECES; ++j) {
      const int d = (g + 16 * j) * 4;
      if (d < p.dim) *reinterpret_cast<float4 *>(y + d) = make_float4(acc[r][j].x * inv, acc[r][j].y * inv, acc[r][j].z * inv, acc[r][j].w * inv);
    }
  }
}

// A wait of a whole warp.  The lanes leave together: one that lagged behind could find the barrier a phase further on, with the parity
// that means "not yet", and wait for good; and all of them agree on a wait that ran out.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int *abort_flag) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag));
}

// The same for waits that are usually long: sleeps between polls.
__device__ __forceinline__ bool warp_wait_long(uint32_t bar, uint32_t parity, volatile int *abort_flag) {
  return __all_sync(0xffffffffu, mbar_wait_relaxed(bar, parity, abort_flag));
}

// ---- bf16 on the tensor cores --------------------------------------------------------------------------------------------------
// max(a, b, c), NaN if one of them is
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float y;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
constexpr float MARGIN = 16.f;   // see prompt_umma_kernel
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
// The loads have arrived; nothing that uses their registers moves above this.
template <int N>
__device__ __forceinline__ void tmem_loaded(uint32_t (&r)[N]) {
  tmem_ld_wait();
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+r"(r[i]));
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// A block works on TILES tiles of 128 rows against the same keys and values.  What sets the sizes:
//  - The way from L2: a tile of keys and values takes about 3000 cycles from request to arrival and an SM sustains about 48 bytes per
//    cycle, while the tensor cores would finish 128 rows x 128 keys of head size 128 (64 KB of keys and values) in 1024 cycles (512 for
//    each product, measured alone).  So at that head size two tiles of rows share every load (32 bytes per cycle at full rate) and
//    160 KB are in flight; one tile a block, two blocks an SM, with 64 KB in flight each, took 964 us where this takes 495 (a prompt
//    of 8192 tokens, 32 heads over 8).  At head size 64 half the bytes are needed per score, and two blocks of one tile share an SM.
//  - Tensor memory, 512 columns.  EARLY: the weights have columns of their own, and the scores of the next tile of keys are computed
//    while this one's are weighed.  At head size 128 two results leave room for that with 64 keys a tile only, where the first product
//    is bound by shared memory (533 us), or 80 keys (678 us, too many registers); there the weights lie over the scores, 128 keys a tile.
//  - Exponentials: the special-function unit does 16 a cycle and SM, 1024 cycles for 128 x 128 scores, as long as both products.  Taking
//    1/8 to 1/2 of them on the FMA pipes (a polynomial of degree 4) made every case slower: a warp is alone on its scheduler's special
//    unit most of the time, and it is the length of its own chain that counts.
template <int DP>
struct UmmaCfg;
template <>
struct UmmaCfg<64> {   // 128 keys a tile, scores read twice from tensor memory: 540 us for 32 full sequences of 2048 tokens, this 457
  static constexpr int TILES = 1, KEYS = 64, BLOCKS = 2, STAGES = 9, QS = 2, COLS = 256;
  static constexpr int S_COL = 0, O_COL = 128, P_COL = 64, STEP = 0;
  static constexpr bool EARLY = true;    // the weights have columns of their own: the next scores are computed meanwhile
};
template <>
struct UmmaCfg<128> {
  static constexpr int TILES = 2, KEYS = 128, BLOCKS = 1, STAGES = 5, QS = 1, COLS = 512;
  static constexpr int S_COL = 0, O_COL = 128, P_COL = 0, STEP = 256;
  static constexpr bool EARLY = false;
};
template <>
struct UmmaCfg<256> {
  static constexpr int TILES = 1, KEYS = 64, BLOCKS = 1, STAGES = 5, QS = 1, COLS = 512;
  static constexpr int S_COL = 0, O_COL = 256, P_COL = 64, STEP = 0;
  static constexpr bool EARLY = true;
};
template <int DP>
struct UmmaSize : UmmaCfg<DP> {
  using C = UmmaCfg<DP>;
  static constexpr int PANELS = DP / 64;                    // a panel: rows x 64 elements, 128-byte swizzle
  static constexpr int Q = C::TILES * PANELS * 16384;
  static constexpr int TILE = C::KEYS * DP * 2;             // keys or values
  static constexpr int PANEL = C::KEYS * 128;
  // Warps of rows; then TMA, MMA.  Where a thread holds a row of 128 scores it needs more than 168 registers (12 warps' share): the block
  // is launched with a whole third group of warps, which hands registers over, 384 x 168 = 256 x 200 + 128 x 104.  The compiler still
  // allots 168 and spills a little, 104 bytes of stores and 156 of loads a thread.
  static constexpr bool MOVE = C::TILES == 2;
  static constexpr int THREADS = C::TILES * 128 + (MOVE ? 128 : 64);
  static constexpr int CONTROL = 512 + 64 + 64 + 4 * (RUNS + 1);   // barriers, mail, answers, table of tiles
  static constexpr int SMEM = C::QS * Q + C::STAGES * TILE + (CONTROL + 127) / 128 * 128 + 1024 /*alignment*/;
};

// The next tile of a block whose first one is blockIdx.x: the hardware hands over a block of the grid that has not begun (cluster
// launch control), so tiles go to whoever is free, the heavy ones first, without a counter in memory that two graphs could share.
__device__ __forceinline__ void ask_for_block(uint32_t answer, uint32_t bar) {
  mbar_arrive_expect_tx(bar, 16);
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(answer), "r"(bar) : "memory");
}
__device__ __forceinline__ bool block_given(uint32_t answer, uint32_t &index) {
  uint32_t given, x = 0;
  asm volatile(
      "{\n.reg .pred p;\n.reg .b128 h;\n"
      "ld.shared.b128 h, [%2];\n"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n"
      "selp.u32 %0, 1, 0, p;\n"
      "mov.u32 %1, 0;\n"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%1, _, _, _}, h;\n}\n"
      : "=r"(given), "=r"(x)
      : "r"(answer)
      : "memory");
  index = x;
  return given != 0;
}

// The result of a row += the NaN and infinities among the values of the sequence's keys [j0, j1), which the product went without.
__device__ __noinline__ void add_nonfinite(const PromptParams &p, long long q_row, int head, int k0, int j0, int j1) {
  __nv_bfloat16 *y = static_cast<__nv_bfloat16 *>(p.y) + q_row * p.ldy + (long long)head * p.dim;
  const __nv_bfloat16 *v = static_cast<const __nv_bfloat16 *>(p.v) + k0 * p.ldv + (long long)(head / p.group) * p.dim;
  for (int d = 0; d < p.dim; d += 8) {
    float sum[8] = {};
    for (int j = j0; j < j1; ++j) {
      const uint4 w = *reinterpret_cast<const uint4 *>(v + j * p.ldv + d);
      const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t bits = e & 1 ? u[e / 2] & 0xffff0000u : u[e / 2] << 16;
        if ((bits & 0x7f800000u) == 0x7f800000u) sum[e] += __uint_as_float(bits);
      }
    }
    for (int e = 0; e < 8; ++e)
      if (sum[e] != 0.f) y[d + e] = __float2bfloat16_rn(__bfloat162float(y[d + e]) + sum[e]);
  }
}

// Blocks stay and take tile after tile.  Roles:
//   a warp           finds the tile, leaves it in the mail for the others, asks for the next; lane 0 loads by TMA: the queries once, then
//                    per tile of keys K and V, from the last to the first, into a ring -- of the next tile while this one is computed
//   a warp           MMA: S = Q K^T (operands in shared memory), O += P V (P in tensor memory, V MN-major in shared memory)
//   4 warps a tile   a thread per row: maximum, exponentials, row sum; P as bf16 back to tensor memory
// The reference maximum of a row moves only when a tile's maximum is 2^16 above it (fp32 and bf16 keep their relative precision up
// there, and numerator and denominator use the same); then O is rescaled in tensor memory, which is rare.
// Only tiles that the sequence's end or the diagonal cross pay for masks.  Every wait has a limit.
// Measured: a causal prompt of 8192 tokens, 32 heads over 8 of 128, 558 to 563 us back to back = 0.98 PFLOP/s (494 to 505 us in short bursts),
// tensor pipe 51 % (60 % with its operand traffic), exponentials 51 %: the two rows' chains of maximum, exponential and hand-over
// fill the gaps of one another only in part.  24 packed prompts of 5 to 2500 tokens 133 us; 512 sequences of 24 to 128, head size 64, full,
// 131 MB: 60 us (a tile is two turns, so beginning and ending it is what counts).
template <int DP>
__global__ void __launch_bounds__(UmmaSize<DP>::THREADS, UmmaSize<DP>::BLOCKS)
prompt_umma_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                   const __grid_constant__ PromptParams p) {
  using Cfg = UmmaSize<DP>;
  constexpr int ST = Cfg::STAGES, KEYS = Cfg::KEYS, TILES = Cfg::TILES, QS = Cfg::QS;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw), pad = (1024u - (raw & 1023u)) & 1023u;
  const uint32_t sm_q = raw + pad, sm_ring = sm_q + QS * Cfg::Q;
  uint8_t *gen = smem_raw + pad;
  uint8_t *tail = gen + QS * Cfg::Q + ST * Cfg::TILE;
  const uint32_t bar_mail = smem_u32(tail);          // [2] a tile is in the mail
  const uint32_t bar_read = bar_mail + 16;           // [2] everybody has read it
  const uint32_t bar_next = bar_read + 16;           // [2] the answer about the next tile is there
  const uint32_t bar_q = bar_next + 16;              // [QS] queries landed
  const uint32_t bar_qe = bar_q + 8 * QS;            // [QS] queries read
  const uint32_t bar_full = bar_qe + 8 * QS;         // [ST] ring: keys or values landed
  const uint32_t bar_empty = bar_full + 8 * ST;      // [ST] the products that read them are complete
  const uint32_t bar_s = bar_empty + 8 * ST;         // [TILES] scores complete in tensor memory
  const uint32_t bar_se = bar_s + 8 * TILES;         // [TILES] scores read (EARLY)
  const uint32_t bar_p = bar_se + 8 * TILES;         // [TILES] weights written to tensor memory
  const uint32_t bar_pv = bar_p + 8 * TILES;        // [TILES] product with the values complete (EARLY)
  const uint32_t bar_o = bar_pv + 8 * TILES;         // [TILES] result complete
  const uint32_t bar_oe = bar_o + 8 * TILES;         // [TILES] result read
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(tail + 448);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tail + 452);
  volatile int *unclean = reinterpret_cast<volatile int *>(tail + 456);   // [4] 1 + number of a tile with non-finite values where the mask hides some
  PromptTile *mail = reinterpret_cast<PromptTile *>(tail + 512);          // [2]
  const uint32_t answer = smem_u32(tail + 576);                           // [2] 16 bytes
  int *table = reinterpret_cast<int *>(tail + 640);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int per = 128 / p.group;                                          // queries of a tile of rows

  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar_mail + 8 * i, 1);
      mbar_init(bar_read + 8 * i, 4 * TILES + 1);
      mbar_init(bar_next + 8 * i, 1);
    }
    for (int i = 0; i < QS; ++i) {
      mbar_init(bar_q + 8 * i, 1);
      mbar_init(bar_qe + 8 * i, 1);
    }
    for (int s = 0; s < ST; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, 1);
    }
    for (int x = 0; x < TILES; ++x) {
      mbar_init(bar_s + 8 * x, 1);
      mbar_init(bar_se + 8 * x, 4);
      mbar_init(bar_p + 8 * x, 4);
      mbar_init(bar_pv + 8 * x, 1);
      mbar_init(bar_o + 8 * x, 2);   // the product, and the issuer's word on `unclean`
      mbar_init(bar_oe + 8 * x, 4);
    }
    *abort_flag = 0;
    for (int i = 0; i < 4; ++i) unclean[i] = 0;
    fence_barrier_init();
    prefetch_tensormap(&tm_q);
    prefetch_tensormap(&tm_k);
    prefetch_tensormap(&tm_v);
  }
  if (warp == 4 * TILES + 1) {
    tmem_alloc(smem_u32(tmem_slot), Cfg::COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  count_tiles(p, table);   // ends with a barrier of the block
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  // The i-th tile of the block from the mail, for the warps that compute.
  auto receive = [&](int i, PromptTile &t) -> bool {
    if (!warp_wait(bar_mail + 8 * (i & 1), (i >> 1) & 1, abort_flag)) return false;
    t = mail[i & 1];
    __syncwarp();
    if (lane == 0) mbar_arrive(bar_read + 8 * (i & 1));
    return true;
  };
  // Tiles of keys are taken from the last to the first.  A tile of rows whose last query sees fewer keys starts later; one without
  // queries or keys has no turn.
  auto first_turn = [&](const PromptTile &t, int n, int x) {
    const int have = min(per, t.queries - x * per);
    return have <= 0 ? n : n - (seen(p, t, x * per + have - 1) + KEYS - 1) / KEYS;
  };

  if (warp < 4 * TILES) {
    if constexpr (Cfg::MOVE) asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    const int x = warp >> 2;                      // tile of rows
    const int row = (warp & 3) * 32 + lane;
    const int in_tile = row / p.group, head = row - in_tile * p.group, query = x * per + in_tile;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + lanes + Cfg::S_COL + x * Cfg::STEP, t_p = tmem + lanes + Cfg::P_COL + x * Cfg::STEP;
    const uint32_t t_o = tmem + lanes + Cfg::O_COL + x * Cfg::STEP;
    const float c = p.scale_log2e;
    const float2 c2 = make_float2(c, c);
    const bool sectors = p.dim % 16 == 0 && p.ldy % 16 == 0 && ((uintptr_t)p.y & 31) == 0;
    uint32_t turns = 0, results = 0;   // of this tile of rows so far: the parities of its barriers
    PromptTile t;
    bool ok = true;
    for (int i = 0; ok && (ok = receive(i, t)) && t.queries > 0; ++i) {
      if (x * per >= t.queries) continue;
      const int lim_lo = seen(p, t, 0), lim_hi = seen(p, t, t.queries - 1);   // keys that the first and the last query see
      const int n = (lim_hi + KEYS - 1) / KEYS, begin = first_turn(t, n, x);
      const bool mine = in_tile < per && query < t.queries;   // rows past the last query (and past per * group) hold anything
      const int lim = mine ? seen(p, t, query) : lim_hi;
      const bool busy = __any_sync(0xffffffffu, mine);        // a warp without rows keeps step and computes nothing
      float m = -INFINITY, l = 0.f;   // reference maximum of the unscaled scores; sum of the weights
      // a tile's maximum: moves the reference maximum if it has to, and with it the sum and O
      auto raise = [&](float top, bool first) {
        if (first) {
          m = top;
          return;
        }
        const bool up = (top - m) * c > MARGIN;
        if (!__any_sync(0xffffffffu, up)) return;
        const float f = up ? ex2((m - top) * c) : 1.f;
        if (up) m = top;
        l *= f;
#pragma unroll
        for (int d = 0; d < DP; d += 16) {
          uint32_t o[16];
          tmem_ld_x16(t_o + d, o);
          tmem_loaded(o);
#pragma unroll
          for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
          tmem_st_x16(t_o + d, o);
        }
      };
      auto hand_over = [&]() {   // P is in tensor memory
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_p + 8 * x);
      };
      for (int it = begin; it < n; ++it, ++turns) {
        const int base = (n - 1 - it) * KEYS;
        if (!(ok = warp_wait(bar_s + 8 * x, turns & 1, abort_flag))) break;
        tc_fence_after();
        const int have = lim - base, some = lim_hi - base;   // keys of this tile that the row sees; that any row sees (the product stops there)
        const bool masked = base + KEYS > lim_lo, first = it == begin;
        if (!busy) {
          if (Cfg::EARLY && lane == 0) mbar_arrive(bar_se + 8 * x);
          __syncwarp();   // what follows (hand_over) takes all lanes
          // in step with the others: two turns ahead, its word would stand for one that is still at work
          if (Cfg::EARLY && !first && !(ok = warp_wait(bar_pv + 8 * x, (turns - 1) & 1, abort_flag))) break;
        } else {
          uint32_t r[KEYS];
#pragma unroll
          for (int k = 0; k < KEYS; k += 32) tmem_ld_x32(t_s + k, r + k);
          tmem_loaded(r);
          float *s = reinterpret_cast<float *>(r);
          if (Cfg::EARLY) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_se + 8 * x);
            __syncwarp();
            if (!first) {   // the previous product has left P and O
              if (!(ok = warp_wait(bar_pv + 8 * x, (turns - 1) & 1, abort_flag))) break;
              tc_fence_after();
            }
          }
          // 32 scores -> 16 columns of P.  The weights are rounded to bf16: the second product takes both operands in the values' type.  That is
          // half a step of the result's type; against 64 bits results were off by 0.0018 to 0.0021 where fp32 weights give 0.0016 (prompts of
          // 40 to 8192 tokens).  Two terms, as over the cache, would double that product and need columns that head size 128 does not have.
          auto weigh = [&](int at, float2 off2, float2 &sum) {
            uint32_t w[16];
            float2 other = make_float2(0.f, 0.f);
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              float2 e = __ffma2_rn(make_float2(s[at + 2 * k], s[at + 2 * k + 1]), c2, off2);
              e.x = ex2(e.x);
              e.y = ex2(e.y);
              if (k & 1) other = __fadd2_rn(other, e);
              else sum = __fadd2_rn(sum, e);
              const __nv_bfloat162 h = __floats2bfloat162_rn(e.x, e.y);
              w[k] = *reinterpret_cast<const uint32_t *>(&h);
            }
            sum = __fadd2_rn(sum, other);
            tmem_st_x16(t_p + at / 2, w);
          };
          bool careful = masked || first;
          if (!careful) {
            // The weights by the reference maximum that is there, without waiting for this tile's own; that one is found beside
            // them and, if it is more than 2^16 above (or a score is NaN or +inf), the tile is done over.
            const float off = -m * c;
            float2 sum = make_float2(0.f, 0.f);
            float x0 = s[0], x1 = s[1];
#pragma unroll
            for (int k = 0; k < KEYS; k += 32) {
              weigh(k, make_float2(off, off), sum);
#pragma unroll
              for (int e = k; e < k + 32; e += 4) {
                x0 = max3_nan(x0, s[e], s[e + 1]);
                x1 = max3_nan(x1, s[e + 2], s[e + 3]);
              }
            }
            const float top = max3_nan(x0, x1, x1);
            careful = __any_sync(0xffffffffu, mine && !((top - m) * c <= MARGIN));
            if (!careful) l += sum.x + sum.y;
          }
          if (careful) {
            tmem_st_wait();   // what the first attempt wrote is written again
            if (masked)
#pragma unroll
              for (int k = 0; k < KEYS; ++k) s[k] = k < have ? s[k] : -INFINITY;
            float x0 = s[0], x1 = s[1];
#pragma unroll
            for (int k = 2; k < KEYS; k += 2) {
              x0 = fmaxf(x0, s[k]);
              x1 = fmaxf(x1, s[k + 1]);
            }
            raise(fmaxf(x0, x1), first);
            const float off = m == -INFINITY ? 0.f : -m * c;
            float2 sum = make_float2(0.f, 0.f);
#pragma unroll
            for (int k = 0; k < KEYS; k += 32)
              if (k < some) weigh(k, make_float2(off, off), sum);
            l += sum.x + sum.y;
          }
        }
        hand_over();
      }
      if (!ok) break;
      const long long q_row = (long long)t.q0 + query;
      const int all_heads = t.kh * p.group + head;
      bool mend = false;   // add the values that were left out of the product
      if (begin < n) {
        if (!(ok = warp_wait(bar_o + 8 * x, results & 1, abort_flag))) break;
        ++results;
        tc_fence_after();
        mend = unclean[i & 3] == i + 1;
      }
      if (!busy) {
        if (begin < n && lane == 0) mbar_arrive(bar_oe + 8 * x);
        continue;
      }
      const float inv = 1.f / l;
      const bool none = begin == n || lim <= 0;
      __nv_bfloat16 *y = static_cast<__nv_bfloat16 *>(p.y) + q_row * p.ldy + (long long)all_heads * p.dim;
#pragma unroll
      for (int d = 0; d < DP; d += 32) {
        uint32_t o[32];
        if (begin < n) {
          tmem_ld_x32(t_o + d, o);
          tmem_loaded(o);
          if (d + 32 == DP) {   // the next tile's products may begin
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_oe + 8 * x);
          }
        }
        uint32_t w[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          const __nv_bfloat162 h = none ? __floats2bfloat162_rn(0.f, 0.f) : __floats2bfloat162_rn(__uint_as_float(o[2 * k]) * inv, __uint_as_float(o[2 * k + 1]) * inv);
          w[k] = *reinterpret_cast<const uint32_t *>(&h);
        }
        if (mine) {
          if (sectors) {   // a lane's row leaves in whole 32-byte sectors
#pragma unroll
            for (int k = 0; k < 16; k += 8)
              if (d + 2 * k < p.dim)
                asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(y + d + 2 * k), "r"(w[k]), "r"(w[k + 1]), "r"(w[k + 2]), "r"(w[k + 3]),
                             "r"(w[k + 4]), "r"(w[k + 5]), "r"(w[k + 6]), "r"(w[k + 7])
                             : "memory");
          } else {
#pragma unroll
            for (int k = 0; k < 16; k += 4)
              if (d + 2 * k < p.dim) *reinterpret_cast<uint4 *>(y + d + 2 * k) = make_uint4(w[k], w[k + 1], w[k + 2], w[k + 3]);
          }
        }
        // A warp that holds some rows only comes together again: the next load from tensor memory takes all its lanes.  (Behind the last
        // one receive() sees to it; here too, the ragged encoder takes 61.5 us instead of 60.4.)
        if (d + 32 < DP) __syncwarp();
      }
      if (mend && mine)   // the tile's first query sees all keys before lim - query: adding an infinity or NaN of those once more changes nothing
        add_nonfinite(p, q_row, all_heads, t.k0, max(0, lim - query), lim);
    }
    if (!ok) {
      *abort_flag = 1;
      report(p.status, DEV_WAIT_TMEM_FULL);
    }
  } else {
    if constexpr (Cfg::MOVE) asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");   // the whole group of warps, the idle ones too
    if (warp == 4 * TILES) {
      uint32_t slot = 0, ph = 0, index = blockIdx.x;   // ring slot of the next load, its parity; the tile at hand
      int sent = 0, loaded = 0;                        // tiles in the mail so far; tiles whose queries were loaded
      bool ok = true;
      auto mail_to_all = [&](const PromptTile &t) -> bool {
        if (!warp_wait_long(bar_read + 8 * (sent & 1), ((sent >> 1) & 1) ^ 1u, abort_flag)) return false;
        if (lane == 0) {
          mail[sent & 1] = t;
          mbar_arrive(bar_mail + 8 * (sent & 1));
        }
        __syncwarp();
        ++sent;
        return true;
      };
      for (int i = 0;; ++i) {
        if (lane == 0) ask_for_block(answer + 16 * (i & 1), bar_next + 8 * (i & 1));
        PromptTile t = find_tile(p, table, index / p.kv_heads);
        if (t.queries > 0) {
          t.kh = index % p.kv_heads;
          if (!(ok = mail_to_all(t))) break;
          const int n = (seen(p, t, t.queries - 1) + KEYS - 1) / KEYS;
          if (n > 0) {
            const int tiles = t.queries > per ? TILES : 1, qs = loaded % QS;
            if (!(ok = warp_wait_long(bar_qe + 8 * qs, ((loaded / QS) & 1) ^ 1u, abort_flag))) break;
            ++loaded;
            if (lane == 0) {
              mbar_arrive_expect_tx(bar_q + 8 * qs, tiles * Cfg::PANELS * 128 * p.group * per);
              for (int x = 0; x < tiles; ++x)
                for (int k = 0; k < Cfg::PANELS; ++k)
                  tma_load_3d(sm_q + qs * Cfg::Q + (x * Cfg::PANELS + k) * 16384, &tm_q, bar_q + 8 * qs, 64 * k, t.kh * p.group, t.q0 + x * per);
            }
            for (int it = 0; it < 2 * n; ++it) {   // K and V in turn
              if (!(ok = warp_wait_long(bar_empty + 8 * slot, ph ^ 1u, abort_flag))) break;
              if (lane == 0) {
                mbar_arrive_expect_tx(bar_full + 8 * slot, Cfg::TILE);
                for (int k = 0; k < Cfg::PANELS; ++k)
                  tma_load_3d(sm_ring + slot * Cfg::TILE + k * Cfg::PANEL, it & 1 ? &tm_v : &tm_k, bar_full + 8 * slot, 64 * k, t.kh,
                              t.k0 + (n - 1 - (it >> 1)) * KEYS);
              }
              if (++slot == ST) slot = 0, ph ^= 1;
            }
            if (!ok) break;
          }
        }
        if (!(ok = warp_wait_long(bar_next + 8 * (i & 1), (i >> 1) & 1, abort_flag))) break;
        const bool given = block_given(answer + 16 * (i & 1), index);
        fence_proxy_async();   // the answer is read before the one after the next may overwrite it
        __syncwarp();
        if (!given) {          // no block is left; nobody asks again
          PromptTile end{};
          end.queries = -1;
          ok = mail_to_all(end);
          break;
        }
      }
      if (!ok && lane == 0) {
        *abort_flag = 1;
        report(p.status, DEV_WAIT_SMEM_EMPTY);
        const uint64_t t0 = globaltimer();   // copies in flight land before the block ends
        while (globaltimer() - t0 < 200000ull) {}
      }
    } else if (warp == 4 * TILES + 1) {
      // descriptors: 128-byte swizzle, 1024 bytes between groups of 8 rows, version 1
      const uint64_t desc_hi = (uint64_t)((1024u >> 4) | (1u << 14) | (2u << 29)) << 32;
      const uint32_t kmajor = 1u << 16, mnmajor = ((uint32_t)Cfg::PANEL >> 4) << 16;   // MN-major: leading offset = one panel
      const uint32_t idesc_s = (1u << 4) | (1u << 7) | (1u << 10) | (((uint32_t)KEYS >> 3) << 17) | ((128u >> 4) << 24);
      const uint32_t idesc_o = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | (((uint32_t)DP >> 3) << 17) | ((128u >> 4) << 24);
      const uint32_t leader = lane == 0;
      const uint32_t q_all = kmajor | uniform(sm_q >> 4), ring = uniform(sm_ring >> 4), tm = uniform(tmem);   // below 2^14: no carry into the next field
      uint32_t ks = 0, kph = 0, vs = 1 % ST, vph = 0;   // ring slots of the next keys and values, with their parities
      auto step = [](uint32_t &slot, uint32_t &ph) {
        slot += 2;
        if (slot >= ST) slot -= ST, ph ^= 1;
      };
      uint32_t scored[TILES] = {}, weighed[TILES] = {}, results[TILES] = {};   // products so far, tile of rows by tile
      int loaded = 0;
      bool ok = true;
      PromptTile t;
      for (int i = 0; ok && (ok = receive(i, t)) && t.queries > 0; ++i) {
        const int lim_lo = seen(p, t, 0), lim_hi = seen(p, t, t.queries - 1);
        const int n = (int)uniform((lim_hi + KEYS - 1) / KEYS), visible = (int)uniform(lim_lo);
        if (n == 0) continue;
        int begin[TILES];
#pragma unroll
        for (int x = 0; x < TILES; ++x) begin[x] = (int)uniform(first_turn(t, n, x));
        const uint32_t qs = loaded % QS, q_lo = q_all + qs * (Cfg::Q >> 4);
        auto scores = [&](int x, int it) -> bool {
          if (it >= begin[x]) {
            if (Cfg::EARLY && scored[x] > 0 && !warp_wait(bar_se + 8 * x, (scored[x] - 1) & 1, abort_flag)) return false;
            if (!warp_wait(bar_full + 8 * ks, kph, abort_flag)) return false;
            tc_fence_after();
            const uint32_t k_lo = kmajor | (ring + ks * (Cfg::TILE >> 4));
#pragma unroll
            for (int kk = 0; kk < DP / 16; ++kk)
              umma_ss(leader, tm + Cfg::S_COL + x * Cfg::STEP, desc_hi | (q_lo + (x * Cfg::PANELS + (kk >> 2)) * 1024 + (kk & 3) * 2),
                      desc_hi | (k_lo + (kk >> 2) * (Cfg::PANEL >> 4) + (kk & 3) * 2), idesc_s, kk != 0);
            commit_if(leader, bar_s + 8 * x);
            ++scored[x];
          }
          if (x == TILES - 1) {   // both tiles' products with these keys are on their way
            commit_if(leader, bar_empty + 8 * ks);
            step(ks, kph);
            if (it + 1 == n) commit_if(leader, bar_qe + 8 * qs);
          }
          return true;
        };
        if (!(ok = warp_wait(bar_q + 8 * qs, (loaded / QS) & 1, abort_flag))) break;
        ++loaded;
#pragma unroll
        for (int x = 0; x < TILES; ++x)
          if (ok) ok = scores(x, 0);
        for (int it = 0; it < n && ok; ++it) {
          const int base = (n - 1 - it) * KEYS;
          if (Cfg::EARLY && it + 1 < n && !(ok = scores(0, it + 1))) break;
          if (!(ok = warp_wait(bar_full + 8 * vs, vph, abort_flag))) break;
          if (base + KEYS > visible) {
            // The product takes 16 keys at a time and stops after the last one that anybody here sees.  Values past that key belong
            // to others and may hold anything: zeros in their place, since the tensor cores multiply every value by every row's
            // weight and 0 * NaN is NaN.  Values on the diagonal are hidden
            // from some rows only: one that is not finite becomes zero here, and the rows that see it add it at the end (any weight
            // above 0 leaves an infinity or NaN what it is).
            uint8_t *v = gen + QS * Cfg::Q + vs * Cfg::TILE;
            constexpr int PIECES = 8 * Cfg::PANELS;   // 16-byte pieces of a key's values
            const int none = max(0, min(KEYS, lim_hi - base)), some = max(0, min(none, lim_lo - base));
            for (int k = none * PIECES + lane; k < (none + 15) / 16 * 16 * PIECES; k += 32) {
              const int key = k / PIECES, piece = k % PIECES;
              *reinterpret_cast<uint4 *>(v + (piece >> 3) * Cfg::PANEL + key * 128 + (piece & 7) * 16) = make_uint4(0, 0, 0, 0);
            }
            bool bad = false;
            for (int k = some * PIECES + lane; k < none * PIECES; k += 32) {
              const int key = k / PIECES, piece = k % PIECES;
              const uint4 w = *reinterpret_cast<const uint4 *>(v + (piece >> 3) * Cfg::PANEL + key * 128 + (piece & 7) * 16);
              for (uint32_t u : {w.x, w.y, w.z, w.w}) bad |= (u & 0x7f80u) == 0x7f80u || (u & 0x7f800000u) == 0x7f800000u;
            }
            if (__any_sync(0xffffffffu, bad)) {
              unclean[i & 3] = i + 1;   // this warp is at most two tiles ahead: the mail has two places
#pragma unroll 1
              for (int k = some * PIECES * 4 + lane; k < none * PIECES * 4; k += 32) {   // words
                const int key = k / (PIECES * 4), word = k % (PIECES * 4);
                uint32_t *w = reinterpret_cast<uint32_t *>(v + (word >> 5) * Cfg::PANEL + key * 128 + (word & 31) * 4);
                *w &= ((*w & 0x7f80u) == 0x7f80u ? 0xffff0000u : 0xffffffffu) & ((*w & 0x7f800000u) == 0x7f800000u ? 0xffffu : 0xffffffffu);
              }
            }
            fence_proxy_async();
            __syncwarp();
          }
          const uint32_t v_lo = mnmajor | (ring + vs * (Cfg::TILE >> 4));
          const int last_key = (int)uniform(lim_hi - base);
#pragma unroll
          for (int x = 0; x < TILES; ++x) {
            if (it >= begin[x]) {
              if (it == begin[x] && results[x] > 0 && !(ok = warp_wait(bar_oe + 8 * x, (results[x] - 1) & 1, abort_flag))) break;
              const uint32_t more = it != begin[x];
              if (!(ok = warp_wait(bar_p + 8 * x, weighed[x] & 1, abort_flag))) break;
              tc_fence_after();
#pragma unroll
              for (int kk = 0; kk < KEYS / 16; ++kk)   // 16 keys: 8 columns of P, 16 rows of V
                umma_ts(16 * kk < last_key ? leader : 0u, tm + Cfg::O_COL + x * Cfg::STEP, tm + Cfg::P_COL + x * Cfg::STEP + 8 * kk,
                        desc_hi | (v_lo + 128 * kk), idesc_o, kk != 0 ? 1u : more);
              ++weighed[x];
              if (Cfg::EARLY) commit_if(leader, bar_pv + 8 * x);
            }
            if (x == TILES - 1) {
              commit_if(leader, bar_empty + 8 * vs);
              step(vs, vph);
            }
            if (it + 1 == n && begin[x] < n) {
              commit_if(leader, bar_o + 8 * x);
              if (lane == 0) mbar_arrive(bar_o + 8 * x);
              ++results[x];
            }
            // Without columns of their own the weights lie where the next scores go.  Both products are this thread's, and the
            // tensor cores take them in order.
            if (!Cfg::EARLY && it + 1 < n && !(ok = scores(x, it + 1))) break;
          }
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
  if (grid > MOST_BLOCKS)
    return fail(SOFIE_B200_ERR_TOO_LARGE, "prompt_attention_enqueue: %lld queries of %d sequences and %d heads", p.q_rows, p.batch, p.heads);
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

template <int DP>
static int launch_fma(sofie_b200_ctx *ctx, PromptParams p) {
  const int parts = (p.group + PF_ROWS - 1) / PF_ROWS;
  p.tokens = parts > 1 ? 1 : PF_ROWS / p.group;
  const long long grid = (p.q_rows / p.tokens + p.batch) * p.kv_heads * parts;
  if (grid > 0x7fffffffLL) return fail(SOFIE_B200_ERR_TOO_LARGE, "prompt_attention_enqueue: %lld queries of %d heads", p.q_rows, p.heads);
  if (!p.k_rows) p.k = p.v = p.q;   // nothing is read, but the address a copy of no bytes is given should exist
  SB_CUDA(cudaFuncSetAttribute(prompt_fma_kernel<DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, FmaCfg<DP>::SMEM));   // per device
  // Few blocks over many keys: clusters of 2, 4 or 8 share the keys of a tile of rows, as long as the blocks fill the GPU at most one and a half
  // times and every team gets a tile of keys.  One block against two: 770 queries of 8 heads over 1770 keys 70 us, 61; 300 queries 21, 19;
  // 20 queries over 2020 keys 99, 56 (four 33, eight 22); but 100 queries 12.9, 13.1; 300 of 16 heads of 128 33, 45; 2048 of 16 heads 290, 316.
  int share = 1;
  while (share < 8 && grid * share * 2 <= (long long)ctx->sm_count * FmaCfg<DP>::BLOCKS * 3 / 2 && p.k_rows / p.batch >= share * 2 * FmaCfg<DP>::TEAMS * PF_KEYS)
    share *= 2;
  cudaLaunchAttribute together{};
  together.id = cudaLaunchAttributeClusterDimension;
  together.val.clusterDim.x = share;
  together.val.clusterDim.y = together.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(grid * share));
  cfg.blockDim = dim3(FmaCfg<DP>::THREADS);
  cfg.dynamicSmemBytes = FmaCfg<DP>::SMEM;
  cfg.stream = ctx->stream;
  cfg.attrs = &together;
  cfg.numAttrs = share > 1;
  SB_CUDA(cudaLaunchKernelEx(&cfg, prompt_fma_kernel<DP>, p, parts, share));
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
  return !plan ? "" : plan->d.dtype == SOFIE_B200_F32 ? "fma" : "umma";
}

int sofie_b200_prompt_attention_enqueue(sofie_b200_prompt_attention_plan *plan, const void *q, const void *k, const void *v, void *y,
                                        const int32_t *cu_seqlens_q, const int32_t *cu_seqlens_k, int64_t batch, int64_t q_tokens,
                                        int64_t k_tokens) {
  if (!plan) return fail(SOFIE_B200_ERR_INVALID, "prompt_attention_enqueue: plan is NULL");
  const sofie_b200_prompt_attention_desc &d = plan->d;
  if (batch < 0 || batch > 0x3fffffff || q_tokens < 0 || q_tokens > (1 << 27) || k_tokens < 0 || k_tokens > (1 << 27))
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
  p.most_keys = d.dtype == SOFIE_B200_BF16 ? MOST_KEYS_BF16 : MOST_KEYS_F32;
  p.scale_log2e = d.scale * 1.4426950408889634f;
  p.status = ctx->d_status;
  if (d.dtype == SOFIE_B200_BF16) {
    if (d.head_dim <= 64) return launch_umma<64>(ctx, p);
    if (d.head_dim <= 128) return launch_umma<128>(ctx, p);
    return launch_umma<256>(ctx, p);
  }
  if (d.head_dim <= 64) return launch_fma<64>(ctx, p);
  if (d.head_dim <= 128) return launch_fma<128>(ctx, p);
  return launch_fma<256>(ctx, p);
}

}  // extern "C"
