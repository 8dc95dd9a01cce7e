// Attention of one new token per sequence over a paged key-value cache:
//     y[b, h] = sum_j softmax_j(scale q[b, h] . k[j, h / g]) v[j, h / g],   j < seq_lens[b],   g = heads / kv_heads.
// Each key and value is read once for the query heads that share it, 16 of them at a time (a larger group reads it once for every 16), so
// the kernel is bound by HBM: 2 D elements per token and key head for 4 g D operations.
//
// Split.  One sequence may be the whole batch and 65,000 tokens long, or a batch may hold hundreds of very different lengths.
// The tokens of all sequences and key heads are one row of units of 16 keys, cut into equal shares, one for every resident warp
// (paged.cuh: split_at).  A warp works by itself down its share, from one sequence or head to the next without meeting another one.
// A share may end inside a sequence; the parts of such a sequence (running maximum, sum, unnormalised result, all fp32) go to the
// workspace and a second kernel joins them in the order of the keys, so results do not depend on timing.  Lengths are read on the
// device: a captured call is replayed for any other lengths.
#include <math.h>
#include <new>

#include "generate.cuh"
#include "ptx.cuh"

namespace sb200 {
using namespace ptx;

constexpr int PA_UNIT = 16;       // keys
constexpr int PA_ROWS = 16;       // query heads of an item at most: the rows of one mma tile
constexpr int PA_LEAST = 3;       // slots that are worth a worker of their own.  2, 3, 4, 6, 9: few short sequences in fp32 17, 19, 21, 24, 29 us;
                                  // one of 3000 tokens in bf16 20.6, 17.2, 19.1, 21.1, 23.2 us
constexpr float PA_MARGIN = 16.f; // the reference maximum moves when a score is 2^16 above it: fp32 keeps its relative precision up there

struct PagedAttnParams {
  PagedView kv;
  const void *q, *cache_k, *cache_v;
  void *y;
  long long ldq, ldy;
  int heads, group, dim;      // group = heads / kv_heads
  int items, parts_per_key;   // items of a sequence = kv_heads * parts_per_key; parts_per_key = ceil(group / 16)
  int rows;                   // min(16, group): what a place of the workspace holds
  float scale_log2e;
  int *status;
  // workspace
  int4 *joins;                // [workers] {sequence, item, parts, 0}: the item that begins with this worker and ends with a later one
  float *part_m, *part_l;     // [workers * 2][rows]
  float *part_o;              // [workers * 2][rows][DP]
};

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}


// Every block sums up the lengths by itself (they are few, and in L2); each of its warps gets its share.  All threads call it.
template <int THREADS>
__device__ __forceinline__ Cursor find_share(const PagedAttnParams &p, long long *slots, int *workers) {
  constexpr int WARPS = THREADS / 32;
  __shared__ long long warp_sum[WARPS];
  __shared__ Cursor s_at[WARPS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (p.kv.batch + THREADS - 1) / THREADS;   // a thread's sequences lie together
  const int b0 = min(p.kv.batch, tid * per), b1 = min(p.kv.batch, b0 + per);
  long long mine = 0;
  bool bad = false;
  for (int b = b0; b < b1; ++b) mine += slots_of(paged_len(p.kv, b, &bad), PA_UNIT, p.items);
  if (bad) report(p.status, DEV_BAD_INDEX);
  long long incl = mine;
  for (int o = 1; o < 32; o <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += x;
  }
  if (lane == 31) warp_sum[warp] = incl;
  if (lane == 0) s_at[warp].left = 0;
  __syncthreads();
  long long before = incl - mine, total = 0;
  for (int w = 0; w < WARPS; ++w) {
    if (w < warp) before += warp_sum[w];
    total += warp_sum[w];
  }
  const int n = split_workers(total, gridDim.x * WARPS, PA_LEAST);
  for (int w = 0; w < WARPS; ++w) {
    const int c = blockIdx.x * WARPS + w;
    if (c >= n) break;
    const long long begin = split_at(total, n, c), end = split_at(total, n, c + 1);
    if (begin < end && begin >= before && begin < before + mine) {   // one thread
      long long at = before;
      for (int b = b0; b < b1; ++b) {
        Cursor k;
        k.len = paged_len(p.kv, b, &bad);
        const long long all = slots_of(k.len, PA_UNIT, p.items);
        if (begin < at + all) {
          k.b = b;
          k.left = end - begin;
          cursor_start(k, begin - at, PA_UNIT);
          s_at[w] = k;
          break;
        }
        at += all;
      }
    }
  }
  __syncthreads();
  *slots = total;
  *workers = n;
  return s_at[warp];
}

// Padding rows: sequences without tokens get zeros.
template <class T>
__device__ __forceinline__ void zero_empty(const PagedAttnParams &p) {
  bool bad = false;
  for (int b = blockIdx.x; b < p.kv.batch; b += gridDim.x)
    if (paged_len(p.kv, b, &bad) == 0) {
      T *y = static_cast<T *>(p.y) + b * p.ldy;
      for (int i = threadIdx.x; i < p.heads * p.dim; i += blockDim.x) from_f32(y + i, 0.f);
    }
}

// The item at the cursor (at its first unit) begins with this worker and goes on: which workers have its parts.
__device__ __forceinline__ void announce_join(const PagedAttnParams &p, const Cursor &c, int worker, long long slots, int workers) {
  const long long item_end = split_at(slots, workers, worker + 1) - c.left + c.units;
  p.joins[worker] = make_int4(c.b, c.item, split_last(slots, workers, item_end) - worker + 1, 0);
}

// ---- loads: each warp has a ring of STAGES units, filled by cp.async through the block table ------------------------------------------
// Lane r < 16 looks up the row of key r of the next unit one step ahead.  A row is CH 16-byte pieces; piece c of row r lies at c ^ (r & 7),
// which keeps eight rows' equal pieces in eight bank groups.  Keys that are not there (past the end, no page) come as zeros.
template <class T, int DP, int STAGES>
struct Loader {
  static constexpr int CH = DP * (int)sizeof(T) / 16, PER = 16 / (int)sizeof(T), TILE = PA_UNIT * DP * (int)sizeof(T);
  const PagedAttnParams &p;
  const T *cache_k, *cache_v;
  uint32_t ring;
  Cursor at;
  long long row;
  bool bad;
  uint32_t valid[STAGES - 1];   // of the units under way: which keys are there

  __device__ __forceinline__ void look_up() {
    const int lane = threadIdx.x & 31;
    row = -1;
    if (at.left <= 0) return;
    const int key = at.unit * PA_UNIT + lane;
    if (lane < PA_UNIT && key < at.len) {
      row = paged_row(p.kv, at.b, key);
      if (row < 0) bad = true;
      else row += (long long)(at.item / p.parts_per_key) * p.kv.head_stride;
    }
  }
  __device__ __forceinline__ uint32_t issue(uint32_t stage) {   // the unit at the cursor, if there is one, and on to the next
    uint32_t there_mask = 0;
    if (at.left > 0) {
      const int lane = threadIdx.x & 31;
      const uint32_t dk = ring + stage * (2 * TILE), dv = dk + TILE;
#pragma unroll
      for (int i = 0; i < PA_UNIT * CH / 32; ++i) {
        const int flat = i * 32 + lane, r = flat / CH, c = flat % CH;
        const long long off = __shfl_sync(0xffffffffu, row, r);
        const bool there = off >= 0 && c * PER < p.dim;
        const long long e = there ? off + c * PER : 0;
        const uint32_t d = r * (CH * 16) + ((c ^ (r & 7)) << 4);
        cp_async_16(dk + d, cache_k + e, there);
        cp_async_16(dv + d, cache_v + e, there);
      }
      there_mask = __ballot_sync(0xffffffffu, row >= 0);
      cursor_next(at, p.kv, p.items, PA_UNIT);
      look_up();
    }
    cp_async_commit();
    return there_mask;
  }
  __device__ __forceinline__ void begin(const Cursor &c, uint32_t ring_, const void *k, const void *v) {
    cache_k = static_cast<const T *>(k);
    cache_v = static_cast<const T *>(v);
    ring = ring_;
    at = c;
    bad = false;
    look_up();
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) valid[s] = issue(s);
  }
  // The unit in `stage` is complete after this; the stage before it, which everybody has read, is filled again.
  __device__ __forceinline__ uint32_t next(uint32_t stage) {
    __syncwarp();
    const uint32_t fresh = issue(stage == 0 ? STAGES - 1 : stage - 1), now = valid[0];
    cp_async_wait<STAGES - 1>();
    __syncwarp();
#pragma unroll
    for (int i = 0; i + 1 < STAGES - 1; ++i) valid[i] = valid[i + 1];
    valid[STAGES - 2] = fresh;
    return now;
  }
};

template <int DP>
struct Bf16Cfg {
  static constexpr int STAGES = DP == 64 ? 6 : 3, THREADS = 128, TILE = PA_UNIT * DP * 2;
  static int smem(int) { return THREADS / 32 * STAGES * 2 * TILE; }
};

// bf16.  Scores and weighted values on mma.m16n8k16 with the 16 rows = query heads of the group (rows past the group cost nothing that HBM
// would not wait for).  The weights of the second product are split into two bf16 terms, high + low (error 2^-16 instead of 2^-8):
// the tensor cores have the time.  The high term is cut, not rounded, and the low one kept above zero (by 2^-20 of the weight), so that
// both have the weight's sign and an infinite value comes out infinite: 0 * inf and inf - inf are NaN.  As fast as rounding (230, 61.5 us).
// Bound by HBM; at head size 128 the rings of two blocks are 192 KB an SM, two thirds of it on the way.  160 sequences, 1.22 GB of cache:
// 209 to 230 us, 5.3 to 5.8 TB/s (DRAM 75 % busy, issue slots 42 %, tensor pipe 28 %); one of 65,543 tokens, 268 MB: 61 us with the launch of
// both kernels, 4.4 TB/s.  A fixed split of every sequence into equal parts, one block each: 66 and 236 us.
template <int DP>
__global__ void __launch_bounds__(128) paged_mma_kernel(const __grid_constant__ PagedAttnParams p) {
  using Cfg = Bf16Cfg<DP>;
  typedef __nv_bfloat16 T;
  extern __shared__ __align__(128) uint8_t smem[];
  asm volatile("griddepcontrol.launch_dependents;");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, worker = blockIdx.x * 4 + warp;
  long long slots;
  int workers;
  Cursor at = find_share<Cfg::THREADS>(p, &slots, &workers);
  if (lane == 0) p.joins[worker] = make_int4(0, 0, 0, 0);
  const uint32_t ring = smem_u32(smem) + warp * (Cfg::STAGES * 2 * Cfg::TILE);
  Loader<T, DP, Cfg::STAGES> load{p};
  load.begin(at, ring, p.cache_k, p.cache_v);
  zero_empty<T>(p);
  uint32_t stage = 0;
  while (at.left > 0) {
    // ---- one segment: the units of one item that lie in this share ----
    const int first_unit = at.unit;
    const int n = (int)min((long long)(at.units - at.unit), at.left);
    const int key_head = at.item / p.parts_per_key, row0 = at.item % p.parts_per_key * PA_ROWS;
    const int rows = min(PA_ROWS, p.group - row0);
    const int r0 = lane >> 2, r1 = r0 + 8;   // this lane's two rows of the mma tiles
    uint32_t qf[DP / 16][4];
    {
      const T *q = static_cast<const T *>(p.q) + at.b * p.ldq + (long long)(key_head * p.group + row0) * p.dim;
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int r = j & 1 ? r1 : r0, d = kk * 16 + (j >> 1) * 8 + (lane & 3) * 2;
          qf[kk][j] = r < rows && d < p.dim ? *reinterpret_cast<const uint32_t *>(q + (long long)r * p.dim + d) : 0u;
        }
    }
    float o[DP / 8][4];
#pragma unroll
    for (int i = 0; i < DP / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;   // maxima in units of log2; -inf: no key yet

    for (int u = 0; u < n; ++u) {
      const uint32_t valid = load.next(stage);
      const uint32_t sk = ring + stage * (2 * Cfg::TILE), sv = sk + Cfg::TILE;
      stage = stage == Cfg::STAGES - 1 ? 0 : stage + 1;
      if (valid == 0) continue;
      // ---- scores: 16 rows x 16 keys ----
      float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
      const int kr = (lane & 7) + ((lane & 16) >> 1);   // matrices: keys 0-7 low dims, keys 0-7 high, keys 8-15 low, keys 8-15 high
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk) {
        uint32_t b[4];
        const int c = kk * 2 + ((lane >> 3) & 1);
        ldmatrix_x4(b, sk + kr * (DP * 2) + ((c ^ (kr & 7)) << 4));
        mma_bf16(s[0], qf[kk], b[0], b[1]);
        mma_bf16(s[1], qf[kk], b[2], b[3]);
      }
      float x0 = -3.0e38f, x1 = -3.0e38f;   // a key is there: the maximum is a number
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int key = t * 8 + (lane & 3) * 2 + j;
          const bool on = valid >> key & 1;
          s[t][j] = on ? s[t][j] * p.scale_log2e : -INFINITY;
          s[t][2 + j] = on ? s[t][2 + j] * p.scale_log2e : -INFINITY;
          x0 = fmaxf(x0, s[t][j]);
          x1 = fmaxf(x1, s[t][2 + j]);
        }
      if (__any_sync(0xffffffffu, x0 > m0 + PA_MARGIN || x1 > m1 + PA_MARGIN)) {
        x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 1));
        x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 1));
        x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 2));
        x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 2));
        const bool up0 = x0 > m0 + PA_MARGIN, up1 = x1 > m1 + PA_MARGIN;
        const float f0 = up0 ? ex2(m0 - x0) : 1.f, f1 = up1 ? ex2(m1 - x1) : 1.f;
        if (up0) m0 = x0;
        if (up1) m1 = x1;
        l0 *= f0;
        l1 *= f1;
#pragma unroll
        for (int i = 0; i < DP / 8; ++i) {
          o[i][0] *= f0; o[i][1] *= f0;
          o[i][2] *= f1; o[i][3] *= f1;
        }
      }
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const float mm = half ? m1 : m0;
          const float e0 = ex2(s[t][2 * half] - mm), e1 = ex2(s[t][2 * half + 1] - mm);
          if (half) l1 += e0 + e1;
          else l0 += e0 + e1;
          const float h0 = __uint_as_float(__float_as_uint(e0) & 0xffff0000u), h1 = __uint_as_float(__float_as_uint(e1) & 0xffff0000u);
          const __nv_bfloat162 r = __floats2bfloat162_rn(fmaxf(e0 - h0, e0 * 0x1p-20f), fmaxf(e1 - h1, e1 * 0x1p-20f));
          hi[t * 2 + half] = __byte_perm(__float_as_uint(e0), __float_as_uint(e1), 0x7632);
          lo[t * 2 + half] = *reinterpret_cast<const uint32_t *>(&r);
        }
      // ---- weighted values: 16 rows x DP ----
      const int vr = lane & 15;   // matrices: keys 0-7, keys 8-15 of dims d .. d + 7, then of d + 8 .. d + 15
#pragma unroll
      for (int dd = 0; dd < DP / 16; ++dd) {
        uint32_t b[4];
        const int c = dd * 2 + (lane >> 4);
        ldmatrix_x4_trans(b, sv + vr * (DP * 2) + ((c ^ (vr & 7)) << 4));
        mma_bf16(o[2 * dd], hi, b[0], b[1]);
        mma_bf16(o[2 * dd + 1], hi, b[2], b[3]);
        mma_bf16(o[2 * dd], lo, b[0], b[1]);
        mma_bf16(o[2 * dd + 1], lo, b[2], b[3]);
      }
    }

    l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
    l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
    const bool begins = first_unit == 0, ends = first_unit + n == at.units;
    if (begins && ends) {
      T *y = static_cast<T *>(p.y) + at.b * p.ldy + (long long)(key_head * p.group + row0) * p.dim;
      const float i0 = m0 == -INFINITY ? 0.f : 1.f / l0, i1 = m1 == -INFINITY ? 0.f : 1.f / l1;
#pragma unroll
      for (int i = 0; i < DP / 8; ++i) {
        const int d = i * 8 + (lane & 3) * 2;
        if (d < p.dim) {
          if (r0 < rows) *reinterpret_cast<__nv_bfloat162 *>(y + (long long)r0 * p.dim + d) = __floats2bfloat162_rn(o[i][0] * i0, o[i][1] * i0);
          if (r1 < rows) *reinterpret_cast<__nv_bfloat162 *>(y + (long long)r1 * p.dim + d) = __floats2bfloat162_rn(o[i][2] * i1, o[i][3] * i1);
        }
      }
    } else {
      const long long place = (long long)worker * 2 + (begins ? 1 : 0);
      float *po = p.part_o + place * p.rows * DP;
      if ((lane & 3) == 0) {
        if (r0 < rows) p.part_m[place * p.rows + r0] = m0, p.part_l[place * p.rows + r0] = l0;
        if (r1 < rows) p.part_m[place * p.rows + r1] = m1, p.part_l[place * p.rows + r1] = l1;
      }
#pragma unroll
      for (int i = 0; i < DP / 8; ++i) {
        const int d = i * 8 + (lane & 3) * 2;
        if (r0 < rows) *reinterpret_cast<float2 *>(po + r0 * DP + d) = make_float2(o[i][0], o[i][1]);
        if (r1 < rows) *reinterpret_cast<float2 *>(po + r1 * DP + d) = make_float2(o[i][2], o[i][3]);
      }
      if (begins && lane == 0) announce_join(p, at, worker, slots, workers);
    }
    at.unit += n - 1;
    at.left -= n - 1;
    cursor_next(at, p.kv, p.items, PA_UNIT);
  }
  cp_async_wait<0>();
  if (load.bad) report(p.status, DEV_BAD_INDEX);
}

template <int DP, int R>
struct F32Cfg {
  static constexpr int STAGES = DP == 128 && R > 4 ? 2 : 3, THREADS = DP == 256 ? 64 : 128, TILE = PA_UNIT * DP * 4;
  static int smem(int rows) { return THREADS / 32 * (STAGES * 2 * TILE + rows * DP * 4 + rows * PA_UNIT * 4); }
};

// fp32, on the CUDA cores.  Scores: a lane has one key and half of its dimensions, the queries are read from shared memory by all lanes
// at once; weights go through shared memory; weighted values: a lane has 4 dimensions (or, at head size 64, every other key of them).
// R: query heads of an item at most.  Six sequences of up to 400 tokens, 2 key heads of 64: 18 us, the way of one launch after another
// (the lengths, the table, a share of three units, the join), 0.38 MB.
template <int DP, int R>
__global__ void __launch_bounds__(F32Cfg<DP, R>::THREADS) paged_fma_kernel(const __grid_constant__ PagedAttnParams p) {
  using Cfg = F32Cfg<DP, R>;
  constexpr int CH = DP / 4, WARPS = Cfg::THREADS / 32;
  constexpr int KPL = CH >= 32 ? 1 : 32 / CH;        // keys side by side in the weighted values
  constexpr int VPL = CH >= 32 ? CH / 32 : 1;        // pieces of a row per lane
  extern __shared__ __align__(128) uint8_t smem[];
  asm volatile("griddepcontrol.launch_dependents;");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, worker = blockIdx.x * WARPS + warp;
  long long slots;
  int workers;
  Cursor at = find_share<Cfg::THREADS>(p, &slots, &workers);
  if (lane == 0) p.joins[worker] = make_int4(0, 0, 0, 0);
  uint8_t *mine = smem + warp * (Cfg::STAGES * 2 * Cfg::TILE);
  float *sq = reinterpret_cast<float *>(smem + WARPS * Cfg::STAGES * 2 * Cfg::TILE) + warp * p.rows * (DP + PA_UNIT);   // [rows][DP], scaled
  float *sp = sq + p.rows * DP;                                                                                        // [rows][16] weights
  Loader<float, DP, Cfg::STAGES> load{p};
  load.begin(at, smem_u32(mine), p.cache_k, p.cache_v);
  zero_empty<float>(p);
  uint32_t stage = 0;
  const int key = lane & 15, half = lane >> 4;
  const int col = KPL > 1 ? lane % CH : lane, sub = KPL > 1 ? lane / CH : 0;
  while (at.left > 0) {
    const int first_unit = at.unit;
    const int n = (int)min((long long)(at.units - at.unit), at.left);
    const int key_head = at.item / p.parts_per_key, row0 = at.item % p.parts_per_key * PA_ROWS;
    const int rows = min(PA_ROWS, p.group - row0);
    const float *q = static_cast<const float *>(p.q) + at.b * p.ldq + (long long)(key_head * p.group + row0) * p.dim;
    __syncwarp();
    for (int i = lane; i < rows * DP; i += 32) {
      const int r = i / DP, d = i % DP;
      sq[i] = d < p.dim ? q[(long long)r * p.dim + d] * p.scale_log2e : 0.f;
    }
    float4 acc[R][VPL];
    float m[R], l[R];   // maxima in units of log2; -inf: no key yet.  Sums: this lane's key
#pragma unroll
    for (int h = 0; h < R; ++h) {
      m[h] = -INFINITY;
      l[h] = 0.f;
#pragma unroll
      for (int v = 0; v < VPL; ++v) acc[h][v] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    for (int u = 0; u < n; ++u) {
      const uint32_t valid = load.next(stage);
      const float4 *tk = reinterpret_cast<const float4 *>(mine + stage * (2 * Cfg::TILE)), *tv = tk + Cfg::TILE / 16;
      stage = stage == Cfg::STAGES - 1 ? 0 : stage + 1;
      if (valid == 0) continue;
      float s[R];
#pragma unroll
      for (int h = 0; h < R; ++h) s[h] = 0.f;
#pragma unroll 4
      for (int i = 0; i < CH / 2; ++i) {
        const int c = half * (CH / 2) + i;
        const float4 k = tk[key * CH + (c ^ (key & 7))];
#pragma unroll
        for (int h = 0; h < R; ++h)
          if (h < rows) {
            const float4 x = *reinterpret_cast<const float4 *>(sq + h * DP + c * 4);
            s[h] = fmaf(k.x, x.x, fmaf(k.y, x.y, fmaf(k.z, x.z, fmaf(k.w, x.w, s[h]))));
          }
      }
      const bool on = valid >> key & 1;
#pragma unroll
      for (int h = 0; h < R; ++h)
        if (h < rows) {
          s[h] += __shfl_xor_sync(0xffffffffu, s[h], 16);
          if (!on) s[h] = -INFINITY;
          if (__any_sync(0xffffffffu, s[h] > m[h] + PA_MARGIN || m[h] == -INFINITY)) {
            float top = s[h];
#pragma unroll
            for (int o = 1; o < 16; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            top = fmaxf(top, fmaxf(m[h], -3.0e38f));   // a key is there: the maximum is a number
            const float f = ex2(m[h] - top);
            m[h] = top;
            l[h] *= f;
#pragma unroll
            for (int v = 0; v < VPL; ++v) { acc[h][v].x *= f; acc[h][v].y *= f; acc[h][v].z *= f; acc[h][v].w *= f; }
          }
          const float e = ex2(s[h] - m[h]);
          l[h] += e;
          if (half == 0) sp[h * PA_UNIT + key] = e;
        }
      __syncwarp();
#pragma unroll
      for (int k0 = 0; k0 < PA_UNIT; k0 += 4 * KPL) {
        float4 val[4][VPL];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int kk = k0 + i * KPL + sub;
#pragma unroll
          for (int v = 0; v < VPL; ++v) val[i][v] = tv[kk * CH + ((col + 32 * v) ^ (kk & 7))];
        }
#pragma unroll
        for (int h = 0; h < R; ++h)
          if (h < rows) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float e = sp[h * PA_UNIT + k0 + i * KPL + sub];
#pragma unroll
              for (int v = 0; v < VPL; ++v) {
                acc[h][v].x = fmaf(e, val[i][v].x, acc[h][v].x);
                acc[h][v].y = fmaf(e, val[i][v].y, acc[h][v].y);
                acc[h][v].z = fmaf(e, val[i][v].z, acc[h][v].z);
                acc[h][v].w = fmaf(e, val[i][v].w, acc[h][v].w);
              }
            }
          }
      }
      __syncwarp();   // the weights are read
    }
    const bool begins = first_unit == 0, ends = first_unit + n == at.units;
    const long long place = (long long)worker * 2 + (begins ? 1 : 0);
    float *y = static_cast<float *>(p.y) + at.b * p.ldy + (long long)(key_head * p.group + row0) * p.dim;
#pragma unroll
    for (int h = 0; h < R; ++h)
      if (h < rows) {
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) l[h] += __shfl_xor_sync(0xffffffffu, l[h], o);
        const float inv = m[h] == -INFINITY ? 0.f : 1.f / l[h];
#pragma unroll
        for (int v = 0; v < VPL; ++v) {
          if (KPL > 1) {
            acc[h][v].x += __shfl_xor_sync(0xffffffffu, acc[h][v].x, 16);
            acc[h][v].y += __shfl_xor_sync(0xffffffffu, acc[h][v].y, 16);
            acc[h][v].z += __shfl_xor_sync(0xffffffffu, acc[h][v].z, 16);
            acc[h][v].w += __shfl_xor_sync(0xffffffffu, acc[h][v].w, 16);
          }
          const int d = (col + 32 * v) * 4;
          if (sub == 0) {
            if (begins && ends) {
              if (d < p.dim) *reinterpret_cast<float4 *>(y + (long long)h * p.dim + d) = make_float4(acc[h][v].x * inv, acc[h][v].y * inv, acc[h][v].z * inv, acc[h][v].w * inv);
            } else {
              *reinterpret_cast<float4 *>(p.part_o + (place * p.rows + h) * DP + d) = acc[h][v];
            }
          }
        }
        if (!(begins && ends) && lane == 0) {
          p.part_m[place * p.rows + h] = m[h];
          p.part_l[place * p.rows + h] = l[h];
        }
      }
    if (begins && !ends && lane == 0) announce_join(p, at, worker, slots, workers);
    at.unit += n - 1;
    at.left -= n - 1;
    cursor_next(at, p.kv, p.items, PA_UNIT);
  }
  cp_async_wait<0>();
  if (load.bad) report(p.status, DEV_BAD_INDEX);
}

// Joins the parts of split items, each in the order of its workers: place 1 of the one it began with, place 0 of the following ones.
// Many items of few parts (a large batch: nearly every warp ends inside an item) go a warp to a row; few items of many parts (one
// long sequence) go a block to 32 dimensions of a row, 16 threads sharing a dimension's parts.  160 sequences: 1183 items of two
// parts; by blocks alone joining them took 100 us.  Launched with programmatic stream serialisation: it waits for the parts here.
constexpr int PJ_THREADS = 512, PJ_SLICES = PJ_THREADS / 32, PJ_FEW = 16;
template <class T>
__global__ void __launch_bounds__(PJ_THREADS) paged_join_kernel(const __grid_constant__ PagedAttnParams p, int workers, int dp) {
  extern __shared__ __align__(16) int4 joins[];   // [workers]
  __shared__ int found[PJ_THREADS / 32], s_first;
  __shared__ float red[PJ_SLICES][32], red_l[PJ_SLICES], found_m[PJ_SLICES];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
#pragma unroll 4
  for (int i = tid; i < workers; i += PJ_THREADS) joins[i] = p.joins[i];
  __syncthreads();
  // ---- items of few parts: those of workers blockIdx.x, blockIdx.x + gridDim.x, ... ----
  for (int task = warp;; task += PJ_THREADS / 32) {
    const int w = blockIdx.x + task / p.rows * gridDim.x, r = task % p.rows;
    if (w >= workers) break;
    const int4 j = joins[w];
    const int parts = j.z, key_head = j.y / p.parts_per_key, row0 = j.y % p.parts_per_key * PA_ROWS;
    if (parts < 2 || parts > PJ_FEW || row0 + r >= p.group) continue;
    auto place = [&](int i) { return ((long long)(w + i) * 2 + (i == 0 ? 1 : 0)) * p.rows + r; };
    const float m = lane < parts ? p.part_m[place(lane)] : -INFINITY, l = lane < parts ? p.part_l[place(lane)] : 0.f;
    float part[2][8];   // the first two parts come with the maxima
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (32 * k < dp) part[i][k] = p.part_o[place(i) * dp + lane + 32 * k];
    float M = m;
    for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    const float f = ex2(m - (M == -INFINITY ? 0.f : M));
    float L = l * f;
    for (int o = 16; o; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
    float acc[8] = {};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float g = __shfl_sync(0xffffffffu, f, i);
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (32 * k < dp) acc[k] = fmaf(g, part[i][k], acc[k]);
    }
#pragma unroll 2
    for (int i = 2; i < parts; ++i) {
      const float g = __shfl_sync(0xffffffffu, f, i);
      const float *src = p.part_o + place(i) * dp + lane;
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (32 * k < dp) acc[k] = fmaf(g, src[32 * k], acc[k]);
    }
    T *y = static_cast<T *>(p.y) + j.x * p.ldy + (long long)(key_head * p.group + row0 + r) * p.dim + lane;
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (32 * k + lane < p.dim) from_f32(y + 32 * k, M == -INFINITY ? 0.f : acc[k] / L);
  }
  // ---- items of many parts: all blocks look for them and take their tasks in turn ----
  const int chunks = dp / 32, per_item = p.rows * chunks;
  int task = blockIdx.x, seen = 0;   // tasks of the items found so far
  for (int base = 0; base < workers; base += PJ_THREADS) {
    const bool many = base + tid < workers && joins[base + tid].z > PJ_FEW;
    const uint32_t mask = __ballot_sync(0xffffffffu, many);
    if (lane == 0) found[warp] = __popc(mask);
    __syncthreads();
    int before = 0, all = 0;
    for (int w = 0; w < PJ_THREADS / 32; ++w) {
      if (w < warp) before += found[w];
      all += found[w];
    }
    const int mine = many ? before + __popc(mask & ((1u << lane) - 1)) : -1;   // this thread's item among those of the round
    while (task < seen + all * per_item) {
      const int t = task - seen, item = t / per_item, r = t % per_item / chunks, d = t % chunks * 32 + lane;
      if (mine == item) s_first = base + tid;
      __syncthreads();
      const int first = s_first;
      const int4 it = joins[first];
      const int parts = it.z, key_head = it.y / p.parts_per_key, row0 = it.y % p.parts_per_key * PA_ROWS;
      if (row0 + r < p.group) {
        auto place = [&](int i) { return ((long long)(first + i) * 2 + (i == 0 ? 1 : 0)) * p.rows + r; };
        // each warp its slice of the parts, by the slice's own maximum
        const int per = (parts + PJ_SLICES - 1) / PJ_SLICES, i0 = min(parts, warp * per), i1 = min(parts, i0 + per);
        float M = -INFINITY, L = 0.f, o = 0.f;
        for (int at = i0; at < i1; at += 32) {
          const int n = min(32, i1 - at);
          const float m = lane < n ? p.part_m[place(at + lane)] : -INFINITY, l = lane < n ? p.part_l[place(at + lane)] : 0.f;
          float top = fmaxf(m, M);
          for (int s = 16; s; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
          const float off = top == -INFINITY ? 0.f : top, again = ex2(M - off), f = ex2(m - off);
          float sum = l * f;
          for (int s = 16; s; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
          L = L * again + sum;
          o *= again;
          M = top;
#pragma unroll 8
          for (int i = 0; i < n; ++i) o = fmaf(__shfl_sync(0xffffffffu, f, i), p.part_o[place(at + i) * dp + d], o);
        }
        red[warp][lane] = o;
        if (lane == 0) red_l[warp] = L, found_m[warp] = M;
        __syncthreads();
        if (warp == 0) {
          float top = -INFINITY;
          for (int w = 0; w < PJ_SLICES; ++w) top = fmaxf(top, found_m[w]);
          const float off = top == -INFINITY ? 0.f : top;
          o = L = 0.f;
          for (int w = 0; w < PJ_SLICES; ++w) {
            const float f = ex2(found_m[w] - off);
            o = fmaf(f, red[w][lane], o);
            L = fmaf(f, red_l[w], L);
          }
          if (d < p.dim)
            from_f32(static_cast<T *>(p.y) + it.x * p.ldy + (long long)(key_head * p.group + row0 + r) * p.dim + d, top == -INFINITY ? 0.f : o / L);
        }
      }
      __syncthreads();
      task += gridDim.x;
    }
    seen += all * per_item;
    __syncthreads();   // `found` is written again
  }
}

template <class T, int DP, int R>
struct PagedKernel;
template <int DP, int R>
struct PagedKernel<__nv_bfloat16, DP, R> : Bf16Cfg<DP> {
  static constexpr int most_rows = R;
  static constexpr auto fn = paged_mma_kernel<DP>;
};
template <int DP, int R>
struct PagedKernel<float, DP, R> : F32Cfg<DP, R> {
  static constexpr int most_rows = R;
  static constexpr auto fn = paged_fma_kernel<DP, R>;
};

// Calls f(kernel traits, DP) for the instance that serves a type, head size and number of rows.
template <class T, int R, class F>
static int with_dim(int dim, F f) {
  if (dim <= 64) return f(PagedKernel<T, 64, R>(), 64);
  if (dim <= 128) return f(PagedKernel<T, 128, R>(), 128);
  return f(PagedKernel<T, 256, R>(), 256);
}
template <class F>
static int with_kernel(int dtype, int dim, int rows, F f) {
  if (dtype == SOFIE_B200_BF16) return with_dim<__nv_bfloat16, PA_ROWS>(dim, f);
  return rows <= 4 ? with_dim<float, 4>(dim, f) : with_dim<float, PA_ROWS>(dim, f);
}

}  // namespace sb200

using namespace sb200;

struct sofie_b200_paged_attention_plan {
  sofie_b200_ctx *ctx = nullptr;
  sofie_b200_paged_attention_desc d{};
  int grid = 0, workers = 0, rows = 0;             // resident blocks of the whole GPU, their warps; rows of a part
  int64_t off_m = 0, off_l = 0, off_o = 0, bytes = 0;
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
  SB_CUDA(cudaSetDevice(ctx->device));
  int per_sm = 0, warps = 0;
  const int rows = d.heads / d.kv_heads < PA_ROWS ? d.heads / d.kv_heads : PA_ROWS;
  rc = with_kernel(d.dtype, d.head_dim, rows, [&](auto k, int) -> int {
    SB_CUDA(cudaFuncSetAttribute(k.fn, cudaFuncAttributeMaxDynamicSharedMemorySize, k.smem(k.most_rows)));   // for every plan of this kernel
    SB_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, k.fn, k.THREADS, k.smem(rows)));
    warps = k.THREADS / 32;
    return 0;
  });
  if (rc) return rc;
  if (per_sm < 1) return fail(SOFIE_B200_ERR_CUDA, "paged_attention_plan_create: the kernel does not fit an SM");
  auto *p = new (std::nothrow) sofie_b200_paged_attention_plan();
  if (!p) return fail(SOFIE_B200_ERR_INVALID, "paged_attention_plan_create: out of host memory");
  p->ctx = ctx;
  p->d = d;
  p->grid = ctx->sm_count * per_sm;
  p->workers = p->grid * warps;
  p->rows = rows;
  const int64_t dp = d.head_dim <= 64 ? 64 : d.head_dim <= 128 ? 128 : 256, places = 2LL * p->workers;
  auto region = [&](int64_t bytes) { const int64_t o = p->bytes; p->bytes += (bytes + 255) / 256 * 256; return o; };
  region((int64_t)p->workers * sizeof(int4));
  p->off_m = region(places * rows * 4);
  p->off_l = region(places * rows * 4);
  p->off_o = region(places * rows * dp * 4);
  *out = p;
  return 0;
}

int sofie_b200_paged_attention_plan_destroy(sofie_b200_paged_attention_plan *plan) {
  delete plan;
  return 0;
}

const char *sofie_b200_paged_attention_plan_kernel(const sofie_b200_paged_attention_plan *plan) {
  return !plan ? "" : plan->d.dtype == SOFIE_B200_F32 ? "fma" : "mma";
}

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
  if (!workspace || ((uintptr_t)workspace % 256))
    return fail(SOFIE_B200_ERR_INVALID, "paged_attention_enqueue: this plan needs a 256-byte aligned workspace");
  sofie_b200_ctx *ctx = plan->ctx;
  SB_CUDA(cudaSetDevice(ctx->device));
  p.q = q; p.y = y;
  p.cache_k = kv->num_pages ? kv->k : q;   // no page: nothing is read, but the address a copy of no bytes is given should exist
  p.cache_v = kv->num_pages ? kv->v : q;
  p.ldq = d.ldq; p.ldy = d.ldy;
  p.heads = d.heads; p.group = d.heads / d.kv_heads; p.dim = d.head_dim;
  p.parts_per_key = (p.group + PA_ROWS - 1) / PA_ROWS;
  p.items = d.kv_heads * p.parts_per_key;
  p.rows = plan->rows;
  p.scale_log2e = d.scale * 1.4426950408889634f;
  p.status = ctx->d_status;
  char *ws = static_cast<char *>(workspace);
  p.joins = reinterpret_cast<int4 *>(ws);
  p.part_m = reinterpret_cast<float *>(ws + plan->off_m);
  p.part_l = reinterpret_cast<float *>(ws + plan->off_l);
  p.part_o = reinterpret_cast<float *>(ws + plan->off_o);
  return with_kernel(d.dtype, d.head_dim, p.rows, [&](auto k, int dp) -> int {
    // never more blocks than the longest lengths that the table allows could fill
    constexpr int warps = k.THREADS / 32;
    const int64_t room = (int64_t)p.kv.table_width * p.kv.page_size;
    const int64_t most = ((room + PA_UNIT - 1) / PA_UNIT + ITEM_COST) * p.items;   // slots of one sequence, below 2^28 * 2^21
    const int64_t slots = most >= (int64_t)plan->workers * PA_LEAST ? (int64_t)plan->workers * PA_LEAST : most * p.kv.batch;
    const int64_t want = (slots / PA_LEAST + warps) / warps;
    const int grid = want > plan->grid ? plan->grid : (int)want;
    k.fn<<<(unsigned)grid, k.THREADS, k.smem(p.rows), ctx->stream>>>(p);
    SB_CUDA(cudaGetLastError());
    ctx->launches++;
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    const int64_t tasks = (int64_t)grid * warps * p.rows * (dp / 32);
    cfg.gridDim = dim3((unsigned)(tasks < ctx->sm_count ? tasks : ctx->sm_count));
    cfg.blockDim = dim3(PJ_THREADS);
    cfg.dynamicSmemBytes = (size_t)grid * warps * sizeof(int4);   // below 48 KB: workers are what an SM keeps, 8 at most
    cfg.stream = ctx->stream;
    cfg.attrs = &early;
    cfg.numAttrs = 1;
    if (d.dtype == SOFIE_B200_F32) SB_CUDA(cudaLaunchKernelEx(&cfg, paged_join_kernel<float>, p, grid * warps, dp));
    else SB_CUDA(cudaLaunchKernelEx(&cfg, paged_join_kernel<__nv_bfloat16>, p, grid * warps, dp));
    ctx->launches++;
    return 0;
  });
}

}  // extern "C"
