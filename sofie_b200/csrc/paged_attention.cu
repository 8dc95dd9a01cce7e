// Attention of one new token per sequence over a paged key-value cache:
//     y[b, h] = sum_j softmax_j(scale q[b, h] . k[j, h / g]) v[j, h / g],   j < seq_lens[b],   g = heads / kv_heads.
// Each key and value is read once for the g query heads that share it, so the kernel is bound by HBM: 2 D elements per token and
// key head for 4 g D operations.
//
// Split.  One sequence may be the whole batch and 65,000 tokens long, or a batch may hold hundreds of very different lengths.
// The tokens of all sequences and key heads are one row of units of 64 (bf16) or 32 (fp32) keys, cut into equal shares, one
// per resident block (paged.cuh: split_at).  A share may end inside a sequence; the parts of such a sequence (running
// maximum, sum, unnormalised result, all fp32) meet in the workspace and a second kernel joins them in the order of the keys, so
// results do not depend on timing.  Lengths are read on the device: a captured call is replayed for any other lengths.
#include <math.h>
#include <new>

#include "generate.cuh"
#include "ptx.cuh"

namespace sb200 {
using namespace ptx;

constexpr int PA_THREADS = 128;   // four warps
constexpr int PA_ROWS = 16;       // query heads of one block's item: the rows of one mma tile
constexpr int PA_LEAST = 2;       // units that are worth a block of their own

struct PagedAttnParams {
  PagedView kv;
  const void *q, *cache_k, *cache_v;
  void *y;
  long long ldq, ldy;
  int heads, group, dim;      // group = heads / kv_heads
  int items, blocks_per_key;  // items of a sequence = kv_heads * blocks_per_key; blocks_per_key = ceil(group / 16)
  float scale_log2e;
  int *status;
  // workspace
  int4 *joins;                // [grid] {sequence, item, parts, 0}: the item that begins in this block and ends in a later one
  float *part_m, *part_l;     // [grid * 2][16]
  float *part_o;              // [grid * 2][16][DP]
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

// Where a block stands in the row of units.
struct Cursor {
  int b, item, unit, units, len;   // sequence, item of the sequence, unit of the item; units and tokens of the sequence
};

template <int UNIT>
__device__ __forceinline__ void cursor_sequence(const PagedView &kv, Cursor &c) {   // from sequence c.b on, the first that has tokens
  bool bad = false;
  while (c.b < kv.batch && (c.len = paged_len(kv, c.b, &bad)) == 0) ++c.b;
  c.units = c.b < kv.batch ? units_of(c.len, UNIT) : 0;
}
template <int UNIT>
__device__ __forceinline__ void cursor_next(const PagedView &kv, int items, Cursor &c) {
  if (++c.unit < c.units) return;
  c.unit = 0;
  if (++c.item < items) return;
  c.item = 0;
  ++c.b;
  cursor_sequence<UNIT>(kv, c);
}

struct Share {
  long long units, begin, end;   // of the batch; of this block
  int blocks;                    // that have work
  Cursor at;
};

// Every block sums up the lengths by itself (they are few, and in L2) and finds its share.  All 128 threads call it.
template <int UNIT>
__device__ __forceinline__ void find_share(const PagedAttnParams &p, Share &s) {
  __shared__ long long warp_sum[PA_THREADS / 32];
  __shared__ Cursor s_at;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (p.kv.batch + PA_THREADS - 1) / PA_THREADS;   // a thread's sequences lie together
  const int b0 = min(p.kv.batch, tid * per), b1 = min(p.kv.batch, b0 + per);
  long long mine = 0;
  bool bad = false;
  for (int b = b0; b < b1; ++b) mine += (long long)units_of(paged_len(p.kv, b, &bad), UNIT) * p.items;
  if (bad) report(p.status, DEV_BAD_INDEX);
  long long incl = mine;
  for (int o = 1; o < 32; o <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += x;
  }
  if (lane == 31) warp_sum[warp] = incl;
  __syncthreads();
  long long before = incl - mine, total = 0;
  for (int w = 0; w < PA_THREADS / 32; ++w) {
    if (w < warp) before += warp_sum[w];
    total += warp_sum[w];
  }
  s.units = total;
  s.blocks = split_blocks(total, gridDim.x, PA_LEAST);
  const int c = blockIdx.x;
  s.begin = c < s.blocks ? split_at(total, s.blocks, c) : total;
  s.end = c < s.blocks ? split_at(total, s.blocks, c + 1) : total;
  if (s.begin < s.end && s.begin >= before && s.begin < before + mine) {   // one thread
    long long at = before;
    Cursor k{};
    for (int b = b0; b < b1; ++b) {
      const int n = paged_len(p.kv, b, &bad), units = units_of(n, UNIT);
      const long long all = (long long)units * p.items;
      if (s.begin < at + all) {
        const long long r = s.begin - at;
        k.b = b; k.len = n; k.units = units;
        k.item = (int)(r / units);
        k.unit = (int)(r % units);
        break;
      }
      at += all;
    }
    s_at = k;
  }
  __syncthreads();
  s.at = s_at;
}

// Padding rows: sequences without tokens get zeros.
template <class T>
__device__ __forceinline__ void zero_empty(const PagedAttnParams &p) {
  bool bad = false;
  for (int b = blockIdx.x; b < p.kv.batch; b += gridDim.x)
    if (paged_len(p.kv, b, &bad) == 0) {
      T *y = static_cast<T *>(p.y) + b * p.ldy;
      for (int i = threadIdx.x; i < p.heads * p.dim; i += PA_THREADS) from_f32(y + i, 0.f);
    }
}

// The item that the cursor's segment [unit, unit + n) is part of: does it begin here, does it end here, which slot takes the part.
__device__ __forceinline__ void announce_join(const PagedAttnParams &p, const Share &s, const Cursor &c, long long item_end) {
  p.joins[blockIdx.x] = make_int4(c.b, c.item, split_last(s.units, s.blocks, item_end) - (int)blockIdx.x + 1, 0);
}

template <int DP>
struct Bf16Cfg {
  static constexpr int UNIT = 64, STAGES = 3;
  static constexpr int TILE = 16 * DP * 2;                     // one warp's 16 keys (or values)
  static constexpr int RING = 4 * STAGES * 2 * TILE;
  static constexpr int MERGE = 2 * PA_ROWS * DP * 4;
  static constexpr int SMEM = RING + MERGE + 4 * PA_ROWS * 8;
};

// bf16.  A unit is 64 keys, 16 to a warp.  Each warp runs by itself down the block's share: its own ring of three stages filled
// by cp.async (keys and values of 16 tokens, found through the block table one step ahead), scores and weighted values on
// mma.m16n8k16 with the 16 rows = query heads of the group (rows past the group cost nothing that HBM would not wait for), its own
// running maximum and sum.  The weights of the second product are split into two bf16 terms, high + low (error 2^-16 instead
// of 2^-8): the tensor cores have the time.  The warps meet once per item.
template <int DP>
__global__ void __launch_bounds__(PA_THREADS) paged_mma_kernel(const __grid_constant__ PagedAttnParams p) {
  using Cfg = Bf16Cfg<DP>;
  extern __shared__ __align__(128) uint8_t smem[];
  asm volatile("griddepcontrol.launch_dependents;");
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  typedef __nv_bfloat16 T;
  zero_empty<T>(p);
  Share sh;
  find_share<Cfg::UNIT>(p, sh);
  if (tid == 0) p.joins[blockIdx.x] = make_int4(0, 0, 0, 0);
  const long long steps = sh.end - sh.begin;
  if (steps <= 0) return;
  const uint32_t ring = smem_u32(smem) + warp * (Cfg::STAGES * 2 * Cfg::TILE);
  float *merge = reinterpret_cast<float *>(smem + Cfg::RING);
  float *merge_m = reinterpret_cast<float *>(smem + Cfg::RING + Cfg::MERGE), *merge_l = merge_m + 4 * PA_ROWS;
  const T *cache_k = static_cast<const T *>(p.cache_k), *cache_v = static_cast<const T *>(p.cache_v);

  // ---- loads: cursor `ld`, one step ahead of it the row offsets of this warp's 16 keys (lane r < 16: key r) ----
  Cursor ld = sh.at;
  long long row = -1;
  bool bad = false;
  auto look_up = [&]() {
    row = -1;
    const int key = ld.unit * Cfg::UNIT + warp * 16 + lane;
    if (lane < 16 && key < ld.len) {
      row = paged_row(p.kv, ld.b, key);
      if (row < 0) bad = true;
      else row += (long long)(ld.item / p.blocks_per_key) * p.kv.head_stride;
    }
  };
  uint32_t valid_ring[Cfg::STAGES];
  auto issue = [&](uint32_t stage) -> uint32_t {
    const uint32_t dk = ring + stage * (2 * Cfg::TILE), dv = dk + Cfg::TILE;
    constexpr int CH = DP / 8;   // 16-byte pieces of a row
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) {
      const int flat = i * 32 + lane, r = flat / CH, c = flat % CH;
      const long long off = __shfl_sync(0xffffffffu, row, r);
      const bool there = off >= 0 && c * 8 < p.dim;
      const long long e = there ? off + c * 8 : 0;
      const uint32_t d = r * (DP * 2) + ((c ^ (r & 7)) << 4);
      cp_async_16(dk + d, cache_k + e, there);
      cp_async_16(dv + d, cache_v + e, there);
    }
    return __ballot_sync(0xffffffffu, row >= 0);
  };
  long long issued = 0;
  look_up();
#pragma unroll
  for (int s = 0; s < Cfg::STAGES - 1; ++s) {
    valid_ring[s] = 0;
    if (issued < steps) {
      valid_ring[s] = issue(s);
      ++issued;
      cursor_next<Cfg::UNIT>(p.kv, p.items, ld);
      if (issued < steps) look_up();
    }
    cp_async_commit();
  }

  Cursor at = sh.at;
  long long done = 0;
  uint32_t stage = 0;
  while (done < steps) {
    // ---- one segment: the units of one item that lie in this block's share ----
    const int first_unit = at.unit;
    const int n = (int)min((long long)(at.units - at.unit), steps - done);
    const int key_head = at.item / p.blocks_per_key, row0 = at.item % p.blocks_per_key * PA_ROWS;
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
      // refill the stage that the previous step has read
      uint32_t fresh = 0;
      const uint32_t into = stage == 0 ? Cfg::STAGES - 1 : stage - 1;
      __syncwarp();
      if (issued < steps) {
        fresh = issue(into);
        ++issued;
        cursor_next<Cfg::UNIT>(p.kv, p.items, ld);
        if (issued < steps) look_up();
      }
      cp_async_commit();
      cp_async_wait<Cfg::STAGES - 1>();
      __syncwarp();
      const uint32_t valid = valid_ring[0];
#pragma unroll
      for (int i = 0; i + 1 < Cfg::STAGES - 1; ++i) valid_ring[i] = valid_ring[i + 1];
      valid_ring[Cfg::STAGES - 2] = fresh;
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
      x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 1));
      x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 1));
      x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 2));
      x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 2));
      // The reference maximum moves only when a new one is 2^8 above it: weights stay below 2^8, and most steps rescale nothing.
      const bool up0 = x0 > m0 + 8.f, up1 = x1 > m1 + 8.f;
      if (__any_sync(0xffffffffu, up0 || up1)) {
        const float n0 = up0 ? x0 : m0, n1 = up1 ? x1 : m1;
        const float f0 = up0 ? ex2(m0 - n0) : 1.f, f1 = up1 ? ex2(m1 - n1) : 1.f;
        m0 = n0;
        m1 = n1;
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
          const __nv_bfloat162 h = __floats2bfloat162_rn(e0, e1);
          const __nv_bfloat162 r = __floats2bfloat162_rn(e0 - __low2float(h), e1 - __high2float(h));
          hi[t * 2 + half] = *reinterpret_cast<const uint32_t *>(&h);
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

    // ---- the four warps' parts of the segment, in their order: 2 and 3 onto 0 and 1, then 1 onto 0 ----
    l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
    l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
    if ((lane & 3) == 0) {
      merge_m[warp * PA_ROWS + r0] = m0;
      merge_m[warp * PA_ROWS + r1] = m1;
      merge_l[warp * PA_ROWS + r0] = l0;
      merge_l[warp * PA_ROWS + r1] = l1;
    }
    __syncthreads();
    float M0 = -INFINITY, M1 = -INFINITY, L0 = 0.f, L1 = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      M0 = fmaxf(M0, merge_m[w * PA_ROWS + r0]);
      M1 = fmaxf(M1, merge_m[w * PA_ROWS + r1]);
    }
    const float B0 = M0 == -INFINITY ? 0.f : M0, B1 = M1 == -INFINITY ? 0.f : M1;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      L0 += merge_l[w * PA_ROWS + r0] * ex2(merge_m[w * PA_ROWS + r0] - B0);
      L1 += merge_l[w * PA_ROWS + r1] * ex2(merge_m[w * PA_ROWS + r1] - B1);
    }
    const float f0 = ex2(m0 - B0), f1 = ex2(m1 - B1);
#pragma unroll
    for (int i = 0; i < DP / 8; ++i) {
      o[i][0] *= f0; o[i][1] *= f0;
      o[i][2] *= f1; o[i][3] *= f1;
    }
    float4 *mb = reinterpret_cast<float4 *>(merge) + (warp & 1) * (PA_ROWS * DP / 4);   // [DP / 8][32 lanes]: each lane meets its own
    if (warp >= 2)
#pragma unroll
      for (int i = 0; i < DP / 8; ++i) mb[i * 32 + lane] = make_float4(o[i][0], o[i][1], o[i][2], o[i][3]);
    __syncthreads();
    if (warp < 2) {
#pragma unroll
      for (int i = 0; i < DP / 8; ++i) {
        const float4 x = mb[i * 32 + lane];
        o[i][0] += x.x; o[i][1] += x.y; o[i][2] += x.z; o[i][3] += x.w;
      }
      if (warp == 1)
#pragma unroll
        for (int i = 0; i < DP / 8; ++i) mb[i * 32 + lane] = make_float4(o[i][0], o[i][1], o[i][2], o[i][3]);
    }
    __syncthreads();
    if (warp == 0) {
      const float4 *other = reinterpret_cast<const float4 *>(merge) + PA_ROWS * DP / 4;
#pragma unroll
      for (int i = 0; i < DP / 8; ++i) {
        const float4 x = other[i * 32 + lane];
        o[i][0] += x.x; o[i][1] += x.y; o[i][2] += x.z; o[i][3] += x.w;
      }
      const bool begins = first_unit == 0, ends = first_unit + n == at.units;
      if (begins && ends) {
        T *y = static_cast<T *>(p.y) + at.b * p.ldy + (long long)(key_head * p.group + row0) * p.dim;
        const float i0 = M0 == -INFINITY ? 0.f : 1.f / L0, i1 = M1 == -INFINITY ? 0.f : 1.f / L1;
#pragma unroll
        for (int i = 0; i < DP / 8; ++i) {
          const int d = i * 8 + (lane & 3) * 2;
          if (d < p.dim) {
            if (r0 < rows) *reinterpret_cast<__nv_bfloat162 *>(y + (long long)r0 * p.dim + d) = __floats2bfloat162_rn(o[i][0] * i0, o[i][1] * i0);
            if (r1 < rows) *reinterpret_cast<__nv_bfloat162 *>(y + (long long)r1 * p.dim + d) = __floats2bfloat162_rn(o[i][2] * i1, o[i][3] * i1);
          }
        }
      } else {
        const long long slot = (long long)blockIdx.x * 2 + (begins ? 1 : 0);
        float *po = p.part_o + slot * PA_ROWS * DP;
        if ((lane & 3) == 0) {
          p.part_m[slot * PA_ROWS + r0] = M0;
          p.part_m[slot * PA_ROWS + r1] = M1;
          p.part_l[slot * PA_ROWS + r0] = L0;
          p.part_l[slot * PA_ROWS + r1] = L1;
        }
#pragma unroll
        for (int i = 0; i < DP / 8; ++i) {
          const int d = i * 8 + (lane & 3) * 2;
          if (r0 < rows) *reinterpret_cast<float2 *>(po + r0 * DP + d) = make_float2(o[i][0], o[i][1]);
          if (r1 < rows) *reinterpret_cast<float2 *>(po + r1 * DP + d) = make_float2(o[i][2], o[i][3]);
        }
        if (begins && lane == 0) announce_join(p, sh, at, sh.begin + done + at.units);
      }
    }
    // the merge buffers are written again after the next item's own first barrier, which warp 0 reaches after reading them
    done += n;
    at.unit += n - 1;
    cursor_next<Cfg::UNIT>(p.kv, p.items, at);
  }
  if (bad) report(p.status, DEV_BAD_INDEX);
}

template <int DP>
struct F32Cfg {
  static constexpr int UNIT = 32, STAGES = 2;
  static constexpr int TILE = 32 * DP * 4;                     // 32 keys (or values)
  static constexpr int RING = STAGES * 2 * TILE;
  static constexpr int MERGE = 2 * PA_ROWS * DP * 4;
  static constexpr int Q = PA_ROWS * DP * 4;
  static constexpr int P = PA_ROWS * 32 * 4;
  static constexpr int SMEM = RING + MERGE + Q + P + (PA_ROWS + 2 * PA_ROWS) * 4 + STAGES * 32 * 4;
};

// fp32, on the CUDA cores.  A unit is a tile of 32 keys that the block works on together: scores with a lane per key and a warp per
// head (heads w, w + 4, ...), weights through shared memory, weighted values with a warp per 8 keys and a lane per 4 dimensions.
template <int DP>
__global__ void __launch_bounds__(PA_THREADS) paged_f32_kernel(const __grid_constant__ PagedAttnParams p) {
  using Cfg = F32Cfg<DP>;
  extern __shared__ __align__(128) uint8_t smem[];
  asm volatile("griddepcontrol.launch_dependents;");
  constexpr int CH = DP / 4;                         // 16-byte pieces of a row
  constexpr int KPL = CH >= 32 ? 1 : 32 / CH;        // keys side by side in a warp's weighted values
  constexpr int VPL = CH >= 32 ? CH / 32 : 1;        // pieces of a row per lane
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  zero_empty<float>(p);
  Share sh;
  find_share<Cfg::UNIT>(p, sh);
  if (tid == 0) p.joins[blockIdx.x] = make_int4(0, 0, 0, 0);
  const long long steps = sh.end - sh.begin;
  if (steps <= 0) return;
  const uint32_t ring = smem_u32(smem);
  float4 *merge = reinterpret_cast<float4 *>(smem + Cfg::RING);
  float *sq = reinterpret_cast<float *>(smem + Cfg::RING + Cfg::MERGE);        // [16][DP], scaled
  float *sp = sq + PA_ROWS * DP;                                               // [16][32] weights
  float *sf = sp + PA_ROWS * 32;                                               // [16] rescaling factors of this step
  float *sm = sf + PA_ROWS, *sl = sm + PA_ROWS;                                // [16] maxima, sums at an item's end
  int *on = reinterpret_cast<int *>(sl + PA_ROWS);                             // [STAGES][32] key is there
  const float *cache_k = static_cast<const float *>(p.cache_k), *cache_v = static_cast<const float *>(p.cache_v);

  Cursor ld = sh.at;
  long long row = -1;   // lane r < 8: key warp * 8 + r of the next tile
  bool bad = false;
  auto look_up = [&]() {
    row = -1;
    const int key = ld.unit * Cfg::UNIT + warp * 8 + lane;
    if (lane < 8 && key < ld.len) {
      row = paged_row(p.kv, ld.b, key);
      if (row < 0) bad = true;
      else row += (long long)(ld.item / p.blocks_per_key) * p.kv.head_stride;
    }
  };
  auto issue = [&](uint32_t stage) {
    const uint32_t dk = ring + stage * (2 * Cfg::TILE), dv = dk + Cfg::TILE;
    if (lane < 8) on[stage * 32 + warp * 8 + lane] = row >= 0;
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) {
      const int flat = i * 32 + lane, r = flat / CH, c = flat % CH, key = warp * 8 + r;
      const long long off = __shfl_sync(0xffffffffu, row, r);
      const bool there = off >= 0 && c * 4 < p.dim;
      const long long e = there ? off + c * 4 : 0;
      const uint32_t d = key * (DP * 4) + ((c ^ (key & 7)) << 4);
      cp_async_16(dk + d, cache_k + e, there);
      cp_async_16(dv + d, cache_v + e, there);
    }
  };
  long long issued = 0;
  look_up();
  issue(0);
  ++issued;
  cursor_next<Cfg::UNIT>(p.kv, p.items, ld);
  if (issued < steps) look_up();
  cp_async_commit();

  Cursor at = sh.at;
  long long done = 0;
  uint32_t stage = 0;
  while (done < steps) {
    const int first_unit = at.unit;
    const int n = (int)min((long long)(at.units - at.unit), steps - done);
    const int key_head = at.item / p.blocks_per_key, row0 = at.item % p.blocks_per_key * PA_ROWS;
    const int rows = min(PA_ROWS, p.group - row0);
    const float *q = static_cast<const float *>(p.q) + at.b * p.ldq + (long long)(key_head * p.group + row0) * p.dim;
    for (int i = tid; i < rows * DP; i += PA_THREADS) {
      const int r = i / DP, d = i % DP;
      sq[i] = d < p.dim ? q[(long long)r * p.dim + d] * p.scale_log2e : 0.f;
    }
    float4 acc[PA_ROWS][VPL];
#pragma unroll
    for (int h = 0; h < PA_ROWS; ++h)
#pragma unroll
      for (int v = 0; v < VPL; ++v) acc[h][v] = make_float4(0.f, 0.f, 0.f, 0.f);
    float m[4], l[4];   // of heads warp, warp + 4, ...: the maximum of the head, this lane's share of its sum
#pragma unroll
    for (int j = 0; j < 4; ++j) m[j] = -INFINITY, l[j] = 0.f;

    for (int u = 0; u < n; ++u) {
      cp_async_wait<0>();
      __syncthreads();   // the tile is there; everybody has left the other stage and the weights
      if (issued < steps) {
        issue(stage ^ 1);
        ++issued;
        cursor_next<Cfg::UNIT>(p.kv, p.items, ld);
        if (issued < steps) look_up();
      }
      cp_async_commit();
      const float4 *tk = reinterpret_cast<const float4 *>(smem + stage * (2 * Cfg::TILE)), *tv = tk + Cfg::TILE / 16;
      const bool there = on[stage * 32 + lane] != 0;
      const bool any = __any_sync(0xffffffffu, there);
      stage ^= 1;
      // ---- scores ----
      if (warp < rows) {
        float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int c = 0; c < CH; ++c) {
          const float4 k = tk[lane * CH + (c ^ (lane & 7))];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (warp + 4 * j < rows) {
              const float4 x = *reinterpret_cast<const float4 *>(sq + (warp + 4 * j) * DP + c * 4);
              s[j] = fmaf(k.x, x.x, fmaf(k.y, x.y, fmaf(k.z, x.z, fmaf(k.w, x.w, s[j]))));
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int h = warp + 4 * j;
          if (h < rows) {
            const float x = there ? s[j] : -INFINITY;
            float top = x;
            for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            if (any) top = fmaxf(top, -3.0e38f);
            float f = 1.f;
            if (top > m[j]) {
              f = exp2f(m[j] - top);
              m[j] = top;
              l[j] *= f;
            }
            const float e = any ? exp2f(x - m[j]) : 0.f;
            l[j] += e;
            sp[h * 32 + lane] = e;
            if (lane == 0) sf[h] = f;
          }
        }
      }
      __syncthreads();
      // ---- weighted values: keys 8 warp .. 8 warp + 7 ----
#pragma unroll
      for (int h = 0; h < PA_ROWS; ++h)
        if (h < rows) {
          const float f = sf[h];
          if (f != 1.f)
#pragma unroll
            for (int v = 0; v < VPL; ++v) { acc[h][v].x *= f; acc[h][v].y *= f; acc[h][v].z *= f; acc[h][v].w *= f; }
        }
#pragma unroll
      for (int k0 = 0; k0 < 8; k0 += 4 * KPL < 8 ? 4 * KPL : 8) {
        constexpr int STEPS = 4 * KPL < 8 ? 4 : 8 / KPL;
        float4 val[STEPS][VPL];
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
          const int key = warp * 8 + k0 + i * KPL + (KPL > 1 ? lane / CH : 0);
#pragma unroll
          for (int v = 0; v < VPL; ++v) val[i][v] = tv[key * CH + ((((KPL > 1 ? lane % CH : lane) + 32 * v)) ^ (key & 7))];
        }
#pragma unroll
        for (int h = 0; h < PA_ROWS; ++h)
          if (h < rows) {
#pragma unroll
            for (int i = 0; i < STEPS; ++i) {
              const float e = sp[h * 32 + warp * 8 + k0 + i * KPL + (KPL > 1 ? lane / CH : 0)];
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
    }

    // ---- sums over the lanes; the warps' values in their order ----
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int h = warp + 4 * j;
      if (h < rows) {
        for (int o = 16; o; o >>= 1) l[j] += __shfl_xor_sync(0xffffffffu, l[j], o);
        if (lane == 0) sm[h] = m[j], sl[h] = l[j];
      }
    }
    if (KPL > 1)
#pragma unroll
      for (int h = 0; h < PA_ROWS; ++h)
        if (h < rows)
#pragma unroll
          for (int v = 0; v < VPL; ++v)
            for (int o = CH; o < 32; o <<= 1) {
              acc[h][v].x += __shfl_xor_sync(0xffffffffu, acc[h][v].x, o);
              acc[h][v].y += __shfl_xor_sync(0xffffffffu, acc[h][v].y, o);
              acc[h][v].z += __shfl_xor_sync(0xffffffffu, acc[h][v].z, o);
              acc[h][v].w += __shfl_xor_sync(0xffffffffu, acc[h][v].w, o);
            }
    float4 *mb = merge + (warp & 1) * (PA_ROWS * CH);
    const int col = KPL > 1 ? lane % CH : lane;
    const bool writes = KPL == 1 || lane < CH;
    if (warp >= 2 && writes)
#pragma unroll
      for (int h = 0; h < PA_ROWS; ++h)
        if (h < rows)
#pragma unroll
          for (int v = 0; v < VPL; ++v) mb[h * CH + col + 32 * v] = acc[h][v];
    __syncthreads();
    if (warp < 2 && writes)
#pragma unroll
      for (int h = 0; h < PA_ROWS; ++h)
        if (h < rows)
#pragma unroll
          for (int v = 0; v < VPL; ++v) {
            const float4 x = mb[h * CH + col + 32 * v];
            acc[h][v].x += x.x; acc[h][v].y += x.y; acc[h][v].z += x.z; acc[h][v].w += x.w;
            if (warp == 1) mb[h * CH + col + 32 * v] = acc[h][v];
          }
    __syncthreads();
    if (warp == 0) {
      const bool begins = first_unit == 0, ends = first_unit + n == at.units;
      const long long slot = (long long)blockIdx.x * 2 + (begins ? 1 : 0);
      float *y = static_cast<float *>(p.y) + at.b * p.ldy + (long long)(key_head * p.group + row0) * p.dim;
      const float4 *other = merge + PA_ROWS * CH;
#pragma unroll
      for (int h = 0; h < PA_ROWS; ++h)
        if (h < rows) {
          const float M = sm[h], L = sl[h];
          const float inv = M == -INFINITY ? 0.f : 1.f / L;
          if (writes)
#pragma unroll
            for (int v = 0; v < VPL; ++v) {
              const float4 x = other[h * CH + col + 32 * v];
              float4 r = make_float4(acc[h][v].x + x.x, acc[h][v].y + x.y, acc[h][v].z + x.z, acc[h][v].w + x.w);
              const int d = (col + 32 * v) * 4;
              if (begins && ends) {
                if (d < p.dim) *reinterpret_cast<float4 *>(y + (long long)h * p.dim + d) = make_float4(r.x * inv, r.y * inv, r.z * inv, r.w * inv);
              } else {
                *reinterpret_cast<float4 *>(p.part_o + (slot * PA_ROWS + h) * DP + d) = r;
              }
            }
          if (!(begins && ends) && lane == 0) {
            p.part_m[slot * PA_ROWS + h] = M;
            p.part_l[slot * PA_ROWS + h] = L;
          }
        }
      if (begins && !ends && lane == 0) announce_join(p, sh, at, sh.begin + done + at.units);
    }
    __syncthreads();   // the next item's queries, maxima and parts go where this one's were read
    done += n;
    at.unit += n - 1;
    cursor_next<Cfg::UNIT>(p.kv, p.items, at);
  }
  if (bad) report(p.status, DEV_BAD_INDEX);
}

// Joins the parts of the item that began in block blockIdx.x: slot 1 of that block, slot 0 of the following ones.  One row per
// blockIdx.y, a thread per dimension.  Launched with programmatic stream serialisation: it waits for the parts here.
template <class T>
__global__ void paged_join_kernel(const __grid_constant__ PagedAttnParams p, int dp) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4 j = p.joins[blockIdx.x];
  const int parts = j.z;
  if (parts <= 1) return;
  const int key_head = j.y / p.blocks_per_key, row0 = j.y % p.blocks_per_key * PA_ROWS;
  const int r = blockIdx.y, d = threadIdx.x;
  if (row0 + r >= p.group) return;
  auto slot = [&](int i) { return ((long long)(blockIdx.x + i) * 2 + (i == 0 ? 1 : 0)) * PA_ROWS + r; };
  float M = -INFINITY;
  for (int i = 0; i < parts; ++i) M = fmaxf(M, p.part_m[slot(i)]);
  const float base = M == -INFINITY ? 0.f : M;
  float L = 0.f, o = 0.f;
#pragma unroll 4
  for (int i = 0; i < parts; ++i) {
    const long long s = slot(i);
    const float f = ex2(p.part_m[s] - base);
    L += p.part_l[s] * f;
    o += p.part_o[s * dp + d] * f;
  }
  if (d < p.dim)
    from_f32(static_cast<T *>(p.y) + j.x * p.ldy + (long long)(key_head * p.group + row0 + r) * p.dim + d, M == -INFINITY ? 0.f : o / L);
}

template <class T, int DP>
struct PagedKernel;
template <int DP>
struct PagedKernel<__nv_bfloat16, DP> {
  static constexpr int smem = Bf16Cfg<DP>::SMEM, unit = Bf16Cfg<DP>::UNIT;
  static constexpr auto fn = paged_mma_kernel<DP>;
};
template <int DP>
struct PagedKernel<float, DP> {
  static constexpr int smem = F32Cfg<DP>::SMEM, unit = F32Cfg<DP>::UNIT;
  static constexpr auto fn = paged_f32_kernel<DP>;
};

// Calls f(kernel traits, DP) for the instance that serves a type and head size.
template <class T, class F>
static int with_dim(int dim, F f) {
  if (dim <= 64) return f(PagedKernel<T, 64>(), 64);
  if (dim <= 128) return f(PagedKernel<T, 128>(), 128);
  return f(PagedKernel<T, 256>(), 256);
}
template <class F>
static int with_kernel(int dtype, int dim, F f) {
  return dtype == SOFIE_B200_F32 ? with_dim<float>(dim, f) : with_dim<__nv_bfloat16>(dim, f);
}

}  // namespace sb200

using namespace sb200;

struct sofie_b200_paged_attention_plan {
  sofie_b200_ctx *ctx = nullptr;
  sofie_b200_paged_attention_desc d{};
  int grid = 0;                                    // resident blocks of the whole GPU
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
  int per_sm = 0;
  rc = with_kernel(d.dtype, d.head_dim, [&](auto k, int) -> int {
    SB_CUDA(cudaFuncSetAttribute(k.fn, cudaFuncAttributeMaxDynamicSharedMemorySize, k.smem));
    SB_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, k.fn, PA_THREADS, k.smem));
    return 0;
  });
  if (rc) return rc;
  if (per_sm < 1) return fail(SOFIE_B200_ERR_CUDA, "paged_attention_plan_create: the kernel does not fit an SM");
  auto *p = new (std::nothrow) sofie_b200_paged_attention_plan();
  if (!p) return fail(SOFIE_B200_ERR_INVALID, "paged_attention_plan_create: out of host memory");
  p->ctx = ctx;
  p->d = d;
  p->grid = ctx->sm_count * per_sm;
  const int64_t dp = d.head_dim <= 64 ? 64 : d.head_dim <= 128 ? 128 : 256, slots = 2LL * p->grid;
  auto region = [&](int64_t bytes) { const int64_t o = p->bytes; p->bytes += (bytes + 255) / 256 * 256; return o; };
  region((int64_t)p->grid * sizeof(int4));
  p->off_m = region(slots * PA_ROWS * 4);
  p->off_l = region(slots * PA_ROWS * 4);
  p->off_o = region(slots * PA_ROWS * dp * 4);
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
  p.blocks_per_key = (p.group + PA_ROWS - 1) / PA_ROWS;
  p.items = d.kv_heads * p.blocks_per_key;
  p.scale_log2e = d.scale * 1.4426950408889634f;
  p.status = ctx->d_status;
  char *ws = static_cast<char *>(workspace);
  p.joins = reinterpret_cast<int4 *>(ws);
  p.part_m = reinterpret_cast<float *>(ws + plan->off_m);
  p.part_l = reinterpret_cast<float *>(ws + plan->off_l);
  p.part_o = reinterpret_cast<float *>(ws + plan->off_o);
  return with_kernel(d.dtype, d.head_dim, [&](auto k, int dp) -> int {
    // never more blocks than the longest lengths that the table allows could fill
    const int64_t room = (int64_t)p.kv.table_width * p.kv.page_size;
    const int64_t most = (room + k.unit - 1) / k.unit * p.items;   // units of one sequence, below 2^31 * 2^12
    const int64_t want = most >= plan->grid ? plan->grid : most * p.kv.batch;
    const unsigned grid = (unsigned)(want < 1 ? 1 : want > plan->grid ? plan->grid : want);
    k.fn<<<grid, PA_THREADS, k.smem, ctx->stream>>>(p);
    SB_CUDA(cudaGetLastError());
    ctx->launches++;
    if (grid == 1) return 0;   // one block has whole items only
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid, (unsigned)(p.group < PA_ROWS ? p.group : PA_ROWS));
    cfg.blockDim = dim3((unsigned)dp);
    cfg.stream = ctx->stream;
    cfg.attrs = &early;
    cfg.numAttrs = 1;
    if (d.dtype == SOFIE_B200_F32) SB_CUDA(cudaLaunchKernelEx(&cfg, paged_join_kernel<float>, p, dp));
    else SB_CUDA(cudaLaunchKernelEx(&cfg, paged_join_kernel<__nv_bfloat16>, p, dp));
    ctx->launches++;
    return 0;
  });
}

}  // extern "C"
