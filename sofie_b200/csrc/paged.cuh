// Index arithmetic of the generation operators (append to a paged cache, attention over packed prompts, attention over the
// cache).  Plain integer functions, for the kernels and for a host compiler alike: tests/test_generate.py builds this
// file with g++ and runs every function over hostile tables and lengths, because an index that leaves its buffer must be
// found there and not on a GPU.
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define SB_HD __host__ __device__ __forceinline__
#else
#define SB_HD inline
#endif

namespace sb200 {

// A paged cache and its sequences (sofie_b200_paged_kv with the defaults filled in).
struct PagedView {
  const int32_t *table;      // [batch, table_width], rows table_pitch apart
  const int32_t *lens;       // [batch]
  long long table_pitch;
  long long page_stride, token_stride, head_stride;   // elements
  int batch, num_pages, table_width, page_size;
};

// Element offset of (position pos of sequence b, head 0) in the cache, or -1 when the position has no page or the page does not
// exist.  64-bit throughout: a cache of 2^31 elements is 4 GB of bf16.
SB_HD long long paged_row(const PagedView &c, int b, int pos) {
  if (pos < 0) return -1;
  const int page_index = pos / c.page_size;
  if (page_index >= c.table_width) return -1;
  const int page = c.table[(long long)b * c.table_pitch + page_index];
  if (page < 0 || page >= c.num_pages) return -1;
  return (long long)page * c.page_stride + (long long)(pos - page_index * c.page_size) * c.token_stride;
}

// Tokens of sequence b that the cache can hold and the length array claims; `bad` is set when the array claims others.
SB_HD int paged_len(const PagedView &c, int b, bool *bad) {
  const int n = c.lens[b];
  const long long room = (long long)c.table_width * c.page_size;
  if (n < 0) { *bad = true; return 0; }
  if (n > room) { *bad = true; return (int)room; }
  return n;
}

// Rows [*begin, *end) of sequence b in a packed tensor of `rows` rows, empty and *bad when the offsets are not 0 <= begin <= end <= rows.
SB_HD void packed_range(const int32_t *cu, int b, long long rows, int *begin, int *end, bool *bad) {
  const int x = cu[b], y = cu[b + 1];
  if (x < 0 || y < x || y > rows) {
    *begin = *end = 0;
    *bad = true;
    return;
  }
  *begin = x;
  *end = y;
}

// The sequence that row t belongs to, cu[b] <= t < cu[b + 1], by a warp: of the sequences [lo, hi) that may hold it lane l looks at
// search_probe (if that is below hi), and with k the highest lane that found cu <= t (0 if none did) search_narrow leaves a 32nd part.
// From [0, batch) it ends at one sequence, to be checked, for any contents of cu.
SB_HD int search_probe(int lo, int hi, int lane) { return lo + lane * ((hi - lo + 31) / 32); }
SB_HD void search_narrow(int &lo, int &hi, int k) {
  const int step = (hi - lo + 31) / 32;
  lo += k * step;
  if (hi > lo + step) hi = lo + step;
}

// ---- attention over the cache: dealing the work of a batch to blocks --------------------------------------------------
// The work is a row of equal units (`unit` keys of one key head of one sequence), ordered by sequence, then head, then key; block c of
// `blocks` takes the units [split_at(U, blocks, c), split_at(U, blocks, c + 1)).  Shares differ by one unit at most, whatever
// the lengths are.  A part of an item (one head of one sequence) that is not the whole of it goes to a slot of the workspace:
// slot 0 of its block when the item began in an earlier block, slot 1 when it begins here and goes on.  A block has at most one of each.
SB_HD long long split_at(long long units, int blocks, int c) { return units / blocks * c + units % blocks * c / blocks; }

// The last block that holds a unit before `end`, 0 < end <= units.
SB_HD int split_last(long long units, int blocks, long long end) {
  int lo = 0, hi = blocks - 1;   // the largest c with split_at(c) < end
  while (lo < hi) {
    const int mid = lo + (hi - lo + 1) / 2;
    if (split_at(units, blocks, mid) < end) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// Blocks that get work: no block fewer than `least` units, unless there are fewer in all.
SB_HD int split_blocks(long long units, int blocks, int least) {
  const long long most = (units + least - 1) / least;
  return most < 1 ? 1 : most < blocks ? (int)most : blocks;
}

// Units of a sequence of n tokens.
SB_HD int units_of(int n, int unit) { return (int)(((long long)n + unit - 1) / unit); }

}  // namespace sb200
