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

// ---- attention over the cache: dealing the work of a batch to workers (warps) ------------------------------------------
// An item is one head of one sequence; it takes ITEM_COST slots (what beginning and ending one costs, in units of time) and then one
// slot for every unit of `unit` keys.  The slots of all items, ordered by sequence, then head, then key, are one row; worker c of
// `workers` takes the slots [split_at(S, workers, c), split_at(S, workers, c + 1)).  Shares differ by one slot at most, whatever the lengths
// are.  A part of an item that is not the whole of it goes to a place of the workspace: place 0 of its worker when the item began
// in an earlier one, place 1 when it begins here and goes on.  A worker has at most one of each.
constexpr int ITEM_COST = 1;

// Quotient of numbers from 0 on; 32 bits where they are enough (a 64-bit division is a routine of a hundred instructions).
SB_HD long long quotient(long long a, long long b) {
  return ((unsigned long long)(a | b) >> 32) == 0 ? (long long)((unsigned)a / (unsigned)b) : a / b;
}

SB_HD long long split_at(long long slots, int workers, int c) {   // workers below 2^15: the rest's share fits 32 bits
  const long long each = quotient(slots, workers);
  return each * c + (unsigned)(slots - each * workers) * (unsigned)c / (unsigned)workers;
}

// The last worker that holds a slot before `end`, 0 < end <= slots.
SB_HD int split_last(long long slots, int workers, long long end) {
  int lo = 0, hi = workers - 1;   // the largest c with split_at(c) < end
  while (lo < hi) {
    const int mid = lo + (hi - lo + 1) / 2;
    if (split_at(slots, workers, mid) < end) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// Workers that get work: as many as shares of `least` slots make, the last one begun counting as one.  So a share may be smaller (4
// slots by 3: two of 2), but holds at least half of `least`, unless there are fewer slots in all.
SB_HD int split_workers(long long slots, int workers, int least) {
  const long long most = quotient(slots + least - 1, least);
  return most < 1 ? 1 : most < workers ? (int)most : workers;
}

// Units of a sequence of n tokens.
SB_HD int units_of(int n, int unit) { return (int)(((unsigned)n + (unsigned)unit - 1u) / (unsigned)unit); }   // n below 2^31

// Slots of all items of a sequence.
SB_HD long long slots_of(int n, int unit, int items) { return n > 0 ? ((long long)units_of(n, unit) + ITEM_COST) * items : 0; }

// A worker's way down its share.  left: slots of the share from `unit` on; nothing is left when it is 0 or less.
struct Cursor {
  int b, item, unit, units, len;   // sequence, item of the sequence, unit of the item; units and tokens of the sequence
  long long left;
};

// From slot `offset` of the items of sequence c.b (whose len is set) on.
SB_HD void cursor_start(Cursor &c, long long offset, int unit) {
  c.units = units_of(c.len, unit);
  const long long per = (long long)c.units + ITEM_COST;
  c.item = (int)quotient(offset, per);
  const long long o = offset - c.item * per;
  c.unit = o > ITEM_COST ? (int)(o - ITEM_COST) : 0;
  if (o < ITEM_COST) c.left -= ITEM_COST - o;
}

// The next unit; lens[] is read where a sequence ends.
SB_HD void cursor_next(Cursor &c, const PagedView &kv, int items, int unit) {
  --c.left;
  if (++c.unit < c.units) return;
  c.unit = 0;
  c.left -= ITEM_COST;
  if (++c.item < items) return;
  c.item = 0;
  bool bad = false;
  do {
    ++c.b;
  } while (c.b < kv.batch && (c.len = paged_len(kv, c.b, &bad)) == 0);
  c.units = c.b < kv.batch ? units_of(c.len, unit) : 0;
  if (c.b >= kv.batch) c.left = 0;
}

}  // namespace sb200
