"""The generation operators without a GPU: what the C entry points refuse, what the Python handles refuse, and the index
arithmetic of their kernels (sofie_b200/csrc/paged.cuh) over hostile tables, built with a host compiler."""
import ctypes as C
import re
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from sofie_b200 import lib as L

ROOT = Path(__file__).resolve().parent.parent


def refused(lib, rc, text):
    assert rc == L.ERR_INVALID, rc
    assert text in lib.sofie_b200_last_error().decode(), lib.sofie_b200_last_error()


# any non-NULL number stands for a pointer: these calls end before anything is read
P = 4096


def cache(**kw):
    kv = L.PagedKv(P, P, P, P, 2, 10, 4, 0, 0, 0, 0, 16)
    for k, v in kw.items():
        setattr(kv, k, v)
    return kv


def append_desc(**kw):
    d = L.KvAppendDesc(tokens=5, heads=4, kv_heads=2, head_dim=64, rotary_dim=64, dtype=L.BF16, max_position=100)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def append(lib, d, kv, cu=P, q=P, k=P, v=P, cos=P, sin=P, qo=2 * P, ko=None):
    return lib.sofie_b200_kv_append_enqueue(None, C.byref(d) if d else None, C.byref(kv) if kv else None, cu, q, k, v, cos, sin, qo, ko)


def test_append_refusals(b200_lib):
    lib = b200_lib
    refused(lib, append(lib, append_desc(), cache()), "ctx is NULL")     # everything else is in order
    refused(lib, append(lib, None, cache()), "desc is NULL")
    refused(lib, append(lib, append_desc(), None), "cache is NULL")
    for kw in ({"tokens": -1}, {"tokens": 1 << 31}, {"kv_heads": 0}, {"head_dim": 0}, {"heads": -1}, {"heads": 1 << 20}):
        refused(lib, append(lib, append_desc(**kw), cache()), "bad extent")
    for dt in (L.I8, L.F8E4M3, L.I32, 17, -1):
        refused(lib, append(lib, append_desc(dtype=dt), cache()), "type")
    for r in (-2, 7, 66):
        refused(lib, append(lib, append_desc(rotary_dim=r), cache()), "rotated dimensions")
    for kw in ({"ldq": 255}, {"ldk": 127}, {"ldv": 1}, {"ldqo": 200}, {"ldko": 100}):
        refused(lib, append(lib, append_desc(**kw), cache()), "pitch is smaller")
    refused(lib, append(lib, append_desc(), cache(), cu=None), "one token")
    refused(lib, append(lib, append_desc(tokens=2), cache(), cu=None), "ctx is NULL")
    for kw in ({"k": None}, {"v": None}, {"q": None}, {"qo": None}):
        refused(lib, append(lib, append_desc(), cache(), **kw), "NULL tensor")
    for kw in ({"cos": None}, {"sin": None}):
        refused(lib, append(lib, append_desc(), cache(), **kw), "cos and sin")
    refused(lib, append(lib, append_desc(max_position=0), cache()), "cos and sin")
    refused(lib, append(lib, append_desc(ldqo=512), cache(), qo=P), "keeps the pitch")
    refused(lib, append(lib, append_desc(ldk=512), cache(), ko=P), "keeps the pitch")


@pytest.mark.parametrize("kw,text", [
    ({"batch": -1}, "batch"), ({"batch": 1 << 31}, "batch"), ({"page_size": 0}, "page size"), ({"num_pages": -1}, "pages"),
    ({"num_pages": 1 << 31}, "pages"), ({"table_width": 1 << 28}, "2^31"), ({"table_width": -1}, "2^31"), ({"table_pitch": 3}, "pitch"),
    ({"page_stride": -8}, "negative"), ({"page_stride": 2048, "token_stride": 128, "head_stride": 56}, "overlap"),
    ({"page_stride": 2047, "token_stride": 128, "head_stride": 64}, "overlap"),
    ({"page_stride": 2048, "token_stride": 64, "head_stride": 64}, "overlap"),
    ({"page_stride": 1 << 62, "token_stride": 128, "head_stride": 64}, "too large"),
    ({"seq_lens": None}, "NULL"), ({"block_table": None}, "NULL"), ({"k": None}, "NULL"), ({"v": None}, "NULL"),
])
def test_cache_refusals(b200_lib, kw, text):
    refused(b200_lib, append(b200_lib, append_desc(), cache(**kw)), text)


def test_cache_layouts_that_are_taken(b200_lib):
    for kw in ({"page_stride": 2048, "token_stride": 64, "head_stride": 1024}, {"page_stride": 4096, "token_stride": 128, "head_stride": 64},
               {"page_stride": 64, "token_stride": 640, "head_stride": 10240}, {"table_pitch": 9}):
        refused(b200_lib, append(b200_lib, append_desc(), cache(**kw)), "ctx is NULL")


def test_attention_plan_refusals(b200_lib):
    lib = b200_lib
    out = C.c_void_p()
    makes = ((lib.sofie_b200_prompt_attention_plan_create, L.PromptAttentionDesc), (lib.sofie_b200_paged_attention_plan_create, L.PagedAttentionDesc))
    for create, desc in makes:
        ok = dict(heads=8, kv_heads=2, head_dim=64, dtype=L.BF16)
        refused(lib, create(None, C.byref(desc(**ok)), C.byref(out)), "ctx is NULL")
        refused(lib, create(None, None, C.byref(out)), "NULL")
        refused(lib, create(None, C.byref(desc(**ok)), None), "NULL")
        for kw, text in (({"dtype": L.I8}, "type"), ({"kv_heads": 3}, "query heads"), ({"kv_heads": 0}, "query heads"), ({"heads": 0}, "query heads"),
                         ({"heads": 130}, "query heads"), ({"head_dim": 0}, "head size"), ({"head_dim": 60}, "head size"), ({"head_dim": 264}, "head size"),
                         ({"scale": -1.0}, "scale"), ({"scale": float("nan")}, "scale"), ({"scale": float("inf")}, "scale"),
                         ({"ldq": 511}, "pitch"), ({"ldq": 516}, "multiples of 8"), ({"ldy": 500}, "pitch"), ({"ldy": 523}, "multiples of 8")):
            refused(lib, create(None, C.byref(desc(**{**ok, **kw})), C.byref(out)), text)
        assert not out.value
    assert lib.sofie_b200_prompt_attention_plan_destroy(None) == 0 and lib.sofie_b200_paged_attention_plan_destroy(None) == 0
    assert lib.sofie_b200_prompt_attention_plan_kernel(None) == b"" and lib.sofie_b200_paged_attention_plan_kernel(None) == b""
    assert lib.sofie_b200_paged_attention_workspace_bytes(None) == 0
    refused(lib, lib.sofie_b200_prompt_attention_enqueue(None, P, P, P, P, P, P, 1, 1, 1), "plan is NULL")
    refused(lib, lib.sofie_b200_paged_attention_enqueue(None, P, C.byref(cache()), P, P), "plan is NULL")


def test_struct_layouts_match_header():
    header = (ROOT / "include" / "sofie_b200.h").read_text()
    for struct, cname in ((L.PagedKv, "sofie_b200_paged_kv"), (L.KvAppendDesc, "sofie_b200_kv_append_desc"),
                          (L.PromptAttentionDesc, "sofie_b200_prompt_attention_desc"), (L.PagedAttentionDesc, "sofie_b200_paged_attention_desc")):
        body = re.sub(r"/\*.*?\*/", "", re.search(r"typedef struct " + cname + r" \{(.*?)\} " + cname, header, re.S).group(1), flags=re.S)
        fields = []
        for decl in filter(None, (d.strip() for d in body.split(";"))):
            names = decl.split(None, 2)[2] if decl.startswith("const") else decl.split(None, 1)[1]
            fields += [n.strip().lstrip("*") for n in names.split(",")]
        assert fields == [f[0] for f in struct._fields_], cname


def test_python_handles_refuse(b200_lib):
    from sofie_b200 import ops
    z = lambda *s, dt=torch.bfloat16: torch.zeros(s, dtype=dt)
    lens, table = z(2, dt=torch.int32), z(2, 3, dt=torch.int32)
    k = z(4, 16, 2, 64)
    for bad in ((z(4, 16, 2), k, table, lens), (k, z(4, 16, 2, 32), table, lens), (k, k.float(), table, lens), (k, k, table.long(), lens),
                (k, k, table, lens.long()), (k, k, table[:1], lens), (k, k, table[0], lens), (k.transpose(2, 3), k.transpose(2, 3), table, lens),
                (k, k.transpose(0, 1).contiguous().transpose(0, 1), table, lens), (k, k, table, lens)):   # the last: not on a GPU
        with pytest.raises(ValueError):
            ops.PagedKV(*bad)
    for bad, text in ((z(5, 4, 64).transpose(1, 2), "one behind another"), (z(5, 8, 64)[:, ::2], "one behind another"), (z(5, 64), "is expected"),
                      (z(5, 12, 64)[:, 2:6], "CUDA")):
        with pytest.raises(ValueError, match=text):
            ops._rows("x", bad, 0)
    for bad in (z(4, dt=torch.int32), z(3), z(3, 1, dt=torch.int32), z(6, dt=torch.int32)[::2], z(3, dt=torch.int32)):   # the last: not on a GPU
        with pytest.raises(ValueError):
            ops._offsets("cu", bad, 2, 0)


def test_rows_that_lie_over_one_another_are_refused(b200_lib):
    """A row stride of 0 (one row expanded over a batch) or below a row's extent is no pitch: 0 means "dense" to the C entry points, which
    would then read and write behind the tensor."""
    from sofie_b200 import ops
    z = lambda *s, dt=torch.bfloat16: torch.zeros(s, dtype=dt)
    for bad in (z(1, 4, 64).expand(5, 4, 64), z(1, 1, 64).expand(2, 1, 64), z(1, 4, 1).expand(3, 4, 1), z(1024).as_strided((5, 4, 64), (128, 64, 1)),
                z(64).as_strided((2, 1, 64), (0, 64, 1))):
        with pytest.raises(ValueError, match="over one another"):
            ops._rows("x", bad, 0)
    for fine in (z(1, 4, 64).expand(1, 4, 64), z(5, 4, 64)[:1], z(0, 4, 64)):      # a stride that is never taken says nothing
        with pytest.raises(ValueError, match="CUDA"):
            ops._rows("x", fine, 0)
    lens, table, k = z(5, dt=torch.int32), z(5, 3, dt=torch.int32), z(4, 16, 2, 64)
    for bad in (z(1, 3, dt=torch.int32).expand(5, 3), z(1, 1, dt=torch.int32).expand(5, 1), z(64, dt=torch.int32).as_strided((5, 3), (2, 1))):
        with pytest.raises(ValueError, match="block_table.*over one another"):
            ops.PagedKV(k, k, bad, lens)
    for bad in (z(64).expand(4, 16, 2, 64), z(1, 16, 2, 64).expand(4, 16, 2, 64), z(4, 1, 2, 64).expand(4, 16, 2, 64), z(4, 16, 1, 64).expand(4, 16, 2, 64)):
        with pytest.raises(ValueError, match="over one another"):
            ops.PagedKV(bad, bad, table, lens)
    for fine in (z(1, 3, dt=torch.int32).expand(1, 3), z(5, 9, dt=torch.int32)[:1, 2:5]):
        with pytest.raises(ValueError, match="CUDA"):
            ops.PagedKV(k, k, fine, lens[:1])
    one = z(1, 1, 1, 64).expand(1, 1, 1, 64)
    with pytest.raises(ValueError, match="CUDA"):
        ops.PagedKV(one, one, table, lens)


HOSTILE = r'''
#include "paged.cuh"
#include <climits>
#include <cstdio>
#include <cstdlib>
#include <vector>
using namespace sb200;
#define NEED(c) do { if (!(c)) { printf("failed: %s (line %d)\n", #c, __LINE__); return 1; } } while (0)
static unsigned rs = 12345;
static int rnd(int n) { rs = rs * 1664525u + 1013904223u; return (int)((rs >> 8) % (unsigned)n); }
static int wild() { static const int w[] = {INT_MIN, -1, 0, 1, 7, INT_MAX, INT_MAX - 1, 100, 50, -1000000}; return rnd(2) ? w[rnd(10)] : rnd(60); }
int main() {
  // pages: every accepted offset lies inside the cache, every position with a page is accepted
  for (int it = 0; it < 20000; ++it) {
    const int size = 1 + rnd(20), width = rnd(6), batch = 1 + rnd(4), pages = rnd(9), kvh = 1 + rnd(3), dim = 8 * (1 + rnd(3));
    std::vector<int> table(batch * width + 1), lens(batch);
    for (auto &x : table) x = rnd(3) ? rnd(pages + 1) : wild();
    for (auto &x : lens) x = wild();
    PagedView c{table.data(), lens.data(), width, (long long)size * kvh * dim, (long long)kvh * dim, dim, batch, pages, width, size};
    const long long total = (long long)pages * size * kvh * dim;
    for (int b = 0; b < batch; ++b) {
      bool bad = false;
      const int n = paged_len(c, b, &bad);
      NEED(n >= 0 && n <= width * size);
      NEED(bad == (lens[b] < 0 || lens[b] > width * size));
      for (int j = 0; j < 200; ++j) {
        const int pos = rnd(2) ? wild() : rnd(width * size + 3);
        const long long r = paged_row(c, b, pos);
        const bool there = pos >= 0 && pos / size < width && table[b * width + pos / size] >= 0 && table[b * width + pos / size] < pages;
        NEED((r >= 0) == there);
        if (there) NEED(r + (long long)(kvh - 1) * dim + dim <= total && r == ((long long)table[b * width + pos / size] * size + pos % size) * kvh * dim);
      }
    }
  }
  // offsets past 32 bits
  {
    int table[1] = {(1 << 20) - 1}, lens[1] = {16};
    PagedView c{table, lens, 1, 16 * 8 * 128, 8 * 128, 128, 1, 1 << 20, 1, 16};
    NEED(paged_row(c, 0, 15) == ((1LL << 20) - 1) * 16 * 1024 + 15 * 1024);
  }
  // packed rows: a range is inside the tensor or refused; a row's sequence holds the row
  for (int it = 0; it < 50000; ++it) {
    const int batch = 1 + rnd(it % 50 ? 8 : 3000), rows = rnd(40);
    std::vector<int> cu(batch + 1);
    const bool ordered = rnd(2);
    int at = 0;
    for (auto &x : cu) { x = ordered ? at : wild(); at += rnd(3) ? rnd(9) : 0; }
    for (int b = 0; b < batch; ++b) {
      int x = -1, y = -1;
      bool bad = false;
      packed_range(cu.data(), b, rows, &x, &y, &bad);
      NEED(x >= 0 && x <= y && y <= rows);
      NEED(bad || (x == cu[b] && y == cu[b + 1]));
    }
    for (int t = 0; t < rows; ++t) {
      int lo = 0, hi = batch, rounds = 0;
      while (hi - lo > 1) {
        int k = 0;
        for (int lane = 0; lane < 32; ++lane) {
          const int at = search_probe(lo, hi, lane);
          if (at < hi && cu[at] <= t) k = lane;
        }
        search_narrow(lo, hi, k);
        NEED(lo >= 0 && lo < hi && hi <= batch && ++rounds < 8);
      }
      const bool found = cu[lo] <= t && t < cu[lo + 1];
      if (ordered) NEED(found == (t >= cu[0] && t < cu[batch]));
    }
  }
  puts("ok");
  return 0;
}
'''


def build_and_run(tmp_path, source):
    cxx = shutil.which("g++")
    src, exe = tmp_path / "t.cxx", tmp_path / "t"
    src.write_text(source)
    subprocess.run([cxx, "-std=c++17", "-O1", "-fsanitize=undefined,address", "-fno-sanitize-recover", f"-I{ROOT / 'sofie_b200' / 'csrc'}", str(src), "-o", str(exe)],
                   check=True, capture_output=True, text=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr


def test_index_arithmetic_over_hostile_tables(tmp_path):
    build_and_run(tmp_path, HOSTILE)


SPLIT = r'''
#include "paged.cuh"
#include <algorithm>
#include <cstdio>
#include <vector>
using namespace sb200;
#define NEED(c) do { if (!(c)) { printf("failed: %s (line %d)\n", #c, __LINE__); return 1; } } while (0)
static unsigned rs = 99;
static int rnd(int n) { rs = rs * 1664525u + 1013904223u; return (int)((rs >> 8) % (unsigned)n); }
int main() {
  for (int it = 0; it < 3000; ++it) {
    const int batch = 1 + rnd(12), items = 1 + rnd(9), unit = 16, all = 1 + rnd(it % 2 ? 30 : 600), least = 1 + rnd(8);
    std::vector<int> n(batch), table(batch * 1000, 0);
    for (auto &x : n) x = rnd(4) ? rnd(it % 3 ? 700 : 9000) : rnd(2);
    PagedView kv{table.data(), n.data(), 1000, 16 * 8, 8, 8, batch, 1, 1000, 16};
    long long slots = 0;
    std::vector<long long> base(batch + 1);
    for (int b = 0; b < batch; ++b) base[b] = slots, slots += slots_of(n[b], unit, items);
    base[batch] = slots;
    const int workers = split_workers(slots, all, least);
    NEED(workers >= 1 && workers <= all && (workers == 1 || slots / workers >= 1));
    std::vector<std::vector<int>> seen(batch * items);   // which worker took each unit
    for (int b = 0; b < batch; ++b)
      for (int i = 0; i < items; ++i) seen[b * items + i].assign(units_of(n[b], unit), -1);
    long long at = 0, lo = 1LL << 60, hi = 0;
    struct Join { int b, item, parts; };
    std::vector<Join> joins(workers, Join{0, 0, 0});
    std::vector<int> place0(workers), place1(workers);
    for (int c = 0; c < workers; ++c) {
      const long long begin = split_at(slots, workers, c), end = split_at(slots, workers, c + 1);
      NEED(begin == at && end >= begin);
      at = end;
      lo = std::min(lo, end - begin);
      hi = std::max(hi, end - begin);
      if (begin == end) continue;
      int b = 0;
      while (base[b + 1] <= begin) ++b;
      Cursor k;
      k.b = b;
      k.len = n[b];
      k.left = end - begin;
      cursor_start(k, begin - base[b], unit);
      while (k.left > 0) {   // a segment, as the kernels take it
        NEED(k.b < batch && k.item < items && k.unit < k.units && k.len == n[k.b]);
        const int first = k.unit, m = (int)std::min((long long)(k.units - k.unit), k.left);
        for (int u = first; u < first + m; ++u) {
          int &s = seen[k.b * items + k.item][u];
          NEED(s == -1);
          s = c;
        }
        const bool begins = first == 0, ends = first + m == k.units;
        if (!(begins && ends)) {
          NEED((begins ? place1 : place0)[c]++ == 0);
          if (begins) {
            const long long item_end = end - k.left + k.units;
            NEED(item_end == base[k.b] + (long long)(k.units + ITEM_COST) * (k.item + 1));
            joins[c] = {k.b, k.item, split_last(slots, workers, item_end) - c + 1};
            NEED(joins[c].parts >= 2 && c + joins[c].parts <= workers);
          }
        }
        k.unit += m - 1;
        k.left -= m - 1;
        cursor_next(k, kv, items, unit);
      }
    }
    NEED(at == slots && (slots == 0 || hi - lo <= 1));
    std::vector<int> joined(batch * items);
    for (int c = 0; c < workers; ++c)
      if (joins[c].parts) {
        const auto &s = seen[joins[c].b * items + joins[c].item];
        ++joined[joins[c].b * items + joins[c].item];
        NEED(s.front() == c && s.back() == c + joins[c].parts - 1);
        for (size_t u = 1; u < s.size(); ++u) NEED(s[u] == s[u - 1] || s[u] == s[u - 1] + 1);   // nobody between has nothing
      }
    for (size_t i = 0; i < seen.size(); ++i)
      if (!seen[i].empty()) {
        for (int c : seen[i]) NEED(c >= 0);
        NEED(joined[i] == (seen[i].front() != seen[i].back()));
      }
  }
  // far: 2^31 - 1 tokens in each of 2^20 sequences of 64 heads
  const long long slots = (1LL << 20) * slots_of(2147483647, 16, 64);
  NEED(units_of(2147483647, 16) == 1 << 27 && split_at(slots, 1184, 1184) == slots && split_at(slots, 1184, 0) == 0 && split_last(slots, 1184, slots) == 1183);
  puts("ok");
  return 0;
}
'''


def test_dealing_of_the_cache_to_warps(tmp_path):
    build_and_run(tmp_path, SPLIT)


WORKERS = r'''
#include "paged.cuh"
#include <algorithm>
#include <cstdio>
using namespace sb200;
#define NEED(c) do { if (!(c)) { printf("failed: %s (line %d)\n", #c, __LINE__); return 1; } } while (0)
int main() {
  for (int least = 1; least <= 9; ++least)
    for (int all : {1, 2, 7, 100, 1184})
      for (long long slots : {1LL, 2LL, 3LL, 4LL, 5LL, 7LL, 8LL, 10LL, 11LL, 16LL, 19LL, 100LL, 101LL, 1184LL, 3551LL, 3553LL, 1LL << 40}) {
        const int n = split_workers(slots, all, least);
        NEED(n >= 1 && n <= all && (n == all || (long long)n * least >= slots) && (n - 1LL) * least < slots);
        long long smallest = slots, sum = 0;
        for (int c = 0; c < n; ++c) {
          const long long share = split_at(slots, n, c + 1) - split_at(slots, n, c);
          smallest = std::min(smallest, share);
          sum += share;
        }
        NEED(sum == slots);
        NEED(2 * smallest >= std::min<long long>(least, slots));
      }
  NEED(split_workers(4, 100, 3) == 2 && split_at(4, 2, 1) == 2);
  NEED(split_workers(0, 100, 3) == 1);
  puts("ok");
  return 0;
}
'''


def test_shares_hold_half_of_the_least_that_is_worth_a_worker(tmp_path):
    build_and_run(tmp_path, WORKERS)
