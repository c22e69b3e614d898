"""The index arithmetic that the cache and attention kernels share
(``csrc/wir_pages.h``), compiled for the CPU and checked against counting:
which positions a block sees, scales, and the division of the work, its
partial results and their slots."""
import os
import shutil
import subprocess

import pytest

from warpir_amd.runtime import PKG_DIR

SOURCE = r"""
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <cmath>
#include <climits>
#include <map>
#include <set>
#include <vector>
#include "wir_pages.h"
using namespace wir;

#define CHECK(x) do { if (!(x)) { std::printf("line %d: %s\n", __LINE__, #x); std::exit(1); } } while (0)

static unsigned long long state = 88172645463325252ull;
static int draw(int lo, int hi) {   // lo .. hi
  state ^= state << 13, state ^= state >> 7, state ^= state << 17;
  return lo + (int)(state % (unsigned long long)(hi - lo + 1));
}

static void spans() {
  const int odd[] = {INT_MIN, -1, 0, 1, 15, 16, 17, 63, 64, 65, 1000, INT_MAX};
  for (int length : odd)
    for (int count : odd)
      for (int tokens : {0, 1, 5, 64, 1 << 30})
        for (int capacity : {0, 16, 1024, 1 << 30}) {
          const Span s = span_of(length, count, tokens, capacity);
          CHECK(s.count >= 0 && s.count <= tokens && s.held >= 0 && s.held <= capacity);
          CHECK((i64)s.start == (i64)(length > 0 ? length : 0) - s.count);
          CHECK(first_new(s) >= 0);
        }
  for (int id : odd) CHECK(checked_page(id, 17) == (id >= 0 && id < 17 ? id : -1));
}

static void keys() {
  for (int it = 0; it < 200000; ++it) {
    const int tokens = draw(1, 40), group = draw(1, 9), rpb = 16 << draw(0, 3), capacity = draw(0, 300);
    const Span s = span_of(draw(-3, 330), draw(-3, 44), tokens, capacity);
    const int rows = tokens * group, blocks = (rows + rpb - 1) / rpb, rb = draw(0, blocks - 1);
    int most = 0;
    for (int r = rb * rpb; r < rows && r < (rb + 1) * rpb; ++r) {
      const int t = r / group;
      if (t >= s.count) continue;
      const int pos = s.start + t, seen = pos + 1 < s.held ? pos + 1 : s.held;
      if (pos >= 0 && seen > most) most = seen;
    }
    const int got = block_keys(s, rb, rpb, rows, group);
    CHECK(got == most);
    CHECK(block_units(got) == (most ? (most + TILE - 1) / TILE : 1));
  }
  CHECK(block_tiles(0) == 0 && block_tiles(1) == 1 && block_tiles(64) == 1 && block_tiles(65) == 2);
  CHECK(slot_of(-5, 3, 4) == 0 && slot_of(INT_MAX, 1, 4) == slots_for(4) - 1);
  CHECK(block_units(INT_MAX) == (int)(((long long)INT_MAX + 63) / 64));
}

static void scales() {
  for (int it = 0; it < 2000000; ++it) {
    unsigned bits = it < 200000 ? (unsigned)it * 21473u : (unsigned)draw(0, 0x7f7fffff);
    if (bits > 0x7f7fffffu) bits %= 0x7f7fffffu;
    float amax, scale;
    std::memcpy(&amax, &bits, 4);
    const unsigned s = scale_bits(bits);
    std::memcpy(&scale, &s, 4);
    CHECK(amax <= 448.0 * scale);
    CHECK(scale == std::ldexp(1.0f, -126) || amax > 448.0 * scale / 2);
  }
}

// Walks the programs as the kernels do.
static void division() {
  for (int it = 0; it < 40000; ++it) {
    const int pairs = draw(1, 12), heads = draw(1, 5), least = draw(1, 9), extra = draw(1, 90);
    std::vector<int> units(pairs);
    for (int& n : units) n = draw(0, 9) ? draw(1, 30) : draw(1, 4000);
    int total = 0;
    for (int n : units) total += heads * n;
    const int share = share_of(total, extra, least), width = slot_width(share);
    std::set<int> used;
    int programs = 0, begin = 0;
    for (int p = 0; p < pairs; ++p) {
      const int parts = parts_of(units[p], share);
      CHECK(parts >= 1 && parts <= units[p]);
      for (int h = 0; h < heads; ++h, begin += units[p], programs += parts) {
        CHECK(part_begin(0, units[p], parts) == 0 && part_begin(parts, units[p], parts) == units[p]);
        for (int n = 0; n < parts; ++n) {
          const int lo = part_begin(n, units[p], parts), hi = part_begin(n + 1, units[p], parts);
          CHECK(hi > lo && hi - lo <= share);
          if (parts == 1) continue;
          CHECK((begin + lo) / width < slots_for(extra));   // (the bound is for lengths that change meanwhile)
          const int slot = slot_of(begin + lo, width, extra);
          CHECK(slot >= 0 && slot < slots_for(extra) && used.insert(slot).second);
        }
      }
    }
    CHECK(programs <= pairs * heads + extra && begin == total);
  }
}

int main() {
  spans();
  keys();
  scales();
  division();
  std::puts("ok");
}
"""


@pytest.mark.skipif(not shutil.which("g++"), reason="no host compiler")
def test_index_arithmetic(tmp_path):
    src = tmp_path / "index.cpp"
    src.write_text(SOURCE)
    exe = str(tmp_path / "index")
    subprocess.run(["g++", "-O1", "-g", "-std=c++17", "-Wall", "-Werror", "-ftrapv", "-I",
                    os.path.join(PKG_DIR, "csrc"), str(src), "-o", exe], check=True)
    run = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and run.stdout.strip() == "ok", run.stdout + run.stderr
