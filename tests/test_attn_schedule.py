"""The cache's page layout and the division of the attention kernels' work, on the CPU: a host program over the same header
that the kernels include (ijah_amd/csrc/attn.h).

  - a block's keys, values and steps occupy every byte of it exactly once, and the granules that the kernels load are whole;
  - the pieces of a write or read fit the grid that is launched for them, whatever the lengths;
  - decode's shares cover every unit once; each group's partials have slots of their own, which the join finds, and counters
    of their own."""
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include <random>
#include <set>
#include <vector>
#include "attn.h"
using namespace ijah;
#define CHECK(c) do { if (!(c)) { printf("%s:%d: %s\n", __FILE__, __LINE__, #c); exit(1); } } while (0)

static void layout() {
  for (int kind : {kKvBf16, kKvF16, kKvI8})
    for (int D : {64, 128, 256}) {
      const int e = kv_esize(kind);
      std::vector<int> hit(kv_block_bytes(kind, D), 0);
      for (int j = 0; j < kKvPage; j++) {
        for (int d = 0; d < D; d++)
          for (int b = 0; b < e; b++) {
            hit[kv_key_at(kind, D, j, d) + b]++;
            hit[kv_value_at(kind, D, j, d) + b]++;
          }
        if (kind == kKvI8)
          for (int v = 0; v < 2; v++)
            for (int b = 0; b < 4; b++) hit[kv_step_at(D, v, j) + b]++;
        // 8 dims of a key from a multiple of 8 on, and the 4 values of keys 4 q .. 4 q + 3, are consecutive
        for (int d = 0; d < D; d += 8)
          for (int k = 0; k < 8; k++) CHECK(kv_key_at(kind, D, j, d + k) == kv_key_at(kind, D, j, d) + k * e);
        if (j % 4 == 0)
          for (int d = 0; d < D; d++)
            for (int k = 0; k < 4; k++) CHECK(kv_value_at(kind, D, j + k, d) == kv_value_at(kind, D, j, d) + k * e);
      }
      for (int h : hit) CHECK(h == 1);
    }
}

struct Batch {
  std::vector<int> lens, rows, table;
  KvSeqs s;
};
static Batch batch(std::mt19937 &r, int n, int maxlen, int maxnew, bool bad) {
  Batch b;
  b.rows.push_back(0);
  for (int i = 0; i < n; i++) {
    b.lens.push_back(bad && r() % 8 == 0 ? (int)r() : (int)(r() % (maxlen + 1)));
    b.rows.push_back(b.rows.back() + r() % (maxnew + 1));
  }
  b.s = KvSeqs{n, maxlen / kKvPage + 1, 100, b.rows.back() ? b.rows.back() : 1, nullptr, b.lens.data(), b.rows.data()};
  if (bad) b.s.R = 1 + r() % b.s.R;
  return b;
}
static void pieces(std::mt19937 &r) {
  for (int it = 0; it < 3000; it++) {
    Batch b = batch(r, 1 + r() % 40, 1 + r() % 700, r() % 3 ? 1 + r() % 300 : 1, it % 2);
    int64_t all = 0, rows = 0;
    for (int i = 0; i < b.s.n; i++) {
      const KvSeq q = kv_seq(b.s, i);
      CHECK(q.len >= 0 && q.len <= b.s.ldt * kKvPage && q.r0 >= 0 && q.nr >= 0 && q.r0 + q.nr <= b.s.R);
      all += kv_pieces(q);
      rows += q.nr;
    }
    CHECK(all <= kv_max_pieces(b.s.n, b.s.R, true));
    KvSeqs one = b.s;
    one.rows = nullptr;
    one.R = one.n;
    all = 0;
    for (int i = 0; i < one.n; i++) all += kv_pieces(kv_seq(one, i));
    CHECK(all == kv_max_pieces(one.n, one.R, false));
  }
}
static void shares(std::mt19937 &r) {
  for (int it = 0; it < 3000; it++) {
    Batch b = batch(r, 1 + r() % 30, 1 + r() % (it % 5 ? 900 : 60000), 1 + r() % 8, it % 2);
    const int W = 1 + r() % (kJoin * kJoins), H = 1 + r() % 8, group = 1 + r() % 20, BR = r() % 2 ? 16 : 32, least = r() % 2 ? 4 : 8;
    // the two forms, as the kernel chooses them
    auto total = [&](int pad) {
      int t = 0;
      for (int i = 0; i < b.s.n; i++) t += dec_units(dec_seq(kv_seq(b.s, i), group, BR), H, pad);
      CHECK(t <= dec_max_units(b.s.n, b.s.ldt, b.s.R, group, H, 16, 8));
      return t;
    };
    int pad = least, all = total(pad), share = least;
    if (all > W * least) {
      pad = 1;
      all = total(pad);
      share = (all + W - 1) / W;
    }
    if (!all) continue;
    CHECK((int64_t)share * W >= all);
    std::set<int> slots, counters, firsts;
    int64_t units = 0;
    int at = 0;
    for (int i = 0; i < b.s.n; i++) {
      const KvSeq q = kv_seq(b.s, i);
      const DecSeq d = dec_seq(q, group, BR);
      CHECK(d.pages >= 1 && d.blocks >= 0);
      for (int k = 0; k < H * d.blocks; k++) {
        const int g0 = at, g1 = g0 + dec_units(d, 1, pad) / d.blocks, first = g0 / share, last = (g1 - 1) / share;
        at = g1;
        CHECK(last < W);
        int real = 0;
        for (int w = first; w <= last; w++) {
          const int lo = std::max(g0, share * w), hi = std::min(g1, share * (w + 1));
          CHECK(lo < hi);
          const int p0 = lo - g0, p1 = std::min(hi - g0, (q.len + kKvPage - 1) / kKvPage);
          CHECK(p0 < p1 || (q.len == 0 && p0 == 0));
          real += std::max(p1 - p0, 0);
          const DecPart p = dec_part(g0, g1, share, w);
          CHECK(p.first == first && p.parts == last - first + 1 && p.parts <= kJoin * kJoins);
          if (p.parts > 1) {
            CHECK(p.slot >= 0 && p.slot < 2 * W && slots.insert(p.slot).second);
            CHECK(p.slot == dec_slot(p, g0, share, w - first));
            if ((w - first) % kJoin == 0) CHECK(counters.insert(p.slot).second);
          }
        }
        CHECK(real == (q.len + kKvPage - 1) / kKvPage);
        units += g1 - g0;
        if (last > first) CHECK(firsts.insert(first).second);
      }
    }
    CHECK(units == all && at == all);
  }
}
int main() {
  std::mt19937 r(7);
  layout();
  pieces(r);
  shares(r);
  puts("ok");
}
"""


def test_layout_pieces_and_shares(tmp_path):
    src, exe = tmp_path / "check.cpp", tmp_path / "check"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-Wall", "-fsanitize=undefined,address", "-fno-sanitize-recover=all",
                    f"-I{ROOT / 'ijah_amd' / 'csrc'}", str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout == "ok\n", r.stdout + r.stderr[-2000:]
