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
    const int W = 1 + r() % (kJoin * kJoins), H = 1 + r() % 8, group = 1 + r() % 20, NB = 1 + r() % 2, BR = 16 * NB;
    int64_t all = 0, groups = 0;
    for (int i = 0; i < b.s.n; i++) {
      const DecSeq d = dec_seq(kv_seq(b.s, i), group, BR, NB);
      CHECK(d.pages >= 1 && d.blocks >= 0 && d.nb >= 1 && d.nb <= NB);
      CHECK((int64_t)d.blocks * d.nb * BR >= (int64_t)kv_seq(b.s, i).nr * group);
      all += dec_units(d, H);
      groups += d.blocks * H;
    }
    CHECK(all <= dec_max_units(b.s.n, b.s.ldt, b.s.R, group, H, 16));
    if (!all) continue;
    const int share = (all + W - 1) / W;
    for (int form = 0; form < 5; form++) {  // shares; chunks of a share and up to three times four units more
      const int C = form ? (share + 3) / 4 * 4 + 4 * (form - 1) : 0;
      int64_t chunks = 0;
      if (form) {
        for (int i = 0; i < b.s.n; i++) {
          const DecSeq d = dec_seq(kv_seq(b.s, i), group, BR, NB);
          chunks += (int64_t)dec_chunks(d, C) * d.blocks * H;
        }
        if (chunks > W) continue;
      }
      std::set<int> slots, counters, firsts;
      int at = 0, item = 0;
      for (int i = 0; i < b.s.n; i++) {
        const KvSeq q = kv_seq(b.s, i);
        const DecSeq d = dec_seq(q, group, BR, NB);
        const int real = (q.len + kKvPage - 1) / kKvPage, size = dec_group(d);
        for (int k = 0; k < H * d.blocks; k++) {
          const int g0 = at, g1 = at + size;
          at = g1;
          const int first = form ? item : g0 / share, parts = form ? dec_chunks(d, C) : (g1 - 1) / share - first + 1;
          CHECK(first + parts <= W && parts <= kJoin * kJoins);
          int page = 0;
          for (int p = 0; p < parts; p++) {
            const int w = first + p;
            const DecPart part = form ? dec_part_chunk(p, parts, w) : dec_part_share(g0, g1, share);
            CHECK(part.first == first && part.parts == parts);
            const int lo = form ? p * C : std::max(g0, share * w) - g0;
            const int hi = form ? std::min(lo + C, size) : std::min(g1, share * (w + 1)) - g0;
            CHECK(lo < hi);
            CHECK(dec_page(d, lo, real) == page);  // the parts' pages follow one another
            page = dec_page(d, hi, real);
            if (parts > 1) {
              const int slot = dec_slot(part, p);
              CHECK(slot >= 0 && slot < 2 * W && slots.insert(slot).second && slot / 2 == w);
              if (p % kJoin == 0) CHECK(counters.insert(slot).second);
            }
          }
          CHECK(page == real);
          if (parts > 1) CHECK(firsts.insert(first).second);
          item += parts;
        }
      }
      CHECK(at == all && (!form || item == chunks));
    }
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
