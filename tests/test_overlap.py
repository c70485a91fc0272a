"""CPU check of csrc/mk_overlap.h, which finds tensors that lie on each other:
against sets of bytes, for every start of a over b and many shapes."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SRC = r"""
#include <cstdio>
#include <set>
#include "mk_overlap.h"
using mk::Span;
static std::set<long long> bytes(const Span& s) {
  std::set<long long> r;
  for (long long t = 0; t < s.tokens; ++t)
    for (long long h = 0; h < s.heads; ++h)
      for (long long w = 0; w < s.width; ++w) r.insert((long long)s.p + t * s.ts + h * s.hs + w);
  return r;
}
int main() {
  long long n = 0, hits = 0;
  for (long long tokens : {1, 2, 3})
    for (long long ha : {1, 2, 3})
      for (long long hb : {1, 2})
        for (long long wa : {2, 4})
          for (long long wb : {2, 4})
            for (long long hs : {4, 6})
              for (long long ts : {4, 10, 12, 23, 40})
                for (long long d = -90; d <= 90; ++d) {
                  const Span a{1000, tokens, ha, ts, hs, wa}, b{(uintptr_t)(1000 + d), tokens, hb, ts, hs, wb};
                  const auto x = bytes(a), y = bytes(b);
                  bool meet = false;
                  for (long long v : y) meet = meet || x.count(v);
                  ++n, hits += meet;
                  if (mk::overlap(a, b) != meet || mk::overlap(b, a) != meet) {
                    std::printf("tokens %lld heads %lld %lld widths %lld %lld strides %lld %lld start %lld: %d, not %d\n", tokens, ha,
                                hb, wa, wb, ts, hs, d, !meet, meet);
                    return 1;
                  }
                }
  // packed rows of 24 heads, queries and keys of one buffer, and of nothing
  const Span q{4096, 1 << 20, 16, 32 * 128, 128, 128}, k{4096 + 16 * 128, 1 << 20, 8, 32 * 128, 128, 128};
  if (mk::overlap(q, k) || mk::overlap(k, q)) return std::puts("packed"), 1;
  if (!mk::overlap(q, Span{k.p - 16, k.tokens, 8, k.ts, k.hs, 128})) return std::puts("shifted"), 1;
  if (mk::overlap(q, Span{q.p, 0, 16, q.ts, q.hs, 128})) return std::puts("nothing"), 1;
  if (!mk::overlap(Span{4096, 4, 2, 256, 128, 128}, Span{4096 + 1000, 9, 1, 100, 0, 100})) return std::puts("dense"), 1;
  if (mk::overlap(Span{4096, 4, 2, 256, 128, 128}, Span{4096 + 1024, 9, 1, 100, 0, 100})) return std::puts("beside"), 1;
  // other strides are not compared, except where a single token or head has none
  if (mk::overlap(q, Span{q.p, 4, 16, 999, 128, 128})) return std::puts("strides"), 1;
  if (!mk::overlap(q, Span{q.p + q.ts, 1, 1, 0, 0, 128})) return std::puts("single"), 1;
  std::printf("ok %d\n", n > 100000 && hits > 10000 && hits < n);
}
"""


def test_overlaps_are_those_of_the_bytes(tmp_path):
    gxx = shutil.which("g++")
    if not gxx:
        pytest.skip("g++ not available")
    src, out = tmp_path / "overlap.cpp", tmp_path / "overlap"
    src.write_text(SRC)
    subprocess.run([gxx, "-std=c++17", "-O1", "-Wall", "-Werror", "-I", os.path.join(ROOT, "megakernel_amd", "csrc"),
                    str(src), "-o", str(out)], check=True, timeout=120)
    r = subprocess.run([str(out)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout == "ok 1\n", r.stdout
