"""Whether two strided operands share a byte (csrc/overlap.hpp), against the sets
of their bytes."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "glt_amd", "csrc")

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include <set>
#include "overlap.hpp"
using glt::ByteRows;
static bool by_bytes(const ByteRows& p, const ByteRows& q) {
  std::set<uintptr_t> s;
  for (int64_t i = 0; i < p.rows; ++i)
    for (int64_t c = 0; c < p.width; ++c) s.insert((uintptr_t)p.at + i * p.ld + c);
  for (int64_t i = 0; i < q.rows; ++i)
    for (int64_t c = 0; c < q.width; ++c)
      if (s.count((uintptr_t)q.at + i * q.ld + c)) return true;
  return false;
}
int main() {
  srand(7);
  auto any = [](int64_t lo, int64_t hi) { return lo + rand() % (hi - lo + 1); };
  int yes = 0, no = 0;
  for (int n = 0; n < 200000; ++n) {
    ByteRows x[2];
    for (auto& r : x) {
      r.rows = any(0, 6);
      r.width = any(0, 9);
      r.ld = r.width + any(r.width ? 0 : 1, 14);
      r.at = (const void*)(uintptr_t)any(1000, 1100);
    }
    if (n & 1) x[1].ld = x[0].ld < x[1].width ? x[1].ld : x[0].ld;
    const bool want = by_bytes(x[0], x[1]);
    (want ? yes : no)++;
    if (glt::overlap(x[0], x[1]) != want || glt::overlap(x[1], x[0]) != want) {
      for (auto& r : x) printf("at %zu rows %ld width %ld ld %ld\n", (size_t)r.at, (long)r.rows, (long)r.width, (long)r.ld);
      return 1;
    }
  }
  printf("%d %d\n", yes, no);
  return yes > 20000 && no > 20000 ? 0 : 2;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="no host compiler")
def test_overlap_against_the_bytes(tmp_path):
    src, exe = tmp_path / "overlap.cpp", tmp_path / "overlap"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O2", "-I", CSRC, str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout
