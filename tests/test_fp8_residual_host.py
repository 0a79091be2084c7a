"""Which bytes of a residual off the 16-byte boundary the many-row product
reads: csrc/fp8_span.h compiled for the host and run over rows shorter than a
block, rows that end just behind a part of 128 columns, and every start."""
import os
import subprocess

from conftest import ROOT

HARNESS = r"""
#include <cstdio>
#include <vector>
#include "fp8_span.h"
using namespace wc;

static int check(int size, int m, int n, int ld, int offset) {
  const uint64_t base = 4096 + offset, limit = base + (uint64_t(m - 1) * ld + n) * size;
  const int part = 128, turns = part * size / kTurnBytes;
  for (int row = 0; row < m; ++row)
    for (int col = 0; col < n; col += part) {
      const int bytes = (n - col < part ? n - col : part) * size;
      const uint64_t from = base + (uint64_t(row) * ld + col) * size;
      const int start = from & 15;
      const uint64_t block = from - start;
      for (int t = 0; t < turns; ++t) {
        const ResidualSpan s = residual_span(from, bytes, base, limit, t);
        const int lo = t * kTurnBytes, hi = lo + kTurnRoom;
        if (s.hi > s.lo) {
          if (s.lo % 16 || s.hi % 16 || s.lo < lo || s.hi > hi) return 1;        // whole blocks, inside the room
          if (block + s.lo < base || block + s.hi > limit) return 2;             // inside the residual
        }
        std::vector<char> have(kTurnRoom, 0);
        for (int b = s.lo; b < s.hi; ++b) have[b - lo] = 1;
        auto elements = [&](int at0) {
          for (int b = at0 > start ? at0 : start; b < at0 + 16 && b < start + bytes; ++b) {
            if (b < lo || b >= hi) return 3;
            have[b - lo] = 1;
          }
          return 0;
        };
        if (s.head && elements(0)) return 3;
        if (s.tail && elements(s.last)) return 3;
        for (int b = lo > start ? lo : start; b < hi && b < start + bytes; ++b)
          if (!have[b - lo]) return 4;                                           // all that the turn needs
      }
    }
  return 0;
}

int main() {
  for (int size = 2; size <= 4; size += 2)
    for (int m : {1, 2, 3, 17, 40})
      for (int n = 1; n <= 300; n += n < 20 || (n > 118 && n < 145) || (n > 250 && n < 275) ? 1 : 13)
        for (int extra : {0, 1, 2, 5, 9})
          for (int offset = 0; offset < 16; offset += size)
            if (int rc = check(size, m, n, n + extra, offset)) {
              std::printf("rule %d broken: size %d m %d n %d ld %d offset %d\n", rc, size, m, n, n + extra, offset);
              return 1;
            }
  return 0;
}
"""


def test_residual_is_read_inside_itself(tmp_path):
    src, exe = tmp_path / "span.cpp", tmp_path / "span"
    src.write_text(HARNESS)
    subprocess.run(["g++", "-O1", "-std=c++17", "-I", os.path.join(ROOT, "witchcraft_b200", "csrc"), str(src), "-o",
                    str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout
