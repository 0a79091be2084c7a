// Which 16-byte blocks of a row of the residual are copied whole and which are
// read by elements (fp8_gemm.cu).  Plain index arithmetic, so that it can be
// run over its sizes on the host.
#pragma once
#include <stdint.h>

namespace wc {

constexpr int kTurnBytes = 128;            // of a row, from the start of its first block on, that a turn takes
constexpr int kTurnRoom = kTurnBytes + 16; // and the block after, where a row that starts inside a block goes on

// Bytes [lo, hi) (hi <= lo: none) are copied whole, counted like the turns from
// the block that the row's part starts in; `head` and `tail` say that the first
// block and the one that starts at `last` are read by elements.
struct ResidualSpan {
  int lo, hi, last;
  bool head, tail;
};

// Turn t of a part of a row, `bytes` long, that starts at address `from` of a
// residual that takes the addresses [base, limit).  A part's first and last
// block may hold bytes of other rows too, which are copied and not used; blocks
// that reach outside the residual, whichever row's they are, are not copied.
constexpr ResidualSpan residual_span(uint64_t from, int bytes, uint64_t base, uint64_t limit, int t) {
  const int start = static_cast<int>(from & 15), end = bytes > 0 ? (start + bytes + 15) & ~15 : 0;
  const uint64_t block = from - start;
  const bool first = bytes > 0 && block < base, past = bytes > 0 && block + end > limit;
  const int at = t * kTurnBytes, to = past ? end - 16 : end;
  ResidualSpan s{};
  s.lo = at + (first && t == 0 ? 16 : 0);
  s.hi = to < at + kTurnRoom ? to : at + kTurnRoom;
  s.last = end - 16;
  s.head = first && t == 0;
  s.tail = past && s.last >= at && s.last < at + kTurnRoom;
  return s;
}

}  // namespace wc
