// How the rows of rotations and appends are dealt out, without device code (a CPU test compiles it).
#pragma once

#include <algorithm>
#include <cstdint>

namespace ghip {
namespace rope {

constexpr int kThreads = 256;
constexpr int kMostTokens = 16;  // of a workgroup

struct Deal {
  int block_tokens = 1;  // tokens of a workgroup
  int splits = 0;        // workgroups that share their rows
  int splits4 = 0;       // and their rows into 4 bits
  int both = 0;          // 4 bits: the one workgroup of a token takes its rows of both kinds
};

// How the rows are dealt out: a row in each slot until 1024 workgroups (four a CU) run, then two,
// beyond eight times as many three, so that a token's angles serve many rows and workgroups still follow each other.
// us with 1, 2, 3, 4, 6, 12 rows a slot (one: a token a workgroup, whose slots its rows may not fill):
//   rope, 16 heads of 128, bf16, 2048 tokens       7.5   6.1   7.2   7.0   8.4  10.8
//   the same, 4 x 2048                            20.2  13.5  15.0  13.9  15.2  15.8
//   the same, 8 x 8192                             151  94.0  98.5  98.8   104   111
//   into 16 bits, 32 heads and 8, f16, 8 x 1024   54.2  37.7  35.2  35.2  35.4  36.3
//   into 4 bits, the same in bf16                 52.0  36.4  36.4  37.8  40.8  51.6
// H: heads of queries; units: threads of a row, units4: of a row into 4 bits.
inline Deal deal(int64_t tokens, int64_t H, int64_t Hkv, int units, int units4, bool four) {
  const int64_t rows = H + (four ? 0 : 2 * Hkv), rows4 = four ? 2 * Hkv : 0;
  const int64_t slots = kThreads / units, slots4 = four ? kThreads / units4 : 1;
  const int64_t all = tokens * (rows * units + rows4 * (four ? units4 : 0));
  const int64_t filled = all / (kThreads * 1024), each = filled < 1 ? 1 : filled < 8 ? 2 : 3;
  Deal d;
  auto parts = [&](int64_t r, int64_t s) {
    return static_cast<int>(r ? std::max<int64_t>(1, (r + s * each - 1) / (s * each)) : 0);
  };
  d.splits = parts(rows, slots);
  d.splits4 = parts(rows4, slots4);
  if (d.splits <= 1 && d.splits4 <= 1 && each > 1) {
    const int64_t by = rows ? std::max<int64_t>(1, slots * each / rows) : kMostTokens;
    const int64_t by4 = rows4 ? std::max<int64_t>(1, slots4 * each / rows4) : kMostTokens;
    d.block_tokens = static_cast<int>(std::min<int64_t>({by, by4, kMostTokens}));
    // Enough tokens for every slot of either kind: the angles are computed once for both.
    if (four && H > 0) {
      d.both = 1;
      d.splits4 = 0;
    }
  }
  return d;
}

// Elements that a thread takes at a time: 16 bytes, or the most that divide the row and half of what
// turns of it.  (bf16, 4 x 16 heads of 80, 40 of them turned: 33 us one by one, 14 four by four.)
inline int width(int D, int half, int most) {
  int n = most;
  while (n > 1 && (D % n || half % n)) n /= 2;
  return n;
}

}  // namespace rope
}  // namespace ghip
