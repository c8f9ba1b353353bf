// Which tiles of queries the workgroups of the windowed attention's dK / dV kernel take, and
// how their sums are dealt out.
#pragma once
#include <stdint.h>

#include <algorithm>

namespace ghip {
namespace win {

constexpr int kKeys = 64;  // keys of a workgroup of dkv_kernel
constexpr int kT = 32;     // queries of a tile there

// The first tile with a query that sees a key of the workgroup's at k0.
constexpr int near_begin(int q_start, int k0) { return (k0 > q_start ? k0 - q_start : 0) / kT; }
// One past the last tile of queries that see, through their windows, a key of the
// workgroup's at k0.
constexpr int near_end(int Sq, int q_start, int window, int k0) {
  const int64_t last = static_cast<int64_t>(k0) + kKeys - 1 + window - q_start;  // one past the last such query
  const int64_t tiles = (static_cast<int64_t>(Sq) + kT - 1) / kT;
  return static_cast<int>(last <= 0 ? 0 : (last + kT - 1) / kT < tiles ? (last + kT - 1) / kT : tiles);
}
// No workgroup has more tiles from near_begin to near_end than this: keys k0 .. k0 + 63 are
// seen by the queries at k0 .. k0 + 62 + window, the first of them in a tile's row r =
// (k0 - q_start) mod 32, the same for every k0, so (r + 63 + window + 31) / 32 tiles.
constexpr int near_most(int Sq, int q_start, int window) {
  return std::min((Sq + kT - 1) / kT, (std::min(window, Sq) + kKeys + kT + (kT - q_start % kT) % kT) / kT);
}

// Sums that several workgroups hold: of the first `blocks` blocks of 32 keys, `shares` each.
struct SharePlan {
  int blocks = 0, shares = 0;
  int chunks = 0, chunk = 0;  // a list of tiles (the heads of a group one after another) in chunks of so many
  bool far = false;           // chunks of the queries beyond the windows of the sinks' workgroups; else of whole lists
};
// For BH (batch, kv head) pairs of G heads each.
constexpr SharePlan plan_shares(int64_t BH, int G, int Sq, int Sk, int q_start, int window, int sinks) {
  SharePlan s;
  const int tiles = (Sq + kT - 1) / kT;
  const int beyond = sinks > 0 ? tiles - near_end(Sq, q_start, window, 0) : 0;
  const int own = near_most(Sq, q_start, window);
  const int64_t grid = static_cast<int64_t>((Sk + kKeys - 1) / kKeys) * BH;
  if (beyond > 0 && beyond >= own && sinks <= 128) {
    // (More sinks are many workgroups of their own.)  Chunks of 8 tiles, us a call with 4 /
    // 8 / 16 / 32: padded batch of 12 heads of 64, window 128, 50.5 / 51.9 / 56 / 65; 4 x 16
    // heads, 2048 tokens, window 512, 200 / 197 / 200 / 209.  The shares take half of q's
    // memory.
    s.far = true;
    s.blocks = (sinks + 31) / 32;
    s.chunk = 8 * s.blocks;
    s.chunks = (beyond * G + s.chunk - 1) / s.chunk;
    s.shares = 1 + s.chunks;
  } else if (grid < 256) {
    // Few workgroups: chunks of at least 4 tiles, towards 512 workgroups.
    const int64_t longest = static_cast<int64_t>(sinks > 0 ? tiles : own) * G;
    const int64_t goal = std::min<int64_t>(grid > 0 ? (512 + grid - 1) / grid : 1, longest / 4);
    if (goal > 1) {
      s.chunk = static_cast<int>((longest + goal - 1) / goal);
      s.chunks = static_cast<int>((longest + s.chunk - 1) / s.chunk);
      s.blocks = (Sk + 31) / 32;
      s.shares = s.chunks;
    }
  }
  return s;
}

}  // namespace win
}  // namespace ghip
