// How the paged attention deals the tiles of all sequences out over its workers.
#pragma once
#include <stdint.h>

namespace ghip {
namespace paged {

// The workers that share the tiles of all sequences: one wave each, four a CU with 32 KiB
// of LDS tiles, most of it in flight.  (268 MB: 65 us; with 1280, 1536, 2048 or 4096 workers,
// which do not all run at once, 85, 77, 68 and 75.)
constexpr int kWorkers = 1024;
constexpr int kMinTiles = 2;  // tiles of a worker at least

// Tiles of a worker, of `total` in all.  (A division in 32 bits where the dividend fits.)
constexpr int64_t share_of(int64_t total) {
  const int64_t up = total + kWorkers - 1;
  const int64_t per = up <= 0xffffffffLL ? static_cast<uint32_t>(up) / kWorkers : up / kWorkers;
  return per < kMinTiles ? kMinTiles : per;
}

}  // namespace paged

// Decoding over 4 bits deals out places: each unit's tiles, and kBegin places ahead of them without
// a tile, what the chain page - rows at a unit's beginning costs a worker beside a tile.
// bf16 D 128, 8 kv heads, us with 0, 1, 2, 3, 4 of them:
//   64 sequences of 1 to 128 tiles            84.7  74.0  71.5  71.5  72.1
//   64 of 1 to 256, as many of each size      77.3  58.3  53.4  54.2  54.3
//   one of 2048, eight of one                 60.8  45.5  43.5  42.8  43.5
//   8 of 1 to 64 / 16 of 1 to 64              15.3 / 20.7  -  13.5 / 19.0
//   64 of 64 / 128 of 32 tiles                64.0 / 66.4  64.9 / 68.2  64.7 / 68.8  64.4 / 69.0  65.0 / 69.6
//   8 of 64 (two tiles a worker)              18.0  20.0  20.0  20.0  19.9
namespace paged4 {

constexpr int kBegin = 2;
constexpr int kLeast = 2;  // places of a worker at least

// Of `workers`, those that have a part of `total` places.
constexpr int used_of(int64_t total, int workers) {
  return total / kLeast >= workers ? workers : total < kLeast ? 1 : static_cast<int>(total / kLeast);
}
// Where worker i of `used` begins, i <= used: parts differ by one place at most.  (Where all have
// one, a shift; else all fits 32 bits.)
template <int WORKERS>
constexpr int64_t first_of(int i, int64_t total, int used) {
  return used == WORKERS ? i * total / WORKERS : static_cast<uint32_t>(i * total) / static_cast<uint32_t>(used);
}
// The worker that has place `at`.
constexpr int worker_of(int64_t at, int64_t total, int used) {
  const int64_t up = (at + 1) * used - 1;
  return static_cast<int>(((up | total) >> 32) == 0 ? static_cast<uint32_t>(up) / static_cast<uint32_t>(total) : up / total);
}

// n / size for 0 <= n < 2^31, by the product with a 33-bit reciprocal: with shift = ceil(log2 size)
// and mul = floor(2^32 (2^shift - size) / size) + 1 the quotient is exact (Granlund and
// Montgomery).  A division costs 25 instructions, two of them a tile of 64 tokens 7% of it.
struct Pages {
  uint32_t mul = 0;
  int shift = 0;
  constexpr Pages() {}
  constexpr explicit Pages(int64_t size) {
    while (int64_t{1} << shift < size) ++shift;
    mul = static_cast<uint32_t>((static_cast<uint64_t>((int64_t{1} << shift) - size) << 32) / static_cast<uint64_t>(size) + 1);
  }
  constexpr int quotient(uint32_t n) const {
    const uint32_t t = static_cast<uint32_t>(static_cast<uint64_t>(mul) * n >> 32);
    return static_cast<int>((t + ((n - t) >> (shift < 1 ? shift : 1))) >> (shift > 1 ? shift - 1 : 0));
  }
};

}  // namespace paged4
}  // namespace ghip
