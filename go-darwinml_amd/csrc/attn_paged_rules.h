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
}  // namespace ghip
