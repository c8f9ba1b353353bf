"""How the paged attention deals its tiles out, on the CPU: the workers hold them all and no
worker that has one begins past the last, for totals around each power of two (32-bit and
64-bit divisions) and up to the largest that the entry point lets through."""
import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "go-darwinml_amd", "csrc")

CODE = r"""
#include <cstdio>
#include "attn_paged_rules.h"
using namespace ghip::paged;

int main() {
  int bad = 0;
  for (int bit = 0; bit < 51; ++bit)  // 2^24 heads of 2^25 tiles and a few
    for (int64_t d = -1100; d <= 1100; ++d) {
      const int64_t total = (int64_t{1} << bit) + d;
      if (total < 0) continue;
      const int64_t per = share_of(total);
      // All are dealt out, in shares as equal as can be or of the least size.
      if (per * kWorkers < total || per < kMinTiles || (per > kMinTiles && (per - 1) * kWorkers >= total)) {
        if (!bad++) printf("%lld tiles: %lld a worker\n", (long long)total, (long long)per);
      }
    }
  return bad != 0;
}
"""


def test_the_workers_hold_every_tile(tmp_path):
    src, exe = tmp_path / "share.cpp", tmp_path / "share"
    src.write_text(CODE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", CSRC, str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout
