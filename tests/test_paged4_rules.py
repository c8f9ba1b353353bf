"""How decoding over 4 bits deals its places out, on the CPU: workers' parts follow one another from
the first place to the last, differ by one place at most, and each place is found in its
worker's part again; for totals around each power of two (32-bit and 64-bit divisions) and up to
the largest that the entry point lets through.  And a token's page without a division."""
import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "go-darwinml_amd", "csrc")

CODE = r"""
#include <cstdio>
#include <initializer_list>
#include "attn_paged_rules.h"
using namespace ghip::paged4;

template <int W>
int check(int64_t total) {
  const int used = used_of(total, W);
  int bad = used < 1 || used > W || (used > 1 && total / used < kLeast) || (used < W && total / (used + 1) >= kLeast);
  bad |= first_of<W>(0, total, used) != 0 || first_of<W>(used, total, used) != total;
  for (int i = 0; i < used && !bad; i += i < 70 || i > used - 70 ? 1 : 61) {
    const int64_t a = first_of<W>(i, total, used), e = first_of<W>(i + 1, total, used);
    bad |= e - a < total / used || e - a > total / used + 1;
    bad |= a < e && (worker_of(a, total, used) != i || worker_of(e - 1, total, used) != i);
  }
  if (bad) printf("%lld places of %d workers\n", (long long)total, W);
  return bad;
}

int main() {
  int bad = 0;
  for (int64_t total = 0; total < 9000; ++total) bad += check<2048>(total) + check<1024>(total);
  for (int bit = 13; bit < 49; ++bit)  // 2^24 heads of 2^23 tiles and two places more each
    for (int64_t d = -40; d <= 40; ++d) bad += check<2048>((int64_t{1} << bit) + d) + check<1024>((int64_t{1} << bit) + d);
  for (uint32_t size = 1; size <= 1u << 29; size = size < 5000 ? size + 1 : size * 2 - size % 7) {
    const Pages pages(size);
    for (int bit = 0; bit < 31; ++bit)
      for (int64_t d = -3; d <= 3; ++d) {
        for (const int64_t n : {(int64_t{1} << bit) + d, ((int64_t{1} << bit) / size) * size + d})
          if (n >= 0 && n < int64_t{1} << 31 && pages.quotient(static_cast<uint32_t>(n)) != n / size) {
            if (!bad++) printf("%lld / %u\n", (long long)n, size);
          }
      }
  }
  return bad != 0;
}
"""


def test_every_place_has_its_worker(tmp_path):
    src, exe = tmp_path / "deal.cpp", tmp_path / "deal"
    src.write_text(CODE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", CSRC, str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout
