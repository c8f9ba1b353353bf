"""How rotations and appends deal their rows out, on the CPU: the sizes of the tests that run on the
device reach every form (rows a slot, tokens of a workgroup, split tokens, one workgroup for both
kinds of rows), and the parts hold all rows, few more than a part has slots for."""
import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "go-darwinml_amd", "csrc")

CODE = r"""
#include <cstdio>
#include "rope_rules.h"
using namespace ghip::rope;

static int bad = 0;

Deal dealt(int64_t tokens, int64_t H, int64_t Hkv, int D, int R, int vec, bool four) {
  int n = width(D, R / 2, vec);
  if (four && n < vec) n = 1;
  return deal(tokens, H, Hkv, (D + 2 * n - 1) / (2 * n), D / 8, four);
}

void expect(int64_t tokens, int64_t H, int64_t Hkv, int D, int R, int vec, bool four, int block, int splits, int splits4, int both) {
  const Deal d = dealt(tokens, H, Hkv, D, R, vec, four);
  if (d.block_tokens == block && d.splits == splits && d.splits4 == splits4 && d.both == both) return;
  ++bad;
  printf("%lld tokens, %lld + %lld heads of %d, four %d: %d %d %d %d\n", (long long)tokens, (long long)H, (long long)Hkv, D, four,
         d.block_tokens, d.splits, d.splits4, d.both);
}

int main() {
  // Prompts (bf16, f16: vectors of 8; fp32: 4), into 16 and into 4 bits.
  expect(7 * 1171, 8, 2, 64, 64, 8, false, 10, 1, 0, 0);
  expect(7 * 1171, 8, 2, 64, 64, 8, true, 16, 1, 0, 1);
  expect(7 * 1171, 32, 8, 128, 128, 8, false, 2, 1, 0, 0);
  expect(7 * 1171, 32, 8, 128, 128, 8, true, 3, 1, 0, 1);
  expect(7 * 1171, 32, 8, 128, 128, 4, false, 1, 1, 0, 0);
  expect(9 * 5003, 1, 1, 32, 32, 8, false, 16, 1, 0, 0);
  expect(9 * 5003, 1, 1, 32, 32, 8, true, 16, 1, 0, 1);
  expect(7 * 2411, 0, 2, 64, 32, 8, false, 16, 1, 0, 0);
  expect(7 * 2411, 0, 2, 64, 32, 8, true, 16, 0, 1, 0);
  expect(2 * 3001, 24, 4, 96, 24, 8, true, 1, 2, 1, 0);
  expect(31 * 67, 4, 4, 256, 256, 8, false, 2, 1, 0, 0);
  expect(31 * 67, 4, 4, 256, 256, 8, true, 2, 1, 0, 1);
  // Rotation alone, three rows a slot.
  expect(2 * 8999, 16, 0, 128, 128, 8, false, 6, 1, 0, 0);
  expect(2 * 8999, 16, 0, 128, 128, 4, false, 3, 1, 0, 0);
  // Single tokens: one row a slot, tokens split over workgroups where their rows are many.
  expect(16, 32, 8, 128, 128, 8, false, 1, 2, 0, 0);
  expect(16, 32, 8, 128, 128, 8, true, 1, 1, 1, 0);
  for (int64_t tokens = 1; tokens < 1 << 22; tokens = tokens * 2 + tokens % 3)
    for (int64_t H = 0; H <= 300; H += 1 + H / 3)
      for (int64_t Hkv = 0; Hkv <= 64; Hkv += 1 + Hkv)
        for (int D = 1; D <= 256; D += D < 8 ? 1 : D % 32 ? 32 - D % 32 : 32)
          for (int four = 0; four < 2; ++four) {
            if ((four && (D % 32 || Hkv == 0)) || H + Hkv == 0) continue;
            const Deal d = dealt(tokens, H, Hkv, D, D / 2 * 2, 8, four);
            const int64_t rows = H + (four ? 0 : 2 * Hkv), rows4 = four ? 2 * Hkv : 0;
            bool ok = d.block_tokens >= 1 && d.block_tokens <= kMostTokens;
            ok = ok && (rows > 0) == (d.splits > 0) && (d.both ? d.splits == 1 : (rows4 > 0) == (d.splits4 > 0));
            ok = ok && (d.block_tokens == 1 || (d.splits <= 1 && d.splits4 <= 1));
            ok = ok && (d.splits <= rows || rows == 0) && d.splits + d.splits4 > 0;
            if (!ok && bad++ < 10) printf("%lld %lld %lld %d %d\n", (long long)tokens, (long long)H, (long long)Hkv, D, four);
          }
  return bad != 0;
}
"""


def test_rows_are_dealt_out(tmp_path):
    src, exe = tmp_path / "deal.cpp", tmp_path / "deal"
    src.write_text(CODE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I", CSRC, str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout
