"""How the windowed attention's gradient deals out the sums of dk and dv, over swept
sizes, on the CPU: every tile of queries that sees a key is in some workgroup's list."""
import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "go-darwinml_amd", "csrc")

# Lists by the definition: the tiles with a query whose window holds a key of the block, or
# with any query at or past a sink.
COVER = r"""
#include <cstdio>
#include "attn_window_rules.h"
using namespace ghip::win;

int main() {
  long plans = 0, split = 0, far = 0;
  for (int start : {0, 1, 6, 16, 31, 32, 33, 63, 100, 127})
    for (int Sq : {1, 5, 32, 33, 64, 100, 127, 200, 257, 600})
      for (int behind : {0, 1, 40, 100})
        for (int w : {1, 2, 3, 4, 31, 32, 33, 34, 35, 50, 64, 66, 90, 97, 128, 302, 1 << 30})
          for (int G : {1, 3, 4})
            for (int BH : {1, 2, 7, 64})
              for (int sinks : {0, 1, 5, 40, 65}) {
                const int Sk = start + Sq + behind, tiles = (Sq + kT - 1) / kT;
                const SharePlan s = plan_shares(BH, G, Sq, Sk, start, w, sinks);
                ++plans;
                split += s.blocks > 0 && !s.far;
                far += s.far;
                for (int k0 = 0; k0 < Sk; k0 += kKeys) {
                  int lo = tiles, hi = 0;  // tiles with a query that sees a key of k0 .. k0 + 63
                  for (int i = 0; i < Sq; ++i)
                    if (start + i >= k0 && ((int64_t)start + i - w < k0 + kKeys - 1 || k0 < sinks)) {
                      lo = i / kT < lo ? i / kT : lo;
                      hi = i / kT + 1;
                    }
                  const int seen = hi > lo ? hi - lo : 0;
                  const int begin = near_begin(start, k0);
                  const int end = k0 < sinks ? (s.far ? near_end(Sq, start, w, k0) : tiles) : near_end(Sq, start, w, k0);
                  bool ok = seen == 0 || (begin <= lo && (end >= hi || (s.far && k0 < sinks)));
                  if (s.blocks && !s.far)  // the chunks hold the list of every head
                    ok = ok && (int64_t)s.chunks * s.chunk >= (int64_t)(end > begin ? end - begin : 0) * G;
                  if (s.far && k0 < sinks)
                    ok = ok && (int64_t)s.chunks * s.chunk >= (int64_t)(tiles - end) * G && s.blocks * 32 >= sinks;
                  if (!ok) {
                    printf("q_start %d Sq %d Sk %d window %d G %d BH %d sinks %d: keys from %d\n", start, Sq, Sk, w, G, BH,
                           sinks, k0);
                    return 1;
                  }
                }
              }
  printf("%ld plans, %ld split, %ld far\n", plans, split, far);
  return split > plans / 10 && far > plans / 50 ? 0 : 2;
}
"""


def _run(tmp_path, code):
    src, exe = tmp_path / "plan.cpp", tmp_path / "plan"
    src.write_text(code)
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", CSRC, str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr


def test_every_tile_is_in_a_list(tmp_path):
    _run(tmp_path, COVER)


def test_plans_of_aligned_starts(tmp_path):
    """The shares of a few calls whose queries begin at a whole tile: blocks, shares, chunks,
    tiles a chunk."""
    _run(tmp_path, r"""
#include "attn_window_rules.h"
using namespace ghip::win;
constexpr bool is(SharePlan s, int blocks, int shares, int chunks, int chunk, bool far) {
  return s.blocks == blocks && s.shares == shares && s.chunks == chunks && s.chunk == chunk && s.far == far;
}
static_assert(is(plan_shares(64, 1, 2048, 2048, 0, 512, 4), 1, 7, 6, 8, true), "");
static_assert(is(plan_shares(64, 1, 2048, 2048, 0, 512, 0), 0, 0, 0, 0, false), "");
static_assert(is(plan_shares(1, 4, 200, 200, 0, 64, 0), 7, 5, 5, 4, false), "");
static_assert(is(plan_shares(2, 2, 300, 332, 32, 0x40000000, 0), 11, 5, 5, 4, false), "");
int main() { return 0; }
""")
