// What the attentions over paged caches share: which tokens a sequence's query sees, how the
// tiles of all sequences are dealt out over the card, and how their shares are joined.
#pragma once

#include "attn_paged_rules.h"
#include "attn_tile.h"

namespace ghip {
namespace paged {

typedef float f32x4 __attribute__((ext_vector_type(4)));

// What both caches' kernels read, and how they join.
struct Common {
  const void* q;
  void* o;
  const int32_t* table;
  const int32_t* lens;
  int64_t q_sb, q_sh, o_sb, o_sh;  // element strides
  int64_t table_stride;
  int B, H, Hkv, D, num_pages, page_size, max_pages;
  int window, sinks;
  float scale;
  int unit_heads;   // min(16, heads of a kv head)
  float* part_o;    // [2 workers][unit_heads][D]: shares of units that several workers hold
  float* part_lse;  // [2 workers][unit_heads]
};

// Heads of one kv head's group that a unit of work holds: the columns of a 16-wide MFMA.
constexpr int kHeads = 16;

template <int N>
__device__ __forceinline__ void wait_vm() {
  static_assert(N < 64, "vmcnt");
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// The tokens that a sequence's query sees, in tiles of KT: those of the sinks (if a gap
// follows them), then those of the window from a multiple of 16 on.
struct Seen {
  int len, lo, ns;  // tokens [0, ns) and [lo, len)
  __device__ __forceinline__ Seen(const Common& p, int n) {
    const int64_t cap = static_cast<int64_t>(p.max_pages) * p.page_size;
    len = static_cast<int>(min(static_cast<int64_t>(max(n, 0)), cap));
    lo = max(0, len - p.window);
    ns = min(p.sinks, lo);
    if (ns == lo) lo = ns = 0;  // no gap between them
  }
  __device__ __forceinline__ int sink_tiles(int kt) const { return (ns + kt - 1) / kt; }
  __device__ __forceinline__ int tiles(int kt) const { return sink_tiles(kt) + (len - (lo & ~15) + kt - 1) / kt; }
};

__device__ __forceinline__ uint32_t lane_of(uint32_t x, int lane) {
  return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(x), lane));
}

// Where the tiles of the sequences lie in the common order (sequence, unit of heads,
// tile), with AHEAD places without a tile before each unit's.  A lane counts one sequence of
// 64; a sequence has fewer than 2^26 tiles (the host checks), so 64 of them fit 32 bits.
template <int KT, int AHEAD = 0>
struct Order {
  int64_t total = 0;  // places of all sequences and units
  int lane, units;
  int len0;           // the first 64 sequences: lengths, tiles, running sums
  uint32_t n0, up0;
  __device__ __forceinline__ Order(const Common& p, int units_) : lane(threadIdx.x & 63), units(units_) {
    if (units == 0) return;
    len0 = lane < p.B ? p.lens[lane] : 0;
    n0 = places(Seen(p, len0).tiles(KT));
    up0 = wave_scan(n0);
    total = lane_of(up0, 63);
    for (int b0 = 64; b0 < p.B; b0 += 64) total += lane_of(wave_scan(count(p, b0 + lane)), 63);
    total *= units;
  }
  static __device__ __forceinline__ uint32_t places(int tiles) { return AHEAD == 0 || tiles > 0 ? tiles + AHEAD : 0; }
  __device__ __forceinline__ uint32_t count(const Common& p, int b) const {
    return b < p.B ? places(Seen(p, p.lens[b]).tiles(KT)) : 0;
  }
  __device__ __forceinline__ int length(const Common& p, int b) const {
    return b < 64 ? static_cast<int>(lane_of(static_cast<uint32_t>(len0), b)) : p.lens[b];
  }
  // The sequence that place `at` < total lies in; *begin: where it begins.
  __device__ __forceinline__ int find(const Common& p, int64_t at, int64_t* begin) const {
    int64_t before = 0;
    for (int b0 = 0;; b0 += 64) {
      const uint32_t n = b0 ? count(p, b0 + lane) : n0, up = b0 ? wave_scan(n) : up0;
      const uint64_t over = __builtin_amdgcn_ballot_w64((before + up) * units > at);
      if (over) {
        const int l = __builtin_ctzll(over);
        *begin = (before + lane_of(up - n, l)) * units;
        return b0 + l;
      }
      before += lane_of(up, 63);
    }
  }
  // Where sequence b begins.
  __device__ __forceinline__ int64_t begin(const Common& p, int b) const {
    int64_t before = 0;
    for (int b0 = 0;; b0 += 64) {
      const uint32_t n = b0 ? count(p, b0 + lane) : n0, up = b0 ? wave_scan(n) : up0;
      if (b < b0 + 64) return (before + lane_of(up - n, b - b0)) * units;
      before += lane_of(up, 63);
    }
  }
  __device__ __forceinline__ int64_t share() const { return share_of(total); }
};

// a / b of non-negative values, in 32 bits where they fit.
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
  if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
  return a / b;
}

// A row of the output (PARTS = 1; else columns of it, by the workgroup's number) from its n
// shares, share i in slot(i): they are dealt out over groups of lanes that each hold the columns
// and a running maximum; the groups are added in order.
template <typename T, int DP, int NT, int PARTS, int AHEAD, typename Slot>
__device__ __forceinline__ void join_shares(const Common& p, T* row, int n, const Slot& slot) {
  constexpr int kCols = DP / PARTS, kLanes = kCols / 4, kGroups = NT / kLanes;
  __shared__ float stat[2][kGroups];
  __shared__ __attribute__((aligned(16))) float sums[kGroups][kCols];
  const int col = threadIdx.x % kLanes * 4, grp = threadIdx.x / kLanes;
  const int d = PARTS == 1 ? col : static_cast<int>(blockIdx.x % PARTS) * kCols + col;
  T* out = row + d;
  if (n == 0) {
    if (grp == 0 && d < p.D) tile::store4(out, 0.f, 0.f, 0.f, 0.f);
    return;
  }
  if (n == 1) return;
  float a[4] = {0.f, 0.f, 0.f, 0.f}, mx = -INFINITY, sum = 0.f;
  for (int i0 = grp; i0 < n; i0 += AHEAD * kGroups) {  // AHEAD shares' loads in flight
    float ls[AHEAD];
    float4 v[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const int i = i0 + j * kGroups;
      ls[j] = i < n ? p.part_lse[slot(i)] : -INFINITY;
      v[j] = i < n && d < p.D ? *reinterpret_cast<const float4*>(p.part_o + slot(i) * p.D + d) : make_float4(0, 0, 0, 0);
    }
    float m = mx;
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) m = fmaxf(m, ls[j]);
    const float old = mx == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mx - m);
    sum *= old;
#pragma unroll
    for (int e = 0; e < 4; ++e) a[e] *= old;
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const float f = ls[j] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ls[j] - m);  // (NaN stays NaN)
      sum += f;
      a[0] += f * v[j].x;
      a[1] += f * v[j].y;
      a[2] += f * v[j].z;
      a[3] += f * v[j].w;
    }
    mx = m;
  }
  *reinterpret_cast<float4*>(&sums[grp][col]) = make_float4(a[0], a[1], a[2], a[3]);
  if (threadIdx.x % kLanes == 0) {
    stat[0][grp] = mx;
    stat[1][grp] = sum;
  }
  __syncthreads();
  if (grp != 0 || d >= p.D) return;
  float m = stat[0][0];
#pragma unroll
  for (int i = 1; i < kGroups; ++i) m = fmaxf(m, stat[0][i]);
  sum = 0.f;
  a[0] = a[1] = a[2] = a[3] = 0.f;
#pragma unroll
  for (int i = 0; i < kGroups; ++i) {
    const float f = stat[0][i] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(stat[0][i] - m);
    const float4 v = *reinterpret_cast<const float4*>(&sums[i][col]);
    sum += f * stat[1][i];
    a[0] += f * v.x;
    a[1] += f * v.y;
    a[2] += f * v.z;
    a[3] += f * v.w;
  }
  const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
  tile::store4(out, a[0] * inv, a[1] * inv, a[2] * inv, a[3] * inv);
}

}  // namespace paged
}  // namespace ghip
