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

// Sum of x over this lane and the lower ones: shifts within the rows of 16 lanes, then the
// rows' totals broadcast to the rows after them (one VALU instruction a step).
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_add(uint32_t x) {
  return x + static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), CTRL, ROWS, 0xf, true));
}
__device__ __forceinline__ uint32_t wave_scan(uint32_t x) {
  x = dpp_add<0x111, 0xf>(x);  // row_shr 1, 2, 4, 8
  x = dpp_add<0x112, 0xf>(x);
  x = dpp_add<0x114, 0xf>(x);
  x = dpp_add<0x118, 0xf>(x);
  x = dpp_add<0x142, 0xa>(x);  // row_bcast 15 into rows 1 and 3
  x = dpp_add<0x143, 0xc>(x);  // row_bcast 31 into rows 2 and 3
  return x;
}
__device__ __forceinline__ uint32_t lane_of(uint32_t x, int lane) {
  return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(x), lane));
}

// Where the tiles of the sequences lie in the common order (sequence, unit of heads,
// tile).  A lane counts one sequence of 64; a sequence has fewer than 2^26 tiles (the host
// checks), so 64 of them fit 32 bits.
template <int KT, int WORKERS = kWorkers>
struct Order {
  int64_t total = 0;  // tiles of all sequences and units
  int lane, units;
  int len0;           // the first 64 sequences: lengths, tiles, running sums
  uint32_t n0, up0;
  __device__ __forceinline__ Order(const Common& p, int units_) : lane(threadIdx.x & 63), units(units_) {
    if (units == 0) return;
    len0 = lane < p.B ? p.lens[lane] : 0;
    n0 = Seen(p, len0).tiles(KT);
    up0 = wave_scan(n0);
    total = lane_of(up0, 63);
    for (int b0 = 64; b0 < p.B; b0 += 64) total += lane_of(wave_scan(count(p, b0 + lane)), 63);
    total *= units;
  }
  __device__ __forceinline__ uint32_t count(const Common& p, int b) const {
    return b < p.B ? Seen(p, p.lens[b]).tiles(KT) : 0;
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
  __device__ __forceinline__ int64_t share() const { return share_of(total, WORKERS); }
};

// a / b of non-negative values, in 32 bits where they fit.
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
  if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
  return a / b;
}

// Joins the shares of units that several workers hold: a workgroup a (sequence, head),
// the shares dealt out over groups of lanes that each hold a row of the output and a
// running maximum; the groups are added in order.  Sequences without a visible token,
// which no worker holds, get zeros.
// Bound by the latency of lengths, then shares: 4.8 us for 8 x 32 heads, 6 us for 64 x 32.
template <typename T, int DP, int KT, int WORKERS, int NT = 256>
__global__ __launch_bounds__(NT) void join_kernel(Common p) {
  constexpr int kLanes = DP / 4, kGroups = NT / kLanes, kAhead = 4;
  __shared__ float stat[2][kGroups];
  __shared__ __attribute__((aligned(16))) float sums[kGroups][DP];
  const int G = p.H / p.Hkv, blocks = (G + kHeads - 1) / kHeads, units = p.Hkv * blocks;
  const int row = blockIdx.x, b = row / p.H, h = row % p.H, hk = h / G;
  const int unit = hk * blocks + (h - hk * G) / kHeads, hd = (h - hk * G) % kHeads;
  const int d = threadIdx.x % kLanes * 4, grp = threadIdx.x / kLanes;
  T* out = static_cast<T*>(p.o) + b * p.o_sb + h * p.o_sh + d;
  const Order<KT, WORKERS> order(p, units);
  const int nt = Seen(p, order.length(p, b)).tiles(KT);
  if (nt == 0) {
    if (grp == 0 && d < p.D) tile::store4(out, 0.f, 0.f, 0.f, 0.f);
    return;
  }
  const int64_t per = order.share(), u0 = order.begin(p, b) + static_cast<int64_t>(unit) * nt;
  const int w0 = static_cast<int>(quotient(u0, per)), n = static_cast<int>(quotient(u0 + nt - 1, per)) - w0 + 1;
  if (n == 1) return;
  // The unit's share in worker w0 + i: its first piece, but for a worker that began before.
  auto slot = [&](int i) {
    return (2 * static_cast<int64_t>(w0 + i) + (i == 0 && u0 != w0 * per ? 1 : 0)) * p.unit_heads + hd;
  };
  float a[4] = {0.f, 0.f, 0.f, 0.f}, mx = -INFINITY, sum = 0.f;
  for (int i0 = grp; i0 < n; i0 += kAhead * kGroups) {  // kAhead shares' loads in flight
    float ls[kAhead];
    float4 v[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int i = i0 + j * kGroups;
      ls[j] = i < n ? p.part_lse[slot(i)] : -INFINITY;
      v[j] = i < n && d < p.D ? *reinterpret_cast<const float4*>(p.part_o + slot(i) * p.D + d) : make_float4(0, 0, 0, 0);
    }
    float m = mx;
#pragma unroll
    for (int j = 0; j < kAhead; ++j) m = fmaxf(m, ls[j]);
    const float old = mx == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mx - m);
    sum *= old;
#pragma unroll
    for (int e = 0; e < 4; ++e) a[e] *= old;
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const float f = ls[j] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ls[j] - m);  // (NaN stays NaN)
      sum += f;
      a[0] += f * v[j].x;
      a[1] += f * v[j].y;
      a[2] += f * v[j].z;
      a[3] += f * v[j].w;
    }
    mx = m;
  }
  *reinterpret_cast<float4*>(&sums[grp][d]) = make_float4(a[0], a[1], a[2], a[3]);
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
    const float4 v = *reinterpret_cast<const float4*>(&sums[i][d]);
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
