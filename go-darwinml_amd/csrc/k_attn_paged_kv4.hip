// Decoding attention over a paged key-value cache of 4 bits.
//
//   o[b, h] = sum_j softmax_j(scale q[b, h].K_b[j]) V_b[j]   over the tokens j that the last
//   token of sequence b sees; K and V as kv4_dev.h defines the cache's values
//
// The values have two significant bits and a power of two, so bf16 holds them exactly: both
// products run on bf16 matrix instructions for queries of every type, which are split into
// bf16 parts (bf16: 1, f16: 2, fp32: 3), and so are the weights (2, 2, 3).  No reference op.
// Bound by the bytes of the codes and scales, of which a value has 4.25 bits.
#include <algorithm>
#include <type_traits>

#include "attn_paged.h"
#include "kv4_dev.h"

namespace ghip {
namespace paged4 {

using paged::Common;
using paged::f32x4;
using paged::kHeads;
using paged::Order;
using paged::quotient;
using paged::Seen;
using paged::wait_vm;

struct Rows {
  const char* codes;
  const char* scales;
  uint32_t sp, st;    // byte strides of page and token of the codes
  uint32_t ssp, sst;  // and of the scales
  int64_t sh, ssh;    // of the heads
};

struct Params : Common {
  Rows k, v;
  Pages pages;  // of page_size tokens
  int2* held;   // [B][units]: slot of a unit's first share, number of its shares
};

constexpr int kTile = 64;  // tokens of a tile

// Waves that share the tiles of all sequences: eight a CU, four with rows of 128 bytes (registers).
constexpr int workers(int DP) { return DP == 256 ? 1024 : 2048; }

// A row of zeros: what lanes without a token load.
__device__ const uint4 kZero4[8] = {};

template <typename T> struct Parts;
// bf16 parts of the queries, and of the weights: their rounding stays below that of the output.
template <> struct Parts<bf16_t> { static constexpr int kQ = 1, kP = 2; };
template <> struct Parts<f16_t> { static constexpr int kQ = 2, kP = 2; };
template <> struct Parts<float> { static constexpr int kQ = 3, kP = 3; };

// x as the sum of N bf16 values (the last one rounds: 2^-9, 2^-17 or 2^-25 of x).  CUT: those before the
// last are cut off, not rounded (three hold an fp32 value's 24 bits either way), so neither they
// nor their sums pass x: near fp32's largest values a rounded part, or it and the next one, is infinite.
template <int N, bool CUT = false>
__device__ __forceinline__ void split8(const float (&x)[8], tile::bf16x8 (&out)[N]) {
  float r[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) r[e] = x[e];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (CUT && n + 1 < N) w[i] = (__float_as_uint(r[2 * i]) >> 16) | (__float_as_uint(r[2 * i + 1]) & 0xffff0000u);
      else w[i] = pack_bf16x2(r[2 * i], r[2 * i + 1]);
      if (n + 1 < N) {
        r[2 * i] -= __uint_as_float(w[i] << 16);
        r[2 * i + 1] -= __uint_as_float(w[i] & 0xffff0000u);
      }
    }
    out[n] = __builtin_bit_cast(tile::bf16x8, make_uint4(w[0], w[1], w[2], w[3]));
  }
}

__device__ __forceinline__ f32x4 mma(const tile::bf16x8& a, const tile::bf16x8& b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// Another lane's pointer.
__device__ __forceinline__ const char* from_lane(const char* x, int lane) {
  const uint64_t u = reinterpret_cast<uint64_t>(x);
  const uint32_t lo = __builtin_amdgcn_ds_bpermute(4 * lane, static_cast<int>(u));
  const uint32_t hi = __builtin_amdgcn_ds_bpermute(4 * lane, static_cast<int>(u >> 32));
  return reinterpret_cast<const char*>(static_cast<uint64_t>(hi) << 32 | lo);
}

// The bytes of a row that hold N values, a lane's share of V.
template <int N> struct Word;
template <> struct Word<4> { using type = uint16_t; };
template <> struct Word<8> { using type = uint32_t; };
template <> struct Word<16> { using type = uint2; };

template <int B>
__device__ __forceinline__ uint32_t decode_byte(uint32_t w, float s) {
  return kv4::decode2<B>(w, s);
}
template <int B>
__device__ __forceinline__ uint32_t decode_byte(uint2 w, float s) {
  return kv4::decode2<(B & 3)>(B < 4 ? w.x : w.y, s);
}

// A wave works alone on tiles of 64 tokens: codes and scales come by per-lane DMA into LDS, from
// there all of the tile goes to registers, and the next tile's DMA runs while it is computed; page
// numbers come one tile further ahead.  S^T = K Q^T, 16 tokens x 16 heads a
// product: lane (c, g) has a quarter g of token c's row, so the contraction runs over d in the
// order quarter, word, value.  O^T += V^T P^T: lane (c, g) has DP / 16 consecutive values of
// tokens 4 g .. 4 g + 3 and 16 more; a conversion makes two of one token, a byte permute
// joins those of two tokens, and product j holds the j-th value of every lane.
// LDS: 16 rows lie in the order 0, 4, 8, 12, 1, ..: the four that one read of V touches
// are neighbours; their 16-byte chunks are exchanged so that a read of K by 16 lanes meets
// every bank once.
// Bound by the bytes and by what comes before and after them: bf16 D 128, 32 heads over 8, 64
// sequences of up to 8192 tokens (291 MB) 62 us; a thousand tokens more each cost their bytes at
// 5.6 TB/s, the rest, 10 us, is the launch, the chain lengths - pages - rows on cold caches
// and the last tiles.  A tile is 500 instructions (67k of 119k cycles of a CU) beside 25k cycles
// of matrix instructions.  Two LDS stages instead of one: 4% slower; three and four waves a
// SIMD: 1% and 55% slower (their registers spill).
template <typename T, int DP, bool SPLIT>
__global__ __launch_bounds__(64, DP == 256 ? 1 : 2) void attend4_kernel(Params p) {
  constexpr int kQ = Parts<T>::kQ, kP = Parts<T>::kP;
  constexpr int kRow = DP / 2, kCh = kRow / 16;         // bytes and 16-byte chunks of a row's codes
  constexpr int kPlanes = DP == 256 ? 2 : 1;            // words of a row's scales
  constexpr int kDma = kTile * kRow / 1024, kPer = 64 / kCh;  // DMA instructions of K's codes, rows of one
  constexpr int kCodes = kTile * kRow, kStage = 2 * kCodes + 2 * kPlanes * 4 * kTile;
  constexpr int kWords = kRow / 16;                     // words of a quarter of a row
  constexpr int kVals = DP / 16;                        // values of V a lane holds of a token
  constexpr int kQuarterGroups = DP == 256 ? 2 : 1;     // scales of a quarter of a row
  __shared__ __attribute__((aligned(1024))) char smem[kStage];
  __shared__ __attribute__((aligned(16))) int32_t page_lds[2][64];

  const int lane = threadIdx.x, g = lane >> 4, col = lane & 15;
  const int G = p.H / p.Hkv, blocks = (G + kHeads - 1) / kHeads, units = p.Hkv * blocks;
  const uint32_t la0 = tile::lds_addr(smem), pa0 = tile::lds_addr(page_lds);
  const float c = p.scale * 1.4426950408889634f;
  const int groups = p.D / kv4::kGroup;
  // A scale's byte as an fp32 power of two; groups past the head dim have none, whatever lies there.
  auto scale_of = [&](uint32_t byte, int group) {
    return __uint_as_float(__umul24(byte, group < groups ? 1u << 23 : 0u));
  };
  auto slot_of = [](int r) { return (r & ~15) | ((r & 3) << 2) | ((r >> 2) & 3); };  // (its own inverse)
  auto swz = [](int s) { return s / (256 / kRow) % kCh; };  // (the same for slots 16 apart)
  const int kslot = slot_of(col);

  int b;
  int64_t at, end, begin;
  const Order<kTile, kBegin> order(p, SPLIT ? units : 0);
  int worker = 0, used = 0;
  if constexpr (SPLIT) {
    // Workgroups go to the eight XCDs in turn; each XCD takes neighbouring workers, so that heads
    // whose rows share cache lines meet in one L2.  (Rows of all heads side by side, 64 x 8192
    // tokens: 197 to 164 us by that alone; a head's rows side by side took the same either way.)
    used = used_of(order.total, workers(DP));
    const int each = (used + 7) >> 3;
    worker = static_cast<int>(blockIdx.x & 7) * each + static_cast<int>(blockIdx.x >> 3);
    if (static_cast<int>(blockIdx.x >> 3) >= each || worker >= used || order.total == 0) return;
    at = first_of<workers(DP)>(worker, order.total, used);
    end = first_of<workers(DP)>(worker + 1, order.total, used);
    b = order.find(p, at, &begin);
  } else {
    b = blockIdx.x / units;
    begin = 0;
    at = end = 0;
  }
  const int64_t first = at;

  for (;;) {
    const Seen seen(p, SPLIT ? order.length(p, b) : p.lens[b]);
    const int nt = seen.tiles(kTile), nst = seen.sink_tiles(kTile);
    int unit, ta, te, taken = 0;
    if constexpr (SPLIT) {
      const int nv = nt + kBegin;
      unit = static_cast<int>(quotient(at - begin, nv));
      const int from = static_cast<int>(at - begin - static_cast<int64_t>(unit) * nv);
      const int to = static_cast<int>(min(static_cast<int64_t>(nv), from + (end - at)));
      taken = to - from;
      ta = max(0, from - kBegin);
      te = to - kBegin;
      if (te <= 0) return;  // (nothing but the unit's beginning: the end of this worker's part)
    } else {
      unit = blockIdx.x % units;
      ta = 0;
      te = nt;
    }
    const int hk = unit / blocks, h0 = hk * G + (unit % blocks) * kHeads;
    const int heads = min(kHeads, (hk + 1) * G - h0);
    if constexpr (SPLIT) {
      // (For the join, which would else have to find the unit's place among all sequences.)
      if (ta == 0 && lane == 0) {
        const int64_t last = begin + static_cast<int64_t>(unit + 1) * (nt + kBegin) - 1;
        const int n = worker_of(last, order.total, used) - worker + 1;
        p.held[static_cast<int64_t>(b) * units + unit] = make_int2(2 * worker + (at == first ? 0 : 1), n);
      }
    }

    const int32_t* table = p.table + b * p.table_stride;
    const char* kc = p.k.codes + hk * p.k.sh;
    const char* vc = p.v.codes + hk * p.v.sh;
    const char* ks = p.k.scales + hk * p.k.ssh;
    const char* vs = p.v.scales + hk * p.v.ssh;
    const char* zero = reinterpret_cast<const char*>(kZero4);

    auto token0 = [&](int t) { return t < nst ? t * kTile : (seen.lo & ~15) + (t - nst) * kTile; };
    auto issue_pages = [&](int t, int slot) {
      const int entry = min(p.pages.quotient(token0(t) + lane), p.max_pages - 1);
      tile::load4(table + entry, pa0 + slot * 256);
    };
    // The DMA of tile t, its page numbers landed; returns its rows that hold a token.  A lane finds
    // the addresses of its token's rows, those that load them fetch them from it.
    auto issue = [&](int t, int slot) -> uint64_t {  // (page numbers from `slot`)
      const int tok = token0(t) + lane;
      const int page = page_lds[slot][lane];
      const uint32_t off = tok - p.pages.quotient(tok) * p.page_size;
      // No branches here: where lanes part, the compiler has put copies of registers in front of the
      // instruction that brings all lanes back, and those of the lanes that had left were lost.
      const int from = t < nst ? 0 : seen.lo, to = t < nst ? seen.ns : seen.len;
      const bool ok = (tok >= from) & (tok < to) & (page >= 0) & (page < p.num_pages);
      const uint32_t pg = ok ? page : 0;
      auto row = [&](const char* base, uint32_t sp, uint32_t st) {
        uint64_t at = reinterpret_cast<uint64_t>(base) + static_cast<uint64_t>(pg) * sp + static_cast<uint64_t>(off) * st;
        asm volatile("" : "+v"(at));  // (computed for all lanes, then selected)
        return ok ? reinterpret_cast<const char*>(at) : zero;
      };
      const char* krow = row(kc, p.k.sp, p.k.st);
      const char* vrow = row(vc, p.v.sp, p.v.st);
#pragma unroll
      for (int i = 0; i < kDma; ++i) {
        const int s = i * kPer + lane / kCh, r = slot_of(s);
        // (Past the head dim: any bytes of the row; their scales count as 2^-127 and q as 0.)
        const int ch = min((lane % kCh) ^ swz(s), groups - 1) * 16;
        tile::load16(from_lane(krow, r) + ch, la0 + i * 1024);
        tile::load16(from_lane(vrow, r) + ch, la0 + kCodes + i * 1024);
      }
      const char* kscale = row(ks, p.k.ssp, p.k.sst);
      const char* vscale = row(vs, p.v.ssp, p.v.sst);
#pragma unroll
      for (int i = 0; i < kPlanes; ++i) {
        tile::load4(kscale + 4 * i, la0 + 2 * kCodes + i * 256);
        tile::load4(vscale + 4 * i, la0 + 2 * kCodes + (kPlanes + i) * 256);
      }
      return __builtin_amdgcn_ballot_w64(ok);
    };

    f32x4 o[kVals];
#pragma unroll
    for (int j = 0; j < kVals; ++j) o[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;

    const int n = te - ta;
    uint64_t next = 0;  // the rows of the tile under way
    if (n > 0) {
      issue_pages(ta, 0);
      if (n > 1) issue_pages(ta + 1, 1);
    }
    tile::bf16x8 qf[kVals / 2][kQ];  // [step][part]
    {
      // (Without branches, so that the loads are under way at once; columns without a head load the last.)
      const T* Q = static_cast<const T*>(p.q) + b * p.q_sb + (h0 + min(col, heads - 1)) * p.q_sh;
      float x[kVals / 2][8];
#pragma unroll
      for (int s = 0; s < kVals / 2; ++s) {
        const int d = g * (DP / 4) + 8 * s;
#pragma unroll
        for (int i = 0; i < 8; i += Elem<T>::kVec) load_vec(Q + (d < p.D ? d : 0) + i, x[s] + i);
      }
#pragma unroll
      for (int s = 0; s < kVals / 2; ++s) {
        const bool in = (col < heads) & (g * (DP / 4) + 8 * s < p.D);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[s][e] = in ? x[s][e] : 0.f;
        split8<kQ, __is_same(T, float)>(x[s], qf[s]);
      }
#pragma unroll
      for (int s = 0; s < kVals / 2; ++s) tile::settle(qf[s]);
    }
    if (n > 0) {
      wait_vm<0>();
      next = issue(ta, 0);
    }
    for (int j = 0; j < n; ++j) {
      wait_vm<0>();  // tile j, and the pages of j + 1
      const char* sk = smem;
      const char* sv = sk + kCodes;
      const uint8_t* ssk = reinterpret_cast<const uint8_t*>(sk + 2 * kCodes);
      const uint8_t* ssv = ssk + kPlanes * 256;
      uint32_t kw[4][kWords];
      float kscale[4][kQuarterGroups];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const char* row = sk + i * 16 * kRow + kslot * kRow;  // token 16 i + col
        if constexpr (kWords == 2) {
          const uint2 v = *reinterpret_cast<const uint2*>(row + (((g >> 1) ^ swz(kslot)) << 4) + (g & 1) * 8);
          kw[i][0] = v.x;
          kw[i][1] = v.y;
        } else {
#pragma unroll
          for (int u = 0; u < kWords / 4; ++u) {
            const uint4 v = *reinterpret_cast<const uint4*>(row + ((((kWords / 4) * g + u) ^ swz(kslot)) << 4));
            kw[i][4 * u] = v.x;
            kw[i][4 * u + 1] = v.y;
            kw[i][4 * u + 2] = v.z;
            kw[i][4 * u + 3] = v.w;
          }
        }
#pragma unroll
        for (int u = 0; u < kQuarterGroups; ++u) {
          const int group = g * (DP / 4) / kv4::kGroup + u;
          kscale[i][u] = scale_of(ssk[64 * i + 4 * col + (group >> 2) * 256 + (group & 3)], group);
        }
      }
      typename Word<kVals>::type vw[2][8];
      float vscale[2][8];
      const int vgroup = col * kVals / kv4::kGroup;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 8; ++e) {  // token 32 t + 16 (e / 4) + 4 g + e % 4, in slot .. + 4 (e % 4) + g
          const int s = 4 * (e & 3) + g, byte = col * (kVals / 2);
          vw[t][e] = *reinterpret_cast<const typename Word<kVals>::type*>(
              sv + (32 * t + 16 * (e >> 2) + 4 * (e & 3)) * kRow + g * kRow + (((byte >> 4) ^ swz(s)) << 4) + (byte & 15));
          const int at = 4 * (32 * t + 16 * (e >> 2) + (e & 3)) + 16 * g;
          vscale[t][e] = scale_of(ssv[at + (vgroup >> 2) * 256 + (vgroup & 3)], vgroup);
        }
      const uint64_t rows = next;
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (j + 1 < n) {
        if (j + 2 < n) issue_pages(ta + j + 2, j & 1);
        next = issue(ta + j + 1, (j + 1) & 1);
      }
      f32x4 x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int u = 0; u < kWords; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint4 values = kv4::decode8(kw[i][u], kscale[i][u * kQuarterGroups / kWords]);
          const tile::bf16x8 kf = __builtin_bit_cast(tile::bf16x8, values);
#pragma unroll
          for (int q = 0; q < kQ; ++q) x[i] = mma(kf, qf[u][q], x[i]);
        }
      // x[i][v]: token 16 i + 4 g + v, head col.
      if (rows != ~0ull) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t bits = static_cast<uint32_t>(rows >> (16 * i + 4 * g));
#pragma unroll
          for (int v = 0; v < 4; ++v) x[i][v] = (bits >> v) & 1 ? x[i][v] : -INFINITY;
        }
      }
      float mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < 4; ++i) mx = fmaxf(fmaxf(fmaxf(x[i][0], x[i][1]), fmaxf(x[i][2], x[i][3])), mx);
      if (__builtin_amdgcn_ballot_w64((mx - m) * c > 8.f)) {  // the maximum may trail by 2^8
        mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const float mnew = fmaxf(m, mx);
        const float alpha = mnew == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - mnew) * c);
        m = mnew;
        l *= alpha;
#pragma unroll
        for (int d = 0; d < kVals; ++d)
#pragma unroll
          for (int v = 0; v < 4; ++v) o[d][v] *= alpha;
      }
      const float nb = m == -INFINITY ? 0.f : -m * c;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        // The weights, at most 2^8, are rounded for the product with V only (to 16 or 24 bits);
        // their sum is not.
        float w8[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          w8[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[2 * t + (e >> 2)][e & 3], c, nb));
          l += w8[e];
        }
        tile::bf16x8 pf[kP];
        split8<kP>(w8, pf);
        auto product = [&](auto B) {
          constexpr int kB = decltype(B)::value;
          uint32_t pair[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) pair[e] = decode_byte<kB>(vw[t][e], vscale[t][e]);
          uint32_t lo[4], hi[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            lo[i] = __builtin_amdgcn_perm(pair[2 * i + 1], pair[2 * i], 0x05040100u);
            hi[i] = __builtin_amdgcn_perm(pair[2 * i + 1], pair[2 * i], 0x07060302u);
          }
          const tile::bf16x8 vl = __builtin_bit_cast(tile::bf16x8, make_uint4(lo[0], lo[1], lo[2], lo[3]));
          const tile::bf16x8 vh = __builtin_bit_cast(tile::bf16x8, make_uint4(hi[0], hi[1], hi[2], hi[3]));
#pragma unroll
          for (int q = 0; q < kP; ++q) {
            o[2 * kB] = mma(vl, pf[q], o[2 * kB]);
            o[2 * kB + 1] = mma(vh, pf[q], o[2 * kB + 1]);
          }
        };
        product(std::integral_constant<int, 0>{});
        product(std::integral_constant<int, 1>{});
        if constexpr (kVals >= 8) {
          product(std::integral_constant<int, 2>{});
          product(std::integral_constant<int, 3>{});
        }
        if constexpr (kVals >= 16) {
          product(std::integral_constant<int, 4>{});
          product(std::integral_constant<int, 5>{});
          product(std::integral_constant<int, 6>{});
          product(std::integral_constant<int, 7>{});
        }
      }
    }

    // o[j][v] is d = kVals (4 g + v) + j of head col.
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;  // no token seen: zeros
    if (col < heads) {
      const bool whole = ta == 0 && te == nt;
      const int64_t r = (2 * static_cast<int64_t>(worker) + (at == first ? 0 : 1)) * p.unit_heads + col;
      T* out = static_cast<T*>(p.o) + b * p.o_sb + (h0 + col) * p.o_sh;
      float* part = SPLIT ? p.part_o + r * p.D : nullptr;
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const int d = kVals * (4 * g + v);
#pragma unroll
        for (int j = 0; j < kVals; j += 4) {
          if (d + j >= p.D) continue;
          const float a0 = o[j][v] * inv, a1 = o[j + 1][v] * inv, a2 = o[j + 2][v] * inv, a3 = o[j + 3][v] * inv;
          if (!SPLIT || whole) tile::store4(out + d + j, a0, a1, a2, a3);
          else tile::store4(part + d + j, a0, a1, a2, a3);
        }
      }
      if (SPLIT && !whole && g == 0) p.part_lse[r] = l > 0.f || l != l ? m * c + __builtin_amdgcn_logf(l) : -INFINITY;
    }
    if constexpr (!SPLIT) {
      return;
    } else {
      at += taken;
      if (at >= end) return;
      if (at - begin >= static_cast<int64_t>(nt + kBegin) * units) b = order.find(p, at, &begin);
    }
  }
}

// Joins the shares of units that several workers hold: a workgroup a (sequence, head) and one of
// PARTS column ranges.  Sequences without a visible token, which no worker holds, get zeros.
// Bound by the latency of a unit's place, then of its shares: 5.2 us for 64 x 32 rows.  Few rows have
// many shares each: 32 of one long sequence, 256 each, 4.9 us in four parts, 10 in one.
template <typename T, int DP, int PARTS, int AHEAD>
__global__ __launch_bounds__(256) void join4_kernel(Params p) {
  const int G = p.H / p.Hkv, blocks = (G + kHeads - 1) / kHeads, units = p.Hkv * blocks;
  const int row = blockIdx.x / PARTS, b = row / p.H, h = row % p.H, hk = h / G;
  const int unit = hk * blocks + (h - hk * G) / kHeads, hd = (h - hk * G) % kHeads;
  const int len = p.lens[b];
  const int2 held = p.held[static_cast<int64_t>(b) * units + unit];
  // The first share is where the worker that began the unit says, the others are in the first slots
  // of the workers after it.
  paged::join_shares<T, DP, 256, PARTS, AHEAD>(
      p, static_cast<T*>(p.o) + b * p.o_sb + h * p.o_sh, Seen(p, len).tiles(kTile) == 0 ? 0 : held.y, [&](int i) {
        return static_cast<int64_t>(i == 0 ? held.x : (held.x & ~1) + 2 * i) * p.unit_heads + hd;
      });
}

template <typename T, int DP>
static void launch_d(const Params& p, hipStream_t s) {
  const int G = p.H / p.Hkv, units = p.Hkv * ((G + kHeads - 1) / kHeads);
  if (p.part_o) {
    hipLaunchKernelGGL((attend4_kernel<T, DP, true>), dim3(workers(DP)), dim3(64), 0, s, p);
    const unsigned rows = static_cast<unsigned>(p.B * p.H);
    constexpr int kParts = DP / 32;
    if (rows <= 128) hipLaunchKernelGGL((join4_kernel<T, DP, kParts, 8>), dim3(rows * kParts), dim3(256), 0, s, p);
    else hipLaunchKernelGGL((join4_kernel<T, DP, 1, 4>), dim3(rows), dim3(256), 0, s, p);
  } else {
    hipLaunchKernelGGL((attend4_kernel<T, DP, false>), dim3(static_cast<unsigned>(p.B * units)), dim3(64), 0, s, p);
  }
}
template <typename T>
static void launch(const Params& p, hipStream_t s) {
  if (p.D <= 64) launch_d<T, 64>(p, s);
  else if (p.D <= 128) launch_d<T, 128>(p, s);
  else launch_d<T, 256>(p, s);
}

}  // namespace paged4
}  // namespace ghip

using namespace ghip;

// No workspace, so a wave for each unit: caches of at most 6 tiles a sequence, 12 with 512 units
// or more, 24 with 1024.  (The second kernel costs 5-7 us; a wave alone takes 1.4 us a tile.)
// bf16 D 128, 32 heads over 8, sequences of one length, us a call in a graph, split / unsplit:
//   units      4 tiles      6           8           12          16          24          32
//   8          11.8 / 8.8   11.8 / 11.6 11.9 / 14.3 11.9 / 19.9 11.8 / 25.3 12.0 / 36.1 11.9 / 46.8
//   256        12.3 / 9.2   12.9 / 11.8 15.1 / 14.8 16.4 / 20.2 18.9 / 26.1 22.5 / 36.9 24.7 / 47.7
//   512        16.3 / 9.6   17.4 / 12.3 19.8 / 16.1 23.0 / 21.9 25.7 / 27.3 31.1 / 39.0 35.2 / 49.4
//   1024       22.7 / 11.7  26.0 / 14.7 28.6 / 17.5 33.1 / 23.4 38.1 / 28.9 47.8 / 40.2 59.2 / 52.4
//   2048       30.3 / 17.2  34.4 / 21.7 39.6 / 26.5 48.8 / 36.4 59.6 / 47.3 93.5 / 81.0 119 / 105
// (Beyond, sequences of one length would still run faster unsplit with 1024 units and more; the
// rule does not know the lengths, and one long sequence would keep the others waiting.)
extern "C" int64_t ghip_sdpa_paged_kv4_workspace_bytes(int64_t B, int64_t H, int64_t Hkv, int64_t D, int64_t page_size,
                                                       int64_t max_pages) {
  if (B <= 0 || Hkv <= 0 || H < Hkv || D <= 0 || D > 256 || page_size <= 0 || max_pages <= 0) return 0;
  const int64_t heads = H / Hkv;
  const int64_t blocks = (heads + paged::kHeads - 1) / paged::kHeads;
  const double units = static_cast<double>(B) * static_cast<double>(Hkv) * static_cast<double>(blocks);
  if (units > tile::kMostGroups) return 0;  // (more than the entry point takes)
  const double tokens = static_cast<double>(page_size) * static_cast<double>(max_pages);
  if (tokens <= paged4::kTile * (units >= 1024 ? 24. : units >= 512 ? 12. : 6.)) return 0;
  return 2 * static_cast<int64_t>(paged4::workers(D <= 128 ? 128 : 256)) * std::min<int64_t>(paged::kHeads, heads) * (D + 1) * 4 +
         8 * B * Hkv * blocks;
}

extern "C" int ghip_sdpa_paged_kv4(int dtype, const void* q, const GHipKv4* k_cache, const GHipKv4* v_cache, void* o,
                                   int64_t B, int64_t H, int64_t Hkv, int64_t D, int64_t num_pages, int64_t page_size,
                                   int64_t max_pages, const int32_t* block_table, int64_t table_stride,
                                   const int32_t* lens, const int64_t* q_strides, const int64_t* o_strides,
                                   int64_t window, int64_t sinks, float scale, void* workspace, int64_t workspace_bytes,
                                   void* stream, GHipError* err) {
  static const char kWhat[] = "sdpa_paged_kv4";
  if (B < 0 || H <= 0 || Hkv <= 0 || D <= 0 || num_pages < 0 || page_size <= 0 || max_pages < 0)
    return set_error(err, GHIP_ERR_INVALID_ARG, "%s: bad sizes", kWhat);
  if (H % Hkv != 0)
    return set_error(err, GHIP_ERR_INVALID_ARG, "%s: num_heads (%lld) must be a multiple of num_kv_heads (%lld)", kWhat,
                     static_cast<long long>(H), static_cast<long long>(Hkv));
  if (window < 0 || sinks < 0)
    return set_error(err, GHIP_ERR_INVALID_ARG, "%s: window and sinks must not be negative", kWhat);
  if (!(scale > 0.f) || !(scale < 1e30f))
    return set_error(err, GHIP_ERR_INVALID_ARG, "%s: the scale must be positive and finite", kWhat);
  const bool f32 = dtype == GHIP_DTYPE_FLOAT32;
  if (!f32 && dtype != GHIP_DTYPE_BFLOAT16 && dtype != GHIP_DTYPE_FLOAT16)
    return set_error(err, GHIP_ERR_UNSUPPORTED, "%s: needs float32, bfloat16 or float16", kWhat);
  if (D % kv4::kGroup != 0 || D > 256)
    return set_error(err, GHIP_ERR_UNSUPPORTED, "%s: needs a head dim that is a multiple of 32 up to 256", kWhat);
  constexpr int64_t kMost = int64_t{1} << 30;
  if (num_pages > kMost || page_size > kMost || max_pages > kMost || page_size * max_pages > kMost / 2 ||
      B > kMost || H > kMost || B * H > tile::kMostGroups)
    return set_error(err, GHIP_ERR_UNSUPPORTED,
                     "%s: at most 2^30 pages, 2^29 tokens of a sequence and fewer than 2^24 heads of all sequences", kWhat);
  if (B == 0) return GHIP_OK;
  if (!q || !o || !lens || !q_strides || !o_strides || !k_cache || !v_cache || !block_table || !k_cache->codes ||
      !k_cache->scales || !v_cache->codes || !v_cache->scales)
    return set_error(err, GHIP_ERR_INVALID_ARG, "%s: null pointer", kWhat);
  if (num_pages == 0 || max_pages == 0)
    return set_error(err, GHIP_ERR_INVALID_ARG, "%s: a cache without pages", kWhat);
  if (table_stride < 0) return set_error(err, GHIP_ERR_INVALID_ARG, "%s: negative table stride", kWhat);
  const int64_t es = f32 ? 4 : 2;
  auto al = [](const void* ptr, uintptr_t a) { return (reinterpret_cast<uintptr_t>(ptr) & (a - 1)) == 0; };
  // (An axis of one entry may have any stride that is not negative.)
  auto whole = [](int64_t stride, int64_t n, int64_t of) { return stride >= 0 && (n <= 1 || stride % of == 0); };
  const int64_t cache[3] = {num_pages, Hkv, page_size}, rows[2] = {B, H};
  bool ok = al(q, 16) && al(o, 4 * es);
  for (int i = 0; i < 2; ++i) ok = ok && whole(q_strides[i], rows[i], 16 / es) && whole(o_strides[i], rows[i], 4);
  if (!ok)
    return set_error(err, GHIP_ERR_UNSUPPORTED,
                     "%s: q must be 16-byte aligned with non-negative strides of whole 16 bytes, o aligned to 4 elements "
                     "with strides of whole 4", kWhat);
  paged4::Params p{};
  paged4::Rows* to[2] = {&p.k, &p.v};
  const GHipKv4* from[2] = {k_cache, v_cache};
  bool near = true;
  for (int j = 0; j < 2; ++j) {
    const GHipKv4& f = *from[j];
    ok = ok && al(f.codes, 16) && al(f.scales, 4);
    for (int i = 0; i < 3; ++i) ok = ok && whole(f.code_strides[i], cache[i], 16) && whole(f.scale_strides[i], cache[i], 4);
    // (A cache of one page, or pages of one token: that stride is not used.)
    const int64_t steps[4] = {num_pages > 1 ? f.code_strides[0] : 0, page_size > 1 ? f.code_strides[2] : 0,
                              num_pages > 1 ? f.scale_strides[0] : 0, page_size > 1 ? f.scale_strides[2] : 0};
    for (const int64_t t : steps) near = near && t <= 0xffffffffLL;
    *to[j] = paged4::Rows{static_cast<const char*>(f.codes), static_cast<const char*>(f.scales),
                          static_cast<uint32_t>(steps[0]), static_cast<uint32_t>(steps[1]),
                          static_cast<uint32_t>(steps[2]), static_cast<uint32_t>(steps[3]),
                          f.code_strides[1], f.scale_strides[1]};
  }
  if (!ok)
    return set_error(err, GHIP_ERR_UNSUPPORTED,
                     "%s: codes must be 16-byte aligned with non-negative strides of whole 16 bytes, scales 4-byte aligned "
                     "with strides of whole 4", kWhat);
  if (!near) return set_error(err, GHIP_ERR_UNSUPPORTED, "%s: pages and tokens at strides of 4 GiB and more", kWhat);
  p.q = q; p.o = o;
  p.table = block_table; p.lens = lens;
  p.q_sb = q_strides[0]; p.q_sh = q_strides[1]; p.o_sb = o_strides[0]; p.o_sh = o_strides[1];
  p.table_stride = table_stride;
  p.B = static_cast<int>(B); p.H = static_cast<int>(H); p.Hkv = static_cast<int>(Hkv); p.D = static_cast<int>(D);
  p.num_pages = static_cast<int>(num_pages); p.page_size = static_cast<int>(page_size);
  p.max_pages = static_cast<int>(max_pages);
  p.window = static_cast<int>(window == 0 || window > kMost ? kMost : window);
  p.sinks = static_cast<int>(sinks > kMost ? kMost : sinks);
  p.scale = scale;
  p.pages = paged4::Pages(page_size);
  p.unit_heads = static_cast<int>(std::min<int64_t>(paged::kHeads, H / Hkv));
  const int64_t need = workspace ? ghip_sdpa_paged_kv4_workspace_bytes(B, H, Hkv, D, page_size, max_pages) : 0;
  if (need > 0) {
    if (workspace_bytes < need)
      return set_error(err, GHIP_ERR_INVALID_ARG, "%s: workspace of %lld bytes, %lld needed", kWhat,
                       static_cast<long long>(workspace_bytes), static_cast<long long>(need));
    if (!al(workspace, 16)) return set_error(err, GHIP_ERR_INVALID_ARG, "%s: workspace must be 16-byte aligned", kWhat);
    p.part_o = static_cast<float*>(workspace);
    const int64_t shares = 2 * static_cast<int64_t>(paged4::workers(D <= 128 ? 128 : 256)) * p.unit_heads;
    p.part_lse = p.part_o + shares * D;
    p.held = reinterpret_cast<int2*>(p.part_lse + shares);
  }
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (f32) paged4::launch<float>(p, s);
  else if (dtype == GHIP_DTYPE_FLOAT16) paged4::launch<f16_t>(p, s);
  else paged4::launch<bf16_t>(p, s);
  GHIP_CHECK(hipGetLastError(), err);
  return GHIP_OK;
}
