// Gradient of the sliding-window attention of k_attn_window.hip, from its output and
// log-sum-exp:
//   P = exp(scale q.k - lse) where the query sees the key,   delta = sum_d do o
//   dV = P^T dO,   dS = P (dO V^T - delta),   dQ = scale dS K,   dK = scale dS^T Q
// (dK and dV summed over the query heads that share a kv head).  Two kernels that each
// evaluate P and dS again, so nothing of size Sq x Sk is stored and no sum depends on
// the order of atomics: the first owns queries (dQ, and delta for the second), the
// second keys.
#include <algorithm>
#include <type_traits>

#include "attn_window.h"

namespace ghip {
namespace win {

using tile::f32x16;

constexpr int kCols = 128;  // queries of a workgroup of dq_kernel
#ifndef KPAIRS
#define KPAIRS 2
#define KTILE 32
#define FARPER 512
#endif
constexpr int kKeys = 32 * KPAIRS;  // keys of a workgroup of dkv_kernel
constexpr float kLog2e = 1.4426950408889634f;

// dQ: the transposed arrangement of the forward kernel.  A lane owns one query; S^T = K
// Q^T and dP^T = V dO^T come out as columns, dS^T enters dQ^T += K^T dS^T from the
// registers.  The product's accumulator starts at -delta, and the scale sits in the
// exponent (P scale = 2^(s c - lse2 + log2 scale)), so an element costs one FMA, one
// exponential and one multiplication.
template <typename T, int DP>
__global__ __launch_bounds__(256, (DP * sizeof(T) > 256 ? 1 : 2)) void dq_kernel(Params p) {
  using Tl = tile::Tile<T, DP>;
  using F = typename Tl::F;
  constexpr int kT = 64, kTile = kT * Tl::kRow, kQW = 32;
  __shared__ __attribute__((aligned(1024))) char smem[2][2][kTile];
  const uint32_t lds0 = tile::lds_addr(smem);

  const int lane = threadIdx.x & 63, h2 = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int nqb = (p.Sq + kCols - 1) / kCols;
  const int nbh = p.B * p.H;
  const int qb = nqb - 1 - static_cast<int>(blockIdx.x / nbh);
  const int bh = blockIdx.x % nbh;
  const int b = bh / p.H, h = bh % p.H, hk = h / (p.H / p.Hkv);
  const int len = length_of(p, b);
  const int q0 = qb * kCols, qw = q0 + wave * kQW, qi = qw + (lane & 31);
  const int pos = p.q_start + qi, pw = p.q_start + qw;
  const bool live = qi < p.Sq && pos < len;

  F qf[DP / 16], gf[DP / 16];
  float nd = 0.f;  // minus delta
  {
    const T* Q = at<T>(p.q, b, h) + static_cast<int64_t>(qi) * p.q.ss;
    const T* G = at<T>(p.dout, b, h) + static_cast<int64_t>(qi) * p.dout.ss;
    const T* O = at<T>(p.o, b, h) + static_cast<int64_t>(qi) * p.o.ss;
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
      qf[s] = Tl::frag_global(Q, s, h2, p.D, live);
      gf[s] = Tl::frag_global(G, s, h2, p.D, live);
      const F of = Tl::frag_global(O, s, h2, p.D, live);
#pragma unroll
      for (int e = 0; e < 8; ++e) nd -= tile::value<T>(gf[s], e) * tile::value<T>(of, e);
    }
  }
  nd += __shfl_xor(nd, 32, 64);
  const int64_t row = (static_cast<int64_t>(b) * p.H + h) * p.Sq + qi;
  if (h2 == 0 && qi < p.Sq) p.ndelta[row] = nd;
  const float c = p.scale * kLog2e;
  float nl = live ? __builtin_amdgcn_logf(p.scale) - p.lse[row] * kLog2e : 0.f;
  tile::settle(qf);
  tile::settle(gf);
  asm volatile("" : "+v"(nl));

  const tile::Rows K = rows_of<T>(p.k, b, hk, len), V = rows_of<T>(p.v, b, hk, len);
  tile::Loader<T, DP, kT, 4> lk, lv;
  lk.init(K.step, p.D, wave, lane);
  lv.init(V.step, p.D, wave, lane);
  const int p0 = p.q_start + q0;
  const Tiles<kT> tl(p, p0, p0 < len ? min(len, p.q_start + min(q0 + kCols, p.Sq)) : 0);
  auto issue = [&](int i) {
    const uint32_t la = lds0 + (i & 1) * (2 * kTile);
    const int r = tl(i) * kT;
    lk.issue(K, r, la, wave);
    lv.issue(V, r, la + kTile, wave);
  };

  f32x16 dq[DP / 32];
#pragma unroll
  for (int db = 0; db < DP / 32; ++db) dq[db] = tile::splat(0.f);

  // Tile i from stage ST, known when compiled.
  auto step = [&](auto st, int i) {
    constexpr int ST = decltype(st)::value;
    tile::landed_barrier();
    if (i + 1 < tl.n) issue(i + 1);
#pragma unroll
    for (int kb = 0; kb < kT / 32; ++kb) {
      const int key0 = tl(i) * kT + 32 * kb;
      if (key0 > pw + kQW - 1 || key0 >= len || (key0 + 31 <= pw - p.window && key0 >= p.sinks)) continue;
      const char* sk = smem[ST][0] + 32 * kb * Tl::kRow;
      const char* sv = smem[ST][1] + 32 * kb * Tl::kRow;
      f32x16 x = tile::splat(0.f), g = tile::splat(nd);
      tile::pipelined<Tl::kRow, F, DP / 8>([&](int j) { return Tl::frag_row(j & 1 ? sv : sk, j >> 1, lane); },
                                 [&](int j, const F& a) {
                                   f32x16& to = j & 1 ? g : x;
                                   to = tile::mma<T>(a, j & 1 ? gf[j >> 1] : qf[j >> 1], to);
                                 });
#pragma unroll
      for (int v = 0; v < 16; ++v) x[v] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[v], c, nl)) * g[v];
      if (key0 + 31 > pw || key0 + 32 > len || key0 <= pw + kQW - 1 - p.window) {
        asm volatile("");  // a branch: most tiles need no mask
        const uint32_t w = seen_keys(p, pos, live, len, key0 + 4 * h2);
#pragma unroll
        for (int v = 0; v < 16; ++v) x[v] = select_bit(w, (v >> 2) * 8 + (v & 3), x[v], 0.f);
      }
      const F df[2] = {tile::pack<T>(x, 0), tile::pack<T>(x, 1)};
      constexpr int ND = DP / 32;
      tile::pipelined<Tl::kRow, F, 2 * ND>([&](int j) { return Tl::frag_tr(sk + 16 * (j / ND) * Tl::kRow, j % ND, lane); },
                                 [&](int j, const F& a) { dq[j % ND] = tile::mma<T>(a, df[j / ND], dq[j % ND]); });
    }
  };
  if (tl.n > 0) issue(0);
  for (int i = 0; i < tl.n; i += 2) {
    step(std::integral_constant<int, 0>{}, i);
    if (i + 1 < tl.n) step(std::integral_constant<int, 1>{}, i + 1);
  }
  if (qi >= p.Sq) return;
  T* out = at<T>(p.dq, b, h) + static_cast<int64_t>(qi) * p.dq.ss;
#pragma unroll
  for (int db = 0; db < DP / 32; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = db * 32 + g * 8 + 4 * h2;
      if (d >= p.D) continue;
      float r[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) r[e] = live ? dq[db][4 * g + e] : 0.f;
      tile::store4(out + d, r[0], r[1], r[2], r[3]);
    }
}

// dK, dV: a lane owns one key; S = Q K^T and dP = dO V^T come out with the lane's key as
// their column, so P and dS enter dV^T += dO^T P and dK^T += Q^T dS from the registers.
// Two waves share 32 keys, half of the registers each (K, V and both sums in one wave
// left one wave a SIMD, which stood waiting 55% of its time): the first holds K and
// the sum dV, and hands P over through LDS in fp32; the second holds V and the sum dK.
// Q and dO stream through two LDS stages, head after head of the group, with each query's
// log-sum-exp and delta beside them.
//
// Every query sees the sinks, so their keys' sums run over the whole sequence, not over a
// window.  Where that matters (plan_far) the queries behind the window of the sinks' block
// are left to workgroups of their own, which deal them out in chunks and hold 32 sinks
// each, every pair of waves another 32 rows of a tile; their fp32 sums and the block's
// own are added by join_kernel in a fixed order.
//
// f16 only: P is at most 1 and of order 1 / window, so it is rounded 2^8 times larger
// (small weights would be subnormal), and dS is rounded with the scale applied.
template <typename T, int DP>
struct Keys {
  using Tl = tile::Tile<T, DP>;
  using F = typename Tl::F;
  static constexpr bool kF16 = __is_same(T, f16_t);
  static constexpr int kPairs = kKeys / 32, kNW = 2 * kPairs;
  static constexpr int kT = Tl::kRow > 256 ? 32 : KTILE;  // rows of a tile
  static constexpr int kTile = kT * Tl::kRow;
  struct Lds {
    __attribute__((aligned(1024))) char tiles[2][2][kTile];      // [stage][Q, dO]
    __attribute__((aligned(16))) float p[kPairs][kT / 32][4][64][4];  // P of a pair's keys, in accumulator order
    __attribute__((aligned(16))) float stat[2][2][kT];           // [stage][-log-sum-exp in base 2, -delta]
  };
  // What a workgroup works on: tiles tbase .. tbase + tcount - 1 of each head of the group
  // as one list, its entries i0 .. i1 - 1; keys from kfirst on.
  struct Work {
    int b, hk, kfirst, tbase, tcount, i0, i1, nq;
    bool far;  // the 32 keys from kfirst on, a pair of waves each 32 rows of the tiles
    float* part;
  };

  // ROLE 0: P and dV; 1: dS and dK.
  template <int ROLE>
  __device__ __forceinline__ static void run(const Params& p, Lds& lds, const Work& w) {
    const uint32_t lds0 = tile::lds_addr(lds.tiles);
    const int lane = threadIdx.x & 63, h2 = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), pair = wave % kPairs;
    const int len = length_of(p, w.b);
    const int kw = w.far ? w.kfirst : w.kfirst + pair * 32, key = kw + (lane & 31);
    const int G = p.H / p.Hkv;
    const float c = p.scale * kLog2e;

    F kf[DP / 16];  // K (ROLE 0) or V
    {
      const Mat3& m = ROLE == 0 ? p.k : p.v;
      const T* K = at<T>(m, w.b, w.hk) + static_cast<int64_t>(key) * m.ss;
#pragma unroll
      for (int s = 0; s < DP / 16; ++s) kf[s] = Tl::frag_global(K, s, h2, p.D, key < len);
    }
    tile::settle(kf);
    tile::Loader<T, DP, kT, kNW> lq, lg;
    lq.init(static_cast<uint32_t>(p.q.ss * Tl::kEs), p.D, wave, lane);
    lg.init(static_cast<uint32_t>(p.dout.ss * Tl::kEs), p.D, wave, lane);
    float st = 0.f;  // this thread's entry of the next tile's statistics
    int tn = w.tbase + w.i0 % max(w.tcount, 1), tc = tn;  // the tile that issue() loads next, the tile worked on
    const int h0 = w.hk * G + w.i0 / max(w.tcount, 1);
    // Its head's rows; the heads of a group follow one another by a head stride.
    tile::Rows Q = rows_of<T>(p.q, w.b, h0, w.nq), dO = rows_of<T>(p.dout, w.b, h0, w.nq);
    const float* stats = (threadIdx.x < kT ? p.lse : p.ndelta) + (static_cast<int64_t>(w.b) * p.H + h0) * p.Sq;
    const float sf = threadIdx.x < kT ? -kLog2e : 1.f, sa = kF16 && threadIdx.x < kT ? 8.f : 0.f;
    auto issue = [&](int stage) {
      // (Rows past the queries, which nothing sees, take the last one's: a load under a
      // condition would be waited for at once.)
      st = stats[min(tn * kT + static_cast<int>(threadIdx.x % kT), w.nq - 1)];
      const uint32_t la = lds0 + stage * (2 * kTile);
      lq.issue(Q, tn * kT, la, wave);
      lg.issue(dO, tn * kT, la + kTile, wave);
      if (++tn == w.tbase + w.tcount) {
        tn = w.tbase;
        Q.base += p.q.sh * Tl::kEs;
        dO.base += p.dout.sh * Tl::kEs;
        stats += p.Sq;
      }
    };
    auto put = [&](int stage) {
      if (threadIdx.x < 2 * kT) lds.stat[stage][threadIdx.x / kT][threadIdx.x % kT] = __builtin_fmaf(st, sf, sa);
    };

    f32x16 sum[DP / 32];  // dV (ROLE 0) or dK
#pragma unroll
    for (int db = 0; db < DP / 32; ++db) sum[db] = tile::splat(0.f);

    // Entry i from stage ST, known when compiled.
    auto step = [&](auto stage, int i) {
      constexpr int ST = decltype(stage)::value;
      tile::landed_barrier();  // the tile is there; nobody reads the other stage or P any more
      if (i + 1 < w.i1) issue(1 - ST);
      const int t0 = p.q_start + tc * kT;  // the tile's first position
      if (++tc == w.tbase + w.tcount) tc = w.tbase;
      f32x16 x[kT / 32];
      F pf[kT / 32][2];
      bool on[kT / 32];
#pragma unroll
      for (int rb = 0; rb < kT / 32; ++rb) {
        const int p0 = t0 + 32 * rb;
        on[rb] = !(p0 + 31 < kw || (p0 >= kw + 31 + p.window && kw >= p.sinks) || p0 - p.q_start >= w.nq) &&
                 (!w.far || rb == pair);
        if (!on[rb]) continue;
        const char* tl = lds.tiles[ST][ROLE] + 32 * rb * Tl::kRow;
        const float* ps = &lds.stat[ST][ROLE][32 * rb + 4 * h2];
        f32x16 stat;
#pragma unroll
        for (int v = 0; v < 16; ++v) stat[v] = ps[(v >> 2) * 8 + (v & 3)];
        x[rb] = ROLE == 0 ? tile::splat(0.f) : stat;
        tile::pipelined<Tl::kRow, F, DP / 16>([&](int s) { return Tl::frag_row(tl, s, lane); },
                                    [&](int s, const F& a) { x[rb] = tile::mma<T>(a, kf[s], x[rb]); });
        if constexpr (ROLE == 0) {
#pragma unroll
          for (int v = 0; v < 16; ++v) x[rb][v] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[rb][v], c, stat[v]));
          if (p0 < kw + 31 || p0 + 31 - p.q_start >= w.nq || (p0 + 31 >= kw + p.window && kw + 31 >= p.sinks)) {
            asm volatile("");  // a branch: most tiles need no mask
            // Rows key - p0 .. min(end, key + window) - p0 - 1 see the key.
            const int end = p.q_start + w.nq;
            const int first = key - p0 - 4 * h2, last = (key < p.sinks ? end : min(end, key + p.window)) - p0 - 4 * h2;
            const uint32_t bits = low_bits(last) & ~low_bits(first);
#pragma unroll
            for (int v = 0; v < 16; ++v) x[rb][v] = select_bit(bits, (v >> 2) * 8 + (v & 3), x[rb][v], 0.f);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j)
            *reinterpret_cast<float4*>(lds.p[pair][rb][j][lane]) =
                make_float4(x[rb][4 * j], x[rb][4 * j + 1], x[rb][4 * j + 2], x[rb][4 * j + 3]);
#pragma unroll
          for (int s = 0; s < 2; ++s) pf[rb][s] = tile::pack<T>(x[rb], s);
        }
      }
      // P is there (the next tile's DMA stays in flight).
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
      for (int rb = 0; rb < kT / 32; ++rb) {
        if (!on[rb]) continue;
        if constexpr (ROLE == 1) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float4 pv = *reinterpret_cast<const float4*>(lds.p[pair][rb][j][lane]);
            const float f = kF16 ? p.scale * 0x1p-8f : 1.f;
            x[rb][4 * j] *= kF16 ? pv.x * f : pv.x;
            x[rb][4 * j + 1] *= kF16 ? pv.y * f : pv.y;
            x[rb][4 * j + 2] *= kF16 ? pv.z * f : pv.z;
            x[rb][4 * j + 3] *= kF16 ? pv.w * f : pv.w;
          }
#pragma unroll
          for (int s = 0; s < 2; ++s) pf[rb][s] = tile::pack<T>(x[rb], s);
        }
        const char* tl = lds.tiles[ST][1 - ROLE] + 32 * rb * Tl::kRow;  // dO for dV, Q for dK
        constexpr int ND = DP / 32;
        tile::pipelined<Tl::kRow, F, 2 * ND>(
            [&](int j) { return Tl::frag_tr(tl + 16 * (j / ND) * Tl::kRow, j % ND, lane); },
            [&](int j, const F& a) { sum[j % ND] = tile::mma<T>(a, pf[rb][j / ND], sum[j % ND]); });
      }
      if (i + 1 < w.i1) put(1 - ST);
    };
    if (w.i0 < w.i1) {
      issue(0);
      put(0);
    }
    for (int i = w.i0; i < w.i1; i += 2) {
      step(std::integral_constant<int, 0>{}, i);
      if (i + 1 < w.i1) step(std::integral_constant<int, 1>{}, i + 1);
    }

    if (w.far ? pair < kT / 32 : w.part && kw < p.sinks) {  // shares of sinks' sums: [dk, dv][32 keys][D]
      const int64_t block = w.far ? 0 : kw / 32 * p.far_stride;
      float* to = w.part + block + (static_cast<int64_t>(w.far ? pair : 0) * 64 + (ROLE == 0 ? 32 : 0) + (lane & 31)) * p.D;
#pragma unroll
      for (int db = 0; db < DP / 32; ++db)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int d = db * 32 + g * 8 + 4 * h2;
          if (d < p.D) tile::store4(to + d, sum[db][4 * g], sum[db][4 * g + 1], sum[db][4 * g + 2], sum[db][4 * g + 3]);
        }
    }
    if (w.far || (w.part && key < p.sinks) || key >= p.Sk) return;
    const Mat3& m = ROLE == 0 ? p.dv : p.dk;
    T* out = at<T>(m, w.b, w.hk) + static_cast<int64_t>(key) * m.ss;
    const float f = ROLE == 0 ? (kF16 ? 0x1p-8f : 1.f) : (kF16 ? 1.f : p.scale);
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int d = db * 32 + g * 8 + 4 * h2;
        if (d >= p.D) continue;
        float r[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = key < len ? sum[db][4 * g + e] * f : 0.f;
        tile::store4(out + d, r[0], r[1], r[2], r[3]);
      }
  }
};

// One past the last tile (of kT rows) of queries that see, through their windows, a key of
// the block at k0.
__device__ __host__ __forceinline__ int near_end(const Params& p, int k0, int kT) {
  const int64_t last = static_cast<int64_t>(k0) + kKeys - 1 + p.window - p.q_start;  // one past the last such query
  const int64_t tiles = (p.Sq + kT - 1) / kT;
  return static_cast<int>(last <= 0 ? 0 : (last + kT - 1) / kT < tiles ? (last + kT - 1) / kT : tiles);
}

template <typename T, int DP>
__global__ __launch_bounds__(128 * KPAIRS, 2) void dkv_kernel(Params p) {
  using K = Keys<T, DP>;
  constexpr int kT = K::kT;
  __shared__ typename K::Lds lds;
  const int nbh = p.B * p.Hkv, G = p.H / p.Hkv;
  const int bh = blockIdx.x % nbh, at_ = blockIdx.x / nbh;
  typename K::Work w;
  w.b = bh / p.Hkv;
  w.hk = bh % p.Hkv;
  const int len = length_of(p, w.b);
  w.nq = max(0, min(p.Sq, len - p.q_start));  // queries that exist
  const int tiles = (w.nq + kT - 1) / kT;
  w.part = p.far_blocks ? p.far + static_cast<int64_t>(bh) * p.far_blocks * p.far_stride : nullptr;
  const int blocks = (p.Sk + kKeys - 1) / kKeys;
  w.far = at_ >= blocks;  // last: the shortest
  if (w.far) {
    // Chunk ck of the queries that see the 32 sinks from 32 sb through no window.
    const int sb = (at_ - blocks) / p.far_chunks, ck = (at_ - blocks) % p.far_chunks;
    w.kfirst = 32 * sb;
    w.tbase = near_end(p, w.kfirst / kKeys * kKeys, kT);
    w.tcount = max(0, tiles - w.tbase);
    w.i0 = min(w.tcount * G, ck * p.far_per);
    w.i1 = min(w.tcount * G, w.i0 + p.far_per);
    w.part += sb * p.far_stride + (1 + kT / 32 * ck) * (64 * static_cast<int64_t>(p.D));
  } else {
    w.kfirst = at_ * kKeys;
    w.tbase = max(0, w.kfirst - p.q_start) / kT;
    const int te = w.kfirst >= len ? 0 : w.kfirst < p.sinks && !w.part ? tiles : min(tiles, near_end(p, w.kfirst, kT));
    w.tcount = max(0, te - w.tbase);
    w.i0 = 0;
    w.i1 = w.tcount * G;
  }
  if (__builtin_amdgcn_readfirstlane(threadIdx.x >> 6) >= K::kPairs) K::template run<1>(p, lds, w);
  else K::template run<0>(p, lds, w);
}

// dk, dv of the sinks: the shares of their block and of the chunks, added in that order.
template <typename T>
__global__ __launch_bounds__(256) void join_kernel(Params p) {
  constexpr bool kF16 = __is_same(T, f16_t);
  const int vecs = p.D / 4, wgs = (p.far_blocks * 64 * vecs + 255) / 256;  // workgroups of a (batch, kv head)
  const int bh = blockIdx.x / wgs, b = bh / p.Hkv, hk = bh % p.Hkv;
  const int e = blockIdx.x % wgs * 256 + threadIdx.x;
  const int row = e / vecs, d = e % vecs * 4;  // row: block, then [dk, dv], then key
  const int sb = row / 64, which = row / 32 % 2, key = sb * 32 + row % 32;
  if (key >= p.sinks || sb >= p.far_blocks) return;
  const float* part = p.far + (static_cast<int64_t>(bh) * p.far_blocks + sb) * p.far_stride +
                      (which * 32 + row % 32) * static_cast<int64_t>(p.D) + d;
  float a[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int i = 0; i < p.far_shares; ++i) {
    const float4 v = *reinterpret_cast<const float4*>(part + i * (2 * 32 * static_cast<int64_t>(p.D)));
    a[0] += v.x;
    a[1] += v.y;
    a[2] += v.z;
    a[3] += v.w;
  }
  const float f = which ? (kF16 ? 0x1p-8f : 1.f) : (kF16 ? 1.f : p.scale);
  const Mat3& m = which ? p.dv : p.dk;
  const bool live = key < length_of(p, b);
  tile::store4(at<T>(m, b, hk) + key * m.ss + d, live ? a[0] * f : 0.f, live ? a[1] * f : 0.f, live ? a[2] * f : 0.f,
               live ? a[3] * f : 0.f);
}

// The workgroups for the queries that see sinks through no window: none unless they are
// as many as a block's own tiles, else in chunks of a block's tiles (each of half its
// work or less).  Fills p's far fields; returns the floats of the shares.
static int64_t plan_far(Params* p, int row_bytes) {
  const int kT = row_bytes > 256 ? 32 : KTILE;
  const int G = p->H / p->Hkv;
  const int beyond = (p->Sq + kT - 1) / kT - near_end(*p, 0, kT);
  const int own = (std::min(p->window, p->Sq) + kKeys) / kT + 1;
  if (p->sinks == 0 || beyond < own) return 0;
  p->far_blocks = (p->sinks + 31) / 32;
  p->far_per = FARPER / kT;
  p->far_chunks = (beyond * G + p->far_per - 1) / p->far_per;
  p->far_shares = 1 + kT / 32 * p->far_chunks;
  p->far_stride = static_cast<int64_t>(p->far_shares) * 64 * p->D;
  return static_cast<int64_t>(p->B) * p->Hkv * p->far_blocks * p->far_stride;
}
static int64_t plan_far(Params* p, bool f32) {
  return plan_far(p, (p->D <= 64 ? 64 : p->D <= 128 ? 128 : 256) * (f32 ? 4 : 2));
}

// Floats of delta, a whole number of 16 bytes.
static int64_t delta_floats(const Params& p) { return (static_cast<int64_t>(p.B) * p.H * p.Sq + 3) / 4 * 4; }

template <typename T, int DP>
static void launch_d(const Params& p, hipStream_t s) {
  const dim3 gq(static_cast<unsigned>((p.Sq + kCols - 1) / kCols * p.B * p.H));
  const dim3 gk(static_cast<unsigned>(((p.Sk + kKeys - 1) / kKeys + p.far_blocks * p.far_chunks) * p.B * p.Hkv));
  if (p.Sq > 0) hipLaunchKernelGGL((dq_kernel<T, DP>), gq, dim3(256), 0, s, p);
  hipLaunchKernelGGL((dkv_kernel<T, DP>), gk, dim3(128 * KPAIRS), 0, s, p);
  if (p.far_blocks)
    hipLaunchKernelGGL((join_kernel<T>), dim3(static_cast<unsigned>((p.far_blocks * 64 * (p.D / 4) + 255) / 256) * p.B * p.Hkv),
                       dim3(256), 0, s, p);
}
template <typename T>
static void launch(const Params& p, hipStream_t s) {
  if (p.D <= 64) launch_d<T, 64>(p, s);
  else if (p.D <= 128) launch_d<T, 128>(p, s);
  else if constexpr (sizeof(T) == 2) launch_d<T, 256>(p, s);
}

}  // namespace win
}  // namespace ghip

using namespace ghip;

extern "C" int64_t ghip_sdpa_window_bwd_workspace_bytes(int dtype, int64_t B, int64_t H, int64_t Hkv, int64_t Sq,
                                                        int64_t Sk, int64_t D, int64_t q_start, int64_t window,
                                                        int64_t sinks) {
  win::Params p{};
  if (win::check_problem("", dtype, B, H, Hkv, Sq, Sk, D, q_start, window, sinks, 1.f, &p, nullptr)) return 0;
  return (win::delta_floats(p) + win::plan_far(&p, dtype == GHIP_DTYPE_FLOAT32)) * 4;
}

extern "C" int ghip_sdpa_window_bwd(int dtype, const void* q, const void* k, const void* v, const void* o,
                                    const void* d_out, const float* lse, void* dq, void* dk, void* dv, int64_t B,
                                    int64_t H, int64_t Hkv, int64_t Sq, int64_t Sk, int64_t D, const int64_t* q_strides,
                                    const int64_t* k_strides, const int64_t* v_strides, const int64_t* o_strides,
                                    const int64_t* d_out_strides, const int64_t* dq_strides, const int64_t* dk_strides,
                                    const int64_t* dv_strides, int64_t q_start, int64_t window, int64_t sinks,
                                    const int32_t* lens, float scale, void* workspace, int64_t workspace_bytes,
                                    void* stream, GHipError* err) {
  static const char kWhat[] = "sdpa_window_bwd";
  win::Params p{};
  if (int rc = win::check_problem(kWhat, dtype, B, H, Hkv, Sq, Sk, D, q_start, window, sinks, scale, &p, err)) return rc;
  if (B == 0 || Sk == 0) return GHIP_OK;
  const struct {
    const char* name;
    const void* ptr;
    const int64_t* strides;
    bool out;
    win::Mat3* to;
  } operands[] = {{"q", q, q_strides, false, &p.q},          {"k", k, k_strides, false, &p.k},
                  {"v", v, v_strides, false, &p.v},          {"o", o, o_strides, false, &p.o},
                  {"do", d_out, d_out_strides, false, &p.dout}, {"dq", dq, dq_strides, true, &p.dq},
                  {"dk", dk, dk_strides, true, &p.dk},       {"dv", dv, dv_strides, true, &p.dv}};
  for (const auto& x : operands) {
    if (Sq == 0 && x.to != &p.k && x.to != &p.v && x.to != &p.dk && x.to != &p.dv) continue;  // empty operands
    if (int rc = win::check_operand(kWhat, x.name, dtype, x.ptr, x.strides, x.out, x.to, err)) return rc;
  }
  if (!lse && Sq > 0) return set_error(err, GHIP_ERR_INVALID_ARG, "%s: lse is null", kWhat);
  const int64_t need = ghip_sdpa_window_bwd_workspace_bytes(dtype, B, H, Hkv, Sq, Sk, D, q_start, window, sinks);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return set_error(err, GHIP_ERR_INVALID_ARG, "%s: workspace of %lld bytes, %lld needed", kWhat,
                     static_cast<long long>(workspace ? workspace_bytes : 0), static_cast<long long>(need));
  if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
    return set_error(err, GHIP_ERR_INVALID_ARG, "%s: workspace must be 16-byte aligned", kWhat);
  p.lse = const_cast<float*>(lse);
  p.ndelta = static_cast<float*>(workspace);
  p.far = p.ndelta + win::delta_floats(p);
  win::plan_far(&p, dtype == GHIP_DTYPE_FLOAT32);
  p.lens = lens;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == GHIP_DTYPE_FLOAT32) win::launch<float>(p, s);
  else if (dtype == GHIP_DTYPE_FLOAT16) win::launch<f16_t>(p, s);
  else win::launch<bf16_t>(p, s);
  GHIP_CHECK(hipGetLastError(), err);
  return GHIP_OK;
}
