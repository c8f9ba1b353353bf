// Gradient of the sliding-window attention of k_attn_window.hip, from its output and
// log-sum-exp:
//   P = exp(scale q.k - lse) where the query sees the key,   delta = sum_d do o
//   dV = P^T dO,   dS = P (dO V^T - delta),   dQ = scale dS K,   dK = scale dS^T Q
// (dK and dV summed over the query heads that share a kv head).  Two kernels that each
// evaluate P and dS again, so nothing of size Sq x Sk is stored and no sum depends on
// the order of atomics: the first owns queries (dQ, and delta for the second), the
// second keys.
#include <type_traits>

#include "attn_window.h"
#include "attn_window_rules.h"

namespace ghip {
namespace win {

using tile::f32x16;

constexpr int kCols = 128;  // queries of a workgroup of dq_kernel
constexpr float kLog2e = 1.4426950408889634f;

// f16 (5 bits of exponent): P, at most 1 and of order 1 / window, is rounded 2^15 times larger,
// and dS, whose size follows d_out's and the window's, times a power of two 2^e that each
// column (a lane's query in dq, its key in dk) finds as its running maximum does in a
// softmax: from first_exponent(), where all that could reach an f16 result is inside the range, e
// falls when a tile's values pass 2^15, so that they end below 2^7 and leave 2^8 for later tiles.  A
// value then keeps all its bits down to 2^-20 of the largest, and none overflows.  The sums
// follow, and lose 2^e at the end, in fp32.  The whole gradient, with a fixed factor / so: 4 x
// 16 heads of 2048 tokens, D 128, window 512 179 / 185 us, padded batch of 12 heads of 64 52.4 /
// 54.4, D 256 (2 x 8 heads of 2048) 111 / 136, where the sums' registers move for the rare branch.
constexpr int kPUp = 15;
__device__ __forceinline__ int first_exponent(float scale) {
  return 60 - max(0, static_cast<int>(__builtin_amdgcn_logf(scale)));  // (P scale 2^e: at most 2^61)
}
// x holds values times 2^e: returns by how much e has to change (0: x and the sums stay).
template <int ND>
__device__ __forceinline__ int make_room(f32x16& x, f32x16 (&sum)[ND]) {
  float mx = 0.f;
#pragma unroll
  for (int v = 0; v < 16; v += 2) mx = fmaxf(fmaxf(fabsf(x[v]), fabsf(x[v + 1])), mx);
  mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
  const bool over = mx > 0x1p15f;
  if (!__builtin_amdgcn_ballot_w64(over)) return 0;
  const int d = over ? min(0, 7 - __builtin_amdgcn_frexp_expf(mx)) : 0;
  const float f = __builtin_amdgcn_ldexpf(1.f, d);
#pragma unroll
  for (int v = 0; v < 16; ++v) x[v] *= f;
#pragma unroll
  for (int db = 0; db < ND; ++db)
#pragma unroll
    for (int v = 0; v < 16; ++v) sum[db][v] *= f;
  return d;
}

// dQ: the transposed arrangement of the forward kernel.  A lane owns one of a wave's 32
// queries; S^T = K Q^T and dP^T = V dO^T come out as columns, dS^T enters dQ^T += K^T dS^T
// from the registers.  The product's accumulator starts at -delta, and the scale sits in
// the exponent (P scale = 2^(s c - lse2 + log2 scale)), so an element costs one FMA, one
// exponential and one multiplication.
template <typename T, int DP>
struct GradQueries {
  using Tl = tile::Tile<T, DP>;
  using F = typename Tl::F;
  static constexpr bool kF16 = __is_same(T, f16_t);
  static constexpr int ND = DP / 32;
  F qf[DP / 16], gf[DP / 16];
  f32x16 dq[ND];
  float c, nl, nd;  // minus the log-sum-exp in base 2 (plus log2 scale, f16: plus e), minus delta
  int e;            // f16: dS and dq are held times 2^e
  int pw, pos;      // positions: the wave's first, the lane's own
  int len;
  bool live;        // the lane's query exists

  __device__ __forceinline__ void place(const Params& p, int b, int qw, int lane) {
    const int qi = qw + (lane & 31);
    len = length_of(p, b);
    pw = p.q_start + qw;
    pos = p.q_start + qi;
    live = qi < p.Sq && pos < len;
    c = p.scale * kLog2e;
  }
  // (Behind the first tile's DMA, so that the two are waited for together.)  tell: this
  // wave leaves the queries' statistics for dkv_kernel.
  __device__ __forceinline__ void load(const Params& p, int b, int h, int qw, int lane, bool tell) {
    const int qi = qw + (lane & 31), h2 = lane >> 5;
    const T* Q = at<T>(p.q, b, h) + static_cast<int64_t>(qi) * p.q.ss;
    const T* G = at<T>(p.dout, b, h) + static_cast<int64_t>(qi) * p.dout.ss;
    const T* O = at<T>(p.o, b, h) + static_cast<int64_t>(qi) * p.o.ss;
    nd = 0.f;
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
      qf[s] = Tl::frag_global(Q, s, h2, p.D, live);
      gf[s] = Tl::frag_global(G, s, h2, p.D, live);
      const F of = Tl::frag_global(O, s, h2, p.D, live);
#pragma unroll
      for (int e = 0; e < 8; ++e) nd -= tile::value<T>(gf[s], e) * tile::value<T>(of, e);
    }
    nd += __shfl_xor(nd, 32, 64);
    const int64_t row = (static_cast<int64_t>(b) * p.H + h) * p.Sq + qi;
    nl = live ? -p.lse[row] * kLog2e : 0.f;
    if (tell && qi < p.Sq && h2 == 0) {
      p.stats[row] = nl + (kF16 ? static_cast<float>(kPUp) : 0.f);
      p.stats[static_cast<int64_t>(p.B) * p.H * p.Sq + row] = nd;
    }
    nl += __builtin_amdgcn_logf(p.scale);
    if constexpr (kF16) {
      e = first_exponent(p.scale);
      nl += e;
    }
    tile::settle(qf);
    tile::settle(gf);
    asm volatile("" : "+v"(nl));
#pragma unroll
    for (int db = 0; db < ND; ++db) dq[db] = tile::splat(0.f);
  }
  // Whether any of the wave's queries, pw .. pw + 31, sees a key of key0 .. key0 + 31.
  __device__ __forceinline__ bool sees(const Params& p, int key0) const {
    return key0 <= pw + 31 && key0 < len && (key0 + 31 > pw - p.window || key0 < p.sinks);
  }
  // Keys key0 .. key0 + 31 from the tiles at sk, sv.
  __device__ __forceinline__ void step(const Params& p, const char* sk, const char* sv, int key0, int lane) {
    f32x16 x = tile::splat(0.f), g = tile::splat(nd);
    tile::pipelined<Tl::kRow, F, DP / 8>([&](int j) { return Tl::frag_row(j & 1 ? sv : sk, j >> 1, lane); },
                                         [&](int j, const F& a) {
                                           // fp32 products are 16 times as long: the padding's are left out.
                                           if (sizeof(T) == 4 && 16 * (j >> 1) >= p.D) return;
                                           f32x16& to = j & 1 ? g : x;
                                           to = tile::mma<T>(a, j & 1 ? gf[j >> 1] : qf[j >> 1], to);
                                         });
#pragma unroll
    for (int v = 0; v < 16; ++v) x[v] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[v], c, nl)) * g[v];
    if (key0 + 31 > pw || key0 + 32 > len || key0 <= pw + 31 - p.window) {
      asm volatile("");  // a branch: most tiles need no mask
      const uint32_t w = seen_keys(p, pos, live, len, key0 + 4 * (lane >> 5));
#pragma unroll
      for (int v = 0; v < 16; ++v) x[v] = select_bit(w, (v >> 2) * 8 + (v & 3), x[v], 0.f);
    }
    if constexpr (kF16) {
      const int d = make_room(x, dq);
      e += d;
      nl += d;
    }
    const F df[2] = {tile::pack<T>(x, 0), tile::pack<T>(x, 1)};
    tile::pipelined<Tl::kRow, F, 2 * ND>([&](int j) { return Tl::frag_tr(sk + 16 * (j / ND) * Tl::kRow, j % ND, lane); },
                                         [&](int j, const F& a) {
                                           if (sizeof(T) == 4 && 32 * (j % ND) >= p.D) return;
                                           dq[j % ND] = tile::mma<T>(a, df[j / ND], dq[j % ND]);
                                         });
  }
  // dq without 2^e.
  __device__ __forceinline__ void settle_sums() {
    if constexpr (kF16) {
      const float f = __builtin_amdgcn_ldexpf(1.f, -e);
#pragma unroll
      for (int db = 0; db < ND; ++db)
#pragma unroll
        for (int v = 0; v < 16; ++v) dq[db][v] *= f;
    }
  }
  __device__ __forceinline__ void finish(const Params& p, int b, int h, int qw, int lane) {
    const int qi = qw + (lane & 31), h2 = lane >> 5;
    if (qi >= p.Sq) return;
    T* out = at<T>(p.dq, b, h) + static_cast<int64_t>(qi) * p.dq.ss;
#pragma unroll
    for (int db = 0; db < ND; ++db)
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
};

// Four waves of 32 queries each; K and V stream through two LDS stages.  Q, dO and dQ take
// 228 registers, so two waves a SIMD: 76 us for 4 x 16 heads of 2048 tokens, window 512, bf16
// D 128 (0.60 PFLOP/s of visible pairs); matrix instructions take 34% of the cycles, vector
// ones 29%, and the rest waits between dependent ones.  Two waves a 32 queries, with Q and with dO, as in dkv_kernel, are three a
// SIMD but took 86 us (K and V twice as often, one wave with twice the products).
template <typename T, int DP>
__global__ __launch_bounds__(256, (DP * sizeof(T) > 256 ? 1 : 2)) void dq_kernel(Params p) {
  using Tl = tile::Tile<T, DP>;
  constexpr int KT = 64, kTile = KT * Tl::kRow;
  __shared__ __attribute__((aligned(1024))) char smem[2][2][kTile];
  const uint32_t lds0 = tile::lds_addr(smem);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int nqb = (p.Sq + kCols - 1) / kCols;
  const int nbh = p.B * p.H;
  const int qb = nqb - 1 - static_cast<int>(blockIdx.x / nbh);
  const int bh = spread(blockIdx.x % nbh, nbh);
  const int b = bh / p.H, h = bh % p.H, hk = h / (p.H / p.Hkv);
  const int q0 = qb * kCols, qw = q0 + wave * 32, p0 = p.q_start + q0;
  GradQueries<T, DP> q;
  q.place(p, b, qw, lane);

  const tile::Rows K = rows_of<T>(p.k, b, hk, q.len), V = rows_of<T>(p.v, b, hk, q.len);
  tile::Loader<T, DP, KT, 4> lk, lv;
  lk.init(K.step, p.D, wave, lane);
  lv.init(V.step, p.D, wave, lane);
  const Tiles<KT> tl(p, p0, p0 < q.len ? min(q.len, p.q_start + min(q0 + kCols, p.Sq)) : 0);
  auto issue = [&](int i) {
    const uint32_t la = lds0 + (i & 1) * (2 * kTile);
    lk.issue(K, tl(i) * KT, la, wave);
    lv.issue(V, tl(i) * KT, la + kTile, wave);
  };
  // Tile i from stage ST, known when compiled.
  auto step = [&](auto st, int i) {
    constexpr int ST = decltype(st)::value;
    tile::landed_barrier();
    if (i + 1 < tl.n) issue(i + 1);
#pragma unroll
    for (int k = 0; k < KT / 32; ++k) {
      const int key0 = tl(i) * KT + 32 * k;
      if (q.sees(p, key0)) q.step(p, smem[ST][0] + 32 * k * Tl::kRow, smem[ST][1] + 32 * k * Tl::kRow, key0, lane);
    }
  };
  if (tl.n > 0) issue(0);
  q.load(p, b, h, qw, lane, true);
  for (int i = 0; i < tl.n; i += 2) {
    step(std::integral_constant<int, 0>{}, i);
    if (i + 1 < tl.n) step(std::integral_constant<int, 1>{}, i + 1);
  }
  q.settle_sums();
  q.finish(p, b, h, qw, lane);
}

// Grids of few workgroups: 32 queries a workgroup, its four waves take the key tiles in
// turn, each with LDS stages of its own and no barrier; their sums are added through LDS.
template <typename T, int DP>
__global__ __launch_bounds__(256, 1) void dq_few_kernel(Params p) {
  using Tl = tile::Tile<T, DP>;
  constexpr int KT = 32, kTile = KT * Tl::kRow, ND = DP / 32;
  constexpr int kStages = Tl::kRow > 256 ? 1 : 2;
  constexpr int kDma = 2 * kTile / 1024;  // DMA instructions of a tile
  __shared__ __attribute__((aligned(1024))) char smem[4][kStages][2][kTile];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t lds0 = tile::lds_addr(smem[wave]);
  const int nbh = p.B * p.H;
  const int bh = spread(blockIdx.x % nbh, nbh), qw = blockIdx.x / nbh * 32;
  const int b = bh / p.H, h = bh % p.H, hk = h / (p.H / p.Hkv);
  GradQueries<T, DP> q;
  q.place(p, b, qw, lane);

  const tile::Rows K = rows_of<T>(p.k, b, hk, q.len), V = rows_of<T>(p.v, b, hk, q.len);
  tile::Loader<T, DP, KT, 1> lk, lv;
  lk.init(K.step, p.D, 0, lane);
  lv.init(V.step, p.D, 0, lane);
  const Tiles<KT> tl(p, q.pw, q.pw < q.len ? min(q.len, p.q_start + min(qw + 32, p.Sq)) : 0);
  auto issue = [&](int i, int stage) {
    const uint32_t la = lds0 + stage * (2 * kTile);
    lk.issue(K, tl(i) * KT, la, 0);
    lv.issue(V, tl(i) * KT, la + kTile, 0);
  };
  int stage = 0;
  if (wave < tl.n) issue(wave, 0);
  q.load(p, b, h, qw, lane, wave == 0);
  for (int i = wave; i < tl.n; i += 4) {
    if (kStages > 1 && i + 4 < tl.n) {
      issue(i + 4, stage ^ 1);
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kDma < 64 ? kDma : 0) : "memory");
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    if (q.sees(p, tl(i) * KT)) q.step(p, smem[wave][stage][0], smem[wave][stage][1], tl(i) * KT, lane);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the stage has been read
    if (kStages > 1) stage ^= 1;
    else if (i + 4 < tl.n) issue(i + 4, 0);
  }

  q.settle_sums();
  float* mine = reinterpret_cast<float*>(smem[wave]);
#pragma unroll
  for (int db = 0; db < ND; ++db)
#pragma unroll
    for (int v = 0; v < 16; ++v) mine[(db * 16 + v) * 64 + lane] = q.dq[db][v];
  __syncthreads();
  if (wave != 0) return;
#pragma unroll
  for (int db = 0; db < ND; ++db)
#pragma unroll
    for (int v = 0; v < 16; ++v) {
      float a = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) a += reinterpret_cast<const float*>(smem[w])[(db * 16 + v) * 64 + lane];
      q.dq[db][v] = a;
      if (v % 8 == 7) __builtin_amdgcn_sched_barrier(0);  // a few shares' reads in flight, not all
    }
  q.finish(p, b, h, qw, lane);
}

// dK, dV: a lane owns one key; S = Q K^T and dP = dO V^T come out with the lane's key as
// their column, so P and dS enter dV^T += dO^T P and dK^T += Q^T dS from the registers.
// Two waves share 32 keys, half of the registers each (K, V and both sums in one wave
// left one wave a SIMD, which stood waiting 55% of its time): the first holds K and
// the sum dV, and hands P over through LDS in fp32; the second holds V and the sum dK.  (A
// second wave one tile behind the first, with one barrier a tile but three stages and two
// P, was no faster at D 128 and 15% slower at 64, where it left room for a workgroup less.)
// Q and dO stream through two LDS stages, head after head of the group, with each query's
// log-sum-exp and delta beside them.
//
// P and dS are rounded once each, to the operands' type, as they enter the second products
// (16-bit matrix instructions take nothing wider; f16: raised, see kPUp); dS is formed from P
// in fp32.
template <typename T, int DP>
struct Keys {
  using Tl = tile::Tile<T, DP>;
  using F = typename Tl::F;
  static constexpr bool kF16 = __is_same(T, f16_t);
  static constexpr int kPairs = kKeys / 32, kNW = 2 * kPairs;
  static constexpr int kTile = kT * Tl::kRow;
  struct Lds {
    __attribute__((aligned(1024))) char tiles[2][2][kTile];    // [stage][Q, dO]
    __attribute__((aligned(16))) float p[kPairs][4][64][4];  // P of a pair's keys, in accumulator order
    __attribute__((aligned(16))) float stat[2][2][kT];       // [stage], as Params::stats
  };
  // What a workgroup works on: tiles tbase .. tbase + tcount - 1 of each head of the group
  // as one list, its entries i0 .. i1 - 1; a pair's keys from kfirst on; where its sums go
  // as a share (null: to the outputs).
  struct Work {
    int b, hk, kfirst, tbase, tcount, i0, i1, nq;
    bool idle;  // the pair only helps to load
    int apart;  // with a share: the keys below this one are the shares', the others go to the outputs
    float* share;
  };

  // ROLE 0: P and dV; 1: dS and dK.
  template <int ROLE>
  __device__ __forceinline__ static void run(const Params& p, Lds& lds, const Work& w) {
    const uint32_t lds0 = tile::lds_addr(lds.tiles);
    const int lane = threadIdx.x & 63, h2 = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), pair = wave % kPairs;
    const int len = length_of(p, w.b);
    const int kw = w.kfirst, key = kw + (lane & 31);
    const int G = p.H / p.Hkv;
    const float c = p.scale * kLog2e;

    tile::Loader<T, DP, kT, kNW> lq, lg;
    lq.init(static_cast<uint32_t>(p.q.ss * Tl::kEs), p.D, wave, lane);
    lg.init(static_cast<uint32_t>(p.dout.ss * Tl::kEs), p.D, wave, lane);
    int tn = w.tbase + w.i0 % max(w.tcount, 1), tc = tn;  // the tile that issue() loads next, the tile worked on
    const int h0 = w.hk * G + w.i0 / max(w.tcount, 1);
    // Its head's rows; the heads of a group follow one another by a head stride.
    tile::Rows Q = rows_of<T>(p.q, w.b, h0, w.nq), dO = rows_of<T>(p.dout, w.b, h0, w.nq);
    // Lanes 0 .. 31: the queries' log-sum-exp, 32 .. 63: their delta.  (Rows past the
    // queries, which nothing sees, take the last one's.)
    const float* stats = p.stats + (lane < 32 ? 0 : static_cast<int64_t>(p.B) * p.H * p.Sq) +
                         (static_cast<int64_t>(w.b) * p.H + h0) * p.Sq;
    auto issue = [&](int stage) {
      if (wave == 0) tile::load4(stats + min(tn * kT + (lane & 31), w.nq - 1), tile::lds_addr(lds.stat[stage]));
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
    if (w.i0 < w.i1) issue(0);  // (waited for together with the rows below)

    F kf[DP / 16];  // K (ROLE 0) or V
    {
      const Mat3& m = ROLE == 0 ? p.k : p.v;
      const T* K = at<T>(m, w.b, w.hk) + static_cast<int64_t>(key) * m.ss;
#pragma unroll
      for (int s = 0; s < DP / 16; ++s) kf[s] = Tl::frag_global(K, s, h2, p.D, key < len);
    }
    tile::settle(kf);
    f32x16 sum[DP / 32];  // dV (ROLE 0) or dK
#pragma unroll
    for (int db = 0; db < DP / 32; ++db) sum[db] = tile::splat(0.f);
    int e = kF16 && ROLE == 1 ? first_exponent(p.scale) : 0;

    // Entry i from stage ST, known when compiled.
    auto step = [&](auto stage, int i) {
      constexpr int ST = decltype(stage)::value, ND = DP / 32;
      tile::landed_barrier();  // the tile is there; nobody reads the other stage or P any more
      if (i + 1 < w.i1) issue(1 - ST);
      const int p0 = p.q_start + tc * kT;  // the tile's first position
      if (++tc == w.tbase + w.tcount) tc = w.tbase;
      const bool on = !(p0 + 31 < kw || (p0 >= kw + 31 + p.window && kw >= p.sinks) || p0 - p.q_start >= w.nq || w.idle);
      float4* pp = reinterpret_cast<float4*>(lds.p[pair]);
      f32x16 x;
      F pf[2];
      if (on) {
        const char* t1 = lds.tiles[ST][ROLE];
        const float* ps = &lds.stat[ST][ROLE][4 * h2];
        if constexpr (ROLE == 0) {
          x = tile::splat(0.f);
        } else {
#pragma unroll
          for (int v = 0; v < 16; ++v) x[v] = ps[(v >> 2) * 8 + (v & 3)];
        }
        f32x16 stat;
        tile::pipelined<Tl::kRow, F, DP / 16>([&](int s) { return Tl::frag_row(t1, s, lane); },
                                              [&](int s, const F& a) {
                                                // (The statistics as the last operands leave registers free.)
                                                if (ROLE == 0 && s == DP / 16 - 2)
#pragma unroll
                                                  for (int v = 0; v < 16; ++v) stat[v] = ps[(v >> 2) * 8 + (v & 3)];
                                                if (sizeof(T) == 4 && 16 * s >= p.D) return;
                                                x = tile::mma<T>(a, kf[s], x);
                                              });
        if constexpr (ROLE == 0) {
#pragma unroll
          for (int v = 0; v < 16; ++v) x[v] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[v], c, stat[v]));
          if (p0 < kw + 31 || p0 + 31 - p.q_start >= w.nq || (p0 + 31 >= kw + p.window && kw + 31 >= p.sinks)) {
            asm volatile("");  // a branch: most tiles need no mask
            // Rows key - p0 .. min(end, key + window) - p0 - 1 see the key.
            const int end = p.q_start + w.nq;
            const int first = key - p0 - 4 * h2, last = (key < p.sinks ? end : min(end, key + p.window)) - p0 - 4 * h2;
            const uint32_t bits = low_bits(last) & ~low_bits(first);
#pragma unroll
            for (int v = 0; v < 16; ++v) x[v] = select_bit(bits, (v >> 2) * 8 + (v & 3), x[v], 0.f);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) pp[64 * j + lane] = make_float4(x[4 * j], x[4 * j + 1], x[4 * j + 2], x[4 * j + 3]);
          pf[0] = tile::pack<T>(x, 0);
          pf[1] = tile::pack<T>(x, 1);
        }
      }
      // P is there (the next tile's DMA stays in flight).
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
      if (!on) return;
      if constexpr (ROLE == 1) {
        const float f = kF16 ? __builtin_amdgcn_ldexpf(p.scale, e - kPUp) : 1.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float4 pv = pp[64 * j + lane];
          x[4 * j] *= kF16 ? pv.x * f : pv.x;
          x[4 * j + 1] *= kF16 ? pv.y * f : pv.y;
          x[4 * j + 2] *= kF16 ? pv.z * f : pv.z;
          x[4 * j + 3] *= kF16 ? pv.w * f : pv.w;
        }
        if constexpr (kF16) e += make_room(x, sum);
        pf[0] = tile::pack<T>(x, 0);
        pf[1] = tile::pack<T>(x, 1);
      }
      const char* t2 = lds.tiles[ST][1 - ROLE];  // dO for dV, Q for dK
      tile::pipelined<Tl::kRow, F, 2 * ND>([&](int j) { return Tl::frag_tr(t2 + 16 * (j / ND) * Tl::kRow, j % ND, lane); },
                                           [&](int j, const F& a) {
                                             if (sizeof(T) == 4 && 32 * (j % ND) >= p.D) return;
                                             sum[j % ND] = tile::mma<T>(a, pf[j / ND], sum[j % ND]);
                                           });
    };
    for (int i = w.i0; i < w.i1; i += 2) {
      step(std::integral_constant<int, 0>{}, i);
      if (i + 1 < w.i1) step(std::integral_constant<int, 1>{}, i + 1);
    }

    if (w.idle) return;
    if constexpr (kF16 && ROLE == 1) {
      const float f = __builtin_amdgcn_ldexpf(1.f, -e);
#pragma unroll
      for (int db = 0; db < DP / 32; ++db)
#pragma unroll
        for (int v = 0; v < 16; ++v) sum[db][v] *= f;
    }
    if (w.share) {  // [dk, dv][32 keys][D] in fp32
      float* to = w.share + ((ROLE == 0 ? 32 : 0) + (lane & 31)) * static_cast<int64_t>(p.D);
#pragma unroll
      for (int db = 0; db < DP / 32; ++db)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int d = db * 32 + g * 8 + 4 * h2;
          if (d < p.D) tile::store4(to + d, sum[db][4 * g], sum[db][4 * g + 1], sum[db][4 * g + 2], sum[db][4 * g + 3]);
        }
    }
    if ((w.share && key < w.apart) || key >= p.Sk) return;
    const Mat3& m = ROLE == 0 ? p.dv : p.dk;
    T* out = at<T>(m, w.b, w.hk) + static_cast<int64_t>(key) * m.ss;
    const float f = ROLE == 0 ? (kF16 ? 1.f / (1 << kPUp) : 1.f) : (kF16 ? 1.f : p.scale);
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

// Bound by the exchange of P with its two barriers a tile: 4 x 16 heads of 2048 tokens,
// window 512, sinks, bf16 D 128 100 us (0.61 PFLOP/s of visible pairs), 34% of the cycles in
// matrix instructions, 28% in vector ones.  Three waves a SIMD instead of two took the whole
// gradient from 187 to 178-184 us.
// A workgroup has 64 keys and every tile of queries that sees any of them, except
//   * far: every query sees the sinks, so their keys' sums run over the whole sequence, not
//     over a window; the queries beyond the window of the sinks' workgroup are left to
//     workgroups of their own, which have 32 sinks and a chunk of those tiles each;
//   * chunks without far (grids of few workgroups): a chunk of the tiles.
// What several workgroups sum is joined in fp32, in a fixed order.
template <typename T, int DP>
__global__ __launch_bounds__(256, (DP * sizeof(T) > 256 ? 1 : DP * sizeof(T) > 128 ? 3 : 4)) void dkv_kernel(Params p) {
  using K = Keys<T, DP>;
  __shared__ typename K::Lds lds;
  const int nbh = p.B * p.Hkv, G = p.H / p.Hkv;
  const int bh = spread(blockIdx.x % nbh, nbh), at_ = blockIdx.x / nbh;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), pair = wave % K::kPairs;
  typename K::Work w;
  w.b = bh / p.Hkv;
  w.hk = bh % p.Hkv;
  const int len = length_of(p, w.b);
  w.nq = max(0, min(p.Sq, len - p.q_start));  // queries that exist
  const int tiles = (w.nq + kT - 1) / kT;
  const int64_t one = 64 * static_cast<int64_t>(p.D);  // floats of a share
  const int blocks = (p.Sk + kKeys - 1) / kKeys;
  float* share = p.share + static_cast<int64_t>(bh) * p.share_blocks * p.share_stride;
  if (p.far && at_ >= blocks) {
    // Chunk ck of the queries that see the 32 sinks from 32 sb through no window.
    const int sb = (at_ - blocks) / p.chunks, ck = (at_ - blocks) % p.chunks;
    w.kfirst = 32 * sb;
    w.tbase = near_end(p.Sq, p.q_start, p.window, w.kfirst / kKeys * kKeys);
    w.tcount = max(0, tiles - w.tbase);
    w.i0 = min(w.tcount * G, ck * p.chunk);
    w.i1 = min(w.tcount * G, w.i0 + p.chunk);
    w.idle = pair > 0;
    w.apart = p.Sk;
    w.share = share + sb * p.share_stride + (1 + ck) * one;
  } else {
    const bool split = !p.far && p.share_blocks > 0;
    const int kb = split ? at_ / p.chunks : at_, ck = split ? at_ % p.chunks : 0, k0 = kb * kKeys;
    w.kfirst = k0 + pair * 32;
    w.tbase = near_begin(p.q_start, k0);
    const int te = k0 >= len ? 0 : k0 < p.sinks && !p.far ? tiles : min(tiles, near_end(p.Sq, p.q_start, p.window, k0));
    w.tcount = max(0, te - w.tbase);
    const int n = w.tcount * G;
    w.i0 = split ? min(n, ck * p.chunk) : 0;
    w.i1 = split ? min(n, w.i0 + p.chunk) : n;
    w.idle = w.kfirst >= p.Sk;
    w.apart = p.far ? p.sinks : p.Sk;
    w.share = w.kfirst < 32 * p.share_blocks ? share + w.kfirst / 32 * p.share_stride + ck * one : nullptr;
  }
  if (wave >= K::kPairs) K::template run<1>(p, lds, w);
  else K::template run<0>(p, lds, w);
}

// join_kernel's workgroups of a (batch, kv head).
__device__ __host__ __forceinline__ int join_groups(const Params& p) { return (p.share_blocks * 64 * (p.D / 4) + 255) / 256; }

// dk, dv of keys whose sums several workgroups hold: the shares, added in order.
template <typename T>
__global__ __launch_bounds__(256) void join_kernel(Params p) {
  constexpr bool kF16 = __is_same(T, f16_t);
  const int vecs = p.D / 4, wgs = join_groups(p);
  const int bh = blockIdx.x / wgs, b = bh / p.Hkv, hk = bh % p.Hkv;
  const int e = blockIdx.x % wgs * 256 + threadIdx.x;
  const int row = e / vecs, d = e % vecs * 4;  // row: block, then [dk, dv], then key
  const int kb = row / 64, which = row / 32 % 2, key = kb * 32 + row % 32;
  if (kb >= p.share_blocks || key >= (p.far ? p.sinks : p.Sk)) return;
  const float* part = p.share + (static_cast<int64_t>(bh) * p.share_blocks + kb) * p.share_stride +
                      (which * 32 + row % 32) * static_cast<int64_t>(p.D) + d;
  float a[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int i = 0; i < p.shares; ++i) {
    const float4 v = *reinterpret_cast<const float4*>(part + i * (64 * static_cast<int64_t>(p.D)));
    a[0] += v.x;
    a[1] += v.y;
    a[2] += v.z;
    a[3] += v.w;
  }
  const float f = which ? (kF16 ? 1.f / (1 << kPUp) : 1.f) : (kF16 ? 1.f : p.scale);
  const Mat3& m = which ? p.dv : p.dk;
  const bool live = key < length_of(p, b);
  tile::store4(at<T>(m, b, hk) + key * m.ss + d, live ? a[0] * f : 0.f, live ? a[1] * f : 0.f, live ? a[2] * f : 0.f,
               live ? a[3] * f : 0.f);
}

// Tiles of a group's heads as one list are counted in 32 bits.
static bool list_too_long(int64_t Sq, int64_t G) { return (Sq / kT + 1) * G > 0x7fffffffLL; }

// How dkv_kernel's work is dealt out (its comment): fills p's share fields.
struct Plan {
  int64_t groups, floats;  // workgroups of dkv_kernel or, if they are more, of join_kernel; floats of the shares
};
static Plan plan(Params* p) {
  const int64_t nbh = static_cast<int64_t>(p->B) * p->Hkv;
  const SharePlan s = plan_shares(nbh, p->H / p->Hkv, p->Sq, p->Sk, p->q_start, p->window, p->sinks);
  p->share_blocks = s.blocks;
  p->shares = s.shares;
  p->chunks = s.chunks;
  p->chunk = s.chunk;
  p->far = s.far;
  p->share_stride = static_cast<int64_t>(s.shares) * 64 * p->D;
  const int64_t grid = static_cast<int64_t>((p->Sk + kKeys - 1) / kKeys) * nbh;
  const int64_t dkv = s.far ? grid + nbh * s.blocks * s.chunks : s.blocks ? grid * s.chunks : grid;
  return {std::max(dkv, nbh * join_groups(*p)), nbh * s.blocks * p->share_stride};
}

// Floats of the statistics, a whole number of 16 bytes.
static int64_t stats_floats(const Params& p) { return (static_cast<int64_t>(p.B) * p.H * p.Sq * 2 + 3) / 4 * 4; }

template <typename T, int DP>
static void launch_d(const Params& p, hipStream_t s) {
  const int nbh = p.B * p.Hkv, blocks = (p.Sk + kKeys - 1) / kKeys;
  const int wgs = p.far ? blocks + p.share_blocks * p.chunks : p.share_blocks ? blocks * p.chunks : blocks;
  // dq_few_kernel by the forward kernels' rule.
  const int64_t bh = static_cast<int64_t>(p.B) * p.H, few = (p.Sq + 31) / 32 * bh;
  constexpr int64_t kMost = few_most(sizeof(T), DP);
  if (p.Sq > 0 && few <= kMost)
    hipLaunchKernelGGL((dq_few_kernel<T, DP>), dim3(static_cast<unsigned>(few)), dim3(256), 0, s, p);
  else if (p.Sq > 0)
    hipLaunchKernelGGL((dq_kernel<T, DP>), dim3(static_cast<unsigned>((p.Sq + kCols - 1) / kCols * bh)), dim3(256), 0, s, p);
  hipLaunchKernelGGL((dkv_kernel<T, DP>), dim3(static_cast<unsigned>(wgs) * nbh), dim3(256), 0, s, p);
  if (p.share_blocks)
    hipLaunchKernelGGL((join_kernel<T>), dim3(static_cast<unsigned>(join_groups(p)) * nbh), dim3(256), 0, s, p);
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
  if (win::list_too_long(Sq, H / Hkv)) return 0;
  return (win::stats_floats(p) + win::plan(&p).floats) * 4;
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
  if (win::list_too_long(Sq, H / Hkv) || (Sq + win::kCols - 1) / win::kCols * B * H > tile::kMostGroups ||
      win::plan(&p).groups > tile::kMostGroups)
    return set_error(err, GHIP_ERR_UNSUPPORTED, "%s: problem too large", kWhat);
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
    const bool kv = x.to == &p.k || x.to == &p.v || x.to == &p.dk || x.to == &p.dv;
    if (Sq == 0 && !kv) continue;  // empty operands
    if (int rc = win::check_operand(kWhat, x.name, dtype, x.ptr, x.strides, p, kv ? p.Hkv : p.H, kv ? p.Sk : p.Sq, x.out,
                                    x.to, err))
      return rc;
  }
  if (!lse && Sq > 0) return set_error(err, GHIP_ERR_INVALID_ARG, "%s: lse is null", kWhat);
  const int64_t need = ghip_sdpa_window_bwd_workspace_bytes(dtype, B, H, Hkv, Sq, Sk, D, q_start, window, sinks);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return set_error(err, GHIP_ERR_INVALID_ARG, "%s: workspace of %lld bytes, %lld needed", kWhat,
                     static_cast<long long>(workspace ? workspace_bytes : 0), static_cast<long long>(need));
  if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
    return set_error(err, GHIP_ERR_INVALID_ARG, "%s: workspace must be 16-byte aligned", kWhat);
  p.lse = const_cast<float*>(lse);
  p.stats = static_cast<float*>(workspace);
  p.share = p.stats + win::stats_floats(p);
  p.lens = lens;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == GHIP_DTYPE_FLOAT32) win::launch<float>(p, s);
  else if (dtype == GHIP_DTYPE_FLOAT16) win::launch<f16_t>(p, s);
  else win::launch<bf16_t>(p, s);
  GHIP_CHECK(hipGetLastError(), err);
  return GHIP_OK;
}
