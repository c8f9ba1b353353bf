// Gradient of the sliding-window attention of k_attn_window.hip, from its output and
// log-sum-exp:
//   P = exp(scale q.k - lse) where the query sees the key,   delta = sum_d do o
//   dV = P^T dO,   dS = P (dO V^T - delta),   dQ = scale dS K,   dK = scale dS^T Q
// (dK and dV summed over the query heads that share a kv head).  Two kernels that each
// evaluate P and dS again, so nothing of size Sq x Sk is stored and no sum depends on
// the order of atomics: the first owns queries (dQ, and delta for the second), the
// second keys.
#include "attn_window.h"

namespace ghip {
namespace win {

using tile::f32x16;

constexpr int kWaves = 4, kRW = 32, kBR = kWaves * kRW, kKT = 64, kQT = 64;
constexpr float kLog2e = 1.4426950408889634f;

// dQ: the transposed arrangement of the forward kernel.  A lane owns one query; S^T = K
// Q^T and dP^T = V dO^T come out as columns, dS^T enters dQ^T += K^T dS^T from the
// registers.  The product's accumulator starts at -delta, and the scale sits in the
// exponent (P scale = 2^(s c - lse2 + log2 scale)), so an element costs one FMA, one
// exponential and one multiplication.
template <typename T, int DP>
__global__ __launch_bounds__(256, DP * sizeof(T) > 256 ? 1 : 2) void dq_kernel(Params p) {
  using Tl = tile::Tile<T, DP>;
  using F = typename Tl::F;
  constexpr int kTile = kKT * Tl::kRow;
  __shared__ __attribute__((aligned(1024))) char smem[2][2][kTile];
  const uint32_t lds0 = tile::lds_addr(smem);

  const int lane = threadIdx.x & 63, h2 = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int nqb = (p.Sq + kBR - 1) / kBR;
  const int nbh = p.B * p.H;
  const int qb = nqb - 1 - static_cast<int>(blockIdx.x / nbh);
  const int bh = blockIdx.x % nbh;
  const int b = bh / p.H, h = bh % p.H, hk = h / (p.H / p.Hkv);
  const int len = length_of(p, b);
  const int q0 = qb * kBR, qw = q0 + wave * kRW, qi = qw + (lane & 31);
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
  const float nl = live ? __builtin_amdgcn_logf(p.scale) - p.lse[row] * kLog2e : 0.f;

  const tile::Rows K = rows_of<T>(p.k, b, hk, len, p.D), V = rows_of<T>(p.v, b, hk, len, p.D);
  tile::Loader<T, DP, kKT, kWaves> lk, lv;
  lk.init(K.step, p.D, wave, lane);
  lv.init(V.step, p.D, wave, lane);
  const int p0 = p.q_start + q0;
  const Tiles<kKT> tl(p, p0, p0 < len ? min(len, p.q_start + min(q0 + kBR, p.Sq)) : 0);
  auto issue = [&](int i) {
    const uint32_t la = lds0 + (i & 1) * (2 * kTile);
    const int64_t r = static_cast<int64_t>(tl(i)) * kKT;
    lk.issue(K, r, la, wave);
    lv.issue(V, r, la + kTile, wave);
  };

  f32x16 dq[DP / 32];
#pragma unroll
  for (int db = 0; db < DP / 32; ++db) dq[db] = tile::splat(0.f);

  if (tl.n > 0) issue(0);
  for (int i = 0; i < tl.n; ++i) {
    tile::landed_barrier();
    if (i + 1 < tl.n) issue(i + 1);
    const int key0 = tl(i) * kKT;
    if (key0 > pw + kRW - 1 || (key0 + kKT - 1 <= pw - p.window && key0 >= p.sinks)) continue;
    const char* sk = smem[i & 1][0];
    const char* sv = smem[i & 1][1];
    const bool masked = key0 + kKT - 1 > pw || key0 + kKT > len || key0 <= pw + kRW - 1 - p.window;
#pragma unroll
    for (int kb = 0; kb < kKT / 32; ++kb) {
      f32x16 x = tile::splat(0.f), g = tile::splat(nd);
#pragma unroll
      for (int s = 0; s < DP / 16; ++s) {
        x = tile::mma<T>(Tl::frag_row(sk, 32 * kb + (lane & 31), s, h2), qf[s], x);
        g = tile::mma<T>(Tl::frag_row(sv, 32 * kb + (lane & 31), s, h2), gf[s], g);
      }
#pragma unroll
      for (int v = 0; v < 16; ++v) x[v] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[v], c, nl)) * g[v];
      if (masked) {
        const int base = key0 + 32 * kb + 4 * h2;
        const int hi = (live ? min(len, pos + 1) : 0) - base, lo = pos - p.window + 1 - base, sn = p.sinks - base;
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const int kv = (v >> 2) * 8 + (v & 3);
          x[v] = kv < hi && (kv >= lo || kv < sn) ? x[v] : 0.f;
        }
      }
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const F df = tile::pack<T>(x, s);
#pragma unroll
        for (int db = 0; db < DP / 32; ++db) dq[db] = tile::mma<T>(Tl::frag_tr(sk, db, 32 * kb, s, lane), df, dq[db]);
      }
    }
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

// dK, dV: a lane owns one key; S = Q K^T and dP = dO V^T come out with the lane's key
// as their column, so P and dS enter dV^T += dO^T P and dK^T += Q^T dS from the
// registers.  K and V stay in registers; Q and dO stream through two LDS stages, head
// after head of the group, with each query's log-sum-exp and delta beside them.
// f16 only: P is at most 1 and of order 1 / window, so it is rounded 2^8 times larger
// (small weights would be subnormal), and dS is rounded with the scale applied.
template <typename T, int DP>
__global__ __launch_bounds__(256, DP * sizeof(T) > 128 ? 1 : 2) void dkv_kernel(Params p) {
  using Tl = tile::Tile<T, DP>;
  using F = typename Tl::F;
  constexpr bool kF16 = __is_same(T, f16_t);
  constexpr int kTile = kQT * Tl::kRow;
  __shared__ __attribute__((aligned(1024))) char smem[2][2][kTile];
  __shared__ __attribute__((aligned(16))) float stat[2][2][kQT];  // -lse in base 2, -delta
  const uint32_t lds0 = tile::lds_addr(smem);

  const int lane = threadIdx.x & 63, h2 = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int nbh = p.B * p.Hkv;
  const int kb = blockIdx.x / nbh;  // the sinks' block, which every query sees, first
  const int b = blockIdx.x % nbh / p.Hkv, hk = blockIdx.x % p.Hkv;
  const int G = p.H / p.Hkv;
  const int len = length_of(p, b);
  const int k0 = kb * kBR, kw = k0 + wave * kRW, key = kw + (lane & 31);
  const bool live = key < len;

  F kf[DP / 16], vf[DP / 16];
  {
    const T* K = at<T>(p.k, b, hk) + static_cast<int64_t>(key) * p.k.ss;
    const T* V = at<T>(p.v, b, hk) + static_cast<int64_t>(key) * p.v.ss;
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
      kf[s] = Tl::frag_global(K, s, h2, p.D, live);
      vf[s] = Tl::frag_global(V, s, h2, p.D, live);
    }
  }
  // Queries qa .. qe - 1 see a key of the block.
  const int nq = max(0, min(p.Sq, len - p.q_start));  // queries that exist
  const int reach = k0 < p.sinks || k0 + kBR - 1 + p.window > p.q_start + p.Sq ? nq
                    : min(nq, max(0, k0 + kBR - 1 + p.window - p.q_start));
  const int ta = max(0, k0 - p.q_start) / kQT;
  const int nt = max(0, (k0 < len ? (reach + kQT - 1) / kQT : 0) - ta);
  const int n = nt * G;

  tile::Loader<T, DP, kQT, kWaves> lq, lg;
  lq.init(p.q.ss * Tl::kEs, p.D, wave, lane);
  lg.init(p.dout.ss * Tl::kEs, p.D, wave, lane);
  const float c = p.scale * kLog2e;
  float st = 0.f;  // this thread's entry of the next tile's statistics
  auto issue = [&](int i) {
    const int h = hk * G + i / nt, t = ta + i % nt;
    const int r = t * kQT + (threadIdx.x & (kQT - 1));
    st = 0.f;
    if (threadIdx.x < 2 * kQT && r < nq) {
      const int64_t at_row = (static_cast<int64_t>(b) * p.H + h) * p.Sq + r;
      st = threadIdx.x < kQT ? (kF16 ? 8.f : 0.f) - p.lse[at_row] * kLog2e : p.ndelta[at_row];
    }
    const uint32_t la = lds0 + (i & 1) * (2 * kTile);
    lq.issue(rows_of<T>(p.q, b, h, nq, p.D), static_cast<int64_t>(t) * kQT, la, wave);
    lg.issue(rows_of<T>(p.dout, b, h, nq, p.D), static_cast<int64_t>(t) * kQT, la + kTile, wave);
  };
  auto put = [&](int i) {
    if (threadIdx.x < 2 * kQT) stat[i & 1][threadIdx.x / kQT][threadIdx.x % kQT] = st;
  };

  f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
  for (int db = 0; db < DP / 32; ++db) dk[db] = dv[db] = tile::splat(0.f);

  if (n > 0) {
    issue(0);
    put(0);
  }
  for (int i = 0; i < n; ++i) {
    tile::landed_barrier();
    if (i + 1 < n) issue(i + 1);
    const char* sq = smem[i & 1][0];
    const char* sg = smem[i & 1][1];
#pragma unroll
    for (int rb = 0; rb < kQT / 32; ++rb) {
      const int p0 = p.q_start + (ta + i % nt) * kQT + 32 * rb;  // the first row's position
      if (p0 + 31 < kw || (p0 >= kw + 31 + p.window && kw >= p.sinks) || p0 - p.q_start >= nq) continue;
      f32x16 x = tile::splat(0.f), g;
      const float* nl = &stat[i & 1][0][32 * rb + 4 * h2];
      const float* nd = &stat[i & 1][1][32 * rb + 4 * h2];
#pragma unroll
      for (int v = 0; v < 16; ++v) g[v] = nd[(v >> 2) * 8 + (v & 3)];
#pragma unroll
      for (int s = 0; s < DP / 16; ++s) {
        x = tile::mma<T>(Tl::frag_row(sq, 32 * rb + (lane & 31), s, h2), kf[s], x);
        g = tile::mma<T>(Tl::frag_row(sg, 32 * rb + (lane & 31), s, h2), vf[s], g);
      }
#pragma unroll
      for (int v = 0; v < 16; ++v) x[v] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[v], c, nl[(v >> 2) * 8 + (v & 3)]));
      if (p0 < kw + 31 || p0 + 31 - p.q_start >= nq || (p0 + 31 >= kw + p.window && kw + 31 >= p.sinks)) {
        const int end = p.q_start + nq;
        const int lo = key - p0 - 4 * h2;
        const int hi = (key < p.sinks ? end : min(end, key + p.window)) - p0 - 4 * h2;
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const int rv = (v >> 2) * 8 + (v & 3);
          x[v] = rv >= lo && rv < hi ? x[v] : 0.f;
        }
      }
#pragma unroll
      for (int v = 0; v < 16; ++v) g[v] *= kF16 ? x[v] * (p.scale * 0x1p-8f) : x[v];
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const F pf = tile::pack<T>(x, s), df = tile::pack<T>(g, s);
#pragma unroll
        for (int db = 0; db < DP / 32; ++db) {
          dv[db] = tile::mma<T>(Tl::frag_tr(sg, db, 32 * rb, s, lane), pf, dv[db]);
          dk[db] = tile::mma<T>(Tl::frag_tr(sq, db, 32 * rb, s, lane), df, dk[db]);
        }
      }
    }
    if (i + 1 < n) put(i + 1);
  }
  if (key >= p.Sk) return;
  T* ok = at<T>(p.dk, b, hk) + static_cast<int64_t>(key) * p.dk.ss;
  T* ov = at<T>(p.dv, b, hk) + static_cast<int64_t>(key) * p.dv.ss;
  const float ck = kF16 ? 1.f : p.scale, cv = kF16 ? 0x1p-8f : 1.f;
#pragma unroll
  for (int db = 0; db < DP / 32; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = db * 32 + g * 8 + 4 * h2;
      if (d >= p.D) continue;
      float rk[4], rv[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        rk[e] = live ? dk[db][4 * g + e] * ck : 0.f;
        rv[e] = live ? dv[db][4 * g + e] * cv : 0.f;
      }
      tile::store4(ok + d, rk[0], rk[1], rk[2], rk[3]);
      tile::store4(ov + d, rv[0], rv[1], rv[2], rv[3]);
    }
}

template <typename T, int DP>
static void launch_d(const Params& p, hipStream_t s) {
  const dim3 gq(static_cast<unsigned>((p.Sq + kBR - 1) / kBR * p.B * p.H));
  const dim3 gk(static_cast<unsigned>((p.Sk + kBR - 1) / kBR * p.B * p.Hkv));
  if (p.Sq > 0) hipLaunchKernelGGL((dq_kernel<T, DP>), gq, dim3(256), 0, s, p);
  hipLaunchKernelGGL((dkv_kernel<T, DP>), gk, dim3(256), 0, s, p);
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
  return B * H * Sq * 4;
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
  p.lens = lens;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == GHIP_DTYPE_FLOAT32) win::launch<float>(p, s);
  else if (dtype == GHIP_DTYPE_FLOAT16) win::launch<f16_t>(p, s);
  else win::launch<bf16_t>(p, s);
  GHIP_CHECK(hipGetLastError(), err);
  return GHIP_OK;
}
