// Causal attention over a sliding window with sinks: the query at position p sees key
// j iff j <= p, j < len, and j > p - window or j < sinks.
//   lse = log sum_j exp(scale q.k_j),   o = sum_j exp(scale q.k_j - lse) v_j
// One pass over the visible keys with the running maximum and sum of the softmax;
// scores never reach memory.  No reference op: this stands beside the causal attention
// of FusedScaledDotProductAttention (mpsgraph/gomlx/function.go:2669-2907), whose mask
// operand would cost Sq x Sk values and every key tile.
#include <type_traits>

#include "attn_window.h"

namespace ghip {
namespace win {

using tile::f32x16;

constexpr int kWaves = 4, kQW = 32, kBQ = kWaves * kQW, kKT = 64;
constexpr float kLazyLog2 = 8.f;  // the reference maximum may trail the true one by 2^8

// S^T = K Q^T and O^T = V^T P^T: a lane owns one query (column), so the softmax's
// maximum, sum and rescale stay in the lane but for one exchange between the halves of
// the wave.  K and V stream through two LDS stages, the next tile's DMA in flight
// during a tile.
template <typename T, int DP>
__global__ __launch_bounds__(256, DP * sizeof(T) > 256 ? 1 : 2) void fwd_kernel(Params p) {
  using Tl = tile::Tile<T, DP>;
  using F = typename Tl::F;
  constexpr int kTile = kKT * Tl::kRow;
  __shared__ __attribute__((aligned(1024))) char smem[2][2][kTile];
  const uint32_t lds0 = tile::lds_addr(smem);

  const int lane = threadIdx.x & 63, h2 = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int nqb = (p.Sq + kBQ - 1) / kBQ;
  const int nbh = p.B * p.H;
  const int qb = nqb - 1 - static_cast<int>(blockIdx.x / nbh);
  const int bh = blockIdx.x % nbh;
  const int b = bh / p.H, h = bh % p.H, hk = h / (p.H / p.Hkv);
  const int len = length_of(p, b);
  const int q0 = qb * kBQ, qw = q0 + wave * kQW, qi = qw + (lane & 31);
  const int pos = p.q_start + qi, pw = p.q_start + qw;
  const bool live = qi < p.Sq && pos < len;

  const T* Q = at<T>(p.q, b, h) + static_cast<int64_t>(qi) * p.q.ss;
  F qf[DP / 16];
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) qf[s] = Tl::frag_global(Q, s, h2, p.D, live);

  tile::settle(qf);

  const tile::Rows K = rows_of<T>(p.k, b, hk, len), V = rows_of<T>(p.v, b, hk, len);
  tile::Loader<T, DP, kKT, kWaves> lk, lv;
  lk.init(K.step, p.D, wave, lane);
  lv.init(V.step, p.D, wave, lane);
  const int p0 = p.q_start + q0;
  const Tiles<kKT> tl(p, p0, p0 < len ? min(len, p.q_start + min(q0 + kBQ, p.Sq)) : 0);
  auto issue = [&](int i) {
    const uint32_t la = lds0 + (i & 1) * (2 * kTile);
    const int row = tl(i) * kKT;
    lk.issue(K, row, la, wave);
    lv.issue(V, row, la + kTile, wave);
  };

  f32x16 o[DP / 32];
#pragma unroll
  for (int db = 0; db < DP / 32; ++db) o[db] = tile::splat(0.f);
  float m = -INFINITY, l = 0.f;
  const float c = p.scale * 1.4426950408889634f;

  // Tile i from stage ST (known when compiled: LDS addresses are a lane's constants plus
  // immediate offsets).
  auto step = [&](auto st, int i) {
    constexpr int ST = decltype(st)::value;
    tile::landed_barrier();  // tile i is there, and nobody reads the other stage any more
    if (i + 1 < tl.n) issue(i + 1);
    const int key0 = tl(i) * kKT;
    // The wave's queries pw .. pw + 31 see nothing of this tile.
    if (key0 > pw + kQW - 1 || (key0 + kKT - 1 <= pw - p.window && key0 >= p.sinks)) return;
    const char* sk = smem[ST][0];
    const char* sv = smem[ST][1];
    f32x16 s0 = tile::splat(0.f), s1 = s0;
    tile::pipelined<Tl::kRow, F, DP / 8>([&](int j) { return Tl::frag_row(sk + (j & 1) * 32 * Tl::kRow, j >> 1, lane); },
                               [&](int j, const F& a) {
                                 f32x16& x = j & 1 ? s1 : s0;
                                 x = tile::mma<T>(a, qf[j >> 1], x);
                               });
    // s{kb}[v] is key key0 + 32 kb + 4 h2 + kv, kv = 8 (v / 4) + v % 4.
    if (key0 + kKT - 1 > pw || key0 + kKT > len || key0 <= pw + kQW - 1 - p.window) {
      asm volatile("");  // a branch: most tiles need no mask
      const uint32_t w0 = seen_keys(p, pos, live, len, key0 + 4 * h2), w1 = seen_keys(p, pos, live, len, key0 + 32 + 4 * h2);
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        const int kv = (v >> 2) * 8 + (v & 3);
        s0[v] = select_bit(w0, kv, s0[v], -INFINITY);
        s1[v] = select_bit(w1, kv, s1[v], -INFINITY);
      }
    }
    // The first maximum is the compiler's, which waits for the products' last results;
    // v_max3_f32 directly for the others (fmaxf would quiet every one of them first).
    float mx = fmaxf(s0[0], s1[0]);
#pragma unroll
    for (int v = 1; v < 16; ++v) asm("v_max3_f32 %0, %0, %1, %2" : "+v"(mx) : "v"(s0[v]), "v"(s1[v]));
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    // The reference maximum moves only when a tile's exceeds it by more than 2^8.
    if (__builtin_amdgcn_ballot_w64((mx - m) * c > kLazyLog2)) {
      const float mnew = fmaxf(m, mx);
      const float alpha = mnew == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - mnew) * c);
      m = mnew;
      l *= alpha;
#pragma unroll
      for (int db = 0; db < DP / 32; ++db)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[db][v] *= alpha;
    }
    const float nb = m == -INFINITY ? 0.f : -m * c;
    float l0 = 0.f, l1 = 0.f;
#pragma unroll
    for (int v = 0; v < 16; ++v) {
      s0[v] = __builtin_amdgcn_exp2f(__builtin_fmaf(s0[v], c, nb));
      s1[v] = __builtin_amdgcn_exp2f(__builtin_fmaf(s1[v], c, nb));
      l0 += s0[v];  // the sum takes the weights before they are rounded for P V
      l1 += s1[v];
    }
    l += l0 + l1;
    F pf[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) pf[s] = s < 2 ? tile::pack<T>(s0, s) : tile::pack<T>(s1, s - 2);
    constexpr int ND = DP / 32;
    tile::pipelined<Tl::kRow, F, 4 * ND>([&](int j) { return Tl::frag_tr(sv + 16 * (j / ND) * Tl::kRow, j % ND, lane); },
                               [&](int j, const F& a) { o[j % ND] = tile::mma<T>(a, pf[j / ND], o[j % ND]); });
  };
  if (tl.n > 0) issue(0);
  for (int i = 0; i < tl.n; i += 2) {
    step(std::integral_constant<int, 0>{}, i);
    if (i + 1 < tl.n) step(std::integral_constant<int, 1>{}, i + 1);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");

  // o[db][v] is d = 32 db + 8 (v / 4) + 4 h2 + v % 4 of query qi.
  const float lt = l + __shfl_xor(l, 32, 64);
  if (qi >= p.Sq) return;
  const float inv = live ? 1.f / lt : 0.f;
  T* O = at<T>(p.o, b, h) + static_cast<int64_t>(qi) * p.o.ss;
#pragma unroll
  for (int db = 0; db < DP / 32; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = db * 32 + g * 8 + 4 * h2;
      if (d >= p.D) continue;
      float r[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) r[e] = live ? o[db][4 * g + e] * inv : 0.f;
      tile::store4(O + d, r[0], r[1], r[2], r[3]);
    }
  if (p.lse && h2 == 0)
    p.lse[(static_cast<int64_t>(b) * p.H + h) * p.Sq + qi] =
        live ? (m * c + __builtin_amdgcn_logf(lt)) * 0.6931471805599453f : -INFINITY;
}

int check_problem(const char* what, int dtype, int64_t B, int64_t H, int64_t Hkv, int64_t Sq, int64_t Sk, int64_t D,
                  int64_t q_start, int64_t window, int64_t sinks, float scale, Params* p, GHipError* err) {
  if (B < 0 || H <= 0 || Hkv <= 0 || Sq < 0 || Sk < 0 || D <= 0)
    return set_error(err, GHIP_ERR_INVALID_ARG, "%s: bad sizes", what);
  if (H % Hkv != 0)
    return set_error(err, GHIP_ERR_INVALID_ARG, "%s: num_heads (%lld) must be a multiple of num_kv_heads (%lld)", what,
                     static_cast<long long>(H), static_cast<long long>(Hkv));
  if (q_start < 0 || q_start > Sk || Sq > Sk - q_start)
    return set_error(err, GHIP_ERR_INVALID_ARG,
                     "%s: queries %lld .. %lld lie outside the %lld keys", what, static_cast<long long>(q_start),
                     static_cast<long long>(q_start + Sq), static_cast<long long>(Sk));
  if (window < 0 || sinks < 0)
    return set_error(err, GHIP_ERR_INVALID_ARG, "%s: window and sinks must not be negative", what);
  if (!(scale > 0.f) || !(scale < 1e30f))
    return set_error(err, GHIP_ERR_INVALID_ARG, "%s: the scale must be positive and finite", what);
  const bool f32 = dtype == GHIP_DTYPE_FLOAT32;
  if (!f32 && dtype != GHIP_DTYPE_BFLOAT16 && dtype != GHIP_DTYPE_FLOAT16)
    return set_error(err, GHIP_ERR_UNSUPPORTED, "%s: needs float32, bfloat16 or float16", what);
  if (D % (f32 ? 4 : 8) != 0 || D > (f32 ? 128 : 256))
    return set_error(err, GHIP_ERR_UNSUPPORTED,
                     "%s: needs a head dim that is a multiple of 8 up to 256 (float32: of 4 up to 128)", what);
  constexpr int64_t kMost = int64_t{1} << 30;
  if (Sk > kMost / 2 || B > kMost || H > kMost || B * H > kMost || ((Sk + 127) / 128) * B * H > 0x7fffffffLL)
    return set_error(err, GHIP_ERR_UNSUPPORTED, "%s: problem too large", what);
  p->B = static_cast<int>(B); p->H = static_cast<int>(H); p->Hkv = static_cast<int>(Hkv);
  p->Sq = static_cast<int>(Sq); p->Sk = static_cast<int>(Sk); p->D = static_cast<int>(D);
  p->q_start = static_cast<int>(q_start);
  p->window = static_cast<int>(window == 0 || window > kMost ? kMost : window);
  p->sinks = static_cast<int>(sinks > Sk ? Sk : sinks);
  p->scale = scale;
  return GHIP_OK;
}

int check_operand(const char* what, const char* name, int dtype, const void* ptr, const int64_t* strides, bool out,
                  Mat3* m, GHipError* err) {
  if (!ptr || !strides) return set_error(err, GHIP_ERR_INVALID_ARG, "%s: %s is null", what, name);
  const int64_t es = dtype == GHIP_DTYPE_FLOAT32 ? 4 : 2;
  const int64_t al = out ? 4 : 16 / es;
  for (int i = 0; i < 3; ++i)
    if (strides[i] < 0 || strides[i] % al != 0)
      return set_error(err, GHIP_ERR_UNSUPPORTED, "%s: %s needs non-negative strides that are multiples of %d elements",
                       what, name, static_cast<int>(al));
  if ((64 * strides[2] + 256) * es >= (int64_t{1} << 31))
    return set_error(err, GHIP_ERR_UNSUPPORTED, "%s: %s needs a sequence stride below 32 MiB", what, name);
  if (reinterpret_cast<uintptr_t>(ptr) % (al * es) != 0)
    return set_error(err, GHIP_ERR_UNSUPPORTED, "%s: %s must be %d-byte aligned", what, name, static_cast<int>(al * es));
  *m = Mat3{ptr, strides[0], strides[1], strides[2]};
  return GHIP_OK;
}

template <typename T>
static void launch_fwd(const Params& p, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>((p.Sq + kBQ - 1) / kBQ * p.B * p.H));
  if (p.D <= 64) hipLaunchKernelGGL((fwd_kernel<T, 64>), grid, dim3(256), 0, s, p);
  else if (p.D <= 128) hipLaunchKernelGGL((fwd_kernel<T, 128>), grid, dim3(256), 0, s, p);
  else if constexpr (sizeof(T) == 2) hipLaunchKernelGGL((fwd_kernel<T, 256>), grid, dim3(256), 0, s, p);
}

}  // namespace win
}  // namespace ghip

using namespace ghip;

extern "C" int ghip_sdpa_window_fwd(int dtype, const void* q, const void* k, const void* v, void* o, float* lse,
                                    int64_t B, int64_t H, int64_t Hkv, int64_t Sq, int64_t Sk, int64_t D,
                                    const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides,
                                    const int64_t* o_strides, int64_t q_start, int64_t window, int64_t sinks,
                                    const int32_t* lens, float scale, void* stream, GHipError* err) {
  static const char kWhat[] = "sdpa_window_fwd";
  win::Params p{};
  if (int rc = win::check_problem(kWhat, dtype, B, H, Hkv, Sq, Sk, D, q_start, window, sinks, scale, &p, err)) return rc;
  if (B == 0 || Sq == 0) return GHIP_OK;
  if (int rc = win::check_operand(kWhat, "q", dtype, q, q_strides, false, &p.q, err)) return rc;
  if (int rc = win::check_operand(kWhat, "k", dtype, k, k_strides, false, &p.k, err)) return rc;
  if (int rc = win::check_operand(kWhat, "v", dtype, v, v_strides, false, &p.v, err)) return rc;
  if (int rc = win::check_operand(kWhat, "o", dtype, o, o_strides, true, &p.o, err)) return rc;
  p.lse = lse;
  p.lens = lens;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == GHIP_DTYPE_FLOAT32) win::launch_fwd<float>(p, s);
  else if (dtype == GHIP_DTYPE_FLOAT16) win::launch_fwd<f16_t>(p, s);
  else win::launch_fwd<bf16_t>(p, s);
  GHIP_CHECK(hipGetLastError(), err);
  return GHIP_OK;
}
