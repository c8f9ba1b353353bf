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

constexpr float kLazyLog2 = 8.f;  // the reference maximum may trail the true one by 2^8
// f16 weights (and their sum) are raised by 2^7, so to 2^15 at most: beside a key that takes
// nearly all of the softmax the others keep all their bits down to 2^-21 of it.
template <typename T>
constexpr float kUpLog2 = __is_same(T, f16_t) ? 7.f : 0.f;

// A wave's 32 queries, one a lane (in both halves): S^T = K Q^T and O^T = V^T P^T, so the
// softmax's running maximum, sum and rescale stay in the lane but for one exchange between
// the halves a tile.
template <typename T, int DP>
struct FwdQueries {
  using Tl = tile::Tile<T, DP>;
  using F = typename Tl::F;
  static constexpr int ND = DP / 32;
  F qf[DP / 16];
  f32x16 o[ND];
  float m, l, c;
  int pw, pos;  // positions: the wave's first, the lane's own
  int len;
  bool live;    // the lane's query exists

  __device__ __forceinline__ void place(const Params& p, int b, int qw, int lane) {
    const int qi = qw + (lane & 31);
    len = length_of(p, b);
    pw = p.q_start + qw;
    pos = p.q_start + qi;
    live = qi < p.Sq && pos < len;
    m = -INFINITY;
    l = 0.f;
    c = p.scale * 1.4426950408889634f;
  }
  // (Behind the first tile's DMA, so that the two are waited for together.)
  __device__ __forceinline__ void load(const Params& p, int b, int h, int qw, int lane) {
    const T* Q = at<T>(p.q, b, h) + static_cast<int64_t>(qw + (lane & 31)) * p.q.ss;
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) qf[s] = Tl::frag_global(Q, s, lane >> 5, p.D, live);
    tile::settle(qf);
#pragma unroll
    for (int db = 0; db < ND; ++db) o[db] = tile::splat(0.f);
  }
  // Whether any of the wave's queries, pw .. pw + 31, sees a key of key0 .. key0 + 31.
  __device__ __forceinline__ bool sees(const Params& p, int key0) const {
    return key0 <= pw + 31 && key0 < len && (key0 + 31 > pw - p.window || key0 < p.sinks);
  }

  // Keys key0 .. key0 + 31 from the tiles at sk, sv.
  __device__ __forceinline__ void step(const Params& p, const char* sk, const char* sv, int key0, int lane) {
    const int h2 = lane >> 5;
    f32x16 x = tile::splat(0.f);
    tile::pipelined<Tl::kRow, F, DP / 16>([&](int s) { return Tl::frag_row(sk, s, lane); },
                                          [&](int s, const F& a) {
                                            // fp32 products are 16 times as long: the padding's are left out.
                                            if (sizeof(T) == 4 && 16 * s >= p.D) return;
                                            x = tile::mma<T>(a, qf[s], x);
                                          });
    // x[v] is key key0 + 4 h2 + 8 (v / 4) + v % 4.
    if (key0 + 31 > pw || key0 + 32 > len || key0 <= pw + 31 - p.window) {
      asm volatile("");  // a branch: most tiles need no mask
      const uint32_t w = seen_keys(p, pos, live, len, key0 + 4 * h2);
#pragma unroll
      for (int v = 0; v < 16; ++v) x[v] = select_bit(w, (v >> 2) * 8 + (v & 3), x[v], -INFINITY);
    }
    // The first maximum is the compiler's, which waits for the products' last results;
    // v_max3_f32 directly for the others (fmaxf would quiet every one of them first).
    float mx = fmaxf(x[0], x[15]);
#pragma unroll
    for (int v = 1; v < 15; v += 2) asm("v_max3_f32 %0, %0, %1, %2" : "+v"(mx) : "v"(x[v]), "v"(x[v + 1]));
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    // The reference maximum moves only when a tile's exceeds it by more than 2^8.
    if (__builtin_amdgcn_ballot_w64((mx - m) * c > kLazyLog2)) {
      const float mnew = fmaxf(m, mx);
      const float alpha = mnew == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - mnew) * c);
      m = mnew;
      l *= alpha;
#pragma unroll
      for (int db = 0; db < ND; ++db)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[db][v] *= alpha;
    }
    const float nb = m == -INFINITY ? 0.f : kUpLog2<T> - m * c;
    float ls = 0.f;
#pragma unroll
    for (int v = 0; v < 16; ++v) {
      x[v] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[v], c, nb));
      ls += x[v];  // the sum takes the weights before they are rounded for P V
    }
    l += ls;
    const F pf[2] = {tile::pack<T>(x, 0), tile::pack<T>(x, 1)};
    tile::pipelined<Tl::kRow, F, 2 * ND>([&](int j) { return Tl::frag_tr(sv + 16 * (j / ND) * Tl::kRow, j % ND, lane); },
                                         [&](int j, const F& a) {
                                           if (sizeof(T) == 4 && 32 * (j % ND) >= p.D) return;
                                           o[j % ND] = tile::mma<T>(a, pf[j / ND], o[j % ND]);
                                         });
  }

  // o[db][v] is d = 32 db + 8 (v / 4) + 4 h2 + v % 4 of the lane's query.
  __device__ __forceinline__ void finish(const Params& p, int b, int h, int qw, int lane) {
    const int qi = qw + (lane & 31), h2 = lane >> 5;
    const float lt = l + __shfl_xor(l, 32, 64);
    if (qi >= p.Sq) return;
    const float inv = live ? 1.f / lt : 0.f;
    T* O = at<T>(p.o, b, h) + static_cast<int64_t>(qi) * p.o.ss;
#pragma unroll
    for (int db = 0; db < ND; ++db)
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
          live ? (m * c + (__builtin_amdgcn_logf(lt) - kUpLog2<T>)) * 0.6931471805599453f : -INFINITY;
  }
};

// Four waves of 32 queries each; K and V stream through two LDS stages, the next tile's DMA
// in flight during a tile.  Bound by a SIMD's matrix and vector cycles, which add up: of a
// 32 x 32 tile at D 128, 512 and about 530.  32-key tiles leave registers for three waves a
// SIMD, each computing in another's waits.  bf16, D 128, counting visible pairs: 32 heads of
// 8192 tokens causal 550 us (1.00 PFLOP/s), with a window of 2048 266 us (0.91; that sum at
// the 1.9 GHz it runs at: 246 us); 4 x 16 heads of 2048 tokens, window 512, 60 us (0.50),
// where 4 workgroups a CU run as three and one.  No faster: three LDS stages (1% at D 128, 4%
// slower at 256), windows walked so that neighbours meet at the same tiles (half the L2 misses,
// 2% faster there, 3-5% slower on windows of 128 and in fp32).
constexpr int kBQ = 128;
template <typename T, int DP>
__global__ __launch_bounds__(256, (DP * sizeof(T) > 256 ? 1 : 3)) void fwd_kernel(Params p) {
  using Tl = tile::Tile<T, DP>;
  constexpr int KT = 32, kTile = KT * Tl::kRow;
  __shared__ __attribute__((aligned(1024))) char smem[2][2][kTile];
  const uint32_t lds0 = tile::lds_addr(smem);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int nqb = (p.Sq + kBQ - 1) / kBQ;
  const int nbh = p.B * p.H;
  const int qb = nqb - 1 - static_cast<int>(blockIdx.x / nbh);
  const int bh = spread(blockIdx.x % nbh, nbh);
  const int b = bh / p.H, h = bh % p.H, hk = h / (p.H / p.Hkv);
  const int q0 = qb * kBQ, qw = q0 + wave * 32, p0 = p.q_start + q0;
  FwdQueries<T, DP> q;
  q.place(p, b, qw, lane);

  const tile::Rows K = rows_of<T>(p.k, b, hk, q.len), V = rows_of<T>(p.v, b, hk, q.len);
  tile::Loader<T, DP, KT, 4> lk, lv;
  lk.init(K.step, p.D, wave, lane);
  lv.init(V.step, p.D, wave, lane);
  const Tiles<KT> tl(p, p0, p0 < q.len ? min(q.len, p.q_start + min(q0 + kBQ, p.Sq)) : 0);
  auto issue = [&](int i) {
    const uint32_t la = lds0 + (i & 1) * (2 * kTile);
    lk.issue(K, tl(i) * KT, la, wave);
    lv.issue(V, tl(i) * KT, la + kTile, wave);
  };
  // Tile i from stage ST (known when compiled: LDS addresses are a lane's constants plus
  // immediate offsets).
  auto step = [&](auto st, int i) {
    constexpr int ST = decltype(st)::value;
    tile::landed_barrier();  // tile i is there, and nobody reads the other stage any more
    if (i + 1 < tl.n) issue(i + 1);
    if (q.sees(p, tl(i) * KT)) q.step(p, smem[ST][0], smem[ST][1], tl(i) * KT, lane);
  };
  if (tl.n > 0) issue(0);
  q.load(p, b, h, qw, lane);
  for (int i = 0; i < tl.n; i += 2) {
    step(std::integral_constant<int, 0>{}, i);
    if (i + 1 < tl.n) step(std::integral_constant<int, 1>{}, i + 1);
  }
  q.finish(p, b, h, qw, lane);
}

// Grids of few workgroups (chunks of a prompt, single tokens): a workgroup has 32 queries,
// and its four waves take the key tiles in turn, each with LDS stages of its own and no
// barrier; their shares are joined through LDS at the end.
template <typename T, int DP>
__global__ __launch_bounds__(256, 1) void fwd_few_kernel(Params p) {
  using Tl = tile::Tile<T, DP>;
  constexpr int KT = 32, kTile = KT * Tl::kRow, ND = DP / 32;
  constexpr int kStages = Tl::kRow > 256 ? 1 : 2;
  constexpr int kDma = 2 * kTile / 1024;  // DMA instructions of a tile
  __shared__ __attribute__((aligned(1024))) char smem[4][kStages][2][kTile];
  __shared__ float stat[4][2][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t lds0 = tile::lds_addr(smem[wave]);
  const int nbh = p.B * p.H;
  const int bh = spread(blockIdx.x % nbh, nbh), qw = blockIdx.x / nbh * 32;
  const int b = bh / p.H, h = bh % p.H, hk = h / (p.H / p.Hkv);
  FwdQueries<T, DP> q;
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
  q.load(p, b, h, qw, lane);
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

  // Every wave's sums against the largest maximum, added in the waves' order by the first.
  float* mine = reinterpret_cast<float*>(smem[wave]);
#pragma unroll
  for (int db = 0; db < ND; ++db)
#pragma unroll
    for (int v = 0; v < 16; ++v) mine[(db * 16 + v) * 64 + lane] = q.o[db][v];
  stat[wave][0][lane] = q.m;
  stat[wave][1][lane] = q.l;
  __syncthreads();
  if (wave != 0) return;
  float m = q.m;
#pragma unroll
  for (int w = 1; w < 4; ++w) m = fmaxf(m, stat[w][0][lane]);
  float f[4];
#pragma unroll
  for (int w = 0; w < 4; ++w) f[w] = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((stat[w][0][lane] - m) * q.c);
  q.l = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) q.l += f[w] * stat[w][1][lane];
  q.m = m;
#pragma unroll
  for (int db = 0; db < ND; ++db)
#pragma unroll
    for (int v = 0; v < 16; ++v) {
      float a = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) a += f[w] * reinterpret_cast<const float*>(smem[w])[(db * 16 + v) * 64 + lane];
      q.o[db][v] = a;
      if (v % 8 == 7) __builtin_amdgcn_sched_barrier(0);  // a few shares' reads in flight, not all
    }
  q.finish(p, b, h, qw, lane);
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

int check_operand(const char* what, const char* name, int dtype, const void* ptr, const int64_t* strides,
                  const Params& p, int heads, int rows, bool out, Mat3* m, GHipError* err) {
  if (!ptr || !strides) return set_error(err, GHIP_ERR_INVALID_ARG, "%s: %s is null", what, name);
  const int64_t es = dtype == GHIP_DTYPE_FLOAT32 ? 4 : 2;
  const int64_t al = out ? 4 : 16 / es;
  const int n[3] = {p.B, heads, rows};
  for (int i = 0; i < 3; ++i)
    if (strides[i] < 0 || (n[i] > 1 && strides[i] % al != 0))
      return set_error(err, GHIP_ERR_UNSUPPORTED, "%s: %s needs non-negative strides that are multiples of %d elements",
                       what, name, static_cast<int>(al));
  if (rows > 1 && strides[2] >= ((int64_t{1} << 31) / es - 256) / 64)
    return set_error(err, GHIP_ERR_UNSUPPORTED, "%s: %s needs a sequence stride below 32 MiB", what, name);
  if (reinterpret_cast<uintptr_t>(ptr) % (al * es) != 0)
    return set_error(err, GHIP_ERR_UNSUPPORTED, "%s: %s must be %d-byte aligned", what, name, static_cast<int>(al * es));
  // (A tile's rows behind the only one lie behind it, so past the descriptor's end.)
  *m = Mat3{ptr, p.B > 1 ? strides[0] : 0, heads > 1 ? strides[1] : 0, rows > 1 ? strides[2] : p.D};
  return GHIP_OK;
}

// Which kernel: fwd_few_kernel while its workgroups, four times as many, run at once (one
// a CU, rows of 128 bytes two).  32 heads over 8, windows of 128 / 1024, us a call in a graph,
// fwd_few_kernel against fwd_kernel at so many workgroups of 32 queries:
//   bf16 D 128, 256: 9.9 / 18.6 against 11.6 / 31.3; 288: 17.6 / 33.2 against 11.7 / 31.1
//   bf16 D 256, 256: 19.4 / 37.5 against 22.0 / 56.6; 288: 35.6 / 68.9 against 22.2 / 56.6
//   f16 D 64, 512: 7.7 / 15.4 against 9.4 / 25.5; 544: 11.8 / 23.3 against 9.5 / 25.6
// In fp32, where a tile's products take 16 times as long, a third round still breaks even:
//   D 64, 512: 21.4 / 55.8 against 23.9 / 88.0; 768: 30.4 / 81.8 against 24.4 / 88.0; 896: 38.9
//   / 108 against 24.6 / 88.5;  D 128, 768: 50.8 / 144 against 44.7 / 166; 896: 66.7 / 190
//   against 45.6 / 167
// (768, windows of 192 to 512: within 5% either way at D 128, 3 to 13% behind at D 64; a
// window of 2048: a quarter ahead.)  The gradient's dq_few_kernel goes by the same rule: whole
// gradients bf16 D 128, 256: 37.3 / 49.8 against 39.1 / 63.6; 288: 46.9 / 68.3 against 40.2 /
// 66.8; fp32 D 64, 768: 103 / 339 against 95 / 346; 896: 116 / 412 against 95 / 383.
template <typename T, int DP>
static void launch_d(const Params& p, hipStream_t s) {
  const int64_t bh = static_cast<int64_t>(p.B) * p.H, few = (p.Sq + 31) / 32 * bh, many = (p.Sq + kBQ - 1) / kBQ * bh;
  constexpr int64_t kMost = few_most(sizeof(T), DP);
  if (few <= kMost)
    hipLaunchKernelGGL((fwd_few_kernel<T, DP>), dim3(static_cast<unsigned>(few)), dim3(256), 0, s, p);
  else
    hipLaunchKernelGGL((fwd_kernel<T, DP>), dim3(static_cast<unsigned>(many)), dim3(256), 0, s, p);
}
template <typename T>
static void launch_fwd(const Params& p, hipStream_t s) {
  if (p.D <= 64) launch_d<T, 64>(p, s);
  else if (p.D <= 128) launch_d<T, 128>(p, s);
  else if constexpr (sizeof(T) == 2) launch_d<T, 256>(p, s);
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
  if ((Sq + win::kBQ - 1) / win::kBQ * B * H > tile::kMostGroups)
    return set_error(err, GHIP_ERR_UNSUPPORTED, "%s: problem too large", kWhat);
  if (int rc = win::check_operand(kWhat, "q", dtype, q, q_strides, p, p.H, p.Sq, false, &p.q, err)) return rc;
  if (int rc = win::check_operand(kWhat, "k", dtype, k, k_strides, p, p.Hkv, p.Sk, false, &p.k, err)) return rc;
  if (int rc = win::check_operand(kWhat, "v", dtype, v, v_strides, p, p.Hkv, p.Sk, false, &p.v, err)) return rc;
  if (int rc = win::check_operand(kWhat, "o", dtype, o, o_strides, p, p.H, p.Sq, true, &p.o, err)) return rc;
  p.lse = lse;
  p.lens = lens;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == GHIP_DTYPE_FLOAT32) win::launch_fwd<float>(p, s);
  else if (dtype == GHIP_DTYPE_FLOAT16) win::launch_fwd<f16_t>(p, s);
  else win::launch_fwd<bf16_t>(p, s);
  GHIP_CHECK(hipGetLastError(), err);
  return GHIP_OK;
}
