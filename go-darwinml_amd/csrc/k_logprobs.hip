// Log probabilities of given tokens, entropy, log-sum-exp and the largest logits of rows, in one
// pass over them, and the gradient of the logits.
//
//   lse = log sum_v exp x_v,  logp = x_id - lse,  entropy = lse - sum_v p_v x_v,  x = scale * logits
//
// No reference op (GoMLX composes it of FusedSoftmax and primitives); beside the log-softmax
// rows, which write V values a row.  Bound by the bytes of the logits, read once.
#include <algorithm>

#include "common.h"

// Products are fused with sums where it says so, nowhere else: the lanes that join their sums in
// pairs then hold the same bits, and a token's log probability is the same in every output.
#pragma clang fp contract(off)

namespace ghip {
namespace logprobs {

constexpr int kMostTop = 32;
constexpr int kMostSlices = 64;
constexpr int kRun = 4;      // vectors a lane takes at a time
constexpr int kQueue = 256;  // candidates a wave holds
constexpr float kLn2 = 0.6931471805599453f, kLog2e = 1.4426950408889634f;
constexpr float kFar = -200.f;  // 2^kFar is 0: what stands for log 0 in a product with a weight of 0
constexpr int64_t kMostGroups = (int64_t{1} << 24) - 1;

struct Params {
  const char* x;
  int64_t stride;  // bytes
  const int32_t* ids;
  int64_t N;
  int V, top, slices, per;  // per: vectors of a slice
  float c;                  // scale * log2 e
  float* logp;
  float* entropy;
  float* lse;
  float* top_logps;
  int32_t* top_ids;
  float4* stats;   // [N][slices]: maximum, sum, sum of weight times exponent
  uint64_t* keys;  // [N][slices][top]
};

// A running softmax in powers of two: m = max of x c, s = sum of w, e = sum of w u, where
// u = x c - m and w = 2^u.
struct Stats {
  float m = -INFINITY, s = 0.f, e = 0.f;
  // The same sums beside another maximum.
  __device__ __forceinline__ void move(float to) {
    const float base = to == -INFINITY ? 0.f : to, d = m - base, f = __builtin_amdgcn_exp2f(d);
    e = f * __builtin_fmaf(fmaxf(d, kFar), s, e);
    s *= f;
    m = to;
  }
  __device__ __forceinline__ void join(Stats o) {
    const float to = fmaxf(m, o.m);
    move(to);
    o.move(to);
    s += o.s;
    e += o.e;
  }
  template <int N>
  __device__ __forceinline__ void add(const float (&x)[N], float most, float c) {
    move(fmaxf(m, most * c));
    const float base = m == -INFINITY ? 0.f : m;
    float s2 = 0.f, e2 = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float u = __builtin_fmaf(x[i], c, -base), w = __builtin_amdgcn_exp2f(u);
      s2 += w;
      e2 = __builtin_fmaf(w, fmaxf(u, kFar), e2);  // (-inf: 0, not 0 times -inf; NaN stays in w)
    }
    s += s2;
    e += e2;
  }
};
__device__ __forceinline__ Stats wave_join(Stats a) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    Stats b;
    b.m = __shfl_xor(a.m, d, 64);
    b.s = __shfl_xor(a.s, d, 64);
    b.e = __shfl_xor(a.e, d, 64);
    a.join(b);
  }
  return a;
}

// Logits in the order of unsigned integers: larger first, NaN above all, -0 as 0; then a key
// whose lower half puts smaller indices first.  No key is 0.
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t order) {
  return __uint_as_float(order & 0x80000000u ? order & 0x7fffffffu : ~order);
}
__device__ __forceinline__ uint64_t key_of(float x, uint32_t i) {
  return static_cast<uint64_t>(order_of(x)) << 32 | static_cast<uint32_t>(~i);
}

__device__ __forceinline__ int rank_in(uint64_t mask) {  // set bits below this lane's
  return __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(mask >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(mask), 0));
}

// The largest number of BITS leading bits (the others 0) that at least k lanes' values reach.
template <typename U, int BITS>
__device__ __forceinline__ U kth_bound(U v, int k) {
  U cur = 0;
  constexpr int kWidth = 8 * static_cast<int>(sizeof(U));
  for (int bit = kWidth - 1; bit >= kWidth - BITS; --bit) {
    const U next = cur | static_cast<U>(1) << bit;
    if (__builtin_popcountll(__builtin_amdgcn_ballot_w64(v >= next)) >= k) cur = next;
  }
  return cur;
}

// This wave's LDS writes are seen by its other lanes.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// A wave's candidates for the largest keys: every key above `tau`, a bound that k keys of the
// row reach.  The bound comes from the lanes' own maxima: k lanes hold k different logits.
struct Queue {
  uint64_t* q;  // [kQueue] in LDS
  int n = 0, k;
  uint64_t tau = 0;
  float tau_x = -INFINITY;  // logits below it are no candidates
  float best = -INFINITY;   // the lane's largest logit so far
  __device__ __forceinline__ Queue(uint64_t* lds, int k_) : q(lds), k(k_) {}
  __device__ __forceinline__ void raise(uint64_t to) {
    if (to > tau) {
      tau = to;
      tau_x = value_of(static_cast<uint32_t>(to >> 32));
    }
  }
  __device__ __forceinline__ void bound(uint32_t order) {  // logits of this order and above are candidates
    if (order) raise((static_cast<uint64_t>(order) << 32) - 1);
    if (order) tau_x = fmaxf(tau_x, value_of(order));
  }
  // Keeps the k largest.
  __device__ __forceinline__ void compact() {
    const int lane = threadIdx.x & 63;
    uint64_t mine[kQueue / 64];
    int above[kQueue / 64];
#pragma unroll
    for (int i = 0; i < kQueue / 64; ++i) {
      mine[i] = lane + 64 * i < n ? q[lane + 64 * i] : 0;
      above[i] = 0;
    }
    for (int j = 0; j < n; ++j) {
      const uint64_t o = q[j];
#pragma unroll
      for (int i = 0; i < kQueue / 64; ++i) above[i] += o > mine[i];
    }
    wave_sync();
#pragma unroll
    for (int i = 0; i < kQueue / 64; ++i)
      if (lane + 64 * i < n && above[i] < k) q[above[i]] = mine[i];
    n = min(n, k);
    wave_sync();
    if (n == k) raise(q[k - 1]);
  }
  __device__ __forceinline__ void push(uint64_t key) {  // 0: none
    const uint64_t mask = __builtin_amdgcn_ballot_w64(key > tau);
    if (mask == 0) return;
    if (key > tau) q[n + rank_in(mask)] = key;
    n += __builtin_popcountll(mask);
    if (n > kQueue - 64) {
      wave_sync();
      compact();
    }
  }
};

// The k largest of n keys in LDS, in order, by how many are above each; NT threads.
template <int NT, typename Out>
__device__ __forceinline__ void select(const uint64_t* list, int n, int k, const Out& out) {
  const int t = NT == 64 ? threadIdx.x & 63 : threadIdx.x;
  for (int i = t; i < n; i += NT) {
    const uint64_t mine = list[i];
    int above = 0;
    for (int j = 0; j < n; ++j) above += list[j] > mine;
    if (above < k) out(above, mine);
  }
}

template <typename T>
__device__ __forceinline__ float logit(const Params& p, int64_t row, uint32_t i) {
  return Elem<T>::load1(reinterpret_cast<const T*>(p.x + row * p.stride) + i);
}

// What a row's statistics give; one thread.
template <typename T>
__device__ __forceinline__ void finish(const Params& p, int64_t row, const Stats& a) {
  const float log_s = a.s == 0.f ? -INFINITY : __builtin_amdgcn_logf(a.s);
  const bool none = a.m == -INFINITY && a.s == a.s;
  const int id = p.ids[row];
  const bool there = id >= 0 && id < p.V;
  float lp = 0.f;
  if (there) lp = none ? -INFINITY : kLn2 * (__builtin_fmaf(logit<T>(p, row, id), p.c, -a.m) - log_s);
  p.logp[row] = lp;
  if (p.entropy) p.entropy[row] = none ? 0.f : kLn2 * (log_s - a.e / a.s);
  if (p.lse) p.lse[row] = none ? -INFINITY : kLn2 * (a.m + log_s);
}
template <typename T>
__device__ __forceinline__ void finish_top(const Params& p, int64_t row, const Stats& a, int rank, uint64_t key) {
  const uint32_t i = ~static_cast<uint32_t>(key);
  p.top_ids[row * p.top + rank] = static_cast<int32_t>(i);
  const bool none = a.m == -INFINITY && a.s == a.s;
  p.top_logps[row * p.top + rank] =
      none ? -INFINITY : kLn2 * (__builtin_fmaf(logit<T>(p, row, i), p.c, -a.m) - __builtin_amdgcn_logf(a.s));
}

// Rows that hold a NaN or +infinity (their sum is NaN, which the bounds above do not see): the
// largest keys one after the other, a pass over the row for each.  Every thread of NT calls it.
template <typename T, int NT>
__device__ __noinline__ void top_of_nan_row(const Params& p, int64_t row, const Stats& a, uint64_t* lds) {
  const int t = NT == 64 ? threadIdx.x & 63 : threadIdx.x;
  uint64_t last = ~0ull;
  for (int r = 0; r < p.top; ++r) {
    uint64_t best = 0;
    for (int i = t; i < p.V; i += NT) {
      const uint64_t key = key_of(logit<T>(p, row, i), i);
      if (key > best && (r == 0 || key < last)) best = key;
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const uint64_t o = __shfl_xor(best, d, 64);
      best = o > best ? o : best;
    }
    if constexpr (NT > 64) {
      __syncthreads();
      if ((t & 63) == 0) lds[t >> 6] = best;
      __syncthreads();
      for (int w = 0; w < NT / 64; ++w) best = lds[w] > best ? lds[w] : best;
    }
    last = best;
    if (t == 0) finish_top<T>(p, row, a, r, best);
  }
}

// A row, or a slice of one, by WAVES waves.  The lanes keep a running softmax each, joined at
// the end; the waves collect candidates for the largest logits above a bound that they share.
// Per logit: one conversion, half a maximum, a multiply-add, an exponential, two sums.
template <typename T, int WAVES, bool TOP>
__global__ __launch_bounds__(256) void stats_kernel(Params p) {
  constexpr int VEC = Elem<T>::kVec, NT = 64 * WAVES;
  __shared__ uint64_t queues[TOP ? 4 : 1][TOP ? kQueue : 1];
  __shared__ uint64_t list[TOP ? 4 * kQueue : 4];
  __shared__ float parts[3][4];
  __shared__ uint32_t shared_tau;
  __shared__ int listed;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, part = WAVES == 1 ? 0 : wave;
  const int64_t unit = WAVES == 1 ? static_cast<int64_t>(blockIdx.x) * 4 + wave : blockIdx.x;
  if (WAVES == 1 && unit >= p.N) return;
  const int64_t row = WAVES == 1 ? unit : unit / p.slices;
  const int slice = WAVES == 1 ? 0 : static_cast<int>(unit - row * p.slices);
  const char* base = p.x + row * p.stride;
  const T* X = reinterpret_cast<const T*>(base);
  // The row's elements before and after its 16-byte vectors.
  const int head = min(static_cast<int>((-reinterpret_cast<uintptr_t>(base) & 15) / sizeof(T)), p.V);
  const int nv = (p.V - head) / VEC, rest = p.V - nv * VEC;
  const int v0 = slice * p.per, v1 = WAVES == 1 ? nv : min(nv, v0 + p.per);
  const uint4* body = reinterpret_cast<const uint4*>(X + head);

  if constexpr (TOP && WAVES > 1) {
    if (threadIdx.x == 0) shared_tau = 0, listed = 0;
    __syncthreads();
  }
  Stats a;
  Queue q(queues[TOP ? wave : 0], p.top);
  uint4 next[kRun];
  auto fetch = [&](int v) {
#pragma unroll
    for (int j = 0; j < kRun; ++j) {
      const int at = v + NT * j + 64 * part + lane;
      if (at < v1) next[j] = body[at];
    }
  };
  fetch(v0);
  if (slice == 0 && part == 0) {  // the single elements, one a lane
    const int i = lane < head ? lane : p.V - rest + lane;
    const bool there = lane < rest;
    float x[1] = {there ? Elem<T>::load1(X + i) : -INFINITY};
    a.add(x, x[0], p.c);
    if constexpr (TOP) q.push(there ? key_of(x[0], i) : 0);
  }
  for (int v = v0; v < v1; v += NT * kRun) {
    float x[kRun][VEC], most[kRun];
#pragma unroll
    for (int j = 0; j < kRun; ++j) {
      const bool there = v + NT * j + 64 * part + lane < v1;
      load_vec(reinterpret_cast<const T*>(&next[j]), x[j]);
      most[j] = -INFINITY;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        x[j][i] = there ? x[j][i] : -INFINITY;
        most[j] = fmaxf(most[j], x[j][i]);
      }
    }
    fetch(v + NT * kRun);
    float all = most[0];
#pragma unroll
    for (int j = 1; j < kRun; ++j) all = fmaxf(all, most[j]);
    a.add(*reinterpret_cast<const float(*)[kRun * VEC]>(&x), all, p.c);
    if constexpr (TOP) {
      q.best = fmaxf(q.best, all);
      if constexpr (WAVES > 1) q.bound(*static_cast<volatile uint32_t*>(&shared_tau));
      if (__builtin_amdgcn_ballot_w64(all >= q.tau_x)) {
        const uint32_t order = kth_bound<uint32_t, 16>(q.best == -INFINITY ? 0u : order_of(q.best), p.top);
        q.bound(order);
        if constexpr (WAVES > 1)
          if (lane == 0 && order) atomicMax(&shared_tau, order);
#pragma unroll
        for (int j = 0; j < kRun; ++j) {
          const int at = v + NT * j + 64 * part + lane;
          if (__builtin_amdgcn_ballot_w64(most[j] >= q.tau_x && at < v1) == 0) continue;
#pragma unroll
          for (int i = 0; i < VEC; ++i)
            q.push(at < v1 && x[j][i] >= q.tau_x ? key_of(x[j][i], head + at * VEC + i) : 0);
        }
      }
    }
  }
  a = wave_join(a);
  if constexpr (WAVES == 1) {
    if (lane == 0) finish<T>(p, row, a);
    if constexpr (TOP) {
      if (a.s != a.s) {
        top_of_nan_row<T, 64>(p, row, a, nullptr);
      } else {
        wave_sync();
        select<64>(q.q, q.n, p.top, [&](int rank, uint64_t key) { finish_top<T>(p, row, a, rank, key); });
      }
    }
  } else {
    if (lane == 0) parts[0][wave] = a.m, parts[1][wave] = a.s, parts[2][wave] = a.e;
    __syncthreads();
    a = Stats();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      Stats o;
      o.m = parts[0][w];
      o.s = parts[1][w];
      o.e = parts[2][w];
      a.join(o);
    }
    const bool whole = p.slices == 1;
    if (threadIdx.x == 0) {
      if (whole) finish<T>(p, row, a);
      else p.stats[unit] = make_float4(a.m, a.s, a.e, 0.f);
    }
    if constexpr (TOP) {
      if (whole && a.s != a.s) {
        top_of_nan_row<T, NT>(p, row, a, list);
        return;
      }
      // The waves' candidates that all their bounds leave.
      const uint64_t tau = shared_tau ? (static_cast<uint64_t>(shared_tau) << 32) - 1 : 0;
      for (int i = lane; i < q.n; i += 64)
        if (q.q[i] > tau) list[atomicAdd(&listed, 1)] = q.q[i];
      __syncthreads();
      const int n = listed;
      if (whole) {
        select<NT>(list, n, p.top, [&](int rank, uint64_t key) { finish_top<T>(p, row, a, rank, key); });
      } else {
        uint64_t* out = p.keys + unit * p.top;
        select<NT>(list, n, p.top, [&](int rank, uint64_t key) { out[rank] = key; });
        for (int i = n + threadIdx.x; i < p.top; i += NT) out[i] = 0;
      }
    }
  }
}

// Joins a row's slices; a wave a row.
template <typename T>
__global__ __launch_bounds__(64) void join_kernel(Params p) {
  __shared__ uint64_t list[kMostSlices * kMostTop];
  const int lane = threadIdx.x;
  const int64_t row = blockIdx.x;
  Stats a;
  if (lane < p.slices) {
    const float4 s = p.stats[row * p.slices + lane];
    a.m = s.x;
    a.s = s.y;
    a.e = s.z;
  }
  const int n = p.slices * p.top;
  const uint64_t* keys = p.keys + row * n;
  uint64_t best = 0;
  for (int i = lane; i < n; i += 64) best = keys[i] > best ? keys[i] : best;
  a = wave_join(a);
  if (lane == 0) finish<T>(p, row, a);
  if (p.top == 0) return;
  if (a.s != a.s) {
    top_of_nan_row<T, 64>(p, row, a, nullptr);
    return;
  }
  const uint64_t bound = kth_bound<uint64_t, 64>(best, p.top);
  int count = 0;
  for (int i0 = 0; i0 < n; i0 += 64) {
    const uint64_t key = i0 + lane < n ? keys[i0 + lane] : 0;
    const bool in = key != 0 && key >= bound;
    const uint64_t mask = __builtin_amdgcn_ballot_w64(in);
    if (in) list[count + rank_in(mask)] = key;
    count += __builtin_popcountll(mask);
  }
  wave_sync();
  select<64>(list, count, p.top, [&](int rank, uint64_t key) { finish_top<T>(p, row, a, rank, key); });
}

// ---------------------------------------------------------------- gradient
struct Grad {
  const char* x;
  char* d;
  int64_t x_stride, d_stride;  // bytes
  const int32_t* ids;
  const float* lse;
  const float* entropy;
  const float* d_logp;
  const float* d_entropy;
  int64_t N;
  int V, runs;  // workgroups of a row
  float scale;
};

// d_v = p_v (A + B t_v) + [v = id] C with t = x - lse, p = e^t, A = -scale (g + h entropy),
// B = -scale h, C = scale g.  WAVES = 4: a workgroup takes a run of a row; 1: a wave a row.
template <typename T, int WAVES, bool WIDE>
__global__ __launch_bounds__(256) void grad_kernel(Grad p) {
  constexpr int VEC = Elem<T>::kVec, NT = 64 * WAVES;
  const int wave = threadIdx.x >> 6, t = WAVES == 1 ? threadIdx.x & 63 : threadIdx.x;
  const int64_t unit = WAVES == 1 ? static_cast<int64_t>(blockIdx.x) * 4 + wave : blockIdx.x;
  const int64_t row = WAVES == 1 ? unit : unit / p.runs;
  if (row >= p.N) return;
  const int run = WAVES == 1 ? 0 : static_cast<int>(unit - row * p.runs);
  const char* xb = p.x + row * p.x_stride;
  char* db = p.d + row * p.d_stride;
  const T* X = reinterpret_cast<const T*>(xb);
  T* D = reinterpret_cast<T*>(db);
  const float lse = p.lse[row];
  const int id = p.ids[row];
  const float g = p.d_logp && id >= 0 && id < p.V ? p.d_logp[row] : 0.f;
  const float h = p.d_entropy ? p.d_entropy[row] : 0.f;
  const float A = -p.scale * (p.d_entropy ? __builtin_fmaf(h, p.entropy[row], g) : g), B = -p.scale * h, C = p.scale * g;
  const bool none = lse == -INFINITY;
  auto value = [&](float x) {
    const float u = __builtin_fmaf(x, p.scale, -lse), w = __builtin_amdgcn_exp2f(u * kLog2e);
    return none ? 0.f : w * __builtin_fmaf(B, fmaxf(u, kFar), A);
  };
  if constexpr (!WIDE) {
    for (int i = run * NT * 8 + t, end = min(p.V, WAVES == 1 ? p.V : (run + 1) * NT * 8); i < end; i += NT) {
      const float d = value(Elem<T>::load1(X + i));
      Elem<T>::store1(D + i, i == id && !none ? d + C : d);
    }
  } else {
    const int head = min(static_cast<int>((-reinterpret_cast<uintptr_t>(xb) & 15) / sizeof(T)), p.V);
    const int nv = (p.V - head) / VEC, rest = p.V - nv * VEC;
    if (run == 0 && t < rest) {
      const int i = t < head ? t : p.V - rest + t;
      const float d = value(Elem<T>::load1(X + i));
      Elem<T>::store1(D + i, i == id && !none ? d + C : d);
    }
    const int at_id = id >= head && !none ? id - head : -1;
    for (int v0 = run * NT * kRun; v0 < nv; v0 += NT * kRun) {
      uint4 raw[kRun];
#pragma unroll
      for (int j = 0; j < kRun; ++j)
        if (v0 + NT * j + t < nv) raw[j] = reinterpret_cast<const uint4*>(X + head)[v0 + NT * j + t];
#pragma unroll
      for (int j = 0; j < kRun; ++j) {
        const int v = v0 + NT * j + t;
        if (v >= nv) break;
        float x[VEC];
        load_vec(reinterpret_cast<const T*>(&raw[j]), x);
#pragma unroll
        for (int i = 0; i < VEC; ++i) x[i] = value(x[i]);
        if (at_id >= 0 && at_id / VEC == v) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) x[i] += i == at_id % VEC ? C : 0.f;
        }
        store_vec(D + head + v * VEC, x);
      }
      if (WAVES > 1) break;
    }
  }
}

// Waves of a row: one where that wave takes it in one run or two, four beyond.
static bool short_rows(int64_t V, int64_t es) { return V * es <= 2 * 64 * 16 * kRun; }

// Workgroups that share a row: so many that about 1024 run, each with a full run at least.
static int64_t slices_of(int64_t N, int64_t V, int64_t es) {
  const int64_t run = 256 * 16 / es * kRun;
  return std::max<int64_t>(1, std::min<int64_t>({(V + run - 1) / run, 1024 / std::max<int64_t>(N, 1), kMostSlices}));
}

template <typename T>
static void launch(const Params& p, hipStream_t s) {
  if (short_rows(p.V, sizeof(T))) {
    const dim3 grid(static_cast<unsigned>((p.N + 3) / 4));
    if (p.top) hipLaunchKernelGGL((stats_kernel<T, 1, true>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((stats_kernel<T, 1, false>), grid, dim3(256), 0, s, p);
    return;
  }
  const dim3 grid(static_cast<unsigned>(p.N * p.slices));
  if (p.top) hipLaunchKernelGGL((stats_kernel<T, 4, true>), grid, dim3(256), 0, s, p);
  else hipLaunchKernelGGL((stats_kernel<T, 4, false>), grid, dim3(256), 0, s, p);
  if (p.slices > 1) hipLaunchKernelGGL((join_kernel<T>), dim3(static_cast<unsigned>(p.N)), dim3(64), 0, s, p);
}

template <typename T>
static int launch_grad(Grad& p, hipStream_t s, GHipError* err, const char* what) {
  const bool wide = (reinterpret_cast<uintptr_t>(p.x) - reinterpret_cast<uintptr_t>(p.d)) % 16 == 0 &&
                    (p.N <= 1 || (p.x_stride - p.d_stride) % 16 == 0);
  const bool one = short_rows(p.V, sizeof(T));
  const int64_t run = 256 * (wide ? static_cast<int64_t>(Elem<T>::kVec) * kRun : 8);
  p.runs = one ? 1 : static_cast<int>((p.V + run - 1) / run);
  const int64_t blocks = one ? (p.N + 3) / 4 : p.N * p.runs;
  if (blocks > kMostGroups) return set_error(err, GHIP_ERR_UNSUPPORTED, "%s: problem too large", what);
  const dim3 grid(static_cast<unsigned>(blocks));
  if (one && wide) hipLaunchKernelGGL((grad_kernel<T, 1, true>), grid, dim3(256), 0, s, p);
  else if (one) hipLaunchKernelGGL((grad_kernel<T, 1, false>), grid, dim3(256), 0, s, p);
  else if (wide) hipLaunchKernelGGL((grad_kernel<T, 4, true>), grid, dim3(256), 0, s, p);
  else hipLaunchKernelGGL((grad_kernel<T, 4, false>), grid, dim3(256), 0, s, p);
  GHIP_CHECK(hipGetLastError(), err);
  return GHIP_OK;
}

// What both entry points ask of the logits.
static int check(int dtype, const void* logits, int64_t row_stride, int64_t N, int64_t V, float scale, GHipError* err,
                 const char* what) {
  if (dtype != GHIP_DTYPE_FLOAT32 && dtype != GHIP_DTYPE_BFLOAT16 && dtype != GHIP_DTYPE_FLOAT16)
    return set_error(err, GHIP_ERR_UNSUPPORTED, "%s: needs float32, bfloat16 or float16", what);
  if (N < 0 || V <= 0) return set_error(err, GHIP_ERR_INVALID_ARG, "%s: bad sizes", what);
  if (!(scale > 0.f) || !(scale < 1e30f))
    return set_error(err, GHIP_ERR_INVALID_ARG, "%s: the scale must be positive and finite", what);
  if (N >= int64_t{1} << 24 || V > int64_t{1} << 30)
    return set_error(err, GHIP_ERR_UNSUPPORTED, "%s: fewer than 2^24 rows of at most 2^30 logits", what);
  if (N > 1 && (row_stride < 0 || row_stride >= int64_t{1} << 40))
    return set_error(err, GHIP_ERR_UNSUPPORTED, "%s: the row stride must not be negative and be below 2^40", what);
  if (N > 0 && reinterpret_cast<uintptr_t>(logits) % (dtype == GHIP_DTYPE_FLOAT32 ? 4 : 2))
    return set_error(err, GHIP_ERR_INVALID_ARG, "%s: pointers are not aligned to elements", what);
  return GHIP_OK;
}

}  // namespace logprobs
}  // namespace ghip

using namespace ghip;

extern "C" int64_t ghip_token_logprobs_workspace_bytes(int dtype, int64_t N, int64_t V, int64_t top) {
  const int64_t es = dtype == GHIP_DTYPE_FLOAT32 ? 4 : 2;
  if (N <= 0 || V <= 0 || top < 0 || top > logprobs::kMostTop || V > int64_t{1} << 30 || logprobs::short_rows(V, es)) return 0;
  const int64_t slices = logprobs::slices_of(N, V, es);
  return slices > 1 ? N * slices * (16 + 8 * top) : 0;
}

extern "C" int ghip_token_logprobs(int dtype, const void* logits, int64_t row_stride, const int32_t* ids, int64_t N,
                                   int64_t V, int64_t top, float scale, float* logp, float* entropy, float* lse,
                                   float* top_logps, int32_t* top_ids, void* workspace, int64_t workspace_bytes,
                                   void* stream, GHipError* err) {
  static const char kWhat[] = "token_logprobs";
  if (int rc = logprobs::check(dtype, logits, row_stride, N, V, scale, err, kWhat)) return rc;
  if (top < 0 || top > logprobs::kMostTop || top > V)
    return set_error(err, GHIP_ERR_INVALID_ARG, "%s: top %lld must be 0 to %d and at most the %lld logits of a row", kWhat,
                     static_cast<long long>(top), logprobs::kMostTop, static_cast<long long>(V));
  if (N == 0) return GHIP_OK;
  if (!logits || !ids || !logp || (top > 0 && (!top_logps || !top_ids)))
    return set_error(err, GHIP_ERR_INVALID_ARG, "%s: null pointer", kWhat);
  const int64_t es = dtype == GHIP_DTYPE_FLOAT32 ? 4 : 2;
  logprobs::Params p{};
  p.x = static_cast<const char*>(logits);
  p.stride = N > 1 ? row_stride * es : 0;
  p.ids = ids;
  p.N = N;
  p.V = static_cast<int>(V);
  p.top = static_cast<int>(top);
  p.c = scale * logprobs::kLog2e;
  p.logp = logp; p.entropy = entropy; p.lse = lse; p.top_logps = top_logps; p.top_ids = top_ids;
  p.slices = 1;
  const int64_t need = workspace ? ghip_token_logprobs_workspace_bytes(dtype, N, V, top) : 0;
  if (need > 0) {
    if (workspace_bytes < need)
      return set_error(err, GHIP_ERR_INVALID_ARG, "%s: workspace of %lld bytes, %lld needed", kWhat,
                       static_cast<long long>(workspace_bytes), static_cast<long long>(need));
    if (reinterpret_cast<uintptr_t>(workspace) & 15)
      return set_error(err, GHIP_ERR_INVALID_ARG, "%s: workspace must be 16-byte aligned", kWhat);
    p.slices = static_cast<int>(logprobs::slices_of(N, V, es));
    p.stats = static_cast<float4*>(workspace);
    p.keys = reinterpret_cast<uint64_t*>(p.stats + N * p.slices);
  }
  p.per = static_cast<int>((V / (16 / es) + p.slices - 1) / p.slices);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == GHIP_DTYPE_FLOAT32) logprobs::launch<float>(p, s);
  else if (dtype == GHIP_DTYPE_FLOAT16) logprobs::launch<f16_t>(p, s);
  else logprobs::launch<bf16_t>(p, s);
  GHIP_CHECK(hipGetLastError(), err);
  return GHIP_OK;
}

extern "C" int ghip_token_logprobs_grad(int dtype, const void* logits, int64_t row_stride, const int32_t* ids,
                                        const float* lse, const float* entropy, const float* d_logp,
                                        const float* d_entropy, int64_t N, int64_t V, float scale, void* d_logits,
                                        int64_t d_row_stride, void* stream, GHipError* err) {
  static const char kWhat[] = "token_logprobs_grad";
  if (int rc = logprobs::check(dtype, logits, row_stride, N, V, scale, err, kWhat)) return rc;
  if (int rc = logprobs::check(dtype, d_logits, d_row_stride, N, V, scale, err, kWhat)) return rc;
  if (N == 0) return GHIP_OK;
  if (!logits || !d_logits || !ids || !lse || (!d_logp && !d_entropy) || (d_entropy && !entropy))
    return set_error(err, GHIP_ERR_INVALID_ARG, "%s: null pointer", kWhat);
  const int64_t es = dtype == GHIP_DTYPE_FLOAT32 ? 4 : 2;
  if (N > 1 && d_row_stride < V)
    return set_error(err, GHIP_ERR_INVALID_ARG, "%s: rows of d_logits overlap", kWhat);
  logprobs::Grad p{};
  p.x = static_cast<const char*>(logits);
  p.d = static_cast<char*>(d_logits);
  p.x_stride = N > 1 ? row_stride * es : 0;
  p.d_stride = N > 1 ? d_row_stride * es : 0;
  p.ids = ids; p.lse = lse; p.entropy = entropy; p.d_logp = d_logp; p.d_entropy = d_entropy;
  p.N = N;
  p.V = static_cast<int>(V);
  p.scale = scale;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == GHIP_DTYPE_FLOAT32) return logprobs::launch_grad<float>(p, s, err, kWhat);
  if (dtype == GHIP_DTYPE_FLOAT16) return logprobs::launch_grad<f16_t>(p, s, err, kWhat);
  return logprobs::launch_grad<bf16_t>(p, s, err, kWhat);
}
