// Log probabilities of given tokens, entropy, log-sum-exp and the largest logits of rows, in one
// pass over them, and the gradient of the logits.
//
//   lse = log sum_v exp x_v,  logp = x_id - lse,  entropy = lse - sum_v p_v x_v,  x = scale * logits
//
// No reference op (GoMLX composes it of FusedSoftmax and primitives); beside the log-softmax
// rows, which write V values a row.  Bound by the bytes of the logits, read once.
#include <algorithm>
#include <type_traits>

#include "common.h"

// Products are fused with sums where it says so, nowhere else: the lanes that join their sums in
// pairs then hold the same bits, and a token's log probability is the same in every output.
#pragma clang fp contract(off)

namespace ghip {
namespace logprobs {

constexpr int kMostTop = 32;
constexpr int kMostSlices = 64;
constexpr int kRun = 4;      // vectors a lane takes at a time
constexpr int kSlots = 16;   // runs of a lane whose maxima are kept apart
constexpr int kQueue = 256;  // candidates a wave holds
constexpr int kAhead = 4;    // vectors under way where a long row is read once more
constexpr float kLn2 = 0.6931471805599453f, kLog2e = 1.4426950408889634f;
constexpr float kFar = -200.f;  // 2^kFar is 0: what stands for log 0 in a product with a weight of 0
constexpr int64_t kMostGroups = (int64_t{1} << 24) - 1;
constexpr int kCus = 256, kStay = 5;  // of an MI355X; workgroups of stream_kernel on each
constexpr int kMostTurns = ((1 << 24) / (kCus * kStay) + 32) / 32 * 32;  // parts that one of them takes, at most

struct Params {
  const char* x;
  int64_t stride;  // bytes
  const int32_t* ids;
  int64_t N;
  int V, top, slices, per;  // per: vectors of a slice
  float c, scale;           // c: scale * log2 e
  float* logp;
  float* entropy;
  float* lse;
  float* top_logps;
  int32_t* top_ids;
  float4* stats;   // [N][slices]: maximum, sum, sum of weight times exponent
  uint64_t* keys;  // [N][slices][top]
};

// A running softmax in powers of two: m = max of x c, s = sum of w, e = sum of w u, where
// u = x c - m and w = 2^u.  m begins at -kLarge, below which weights are 0: the rounding of a
// larger maximum's product with c would reach the weights.  A row that has nothing above, or a
// maximum beyond kLarge, is summed by exact_sums.
constexpr float kLarge = 1048576.f;
struct Stats {
  float m = -kLarge, s = 0.f, e = 0.f;
  // The same sums beside another maximum.
  __device__ __forceinline__ void move(float to) {
    const float d = m - to, f = __builtin_amdgcn_exp2f(d);
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
};
// The lanes' sums beside their wave's one maximum.
__device__ __forceinline__ Stats wave_join(Stats a) {
  a.s = wave_sum(a.s);
  a.e = wave_sum(a.e);
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

// The largest number of BITS leading bits (the others 0) that at least k of the lanes' M values reach.
template <typename U, int BITS, int M>
__device__ __forceinline__ U kth_bound(const U (&v)[M], int k) {
  U cur = 0;
  constexpr int kWidth = 8 * static_cast<int>(sizeof(U));
#pragma unroll
  for (int bit = kWidth - 1; bit >= kWidth - BITS; --bit) {
    const U next = cur | static_cast<U>(1) << bit;
    int n = 0;
#pragma unroll
    for (int i = 0; i < M; ++i) n += __builtin_popcountll(__builtin_amdgcn_ballot_w64(v[i] >= next));
    if (n >= k) cur = next;
  }
  return cur;
}

// This wave's LDS writes are seen by its other lanes.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// The largest keys of rows where many logits are equal (constant rows, masks of the lowest value
// or -infinity, fewer tokens than `top`): a wave's second pass over its part, in the order of
// the indices.  Every key above `tau`, a bound that k keys of the row reach, is a candidate;
// the bound comes from the lanes' own maxima (k lanes hold k different logits) and, when
// candidates are many, from the k-th of them.
struct Queue {
  uint64_t* q;  // [kQueue] in LDS
  int n = 0, k;
  uint64_t tau = 0;
  float tau_x = -INFINITY;  // logits below it are no candidates
  float best = -INFINITY;   // the lane's largest logit so far
  __device__ __forceinline__ Queue(uint64_t* lds, int k_) : q(lds), k(k_) {}
  // Logits of this order and above are candidates (0: all); whether that is news.
  __device__ __forceinline__ bool bound(uint32_t order) {
    const uint64_t to = (static_cast<uint64_t>(order) << 32) - 1;
    if (order == 0 || to <= tau) return false;
    tau = to;
    tau_x = value_of(order);
    return true;
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
    if (n == k && q[k - 1] > tau) {
      tau = q[k - 1];
      tau_x = value_of(static_cast<uint32_t>(tau >> 32));
    }
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
  for (int i0 = 0; i0 < n; i0 += NT) {
    const uint64_t mine = i0 + t < n ? list[i0 + t] : ~0ull;
    int above = 0, j = 0;
    for (; j + 8 <= n; j += 8) {
#pragma unroll
      for (int u = 0; u < 8; ++u) above += list[j + u] > mine;
    }
    for (; j < n; ++j) above += list[j] > mine;
    if (i0 + t < n && above < k) out(above, mine);
  }
}

template <typename T>
__device__ __forceinline__ float logit(const Params& p, int64_t row, uint32_t i) {
  return Elem<T>::load1(reinterpret_cast<const T*>(p.x + row * p.stride) + i);
}

// The row's token and its logit; one thread, ahead of the row's pass.
struct Given {
  bool there = false;
  float x = 0.f;
  template <typename T>
  __device__ __forceinline__ void load(const Params& p, int64_t row) {
    const int id = p.ids[row];
    there = id >= 0 && id < p.V;
    if (there) x = logit<T>(p, row, id);
  }
};

// A row's sums: u = (x - x0) c - m.
struct Sums : Stats {
  float x0 = 0.f;
  bool none = false;  // nothing but -infinity
  Sums() = default;
  __device__ __forceinline__ explicit Sums(const Stats& a) : Stats(a) {}
  __device__ __forceinline__ float exponent(float x, float c) const { return __builtin_fmaf(x - x0, c, -m); }
  __device__ __forceinline__ bool usual() const { return fabsf(m) < kLarge && s > 0.f && s < INFINITY; }
};
// A row's logits to f(x, first index, there), thread t of NT: one by one, or (AHEAD > 0) AHEAD vectors at a
// time and the logits around the row's vectors one by one.  The lanes of a wave are in every call
// together; -infinity where a lane has none.
template <typename T, int NT, int AHEAD, typename F>
__device__ __forceinline__ void each_logit(const Params& p, int64_t row, int t, const F& f) {
  const char* base = p.x + row * p.stride;
  const T* x = reinterpret_cast<const T*>(base);
  auto one = [&](int i, bool there) {
    float v[1] = {-INFINITY};
    if (there) v[0] = Elem<T>::load1(x + i);
    f(v, i, there);
  };
  if constexpr (AHEAD == 0) {
    for (int i = t; i - t < p.V; i += NT) one(i, i < p.V);
  } else {
    constexpr int VEC = Elem<T>::kVec;
    const int head = min(static_cast<int>((-reinterpret_cast<uintptr_t>(base) & 15) / sizeof(T)), p.V);
    const int nv = (p.V - head) / VEC, rest = p.V - nv * VEC;
    one(t < head ? t : p.V - rest + t, t < rest);
    const uint4* body = reinterpret_cast<const uint4*>(x + head);
#pragma unroll 1
    for (int v0 = 0; v0 < nv; v0 += NT * AHEAD) {
      uint4 raw[AHEAD];
#pragma unroll
      for (int j = 0; j < AHEAD; ++j)
        if (v0 + NT * j + t < nv) raw[j] = body[v0 + NT * j + t];
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        const int v = v0 + NT * j + t;
        float many[VEC];
        __builtin_amdgcn_sched_barrier(0);  // (one vector widened at a time)
        load_vec(reinterpret_cast<const T*>(&raw[j]), many);
#pragma unroll
        for (int e = 0; e < VEC; ++e) many[e] = v < nv ? many[e] : -INFINITY;
        f(many, head + v * VEC, v < nv);
      }
    }
  }
}
// The largest, the sum (wave after wave) of NT threads' values; `lds` of the workgroup's waves.
template <int NT>
__device__ __forceinline__ float group_max(float x, float* lds) {
  x = wave_max(x);
  if constexpr (NT > 64) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
    __syncthreads();
    for (int w = 0; w < NT / 64; ++w) x = fmaxf(x, lds[w]);
  }
  return x;
}
template <int NT>
__device__ __forceinline__ float group_sum(float x, float* lds) {
  x = wave_sum(x);
  if constexpr (NT > 64) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
    __syncthreads();
    x = 0.f;
    for (int w = 0; w < NT / 64; ++w) x += lds[w];
  }
  return x;
}
// Rows of one mask, -infinity, 1e10 or a type's lowest number, and rows with a NaN or infinity: the
// largest logit itself, then u = (x - x0) c.  Every thread of NT calls it, and gets the same.
// (Padding is such a row.  16 rows of 131072 bf16 logits, one of them nothing but -infinity: 24 us as without it;
// 439 by one wave that reads its logits one by one.  One with a NaN, and a top of 20: 84 us for 22.)
template <typename T, int NT, int AHEAD>
__device__ __forceinline__ Sums exact_sums(const Params& p, int64_t row, int t, float* lds) {
  Sums a;
  float most = -INFINITY;
  bool nan = false;
  each_logit<T, NT, AHEAD>(p, row, t, [&](const auto& x, int, bool) {
#pragma unroll
    for (const float v : x) {
      most = fmaxf(most, v);
      nan |= v != v;
    }
  });
  a.m = 0.f;
  a.x0 = group_max<NT>(nan ? INFINITY : most, lds);
  if (a.x0 == -INFINITY) {
    a.x0 = 0.f;
    a.none = true;
    return a;
  }
  if (a.x0 == INFINITY) {
    a.s = a.e = NAN;
    return a;
  }
  each_logit<T, NT, AHEAD>(p, row, t, [&](const auto& x, int, bool) {
#pragma unroll
    for (const float v : x) {
      const float u = a.exponent(v, p.c), w = __builtin_amdgcn_exp2f(u);
      a.s += w;
      a.e = __builtin_fmaf(w, fmaxf(u, kFar), a.e);
    }
  });
  a.s = group_sum<NT>(a.s, lds);
  a.e = group_sum<NT>(a.e, lds);
  return a;
}
template <typename T, int NT, int AHEAD>
__device__ __forceinline__ Sums sums_of(const Params& p, int64_t row, const Stats& a, int t, float* lds) {
  const Sums r(a);
  return r.usual() ? r : exact_sums<T, NT, AHEAD>(p, row, t, lds);
}

// What a row's sums give; one thread.
__device__ __forceinline__ void finish(const Params& p, int64_t row, const Sums& a, const Given& id) {
  const float log_s = __builtin_amdgcn_logf(a.s);
  float lp = 0.f;
  if (id.there) lp = a.none ? -INFINITY : kLn2 * (a.exponent(id.x, p.c) - log_s);
  p.logp[row] = lp;
  if (p.entropy) p.entropy[row] = a.none ? 0.f : kLn2 * (log_s - a.e / a.s);
  if (p.lse) p.lse[row] = a.none ? -INFINITY : __builtin_fmaf(a.x0, p.scale, kLn2 * (a.m + log_s));
}
__device__ __forceinline__ void finish_top(const Params& p, int64_t row, const Sums& a, int rank, uint64_t key) {
  p.top_ids[row * p.top + rank] = static_cast<int32_t>(~static_cast<uint32_t>(key));
  const float x = value_of(static_cast<uint32_t>(key >> 32));
  p.top_logps[row * p.top + rank] = a.none ? -INFINITY : kLn2 * (a.exponent(x, p.c) - __builtin_amdgcn_logf(a.s));
}

// The largest logits of a row by comparisons of orders, in one pass: rows that hold a NaN or +infinity,
// which the bounds by floating-point maxima do not see (their sum is NaN), and others of no usual sum.
// Every thread of NT calls it; `queues`: [NT / 64][kQueue], `list`: [NT / 64][kMostTop] (one wave: none).
template <typename T, int NT, int AHEAD>
__device__ __forceinline__ void top_by_order(const Params& p, int64_t row, const Sums& a, int t, uint64_t* queues,
                                             uint64_t* list) {
  const int lane = t & 63, wave = t >> 6;
  Queue q(queues + wave * kQueue, p.top);
  uint32_t best = 0;
  each_logit<T, NT, AHEAD>(p, row, t, [&](const auto& x, int i, bool there) {
    constexpr int kN = sizeof(x) / sizeof(float);
    uint32_t order[kN], most = 0;
#pragma unroll
    for (int e = 0; e < kN; ++e) {
      order[e] = there ? order_of(x[e]) : 0u;
      most = max(most, order[e]);
    }
    best = max(best, most);
    // (No key of these is above that of their largest at the first's place.)
    const uint64_t top = static_cast<uint64_t>(most) << 32 | static_cast<uint32_t>(~i);
    if (__builtin_amdgcn_ballot_w64(there && top > q.tau) == 0) return;
    const uint32_t bests[1] = {best};
    q.bound(kth_bound<uint32_t, 16>(bests, p.top));
    uint32_t marks = 0;
#pragma unroll
    for (int e = 0; e < kN; ++e) marks |= there && order[e] >= static_cast<uint32_t>(q.tau >> 32) ? 1u << e : 0u;
    while (__builtin_amdgcn_ballot_w64(marks != 0)) {  // (looked up once more: one place that pushes, not kN)
      const int at = i + __builtin_ctz(marks | 1u << 31);
      q.push(marks ? key_of(logit<T>(p, row, at), at) : 0);
      marks &= marks - 1;
    }
  });
  wave_sync();
  q.compact();
  if constexpr (NT == 64) {
    if (lane < q.n) finish_top(p, row, a, lane, q.q[lane]);
    wave_sync();
  } else {
    if (lane < kMostTop) list[wave * kMostTop + lane] = lane < q.n ? q.q[lane] : 0;
    __syncthreads();
    select<NT>(list, NT / 64 * kMostTop, p.top, [&](int rank, uint64_t key) { finish_top(p, row, a, rank, key); });
  }
}

// The largest of three, without the two instructions that quiet a signalling NaN in each (rows
// with a NaN are found by their sums).
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// The order of a lane's largest logit, 0 if there is none above -infinity: the lanes' k-th bounds the
// row's, since k lanes hold k different logits.
__device__ __forceinline__ uint32_t order_of_best(float best) { return best == -INFINITY ? 0u : order_of(best); }
__device__ __forceinline__ uint32_t bound_of(float best, int k) {
  const uint32_t v[1] = {order_of_best(best)};
  return kth_bound<uint32_t, 16>(v, k);
}
// The same of four waves' lanes, from the upper halves of their orders; in the order's upper half.
__device__ __forceinline__ uint32_t bound_of(const uint16_t (&bests)[256], int lane, int k) {
  const uint2 v = reinterpret_cast<const uint2*>(bests)[lane];
  const uint32_t four[4] = {v.x << 16, v.x & 0xffff0000u, v.y << 16, v.y & 0xffff0000u};
  return kth_bound<uint32_t, 16>(four, k);
}

// A wave's candidates by Queue: vectors [v0, v1) of the row, one a lane at a time.
template <typename T>
__device__ __forceinline__ void scan(Queue& q, const T* body, int head, int first, int step, int v0, int v1) {
  constexpr int VEC = Elem<T>::kVec;
  const int lane = threadIdx.x & 63;
  for (int v = v0 + first; v < v1; v += step) {
    const int at = v + lane;
    float x[VEC], most = -INFINITY;
    if (at < v1) load_vec(body + static_cast<int64_t>(at) * VEC, x);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      if (at >= v1) x[i] = -INFINITY;
      most = fmaxf(most, x[i]);
    }
    q.best = fmaxf(q.best, most);
    if (__builtin_amdgcn_ballot_w64(most >= q.tau_x && at < v1) == 0) continue;
    q.bound(bound_of(q.best, q.k));
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const bool in = at < v1 && x[i] >= q.tau_x;
      if (__builtin_amdgcn_ballot_w64(in)) q.push(in ? key_of(x[i], head + at * VEC + i) : 0);
    }
  }
}

// Where a row, or a slice of one, lies.
template <typename T>
struct Part {
  static constexpr int VEC = Elem<T>::kVec;
  int64_t row;
  int slice, head, rest, v0, v1;  // rest: elements before (head) and after the row's 16-byte vectors
  const T* x;
  const uint4* body;
  __device__ __forceinline__ Part(const Params& p, int64_t unit) {
    row = p.slices == 1 ? unit : unit / p.slices;
    slice = static_cast<int>(unit - row * p.slices);
    const char* base = p.x + row * p.stride;
    x = reinterpret_cast<const T*>(base);
    head = min(static_cast<int>((-reinterpret_cast<uintptr_t>(base) & 15) / sizeof(T)), p.V);
    const int nv = (p.V - head) / VEC;
    rest = p.V - nv * VEC;
    v0 = min(slice * p.per, nv);
    v1 = min(nv, v0 + p.per);
    body = reinterpret_cast<const uint4*>(x + head);
    if (slice != 0) rest = 0;  // (the first slice's)
  }
  __device__ __forceinline__ int single(const Params& p, int lane) const { return lane < head ? lane : p.V - rest + lane; }
};

// Thread t's vector of those from `v` on: the address of the workgroup's in scalar registers, the
// lane's in one.
__device__ __forceinline__ uint4 vector_at(const uint4* body, int v, int t) {
  return *reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(body + v) + 16u * static_cast<uint32_t>(t));
}

// A run of R vectors a lane, NT lanes: from vector v on, thread t's.
template <int NT, int R>
__device__ __forceinline__ void fetch(uint4 (&next)[R], const uint4* body, int v, int t, int v1) {
  if (v + NT * R <= v1) {
#pragma unroll
    for (int j = 0; j < R; ++j) next[j] = vector_at(body, v + NT * j, t);
  } else {
#pragma unroll
    for (int j = 0; j < R; ++j)
      if (v + NT * j + t < v1) next[j] = vector_at(body, v + NT * j, t);
  }
}
template <int N>
__device__ __forceinline__ float most_of(const float (&x)[N]) {
  float m = x[0];
#pragma unroll
  for (int i = 1; i + 1 < N; i += 2) m = max3(m, x[i], x[i + 1]);
  return N % 2 == 0 ? max3(m, x[N - 1], x[N - 1]) : m;
}
// Vector j of a run, widened; -infinity where there is none.
template <typename T, int NT, int R>
struct Run {
  static constexpr bool kFromMemory = false;
  static constexpr int kVectors = R;
  const uint4 (&raw)[R];
  int v, t, v1;
  __device__ __forceinline__ bool there(int j) const { return v + NT * j + t < v1; }
  // FRESH: widened once more; left alone, the compiler keeps a whole run's values for a second use.
  template <bool FRESH = false>
  __device__ __forceinline__ void get(int j, float (&x)[Elem<T>::kVec]) const {
    uint4 r = raw[j];
    if constexpr (FRESH) asm volatile("" : "+v"(r.x), "+v"(r.y), "+v"(r.z), "+v"(r.w));
    load_vec(reinterpret_cast<const T*>(&r), x);
    if (v + NT * R > v1) {
#pragma unroll
      for (int i = 0; i < Elem<T>::kVec; ++i) x[i] = there(j) ? x[i] : -INFINITY;
    }
  }
};
// The same of a run that streams: as soon as a vector is widened, that of the next run loads into its
// registers (past its end: the last one once more).  A second look reads memory again (it is
// rare, and a run's copy costs 16 registers).  FULL: every lane has all of its vectors.
template <typename T, int NT, bool FULL>
struct Streamed {
  static constexpr bool kFromMemory = true;
  static constexpr int kVectors = kRun;
  uint4 (&raw)[kRun];
  const uint4* body;
  int v, t, v1;
  const uint4* then;  // the next run's
  int nv, nv1;
  template <bool AGAIN = false>
  __device__ __forceinline__ void get(int j, float (&x)[Elem<T>::kVec]) const {
    const bool there = FULL || v + NT * j + t < v1;
    if constexpr (AGAIN) {
      uint4 r{};
      if (there) r = vector_at(body, 0, v + NT * j + t);
      load_vec(reinterpret_cast<const T*>(&r), x);
    } else {
      // (Kept apart, or the compiler widens all vectors ahead of the branch between the two forms.)
      if constexpr (FULL) asm volatile("; whole run" : "+v"(raw[j].x), "+v"(raw[j].y), "+v"(raw[j].z), "+v"(raw[j].w));
      else asm volatile("; last run" : "+v"(raw[j].x), "+v"(raw[j].y), "+v"(raw[j].z), "+v"(raw[j].w));
      load_vec(reinterpret_cast<const T*>(&raw[j]), x);
      raw[j] = vector_at(then, 0, min(nv + NT * j + t, nv1 - 1));
    }
    if constexpr (!FULL) {
#pragma unroll
      for (int i = 0; i < Elem<T>::kVec; ++i) x[i] = there ? x[i] : -INFINITY;
    }
  }
};
struct Single {
  static constexpr bool kFromMemory = false;
  static constexpr int kVectors = 1;
  float value;
  template <bool FRESH = false>
  __device__ __forceinline__ void get(int, float (&x)[1]) const { x[0] = value; }
};

// What stands before is computed before what follows.
__device__ __forceinline__ void here(float (&x)[2], float (&y)[2]) {
  asm volatile("" : "+v"(x[0]), "+v"(x[1]), "+v"(y[0]), "+v"(y[1]));
  __builtin_amdgcn_sched_barrier(0);
}

// The first run's maximum, ahead of its sums, which would be taken twice without it.
template <typename T, int NT, int R>
__device__ __forceinline__ void look(Stats& a, const uint4 (&raw)[R], int v, int t, int v1, float c) {
  float most = -INFINITY;
#pragma unroll
  for (int j = 0; j < R; ++j) {
    float x[Elem<T>::kVec];
    load_vec(reinterpret_cast<const T*>(&raw[j]), x);
    const float m = most_of(x);
    most = v + NT * j + t < v1 ? fmaxf(most, m) : most;
  }
  a.move(fmaxf(a.m, wave_max(most) * c));
}

// A run's sums into the lane's; a.m is the wave's maximum, and moves only where a run's weights say
// that it has grown (kGrown).  Per logit: a conversion, a multiply-add, an exponential (four issue
// slots), two sums.  Returns the lane's largest of the run, with MOST at half an instruction a
// logit.
template <int M, bool MOST, typename Values>
__device__ __forceinline__ float add_run(Stats& a, const Values& values, float c) {
  constexpr float kGrown = 256.f;
  constexpr int kVectors = Values::kVectors;
  float most = -INFINITY, s[2] = {0.f, 0.f}, e[2] = {0.f, 0.f}, shift = -a.m;
  auto weigh = [&](auto again, int j) {
    float x[M];
    values.template get<decltype(again)::value>(j, x);
    if constexpr (MOST && !decltype(again)::value) {
      if constexpr (M == 1) most = fmaxf(most, x[0]);
      else most = max3(most, most_of(x), most);
    }
#pragma unroll
    for (int i = 0; i < M; ++i) {
      const float u = __builtin_fmaf(x[i], c, shift), w = __builtin_amdgcn_exp2f(u);
      s[i & 1] += w;
      e[i & 1] = __builtin_fmaf(w, decltype(again)::value ? fmaxf(u, kFar) : u, e[i & 1]);
    }
  };
#pragma unroll
  for (int j = 0; j < kVectors; ++j) {
    weigh(std::integral_constant<bool, false>{}, j);
    here(s, e);  // (all vectors at once take 32 registers more)
  }
  // A maximum that has grown, NaN, infinities: once more beside the run's own maximum, and with
  // 0 for 0 times -infinity.
  if (__builtin_amdgcn_ballot_w64(!(s[0] + s[1] < kGrown) || e[0] + e[1] != e[0] + e[1])) {
    auto each = [&](auto f) {
      if constexpr (Values::kFromMemory) {
#pragma unroll 1
        for (int j = 0; j < kVectors; ++j) f(j);
      } else {
#pragma unroll
        for (int j = 0; j < kVectors; ++j) {
          f(j);
          here(s, e);
        }
      }
    };
    if constexpr (!MOST) {
      each([&](int j) {
        float x[M];
        values.template get<true>(j, x);
#pragma unroll
        for (int i = 0; i < M; ++i) most = fmaxf(most, x[i]);
      });
    }
    a.move(fmaxf(a.m, wave_max(most) * c));
    shift = -a.m;
    s[0] = s[1] = e[0] = e[1] = 0.f;
    each([&](int j) { weigh(std::integral_constant<bool, true>{}, j); });
  }
  const float ss = s[0] + s[1], es = e[0] + e[1];
  a.s += ss;
  a.e += es;
  return most;
}
// Joins the four waves' statistics.
__device__ __forceinline__ Stats waves_join(const float (&parts)[3][4]) {
  Stats a;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    Stats o;
    o.m = parts[0][w];
    o.s = parts[1][w];
    o.e = parts[2][w];
    a.join(o);
  }
  return a;
}
// Rows (WAVES = 1: a wave a row) and slices (4) of one run of R vectors a lane: the logits stay in
// registers, so candidates are taken from there.  A run in which a lane has no vector is weighed twice (0
// times -infinity), and a wave ends with its row: 65536 rows of 2000 bf16 logits 80 us where their bytes take 47.
// Bound by the chain of its steps: 16 rows of 131072 bf16 logits in 16 slices each 6.6 us, and 4.3
// for their join.
template <typename T, int WAVES, int R, bool TOP>
__global__ __launch_bounds__(256) void run_kernel(Params p) {
  constexpr int VEC = Elem<T>::kVec, NT = 64 * WAVES;
  constexpr int kKeys = WAVES * kQueue;
  __shared__ uint64_t lists[TOP ? 4 * kQueue : 1];
  __shared__ uint64_t queues[TOP ? 4 * kQueue : 1];
  __shared__ __attribute__((aligned(16))) uint16_t bests[256];
  __shared__ float parts[3][4];
  __shared__ int counts[4];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, own = WAVES == 1 ? wave : 0;
  const int t = WAVES == 1 ? lane : threadIdx.x;  // among the part's threads
  const int64_t unit = WAVES == 1 ? static_cast<int64_t>(blockIdx.x) * 4 + wave : blockIdx.x;
  if (WAVES == 1 && unit >= p.N) return;
  auto sync = [] {
    if constexpr (WAVES == 1) wave_sync();
    else __syncthreads();
  };
  const Part<T> at(p, unit);
  const bool whole = p.slices == 1;
  uint4 raw[R];
  fetch<NT>(raw, at.body, at.v0, t, at.v1);
  Given given;
  if (t == 0 && whole) given.load<T>(p, at.row);
  Stats a;
  float single = -INFINITY, best;
  const bool alone = t < at.rest;
  if (at.rest > 0 && (WAVES == 1 || wave == 0)) {
    if (alone) single = Elem<T>::load1(at.x + at.single(p, t));
    add_run<1, true>(a, Single{single}, p.c);
  }
  const Run<T, NT, R> values{raw, at.v0, t, at.v1};
  look<T, NT>(a, raw, at.v0, t, at.v1, p.c);
  best = fmaxf(add_run<VEC, TOP>(a, values, p.c), single);
  a = wave_join(a);
  uint32_t tau = 0;  // logits of this order and above are candidates (0: all)
  if constexpr (WAVES > 1) {
    if (lane == 0) parts[0][wave] = a.m, parts[1][wave] = a.s, parts[2][wave] = a.e;
    if (threadIdx.x == 0) counts[0] = 0;
    if constexpr (TOP) bests[t] = static_cast<uint16_t>(order_of_best(best) >> 16);
    __syncthreads();
    a = waves_join(parts);
    if constexpr (TOP) tau = bound_of(bests, lane, p.top);
  } else if constexpr (TOP) {
    tau = bound_of(best, p.top);
  }
  Sums row;
  if (whole) row = sums_of<T, NT, 0>(p, at.row, a, t, parts[0]);
  if (t == 0) {
    if (whole) finish(p, at.row, row, given);
    else p.stats[unit] = make_float4(a.m, a.s, a.e, 0.f);
  }
  if constexpr (TOP) {
    uint64_t* list = lists + own * kQueue;
    if (whole && row.s != row.s) {
      top_by_order<T, NT, 0>(p, at.row, row, t, queues + own * kQueue, lists);
      return;
    }
    const float tau_x = tau ? value_of(tau) : -INFINITY;
    // A lane marks its candidates (a bit each, the single element last), then writes them behind those
    // of the lanes before it, each looked up once more by its index.
    constexpr int kBits = R * VEC;
    uint64_t marks = static_cast<uint64_t>(alone && single >= tau_x) << kBits;
#pragma unroll
    for (int j = 0; j < R; ++j) {
      const bool there = values.there(j);
      float x[VEC];
      values.template get<true>(j, x);
      if (__builtin_amdgcn_ballot_w64(there && most_of(x) >= tau_x) == 0) continue;
      uint32_t bits = 0;
#pragma unroll
      for (int i = 0; i < VEC; ++i) bits |= x[i] >= tau_x ? 1u << i : 0u;
      marks |= static_cast<uint64_t>(there ? bits : 0u) << (VEC * j);
    }
    const int mine = __builtin_popcountll(marks), upto = static_cast<int>(wave_scan(static_cast<uint32_t>(mine)));
    int n = __builtin_amdgcn_readlane(upto, 63), to = upto - mine;
    if constexpr (WAVES > 1) {
      int first = 0;
      if (lane == 0) first = atomicAdd(&counts[0], n);
      to += __builtin_amdgcn_readfirstlane(first);
    }
    while (marks) {
      const int i = __builtin_ctzll(marks);
      marks &= marks - 1;
      const int at_i = i == kBits ? at.single(p, t) : at.head + (at.v0 + NT * (i / VEC) + t) * VEC + i % VEC;
      if (to < kKeys) list[to] = key_of(Elem<T>::load1(at.x + at_i), at_i);
      ++to;
    }
    sync();
    if constexpr (WAVES > 1) n = counts[0];
    if (n > kKeys) {
      Queue q(queues + wave * kQueue, p.top);
      q.bound(tau);
      q.best = single;
      if (WAVES == 1 || wave == 0) q.push(alone && single >= q.tau_x ? key_of(single, at.single(p, t)) : 0);
      scan<T>(q, at.x + at.head, at.head, WAVES == 1 ? 0 : 64 * wave, NT, at.v0, at.v1);
      sync();
      if (t == 0) counts[own] = 0;
      sync();
      for (int i = lane; i < q.n; i += 64) list[atomicAdd(&counts[own], 1)] = q.q[i];
      sync();
      n = counts[own];
    }
    if (whole) {
      select<NT>(list, n, p.top, [&](int rank, uint64_t key) { finish_top(p, at.row, row, rank, key); });
    } else {
      uint64_t* out = p.keys + unit * p.top;
      select<NT>(list, n, p.top, [&](int rank, uint64_t key) { out[rank] = key; });
      for (int i = n + t; i < p.top; i += NT) out[i] = 0;
    }
  }
}

// Longer rows and slices: workgroups that stay, four waves that stream one part after the other and,
// with a top, a fifth that picks each part's largest logits while the next one streams.  A lane
// keeps the largest of each of its runs (half an instruction a logit), as the upper half of its
// order; the k-th largest of a wave's lanes bounds the k-th of the part, and the runs that reach
// the bound, few more than `top`, are read again.
// Bound by the bytes: 4096 rows of 131072 bf16 logits 187 us without a top (5.75 TB/s), 198 with one
// of 5.  That the fifth wave picks is what hides it: candidates queued by the waves that stream
// 287 us, a part's end in these waves 260.  Five workgroups a CU, in the registers of seven waves
// a SIMD; four, without that bound, 209 us, six in the registers of eight 243.
// No register spills.  A run in which a lane has no vector (a part's last one) or a logit of -infinity is weighed
// twice and read again, so a row of 32000 a quarter of it, and one of which most is masked all: 340 us for 191.
template <typename T, bool TOP>
__global__ __launch_bounds__(TOP ? 320 : 256, TOP ? 7 : 1) void stream_kernel(Params p, int64_t parts_n) {
  constexpr int VEC = Elem<T>::kVec, NT = 256, kStep = NT * kRun;
  constexpr int kKeys = 512, kPicks = 512;
  __shared__ __attribute__((aligned(16))) uint16_t slots[TOP ? 2 : 1][TOP ? kSlots : 1][NT];
  __shared__ uint64_t list[TOP ? kKeys : 1];
  __shared__ uint64_t queue[TOP ? kQueue : 1];
  __shared__ uint16_t picks[TOP ? kPicks : 1];
  __shared__ __attribute__((aligned(16))) uint16_t bests[2][256];
  __shared__ float parts[2][3][4];
  __shared__ uint32_t unusual[TOP ? kMostTurns / 32 : 1];  // rows without usual sums, a bit each
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, t = threadIdx.x;
  int parity = 0;
  if (!TOP || wave < 4) {
    int64_t unit = blockIdx.x;
    uint4 raw[kRun];
    {
      const Part<T> at(p, unit);
      fetch<NT>(raw, at.body, at.v0, t, at.v1);
    }
    for (; unit < parts_n; unit += gridDim.x, parity ^= 1) {
      const Part<T> at(p, unit);
      const bool more = unit + gridDim.x < parts_n;
      const Part<T> after(p, more ? unit + gridDim.x : unit);
      Stats a;
      float best = -INFINITY;
      if (at.rest > 0 && wave == 0) {
        best = lane < at.rest ? Elem<T>::load1(at.x + at.single(p, lane)) : -INFINITY;
        add_run<1, true>(a, Single{best}, p.c);
      }
      int run = 0;
      if (at.v0 < at.v1) look<T, NT>(a, raw, at.v0, t, at.v1, p.c);
      for (int v = at.v0; v < at.v1; v += kStep, ++run) {
        // (The next part's first run loads while this part ends; without one, a single vector.)
        const bool last = v + kStep >= at.v1;
        const uint4* then = last ? after.body : at.body;
        const int nv = last ? after.v0 : v + kStep, nv1 = !last ? at.v1 : more ? after.v1 : after.v0 + 1;
        const float most = v + kStep <= at.v1
                               ? add_run<VEC, TOP>(a, Streamed<T, NT, true>{raw, at.body, v, t, at.v1, then, nv, nv1}, p.c)
                               : add_run<VEC, TOP>(a, Streamed<T, NT, false>{raw, at.body, v, t, at.v1, then, nv, nv1}, p.c);
        if constexpr (TOP) {
          best = fmaxf(best, most);
          const uint32_t held = v + t < at.v1 ? order_of(most) >> 16 : 0u;  // 0: no vector
          uint16_t* slot = &slots[parity][run % kSlots][t];
          *slot = static_cast<uint16_t>(run < kSlots ? held : max(held, static_cast<uint32_t>(*slot)));
        }
      }
      a = wave_join(a);
      if (lane == 0) parts[parity][0][wave] = a.m, parts[parity][1][wave] = a.s, parts[parity][2][wave] = a.e;
      if constexpr (TOP) bests[parity][t] = static_cast<uint16_t>(order_of_best(best) >> 16);
      __syncthreads();
      if constexpr (!TOP) {  // (the workgroup's one part)
        a = waves_join(parts[parity]);
        if (p.slices == 1) {
          const Sums row = sums_of<T, NT, kAhead>(p, at.row, a, t, parts[parity ^ 1][0]);
          Given given;
          if (t == 0) given.load<T>(p, at.row), finish(p, at.row, row, given);
        } else if (t == 0) {
          p.stats[unit] = make_float4(a.m, a.s, a.e, 0.f);
        }
      }
    }
  } else if constexpr (TOP) {
    for (int i = lane; i < kMostTurns / 32; i += 64) unusual[i] = 0;
    wave_sync();
    int turn = 0;
    for (int64_t unit = blockIdx.x; unit < parts_n; unit += gridDim.x, parity ^= 1, ++turn) {
      const Part<T> at(p, unit);
      const bool whole = p.slices == 1;
      Given given;
      if (whole && lane == 0) given.load<T>(p, at.row);
      const bool alone = lane < at.rest;
      const float single = alone ? Elem<T>::load1(at.x + at.single(p, lane)) : -INFINITY;
      __syncthreads();  // the part has been streamed
      const Stats a = waves_join(parts[parity]);
      const Sums row(a);
      if (whole && !row.usual()) {
        if (lane == 0) unusual[turn >> 5] |= 1u << (turn & 31);
        continue;
      }
      if (lane == 0) {
        if (whole) finish(p, at.row, row, given);
        else p.stats[unit] = make_float4(a.m, a.s, a.e, 0.f);
      }
      const uint32_t tau = bound_of(bests[parity], lane, p.top);
      const float tau_x = tau ? value_of(tau) : -INFINITY;
      int n = 0, runs = 0;
      auto add = [&](bool in, float value, int i) {
        const uint64_t mask = __builtin_amdgcn_ballot_w64(in);
        if (mask == 0) return;
        const int to = n + rank_in(mask);
        if (in && to < kKeys) list[to] = key_of(value, i);
        n += __builtin_popcountll(mask);
      };
      add(alone && single >= tau_x, single, at.single(p, lane));
      const int held = min(kSlots, (at.v1 - at.v0 + kStep - 1) / kStep);
      const uint32_t least = max(tau >> 16, 1u);
      for (int k = 0; k < held; ++k) {
        const uint2 four = reinterpret_cast<const uint2*>(slots[parity][k])[lane];
        const uint32_t order[4] = {four.x & 0xffff, four.x >> 16, four.y & 0xffff, four.y >> 16};
        if (__builtin_amdgcn_ballot_w64(max(max(order[0], order[1]), max(order[2], order[3])) >= least) == 0) continue;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint64_t mask = __builtin_amdgcn_ballot_w64(order[j] >= least);
          const int to = runs + rank_in(mask);
          if (order[j] >= least && to < kPicks) picks[to] = static_cast<uint16_t>(k * NT + 4 * lane + j);
          runs += __builtin_popcountll(mask);
        }
      }
      wave_sync();
      for (int i0 = 0; i0 < runs && runs <= kPicks; i0 += 64) {
        const bool mine = i0 + lane < runs;
        const int pick = mine ? picks[i0 + lane] : 0;
        for (int v0 = at.v0; v0 < at.v1; v0 += kSlots * kStep) {  // (runs of one slot)
          const int v = v0 + pick / NT * kStep + pick % NT;
          uint4 raw[kRun];
#pragma unroll
          for (int j = 0; j < kRun; ++j)
            if (mine && v + NT * j < at.v1) raw[j] = at.body[v + NT * j];
#pragma unroll
          for (int j = 0; j < kRun; ++j) {
            float x[VEC];
            load_vec(reinterpret_cast<const T*>(&raw[j]), x);
            const bool there = mine && v + NT * j < at.v1;
            if (__builtin_amdgcn_ballot_w64(there && most_of(x) >= tau_x) == 0) continue;
#pragma unroll
            for (int i = 0; i < VEC; ++i) add(there && x[i] >= tau_x, x[i], at.head + (v + NT * j) * VEC + i);
          }
        }
      }
      if (runs > kPicks || n > kKeys) {
        Queue q(queue, p.top);
        q.bound(tau);
        q.best = single;
        q.push(alone && single >= q.tau_x ? key_of(single, at.single(p, lane)) : 0);
        scan<T>(q, at.x + at.head, at.head, 0, 64, at.v0, at.v1);
        wave_sync();
        for (int i = lane; i < q.n; i += 64) list[i] = q.q[i];
        n = q.n;
      }
      wave_sync();
      if (whole) {
        select<64>(list, n, p.top, [&](int rank, uint64_t key) { finish_top(p, at.row, row, rank, key); });
      } else {
        uint64_t* out = p.keys + unit * p.top;
        select<64>(list, n, p.top, [&](int rank, uint64_t key) { out[rank] = key; });
        for (int i = n + lane; i < p.top; i += 64) out[i] = 0;
      }
      wave_sync();
    }
  }
  if constexpr (TOP) {
    // Rows without usual sums, by all waves, behind the others (in the fifth wave's turn they held up
    // the stream, and their registers spilled in it).
    constexpr int kAll = NT + 64;
    static_assert(sizeof(slots) >= kAll / 64 * kQueue * sizeof(uint64_t) && kKeys >= kAll / 64 * kMostTop,
                  "queues of all waves");
    __shared__ float of_waves[kAll / 64];
    if (p.slices > 1) return;
    __syncthreads();
    int64_t unit = blockIdx.x;
    for (int turn = 0; unit < parts_n; unit += gridDim.x, ++turn) {
      if (!(unusual[turn >> 5] >> (turn & 31) & 1)) continue;
      const Sums row = exact_sums<T, kAll, kAhead>(p, unit, t, of_waves);
      if (t == 0) {
        Given given;
        given.load<T>(p, unit);
        finish(p, unit, row, given);
      }
      top_by_order<T, kAll, kAhead>(p, unit, row, t, reinterpret_cast<uint64_t*>(slots), list);
      __syncthreads();
    }
  }
}

// Joins a row's slices; a wave a row, and three more for rows outside the usual sums.  Bound by the
// chain of its loads: 4.3 us for 16 rows.
template <typename T>
__global__ __launch_bounds__(256) void join_kernel(Params p) {
  constexpr int kHeld = 8;  // keys of a lane in registers
  __shared__ uint64_t list[kMostSlices * kMostTop];
  __shared__ uint64_t best_of_waves[4 * kMostTop];
  __shared__ float parts[4];
  __shared__ int unusual;
  static_assert(kMostSlices * kMostTop >= 4 * kQueue, "queues of four waves");
  const int lane = threadIdx.x & 63, t = threadIdx.x;
  const int64_t row = blockIdx.x;
  const int n = p.slices * p.top;
  const uint64_t* keys = p.keys + row * n;
  Given given;
  Sums sums;
  uint64_t best = 0, held[kHeld] = {};
  if (t < 64) {
    Stats a;
    if (lane == 0) given.load<T>(p, row);
    if (lane < p.slices) {
      const float4 s = p.stats[row * p.slices + lane];
      a.m = s.x;
      a.s = s.y;
      a.e = s.z;
    }
#pragma unroll
    for (int i = 0; i < kHeld; ++i) held[i] = lane + 64 * i < n ? keys[lane + 64 * i] : 0;
    a.move(wave_max(a.m));
    sums = Sums(wave_join(a));
    if (lane == 0) unusual = !sums.usual();
  }
  __syncthreads();
  const bool exact = unusual != 0;
  if (exact) sums = exact_sums<T, 256, kAhead>(p, row, t, parts);
  if (t == 0) finish(p, row, sums, given);
  if (p.top == 0) return;
  if (exact && sums.s != sums.s) {
    top_by_order<T, 256, kAhead>(p, row, sums, t, list, best_of_waves);
    return;
  }
  if (t >= 64) return;
#pragma unroll
  for (int i = 0; i < kHeld; ++i) best = held[i] > best ? held[i] : best;
  for (int i = lane + 64 * kHeld; i < n; i += 64) best = keys[i] > best ? keys[i] : best;
  const uint32_t high[1] = {static_cast<uint32_t>(best >> 32)};
  const uint64_t bound = static_cast<uint64_t>(kth_bound<uint32_t, 32>(high, p.top)) << 32;
  int count = 0;
  auto take = [&](uint64_t key) {
    const bool in = key != 0 && key >= bound;
    const uint64_t mask = __builtin_amdgcn_ballot_w64(in);
    if (in) list[count + rank_in(mask)] = key;
    count += __builtin_popcountll(mask);
  };
#pragma unroll
  for (int i = 0; i < kHeld; ++i) take(held[i]);
  for (int i0 = 64 * kHeld; i0 < n; i0 += 64) take(i0 + lane < n ? keys[i0 + lane] : 0);
  wave_sync();
  select<64>(list, count, p.top, [&](int rank, uint64_t key) { finish_top(p, row, sums, rank, key); });
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
// Bound by the bytes: 8192 rows of 32000 bf16 logits (1.05 GB) 190 us, 5.5 TB/s.
template <typename T, int WAVES>
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
  // (Vectors as the gradient's row lies; the logits' may lie otherwise: a load of 16 bytes needs no
  // alignment.  2048 rows of 32003 bf16 logits, 32064 apart: 70 us one by one, 41.5 so.)
  const int head = min(static_cast<int>((-reinterpret_cast<uintptr_t>(db) & 15) / sizeof(T)), p.V);
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
      if (v0 + NT * j + t < nv) __builtin_memcpy(&raw[j], X + head + static_cast<int64_t>(v0 + NT * j + t) * VEC, 16);
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


// Logits of a run of `waves` waves.
constexpr int64_t run_of(int64_t es, int waves) { return waves * 64 * kRun * 16 / es; }

// A wave takes a row alone where one run (the gradient: two) holds it.
static bool short_rows(int64_t V, int64_t es, int runs = 1) { return V <= runs * run_of(es, 1); }

// Workgroups that share a row: so many that about 1024 run, each with a full run at least.
static int64_t slices_of(int64_t N, int64_t V, int64_t es) {
  const int64_t run = run_of(es, 4);
  return std::max<int64_t>(1, std::min<int64_t>({(V + run - 1) / run, 1024 / std::max<int64_t>(N, 1), kMostSlices}));
}

template <typename T, int WAVES, int R>
static void launch_run(const Params& p, int64_t groups, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(groups));
  if (p.top) hipLaunchKernelGGL((run_kernel<T, WAVES, R, true>), grid, dim3(256), 0, s, p);
  else hipLaunchKernelGGL((run_kernel<T, WAVES, R, false>), grid, dim3(256), 0, s, p);
}
// As many vectors a lane as the longest row or slice needs: those that it does not have cost their
// instructions all the same.  (100000 rows of 500 bf16 logits: 126 us with four, 53 with one.)
template <typename T, int WAVES>
static void launch_runs(const Params& p, int64_t groups, hipStream_t s) {
  const int64_t lanes = 64 * WAVES, vectors = p.slices == 1 ? p.V / Elem<T>::kVec : p.per;
  if (vectors <= lanes) launch_run<T, WAVES, 1>(p, groups, s);
  else if (vectors <= 2 * lanes) launch_run<T, WAVES, 2>(p, groups, s);
  else launch_run<T, WAVES, kRun>(p, groups, s);
}

template <typename T>
static void launch(const Params& p, hipStream_t s) {
  if (short_rows(p.V, sizeof(T))) {
    launch_runs<T, 1>(p, (p.N + 3) / 4, s);
    return;
  }
  const int64_t parts = p.N * p.slices;  // (below 2^24: one row each, or 1024 of them)
  if (p.per <= 256 * kRun) {
    launch_runs<T, 4>(p, parts, s);
  } else {
    // Workgroups that stay, as many as run at once, with as many parts each as can be alike.
    const int64_t most = kCus * kStay, turns = (parts + most - 1) / most;
    const dim3 grid(static_cast<unsigned>(p.top ? (parts + turns - 1) / turns : parts));
    if (p.top) hipLaunchKernelGGL((stream_kernel<T, true>), grid, dim3(320), 0, s, p, parts);
    else hipLaunchKernelGGL((stream_kernel<T, false>), grid, dim3(256), 0, s, p, parts);
  }
  if (p.slices > 1) hipLaunchKernelGGL((join_kernel<T>), dim3(static_cast<unsigned>(p.N)), dim3(256), 0, s, p);
}

template <typename T>
static int launch_grad(Grad& p, hipStream_t s, GHipError* err, const char* what) {
  const bool one = short_rows(p.V, sizeof(T), 2);
  const int64_t run = run_of(sizeof(T), 4);
  p.runs = one ? 1 : static_cast<int>((p.V + run - 1) / run);
  const int64_t blocks = one ? (p.N + 3) / 4 : p.N * p.runs;
  if (blocks > kMostGroups) return set_error(err, GHIP_ERR_UNSUPPORTED, "%s: problem too large", what);
  const dim3 grid(static_cast<unsigned>(blocks));
  if (one) hipLaunchKernelGGL((grad_kernel<T, 1>), grid, dim3(256), 0, s, p);
  else hipLaunchKernelGGL((grad_kernel<T, 4>), grid, dim3(256), 0, s, p);
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
  p.scale = scale;
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
