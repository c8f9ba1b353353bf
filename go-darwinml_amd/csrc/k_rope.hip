// Rotary positions, alone and on the way into a paged key-value cache of 16 or 4 bits, and
// the way back out of 4 bits.
//
//   pair i of a row at token (b, s):  a = position * freqs[i],  (x, y) -> (x cos a - y sin a, x sin a + y cos a)
//
// No reference op (GoMLX composes it of primitives).  Bound by the bytes of the rows.
#include "kv4_dev.h"
#include "rope_dev.h"
#include "rope_rules.h"

namespace ghip {
namespace rope {

constexpr int64_t kMostGroups = (int64_t{1} << 24) - 1;  // workgroups of a launch (HIP: fewer than 2^32 threads)

struct Rows {  // [B, heads, S, D]
  char* p;
  int64_t sb, sh, ss;  // byte strides
};
struct Cache {  // rows of a page
  char* p;
  int64_t sp, sh, st;  // byte strides
};

struct Params {
  Angles a;
  Rows q, qo, k, v;
  Cache kc, vc;  // 16 bits and more: the rows; 4 bits: the codes
  Cache ks, vs;  // 4 bits: the scales
  const int32_t* table;
  const int32_t* counts;
  int64_t table_stride;
  int64_t tokens;  // B S
  int S, H, Hkv, D, R, num_pages, page_size, max_pages;
  int units, units4;  // threads of a row
  Deal deal;
};

// What the workgroup's tokens need: the angles of their pairs, and where their rows go.
struct Shared {
  float2 cs[kMostTokens][kMostHalf];
  int b[kMostTokens], s[kMostTokens], page[kMostTokens], at[kMostTokens];
};

__device__ __forceinline__ void prepare(const Params& p, Shared& sh, int64_t first, int n, bool turns) {
  for (int t = threadIdx.x; t < n; t += kThreads) {
    const int64_t token = first + t;
    const int b = static_cast<int>(token / p.S), s = static_cast<int>(token - static_cast<int64_t>(b) * p.S);
    sh.b[t] = b;
    sh.s[t] = s;
    int page = -1, at = 0;
    if (p.table && (!p.counts || s < p.counts[b])) {
      const int64_t pos = static_cast<int64_t>(p.a.starts[b]) + s;
      if (pos >= 0 && pos < static_cast<int64_t>(p.max_pages) * p.page_size) {
        const uint32_t entry = static_cast<uint32_t>(pos) / static_cast<uint32_t>(p.page_size);
        page = p.table[b * p.table_stride + entry];
        if (page >= p.num_pages) page = -1;
        at = static_cast<int>(static_cast<uint32_t>(pos) - entry * static_cast<uint32_t>(p.page_size));
      }
    }
    sh.page[t] = page;
    sh.at[t] = at;
  }
  if (turns) {
    for (int j = threadIdx.x; j < n * p.a.half; j += kThreads) {
      const int t = j / p.a.half, i = j - t * p.a.half;
      const int64_t token = first + t;
      const int b = static_cast<int>(token / p.S), s = static_cast<int>(token - static_cast<int64_t>(b) * p.S);
      sh.cs[t][i] = turn(position(p.a, b, s, i), p.a.freqs[i], p.a.inverse);
    }
  }
  __syncthreads();
}

// N elements at any element's alignment: loads and stores of up to 16 bytes need none.
template <typename T, int N>
struct alignas(N * sizeof(T)) Few {
  T v[N];
};
template <typename T, int N>
__device__ __forceinline__ void load_n(const T* p, float* x) {
  Few<T, N> few;
  __builtin_memcpy(&few, p, sizeof(few));
  if constexpr (N == Elem<T>::kVec) {
    load_vec(few.v, x);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = Elem<T>::load1(&few.v[e]);
  }
}
template <typename T, int N>
__device__ __forceinline__ void store_n(T* p, const float* x) {
  Few<T, N> few;
  if constexpr (N == Elem<T>::kVec) {
    store_vec(few.v, x);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) Elem<T>::store1(&few.v[e], x[e]);
  }
  __builtin_memcpy(p, &few, sizeof(few));
}

// Rows of whole elements.  A thread holds N pairs of a row, as two runs of N elements: run
// `a` and the one half a row behind it, or two runs one after the other.  Units past the
// pairs copy the row's other elements, two runs each.
template <typename T, int N>
__device__ __forceinline__ void row_unit(const Params& p, const T* src, T* dst, const float2* cs, int u, bool turns) {
  const int pairs = turns ? p.a.half / N : 0, R = turns ? p.R : 0;
  float x[N], y[N];
  if (u < pairs) {
    const int a = p.a.neighbours ? 2 * N * u : N * u, c = p.a.neighbours ? a + N : p.a.half + a;
    load_n<T, N>(src + a, x);
    load_n<T, N>(src + c, y);
    if (!p.a.neighbours) {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float2 r = turned(x[e], y[e], cs[N * u + e]);
        x[e] = r.x;
        y[e] = r.y;
      }
    } else if constexpr (N == 1) {
      const float2 r = turned(x[0], y[0], cs[u]);
      x[0] = r.x;
      y[0] = r.y;
    } else {
#pragma unroll
      for (int e = 0; e < N; e += 2) {
        const float2 r = turned(x[e], x[e + 1], cs[N * u + e / 2]);
        x[e] = r.x;
        x[e + 1] = r.y;
        const float2 w = turned(y[e], y[e + 1], cs[N * u + N / 2 + e / 2]);
        y[e] = w.x;
        y[e + 1] = w.y;
      }
    }
    store_n<T, N>(dst + a, x);
    store_n<T, N>(dst + c, y);
  } else {
    const int a = R + 2 * N * (u - pairs);
    const bool two = a + N < p.D;
    load_n<T, N>(src + a, x);
    if (two) load_n<T, N>(src + a + N, y);
    store_n<T, N>(dst + a, x);
    if (two) store_n<T, N>(dst + a + N, y);
  }
}

// Rows on their way into 4 bits.  A thread holds 8 consecutive values; four neighbours share
// a scale, found by two exchanges inside each four lanes.
template <typename T, bool WIDE>
__device__ __forceinline__ void row_unit4(const Params& p, const T* src, char* codes, char* scales, const float2* cs,
                                          int u, bool turns) {
  float x[8];
  const int d = 8 * u, R = turns ? p.R : 0;
  if constexpr (WIDE) {  // whole units turn, or none of a unit
    constexpr int V = Elem<T>::kVec;
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; i += V) load_n<T, V>(src + d + i, x + i);
    if (d < R) {
      if (p.a.neighbours) {
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const float2 r = turned(x[e], x[e + 1], cs[4 * u + e / 2]);
          x[e] = r.x;
          x[e + 1] = r.y;
        }
      } else {
        const bool low = d < p.a.half;
        const int other = low ? d + p.a.half : d - p.a.half, i0 = low ? d : other;
#pragma unroll
        for (int i = 0; i < 8; i += V) load_n<T, V>(src + other + i, y + i);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float2 r = low ? turned(x[e], y[e], cs[i0 + e]) : turned(y[e], x[e], cs[i0 + e]);
          x[e] = low ? r.x : r.y;
        }
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int c = d + e;
      x[e] = Elem<T>::load1(src + c);
      if (c < R) {
        const bool first = p.a.neighbours ? (c & 1) == 0 : c < p.a.half;
        const int i = p.a.neighbours ? c >> 1 : first ? c : c - p.a.half;
        const int other = p.a.neighbours ? c ^ 1 : first ? c + p.a.half : i;
        const float y = Elem<T>::load1(src + other);
        const float2 r = first ? turned(x[e], y, cs[i]) : turned(y, x[e], cs[i]);
        x[e] = first ? r.x : r.y;
      }
    }
  }
  uint32_t most = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) most = max(most, __float_as_uint(x[e]) & 0x7fffffffu);
  most = max(most, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(most), 0xb1, 0xf, 0xf, false)));
  most = max(most, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(most), 0x4e, 0xf, 0xf, false)));
  const uint32_t scale = kv4::scale_of(most);
  *reinterpret_cast<uint32_t*>(codes + 4 * u) = kv4::encode8(x, scale);
  if ((u & 3) == 0) scales[u >> 2] = static_cast<char>(scale);
}

// A slot of a workgroup (the threads of a row) and the rows that it takes: (token, head) of `n`
// tokens and `nh` heads, one slot after the other.
struct Slots {
  int u, t, h, dt, dh, nh;
  bool any;
  __device__ __forceinline__ Slots(int units, int nh_) : nh(nh_) {
    const int slots = kThreads / units, slot = threadIdx.x / units;
    u = threadIdx.x - slot * units;
    any = slot < slots && nh > 0;
    if (!any) return;
    dt = slots / nh;
    dh = slots - dt * nh;
    t = slot / nh;
    h = slot - t * nh;
  }
  __device__ __forceinline__ void next() {
    t += dt;
    h += dh;
    if (h >= nh) {
      h -= nh;
      ++t;
    }
  }
};

// A workgroup takes some tokens and all their rows, or, where the tokens are few, a share of
// one token's rows: the angles are computed once for all of its heads.  FOUR: the rows of
// keys and values go into 4 bits, by threads of their own share of a row.
// Bound by the bytes of the rows, then, for a few tokens, by the chain position - angle - row:
// 8192 tokens of 16 heads of 128 in bf16 (67 MB) 12.8 us, 8 prompts of 1024 tokens, 32 heads and
// 8, into 16 bits (172 MB) 36 us, into 4 bits 38; 16 tokens 4.3 and 5.8.  Two rows of a thread
// under way at once: 59 us for 35.7 (88 registers).
template <typename T, int N, bool FOUR, bool WIDE>
__global__ __launch_bounds__(kThreads) void rope_kernel(Params p) {
  __shared__ Shared sh;
  const int splits = p.deal.splits + (FOUR ? p.deal.splits4 : 0);
  const int64_t block = blockIdx.x / splits;
  const int split = blockIdx.x - static_cast<int>(block) * splits;
  const int64_t first = block * p.deal.block_tokens;
  const int n = static_cast<int>(min(static_cast<int64_t>(p.deal.block_tokens), p.tokens - first));
  prepare(p, sh, first, n, p.R > 0);
  if (split < p.deal.splits) {
    const int heads = FOUR ? p.H : p.H + 2 * p.Hkv, per = (heads + p.deal.splits - 1) / p.deal.splits, h0 = split * per;
    Slots at(p.units, min(per, heads - h0));
    for (; at.any && at.t < n; at.next()) {
      const int b = sh.b[at.t], s = sh.s[at.t], head = h0 + at.h;
      if (FOUR || head < p.H) {
        row_unit<T, N>(p, reinterpret_cast<const T*>(p.q.p + b * p.q.sb + head * p.q.sh + s * p.q.ss),
                       reinterpret_cast<T*>(p.qo.p + b * p.qo.sb + head * p.qo.sh + s * p.qo.ss), sh.cs[at.t], at.u, p.R > 0);
      } else if (const int page = sh.page[at.t]; page >= 0) {
        const bool key = head < p.H + p.Hkv;
        const int hk = head - p.H - (key ? 0 : p.Hkv);
        const Rows& r = key ? p.k : p.v;
        const Cache& c = key ? p.kc : p.vc;
        row_unit<T, N>(p, reinterpret_cast<const T*>(r.p + b * r.sb + hk * r.sh + s * r.ss),
                       reinterpret_cast<T*>(c.p + page * c.sp + hk * c.sh + static_cast<int64_t>(sh.at[at.t]) * c.st),
                       sh.cs[at.t], at.u, key && p.R > 0);
      }
    }
  }
  if constexpr (FOUR) {
    const int part = split - (p.deal.both ? 0 : p.deal.splits);  // (both: this workgroup takes all rows)
    if (part < 0) return;
    const int parts = p.deal.both ? 1 : p.deal.splits4, heads = 2 * p.Hkv, per = (heads + parts - 1) / parts, h0 = part * per;
    Slots at(p.units4, min(per, heads - h0));
    for (; at.any && at.t < n; at.next()) {
      const int b = sh.b[at.t], s = sh.s[at.t], head = h0 + at.h, page = sh.page[at.t];
      if (page < 0) continue;
      const bool key = head < p.Hkv;
      const int hk = key ? head : head - p.Hkv;
      const int64_t row = sh.at[at.t];
      const Rows& r = key ? p.k : p.v;
      const Cache& c = key ? p.kc : p.vc;
      const Cache& w = key ? p.ks : p.vs;
      row_unit4<T, WIDE>(p, reinterpret_cast<const T*>(r.p + b * r.sb + hk * r.sh + s * r.ss),
                         c.p + page * c.sp + hk * c.sh + row * c.st, w.p + page * w.sp + hk * w.sh + row * w.st, sh.cs[at.t],
                         at.u, key && p.R > 0);
    }
  }
}

// ---------------------------------------------------------------- out of 4 bits
struct Read {
  Cache kc, ks, vc, vs;
  Rows k, v;
  const int32_t* table;
  const int32_t* lens;
  int64_t table_stride;
  int S, Hkv, units, num_pages, page_size;
};

// A thread widens 8 values of a token's key and of its value; a workgroup takes neighbouring
// tokens of one head, and rows past a sequence's length and on no page get zeros.
// Bound by the bytes written: 8 x 1280 tokens, 8 heads of 128, to bf16 10.6 us (5.0 TB/s; two heads a
// thread 11.5, four 12.2).
template <typename T>
__global__ __launch_bounds__(kThreads) void read4_kernel(Read p) {
  const int slots = kThreads / p.units, slot = threadIdx.x / p.units, u = threadIdx.x - slot * p.units;
  const int s = blockIdx.x * slots + slot, b = blockIdx.y, h = blockIdx.z;
  if (slot >= slots || s >= p.S) return;
  const int entry = s / p.page_size, at = s - entry * p.page_size;
  int page = -1;
  if (!p.lens || s < p.lens[b]) page = p.table[b * p.table_stride + entry];
  uint32_t codes[2] = {0, 0}, scales[2] = {0, 0};
  if (page >= 0 && page < p.num_pages) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const Cache& c = j ? p.vc : p.kc;
      const Cache& w = j ? p.vs : p.ks;
      codes[j] = *reinterpret_cast<const uint32_t*>(c.p + page * c.sp + h * c.sh + at * c.st + 4 * u);
      scales[j] = *reinterpret_cast<const uint8_t*>(w.p + page * w.sp + h * w.sh + at * w.st + (u >> 2));
    }
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const Rows& r = j ? p.v : p.k;
    T* out = reinterpret_cast<T*>(r.p + b * r.sb + h * r.sh + s * r.ss) + 8 * u;
    const uint4 d = kv4::decode8(codes[j], kv4::scale_f32(scales[j]));
    if constexpr (__is_same(T, bf16_t)) {
      *reinterpret_cast<uint4*>(out) = d;
    } else {
      const uint32_t words[4] = {d.x, d.y, d.z, d.w};
      float x[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[2 * e] = __uint_as_float(words[e] << 16);
        x[2 * e + 1] = __uint_as_float(words[e] & 0xffff0000u);
      }
#pragma unroll
      for (int e = 0; e < 8; e += Elem<T>::kVec) store_vec(out + e, x + e);
    }
  }
}

template <typename T, bool FOUR>
static int launch(Params& p, bool wide4, hipStream_t s, GHipError* err, const char* what) {
  constexpr int V = Elem<T>::kVec;
  int n = width(p.D, p.a.half, V);
  // (Beside rows into 4 bits there are no kernels of the widths between: bf16, 8 x 1024 tokens, 32 heads and
  // 8 of 96, 24 of them turned, 134 us; q alone four at a time 28, and the call without q 33.)
  if (FOUR && n < V) n = 1;
  p.units = (p.D + 2 * n - 1) / (2 * n);  // (half a row's pairs are a multiple of n)
  p.units4 = p.D / 8;
  p.deal = deal(p.tokens, p.H, p.Hkv, p.units, p.units4, FOUR);
  const int64_t blocks = (p.tokens + p.deal.block_tokens - 1) / p.deal.block_tokens * (p.deal.splits + p.deal.splits4);
  if (blocks > kMostGroups) return set_error(err, GHIP_ERR_UNSUPPORTED, "%s: problem too large", what);
  const dim3 grid(static_cast<unsigned>(blocks));
  if constexpr (FOUR) {
    if (n == V && wide4) hipLaunchKernelGGL((rope_kernel<T, V, true, true>), grid, dim3(kThreads), 0, s, p);
    else if (n == V) hipLaunchKernelGGL((rope_kernel<T, V, true, false>), grid, dim3(kThreads), 0, s, p);
    else if (wide4) hipLaunchKernelGGL((rope_kernel<T, 1, true, true>), grid, dim3(kThreads), 0, s, p);
    else hipLaunchKernelGGL((rope_kernel<T, 1, true, false>), grid, dim3(kThreads), 0, s, p);
  } else {
    if (n == V) hipLaunchKernelGGL((rope_kernel<T, V, false, false>), grid, dim3(kThreads), 0, s, p);
    else if (V == 8 && n == 4) hipLaunchKernelGGL((rope_kernel<T, V / 2, false, false>), grid, dim3(kThreads), 0, s, p);
    else if (n == 2) hipLaunchKernelGGL((rope_kernel<T, 2, false, false>), grid, dim3(kThreads), 0, s, p);
    else hipLaunchKernelGGL((rope_kernel<T, 1, false, false>), grid, dim3(kThreads), 0, s, p);
  }
  GHIP_CHECK(hipGetLastError(), err);
  return GHIP_OK;
}

}  // namespace rope
}  // namespace ghip

using namespace ghip;

namespace {

int64_t elem(int dtype) { return dtype == GHIP_DTYPE_FLOAT32 ? 4 : 2; }

// The rotation's plan; `positions` are needed where there are no starts.
int read_rope(const GHipRope* r, int64_t D, int64_t S, const int32_t* starts, rope::Params& p, GHipError* err,
              const char* what) {
  if (r->rotary_dim < 0 || r->rotary_dim > D || r->rotary_dim % 2 != 0)
    return set_error(err, GHIP_ERR_INVALID_ARG, "%s: rotary_dim %lld must be even and at most the head dim %lld", what,
                     static_cast<long long>(r->rotary_dim), static_cast<long long>(D));
  if (r->rotary_dim == 0) return GHIP_OK;
  if (r->axes < 1 || r->axes > rope::kMostAxes)
    return set_error(err, GHIP_ERR_INVALID_ARG, "%s: 1 to %d axes of positions", what, rope::kMostAxes);
  if (!r->freqs) return set_error(err, GHIP_ERR_INVALID_ARG, "%s: freqs is null", what);
  if (!r->positions && (!starts || r->axes != 1))
    return set_error(err, GHIP_ERR_INVALID_ARG, "%s: positions are needed", what);
  int64_t end = 0;
  for (int i = 0; i < rope::kMostAxes; ++i) {
    if (i < r->axes) {
      if (r->sections[i] < 0) return set_error(err, GHIP_ERR_INVALID_ARG, "%s: negative section", what);
      end += std::min<int64_t>(r->sections[i], int64_t{1} << 60);  // (so that the sum cannot wrap around)
    }
    p.a.ends[i] = static_cast<int>(std::min<int64_t>(end, rope::kMostHalf));
  }
  if (end != r->rotary_dim / 2)
    return set_error(err, GHIP_ERR_INVALID_ARG, "%s: the sections hold %lld pairs, not rotary_dim / 2 = %lld", what,
                     static_cast<long long>(end), static_cast<long long>(r->rotary_dim / 2));
  if (r->positions && (r->position_strides[0] < 0 || r->position_strides[1] < 0 || r->position_strides[2] < 0))
    return set_error(err, GHIP_ERR_UNSUPPORTED, "%s: negative strides", what);
  p.a.positions = r->positions;
  p.a.freqs = r->freqs;
  p.a.p_sa = r->position_strides[0]; p.a.p_sb = r->position_strides[1]; p.a.p_ss = r->position_strides[2];
  p.a.half = static_cast<int>(r->rotary_dim / 2);
  p.a.neighbours = r->interleaved != 0;
  p.R = static_cast<int>(r->rotary_dim);
  return GHIP_OK;
}

int check_sizes(int dtype, int64_t B, int64_t H, int64_t Hkv, int64_t S, int64_t D, GHipError* err, const char* what) {
  if (dtype != GHIP_DTYPE_FLOAT32 && dtype != GHIP_DTYPE_BFLOAT16 && dtype != GHIP_DTYPE_FLOAT16)
    return set_error(err, GHIP_ERR_UNSUPPORTED, "%s: needs float32, bfloat16 or float16", what);
  if (B < 0 || S < 0 || H < 0 || Hkv < 0 || D <= 0) return set_error(err, GHIP_ERR_INVALID_ARG, "%s: bad sizes", what);
  if (D > 2 * rope::kMostHalf)
    return set_error(err, GHIP_ERR_UNSUPPORTED, "%s: needs a head dim of at most %d", what, 2 * rope::kMostHalf);
  constexpr int64_t kMost = int64_t{1} << 30;
  if (B > kMost || S > kMost || H > (1 << 20) || Hkv > (1 << 20) || B * S > kMost)
    return set_error(err, GHIP_ERR_UNSUPPORTED, "%s: problem too large", what);
  return GHIP_OK;
}

int check_pages(int64_t num_pages, int64_t page_size, int64_t max_pages, const int32_t* table, int64_t table_stride,
                GHipError* err, const char* what) {
  if (num_pages < 0 || page_size <= 0 || max_pages < 0)
    return set_error(err, GHIP_ERR_INVALID_ARG, "%s: bad sizes", what);
  constexpr int64_t kMost = int64_t{1} << 30;
  if (num_pages > kMost || page_size > kMost || max_pages > kMost || page_size * max_pages > kMost)
    return set_error(err, GHIP_ERR_UNSUPPORTED, "%s: problem too large", what);
  if (num_pages == 0 || max_pages == 0)
    return set_error(err, GHIP_ERR_INVALID_ARG, "%s: a cache without pages", what);
  if (!table) return set_error(err, GHIP_ERR_INVALID_ARG, "%s: null pointer", what);
  if (table_stride < 0) return set_error(err, GHIP_ERR_INVALID_ARG, "%s: negative table stride", what);
  return GHIP_OK;
}

// Strides in elements of `es` bytes; `n`: entries of each axis (one: its stride is not looked at,
// but for its sign).  false: a negative one, or one of 2^48 and more.
template <typename R>
bool take(R& r, const void* ptr, const int64_t* st, const int64_t (&n)[3], int64_t es, uint64_t* bits) {
  int64_t step[3];
  *bits |= reinterpret_cast<uint64_t>(ptr);
  for (int i = 0; i < 3; ++i) {
    if (st[i] < 0 || (n[i] > 1 && st[i] >= int64_t{1} << 48)) return false;
    step[i] = n[i] > 1 ? st[i] * es : 0;
    *bits |= static_cast<uint64_t>(step[i]);
  }
  r = R{const_cast<char*>(static_cast<const char*>(ptr)), step[0], step[1], step[2]};
  return true;
}

int launch_rope(int dtype, rope::Params& p, uint64_t bits, uint64_t bits4, bool four, hipStream_t s, GHipError* err,
                const char* what) {
  const int64_t es = elem(dtype);
  if ((bits | bits4) % es) return set_error(err, GHIP_ERR_INVALID_ARG, "%s: pointers are not aligned to elements", what);
  const bool wide4 = p.a.neighbours ? p.R % 8 == 0 : p.a.half % 8 == 0;
  if (dtype == GHIP_DTYPE_FLOAT32)
    return four ? rope::launch<float, true>(p, wide4, s, err, what) : rope::launch<float, false>(p, false, s, err, what);
  if (dtype == GHIP_DTYPE_FLOAT16)
    return four ? rope::launch<f16_t, true>(p, wide4, s, err, what) : rope::launch<f16_t, false>(p, false, s, err, what);
  return four ? rope::launch<bf16_t, true>(p, wide4, s, err, what) : rope::launch<bf16_t, false>(p, false, s, err, what);
}

// A 4-bit cache's tensors; false and the error set if they are not as the kernels read them.
bool take4(const GHipKv4* c, const int64_t (&n)[3], int64_t D, rope::Cache& codes, rope::Cache& scales) {
  uint64_t b0 = 0, b1 = 0;
  if (!take(codes, c->codes, c->code_strides, n, 1, &b0) || !take(scales, c->scales, c->scale_strides, n, 1, &b1)) return false;
  return b0 % 16 == 0 && b1 % 4 == 0;
}
const char kLayout4[] =
    "%s: codes must be 16-byte aligned with non-negative strides of whole 16 bytes, scales 4-byte aligned with strides of "
    "whole 4";

}  // namespace

extern "C" int ghip_rope(int dtype, const void* x, void* out, int64_t B, int64_t H, int64_t S, int64_t D,
                         const int64_t* x_strides, const int64_t* out_strides, const GHipRope* r, int inverse, void* stream,
                         GHipError* err) {
  static const char kWhat[] = "rope";
  if (int rc = check_sizes(dtype, B, H, 0, S, D, err, kWhat)) return rc;
  if (!r) return set_error(err, GHIP_ERR_INVALID_ARG, "%s: null pointer", kWhat);
  if (B == 0 || H == 0 || S == 0) return GHIP_OK;
  rope::Params p{};
  if (int rc = read_rope(r, D, S, nullptr, p, err, kWhat)) return rc;
  if (!x || !out || !x_strides || !out_strides) return set_error(err, GHIP_ERR_INVALID_ARG, "%s: null pointer", kWhat);
  const int64_t n[3] = {B, H, S}, es = elem(dtype);
  uint64_t bits = 0;
  if (!take(p.q, x, x_strides, n, es, &bits) || !take(p.qo, out, out_strides, n, es, &bits))
    return set_error(err, GHIP_ERR_UNSUPPORTED, "%s: negative strides", kWhat);
  p.a.inverse = inverse != 0;
  p.tokens = B * S;
  p.S = static_cast<int>(S); p.H = static_cast<int>(H); p.D = static_cast<int>(D);
  return launch_rope(dtype, p, bits, 0, false, static_cast<hipStream_t>(stream), err, kWhat);
}

namespace {

// What the two appends share; the caches' rows are taken by the caller.
int append_common(int dtype, const void* q, void* q_out, const void* k, const void* v, int64_t B, int64_t H, int64_t Hkv,
                  int64_t S, int64_t D, int64_t num_pages, int64_t page_size, int64_t max_pages,
                  const int32_t* block_table, int64_t table_stride, const int32_t* starts, const int32_t* counts,
                  const int64_t* q_strides, const int64_t* q_out_strides, const int64_t* k_strides,
                  const int64_t* v_strides, const GHipRope* r, rope::Params& p, uint64_t* bits, uint64_t* kv_bits,
                  GHipError* err, const char* what) {
  if (int rc = check_sizes(dtype, B, H, Hkv, S, D, err, what)) return rc;
  if (Hkv <= 0) return set_error(err, GHIP_ERR_INVALID_ARG, "%s: bad sizes", what);
  if (B == 0 || S == 0) return GHIP_OK;
  if (int rc = check_pages(num_pages, page_size, max_pages, block_table, table_stride, err, what)) return rc;
  if (!k || !v || !starts || !k_strides || !v_strides || (H > 0 && (!q || !q_out || !q_strides || !q_out_strides)))
    return set_error(err, GHIP_ERR_INVALID_ARG, "%s: null pointer", what);
  p.a.starts = starts;
  if (r)
    if (int rc = read_rope(r, D, S, starts, p, err, what)) return rc;
  const int64_t nq[3] = {B, H, S}, nk[3] = {B, Hkv, S}, es = elem(dtype);
  bool ok = take(p.k, k, k_strides, nk, es, kv_bits) && take(p.v, v, v_strides, nk, es, kv_bits);
  if (H > 0) ok = ok && take(p.q, q, q_strides, nq, es, bits) && take(p.qo, q_out, q_out_strides, nq, es, bits);
  if (!ok) return set_error(err, GHIP_ERR_UNSUPPORTED, "%s: negative strides", what);
  p.table = block_table;
  p.table_stride = table_stride;
  p.counts = counts;
  p.tokens = B * S;
  p.S = static_cast<int>(S); p.H = static_cast<int>(H); p.Hkv = static_cast<int>(Hkv); p.D = static_cast<int>(D);
  p.num_pages = static_cast<int>(num_pages); p.page_size = static_cast<int>(page_size);
  p.max_pages = static_cast<int>(max_pages);
  return GHIP_OK;
}

}  // namespace

extern "C" int ghip_kv_append_rope(int dtype, const void* q, void* q_out, const void* k, const void* v, void* k_cache,
                                   void* v_cache, int64_t B, int64_t H, int64_t Hkv, int64_t S, int64_t D,
                                   int64_t num_pages, int64_t page_size, int64_t max_pages, const int32_t* block_table,
                                   int64_t table_stride, const int32_t* starts, const int32_t* counts,
                                   const int64_t* q_strides, const int64_t* q_out_strides, const int64_t* k_strides,
                                   const int64_t* v_strides, const int64_t* k_cache_strides,
                                   const int64_t* v_cache_strides, const GHipRope* r, void* stream, GHipError* err) {
  static const char kWhat[] = "kv_append_rope";
  rope::Params p{};
  uint64_t bits = 0;
  if (int rc = append_common(dtype, q, q_out, k, v, B, H, Hkv, S, D, num_pages, page_size, max_pages, block_table,
                             table_stride, starts, counts, q_strides, q_out_strides, k_strides, v_strides, r, p, &bits,
                             &bits, err, kWhat))
    return rc;
  if (p.tokens == 0) return GHIP_OK;
  if (!k_cache || !v_cache || !k_cache_strides || !v_cache_strides)
    return set_error(err, GHIP_ERR_INVALID_ARG, "%s: null pointer", kWhat);
  const int64_t n[3] = {num_pages, Hkv, page_size}, es = elem(dtype);
  if (!take(p.kc, k_cache, k_cache_strides, n, es, &bits) || !take(p.vc, v_cache, v_cache_strides, n, es, &bits))
    return set_error(err, GHIP_ERR_UNSUPPORTED, "%s: negative strides", kWhat);
  return launch_rope(dtype, p, bits, 0, false, static_cast<hipStream_t>(stream), err, kWhat);
}

extern "C" int ghip_kv4_append_rope(int dtype, const void* q, void* q_out, const void* k, const void* v,
                                    const GHipKv4* k_cache, const GHipKv4* v_cache, int64_t B, int64_t H, int64_t Hkv,
                                    int64_t S, int64_t D, int64_t num_pages, int64_t page_size, int64_t max_pages,
                                    const int32_t* block_table, int64_t table_stride, const int32_t* starts,
                                    const int32_t* counts, const int64_t* q_strides, const int64_t* q_out_strides,
                                    const int64_t* k_strides, const int64_t* v_strides, const GHipRope* r, void* stream,
                                    GHipError* err) {
  static const char kWhat[] = "kv4_append_rope";
  rope::Params p{};
  uint64_t bits = 0, kv_bits = 0;
  if (D > 0 && D % kv4::kGroup != 0)
    return set_error(err, GHIP_ERR_UNSUPPORTED, "%s: needs a head dim that is a multiple of 32", kWhat);
  if (int rc = append_common(dtype, q, q_out, k, v, B, H, Hkv, S, D, num_pages, page_size, max_pages, block_table,
                             table_stride, starts, counts, q_strides, q_out_strides, k_strides, v_strides, r, p, &bits,
                             &kv_bits, err, kWhat))
    return rc;
  if (p.tokens == 0) return GHIP_OK;
  if (!k_cache || !v_cache || !k_cache->codes || !k_cache->scales || !v_cache->codes || !v_cache->scales)
    return set_error(err, GHIP_ERR_INVALID_ARG, "%s: null pointer", kWhat);
  const int64_t n[3] = {num_pages, Hkv, page_size};
  if (!take4(k_cache, n, D, p.kc, p.ks) || !take4(v_cache, n, D, p.vc, p.vs))
    return set_error(err, GHIP_ERR_UNSUPPORTED, kLayout4, kWhat);
  return launch_rope(dtype, p, bits, kv_bits, true, static_cast<hipStream_t>(stream), err, kWhat);
}

extern "C" int ghip_kv4_read(int dtype, const GHipKv4* k_cache, const GHipKv4* v_cache, void* k, void* v, int64_t B,
                             int64_t Hkv, int64_t S, int64_t D, int64_t num_pages, int64_t page_size, int64_t max_pages,
                             const int32_t* block_table, int64_t table_stride, const int32_t* lens,
                             const int64_t* k_strides, const int64_t* v_strides, void* stream, GHipError* err) {
  static const char kWhat[] = "kv4_read";
  if (D > 0 && D % kv4::kGroup != 0)
    return set_error(err, GHIP_ERR_UNSUPPORTED, "%s: needs a head dim that is a multiple of 32", kWhat);
  if (int rc = check_sizes(dtype, B, 0, Hkv, S, D, err, kWhat)) return rc;
  if (Hkv == 0) return set_error(err, GHIP_ERR_INVALID_ARG, "%s: bad sizes", kWhat);
  if (B == 0 || S == 0) return GHIP_OK;
  if (int rc = check_pages(num_pages, page_size, max_pages, block_table, table_stride, err, kWhat)) return rc;
  if (S > page_size * max_pages)
    return set_error(err, GHIP_ERR_INVALID_ARG, "%s: %lld tokens where a sequence's pages hold %lld", kWhat,
                     static_cast<long long>(S), static_cast<long long>(page_size * max_pages));
  if (!k || !v || !k_strides || !v_strides || !k_cache || !v_cache || !k_cache->codes || !k_cache->scales ||
      !v_cache->codes || !v_cache->scales)
    return set_error(err, GHIP_ERR_INVALID_ARG, "%s: null pointer", kWhat);
  rope::Read p{};
  const int64_t n[3] = {num_pages, Hkv, page_size}, rows[3] = {B, Hkv, S}, es = elem(dtype);
  if (!take4(k_cache, n, D, p.kc, p.ks) || !take4(v_cache, n, D, p.vc, p.vs))
    return set_error(err, GHIP_ERR_UNSUPPORTED, kLayout4, kWhat);
  uint64_t bits = 0;
  if (!take(p.k, k, k_strides, rows, es, &bits) || !take(p.v, v, v_strides, rows, es, &bits) || bits % 16 != 0)
    return set_error(err, GHIP_ERR_UNSUPPORTED, "%s: k and v must be 16-byte aligned with non-negative strides of whole 16 bytes",
                     kWhat);
  p.table = block_table;
  p.lens = lens;
  p.table_stride = table_stride;
  p.S = static_cast<int>(S); p.Hkv = static_cast<int>(Hkv); p.units = static_cast<int>(D / 8);
  p.num_pages = static_cast<int>(num_pages); p.page_size = static_cast<int>(page_size);
  const int64_t slots = rope::kThreads / p.units, blocks = (S + slots - 1) / slots;
  if (B > 65535 || Hkv > 65535 || blocks > rope::kMostGroups)
    return set_error(err, GHIP_ERR_UNSUPPORTED, "%s: problem too large", kWhat);
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(B), static_cast<unsigned>(Hkv));
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == GHIP_DTYPE_FLOAT32) hipLaunchKernelGGL((rope::read4_kernel<float>), grid, dim3(rope::kThreads), 0, s, p);
  else if (dtype == GHIP_DTYPE_FLOAT16) hipLaunchKernelGGL((rope::read4_kernel<f16_t>), grid, dim3(rope::kThreads), 0, s, p);
  else hipLaunchKernelGGL((rope::read4_kernel<bf16_t>), grid, dim3(rope::kThreads), 0, s, p);
  GHIP_CHECK(hipGetLastError(), err);
  return GHIP_OK;
}
