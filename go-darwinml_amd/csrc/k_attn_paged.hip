// A key-value cache in pages: the append of new tokens, and the attention of one new
// token a sequence over its pages (decoding).
//
//   o[b, h] = sum_j softmax_j(scale q[b, h].K_b[j]) V_b[j]   over the tokens j of sequence
//   b that its last token, at position len - 1, sees: j >= len - window or j < sinks
//
// where token j of sequence b lies in row j % page_size of page table[b][j /
// page_size].  No reference op (the reference keeps dense caches, which
// ghip_sdpa_fwd_masked_ws reads); bound by the bytes of K and V.
#include <algorithm>

#include "attn_paged.h"

namespace ghip {
namespace paged {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

struct Params : Common {
  const void* k;
  const void* v;
  int64_t k_sp, k_sh, k_st, v_sp, v_sh, v_st;  // byte strides of page, head, token
};

// 16 zero bytes: what lanes without a token load.
__device__ const uint4 kZero[1] = {};

template <typename T> struct Op;
template <> struct Op<float> {
  typedef float f8 __attribute__((ext_vector_type(8)));
  __device__ static f32x4 qk(const f8& a, const f8& b, f32x4 c) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
    return c;
  }
  using P = f32x4;
  __device__ static P pack(const f32x4& x) { return x; }
  __device__ static f32x4 pv(const P& a, const P& b, f32x4 c) {
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
    return c;
  }
};
template <> struct Op<bf16_t> {
  __device__ static f32x4 qk(const tile::bf16x8& a, const tile::bf16x8& b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  using P = s16x4;
  __device__ static P pack(const f32x4& x) {
    return __builtin_bit_cast(s16x4, make_uint2(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3])));
  }
  __device__ static f32x4 pv(const P& a, const P& b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(a, b, c, 0, 0, 0);
  }
};
template <> struct Op<f16_t> {
  __device__ static f32x4 qk(const tile::bf16x8& a, const tile::bf16x8& b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(tile::f16x8, a), __builtin_bit_cast(tile::f16x8, b), c,
                                                  0, 0, 0);
  }
  using P = s16x4;
  __device__ static P pack(const f32x4& x) {
    return __builtin_bit_cast(s16x4, make_uint2(pack_f16x2(x[0], x[1]), pack_f16x2(x[2], x[3])));
  }
  __device__ static f32x4 pv(const P& a, const P& b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4, a), __builtin_bit_cast(f16x4, b), c, 0, 0, 0);
  }
};

// A wave works alone on tiles of KT tokens: K and V rows come by per-lane DMA into
// two LDS stages, page numbers one tile further ahead by the same path, so one
// in-order counter (vmcnt) tells what has landed.  S^T = K Q^T with 16 tokens x 16
// heads a product and the softmaxed columns as the operand of O^T += V^T P^T, as in the
// prompt kernels.  SPLIT: the tiles of all sequences are dealt out evenly, whatever the
// lengths; a unit that several workers hold is joined by the second kernel.
// Bound by the bytes of K and V, each read once: bf16 D 128, 32 heads over 8, 64 sequences
// of 4096 tokens (1.07 GB) 203 us with the join (5.3 TB/s; pages with the heads of a token
// together 216 us, 5.0), 8 of 8192 (268 MB) 64 us, of which the loads at that rate are 50: the
// rest is the chain length - page number - row on cold caches (10 us) and the join.  (A
// stream of LDS loads of one large buffer reads 5.9 TB/s.)
template <typename T, int DP, bool SPLIT>
__global__ __launch_bounds__(64, 1) void attend_kernel(Params p) {
  constexpr int kEs = static_cast<int>(sizeof(T));
  constexpr int kRow = DP * kEs, kCh = kRow / 16;
  constexpr int KT = 8192 / kRow;              // 64, 32 or 16 tokens: 8 KiB of K and of V
  constexpr int kN = 8, kPer = 1024 / kRow;    // DMA instructions of a K (V) tile, rows of one
  constexpr int kTile = 8192;
  // f16 weights (and their sum, in every share alike) are raised by 2^7: beside a token that
  // takes nearly all of the softmax the others keep all their bits down to 2^-21 of it.
  constexpr float kUpLog2 = __is_same(T, f16_t) ? 7.f : 0.f;
  using O = Op<T>;
  using F = typename tile::Frag<T>::type;
  __shared__ __attribute__((aligned(1024))) char smem[2][2][kTile];
  __shared__ __attribute__((aligned(16))) int32_t page_lds[2][64];

  const int lane = threadIdx.x, g = lane >> 4, col = lane & 15;
  const int G = p.H / p.Hkv, blocks = (G + kHeads - 1) / kHeads, units = p.Hkv * blocks;
  const uint32_t la0 = tile::lds_addr(smem), pa0 = tile::lds_addr(page_lds);
  const float c = p.scale * 1.4426950408889634f;

  int b;
  int64_t at, end, begin;
  const Order<KT> order(p, SPLIT ? units : 0);
  if constexpr (SPLIT) {
    const int64_t per = order.share();
    at = blockIdx.x * per;
    end = min(order.total, at + per);
    if (at >= end) return;
    b = order.find(p, at, &begin);
  } else {
    b = blockIdx.x / units;
    begin = 0;
    at = end = 0;
  }
  const int64_t first = at;

  for (;;) {
    const Seen seen(p, SPLIT ? order.length(p, b) : p.lens[b]);
    const int nt = seen.tiles(KT), nst = seen.sink_tiles(KT);
    int unit, ta, te;
    if constexpr (SPLIT) {
      unit = static_cast<int>(quotient(at - begin, nt));
      ta = static_cast<int>(at - begin - static_cast<int64_t>(unit) * nt);
      te = static_cast<int>(min(static_cast<int64_t>(nt), ta + (end - at)));
    } else {
      unit = blockIdx.x % units;
      ta = 0;
      te = nt;
    }
    const int hk = unit / blocks, h0 = hk * G + (unit % blocks) * kHeads;
    const int heads = min(kHeads, (hk + 1) * G - h0);

    F qf[DP / 32];
    {
      const T* Q = static_cast<const T*>(p.q) + b * p.q_sb + (h0 + col) * p.q_sh;
#pragma unroll
      for (int s = 0; s < DP / 32; ++s) {
        const int d = 32 * s + 8 * g;
        F f{};
        if (col < heads && d < p.D) {
          if constexpr (kEs == 2) {
            f = *reinterpret_cast<const F*>(Q + d);
          } else {
            const float4 lo = *reinterpret_cast<const float4*>(Q + d);
            const float4 hi = d + 4 < p.D ? *reinterpret_cast<const float4*>(Q + d + 4) : make_float4(0.f, 0.f, 0.f, 0.f);
            f = F{lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
          }
        }
        qf[s] = f;
      }
    }
    const char* K = static_cast<const char*>(p.k) + hk * p.k_sh;
    const char* V = static_cast<const char*>(p.v) + hk * p.v_sh;
    const int32_t* table = p.table + b * p.table_stride;

    // Tile t's first token, and the rows of it that hold visible tokens.
    auto token0 = [&](int t) { return t < nst ? t * KT : (seen.lo & ~15) + (t - nst) * KT; };
    auto issue_pages = [&](int t, int slot) {
      const int entry = min((token0(t) + (lane & (KT - 1))) / p.page_size, p.max_pages - 1);
      tile::load4(table + entry, pa0 + slot * 256);
    };
    // The DMA of tile t, its page numbers landed; returns its rows that hold a token.
    auto issue = [&](int t, int slot) -> uint64_t {
      const int tok = token0(t) + (lane & (KT - 1));
      const int page = page_lds[slot][lane];
      const int off = tok % p.page_size;
      const bool ok = (t < nst ? tok < seen.ns : tok >= seen.lo && tok < seen.len) && page >= 0 && page < p.num_pages;
      const uint64_t rows = __builtin_amdgcn_ballot_w64(ok);
      const uint32_t la = la0 + slot * (2 * kTile);
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const int r = i * kPer + lane / kCh;
        const int ch = (lane % kCh) ^ tile::swz<kCh>(r);
        const int64_t pg = __shfl(page, r, 64), of = __shfl(off, r, 64);
        const bool there = ((rows >> r) & 1) && ch * 16 < p.D * kEs;
        const char* zero = reinterpret_cast<const char*>(kZero);
        tile::load16(there ? K + pg * p.k_sp + of * p.k_st + ch * 16 : zero, la + i * 1024);
        tile::load16(there ? V + pg * p.v_sp + of * p.v_st + ch * 16 : zero, la + kTile + i * 1024);
      }
      return rows;
    };

    f32x4 o[DP / 16];
#pragma unroll
    for (int db = 0; db < DP / 16; ++db) o[db] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;

    // The order of the DMA is pages(j + 1), K and V(j) (the first two tiles' pages together).
    const int n = te - ta;
    auto tile_of = [&](int j) { return ta + j; };
    uint64_t rows0 = 0, rows1 = 0;  // of tiles j and j + 1
    if (n > 0) {
      issue_pages(tile_of(0), 0);
      if (n > 1) issue_pages(tile_of(1), 1);
      wait_vm<0>();
      rows0 = issue(tile_of(0), 0);
      if (n > 1) {
        if (n > 2) issue_pages(tile_of(2), 0);
        rows1 = issue(tile_of(1), 1);
      }
    }
    for (int j = 0; j < n; ++j) {
      // Everything older than tile j + 1's own DMA has landed (and its successor's pages).
      if (j + 2 < n) wait_vm<2 * kN + 1>();
      else if (j + 1 < n) wait_vm<2 * kN>();
      else wait_vm<0>();
      const char* sk = smem[j & 1][0];
      const char* sv = smem[j & 1][1];
      f32x4 x[KT / 16];
#pragma unroll
      for (int i = 0; i < KT / 16; ++i) {
        x[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        const int r = 16 * i + col;
#pragma unroll
        for (int s = 0; s < DP / 32; ++s) {
          F f;
          if constexpr (kEs == 2) {
            f = *reinterpret_cast<const F*>(sk + r * kRow + (((4 * s + g) ^ tile::swz<kCh>(r)) << 4));
          } else {
            const float4 lo = *reinterpret_cast<const float4*>(sk + r * kRow + (((8 * s + 2 * g) ^ tile::swz<kCh>(r)) << 4));
            const float4 hi = *reinterpret_cast<const float4*>(sk + r * kRow + (((8 * s + 2 * g + 1) ^ tile::swz<kCh>(r)) << 4));
            f = F{lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
          }
          x[i] = O::qk(f, qf[s], x[i]);
        }
      }
      // x[i][v]: row 16 i + 4 g + v, head col.
      if (rows0 != ~0ull) {
#pragma unroll
        for (int i = 0; i < KT / 16; ++i) {
          const uint32_t bits = static_cast<uint32_t>(rows0 >> (16 * i + 4 * g));
#pragma unroll
          for (int v = 0; v < 4; ++v) x[i][v] = (bits >> v) & 1 ? x[i][v] : -INFINITY;
        }
      }
      float mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < KT / 16; ++i) mx = fmaxf(fmaxf(fmaxf(x[i][0], x[i][1]), fmaxf(x[i][2], x[i][3])), mx);
      mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
      mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
      if (__builtin_amdgcn_ballot_w64((mx - m) * c > 8.f)) {  // the maximum may trail by 2^8
        const float mnew = fmaxf(m, mx);
        const float alpha = mnew == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - mnew) * c);
        m = mnew;
        l *= alpha;
#pragma unroll
        for (int db = 0; db < DP / 16; ++db)
#pragma unroll
          for (int v = 0; v < 4; ++v) o[db][v] *= alpha;
      }
      const float nb = m == -INFINITY ? 0.f : kUpLog2 - m * c;
#pragma unroll
      for (int i = 0; i < KT / 16; ++i) {
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          x[i][v] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i][v], c, nb));
          l += x[i][v];
        }
        // The weights, at most 2^8 (f16: 2^15), are rounded for the product with V only: half a
        // step of the type beside V's own rounding; their sum above is not.
        const typename O::P pf = O::pack(x[i]);
#pragma unroll
        for (int db = 0; db < DP / 16; ++db) {
          typename O::P vf;
          if constexpr (kEs == 2) {
            const int r = 16 * i + 4 * g + (col >> 2), cc = 16 * db + 4 * (lane & 3);
            const char* a = sv + r * kRow + (((cc >> 3) ^ tile::swz<kCh>(r)) << 4) + (cc & 7) * 2;
            vf = __builtin_bit_cast(typename O::P, __builtin_amdgcn_ds_read_tr16_b64_v4bf16((GHIP_LDS tile::bf16x4*)(a)));
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int r = 16 * i + 4 * g + e, cc = 16 * db + col;
              vf[e] = *reinterpret_cast<const float*>(sv + r * kRow + (((cc >> 2) ^ tile::swz<kCh>(r)) << 4) + (cc & 3) * 4);
            }
          }
          o[db] = O::pv(vf, pf, o[db]);
        }
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the stage has been read
      rows0 = rows1;
      if (j + 2 < n) {
        wait_vm<2 * kN>();  // its page numbers
        if (j + 3 < n) issue_pages(tile_of(j + 3), (j + 1) & 1);
        rows1 = issue(tile_of(j + 2), j & 1);
      }
    }

    // o[db][v] is d = 16 db + 4 g + v of head col.
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;  // no token seen: zeros
    if (col < heads) {
      if (ta == 0 && te == nt) {
        T* out = static_cast<T*>(p.o) + b * p.o_sb + (h0 + col) * p.o_sh + 4 * g;
#pragma unroll
        for (int db = 0; db < DP / 16; ++db)
          if (16 * db + 4 * g < p.D)
            tile::store4(out + 16 * db, o[db][0] * inv, o[db][1] * inv, o[db][2] * inv, o[db][3] * inv);
      } else {
        const int64_t r = (2 * static_cast<int64_t>(blockIdx.x) + (at == first ? 0 : 1)) * p.unit_heads + col;
        float* out = p.part_o + r * p.D + 4 * g;
#pragma unroll
        for (int db = 0; db < DP / 16; ++db)
          if (16 * db + 4 * g < p.D)
            tile::store4(out + 16 * db, o[db][0] * inv, o[db][1] * inv, o[db][2] * inv, o[db][3] * inv);
        if (g == 0) p.part_lse[r] = l > 0.f || l != l ? m * c + __builtin_amdgcn_logf(l) : -INFINITY;
      }
    }
    if constexpr (!SPLIT) {
      return;
    } else {
      at += te - ta;
      if (at >= end) return;
      if (at - begin >= static_cast<int64_t>(nt) * units) b = order.find(p, at, &begin);
    }
  }
}

// Joins the shares of units that several workers hold; a workgroup a (sequence, head).
// Sequences without a visible token, which no worker holds, get zeros.
// Bound by the latency of lengths, then shares: 4.8 us for 8 x 32 heads, 6 us for 64 x 32.
template <typename T, int DP>
__global__ __launch_bounds__(256) void join_kernel(Params p) {
  constexpr int KT = 8192 / (DP * static_cast<int>(sizeof(T)));
  const int G = p.H / p.Hkv, blocks = (G + kHeads - 1) / kHeads, units = p.Hkv * blocks;
  const int row = blockIdx.x, b = row / p.H, h = row % p.H, hk = h / G;
  const int unit = hk * blocks + (h - hk * G) / kHeads, hd = (h - hk * G) % kHeads;
  const Order<KT> order(p, units);
  const int nt = Seen(p, order.length(p, b)).tiles(KT);
  const int64_t per = order.share(), u0 = order.begin(p, b) + static_cast<int64_t>(unit) * nt;
  const int w0 = static_cast<int>(quotient(u0, per));
  const int n = nt == 0 ? 0 : static_cast<int>(quotient(u0 + nt - 1, per)) - w0 + 1;
  // The unit's share in worker w0 + i: its first piece, but for a worker that began before.
  join_shares<T, DP, 256, 1, 4>(p, static_cast<T*>(p.o) + b * p.o_sb + h * p.o_sh, n, [&](int i) {
    return (2 * static_cast<int64_t>(w0 + i) + (i == 0 && u0 != w0 * per ? 1 : 0)) * p.unit_heads + hd;
  });
}

template <typename T, int DP>
static void launch_d(const Params& p, hipStream_t s) {
  const int G = p.H / p.Hkv, units = p.Hkv * ((G + kHeads - 1) / kHeads);
  if (p.part_o) {
    hipLaunchKernelGGL((attend_kernel<T, DP, true>), dim3(kWorkers), dim3(64), 0, s, p);
    hipLaunchKernelGGL((join_kernel<T, DP>), dim3(static_cast<unsigned>(p.B * p.H)), dim3(256), 0, s, p);
  } else {
    hipLaunchKernelGGL((attend_kernel<T, DP, false>), dim3(static_cast<unsigned>(p.B * units)), dim3(64), 0, s, p);
  }
}
template <typename T>
static void launch(const Params& p, hipStream_t s) {
  if (p.D <= 64) launch_d<T, 64>(p, s);
  else if (p.D <= 128) launch_d<T, 128>(p, s);
  else if constexpr (sizeof(T) == 2) launch_d<T, 256>(p, s);
}

// ---------------------------------------------------------------- append
struct Append {
  const char* k;
  const char* v;
  char* kc;
  char* vc;
  const int32_t* table;
  const int32_t* starts;
  const int32_t* counts;
  int64_t k_sb, k_sh, k_ss, v_sb, v_sh, v_ss;      // byte strides of batch, head, token
  int64_t kc_sp, kc_sh, kc_st, vc_sp, vc_sh, vc_st;  // of page, head, row
  int64_t table_stride;
  int S, Hkv, chunks, num_pages, page_size, max_pages;
};

// One thread moves the same U-byte piece of one token's K and V; the pieces of a row,
// then the heads, are neighbours.
// Bound by the bytes: 8 prompts of up to 1024 tokens, 8 heads of 128 in bf16 (38 MB read and
// written) 8.5 us, 4.4 TB/s, near a large copy's 4.9; 16 single tokens 2.6 us, the launch.
template <typename U>
__global__ __launch_bounds__(256) void append_kernel(Append p) {
  const int64_t n = static_cast<int64_t>(p.S) * p.Hkv * p.chunks;
  const int64_t e = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (e >= n) return;
  const int b = blockIdx.y;
  const uint32_t rowi = static_cast<uint32_t>(e / p.chunks), ch = static_cast<uint32_t>(e - static_cast<int64_t>(rowi) * p.chunks);
  const uint32_t i = rowi / p.Hkv, h = rowi - i * p.Hkv;
  if (p.counts && static_cast<int>(i) >= p.counts[b]) return;
  const int64_t pos = static_cast<int64_t>(p.starts[b]) + i;
  if (pos < 0 || pos >= static_cast<int64_t>(p.max_pages) * p.page_size) return;
  const uint32_t entry = static_cast<uint32_t>(pos / p.page_size), at = static_cast<uint32_t>(pos - static_cast<int64_t>(entry) * p.page_size);
  const int64_t src = static_cast<int64_t>(sizeof(U)) * ch;
  const U kx = *reinterpret_cast<const U*>(p.k + b * p.k_sb + h * p.k_sh + i * p.k_ss + src);
  const U vx = *reinterpret_cast<const U*>(p.v + b * p.v_sb + h * p.v_sh + i * p.v_ss + src);
  const int page = p.table[b * p.table_stride + entry];
  if (page < 0 || page >= p.num_pages) return;
  *reinterpret_cast<U*>(p.kc + page * p.kc_sp + h * p.kc_sh + at * p.kc_st + src) = kx;
  *reinterpret_cast<U*>(p.vc + page * p.vc_sp + h * p.vc_sh + at * p.vc_st + src) = vx;
}

}  // namespace paged
}  // namespace ghip

using namespace ghip;

// No workspace, so a wave for each unit: caches of at most 4 tiles a sequence, or 12 with
// 512 units or more.  (More units hide the two kernels' latencies, not the second launch.)
// bf16 D 128, sequences of one length, us a call in a graph, split / unsplit:
//   units      4 tiles      6           8           12          16          24
//   64         11.0 / 10.3  11.3 / 13.7  11.3 / 17.2  11.7 / 23.8
//   256        12.9 / 10.4  13.8 / 13.9  14.7 / 18.3  19.1 / 25.5
//   512        16.6 / 11.7  21.1 / 16.2  24.3 / 20.4  30.2 / 28.4  35.9 / 36.5  46.9 / 52.5
//   1024       26.7 / 15.7  32.2 / 21.3  38.2 / 26.6  49.7 / 37.6  60.4 / 46.9  97.8 / 81.9
// (As many units as workers and more fill the card unsplit when the lengths are alike; the
// rule, which does not know them, splits from 13 tiles on: one sequence of the whole cache
// among short ones would keep the others waiting.)
extern "C" int64_t ghip_sdpa_paged_workspace_bytes(int dtype, int64_t B, int64_t H, int64_t Hkv, int64_t D,
                                                   int64_t page_size, int64_t max_pages) {
  if (B <= 0 || Hkv <= 0 || H < Hkv || D <= 0 || D > 256 || page_size <= 0 || max_pages <= 0) return 0;
  const int64_t heads = H / Hkv, units = B * Hkv * ((heads + paged::kHeads - 1) / paged::kHeads);
  const int64_t row = (D <= 64 ? 64 : D <= 128 ? 128 : 256) * (dtype == GHIP_DTYPE_FLOAT32 ? 4 : 2);
  const double tokens = static_cast<double>(page_size) * static_cast<double>(max_pages);
  if (tokens * row <= 8192. * (units >= 512 ? 12 : 4)) return 0;
  return 2 * static_cast<int64_t>(paged::kWorkers) * std::min<int64_t>(paged::kHeads, heads) * (D + 1) * 4;
}

extern "C" int ghip_sdpa_paged(int dtype, const void* q, const void* k_cache, const void* v_cache, void* o, int64_t B,
                               int64_t H, int64_t Hkv, int64_t D, int64_t num_pages, int64_t page_size,
                               int64_t max_pages, const int32_t* block_table, int64_t table_stride,
                               const int32_t* lens, const int64_t* q_strides, const int64_t* k_strides,
                               const int64_t* v_strides, const int64_t* o_strides, int64_t window, int64_t sinks,
                               float scale, void* workspace, int64_t workspace_bytes, void* stream, GHipError* err) {
  static const char kWhat[] = "sdpa_paged";
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
  if (D % (f32 ? 4 : 8) != 0 || D > (f32 ? 128 : 256))
    return set_error(err, GHIP_ERR_UNSUPPORTED,
                     "%s: needs a head dim that is a multiple of 8 up to 256 (float32: of 4 up to 128)", kWhat);
  constexpr int64_t kMost = int64_t{1} << 30;
  if (num_pages > kMost || page_size > kMost || max_pages > kMost || page_size * max_pages > kMost / 2 ||
      B > kMost || H > kMost || B * H > tile::kMostGroups)
    return set_error(err, GHIP_ERR_UNSUPPORTED,
                     "%s: at most 2^30 pages, 2^29 tokens of a sequence and fewer than 2^24 heads of all sequences", kWhat);
  if (B == 0) return GHIP_OK;
  if (!q || !o || !lens || !q_strides || !k_strides || !v_strides || !o_strides || !k_cache || !v_cache || !block_table)
    return set_error(err, GHIP_ERR_INVALID_ARG, "%s: null pointer", kWhat);
  if (num_pages == 0 || max_pages == 0)
    return set_error(err, GHIP_ERR_INVALID_ARG, "%s: a cache without pages", kWhat);
  if (table_stride < 0) return set_error(err, GHIP_ERR_INVALID_ARG, "%s: negative table stride", kWhat);
  const int64_t es = f32 ? 4 : 2;
  auto al = [](const void* ptr, uintptr_t a) { return (reinterpret_cast<uintptr_t>(ptr) & (a - 1)) == 0; };
  bool ok = al(q, 16) && al(k_cache, 16) && al(v_cache, 16) && al(o, 4 * es);
  // (An axis of one entry may have any stride that is not negative.)
  auto whole = [](int64_t stride, int64_t n, int64_t of) { return stride >= 0 && (n <= 1 || stride % of == 0); };
  const int64_t cache[3] = {num_pages, Hkv, page_size}, rows[2] = {B, H};
  for (int i = 0; i < 3; ++i) ok = ok && whole(k_strides[i], cache[i], 16 / es) && whole(v_strides[i], cache[i], 16 / es);
  for (int i = 0; i < 2; ++i) ok = ok && whole(q_strides[i], rows[i], 16 / es) && whole(o_strides[i], rows[i], 4);
  if (!ok)
    return set_error(err, GHIP_ERR_UNSUPPORTED,
                     "%s: q and the caches must be 16-byte aligned with non-negative strides of whole 16 bytes, o "
                     "aligned to 4 elements with strides of whole 4", kWhat);
  paged::Params p{};
  p.q = q; p.k = k_cache; p.v = v_cache; p.o = o;
  p.table = block_table; p.lens = lens;
  p.q_sb = q_strides[0]; p.q_sh = q_strides[1]; p.o_sb = o_strides[0]; p.o_sh = o_strides[1];
  p.k_sp = k_strides[0] * es; p.k_sh = k_strides[1] * es; p.k_st = k_strides[2] * es;
  p.v_sp = v_strides[0] * es; p.v_sh = v_strides[1] * es; p.v_st = v_strides[2] * es;
  p.table_stride = table_stride;
  p.B = static_cast<int>(B); p.H = static_cast<int>(H); p.Hkv = static_cast<int>(Hkv); p.D = static_cast<int>(D);
  p.num_pages = static_cast<int>(num_pages); p.page_size = static_cast<int>(page_size);
  p.max_pages = static_cast<int>(max_pages);
  p.window = static_cast<int>(window == 0 || window > kMost ? kMost : window);
  p.sinks = static_cast<int>(sinks > kMost ? kMost : sinks);
  p.scale = scale;
  p.unit_heads = static_cast<int>(std::min<int64_t>(paged::kHeads, H / Hkv));
  const int64_t need = workspace ? ghip_sdpa_paged_workspace_bytes(dtype, B, H, Hkv, D, page_size, max_pages) : 0;
  if (need > 0) {
    if (workspace_bytes < need)
      return set_error(err, GHIP_ERR_INVALID_ARG, "%s: workspace of %lld bytes, %lld needed", kWhat,
                       static_cast<long long>(workspace_bytes), static_cast<long long>(need));
    if (!al(workspace, 16)) return set_error(err, GHIP_ERR_INVALID_ARG, "%s: workspace must be 16-byte aligned", kWhat);
    p.part_o = static_cast<float*>(workspace);
    p.part_lse = p.part_o + 2 * static_cast<int64_t>(paged::kWorkers) * p.unit_heads * D;
  }
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (f32) paged::launch<float>(p, s);
  else if (dtype == GHIP_DTYPE_FLOAT16) paged::launch<f16_t>(p, s);
  else paged::launch<bf16_t>(p, s);
  GHIP_CHECK(hipGetLastError(), err);
  return GHIP_OK;
}

extern "C" int ghip_kv_append(int elem_bytes, const void* k, const void* v, void* k_cache, void* v_cache, int64_t B,
                              int64_t S, int64_t Hkv, int64_t D, int64_t num_pages, int64_t page_size,
                              int64_t max_pages, const int32_t* block_table, int64_t table_stride,
                              const int32_t* starts, const int32_t* counts, const int64_t* k_strides,
                              const int64_t* v_strides, const int64_t* k_cache_strides,
                              const int64_t* v_cache_strides, void* stream, GHipError* err) {
  static const char kWhat[] = "kv_append";
  if (elem_bytes != 1 && elem_bytes != 2 && elem_bytes != 4 && elem_bytes != 8)
    return set_error(err, GHIP_ERR_UNSUPPORTED, "%s: elements of 1, 2, 4 or 8 bytes", kWhat);
  if (B < 0 || S < 0 || Hkv <= 0 || D <= 0 || num_pages < 0 || page_size <= 0 || max_pages < 0)
    return set_error(err, GHIP_ERR_INVALID_ARG, "%s: bad sizes", kWhat);
  constexpr int64_t kMost = int64_t{1} << 30;
  if (num_pages > kMost || page_size > kMost || max_pages > kMost || page_size * max_pages > kMost || B > 65535 ||
      S > kMost || Hkv > kMost || S * Hkv > kMost || D > (1 << 20))
    return set_error(err, GHIP_ERR_UNSUPPORTED, "%s: problem too large", kWhat);
  if (B == 0 || S == 0) return GHIP_OK;
  if (!k || !v || !k_cache || !v_cache || !block_table || !starts || !k_strides || !v_strides || !k_cache_strides ||
      !v_cache_strides)
    return set_error(err, GHIP_ERR_INVALID_ARG, "%s: null pointer", kWhat);
  if (num_pages == 0 || max_pages == 0)
    return set_error(err, GHIP_ERR_INVALID_ARG, "%s: a cache without pages", kWhat);
  if (table_stride < 0) return set_error(err, GHIP_ERR_INVALID_ARG, "%s: negative table stride", kWhat);
  // The widest unit that every row and stride (of an axis of several entries) is a multiple of.
  uint64_t bits = reinterpret_cast<uint64_t>(k) | reinterpret_cast<uint64_t>(v) | reinterpret_cast<uint64_t>(k_cache) |
                  reinterpret_cast<uint64_t>(v_cache) | static_cast<uint64_t>(D * elem_bytes);
  const int64_t fresh[3] = {B, Hkv, S}, cache[3] = {num_pages, Hkv, page_size};
  for (const int64_t* s : {k_strides, v_strides, k_cache_strides, v_cache_strides})
    for (int i = 0; i < 3; ++i) {
      if (s[i] < 0) return set_error(err, GHIP_ERR_UNSUPPORTED, "%s: negative strides", kWhat);
      if ((s == k_strides || s == v_strides ? fresh : cache)[i] > 1) bits |= static_cast<uint64_t>(s[i] * elem_bytes);
    }
  if (bits % elem_bytes) return set_error(err, GHIP_ERR_INVALID_ARG, "%s: pointers are not aligned to elements", kWhat);
  const int unit = bits % 16 == 0 ? 16 : bits % 8 == 0 ? 8 : bits % 4 == 0 ? 4 : bits % 2 == 0 ? 2 : 1;
  const int64_t es = elem_bytes;
  paged::Append p{};
  p.k = static_cast<const char*>(k); p.v = static_cast<const char*>(v);
  p.kc = static_cast<char*>(k_cache); p.vc = static_cast<char*>(v_cache);
  p.table = block_table; p.starts = starts; p.counts = counts;
  p.k_sb = k_strides[0] * es; p.k_sh = k_strides[1] * es; p.k_ss = k_strides[2] * es;
  p.v_sb = v_strides[0] * es; p.v_sh = v_strides[1] * es; p.v_ss = v_strides[2] * es;
  p.kc_sp = k_cache_strides[0] * es; p.kc_sh = k_cache_strides[1] * es; p.kc_st = k_cache_strides[2] * es;
  p.vc_sp = v_cache_strides[0] * es; p.vc_sh = v_cache_strides[1] * es; p.vc_st = v_cache_strides[2] * es;
  p.table_stride = table_stride;
  p.S = static_cast<int>(S); p.Hkv = static_cast<int>(Hkv); p.chunks = static_cast<int>(D * es / unit);
  p.num_pages = static_cast<int>(num_pages); p.page_size = static_cast<int>(page_size);
  p.max_pages = static_cast<int>(max_pages);
  const int64_t n = S * Hkv * p.chunks;
  if (n > tile::kMostGroups * 256) return set_error(err, GHIP_ERR_UNSUPPORTED, "%s: problem too large", kWhat);
  const dim3 grid(static_cast<unsigned>((n + 255) / 256), static_cast<unsigned>(B));
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (unit == 16) hipLaunchKernelGGL((paged::append_kernel<uint4>), grid, dim3(256), 0, s, p);
  else if (unit == 8) hipLaunchKernelGGL((paged::append_kernel<uint2>), grid, dim3(256), 0, s, p);
  else if (unit == 4) hipLaunchKernelGGL((paged::append_kernel<uint32_t>), grid, dim3(256), 0, s, p);
  else if (unit == 2) hipLaunchKernelGGL((paged::append_kernel<uint16_t>), grid, dim3(256), 0, s, p);
  else hipLaunchKernelGGL((paged::append_kernel<uint8_t>), grid, dim3(256), 0, s, p);
  GHIP_CHECK(hipGetLastError(), err);
  return GHIP_OK;
}
