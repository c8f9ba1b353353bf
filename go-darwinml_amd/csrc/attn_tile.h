// What the windowed attention kernels share (gfx950): LDS tiles of K / V / Q / dO rows
// filled by DMA, the MFMA operands read from them, and the rule of which key a query
// sees.  One set of index formulas serves bf16, f16 and fp32:
//
//   * operands are "fragments" of 8 values a lane: lane l of a wave (c = l % 32, h =
//     l / 32) holds values 8h .. 8h + 7 of a 16-step contraction for row (or column) c.
//     16-bit types: one v_mfma_f32_32x32x16; fp32: eight v_mfma_f32_32x32x2_f32, the
//     e-th of them contracting steps e (lane half 0) and 8 + e (lane half 1);
//   * accumulators: register v of lane (c, h) is row 8 (v / 4) + 4 h + v % 4, column c.
//     Registers 8 s .. 8 s + 7 are thereby a fragment of a contraction over the rows in
//     the order 16 s + 4 h + {0..3}, 16 s + 8 + 4 h + {0..3}: scores enter the next
//     product without leaving registers, and frag_tr reads the other operand in that
//     same order.
#pragma once

#include "common.h"

#define GHIP_LDS __attribute__((address_space(3)))

namespace ghip {
namespace tile {

// Workgroups of 256 threads that one launch holds (HIP: fewer than 2^32 threads).
constexpr int64_t kMostGroups = (int64_t{1} << 24) - 1;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

template <typename T> struct Frag { using type = bf16x8; };  // 16-bit: raw bits
template <> struct Frag<float> { using type = f32x8; };

template <typename T>
__device__ __forceinline__ f32x16 mma(const typename Frag<T>::type& a, const typename Frag<T>::type& b, f32x16 c) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
    return c;
  } else if constexpr (__is_same(T, f16_t)) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
}

// Rounds registers 8 s .. 8 s + 7 of an accumulator to the operands' type (fp32: none).
template <typename T>
__device__ __forceinline__ typename Frag<T>::type pack(const f32x16& x, int s) {
  if constexpr (sizeof(T) == 4) {
    f32x8 r;
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = x[8 * s + e];
    return r;
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (__is_same(T, f16_t)) w[i] = pack_f16x2(x[8 * s + 2 * i], x[8 * s + 2 * i + 1]);
      else w[i] = pack_bf16x2(x[8 * s + 2 * i], x[8 * s + 2 * i + 1]);
    }
    return __builtin_bit_cast(bf16x8, make_uint4(w[0], w[1], w[2], w[3]));
  }
}

// Value e of a fragment, widened.
template <typename T>
__device__ __forceinline__ float value(const typename Frag<T>::type& f, int e) {
  if constexpr (sizeof(T) == 4) return f[e];
  else if constexpr (__is_same(T, f16_t)) return static_cast<float>(__builtin_bit_cast(f16x8, f)[e]);
  else return static_cast<float>(f[e]);
}

__device__ __forceinline__ f32x16 splat(float x) {
  f32x16 r;
#pragma unroll
  for (int v = 0; v < 16; ++v) r[v] = x;
  return r;
}

// LDS tiles are [rows][DP] values, 16-byte chunk j of row r at slot j ^ swz(r).  With
// r's bits r0 .. r3: any 8 aligned consecutive rows differ in slot bits 0..2 and 16 in
// bits 0..3 (the ds_read_b128 of frag_row), and the 4 consecutive rows of a transpose
// read (frag_tr: pairs or quads of chunks) differ in bits 1..2 and in bits 2..3, so
// both kinds of read of one tile spread over the banks.
template <int NCH>
__device__ __forceinline__ int swz(int r) {
  return (((r >> 2) & 1) | (r & 2) | (((r ^ (r >> 1)) & 1) << 2) | ((((r >> 1) ^ (r >> 3)) & 1) << 3)) & (NCH - 1);
}

template <typename T, int DP>
struct Tile {
  static constexpr int kEs = static_cast<int>(sizeof(T));
  static constexpr int kRow = DP * kEs;      // bytes of a row
  static constexpr int kCh = kRow / 16;      // 16-byte chunks of a row
  using F = typename Frag<T>::type;

  // Values 16 s + 8 h .. + 8 of row lane % 32 of the 32 rows at `lds` (A operand whose
  // rows are the tile's rows); `lds` at a multiple of 16 rows.
  __device__ __forceinline__ static F frag_row(const char* lds, int s, int lane) {
    const int r = lane & 31, h = lane >> 5, f = swz<kCh>(r);
    if constexpr (kEs == 2) {
      return *reinterpret_cast<const F*>(lds + (r * kRow + (((2 * s + h) ^ f) << 4)));
    } else {
      const float4 lo = *reinterpret_cast<const float4*>(lds + (r * kRow + (((4 * s + 2 * h) ^ f) << 4)));
      const float4 hi = *reinterpret_cast<const float4*>(lds + (r * kRow + (((4 * s + 2 * h + 1) ^ f) << 4)));
      return F{lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    }
  }
  // Column 32 db + lane % 32 of rows 4 h + {0..3} and 8 + 4 h + {0..3} of the 16 rows at
  // `lds` (A operand of the transposed tile).  16-bit: ds_read_b64_tr_b16 hands lane j of
  // each 16-lane group element j of the four 4-element rows that the group points at.
  __device__ __forceinline__ static F frag_tr(const char* lds, int db, int lane) {
    const int h = lane >> 5;
    if constexpr (kEs == 2) {
      const int r = 4 * h + ((lane & 15) >> 2);
      const int col = db * 32 + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
      const char* p0 = lds + (r * kRow + (((col >> 3) ^ swz<kCh>(r)) << 4) + (col & 7) * 2);
      const char* p1 = lds + (r * kRow + (((col >> 3) ^ swz<kCh>(r + 8)) << 4) + (col & 7) * 2) + 8 * kRow;
      const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((GHIP_LDS bf16x4*)(p0));
      const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((GHIP_LDS bf16x4*)(p1));
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    } else {
      F r;
      const int col = db * 32 + (lane & 31);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int row = 8 * (e >> 2) + 4 * h + (e & 3);
        r[e] = *reinterpret_cast<const float*>(lds + (row * kRow + (((col >> 2) ^ swz<kCh>(row)) << 4) + (col & 3) * 4));
      }
      return r;
    }
  }
  // Values 16 s + 8 h .. + 8 of a row in global memory (B operand whose columns are
  // rows); zeros past D and where !ok.
  __device__ __forceinline__ static F frag_global(const T* row, int s, int h, int D, bool ok) {
    const int d = 16 * s + 8 * h;
    F r{};
    if (ok && d < D) {
      if constexpr (kEs == 2) {
        r = *reinterpret_cast<const F*>(row + d);
      } else {
        const float4 lo = *reinterpret_cast<const float4*>(row + d);
        const float4 hi = d + 4 < D ? *reinterpret_cast<const float4*>(row + d + 4) : make_float4(0.f, 0.f, 0.f, 0.f);
        r = F{lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
      }
    }
    return r;
  }
};

// use(j, read(j)) for j < N with several reads in flight: left alone, the compiler reads an
// operand from LDS right before the instruction that takes it and waits for each (1200
// cycles for 8 matrix instructions that take 256).
// Rows of 512 bytes leave registers for fewer.
template <int ROW, typename F, int N, typename Read, typename Use>
__device__ __forceinline__ void pipelined(const Read& read, const Use& use) {
  constexpr int kAhead = ROW > 256 ? 2 : 4, A = N < kAhead ? N : kAhead;
  F a[A];
#pragma unroll
  for (int j = 0; j < A; ++j) a[j] = read(j);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int j = 0; j < N; ++j) {
    use(j, a[j % A]);
    if (j + A < N) a[j % A] = read(j + A);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// The fragments are there: the compiler's wait for their loads falls here.  Left to their
// first use, inside the loop over the tiles, that wait would also be one for each next
// tile's DMA (both count in vmcnt).
template <typename F, int N>
__device__ __forceinline__ void settle(F (&f)[N]) {
#pragma unroll
  for (int s = 0; s < N; ++s) asm volatile("" : "+v"(f[s]));
}

// Four consecutive values of an accumulator column, rounded once.
__device__ __forceinline__ void store4(float* p, float a, float b, float c, float d) {
  *reinterpret_cast<float4*>(p) = make_float4(a, b, c, d);
}
__device__ __forceinline__ void store4(bf16_t* p, float a, float b, float c, float d) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(a, b), pack_bf16x2(c, d));
}
__device__ __forceinline__ void store4(f16_t* p, float a, float b, float c, float d) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_f16x2(a, b), pack_f16x2(c, d));
}

// 16 bytes per lane from buffer offset voff to LDS byte address la + lane * 16 (la
// wave-uniform).  m0 is set and used inside this one statement; nothing else in these
// kernels reads it.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void dma16(i32x4 rsrc, uint32_t la, uint32_t voff) {
  asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               ::"s"(la), "v"(voff), "s"(rsrc) : "memory", "m0");
}
// The same from per-lane addresses, 16 or 4 bytes a lane (LDS address la + lane * 16, * 4).
__device__ __forceinline__ void load16(const void* p, uint32_t la) {
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(la), "v"(p) : "memory", "m0");
}
__device__ __forceinline__ void load4(const void* p, uint32_t la) {
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dword %1, off" ::"s"(la), "v"(p) : "memory", "m0");
}
#pragma clang diagnostic pop

constexpr uint32_t kPastEnd = 0x80000000u;  // past every descriptor's records: loads zeros

// A matrix in global memory whose rows are loaded as tiles; rows from `rows` on read zeros.
struct Rows {
  const char* base;
  uint32_t step;  // bytes from row to row (the host checks 64 of them against 2 GiB)
  int rows;
};

// The wave's share of the DMA of ROWS-row tiles (NW waves): per-lane offsets, computed once.
template <typename T, int DP, int ROWS, int NW>
struct Loader {
  static constexpr int kN = ROWS * DP * static_cast<int>(sizeof(T)) / 1024 / NW;
  static constexpr int kPer = 1024 / (DP * static_cast<int>(sizeof(T)));  // rows of one DMA instruction
  static_assert(kN >= 1, "a wave loads at least 1 KiB of a tile");
  uint32_t off[kN];
  uint32_t row_bytes;
  __device__ __forceinline__ void init(uint32_t step, int D, int wave, int lane) {
    constexpr int NCH = DP * static_cast<int>(sizeof(T)) / 16;
    row_bytes = D * static_cast<int>(sizeof(T));
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int r = (wave * kN + i) * kPer + lane / NCH;
      const int c = (lane % NCH) ^ swz<NCH>(r);
      off[i] = c * 16u < row_bytes ? r * step + c * 16 : kPastEnd;
    }
  }
  // Rows row0 .. row0 + ROWS of m to the tile at LDS address la.  The descriptor begins at
  // row0 and holds the rows of the tile that exist, so its sizes stay within 32 bits.
  __device__ __forceinline__ void issue(const Rows& m, int row0, uint32_t la, int wave) const {
    const int left = min(m.rows - row0, ROWS);
    const uint64_t b = reinterpret_cast<uint64_t>(m.base) + static_cast<uint64_t>(static_cast<uint32_t>(row0)) * m.step;
    i32x4 rs;
    rs.x = __builtin_amdgcn_readfirstlane(static_cast<int>(b));
    rs.y = __builtin_amdgcn_readfirstlane(static_cast<int>((b >> 32) & 0xffff));
    rs.z = __builtin_amdgcn_readfirstlane(left <= 0 ? 0 : static_cast<int>((left - 1) * m.step + row_bytes));
    rs.w = 0x00020000;
#pragma unroll
    for (int i = 0; i < kN; ++i) dma16(rs, la + (wave * kN + i) * 1024, off[i]);
  }
};

__device__ __forceinline__ uint32_t lds_addr(const void* p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((GHIP_LDS const void*)p));
}
// This wave's DMA has landed and its LDS reads and writes are done; then the workgroup's.
__device__ __forceinline__ void landed_barrier() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __syncthreads();
}

}  // namespace tile
}  // namespace ghip
