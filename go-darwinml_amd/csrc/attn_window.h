// Arguments of the windowed attention kernels and the checks their entry points share.
#pragma once

#include "attn_tile.h"

namespace ghip {
namespace win {

struct Mat3 {
  const void* p;
  int64_t sb, sh, ss;  // element strides of batch, head, sequence (head dim contiguous)
};

struct Params {
  Mat3 q, k, v, o, dout, dq, dk, dv;
  float* lse;        // [B, H, Sq]; forward: written (may be null), gradient: read
  // Gradient, [2][B, H, Sq]: minus the log-sum-exp in base 2 (f16: plus 15), and minus delta,
  // the row sums of do * o.
  float* stats;
  // Gradient: shares of dk and dv that join_kernel adds, of the first share_blocks blocks of
  // 32 keys: [B, Hkv, share_blocks][shares][dk, dv][32][D].
  float* share;
  int64_t share_stride;  // floats of one block's shares
  int share_blocks, shares, chunks, chunk;  // chunks of so many tiles
  bool far;  // shares: 0 the block's own workgroup, the others chunks of the queries beyond; else all chunks
  const int32_t* lens;
  int B, H, Hkv, Sq, Sk, D;
  int q_start, window, sinks;
  float scale;
};

// The workgroups of 32 queries up to which the kernels that share their keys among the waves
// are taken (measured at the forward kernels' launch): one round of the card, one
// workgroup a CU (rows of 128 bytes: two); in fp32 three.
constexpr int64_t few_most(int elem_bytes, int dp) {
  return elem_bytes == 4 ? 768 : dp * elem_bytes > 128 ? 256 : 512;
}

// The tokens of sequence b that exist: lens[b] clamped to [0, Sk].
__device__ __forceinline__ int length_of(const Params& p, int b) {
  return p.lens ? min(max(p.lens[b], 0), p.Sk) : p.Sk;
}

template <typename T>
__device__ __forceinline__ T* at(const Mat3& m, int b, int h) {
  return static_cast<T*>(const_cast<void*>(m.p)) + b * m.sb + h * m.sh;
}
template <typename T>
__device__ __forceinline__ tile::Rows rows_of(const Mat3& m, int b, int h, int rows) {
  return tile::Rows{reinterpret_cast<const char*>(at<T>(m, b, h)), static_cast<uint32_t>(m.ss * sizeof(T)), rows};
}

// The key tiles of queries at positions [p0, p1]: those of the sinks, then those of the
// windows; tile(i) for i < n.
template <int kKT>
struct Tiles {
  int n, ns, first;
  __device__ __forceinline__ Tiles(const Params& p, int p0, int end) {
    const int lo = max(0, p0 - p.window + 1) / kKT;
    const int hi = (end + kKT - 1) / kKT;  // end: one past the last key that any query sees
    ns = min((min(p.sinks, end) + kKT - 1) / kKT, lo);
    first = lo;
    n = end > 0 ? ns + max(0, hi - lo) : 0;
  }
  __device__ __forceinline__ int operator()(int i) const { return i < ns ? i : first + i - ns; }
};

// The (batch, head) that workgroup i of each n works on.  Consecutive workgroups go to the
// 8 XCDs in turn; neighbouring heads, which share K and V, should share an L2.
__device__ __forceinline__ int spread(int i, int n) { return n % 8 == 0 ? i % 8 * (n / 8) + i / 8 : i; }

// Bits [0, n) of a word, n clamped to 0 .. 32.
__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; }
// Which of keys key0 + kv, kv < 32, the query at position pos sees, as bits (none unless live).
__device__ __forceinline__ uint32_t seen_keys(const Params& p, int pos, bool live, int len, int key0) {
  if (!live) return 0u;
  return low_bits(min(len, pos + 1) - key0) & (~low_bits(pos - p.window + 1 - key0) | low_bits(p.sinks - key0));
}
// x where bit `bit` of word is set, otherwise `other` (two instructions an element).
__device__ __forceinline__ float select_bit(uint32_t word, int bit, float x, float other) {
  const uint32_t t = static_cast<uint32_t>(__builtin_amdgcn_sbfe(static_cast<int>(word), bit, 1));
  return __uint_as_float((t & __float_as_uint(x)) | (~t & __float_as_uint(other)));
}

// The problem's sizes and types; fills p.  Returns GHIP_OK or the error.
int check_problem(const char* what, int dtype, int64_t B, int64_t H, int64_t Hkv, int64_t Sq, int64_t Sk, int64_t D,
                  int64_t q_start, int64_t window, int64_t sinks, float scale, Params* p, GHipError* err);
// One operand of p's batch, `heads` heads, `rows` rows: its strides (an axis of one entry may
// have any that is not negative) and alignment (out: 8-byte rows of 16-bit values suffice).
int check_operand(const char* what, const char* name, int dtype, const void* ptr, const int64_t* strides,
                  const Params& p, int heads, int rows, bool out, Mat3* m, GHipError* err);

}  // namespace win
}  // namespace ghip
