// The 8-bit key/value cache and the trees of drafted tokens, as the kernels
// that write (kv8.cu) and read (kv8.cu, tree_attn.cu) them agree on them.
//
// A head vector x [head_dim] is held as e4m3 codes and one exponent byte:
// x ~ code * 2^(byte - 127), with the smallest exponent e for which
// max |x| <= 448 * 2^e.  A power of two costs no precision against
// max|x| / 448 (e4m3 is a floating-point format: its relative step is the
// same at every exponent; only the 2^-9 underflow threshold moves, by less
// than a factor of two), and it makes every use of the factor exact: the
// quotient before the rounding, the score's product, the value's weight.
#pragma once
#include "common.cuh"

namespace fpb {

constexpr int kKv8MinExp = -100, kKv8MaxExp = 120, kKv8ZeroExp = -8, kTreeMaxNodes = 64;
// Device error codes of these operators (fpb_device_error).
constexpr int kErrPosition = 502, kErrParent = 504, kErrToken = 505;

// 2^e for e in [-126, 127].
__device__ __forceinline__ float pow2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
// 2^(byte - 127) of a cache exponent byte (any byte).
__device__ __forceinline__ float kv8_factor(uint32_t byte) {
  return __uint_as_float(byte ? byte << 23 : 0x00400000u);
}

// A value vector's exponent as the attention uses it: within the cache's
// range whatever a row that nobody wrote may hold, so that it and its inverse
// stay finite.
__device__ __forceinline__ float kv8_value_exponent(uint32_t byte) {
  return (float)min(kKv8MaxExp, max(kKv8MinExp, (int)byte - 127));
}

// The exponent for a head vector whose largest magnitude is amax: 448 = 1.75
// * 2^8, so with amax = m * 2^x, m in [1, 2), it is x - 8, or x - 7 past 1.75.
// Zero vectors take a middling exponent (the attention weighs each row by it).
// Subnormal and infinite maxima end at the clamps.
__device__ __forceinline__ int kv8_exponent(float amax) {
  const uint32_t u = __float_as_uint(amax);
  if (u == 0) return kKv8ZeroExp;
  const int e = (int)(u >> 23) - 127 - ((u & 0x7fffffu) <= 0x600000u ? 8 : 7);
  return min(kKv8MaxExp, max(kKv8MinExp, e));
}

// Depth of node n in a session's tree (`parents` [nodes], null: a chain), or
// -1 where it is not there: a negative parent past node 0, an ancestor that
// is not there, or node 0 other than -1.  A parent that is not an earlier
// node is a fault of the tree: *bad is set and the node is not there.
__device__ __forceinline__ int tree_depth(const int32_t *parents, int n, bool *bad) {
  if (!parents) return n;
  int d = 0;
  for (int j = n; j > 0; ++d) {
    const int p = parents[j];
    if (p < 0 || p >= j) {
      if (p >= j) *bad = true;
      return -1;
    }
    j = p;
  }
  return parents[0] == -1 ? d : -1;
}

}  // namespace fpb
