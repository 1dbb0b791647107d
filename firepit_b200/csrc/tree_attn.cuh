// What the attention kernels over the 8-bit cache share: the call's arguments,
// what a row sees, the scaling of queries and weights.
#pragma once
#include "kv8.cuh"

namespace fpb {

struct TreeArgs {
  const void *q;
  const float *gate;
  const uint8_t *k_codes, *v_codes, *k_exp, *v_exp;
  const int32_t *positions, *parents;
  long long q_pitch, q_head, gate_pitch, gate_head;  // elements
  int batch, nodes, q_heads, kv_heads, group, head_dim, max_seq, q_bf16, q_vec, splits;
  float scale_log2;  // scale * log2(e): scores and maxima are held in powers of two
  __nv_bfloat16 *out;
  float *part;     // [session, kv head, row tile][split][row][head_dim] numerators
  float2 *part_ml; // [session, kv head, row tile][split][row] maximum, sum
  // for the tiles: queries as f16, their factors, what each node sees [session,
  // 64], [session, kv head, row tile] first slot and last block
  uint4 *q16;
  float *q_fac;
  uint64_t *sights;
  int2 *shares;
  int *error;
};

// What a row (node n's query head) sees: rows before `pos`, then the tree
// rows of `bits` (a tree), or the first `upto` of them (a chain); upto < 0:
// the node is not there.
struct Sight {
  int upto;
  uint64_t bits;
  // Which of the 64 rows from t0 on it sees.
  __device__ __forceinline__ uint64_t seen64(int t0, int pos, bool tree) const {
    const int k = pos - t0;  // rows of the context among them
    if (!tree) {
      const int c = k + max(upto, 0);
      return c >= 64 ? ~0ull : c <= 0 ? 0ull : (1ull << c) - 1;
    }
    if (k >= 64) return ~0ull;
    if (k > 0) return ((1ull << k) - 1) | bits << k;
    return k > -64 ? bits >> -k : 0ull;
  }
  __device__ __forceinline__ bool sees(int t, int pos, bool tree) const {
    const int j = t - pos;
    if (j < 0) return true;
    return tree ? j < kTreeMaxNodes && (bits >> j & 1) : j < upto;
  }
};

// The tree is walked through the warp's registers: all 32 lanes call this, each
// with its own node (n >= nodes: none).  A row outside the cache is an error of a
// node that would be there.
__device__ __forceinline__ Sight sight_of(const TreeArgs &a, int b, int n, int pos) {
  Sight s{-1, 0};
  const bool in = n < a.nodes;
  const bool inside = pos >= 0 && pos < a.max_seq - n;
  if (!a.parents) {
    if (in && inside) s.upto = n + 1;
    if (in && !inside && a.error) atomicCAS(a.error, 0, kErrPosition);
    return s;
  }
  const int32_t *par = a.parents + (size_t)b * a.nodes;
  const int lane = threadIdx.x & 31;
  const int p0 = lane < a.nodes ? par[lane] : -2, p1 = lane + 32 < a.nodes ? par[lane + 32] : -2;
  const int root = __shfl_sync(0xffffffffu, p0, 0);  // (by every lane, outside the conditions)
  bool there = in && root == -1;
  bool going = there && n > 0;
  int j = in ? n : 0;
  while (__any_sync(0xffffffffu, going)) {
    const int lo = __shfl_sync(0xffffffffu, p0, j & 31), hi = __shfl_sync(0xffffffffu, p1, j & 31);
    const int p = j < 32 ? lo : hi;
    if (going) {
      if (p < 0 || p >= j) {
        if (p >= j && a.error) atomicCAS(a.error, 0, kErrParent);
        there = going = false;
      } else {
        s.bits |= 1ull << j;
        j = p;
        going = j > 0;
      }
    }
  }
  if (there && !inside) {
    there = false;
    if (a.error) atomicCAS(a.error, 0, kErrPosition);
  }
  if (there) {
    s.upto = n + 1;
    s.bits |= 1;
  } else {
    s.bits = 0;
  }
  return s;
}

// Rows of the cache that this session's nodes can see (0: none).
__device__ __forceinline__ int seen_rows(const TreeArgs &a, int pos, int last_node) {
  if (pos < 0 || pos >= a.max_seq) return 0;
  return min(pos + last_node + 1, a.max_seq);
}

__device__ __forceinline__ float load_q(const TreeArgs &a, size_t at) {
  return a.q_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16 *>(a.q)[at])
                  : static_cast<const float *>(a.q)[at];
}

// Eight elements of q from `at` on (a multiple of 8).
__device__ __forceinline__ void load_q8(const TreeArgs &a, size_t at, float (&x)[8]) {
  if (!a.q_vec) {
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = load_q(a, at + k);
  } else if (a.q_bf16) {
    const uint4 v = *reinterpret_cast<const uint4 *>(static_cast<const __nv_bfloat16 *>(a.q) + at);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      x[2 * k] = __uint_as_float(w[k] << 16);
      x[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
    }
  } else {
    const float4 *p = reinterpret_cast<const float4 *>(static_cast<const float *>(a.q) + at);
    const float4 u = p[0], v = p[1];
    x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w;
    x[4] = v.x; x[5] = v.y; x[6] = v.z; x[7] = v.w;
  }
}

// Power of two that takes a query row into f16: its largest magnitude to
// [2^8, 2^9), so that f16's 11 bits hold down to 2^-22 of it (f16 products
// round at 2^-11; the scores' f32 sums and the factor are exact in it).
__device__ __forceinline__ int q_exponent(float amax) {
  const uint32_t u = __float_as_uint(amax);
  if (u < 0x00800000u || u >= 0x7f800000u) return 0;  // zero, subnormal, infinite
  return max(-118, (int)(u >> 23) - 127 - 8);
}

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Weights are held as 2^(y - m + kHead), y the score (in powers of two) plus
// the value vector's own exponent: f16 then holds a weight down to 2^-32 of
// the row's largest.  The maximum may lag by kLag before the sums are rescaled
// (weights up to 2^(kHead + kLag)).
constexpr float kHead = 7.0f, kLag = 8.0f, kMost = 32768.0f, kLowest = -1e30f;
// Their sum takes them without the values' exponents v, which lie within [-100,
// 120]: a value's size is no part of its weight.  Since m >= y + v - kLag (in the
// tiles a half less) for every score y, 2^(y - m + kHead) could reach 2^115.5, and
// the largest be 2^-113; times 2^kSpread that becomes 2^126.5 and 2^-102, so that
// no weight overflows and none is lost that is above 2^-24 of the largest.  The
// value's factor takes 2^kSpread back, and the sum is held times kSumScale (2^20 weights fit), what
// 1 / sum has to be multiplied by kSumBack for.
constexpr int kSpread = 11;
constexpr float kSumScale = 0x1p-20f, kSumBack = 0x1p-9f;
static_assert(kSumScale / kSumBack == 1.0f / (1 << kSpread));
// A zero value vector adds to the sum only: it takes part in the maximum as
// one of the smallest exponent, so that a large weight of its own (a row that
// the model rests attention on) does not push what the others give out of f16.
// Found where a maximum is about to be raised, from the codes.
constexpr float kZeroExp = kKv8MinExp;
// A sum of weights taken from one maximum to another that is `by` (<= 0) higher.
// Two maxima may lie 220 and more apart, where the factor is no f32 but the
// sum's two ends are: it goes by halves.
__device__ __forceinline__ float sum_to(float l, float by) {
  const float half = exp2_approx(0.5f * by);
  return l * half * half;
}

// The tcgen05 kernel (tree_attn_tile.cu): token tiles of BT rows, `blocks` of
// them, their partial results and the items' shares of them in the workspace.
struct TilePlan {
  int BT, blocks;
  size_t batch, items, units;  // units: a bound
};
TilePlan tile_plan(size_t batch, size_t nodes, size_t q_heads, size_t kv_heads, size_t head_dim, size_t max_seq);
size_t tile_workspace_bytes(const TilePlan &p, size_t head_dim);
int run_tree_tiles(TreeArgs a, const TilePlan &p, void *workspace, cudaStream_t s);

}  // namespace fpb
