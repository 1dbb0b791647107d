// Attention of a tree of drafted tokens over the 8-bit cache (kv8.cuh).
//
// Node i of session b sees the cache rows before position[b], its ancestors'
// rows and its own (row position + j of node j).  With s_t = scale q . k_t:
//   out = sum_t softmax(s)_t v_t, times sigmoid(gate) where a gate is given.
#include <algorithm>
#include <cmath>
#include <mutex>
#include <vector>

#include "kv8.cuh"
#include "sm100.cuh"

namespace fpb {
namespace {

using namespace sm100;

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
// with its own node (n >= nodes: none).
__device__ __forceinline__ Sight sight_of(const TreeArgs &a, int b, int n, int pos) {
  Sight s{-1, 0};
  const bool in = n < a.nodes;
  const bool inside = pos >= 0 && pos < a.max_seq - n;
  if (in && !inside && a.error) atomicCAS(a.error, 0, kErrPosition);
  if (!a.parents) {
    if (in && inside) s.upto = n + 1;
    return s;
  }
  const int32_t *par = a.parents + (size_t)b * a.nodes;
  const int lane = threadIdx.x & 31;
  const int p0 = lane < a.nodes ? par[lane] : -2, p1 = lane + 32 < a.nodes ? par[lane + 32] : -2;
  const int root = __shfl_sync(0xffffffffu, p0, 0);  // (by every lane, outside the conditions)
  bool there = in && inside && root == -1;
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

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Weights are held as 2^(y - m + kHead), y the score (in powers of two) plus
// the value vector's own exponent: f16 then holds a weight down to 2^-32 of
// the row's largest, and the exponent costs no multiplication.  The maximum
// may lag by kLag before the sums are rescaled (weights up to 2^(kHead + kLag)).
constexpr float kHead = 7.0f, kLag = 8.0f, kMost = 32768.0f, kLowest = -1e30f;

// ---- few rows: tokens streamed through registers ---------------------------------------------
// Block (split, session * kv head * row tile): NR rows (8 or 16) of one kv
// head, four warps that take steps of 16 tokens in turn, all on their own:
// codes go from memory to registers to the tensor cores with no shared memory
// between.
//  S = Q K^T   m16n8k16, the rows as M (NR = 8 leaves half of it zero).  The
//              order of the summed dimension is free as long as both sides
//              agree, so a lane's 16-byte piece of a key (16 dimensions) is
//              its operand of four instructions as it lies.
//  O^T = V^T P^T  the dimensions as M, the rows as N: P^T's operand is S's
//              result as it lies.  V's needs pairs of tokens in a word: byte
//              permutes of two tokens' pieces before the conversion.
// Each e4m3 is converted to f16 (exact); the key's factor goes to the score,
// the value's to the weight's exponent.
constexpr int kRowsThreads = 128, kRowsWarps = 4;

template <int DP, int NR>
struct RowsShape {
  static constexpr bool kQShared = NR * DP > 16 * 128;  // 64 registers of queries are too many beside 128 of sums
  static constexpr int kQPitch = DP + 8;                // f16 elements: 16-byte reads of eight rows on distinct banks
  static constexpr size_t smem = (size_t)kRowsWarps * NR * (DP + 2) * 4;
};

template <int DP, int NR>
__global__ void __launch_bounds__(kRowsThreads, 2) tree_attn_rows_kernel(const __grid_constant__ TreeArgs a) {
  pdl_enter();
  using Sh = RowsShape<DP, NR>;
  constexpr int kPieces = DP / 64, kVPieces = DP >= 128 ? DP / 128 : 1, kVBytes = DP >= 128 ? 16 : 8;
  constexpr int kMT = DP / 16, kNT = NR / 8;
  extern __shared__ __align__(16) float sm[];  // queries (f16) first, then the warps' results
  __shared__ float m_s[kRowsWarps][NR], l_s[kRowsWarps][NR];
  __shared__ float fac_s[NR];
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, g = lane >> 2, c = lane & 3;
  const int rows = a.nodes * a.group, tiles = (rows + NR - 1) / NR;
  const int item = blockIdx.y, tile = item % tiles, bk = item / tiles;
  const int b = bk / a.kv_heads, kvh = bk % a.kv_heads, D = a.head_dim;
  const int pos = a.positions[b];
  const bool tree = a.parents != nullptr;
  const int last = min(a.nodes - 1, (tile * NR + NR - 1) / a.group);
  const int total = seen_rows(a, pos, last);
  // this split's tokens, in whole steps
  const int steps = (total + 15) / 16, per = (steps + a.splits - 1) / a.splits;
  const int s0 = blockIdx.x * per, s1 = min(steps, s0 + per);

  // queries: a warp takes rows w, w + 4, ...; eight columns a lane
  __half *qs = reinterpret_cast<__half *>(sm);
  for (int r = w; r < NR; r += kRowsWarps) {
    const int row = tile * NR + r, n = row / a.group, h = kvh * a.group + row % a.group;
    float x[8];
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int col = lane * 8 + i;
      x[i] = row < rows && col < D
                 ? load_q(a, ((size_t)b * a.nodes + n) * a.q_pitch + (size_t)h * a.q_head + col) : 0.0f;
      amax = fmaxf(amax, fabsf(x[i]));
    }
    amax = warp_max(amax);
    const int e = q_exponent(amax);
    const float f = pow2i(-e);
    if (lane * 8 < DP) {
      uint4 o;
      o.x = pack_f16x2(x[0] * f, x[1] * f);
      o.y = pack_f16x2(x[2] * f, x[3] * f);
      o.z = pack_f16x2(x[4] * f, x[5] * f);
      o.w = pack_f16x2(x[6] * f, x[7] * f);
      *reinterpret_cast<uint4 *>(qs + r * Sh::kQPitch + lane * 8) = o;
    }
    if (lane == 0) fac_s[r] = pow2i(e) * a.scale_log2;
  }
  __syncthreads();
  // the lane's rows of S: g and, with 16 rows, g + 8
  Sight sight[kNT];
  float fac[kNT];
#pragma unroll
  for (int i = 0; i < kNT; ++i) {
    const int row = tile * NR + g + 8 * i;
    sight[i] = sight_of(a, b, row < rows ? row / a.group : a.nodes, pos);
    fac[i] = fac_s[g + 8 * i];
  }
  // Q operands of piece p: row's dimensions 64 p + 16 c + [0, 16)
  uint32_t qr[Sh::kQShared ? 1 : kPieces * kNT * 8];
  if constexpr (!Sh::kQShared) {
#pragma unroll
    for (int p = 0; p < kPieces; ++p)
#pragma unroll
      for (int i = 0; i < kNT; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint4 v = *reinterpret_cast<const uint4 *>(qs + (g + 8 * i) * Sh::kQPitch + 64 * p + 16 * c + 8 * j);
          uint32_t *o = qr + (p * kNT + i) * 8 + 4 * j;
          o[0] = v.x; o[1] = v.y; o[2] = v.z; o[3] = v.w;
        }
  }

  const size_t pitch = (size_t)a.kv_heads * D;
  const uint8_t *kc = a.k_codes + ((size_t)b * a.max_seq * a.kv_heads + kvh) * D;
  const uint8_t *vc = a.v_codes + ((size_t)b * a.max_seq * a.kv_heads + kvh) * D;
  const uint8_t *ex = (lane < 16 ? a.k_exp : a.v_exp) + (size_t)b * a.max_seq * a.kv_heads + kvh;
  uint4 kr[2][kPieces];
  uint32_t vr[4][kVPieces][kVBytes / 4];
  uint32_t xr = 0;
  auto load_k = [&](int step) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int t = step * 16 + 8 * u + g;
#pragma unroll
      for (int p = 0; p < kPieces; ++p) {
        const int d = 64 * p + 16 * c;
        kr[u][p] = t < total && d < D ? __ldg(reinterpret_cast<const uint4 *>(kc + (size_t)t * pitch + d))
                                      : make_uint4(0, 0, 0, 0);
      }
    }
    const int t = step * 16 + (lane & 15);
    xr = t < total ? ex[(size_t)t * a.kv_heads] : 127;
  };
  auto load_v = [&](int step) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int t = step * 16 + 2 * c + (i & 1) + 8 * (i >> 1);
#pragma unroll
      for (int p = 0; p < kVPieces; ++p) {
        const int d = 128 * p + kVBytes * g;
        if constexpr (kVBytes == 16) {
          const uint4 v = t < total && d < D ? __ldg(reinterpret_cast<const uint4 *>(vc + (size_t)t * pitch + d))
                                             : make_uint4(0, 0, 0, 0);
          vr[i][p][0] = v.x; vr[i][p][1] = v.y; vr[i][p][2] = v.z; vr[i][p][3] = v.w;
        } else {
          const uint2 v = t < total && d < D ? __ldg(reinterpret_cast<const uint2 *>(vc + (size_t)t * pitch + d))
                                             : make_uint2(0, 0);
          vr[i][p][0] = v.x; vr[i][p][1] = v.y;
        }
      }
    }
  };

  float acc[kMT][kNT][4];
#pragma unroll
  for (int i = 0; i < kMT; ++i)
#pragma unroll
    for (int j = 0; j < kNT; ++j)
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[i][j][k] = 0.0f;
  float m[kNT], l[kNT];
#pragma unroll
  for (int i = 0; i < kNT; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.0f;
  }
  int step = s0 + w;
  if (step < s1) {
    load_k(step);
    load_v(step);
  }
  for (; step < s1; step += kRowsWarps) {
    // scores of 16 tokens: s[u] tokens 8 u + 2 c, 2 c + 1 of row g (and g + 8)
    float s[2][4];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int k = 0; k < 4; ++k) s[u][k] = 0.0f;
#pragma unroll
    for (int p = 0; p < kPieces; ++p) {
      uint32_t q0[8], q1[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) q1[j] = 0;
      if constexpr (Sh::kQShared) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint4 v = *reinterpret_cast<const uint4 *>(qs + g * Sh::kQPitch + 64 * p + 16 * c + 8 * j);
          q0[4 * j] = v.x; q0[4 * j + 1] = v.y; q0[4 * j + 2] = v.z; q0[4 * j + 3] = v.w;
          if constexpr (NR == 16) {
            const uint4 y = *reinterpret_cast<const uint4 *>(qs + (g + 8) * Sh::kQPitch + 64 * p + 16 * c + 8 * j);
            q1[4 * j] = y.x; q1[4 * j + 1] = y.y; q1[4 * j + 2] = y.z; q1[4 * j + 3] = y.w;
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          q0[j] = qr[p * kNT * 8 + j];
          if constexpr (NR == 16) q1[j] = qr[(p * kNT + 1) * 8 + j];
        }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const uint32_t kw[4] = {kr[u][p].x, kr[u][p].y, kr[u][p].z, kr[u][p].w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
          mma_f16(s[u], q0[2 * j], q1[2 * j], q0[2 * j + 1], q1[2 * j + 1], e4m3x2_to_f16x2((uint16_t)kw[j]),
                  e4m3x2_to_f16x2((uint16_t)(kw[j] >> 16)));
      }
    }
    const uint32_t xb = xr;
    const int t0 = step * 16;
    const bool open = t0 + 16 > pos;  // warp-uniform: the tree's rows, or the end
    if (step + kRowsWarps < s1) load_k(step + kRowsWarps);
    uint32_t nan[4] = {0, 0, 0, 0};
    if (open) {  // a value vector that some row does not see must not reach it through 0 * NaN
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int p = 0; p < kVPieces; ++p)
#pragma unroll
          for (int j = 0; j < kVBytes / 4; ++j) {
            const uint32_t bad = __vcmpeq4(vr[i][p][j] & 0x7f7f7f7fu, 0x7f7f7f7fu);
            vr[i][p][j] &= ~bad;
            nan[i] |= bad;
          }
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) nan[i] |= __shfl_xor_sync(0xffffffffu, nan[i], o);
      }
    }
    // y = score + the value's exponent, and the rows' maxima
    float y[kNT][4], ve[4], mx[kNT];
#pragma unroll
    for (int i = 0; i < kNT; ++i) mx[i] = -INFINITY;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int u = k >> 1, e = k & 1, tl = 8 * u + 2 * c + e, t = t0 + tl;
      const float kf = kv8_factor(__shfl_sync(0xffffffffu, xb, tl));
      ve[k] = kv8_value_exponent(__shfl_sync(0xffffffffu, xb, 16 + tl));
#pragma unroll
      for (int i = 0; i < kNT; ++i) {
        float v = fmaf(s[u][2 * i + e], kf * fac[i], ve[k]);
        if (open) {
          if (nan[k]) v = __int_as_float(0x7fc00000);
          if (t >= total || !sight[i].sees(t, pos, tree)) v = -INFINITY;
        }
        y[i][k] = v;
        mx[i] = fmaxf(mx[i], v);
      }
    }
    bool grow = false;
#pragma unroll
    for (int i = 0; i < kNT; ++i) {
      mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
      mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
      grow |= mx[i] > m[i] + kLag || (m[i] == -INFINITY && mx[i] > m[i]);
    }
    if (__any_sync(0xffffffffu, grow)) {
      float old[kNT];
#pragma unroll
      for (int i = 0; i < kNT; ++i) {
        const float mn = fmaxf(m[i], mx[i]);
        old[i] = m[i] == -INFINITY ? 0.0f : exp2_approx(m[i] - mn);
        l[i] *= old[i];
        m[i] = mn;
      }
#pragma unroll
      for (int j = 0; j < kNT; ++j)  // the sums hold rows 2 c, 2 c + 1 (+ 8 j): their factors are lanes 8 c and 8 c + 4's
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float f = __shfl_sync(0xffffffffu, old[j], 8 * c + 4 * e);
#pragma unroll
          for (int i = 0; i < kMT; ++i) {
            acc[i][j][e] *= f;
            acc[i][j][2 + e] *= f;
          }
        }
    }
    uint32_t pb[kNT][2];
#pragma unroll
    for (int i = 0; i < kNT; ++i) {
      const float base = m[i] == -INFINITY ? 0.0f : kHead - m[i];
      float p[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        p[k] = exp2_approx(y[i][k] + base);
        l[i] = fmaf(p[k], pow2i(-(int)ve[k]), l[i]);
      }
      pb[i][0] = pack_f16x2(p[0], p[1]);
      pb[i][1] = pack_f16x2(p[2], p[3]);
    }
#pragma unroll
    for (int p = 0; p < kVPieces; ++p)
#pragma unroll
      for (int j = 0; j < kVBytes / 4; ++j) {
        const uint32_t x0 = __byte_perm(vr[0][p][j], vr[1][p][j], 0x5140);
        const uint32_t x1 = __byte_perm(vr[0][p][j], vr[1][p][j], 0x7362);
        const uint32_t z0 = __byte_perm(vr[2][p][j], vr[3][p][j], 0x5140);
        const uint32_t z1 = __byte_perm(vr[2][p][j], vr[3][p][j], 0x7362);
        const int mt = (p * kVBytes / 4 + j) * 2;
#pragma unroll
        for (int i = 0; i < kNT; ++i) {
          mma_f16(acc[mt][i], e4m3x2_to_f16x2((uint16_t)x0), e4m3x2_to_f16x2((uint16_t)(x0 >> 16)),
                  e4m3x2_to_f16x2((uint16_t)z0), e4m3x2_to_f16x2((uint16_t)(z0 >> 16)), pb[i][0], pb[i][1]);
          mma_f16(acc[mt + 1][i], e4m3x2_to_f16x2((uint16_t)x1), e4m3x2_to_f16x2((uint16_t)(x1 >> 16)),
                  e4m3x2_to_f16x2((uint16_t)z1), e4m3x2_to_f16x2((uint16_t)(z1 >> 16)), pb[i][0], pb[i][1]);
        }
      }
    if (step + kRowsWarps < s1) load_v(step + kRowsWarps);
  }

  // the warps' results meet: maxima, then sums over one maximum in warp order
#pragma unroll
  for (int i = 0; i < kNT; ++i) {
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    if (c == 0) {
      m_s[w][g + 8 * i] = m[i];
      l_s[w][g + 8 * i] = l[i];
    }
  }
  __syncthreads();  // also: every warp is done with the queries that `sm` held
  float *mine = sm + (size_t)w * NR * (DP + 2);
#pragma unroll
  for (int p = 0; p < kVPieces; ++p)
#pragma unroll
    for (int j = 0; j < kVBytes / 4; ++j)
#pragma unroll
      for (int i = 0; i < kNT; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int mt = (p * kVBytes / 4 + j) * 2, d = 128 * p + kVBytes * g + 4 * j;
          float *o = mine + (size_t)(8 * i + 2 * c + e) * (DP + 2) + d;
          *reinterpret_cast<float2 *>(o) = make_float2(acc[mt][i][e], acc[mt][i][2 + e]);
          *reinterpret_cast<float2 *>(o + 2) = make_float2(acc[mt + 1][i][e], acc[mt + 1][i][2 + e]);
        }
  __syncthreads();
  for (int r = w; r < NR; r += kRowsWarps) {
    const int row = tile * NR + r;
    if (row >= rows) break;
    float mt = -INFINITY, f[kRowsWarps], lt = 0.0f;
#pragma unroll
    for (int x = 0; x < kRowsWarps; ++x) mt = fmaxf(mt, m_s[x][r]);
#pragma unroll
    for (int x = 0; x < kRowsWarps; ++x) {
      f[x] = m_s[x][r] == -INFINITY ? 0.0f : exp2_approx(m_s[x][r] - mt);
      lt += l_s[x][r] * f[x];
    }
    const int n = row / a.group, h = kvh * a.group + row % a.group;
    const bool there = sight_of(a, b, n, pos).upto >= 0;
    for (int d = lane * 2; d < D; d += 64) {
      float2 o = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int x = 0; x < kRowsWarps; ++x) {
        const float2 v = *reinterpret_cast<const float2 *>(sm + ((size_t)x * NR + r) * (DP + 2) + d);
        o.x = fmaf(v.x, f[x], o.x);
        o.y = fmaf(v.y, f[x], o.y);
      }
      if (a.splits > 1) {
        *reinterpret_cast<float2 *>(a.part + (((size_t)item * a.splits + blockIdx.x) * NR + r) * D + d) = o;
      } else {
        const size_t node = (size_t)b * a.nodes + n;
        const float inv = there ? 1.0f / lt : 0.0f;
        o.x = there ? o.x * inv : 0.0f;
        o.y = there ? o.y * inv : 0.0f;
        if (a.gate && there) {
          const float *gt = a.gate + node * a.gate_pitch + (size_t)h * a.gate_head + d;
          o.x /= 1.0f + expf(-gt[0]);
          o.y /= 1.0f + expf(-gt[1]);
        }
        *reinterpret_cast<uint32_t *>(a.out + (node * a.q_heads + h) * D + d) = pack_bf16x2(o.x, o.y);
      }
    }
    if (a.splits > 1 && lane == 0)
      a.part_ml[((size_t)item * a.splits + blockIdx.x) * NR + r] = make_float2(mt, lt);
  }
}

// The splits of a row meet: one warp a (session, node, query head), the
// splits in order.
__global__ void __launch_bounds__(256) tree_attn_merge_kernel(const __grid_constant__ TreeArgs a, int NR, int count) {
  pdl_enter();
  const int lane = threadIdx.x & 31, i = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (i >= count) return;
  const int h = i % a.q_heads, node = i / a.q_heads, b = node / a.nodes, n = node % a.nodes, D = a.head_dim;
  const int kvh = h / a.group, row = n * a.group + h % a.group;
  const int tiles = (a.nodes * a.group + NR - 1) / NR;
  const size_t item = ((size_t)b * a.kv_heads + kvh) * tiles + row / NR;
  const int r = row % NR, pos = a.positions[b];
  const bool there = sight_of(a, b, n, pos).upto >= 0;
  const float2 *ml = a.part_ml + item * a.splits * NR + r;
  float m = -INFINITY, l = 0.0f;
  for (int s = lane; s < a.splits; s += 32) m = fmaxf(m, ml[(size_t)s * NR].x);
  m = warp_max(m);
  float acc[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) acc[k] = 0.0f;
  const int d = lane * 8;
  for (int s = 0; s < a.splits; ++s) {
    const float2 v = ml[(size_t)s * NR];
    const float f = v.x == -INFINITY ? 0.0f : exp2_approx(v.x - m);
    l = fmaf(v.y, f, l);
    if (d < D && f != 0.0f) {
      const float4 *p = reinterpret_cast<const float4 *>(a.part + ((item * a.splits + s) * NR + r) * D + d);
      const float4 x = p[0], z = p[1];
      acc[0] = fmaf(x.x, f, acc[0]); acc[1] = fmaf(x.y, f, acc[1]);
      acc[2] = fmaf(x.z, f, acc[2]); acc[3] = fmaf(x.w, f, acc[3]);
      acc[4] = fmaf(z.x, f, acc[4]); acc[5] = fmaf(z.y, f, acc[5]);
      acc[6] = fmaf(z.z, f, acc[6]); acc[7] = fmaf(z.w, f, acc[7]);
    }
  }
  if (d >= D) return;
  const float inv = 1.0f / l;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    acc[k] = there ? acc[k] * inv : 0.0f;
    if (there && a.gate)
      acc[k] /= 1.0f + expf(-a.gate[(size_t)node * a.gate_pitch + (size_t)h * a.gate_head + d + k]);
  }
  *reinterpret_cast<uint4 *>(a.out + ((size_t)node * a.q_heads + h) * D + d) =
      make_uint4(pack_bf16x2(acc[0], acc[1]), pack_bf16x2(acc[2], acc[3]), pack_bf16x2(acc[4], acc[5]),
                 pack_bf16x2(acc[6], acc[7]));
}

// ---- many rows: tiles on tcgen05 ----------------------------------------------------------------
// Block: a share of the call's (session, kv head, 128-row tile, token tile)
// units, in that order, so that sessions of any lengths load the SMs evenly;
// a (row tile)'s token tiles that fall to several blocks meet in the merge.
//   warps 0-7   softmax: thread (half, r) owns half of row r's tokens (TMEM
//               lane r)
//   warp 8      issues the MMAs
//   warps 9-15  read codes and convert them to f16 tiles in shared memory
// S = Q K^T and O += P V with Q and P as the A operand in TMEM, so shared
// memory carries only what K and V need: 64 KB written and 64 KB read a tile
// of 16384 elements each, against 1024 cycles of MMA.  A tile is 64 tokens at
// head_dim 256, else 128: TMEM then holds O [DP], two S [BT] (P overwrites
// its S) and Q [DP / 2 columns].
//   K tile: tokens as rows of 128-byte swizzled lines, 64 dimensions a chunk
//           (K-major).
//   V tile: the same bytes read as the transposed operand (N-major).
// The tokens' factors stay out of the tiles: the key's multiplies the score,
// the value's the weight, both in f32 (see kHead).
constexpr int kSoftThreads = 256, kMmaWarp = 8, kConvThreads = 224, kTileRows = 128;
constexpr int kTileThreads = kSoftThreads + 32 + kConvThreads;
constexpr int kErrTileWait = 503;

template <int DP>
struct TileShape {
  static constexpr int BT = DP == 256 ? 64 : 128, ST = 3, META = 8;
  static constexpr uint32_t kBytes = BT * DP * 2;
  static constexpr uint32_t kTmemO = 0, kTmemS = DP, kTmemQ = DP + 2 * BT;
  static constexpr int kPieces = (BT * DP / 16 + kConvThreads - 1) / kConvThreads;  // 16-byte pieces of codes a thread and tile
  static constexpr int kQPitch = 40;  // f16 elements of a staged query row's 32 columns: rows on distinct banks
  static constexpr size_t smem = 1024 + 2 * ST * (size_t)kBytes + META * BT * 8 + kSoftThreads * kQPitch * 2;

};

// Token tiles of session b (0: none of its nodes is there).
__device__ __forceinline__ int session_tiles(const TreeArgs &a, int b, int BT) {
  if (a.parents && a.parents[(size_t)b * a.nodes] != -1) return 0;
  return (seen_rows(a, a.positions[b], a.nodes - 1) + BT - 1) / BT;
}

// Units before session b (b = batch: all), warp-collective.
__device__ __forceinline__ long long units_before(const TreeArgs &a, int b, int BT, int items) {
  long long n = 0;
  const int lane = threadIdx.x & 31;
  for (int i = lane; i < b; i += 32) n += session_tiles(a, i, BT);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
  return n * items;
}

struct Segment {
  int b, kvh, rt, j0, j1, pos, total;
};

// A block's units, one segment (token tiles [j0, j1) of one row tile) at a time.
struct Walk {
  int b, tiles, row_tiles;
  int rem, left;
  __device__ __forceinline__ bool next(const TreeArgs &a, int BT, Segment &s) {
    if (left <= 0) return false;
    const int items = a.kv_heads * row_tiles;
    while (rem >= items * tiles) {
      rem -= items * tiles;
      tiles = session_tiles(a, ++b, BT);
    }
    const int item = rem / tiles;
    s.j0 = rem % tiles;
    const int n = min(left, tiles - s.j0);
    left -= n;
    rem += n;
    s.b = b;
    s.kvh = item / row_tiles;
    s.rt = item % row_tiles;
    s.pos = a.positions[b];
    // a chain's row tile ends at its last node's own row
    s.total = seen_rows(a, s.pos, min(a.nodes - 1, (s.rt * kTileRows + kTileRows - 1) / a.group));
    s.j1 = min(s.j0 + n, (s.total + BT - 1) / BT);
    return true;
  }
};

__device__ __forceinline__ void give_up(int *error, volatile int *abort) {
  *abort = 1;
  if (error) atomicCAS(error, 0, kErrTileWait);
}

// Codes pass by once: they leave L1 to what is used again.
__device__ __forceinline__ uint4 load_once(const uint8_t *p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float &a, float &b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// Half a row of S (NT tokens from TMEM column s_tmem, factors fac: two keys',
// two values' of each pair): weights e = 2^(s * kf * f + base), their sums in l,
// e * vf as f16 pairs in p; returns the largest e * vf.  OPEN: a tile that not
// every row sees whole, only its tokens `seen`.
template <int NT, bool OPEN>
__device__ __forceinline__ float weigh_pass(uint32_t s_tmem, const float4 *fac, float f, float base, uint64_t seen,
                                            uint32_t (&p)[NT / 2], uint64_t &l) {
  const uint64_t f2 = pack2(f, f), b2 = pack2(base, base);
  float mx[2] = {0.0f, 0.0f};
#pragma unroll
  for (int c = 0; c < NT / 16; ++c) {
    uint32_t r[16];
    tmem_ld16(s_tmem + c * 16, r);
    tmem_ld_wait(r);
#pragma unroll
    for (int e = 0; e < 16; e += 2) {
      const float4 ft = fac[(c * 16 + e) / 2];
      const uint64_t x = mul2(pack2(__uint_as_float(r[e]), __uint_as_float(r[e + 1])), pack2(ft.x, ft.y));
      float e0, e1, w0, w1;
      unpack2(fma2(x, f2, b2), e0, e1);
      e0 = exp2_approx(e0);
      e1 = exp2_approx(e1);
      if (OPEN) {
        if (!(seen >> (c * 16 + e) & 1)) e0 = 0.0f;
        if (!(seen >> (c * 16 + e + 1) & 1)) e1 = 0.0f;
      }
      const uint64_t e2 = pack2(e0, e1);
      l = add2(l, e2);
      unpack2(mul2(e2, pack2(ft.z, ft.w)), w0, w1);
      mx[(e >> 1) & 1] = fmaxf(mx[(e >> 1) & 1], fmaxf(w0, w1));
      p[(c * 16 + e) / 2] = pack_f16x2(w0, w1);
    }
  }
  return fmaxf(mx[0], mx[1]);
}

// The largest y = s * kf * f + log2(vf) of the same tokens.
template <int NT>
__device__ __forceinline__ float max_pass(uint32_t s_tmem, const float4 *fac, float f, uint64_t seen) {
  float mx = -INFINITY;
#pragma unroll
  for (int c = 0; c < NT / 16; ++c) {
    uint32_t r[16];
    tmem_ld16(s_tmem + c * 16, r);
    tmem_ld_wait(r);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float4 ft = fac[(c * 16 + e) / 2];
      const float v = (float)((int)(__float_as_uint(e & 1 ? ft.w : ft.z) >> 23) - 127);
      const float y = fmaf(__uint_as_float(r[e]) * (e & 1 ? ft.y : ft.x), f, v);
      if (seen >> (c * 16 + e) & 1) mx = fmaxf(mx, y);
    }
  }
  return mx;
}

// The converting threads meet.
__device__ __forceinline__ void conv_sync() { asm volatile("bar.sync 1, 224;" ::: "memory"); }
// All of the softmax threads: meet / meet and learn whether any says yes.
__device__ __forceinline__ void soft_sync() {
  tc_fence_before();
  asm volatile("bar.sync 2, 256;" ::: "memory");
  tc_fence_after();
}
__device__ __forceinline__ bool soft_any(bool v) {
  int r;
  tc_fence_before();
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\tbar.red.or.pred q, 2, 256, p;\n\tselp.b32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"((int)v)
      : "memory");
  tc_fence_after();
  return r != 0;
}

template <int DP>
__global__ void __launch_bounds__(kTileThreads, 1) tree_attn_tile_kernel(const __grid_constant__ TreeArgs a) {
  pdl_enter();
  using Sh = TileShape<DP>;
  constexpr int BT = Sh::BT, ST = Sh::ST, META = Sh::META;
  extern __shared__ uint8_t raw_sm[];
  __shared__ uint64_t kfull[ST], kempty[ST], vfull[ST], vempty[ST], sfull[2], pready[2], metafull[META], qready, drain;
  __shared__ float mx_s[2][kTileRows];
  __shared__ uint32_t tmem_s;
  __shared__ int abort_word, never_s;
  __shared__ Walk walk_s, soft_walk_s;
  __shared__ Segment seg_s;
  __shared__ bool more_s;
  __shared__ uint64_t sight_s[kTileRows];
  volatile int *abort_s = &abort_word;
  uint8_t *sK = reinterpret_cast<uint8_t *>(((uintptr_t)raw_sm + 1023) & ~(uintptr_t)1023);
  uint8_t *sV = sK + ST * Sh::kBytes;
  float4 *fac_s = reinterpret_cast<float4 *>(sV + ST * Sh::kBytes);  // [META][BT / 2]
  __half *q_s = reinterpret_cast<__half *>(fac_s + META * (BT / 2));  // [8 warps][32][kQPitch]
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rows = a.nodes * a.group, row_tiles = (rows + kTileRows - 1) / kTileRows, D = a.head_dim;
  const bool tree = a.parents != nullptr;
  if (warp == 0) {  // this block's share of the units
    const int items = a.kv_heads * row_tiles;
    const long long units = units_before(a, a.batch, BT, items);
    const long long blocks = min((long long)gridDim.x, units);
    long long u0 = 0, u1 = 0;
    if (blockIdx.x < blocks) {
      u0 = units * blockIdx.x / blocks;
      u1 = units * (blockIdx.x + 1) / blocks;
    }
    int b = 0;  // the session that holds unit u0
    long long before = 0;
    if (u1 > u0)
      for (int i0 = 0; i0 < a.batch; i0 += 32) {
        const int n = i0 + lane < a.batch ? session_tiles(a, i0 + lane, BT) : 0;
        long long sum = (long long)n * items;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const long long v = __shfl_up_sync(0xffffffffu, sum, o);
          if (lane >= o) sum += v;
        }
        const unsigned past = __ballot_sync(0xffffffffu, before + sum > u0);
        if (past) {
          const int k = __ffs(past) - 1;
          b = i0 + k;
          before += __shfl_sync(0xffffffffu, sum - (long long)n * items, k);
          break;
        }
        before += __shfl_sync(0xffffffffu, sum, 31);
      }
    if (lane == 0) {
      walk_s = soft_walk_s = Walk{b, u1 > u0 ? session_tiles(a, b, BT) : 1, row_tiles, (int)(u0 - before),
                                  (int)(u1 - u0)};
    }
  }
  if (warp == kMmaWarp) {
    if (lane == 0) {
      for (int i = 0; i < ST; ++i) {
        mbar_init(&kfull[i], kConvThreads / 32);
        mbar_init(&vfull[i], kConvThreads / 32);
        mbar_init(&kempty[i], 1);
        mbar_init(&vempty[i], 1);
      }
      for (int i = 0; i < 2; ++i) {
        mbar_init(&sfull[i], 1);
        mbar_init(&pready[i], 8);
      }
      for (int i = 0; i < META; ++i) mbar_init(&metafull[i], 1);
      mbar_init(&qready, 8);
      mbar_init(&drain, 1);
      abort_word = never_s = 0;
      fence_barrier_init();
    }
    __syncwarp();
    tmem_alloc(&tmem_s, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();

  if (warp < 8) {
    // ---- softmax ----
    constexpr int NT = BT / 2;
    const int quad = warp & 3, half = warp >> 2, r_own = quad * 32 + lane;
    const uint32_t my = tmem_s + ((uint32_t)(quad * 32) << 16);
    __half *stage = q_s + (size_t)warp * 32 * Sh::kQPitch;
    uint32_t g = 0;  // tiles so far
    // After a wait that ran out this role goes on to its end without waiting
    // (the results are void): its warps meet at barriers.
    bool ok = true;
    // The walk and what a segment needs once lie in shared memory: the loop
    // over its tiles wants the registers.
    for (int seg = 0;; ++seg) {
      if (tid == 0) {
        Walk w = soft_walk_s;
        Segment next;
        more_s = w.next(a, BT, next);
        soft_walk_s = w;
        seg_s = next;
      }
      soft_sync();
      if (!more_s) break;
      const int j0 = seg_s.j0, j1 = seg_s.j1, pos = seg_s.pos;
      {
        const int row = seg_s.rt * kTileRows + r_own;
        const Sight sight = sight_of(a, seg_s.b, row < rows ? row / a.group : a.nodes, pos);
        if (half == 0) sight_s[r_own] = tree ? sight.bits : (uint64_t)max(sight.upto, 0);
      }
      float m = kLowest;
      uint64_t l2 = 0;
      // Queries: 32 columns of the warp's 32 rows at a time, four rows a load
      // (8 lanes, four columns each), the halves taking the columns' chunks in
      // turn; as f16 through shared memory to the rows' TMEM lanes.  They are
      // taken as they are where every row's largest magnitude lies well
      // inside f16's range, else again with each row's power of two.
      const int r_sub = lane >> 3, c_sub = 4 * (lane & 7);
      long long at[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = seg_s.rt * kTileRows + quad * 32 + 4 * i + r_sub, n = r / a.group;
        at[i] = r < rows ? ((long long)seg_s.b * a.nodes + n) * a.q_pitch +
                               (long long)(seg_s.kvh * a.group + (r - n * a.group)) * a.q_head + c_sub
                         : -1;
      }
      int qe = 0;
      for (int round = 0; round < 2; ++round) {
        float am[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) am[i] = 0.0f;
        for (int d = 32 * half; d < D; d += 64) {
          float4 x[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            x[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (at[i] < 0 || d + c_sub >= D) continue;
            const size_t o = (size_t)at[i] + d;
            if (!a.q_vec) {
              x[i] = make_float4(load_q(a, o), load_q(a, o + 1), load_q(a, o + 2), load_q(a, o + 3));
            } else if (a.q_bf16) {
              const uint2 v = *reinterpret_cast<const uint2 *>(static_cast<const __nv_bfloat16 *>(a.q) + o);
              x[i] = make_float4(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u),
                                 __uint_as_float(v.y << 16), __uint_as_float(v.y & 0xffff0000u));
            } else {
              x[i] = *reinterpret_cast<const float4 *>(static_cast<const float *>(a.q) + o);
            }
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            am[i] = fmaxf(am[i], fmaxf(fmaxf(fabsf(x[i].x), fabsf(x[i].y)), fmaxf(fabsf(x[i].z), fabsf(x[i].w))));
            const float f = pow2i(-__shfl_sync(0xffffffffu, qe, 4 * i + r_sub));
            *reinterpret_cast<uint2 *>(stage + (4 * i + r_sub) * Sh::kQPitch + c_sub) =
                make_uint2(pack_f16x2(x[i].x * f, x[i].y * f), pack_f16x2(x[i].z * f, x[i].w * f));
          }
          __syncwarp();
          uint32_t w[16];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint4 v = *reinterpret_cast<const uint4 *>(stage + lane * Sh::kQPitch + 8 * i);
            w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
          }
          tmem_st16(my + Sh::kTmemQ + d / 2, w);
          __syncwarp();
        }
        if (round) break;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
#pragma unroll
          for (int o = 4; o > 0; o >>= 1) am[i] = fmaxf(am[i], __shfl_xor_sync(0xffffffffu, am[i], o));
          if ((lane & 7) == 0) mx_s[half][quad * 32 + 4 * i + r_sub] = am[i];
        }
        soft_sync();
        const float big = fmaxf(mx_s[0][r_own], mx_s[1][r_own]);
        if (!soft_any(big != 0.0f && !(big >= 0x1p-3f && big < 0x1p15f))) break;
        qe = q_exponent(big);
      }
      const float f = pow2i(qe) * a.scale_log2;
      tmem_st_wait();
      soft_sync();
      if (lane == 0) mbar_arrive(&qready);
      for (int j = j0; j < j1; ++j, ++g) {
        const int t0 = j * BT;
        const bool open = t0 + BT > pos;
        if (ok)
          ok = mbar_wait(&sfull[g & 1], (g >> 1) & 1, abort_s) &&
               mbar_wait(&metafull[g % META], (g / META) & 1, abort_s);
        if (!ok) give_up(a.error, abort_s);
        __syncwarp();
        tc_fence_after();
        const uint32_t s_tmem = my + Sh::kTmemS + (g & 1) * BT + half * NT;
        const float4 *fac = fac_s + ((size_t)(g % META) * BT + half * NT) / 2;
        uint64_t seen = ~0ull;
        if (open) {
          const uint64_t b = sight_s[r_own];
          seen = Sight{(int)b, b}.seen64(t0 + half * NT, pos, tree);
        }
        uint32_t p[NT / 2];
        // With the maximum so far; where a weight has outgrown it (and for a
        // segment's first tile) the maximum is raised and the weights taken
        // again, once.
        uint64_t l_new;
        for (bool raise = j == j0;;) {
          if (raise) {
            mx_s[half][r_own] = max_pass<NT>(s_tmem, fac, f, seen);
            soft_sync();
            // (a row that has seen nothing yet keeps a floor that no score is under)
            const float mn = fmaxf(m, fmaxf(mx_s[0][r_own], mx_s[1][r_own]));
            const float old = exp2_approx(m - mn);
            m = mn;
            l2 = mul2(l2, pack2(old, old));
            if (j > j0) {  // O of the tiles before takes the new maximum, once they are in it
              const uint32_t q = g - 1;
              if (ok) ok = mbar_wait(&vempty[q % ST], (q / ST) & 1, abort_s);
              if (!ok) give_up(a.error, abort_s);
              __syncwarp();
              tc_fence_after();
#pragma unroll 1
              for (int d = 16 * half; d < D; d += 32) {
                uint32_t r[16];
                tmem_ld16(my + Sh::kTmemO + d, r);
                tmem_ld_wait(r);
#pragma unroll
                for (int i = 0; i < 16; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * old);
                tmem_st16(my + Sh::kTmemO + d, r);
              }
            }
          }
          l_new = l2;
          const float mx = open ? weigh_pass<NT, true>(s_tmem, fac, f, kHead - m, seen, p, l_new)
                                : weigh_pass<NT, false>(s_tmem, fac, f, kHead - m, seen, p, l_new);
          if (raise) {
            soft_sync();
            break;
          }
          raise = soft_any(mx > kMost);
          if (!raise) break;
        }
        l2 = l_new;
        // P goes over the S that both halves have read, by the barriers above
        const uint32_t p_tmem = my + Sh::kTmemS + (g & 1) * BT + half * (NT / 2);
        if constexpr (NT == 64)
          tmem_st32(p_tmem, p);
        else
          tmem_st16(p_tmem, p);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&pready[g & 1]);
      }
      float l0, l1;
      unpack2(l2, l0, l1);
      const size_t slot = (size_t)blockIdx.x * 2 + (seg ? 1 : 0);
      mx_s[half][r_own] = l0 + l1;
      soft_sync();
      if (half == 0)
        a.part_ml[slot * kTileRows + r_own] =
            make_float2(j1 > j0 ? fmaxf(m, kLowest) : -INFINITY, mx_s[0][r_own] + mx_s[1][r_own]);
      if (j1 > j0) {
        const uint32_t q = g - 1;
        if (ok) ok = mbar_wait(&vempty[q % ST], (q / ST) & 1, abort_s);
        if (!ok) give_up(a.error, abort_s);
        __syncwarp();
        tc_fence_after();
        // four columns of 128 rows lie together: a warp stores 512 bytes
        float4 *o = reinterpret_cast<float4 *>(a.part) + slot * (kTileRows * (size_t)D / 4) + r_own;
        for (int d = 32 * half; d < D; d += 64) {
          uint32_t r[32];
          tmem_ld32(my + Sh::kTmemO + d, r);
          tmem_ld_wait(r);
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (d + 4 * i < D)
              o[(size_t)(d / 4 + i) * kTileRows] =
                  make_float4(__uint_as_float(r[4 * i]), __uint_as_float(r[4 * i + 1]),
                              __uint_as_float(r[4 * i + 2]), __uint_as_float(r[4 * i + 3]));
        }
      }
      soft_sync();  // O and mx_s are read: the next segment may overwrite them
    }
  } else if (warp == kMmaWarp) {
    // ---- MMA issue ----
    if (lane == 0) {
      const uint32_t idesc_s = idesc_f16(128, BT, false), idesc_o = idesc_f16(128, D, true);
      const uint32_t tmem = tmem_s;
      Walk walk = walk_s;
      Segment sg;
      uint32_t g = 0;
      bool ok = true;
      auto scores = [&](uint32_t i) {
        const int st = i % ST;
        ok = ok && mbar_wait(&kfull[st], (i / ST) & 1, abort_s);
        // S of tile i lies where P of tile i - 2 was: its product is done
        if (ok && i >= 2) ok = mbar_wait(&vempty[(i - 2) % ST], ((i - 2) / ST) & 1, abort_s);
        if (!ok) return;
        tc_fence_after();
        const uint32_t base = smem_u32(sK + st * Sh::kBytes);
        for (int k = 0; k < D / 16; ++k)
          mma_f16_ts(tmem + Sh::kTmemS + (i & 1) * BT, tmem + Sh::kTmemQ + 8 * k,
                     smem_desc(base + (k >> 2) * (BT * 128) + (k & 3) * 32, 16, 1024, 2), idesc_s, k > 0);
        tc_commit(&kempty[st]);
        tc_commit(&sfull[i & 1]);
      };
      for (int seg = 0; ok && walk.next(a, BT, sg); ++seg) {
        ok = mbar_wait(&qready, seg & 1, abort_s);
        if (!ok) break;
        tc_fence_after();
        const uint32_t g0 = g, g1 = g + max(0, sg.j1 - sg.j0);
        if (g1 > g0) scores(g0);
        for (; ok && g < g1; ++g) {
          if (g + 1 < g1) scores(g + 1);
          const int st = g % ST;
          ok = ok && mbar_wait(&pready[g & 1], (g >> 1) & 1, abort_s) && mbar_wait(&vfull[st], (g / ST) & 1, abort_s);
          if (!ok) break;
          tc_fence_after();
          const uint32_t base = smem_u32(sV + st * Sh::kBytes);
          for (int k = 0; k < BT / 16; ++k)
            mma_f16_ts(tmem + Sh::kTmemO, tmem + Sh::kTmemS + (g & 1) * BT + 8 * k,
                       smem_desc(base + k * 2048, BT * 128, 1024, 2), idesc_o, g > g0 || k > 0);
          tc_commit(&vempty[st]);
        }
      }
      if (!ok) {  // what was issued ends before its TMEM is given back
        give_up(a.error, abort_s);
        tc_commit(&drain);
        mbar_wait(&drain, 0, &never_s);
      }
    }
    __syncwarp();
  } else {
    // ---- codes to f16 tiles ----
    const int ct = tid - kSoftThreads - 32, cw = ct >> 5;
    constexpr int P = Sh::kPieces, X = BT / 32;
    const int per = D / 16;  // pieces a token
    const uint32_t pitch = (uint32_t)(a.kv_heads * D);
    int tok[P];
    uint32_t src[P], dst[P];
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int idx = i * kConvThreads + ct;
      tok[i] = idx / per;
      const int ch = idx - tok[i] * per;
      // the lanes of odd chunks write their second half first, so that eight
      // lanes' 16-byte stores fall on all banks (bit 31 of src)
      const int first = (ch >> 2) & 1;
      src[i] = (uint32_t)tok[i] * pitch + (uint32_t)ch * 16;
      dst[i] = (uint32_t)((ch >> 2) * (BT * 128) + tok[i] * 128 + (((2 * (ch & 3) + first) ^ (tok[i] & 7)) * 16));
      if (first) dst[i] |= 1u << 31;
      if (tok[i] >= BT) tok[i] = 1 << 30;
    }
    Walk ahead = walk_s;
    Segment na;
    bool more = ahead.next(a, BT, na);
    while (more && na.j1 <= na.j0) more = ahead.next(a, BT, na);
    int jn = more ? na.j0 : 0;
    uint4 kb[P], vb[P];
    uint32_t xk[X], xv[X];
    auto load = [&](const uint8_t *codes, uint4(&r)[P]) {
      const uint8_t *c = codes + (((size_t)na.b * a.max_seq + (size_t)jn * BT) * a.kv_heads + na.kvh) * D;
      const int live = min(BT, na.total - jn * BT);
#pragma unroll
      for (int i = 0; i < P; ++i)
        r[i] = tok[i] < live ? load_once(c + src[i]) : make_uint4(0, 0, 0, 0);
    };
    auto load_exps = [&]() {
      const size_t row = ((size_t)na.b * a.max_seq + (size_t)jn * BT) * a.kv_heads + na.kvh;
      const int live = na.total - jn * BT;
#pragma unroll
      for (int i = 0; i < X; ++i) {
        const int t = lane + 32 * i;
        xk[i] = t < live ? a.k_exp[row + (size_t)t * a.kv_heads] : 127;
        xv[i] = t < live ? a.v_exp[row + (size_t)t * a.kv_heads] : 127;
      }
    };
    auto store = [&](uint8_t *stage, const uint4(&v)[P]) {
#pragma unroll
      for (int i = 0; i < P; ++i) {
        if (tok[i] >= BT) continue;
        const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
        uint32_t o[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          o[2 * k] = e4m3x2_to_f16x2((uint16_t)w[k]);
          o[2 * k + 1] = e4m3x2_to_f16x2((uint16_t)(w[k] >> 16));
        }
        const uint4 lo = make_uint4(o[0], o[1], o[2], o[3]), hi = make_uint4(o[4], o[5], o[6], o[7]);
        const bool fl = dst[i] >> 31;
        uint8_t *to = stage + (dst[i] & 0x7fffffffu);
        *reinterpret_cast<uint4 *>(to) = fl ? hi : lo;
        *reinterpret_cast<uint4 *>(stage + ((dst[i] & 0x7fffffffu) ^ 16)) = fl ? lo : hi;
      }
    };
    if (more) {
      load(a.k_codes, kb);
      load(a.v_codes, vb);
      if (cw == 0) load_exps();
    }
    // After a wait that ran out this role goes on to its end without waiting
    // (the results are void): its warps meet at a barrier in open tiles.
    bool ok = true;
    for (uint32_t g = 0; more; ++g) {
      const int st = g % ST;
      const bool open = (jn + 1) * BT > na.pos;
      float *ft = reinterpret_cast<float *>(fac_s + (size_t)(g % META) * (BT / 2));
      if (g >= ST && ok) ok = mbar_wait(&kempty[st], ((g / ST) - 1) & 1, abort_s);
      if (!ok) give_up(a.error, abort_s);
      __syncwarp();
      if (cw == 0) {
#pragma unroll
        for (int i = 0; i < X; ++i) {
          const int t = lane + 32 * i;
          ft[(t >> 1) * 4 + (t & 1)] = kv8_factor(xk[i]);
          ft[(t >> 1) * 4 + 2 + (t & 1)] = pow2i((int)kv8_value_exponent(xv[i]));
        }
      }
      if (open) {  // values that are not a number: zero in the product, and the token's score NaN for those who see it
        conv_sync();
#pragma unroll
        for (int i = 0; i < P; ++i) {
          uint32_t w[4] = {vb[i].x, vb[i].y, vb[i].z, vb[i].w}, any = 0;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t bad = __vcmpeq4(w[k] & 0x7f7f7f7fu, 0x7f7f7f7fu);
            w[k] &= ~bad;
            any |= bad;
          }
          vb[i] = make_uint4(w[0], w[1], w[2], w[3]);
          if (any && tok[i] < BT) ft[(tok[i] >> 1) * 4 + (tok[i] & 1)] = __int_as_float(0x7fc00000);
        }
        conv_sync();
      }
      __syncwarp();
      if (cw == 0 && lane == 0) mbar_arrive(&metafull[g % META]);
      store(sK + st * Sh::kBytes, kb);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&kfull[st]);
      // the next tile's keys are on their way while this one's values are stored
      if (jn + 1 >= na.j1) {
        more = ahead.next(a, BT, na);
        while (more && na.j1 <= na.j0) more = ahead.next(a, BT, na);
        jn = more ? na.j0 : 0;
      } else {
        ++jn;
      }
      if (more) {
        load(a.k_codes, kb);
        if (cw == 0) load_exps();
      }
      if (g >= ST && ok) ok = mbar_wait(&vempty[st], ((g / ST) - 1) & 1, abort_s);
      if (!ok) give_up(a.error, abort_s);
      __syncwarp();
      store(sV + st * Sh::kBytes, vb);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&vfull[st]);
      if (more) load(a.v_codes, vb);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem_s, 512);
  }
}

// The blocks that share a row tile's tokens meet, in order, with the gate:
// block (16 rows of a row tile, 64 columns); thread (row, four columns, one of
// four shares of the blocks).  Rows of nodes that are not there become zeros.
constexpr int kMergeThreads = 1024, kMergeShares = 4;
__global__ void __launch_bounds__(kMergeThreads, 1) tree_attn_tile_merge_kernel(const __grid_constant__ TreeArgs a,
                                                                             int BT, int grid) {
  pdl_enter();
  __shared__ float4 acc_s[kMergeShares - 1][256];
  __shared__ float2 ml_s[kMergeShares - 1][256];
  const int tid = threadIdx.x, share = tid >> 8, t = tid & 255, D = a.head_dim;
  const int rows = a.nodes * a.group, row_tiles = (rows + kTileRows - 1) / kTileRows, items = a.kv_heads * row_tiles;
  const int item = blockIdx.x / (kTileRows / 16), r = blockIdx.x % (kTileRows / 16) * 16 + (t & 15);
  const int b = item / items, kvh = item % items / row_tiles, row = item % row_tiles * kTileRows + r;
  const int d = blockIdx.y * 64 + 4 * (t >> 4);
  const bool live = row < rows && d < D;
  const int n = row / a.group, h = kvh * a.group + row % a.group;
  const int tiles = session_tiles(a, b, BT);
  float m = -INFINITY, l = 0.0f;
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (tiles > 0) {
    const long long before = units_before(a, b, BT, items), units = units_before(a, a.batch, BT, items);
    const long long blocks = min((long long)grid, units);
    const long long ua = before + (long long)(item % items) * tiles, ub = ua + tiles;
    const int c0 = (int)(((ua + 1) * blocks - 1) / units), c1 = (int)((ub * blocks - 1) / units);
    // the block that the row tile begins in holds it as a later segment, unless it begins there
    const int first = units * c0 / blocks < ua ? 1 : 0;
    const float4 *part = reinterpret_cast<const float4 *>(a.part);
#pragma unroll 4
    for (int c = c0 + share; c <= c1; c += kMergeShares) {
      const size_t slot = (size_t)c * 2 + (c == c0 ? first : 0);
      const float2 v = a.part_ml[slot * kTileRows + r];
      if (v.x == -INFINITY || !live) continue;
      const float4 x = part[slot * (kTileRows * (size_t)D / 4) + (size_t)(d / 4) * kTileRows + r];
      const float mn = fmaxf(m, v.x), fo = exp2_approx(m - mn), fn = exp2_approx(v.x - mn);
      l = l * fo + v.y * fn;
      acc.x = acc.x * fo + x.x * fn;
      acc.y = acc.y * fo + x.y * fn;
      acc.z = acc.z * fo + x.z * fn;
      acc.w = acc.w * fo + x.w * fn;
      m = mn;
    }
  }
  if (share > 0) {
    acc_s[share - 1][t] = acc;
    ml_s[share - 1][t] = make_float2(m, l);
  }
  __syncthreads();
  if (share > 0) return;
  const bool there = tiles > 0 && sight_of(a, b, row < rows ? n : a.nodes, a.positions[b]).upto >= 0;
  if (!live) return;
  for (int i = 0; i < kMergeShares - 1; ++i) {
    const float2 v = ml_s[i][t];
    if (v.x == -INFINITY) continue;
    const float4 x = acc_s[i][t];
    const float mn = fmaxf(m, v.x), fo = m == -INFINITY ? 0.0f : exp2_approx(m - mn), fn = exp2_approx(v.x - mn);
    l = l * fo + v.y * fn;
    acc.x = acc.x * fo + x.x * fn;
    acc.y = acc.y * fo + x.y * fn;
    acc.z = acc.z * fo + x.z * fn;
    acc.w = acc.w * fo + x.w * fn;
    m = mn;
  }
  const size_t node = (size_t)b * a.nodes + n;
  float o[4] = {acc.x, acc.y, acc.z, acc.w};
  const float inv = 1.0f / l;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    o[i] = there ? o[i] * inv : 0.0f;
    if (there && a.gate) o[i] /= 1.0f + expf(-a.gate[node * a.gate_pitch + (size_t)h * a.gate_head + d + i]);
  }
  *reinterpret_cast<uint2 *>(a.out + (node * a.q_heads + h) * D + d) =
      make_uint2(pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3]));
}

// How a call is cut.  tiles: the tcgen05 kernel, `blocks` of them; else rows a
// tile, tiles and splits of the tokens.
struct Plan {
  bool tiles;
  int rows_tile, splits, blocks, BT;
  size_t items, units;
};

Plan plan_for(size_t batch, size_t nodes, size_t q_heads, size_t kv_heads, size_t head_dim, size_t max_seq) {
  Plan p{};
  const size_t rows = nodes * (q_heads / kv_heads);
  if (rows > 16) {
    p.tiles = true;
    p.BT = head_dim > 128 ? 64 : 128;
    p.items = batch * kv_heads * ((rows + kTileRows - 1) / kTileRows);
    const size_t most = p.items * ((max_seq + p.BT - 1) / p.BT);
    p.units = most;
    p.blocks = (int)std::min<size_t>(sm_count(), most);
    return p;
  }
  p.rows_tile = rows <= 8 ? 8 : 16;
  p.items = batch * kv_heads * ((rows + p.rows_tile - 1) / p.rows_tile);
  // two blocks an SM; at least 64 tokens a split (a step for each warp)
  const size_t want = ((size_t)sm_count() * 2 + p.items - 1) / p.items;
  p.splits = (int)std::max<size_t>(1, std::min(want, (max_seq + 63) / 64));
  return p;
}

template <int DP>
int run_tiles(const TreeArgs &a, const Plan &p, cudaStream_t s) {
  constexpr size_t smem = TileShape<DP>::smem;
  {
    static std::mutex mu;
    static std::vector<int> done;
    int dev = 0;
    FPB_CUDA_TRY(cudaGetDevice(&dev));
    std::lock_guard<std::mutex> lock(mu);
    if (std::find(done.begin(), done.end(), dev) == done.end()) {
      FPB_CUDA_TRY(cudaFuncSetAttribute(tree_attn_tile_kernel<DP>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        (int)smem));
      done.push_back(dev);
    }
  }
  cudaError_t e = launch_pdl(tree_attn_tile_kernel<DP>, dim3((unsigned)p.blocks), kTileThreads, smem, s, a);
  if (e != cudaSuccess) return cuda_fail(e, "tree_attn_tile_kernel");
  FPB_LAUNCH_CHECK("tree_attn_tile_kernel");
  e = launch_pdl(tree_attn_tile_merge_kernel,
                 dim3((unsigned)(p.items * (kTileRows / 16)), (unsigned)((a.head_dim + 63) / 64)), kMergeThreads, 0, s, a,
                 p.BT, p.blocks);
  if (e != cudaSuccess) return cuda_fail(e, "tree_attn_tile_merge_kernel");
  FPB_LAUNCH_CHECK("tree_attn_tile_merge_kernel");
  return FPB_OK;
}

template <int DP, int NR>
int run_rows(const TreeArgs &a, const Plan &p, cudaStream_t s) {
  constexpr size_t smem = std::max(RowsShape<DP, NR>::smem, (size_t)NR * RowsShape<DP, NR>::kQPitch * 2);
  if (smem > 40 * 1024) {
    static std::mutex mu;
    static std::vector<int> done;
    int dev = 0;
    FPB_CUDA_TRY(cudaGetDevice(&dev));
    std::lock_guard<std::mutex> lock(mu);
    if (std::find(done.begin(), done.end(), dev) == done.end()) {
      FPB_CUDA_TRY(cudaFuncSetAttribute(tree_attn_rows_kernel<DP, NR>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        (int)smem));
      done.push_back(dev);
    }
  }
  cudaError_t e = launch_pdl(tree_attn_rows_kernel<DP, NR>, dim3((unsigned)p.splits, (unsigned)p.items), kRowsThreads,
                             smem, s, a);
  if (e != cudaSuccess) return cuda_fail(e, "tree_attn_rows_kernel");
  FPB_LAUNCH_CHECK("tree_attn_rows_kernel");
  return FPB_OK;
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace fpb

using namespace fpb;

extern "C" size_t fpb_tree_attn_workspace_bytes(size_t batch, size_t nodes, size_t q_heads, size_t kv_heads,
                                                size_t head_dim, size_t max_seq) {
  if (batch == 0 || nodes == 0 || kv_heads == 0 || q_heads == 0 || q_heads % kv_heads) return 16;
  const Plan p = plan_for(batch, nodes, q_heads, kv_heads, head_dim, max_seq);
  if (p.tiles) return (size_t)p.blocks * 2 * kTileRows * (head_dim + 2) * sizeof(float);
  return p.splits == 1 ? 16 : p.items * p.splits * p.rows_tile * (head_dim + 2) * sizeof(float);
}

extern "C" int fpb_tree_attn(const void *q, int q_dtype, size_t q_pitch, size_t q_head_pitch, const uint8_t *k_codes,
                             const uint8_t *v_codes, const uint8_t *k_exp, const uint8_t *v_exp,
                             const int32_t *positions, const int32_t *parents, const float *gate, size_t gate_pitch,
                             size_t gate_head_pitch, size_t batch, size_t nodes, size_t q_heads, size_t kv_heads,
                             size_t head_dim, size_t max_seq, float scale, void *workspace, size_t workspace_bytes,
                             void *out_bf16, void *stream) {
  if (!q || !k_codes || !v_codes || !k_exp || !v_exp || !positions || !workspace || !out_bf16)
    return fail(FPB_ERR_INVALID_ARGUMENT, "fpb_tree_attn: null pointer");
  if (q_dtype != FPB_F32 && q_dtype != FPB_BF16) return fail(FPB_ERR_INVALID_ARGUMENT, "fpb_tree_attn: dtype");
  if (batch == 0 || batch > 65535 || kv_heads == 0 || kv_heads > 4096 || q_heads == 0 || q_heads % kv_heads ||
      q_heads > 65535 || head_dim == 0 || head_dim > 256 || head_dim % 16 || max_seq == 0 || max_seq > (1u << 30))
    return fail(FPB_ERR_SHAPE, "fpb_tree_attn: shape (batch %zu, heads %zu / %zu, head_dim %zu: a multiple of 16 up "
                "to 256, max_seq %zu)", batch, q_heads, kv_heads, head_dim, max_seq);
  if (nodes == 0 || nodes > max_seq || batch * nodes > 65535 || (parents && nodes > (size_t)kTreeMaxNodes))
    return fail(FPB_ERR_SHAPE, "fpb_tree_attn: nodes %zu (a tree has at most %d)", nodes, kTreeMaxNodes);
  if (q_head_pitch < head_dim || (gate && gate_head_pitch < head_dim) || !std::isfinite(scale))
    return fail(FPB_ERR_SHAPE, "fpb_tree_attn: pitches or scale");
  if (!aligned16(k_codes) || !aligned16(v_codes) || !aligned16(workspace) || !aligned16(out_bf16) ||
      reinterpret_cast<uintptr_t>(q) % (q_dtype == FPB_F32 ? 4 : 2) || reinterpret_cast<uintptr_t>(gate) % 4)
    return fail(FPB_ERR_INVALID_ARGUMENT, "fpb_tree_attn: alignment (codes, workspace and out: 16 bytes)");
  const size_t need = fpb_tree_attn_workspace_bytes(batch, nodes, q_heads, kv_heads, head_dim, max_seq);
  if (workspace_bytes < need)
    return fail(FPB_ERR_WORKSPACE, "fpb_tree_attn: workspace %zu < %zu bytes", workspace_bytes, need);
  const Plan p = plan_for(batch, nodes, q_heads, kv_heads, head_dim, max_seq);
  if (p.items > 65535 || p.units > 0x7fffffff)
    return fail(FPB_ERR_SHAPE, "fpb_tree_attn: %zu tiles of rows in one call (at most 65535, and 2^31 with their tiles "
                "of tokens)", p.items);
  TreeArgs a{};
  a.q = q;
  a.gate = gate;
  a.k_codes = k_codes;
  a.v_codes = v_codes;
  a.k_exp = k_exp;
  a.v_exp = v_exp;
  a.positions = positions;
  a.parents = parents;
  a.q_pitch = (long long)q_pitch;
  a.q_head = (long long)q_head_pitch;
  a.gate_pitch = (long long)gate_pitch;
  a.gate_head = (long long)gate_head_pitch;
  a.batch = (int)batch;
  a.nodes = (int)nodes;
  a.q_heads = (int)q_heads;
  a.kv_heads = (int)kv_heads;
  a.group = (int)(q_heads / kv_heads);
  a.head_dim = (int)head_dim;
  a.max_seq = (int)max_seq;
  a.q_bf16 = q_dtype == FPB_BF16;
  a.q_vec = aligned16(q) && (q_pitch | q_head_pitch) * (q_dtype == FPB_F32 ? 4 : 2) % 16 == 0;
  a.splits = p.splits;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.out = static_cast<__nv_bfloat16 *>(out_bf16);
  a.part = static_cast<float *>(workspace);
  a.part_ml = reinterpret_cast<float2 *>(
      a.part + (p.tiles ? (size_t)p.blocks * 2 * kTileRows : p.items * p.splits * p.rows_tile) * head_dim);
  a.error = device_error_ptr();
  cudaStream_t s = as_stream(stream);
  if (p.tiles)
    return head_dim <= 64 ? run_tiles<64>(a, p, s) : head_dim <= 128 ? run_tiles<128>(a, p, s) : run_tiles<256>(a, p, s);
  const bool few = p.rows_tile == 8;
  const int st = head_dim <= 64    ? (few ? run_rows<64, 8>(a, p, s) : run_rows<64, 16>(a, p, s))
                 : head_dim <= 128 ? (few ? run_rows<128, 8>(a, p, s) : run_rows<128, 16>(a, p, s))
                                   : (few ? run_rows<256, 8>(a, p, s) : run_rows<256, 16>(a, p, s));
  if (st || p.splits == 1) return st;
  const int count = (int)(batch * nodes * q_heads);
  cudaError_t e = launch_pdl(tree_attn_merge_kernel, dim3((unsigned)((count + 7) / 8)), 256, 0, s, a, p.rows_tile,
                             count);
  if (e != cudaSuccess) return cuda_fail(e, "tree_attn_merge_kernel");
  FPB_LAUNCH_CHECK("tree_attn_merge_kernel");
  return FPB_OK;
}
