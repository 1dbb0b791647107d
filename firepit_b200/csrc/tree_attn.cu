// Attention of a tree of drafted tokens over the 8-bit cache (kv8.cuh).
//
// Node i of session b sees the cache rows before position[b], its ancestors'
// rows and its own (row position + j of node j).  With s_t = scale q . k_t:
//   out = sum_t softmax(s)_t v_t, times sigmoid(gate) where a gate is given.
#include <algorithm>
#include <cmath>
#include <mutex>
#include <vector>

#include "sm100.cuh"
#include "tma_host.cuh"
#include "tree_attn.cuh"

namespace fpb {
namespace {

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

using namespace sm100;

// ---- few rows: warps that stream tokens on their own -------------------------------------------
// Block (split, session * kv head): NR rows (8 or 16) of one kv head, four
// warps that take steps of 16 tokens in turn.  Each warp has its own ring of
// kRowsStages steps of codes, filled by TMA (128-byte swizzle: its 16-byte
// reads fall on distinct banks), so that 24 KB a warp are on their way however
// long a step takes; nothing is shared between the warps before the end.
//  S = Q K^T   m16n8k16, the rows as M (NR = 8 leaves half of it zero).  The
//              order of the summed dimension is free as long as both sides
//              agree, so a lane's 16-byte piece of a key (16 dimensions) is
//              its operand of four instructions as it lies.
//  O^T = V^T P^T  the dimensions as M, the rows as N: P^T's operand is S's
//              result as it lies.  V's needs pairs of tokens in a word: byte
//              permutes of two tokens' pieces before the conversion.
// Each e4m3 is converted to f16 (exact); the key's factor goes to the score,
// the value's to the weight's exponent.
constexpr int kRowsThreads = 128, kRowsWarps = 4, kRowsStages = 3;
constexpr int kErrRowsWait = 503;

template <int DP, int NR>
struct RowsShape {
  static constexpr bool kQShared = NR * DP > 16 * 128;  // 64 registers of queries are too many beside 128 of sums
  static constexpr int kQPitch = DP + 8;                // f16 elements: 16-byte reads of eight rows on distinct banks
  static constexpr int kBox = DP == 64 ? 64 : 128;
  static constexpr uint32_t kStage = 2 * 16 * DP;  // a step's codes, keys then values
  static constexpr size_t kRing = (size_t)kRowsWarps * kRowsStages * kStage;
  static constexpr size_t kEnd = (size_t)kRowsWarps * NR * (DP + 2) * 4;  // the warps' results, over the ring
  static constexpr size_t kQueries = (size_t)NR * kQPitch * 2;
  static constexpr size_t smem = 1023 + (kRing > kEnd ? kRing : kEnd) + kQueries;
};

template <int DP, int NR>
__global__ void __launch_bounds__(kRowsThreads, 2)
    tree_attn_rows_kernel(const __grid_constant__ TreeArgs a, const __grid_constant__ CUtensorMap k_map,
                          const __grid_constant__ CUtensorMap v_map) {
  using Sh = RowsShape<DP, NR>;
  constexpr int kPieces = DP / 64, kVPieces = DP >= 128 ? DP / 128 : 1, kVBytes = DP >= 128 ? 16 : 8;
  constexpr int kMT = DP / 16, kNT = NR / 8;
  extern __shared__ uint8_t raw_sm[];
  uint8_t *const ring = raw_sm + (-smem_u32(raw_sm) & 1023);  // the swizzle goes by the address
  float *const sm = reinterpret_cast<float *>(ring);  // at the end: the warps' results
  __half *const qs = reinterpret_cast<__half *>(ring + (Sh::kRing > Sh::kEnd ? Sh::kRing : Sh::kEnd));
  __shared__ uint64_t full[kRowsWarps][kRowsStages];
  __shared__ int abort_s;
  __shared__ float m_s[kRowsWarps][NR], l_s[kRowsWarps][NR];
  __shared__ float fac_s[NR];
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, g = lane >> 2, c = lane & 3;
  const int rows = a.nodes * a.group;
  const int item = blockIdx.y, b = item / a.kv_heads, kvh = item % a.kv_heads, D = a.head_dim;
  if (lane == 0) {
    for (int i = 0; i < kRowsStages; ++i) mbar_init(&full[w][i], 1);
    if (w == 0) abort_s = 0;
    fence_barrier_init();
  }
  __syncwarp();
  pdl_enter();
  const int pos = a.positions[b];
  const bool tree = a.parents != nullptr;
  const int total = seen_rows(a, pos, a.nodes - 1);
  // this split's tokens, in whole steps
  const int steps = (total + 15) / 16, per = (steps + a.splits - 1) / a.splits;
  const int s0 = blockIdx.x * per, s1 = min(steps, s0 + per);

  // the ring's first steps are on their way before anything else
  const int first = s0 + w, boxes = (D + Sh::kBox - 1) / Sh::kBox;
  uint8_t *const mine_ring = ring + (size_t)w * kRowsStages * Sh::kStage;
  auto fetch = [&](int i) {  // the warp's i-th step, one lane
    uint8_t *to = mine_ring + (i % kRowsStages) * Sh::kStage;
    uint64_t *bar = &full[w][i % kRowsStages];
    const int t0 = (first + i * kRowsWarps) * 16;
    mbar_arrive_expect_tx(bar, 2u * boxes * (16 * Sh::kBox));
    for (int x = 0; x < boxes; ++x) {
      tma_load_4d(to + x * (16 * Sh::kBox), &k_map, x * Sh::kBox, kvh, t0, b, bar);
      tma_load_4d(to + Sh::kStage / 2 + x * (16 * Sh::kBox), &v_map, x * Sh::kBox, kvh, t0, b, bar);
    }
  };
  const int count = first < s1 ? (s1 - first + kRowsWarps - 1) / kRowsWarps : 0;
  if (lane == 0)
    for (int i = 0; i < min(count, kRowsStages); ++i) fetch(i);
  __syncwarp();

  // queries: a warp takes rows w, w + 4, ...; eight columns a lane
  for (int r = w; r < NR; r += kRowsWarps) {
    const int row = r, n = row / a.group, h = kvh * a.group + row % a.group;
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
    const int row = g + 8 * i;
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

  const uint8_t *ex = (lane < 16 ? a.k_exp : a.v_exp) + (size_t)b * a.max_seq * a.kv_heads + kvh;
  auto load_exp = [&](int step) -> uint32_t {
    const int t = step * 16 + (lane & 15);
    return t < total ? ex[(size_t)t * a.kv_heads] : 127;
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
  uint32_t xr = count > 0 ? load_exp(first) : 127;
  bool ok = true;
  for (int i = 0; i < count; ++i) {
    const int step = first + i * kRowsWarps;
    const uint8_t *kst = mine_ring + (i % kRowsStages) * Sh::kStage, *vst = kst + Sh::kStage / 2;
    if (ok) ok = mbar_wait(&full[w][i % kRowsStages], (i / kRowsStages) & 1, &abort_s);
    if (!ok && a.error) {  // (a wait that ran out: the results are void, but the loop ends)
      *(volatile int *)&abort_s = 1;
      atomicCAS(a.error, 0, kErrRowsWait);
    }
    __syncwarp();
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
        const int at = DP == 64 ? (8 * u + g) * 64 + ((c ^ ((g >> 1) & 3)) * 16)
                                : (p >> 1) * 2048 + (8 * u + g) * 128 + (((4 * (p & 1) + c) ^ g) * 16);
        const uint4 kv = *reinterpret_cast<const uint4 *>(kst + at);
        const uint32_t kw[4] = {kv.x, kv.y, kv.z, kv.w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
          mma_f16(s[u], q0[2 * j], q1[2 * j], q0[2 * j + 1], q1[2 * j + 1], e4m3x2_to_f16x2((uint16_t)kw[j]),
                  e4m3x2_to_f16x2((uint16_t)(kw[j] >> 16)));
      }
    }
    const uint32_t xb = xr;
    const int t0 = step * 16;
    const bool open = t0 + 16 > pos;  // warp-uniform: the tree's rows, or the end
    if (i + 1 < count) xr = load_exp(step + kRowsWarps);
    uint32_t vr[4][kVPieces][kVBytes / 4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int row = 2 * c + (t & 1) + 8 * (t >> 1);
#pragma unroll
      for (int p = 0; p < kVPieces; ++p) {
        if constexpr (kVBytes == 16) {
          const uint4 v = *reinterpret_cast<const uint4 *>(vst + p * 2048 + row * 128 + ((g ^ (row & 7)) * 16));
          vr[t][p][0] = v.x; vr[t][p][1] = v.y; vr[t][p][2] = v.z; vr[t][p][3] = v.w;
        } else {
          const uint2 v = *reinterpret_cast<const uint2 *>(vst + row * 64 + (((g >> 1) ^ ((row >> 1) & 3)) * 16) + (g & 1) * 8);
          vr[t][p][0] = v.x; vr[t][p][1] = v.y;
        }
      }
    }
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
    __syncwarp();  // the stage is read
    if (lane == 0 && i + kRowsStages < count) fetch(i + kRowsStages);
    __syncwarp();
  }
  if (!ok)  // copies still in flight land before the block ends
    for (int i = 0; i < kRowsStages; ++i) {
      int never = 0;
      for (uint32_t k = 0; k < 2; ++k) mbar_wait(&full[w][i], k, &never);
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
    const int row = r;
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

// How a call of few rows is cut: rows a tile, tiles, splits of the tokens.
struct Plan {
  int rows_tile, splits;
  size_t items;
};

// Rows a key/value head from which the tcgen05 kernel takes over.
bool wants_tiles(size_t nodes, size_t q_heads, size_t kv_heads) { return nodes * (q_heads / kv_heads) > 16; }

Plan plan_for(size_t batch, size_t nodes, size_t q_heads, size_t kv_heads, size_t max_seq) {
  Plan p{};
  const size_t rows = nodes * (q_heads / kv_heads);
  p.rows_tile = rows <= 8 ? 8 : 16;
  p.items = batch * kv_heads;
  // two blocks an SM; at least 64 tokens a split (a step for each warp)
  const size_t want = std::max<size_t>(1, (size_t)sm_count() * 2 / p.items);  // one wave
  p.splits = (int)std::max<size_t>(1, std::min(want, (max_seq + 63) / 64));
  return p;
}

template <int DP, int NR>
int run_rows(const TreeArgs &a, const Plan &p, cudaStream_t s) {
  using Sh = RowsShape<DP, NR>;
  {
    static std::mutex mu;
    static std::vector<int> done;
    int dev = 0;
    FPB_CUDA_TRY(cudaGetDevice(&dev));
    std::lock_guard<std::mutex> lock(mu);
    if (std::find(done.begin(), done.end(), dev) == done.end()) {
      FPB_CUDA_TRY(cudaFuncSetAttribute(tree_attn_rows_kernel<DP, NR>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        (int)Sh::smem));
      done.push_back(dev);
    }
  }
  CUtensorMap k_map, v_map;
  if (int st = encode_cache_u8(&k_map, a.k_codes, a.batch, a.max_seq, a.kv_heads, a.head_dim, Sh::kBox, 16)) return st;
  if (int st = encode_cache_u8(&v_map, a.v_codes, a.batch, a.max_seq, a.kv_heads, a.head_dim, Sh::kBox, 16)) return st;
  cudaError_t e = launch_pdl(tree_attn_rows_kernel<DP, NR>, dim3((unsigned)p.splits, (unsigned)p.items), kRowsThreads,
                             Sh::smem, s, a, k_map, v_map);
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
  if (wants_tiles(nodes, q_heads, kv_heads))
    return tile_workspace_bytes(tile_plan(batch, nodes, q_heads, kv_heads, head_dim, max_seq), head_dim);
  const Plan p = plan_for(batch, nodes, q_heads, kv_heads, max_seq);
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
  a.scale_log2 = scale * 1.4426950408889634f;
  a.out = static_cast<__nv_bfloat16 *>(out_bf16);
  a.error = device_error_ptr();
  cudaStream_t s = as_stream(stream);
  if (wants_tiles(nodes, q_heads, kv_heads)) {
    const TilePlan p = tile_plan(batch, nodes, q_heads, kv_heads, head_dim, max_seq);
    if (p.items > 65535 || p.units > 0x7fffffff)
      return fail(FPB_ERR_SHAPE, "fpb_tree_attn: %zu tiles of rows in one call (at most 65535, and 2^31 with their "
                  "tiles of tokens)", p.items);
    return run_tree_tiles(a, p, workspace, s);
  }
  const Plan p = plan_for(batch, nodes, q_heads, kv_heads, max_seq);
  if (p.items > 65535) return fail(FPB_ERR_SHAPE, "fpb_tree_attn: %zu key/value heads in one call", p.items);
  a.splits = p.splits;
  a.part = static_cast<float *>(workspace);
  a.part_ml = reinterpret_cast<float2 *>(a.part + p.items * p.splits * p.rows_tile * head_dim);
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
