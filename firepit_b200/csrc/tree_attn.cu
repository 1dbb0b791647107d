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

// An 8 x 8 matrix of f16 pairs (lane 4 r + c: row r, columns 2 c and 2 c + 1), transposed.
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

using namespace sm100;

// ---- few rows: warps that stream tokens on their own -------------------------------------------
// Block (split, session * kv head): NR rows (8 or 16) of one kv head, four
// warps that take steps of 16 tokens in turn.  Each warp has its own ring of
// kStages steps of codes, filled by TMA, so that up to 16 KB a warp are on their
// way however long a step takes (three stages: 21.4 us instead of 20.9 at 8 x
// 8192 x 256, 56.4 instead of 52.5 at 8 x 65536 x 128); nothing is shared between
// the warps before the end.
//  S^T = K Q^T  m16n8k16, the tokens as M, the rows as N.  The order of the
//               summed dimension is free as long as both sides agree, so a
//               lane's 16-byte piece of a key (16 dimensions) is its operand
//               of four instructions as it lies.
//  O^T = V^T P^T  the dimensions as M, the rows as N: P^T's operand is S^T's
//               result, transposed eight by eight.  V's needs pairs of tokens
//               in a word: byte permutes of two tokens' pieces before the
//               conversion.
// Row i of an operand of eight is token token_at(i), and piece i of a value
// piece_at(i): a quarter of a warp then reads 16 bytes from all of the banks.
// Each e4m3 is converted to f16 (exact); the key's factor goes to the score,
// the value's to the weight's exponent.
// The tokens as M, not the rows: eight rows take half as many instructions, and
// a token's exponents belong to one lane (8 x 8192 tokens x 2 heads x 256, 16
// rows: 27.9 us against 32 with the rows as M; 24.5 now).
// Long caches are bound by their bytes (from 8 x 16384 to 8 x 32768 tokens, 8 rows
// x 256: 134 MB more in 20 us, 6.7 TB/s), shorter ones by some 10 us besides:
// the launches, the start (positions, then the first codes), the last steps'
// latency, the splits' results and their merge.  16 x 1 node x 16 heads (2 kv) x
// 256, 8192 tokens: 30.4 us, 3.9 TB/s.
constexpr int kRowsThreads = 128, kRowsWarps = 4;
constexpr int kErrRowsWait = 503;

// Blocks an SM.  Their registers would allow three at 256 columns and eight
// rows, and four at fewer columns, but more splits cost the merge what they
// gain (1 x 30000, 256 columns: 20.7 us with two, 23.7 with three; 8 x 8192, 64
// columns, 16 rows: 19.7 us with two, 17.7 with three, 18.3 with four).
constexpr int rows_blocks(int DP) { return DP == 256 ? 2 : 3; }

template <int DP, int NR>
struct RowsShape {
  static constexpr int kBlocks = rows_blocks(DP), kStages = 2;
  static constexpr bool kQShared = NR * DP > 16 * 128;  // 64 registers of queries are too many beside 128 of sums
  static constexpr int kQPitch = DP + 8;                // f16 elements: 16-byte reads of eight rows on distinct banks
  static constexpr int kBox = DP == 64 ? 64 : 128;
  static constexpr uint32_t kStage = 2 * 16 * DP;  // a step's codes, keys then values
  static constexpr size_t kRing = (size_t)kRowsWarps * kStages * kStage;
  static constexpr size_t kEnd = (size_t)kRowsWarps * NR * (DP + 2) * 4;  // the warps' results, over the ring
  static constexpr size_t kQueries = (size_t)NR * kQPitch * 2;
  static constexpr size_t smem = 1023 + (kRing > kEnd ? kRing : kEnd) + kQueries;
};

// Steps of a split: what the call's splits share of a session's, in whole
// rounds of a block's warps; a session of few tokens leaves splits unused (1000
// tokens in a cache of 32768: 7.8 us, 9.1 with 63 splits of one step; elsewhere
// alike).
__device__ __forceinline__ int steps_a_split(int steps, int splits) {
  return ((steps + splits - 1) / splits + kRowsWarps - 1) / kRowsWarps * kRowsWarps;
}

template <int DP>
__device__ __forceinline__ int token_at(int i) {
  return DP == 64 ? i ^ ((i >> 1) & 1) : (i >> 1) | (i & 1) << 2;
}
template <int DP>
__device__ __forceinline__ int piece_at(int i) {
  return DP == 64 ? i : token_at<DP>(i);
}

template <int DP, int NR>
__global__ void __launch_bounds__(kRowsThreads, (RowsShape<DP, NR>::kBlocks))
    tree_attn_rows_kernel(const __grid_constant__ TreeArgs a, const __grid_constant__ CUtensorMap k_map,
                          const __grid_constant__ CUtensorMap v_map) {
  using Sh = RowsShape<DP, NR>;
  constexpr int kStages = Sh::kStages, kPieces = DP / 64, kVPieces = DP >= 128 ? DP / 128 : 1, kVBytes = DP >= 128 ? 16 : 8;
  constexpr int kMT = DP / 16, kNT = NR / 8;
  extern __shared__ uint8_t raw_sm[];
  uint8_t *const ring = raw_sm + (-smem_u32(raw_sm) & 1023);  // the swizzle goes by the address
  float *const sm = reinterpret_cast<float *>(ring);  // at the end: the warps' results
  __half *const qs = reinterpret_cast<__half *>(ring + (Sh::kRing > Sh::kEnd ? Sh::kRing : Sh::kEnd));
  __shared__ uint64_t full[kRowsWarps][kStages];
  __shared__ int abort_s;
  __shared__ float m_s[kRowsWarps][NR], l_s[kRowsWarps][NR];
  __shared__ float fac_s[NR];
  __shared__ Sight sight_s[NR];
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, g = lane >> 2, c = lane & 3;
  const int rows = a.nodes * a.group;
  const int item = blockIdx.y, b = item / a.kv_heads, kvh = item % a.kv_heads, D = a.head_dim;
  if (lane == 0) {
    for (int i = 0; i < kStages; ++i) mbar_init(&full[w][i], 1);
    if (w == 0) abort_s = 0;
    fence_barrier_init();
  }
  __syncwarp();
  pdl_enter();
  const int pos = a.positions[b];
  const bool tree = a.parents != nullptr;
  const int total = seen_rows(a, pos, a.nodes - 1);
  // this split's tokens, in whole steps
  const int steps = (total + 15) / 16, per = steps_a_split(steps, a.splits);
  const int s0 = blockIdx.x * per, s1 = min(steps, s0 + per);
  if (blockIdx.x > 0 && s0 >= steps) return;

  // the ring's first steps are on their way before anything else
  const int first = s0 + w, boxes = (D + Sh::kBox - 1) / Sh::kBox;
  uint8_t *const mine_ring = ring + (size_t)w * kStages * Sh::kStage;
  auto fetch = [&](int i) {  // the warp's i-th step, one lane
    uint8_t *to = mine_ring + (i % kStages) * Sh::kStage;
    uint64_t *bar = &full[w][i % kStages];
    const int t0 = (first + i * kRowsWarps) * 16;
    mbar_arrive_expect_tx(bar, 2u * boxes * (16 * Sh::kBox));
    for (int x = 0; x < boxes; ++x) {
      tma_load_4d(to + x * (16 * Sh::kBox), &k_map, x * Sh::kBox, kvh, t0, b, bar);
      tma_load_4d(to + Sh::kStage / 2 + x * (16 * Sh::kBox), &v_map, x * Sh::kBox, kvh, t0, b, bar);
    }
  };
  const int count = first < s1 ? (s1 - first + kRowsWarps - 1) / kRowsWarps : 0;
  if (lane == 0)
    for (int i = 0; i < min(count, kStages); ++i) fetch(i);
  __syncwarp();

  // the exponents of the lane's tokens, token_at(g) and that + 8
  const int own = token_at<DP>(g);
  const size_t ex0 = (size_t)b * a.max_seq * a.kv_heads + kvh;
  auto load_exps = [&](int step, uint32_t(&x)[4]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int t = step * 16 + own + 8 * h;
      const size_t at = ex0 + (size_t)t * a.kv_heads;
      x[h] = t < total ? a.k_exp[at] : 127;
      x[2 + h] = t < total ? a.v_exp[at] : 127;
    }
  };
  uint32_t xr[4] = {127, 127, 127, 127};
  if (count > 0) load_exps(first, xr);

  // queries: a warp takes rows w, w + 4, ...; eight columns a lane, all rows' asked for at once
  constexpr int kMine = NR / kRowsWarps;
  float x[kMine][8];
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    const int row = w + i * kRowsWarps, n = row / a.group, col = lane * 8;
#pragma unroll
    for (int k = 0; k < 8; ++k) x[i][k] = 0.0f;
    if (row < rows && col < D)
      load_q8(a, ((size_t)b * a.nodes + n) * a.q_pitch + (size_t)(kvh * a.group + row - n * a.group) * a.q_head + col, x[i]);
  }
  if (w == 0) {
    const Sight s = sight_of(a, b, lane < rows ? lane / a.group : a.nodes, pos);
    if (lane < NR) sight_s[lane] = s;
  }
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    const int r = w + i * kRowsWarps;
    float amax = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k) amax = fmaxf(amax, fabsf(x[i][k]));
    const int e = q_exponent(warp_max(amax));
    const float f = pow2i(-e);
    if (lane * 8 < DP)
      *reinterpret_cast<uint4 *>(qs + r * Sh::kQPitch + lane * 8) =
          make_uint4(pack_f16x2(x[i][0] * f, x[i][1] * f), pack_f16x2(x[i][2] * f, x[i][3] * f),
                     pack_f16x2(x[i][4] * f, x[i][5] * f), pack_f16x2(x[i][6] * f, x[i][7] * f));
    if (lane == 0) fac_s[r] = pow2i(e) * a.scale_log2;
  }
  __syncthreads();
  // the lane's rows: 2 c, 2 c + 1 and, with 16 rows, those + 8
  float fac[kNT][2];
#pragma unroll
  for (int i = 0; i < kNT; ++i)
#pragma unroll
    for (int e = 0; e < 2; ++e) fac[i][e] = fac_s[8 * i + 2 * c + e];
  // Q operands of piece p: row g (+ 8 i)'s dimensions 64 p + 16 c + [0, 16)
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

  float acc[kMT][kNT][4];
#pragma unroll
  for (int i = 0; i < kMT; ++i)
#pragma unroll
    for (int j = 0; j < kNT; ++j)
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[i][j][k] = 0.0f;
  float m[kNT][2], l[kNT][2];
#pragma unroll
  for (int i = 0; i < kNT; ++i)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      m[i][e] = -INFINITY;
      l[i][e] = 0.0f;
    }
  bool ok = true, nan = false;  // nan: a NaN among the lane's values of open steps
  for (int at_step = 0; at_step < count; ++at_step) {
    const int step = first + at_step * kRowsWarps;
    const uint8_t *kst = mine_ring + (at_step % kStages) * Sh::kStage, *vst = kst + Sh::kStage / 2;
    if (ok) ok = mbar_wait(&full[w][at_step % kStages], (at_step / kStages) & 1, &abort_s);
    if (!ok && a.error) {  // (a wait that ran out: the results are void, but the loop ends)
      *(volatile int *)&abort_s = 1;
      atomicCAS(a.error, 0, kErrRowsWait);
    }
    __syncwarp();
    // scores of 16 tokens: s[i][.][2 h + e] token token_at(g) + 8 h, row 2 c + e + 8 i,
    // with eight rows in two sums that do not wait for one another
    constexpr int kChains = NR == 8 ? 2 : 1;
    float s[kNT][kChains][4];
#pragma unroll
    for (int i = 0; i < kNT; ++i)
#pragma unroll
      for (int u = 0; u < kChains; ++u)
#pragma unroll
        for (int k = 0; k < 4; ++k) s[i][u][k] = 0.0f;
#pragma unroll
    for (int p = 0; p < kPieces; ++p) {
      uint32_t kw[2][4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int at = DP == 64 ? (8 * h + own) * 64 + ((c ^ ((own >> 1) & 3)) * 16)
                                : (p >> 1) * 2048 + (8 * h + own) * 128 + (((4 * (p & 1) + c) ^ own) * 16);
        const uint4 kv = *reinterpret_cast<const uint4 *>(kst + at);
        kw[h][0] = kv.x; kw[h][1] = kv.y; kw[h][2] = kv.z; kw[h][3] = kv.w;
      }
      uint32_t q[kNT][8];
#pragma unroll
      for (int i = 0; i < kNT; ++i) {
        if constexpr (Sh::kQShared) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint4 v = *reinterpret_cast<const uint4 *>(qs + (g + 8 * i) * Sh::kQPitch + 64 * p + 16 * c + 8 * j);
            q[i][4 * j] = v.x; q[i][4 * j + 1] = v.y; q[i][4 * j + 2] = v.z; q[i][4 * j + 3] = v.w;
          }
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) q[i][j] = qr[(p * kNT + i) * 8 + j];
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t a0 = e4m3x2_to_f16x2((uint16_t)kw[0][j]), a1 = e4m3x2_to_f16x2((uint16_t)kw[1][j]),
                       a2 = e4m3x2_to_f16x2((uint16_t)(kw[0][j] >> 16)), a3 = e4m3x2_to_f16x2((uint16_t)(kw[1][j] >> 16));
#pragma unroll
        for (int i = 0; i < kNT; ++i) mma_f16(s[i][j % kChains], a0, a1, a2, a3, q[i][2 * j], q[i][2 * j + 1]);
      }
    }
    if constexpr (kChains == 2) {
#pragma unroll
      for (int i = 0; i < kNT; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) s[i][0][k] += s[i][1][k];
    }
    const int t0 = step * 16;
    const bool open = t0 + 16 > pos;  // warp-uniform: the tree's rows, or the end
    float kf[2], ve[2], vf[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      kf[h] = kv8_factor(xr[h]);
      ve[h] = kv8_value_exponent(xr[2 + h]);
      vf[h] = pow2i((int)ve[h] - kSpread);
    }
    if (at_step + 1 < count) load_exps(step + kRowsWarps, xr);
    uint32_t vr[4][kVPieces][kVBytes / 4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int row = token_at<DP>(2 * c + (t & 1)) + 8 * (t >> 1), at = piece_at<DP>(g);
#pragma unroll
      for (int p = 0; p < kVPieces; ++p) {
        if constexpr (kVBytes == 16) {
          const uint4 v = *reinterpret_cast<const uint4 *>(vst + p * 2048 + row * 128 + ((at ^ (row & 7)) * 16));
          vr[t][p][0] = v.x; vr[t][p][1] = v.y; vr[t][p][2] = v.z; vr[t][p][3] = v.w;
        } else {
          const uint2 v = *reinterpret_cast<const uint2 *>(vst + row * 64 + (((at >> 1) ^ ((row >> 1) & 3)) * 16) + (at & 1) * 8);
          vr[t][p][0] = v.x; vr[t][p][1] = v.y;
        }
      }
    }
    if (open) {  // a value vector that some row does not see must not reach it through 0 * NaN
      uint32_t any = 0;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int p = 0; p < kVPieces; ++p)
#pragma unroll
          for (int j = 0; j < kVBytes / 4; ++j) {
            const uint32_t bad = __vcmpeq4(vr[t][p][j] & 0x7f7f7f7fu, 0x7f7f7f7fu);
            vr[t][p][j] &= ~bad;
            any |= bad;
          }
      nan |= any != 0;
    }
    float y[kNT][2][2];  // scores: row, token
    bool grow = false;
#pragma unroll
    for (int i = 0; i < kNT; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float v = s[i][0][2 * h + e] * (kf[h] * fac[i][e]);
          if (open) {
            const int t = t0 + own + 8 * h;
            if (t >= total || !sight_s[8 * i + 2 * c + e].sees(t, pos, tree)) v = -INFINITY;
          }
          y[i][e][h] = v;
        }
        grow |= fmaxf(y[i][e][0] + ve[0], y[i][e][1] + ve[1]) > m[i][e] + kLag;
      }
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        uint32_t any = 0;
#pragma unroll
        for (int p = 0; p < kVPieces; ++p)
#pragma unroll
          for (int j = 0; j < kVBytes / 4; ++j) any |= vr[t][p][j];
        // operand row 2 c + t % 2 (+ 8) lies over the lanes of this c
        const uint32_t lanes = __ballot_sync(0xffffffffu, (any & 0x7f7f7f7fu) != 0) & (0x11111111u << (g >> 1));
        if ((g & 1) == (t & 1) && !lanes) {
          ve[t >> 1] = kZeroExp;
          vf[t >> 1] = 0.0f;
        }
      }
#pragma unroll
      for (int i = 0; i < kNT; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float mn = fmaxf(m[i][e], fmaxf(y[i][e][0] + ve[0], y[i][e][1] + ve[1]));
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
          const float by = m[i][e] == -INFINITY ? -INFINITY : m[i][e] - mn, old = exp2_approx(by);
          l[i][e] = sum_to(l[i][e], by);
          m[i][e] = mn;
#pragma unroll
          for (int k = 0; k < kMT; ++k) {
            acc[k][i][e] *= old;
            acc[k][i][2 + e] *= old;
          }
        }
    }
    uint32_t pb[kNT][2];
#pragma unroll
    for (int i = 0; i < kNT; ++i) {
      float p[2][2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float base = m[i][e] == -INFINITY ? 0.0f : kHead + kSpread - m[i][e];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float x = exp2_approx(y[i][e][h] + base);
          l[i][e] = fmaf(x, kSumScale, l[i][e]);
          p[e][h] = x * vf[h];
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) pb[i][h] = transposed(pack_f16x2(p[0][h], p[1][h]));
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
    if (lane == 0 && at_step + kStages < count) fetch(at_step + kStages);
    __syncwarp();
  }
  if (!ok)  // copies still in flight land before the block ends
    for (int i = 0; i < kStages; ++i) {
      int never = 0;
      for (uint32_t k = 0; k < 2; ++k) mbar_wait(&full[w][i], k, &never);
    }

  // Those who see a value with NaN codes have NaN in its columns (the lane's:
  // whichever lane has met one, all look).
  if (__any_sync(0xffffffffu, nan))
    for (int t = max(s0 * 16, pos / 16 * 16); t < min(s1 * 16, total); ++t) {
      if ((t / 16 - first) % kRowsWarps) continue;  // another warp's step
      const uint8_t *v = a.v_codes + (((size_t)b * a.max_seq + t) * a.kv_heads + kvh) * D;
#pragma unroll
      for (int p = 0; p < kVPieces; ++p)
#pragma unroll
        for (int j = 0; j < kVBytes / 4; ++j) {
          const int d = 128 * p + kVBytes * piece_at<DP>(g) + 4 * j, mt = (p * kVBytes / 4 + j) * 2;
          const uint32_t w = d < D ? __ldg(reinterpret_cast<const uint32_t *>(v + d)) : 0;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if ((w >> (8 * k) & 0x7f) == 0x7f) {
#pragma unroll
              for (int i = 0; i < kNT; ++i)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                  if (sight_s[8 * i + 2 * c + e].sees(t, pos, tree))
                    acc[mt + (k >> 1)][i][2 * (k & 1) + e] = __int_as_float(0x7fc00000);
            }
        }
    }

  // the warps' results meet: maxima, then sums over one maximum in warp order
#pragma unroll
  for (int i = 0; i < kNT; ++i)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) l[i][e] += __shfl_xor_sync(0xffffffffu, l[i][e], o);
      if (g == 0) {
        m_s[w][8 * i + 2 * c + e] = m[i][e];
        l_s[w][8 * i + 2 * c + e] = l[i][e];
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
          const int mt = (p * kVBytes / 4 + j) * 2, d = 128 * p + kVBytes * piece_at<DP>(g) + 4 * j;
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
      const float by = m_s[x][r] == -INFINITY ? -INFINITY : m_s[x][r] - mt;
      f[x] = exp2_approx(by);
      lt += sum_to(l_s[x][r], by);
    }
    const int n = row / a.group, h = kvh * a.group + row % a.group;
    const bool there = sight_s[r].upto >= 0;
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
        const float inv = there ? kSumBack / lt : 0.0f;
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

// The splits of a row (session, node, query head) meet, in order: blockDim.y
// warps a row and 128 columns share them, four columns a lane.  What the rows
// kernel does not write is read before it is waited for.  Bound by the latency
// of two reads in a row (maxima, then values, in L2).
constexpr int kMergeWarps = 16;
__global__ void __launch_bounds__(kMergeWarps * 32, 2) tree_attn_merge_kernel(const __grid_constant__ TreeArgs a, int NR,
                                                                            int count) {
  __shared__ float4 acc_s[kMergeWarps][32];
  __shared__ float l_s[kMergeWarps];
  const int lane = threadIdx.x, share = threadIdx.y, shares = blockDim.y, w = threadIdx.z * shares + share;
  const int i = blockIdx.x * blockDim.z + threadIdx.z, d = blockIdx.y * 128 + lane * 4, D = a.head_dim;
  const bool in = i < count;
  const int h = i % a.q_heads, node = in ? i / a.q_heads : 0, b = node / a.nodes, n = node % a.nodes;
  const int kvh = h / a.group, r = n * a.group + h % a.group, pos = a.positions[b];
  const size_t slot0 = ((size_t)b * a.kv_heads + kvh) * a.splits * NR + r;
  asm volatile("griddepcontrol.launch_dependents;");
  const int steps = (seen_rows(a, pos, a.nodes - 1) + 15) / 16, per = max(1, steps_a_split(steps, a.splits));
  const int splits = max(1, (steps + per - 1) / per);
  const bool there = sight_of(a, b, n, pos).upto >= 0;
  float gate[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (there && a.gate && d < D && share == 0) {
    const float *g = a.gate + (size_t)node * a.gate_pitch + (size_t)h * a.gate_head + d;
#pragma unroll
    for (int k = 0; k < 4; ++k) gate[k] = expf(-g[k]);
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const float2 *ml = a.part_ml + slot0;
  float m = -INFINITY, l = 0.0f;
  for (int s = lane; s < splits; s += 32) m = fmaxf(m, ml[(size_t)s * NR].x);
  m = warp_max(m);
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  auto add = [&](float4 x, float f) {
    acc.x = fmaf(x.x, f, acc.x);
    acc.y = fmaf(x.y, f, acc.y);
    acc.z = fmaf(x.z, f, acc.z);
    acc.w = fmaf(x.w, f, acc.w);
  };
  const float *part = a.part + slot0 * D + (d < D ? d : 0);
#pragma unroll 4
  for (int s = share; s < splits; s += shares) {
    const float2 v = ml[(size_t)s * NR];
    const float4 x = *reinterpret_cast<const float4 *>(part + (size_t)s * NR * D);
    const float by = v.x == -INFINITY ? -INFINITY : v.x - m;
    l += sum_to(v.y, by);
    add(x, exp2_approx(by));
  }
  if (shares > 1) {
    if (share > 0) {
      acc_s[w][lane] = acc;
      if (lane == 0) l_s[w] = l;
    }
    __syncthreads();
    if (share > 0) return;
    for (int k = w + 1; k < w + shares; ++k) {
      add(acc_s[k][lane], 1.0f);
      l += l_s[k];
    }
  }
  if (!in || d >= D) return;
  const float inv = there ? kSumBack / l : 0.0f;
  const float x[4] = {acc.x, acc.y, acc.z, acc.w};
  float o[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) o[k] = there ? x[k] * inv / (1.0f + gate[k]) : 0.0f;
  *reinterpret_cast<uint2 *>(a.out + ((size_t)node * a.q_heads + h) * D + d) =
      make_uint2(pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3]));
}

// How a call of few rows is cut: rows a tile, tiles, splits of the tokens.
struct Plan {
  int rows_tile, splits;
  size_t items;
};

// Past 16 rows a key/value head the tcgen05 kernel takes over, which takes 128 of
// them in the time of 17.  Up to 16 it is the slower one: 16 rows x 256 columns,
// 8 x 8192 tokens 47 us, here 24.5, 1 x 30000 36 and 22, 64 x 1000 51 and 28.
bool wants_tiles(size_t nodes, size_t q_heads, size_t kv_heads) { return nodes * (q_heads / kv_heads) > 16; }

Plan plan_for(size_t batch, size_t nodes, size_t q_heads, size_t kv_heads, size_t head_dim, size_t max_seq) {
  Plan p{};
  const size_t rows = nodes * (q_heads / kv_heads);
  // (eight rows as 16: 25.9 us instead of 21.5 at 8 x 8192 x 256, 9.0 instead of 7.7 at 1 x 1000)
  p.rows_tile = rows <= 8 ? 8 : 16;
  p.items = batch * kv_heads;
  // One wave of blocks; at least 64 tokens a split, a step for each warp (1 x 1000
  // tokens: 7.8 us, with 128 tokens 8.7, with 256 11.1).
  const size_t resident = (size_t)sm_count() * rows_blocks(head_dim <= 128 ? 128 : 256);
  const size_t want = std::max<size_t>(1, resident / p.items);
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
  const Plan p = plan_for(batch, nodes, q_heads, kv_heads, head_dim, max_seq);
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
  const Plan p = plan_for(batch, nodes, q_heads, kv_heads, head_dim, max_seq);
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
  // As many warps a row as it has splits, while all of them run at once (whole
  // calls, one warp a row and shared: 1 x 30000 28.5 and 16.9 us, 8 x 8192 with 16
  // rows 29.3 and 27.5; shared past what runs at once: 31).
  const unsigned halves = head_dim > 128 ? 2 : 1;
  unsigned shares = 1;
  while (shares < (unsigned)kMergeWarps && 2 * shares <= (unsigned)p.splits &&
         2 * shares * halves * (size_t)count <= (size_t)sm_count() * 16)
    shares *= 2;
  const unsigned per = std::max(1u, 8 / shares);
  cudaError_t e = launch_pdl(tree_attn_merge_kernel, dim3((unsigned)((count + per - 1) / per), halves),
                             dim3(32, shares, per), 0, s, a, p.rows_tile, count);
  if (e != cudaSuccess) return cuda_fail(e, "tree_attn_merge_kernel");
  FPB_LAUNCH_CHECK("tree_attn_merge_kernel");
  return FPB_OK;
}
