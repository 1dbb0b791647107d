// Tree attention for many rows a key/value head: 128-row tiles on tcgen05.
//
// A block takes a share of the call's (session, kv head, row tile, token tile)
// units, in that order, so that sessions of any lengths load the SMs evenly.
// Token tiles of one row tile that fall to several blocks meet in the merge.
//   warps 0-15   softmax: thread (part, r) owns a quarter of row r's tokens
//                (TMEM lane r); the four warps of a 32-row quad keep step
//   warp 16      issues the MMAs
//   warp 17      brings the codes to shared memory by TMA, two tiles ahead
//   warps 18-25  convert them to f16 tiles
// S = Q K^T and O += P V, with Q and P as the A operand in TMEM: shared memory
// carries only what K and V need.  A tile is 64 tokens at head_dim 256, else
// 128; TMEM then holds O [DP], two S [BT] (P overwrites its S) and Q [DP / 2
// columns].
//   K tile: tokens as rows of 128-byte swizzled lines, 64 dimensions a chunk
//           (K-major).
//   V tile: the same bytes read as the transposed operand (N-major).
// The tokens' factors stay out of the tiles: the key's multiplies the score,
// the value's the weight, both in f32 (see kHead).
// Neither the cache's bytes nor the tensor cores bound it.  A unit of 128 tokens
// and 128 columns takes 2600 cycles, of which the two products need 1280, the
// softmax's and the converters' instructions 1350 issue cycles a scheduler, and
// shared memory about 1800 (copies in, converters' reads and writes, operands,
// factors).  Issue slots 54% busy, tensor cores 33%.
//   8 sessions x 16 nodes x 16 heads (2 kv) x 256, 16384 tokens: 61 us with its
//     two helpers; 2.05 TB/s of the cache, 443 TFLOP/s
//   4 x 61 x 32 (4) x 128, 30011 tokens: 183 us, 525 TFLOP/s
//   a prompt's chunk of 2048 rows x 16 heads (2 kv) x 256: 163 us from position 0
//     (211 TFLOP/s: a row tile's share counts its session's tiles, of which it
//     sees half), 436 us from 8192 (710 TFLOP/s)
// Before the first products the block spends 8 us (start, shares, queries), at
// its end 4 us on the 64 to 128 KB of its partial result.
#include <algorithm>
#include <cfloat>
#include <mutex>
#include <vector>

#include "sm100.cuh"
#include "tma_host.cuh"
#include "tree_attn.cuh"

namespace fpb {
namespace {

using namespace sm100;

constexpr int kParts = 4, kSoftWarps = 4 * kParts, kSoftThreads = kSoftWarps * 32, kConvWarps = 8, kTileRows = 128;
constexpr int kMmaWarp = kSoftWarps, kLoadWarp = kMmaWarp + 1, kConvWarp = kLoadWarp + 1;
constexpr int kTileThreads = (kConvWarp + kConvWarps) * 32;
constexpr int kErrTileWait = 503;
// A score is (s * kf) * f: f16 products s of up to 2^26, the key's factor of up
// to 2^120, the query's.  kKeyShift of kf is in f, so that s * kf is an f32
// whatever the key's size; s * (kf * f) would do without, and takes the tiles 3 %
// longer (4 x 61 at 30011 184 us, 178 to 181 so).
constexpr float kKeyShift = 0x1p-24f;

template <int DP>
struct TileShape {
  static constexpr int BT = DP == 256 ? 64 : 128;
  static constexpr int ST = 2, RAW = 2, META = 4;  // f16 stages, stages of codes, of factors (at least ST + 2)
  static constexpr uint32_t kBytes = BT * DP * 2, kRawBytes = BT * DP;
  static constexpr uint32_t kTmemO = 0, kTmemS = DP, kTmemQ = DP + 2 * BT;
  static constexpr int kPieces = BT * DP / 16 / (kConvWarps * 32);  // 16-byte pieces of codes a thread and tile
  static constexpr int kBox = DP == 64 ? 64 : 128;
};

struct Segment {
  int b, kvh, rt, item, j0, j1, pos, total;
  bool starts, ends;
};

// A block's units, one segment (token tiles [j0, j1) of one row tile) at a time.
// A row tile counts for kTakeUp / BT units more than it has token tiles, what a
// block spends on taking up another one (its end's and the next one's queries,
// first scores: 7 us, five tiles of 64 tokens at 256 columns).  8 x 16 nodes at
// 16384: 64.8 us, 68.5 without.
constexpr int kTakeUp = 320;  // tokens
struct Walk {
  int b, units, row_tiles, rem, left;
  __device__ __forceinline__ bool next(const TreeArgs &a, int BT, Segment &s);
};

// Fixed part of the block's shared memory; the stages follow, 1024-byte aligned.
struct TileShared {
  uint64_t kfull[2], kempty[2], vfull[2], vempty[2], rkfull[2], rvfull[2], rkempty[2], rvempty[2], sfull[2], pready[2],
      metafull[4], qready, drain;
  Walk walk, soft_walk;
  Segment seg;
  uint32_t tmem;
  int abort, never, more, nan;  // nan: there has been a NaN among the values of an open tile
  float red[kParts][kTileRows];  // maxima, then sums, of the rows' parts
  uint64_t sight[kTileRows];     // a tree: the bits; a chain: the limit
  float4 fac[4][64];             // [META][pair of tokens]: two keys' factors, two values'
};

// Token tiles of session b (0: none of its nodes is there).
__device__ __forceinline__ int session_tiles(const TreeArgs &a, int b, int BT) {
  const int root = a.parents ? a.parents[(size_t)b * a.nodes] : -1, pos = a.positions[b];  // (both asked for at once)
  return root == -1 ? (seen_rows(a, pos, a.nodes - 1) + BT - 1) / BT : 0;
}

__device__ __forceinline__ int session_units(const TreeArgs &a, int b, int BT) {
  const int tiles = session_tiles(a, b, BT);
  return tiles ? tiles + kTakeUp / BT : 0;
}

__device__ __forceinline__ bool Walk::next(const TreeArgs &a, int BT, Segment &s) {
  if (left <= 0) return false;
  const int items = a.kv_heads * row_tiles, skip = kTakeUp / BT;
  while (rem >= items * units) {
    rem -= items * units;
    units = session_units(a, ++b, BT);
  }
  const int item = rem / units, u0 = rem % units, n = min(left, units - u0);
  s.starts = u0 == 0;
  s.ends = u0 + n == units;
  s.j0 = max(0, u0 - skip);
  left -= n;
  rem += n;
  s.b = b;
  s.item = b * items + item;
  s.kvh = item / row_tiles;
  s.rt = item % row_tiles;
  s.pos = a.positions[b];
  // a chain's row tile ends at its last node's own row
  s.total = seen_rows(a, s.pos, min(a.nodes - 1, (s.rt * kTileRows + kTileRows - 1) / a.group));
  s.j1 = min(u0 + n - skip, (s.total + BT - 1) / BT);
  return true;
}

__device__ __forceinline__ void give_up(int *error, volatile int *abort) {
  *abort = 1;
  if (error) atomicCAS(error, 0, kErrTileWait);
}

// Packed pairs of f32.
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

// Barriers of the roles: a quad's softmax warps (ids 1-4), the converting
// warps (5), all of the softmax (6).  TMEM accesses are ordered across them.
__device__ __forceinline__ void quad_sync(int quad) {
  tc_fence_before();
  asm volatile("bar.sync %0, %1;" ::"r"(1 + quad), "n"(kParts * 32) : "memory");
  tc_fence_after();
}
__device__ __forceinline__ bool quad_any(int quad, bool v) {
  int r;
  tc_fence_before();
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\tbar.red.or.pred q, %2, %3, p;\n\tselp.b32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"((int)v), "r"(1 + quad), "n"(kParts * 32)
      : "memory");
  tc_fence_after();
  return r != 0;
}
__device__ __forceinline__ void conv_sync() { asm volatile("bar.sync 5, %0;" ::"n"(kConvWarps * 32) : "memory"); }
__device__ __forceinline__ void soft_sync() {
  tc_fence_before();
  asm volatile("bar.sync 6, %0;" ::"n"(kSoftThreads) : "memory");
  tc_fence_after();
}

// A part of a row of S (NT tokens from TMEM column s_tmem, factors fac: two
// keys', two values' of each pair): weights e = 2^(s * kf * f + base), kSumScale
// of their sums in l, e * vf as f16 pairs in p; returns the largest e * vf.  OPEN: a
// tile that not every row sees whole, only its tokens `seen`.
template <int NT, bool OPEN>
__device__ __forceinline__ float weigh_pass(uint32_t s_tmem, const float4 *fac, float f, float base, uint64_t seen,
                                            uint32_t (&p)[NT / 2], uint64_t &l) {
  const uint64_t f2 = pack2(f, f), b2 = pack2(base, base), k2 = pack2(kSumScale, kSumScale);
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
      l = fma2(e2, k2, l);
      unpack2(mul2(e2, pack2(ft.z, ft.w)), w0, w1);
      mx[(e >> 1) & 1] = fmaxf(mx[(e >> 1) & 1], fmaxf(w0, w1));
      p[(c * 16 + e) / 2] = pack_f16x2(w0, w1);
    }
  }
  return fmaxf(mx[0], mx[1]);
}

// Bytes of four codes that are not a number.
__device__ __forceinline__ uint32_t not_numbers(uint32_t w) { return __vcmpeq4(w & 0x7f7f7f7fu, 0x7f7f7f7fu); }

// What happens seldom stays out of line, so that the loop over tiles keeps its
// registers.
template <int NT>
__device__ __noinline__ float weigh_open(uint32_t s_tmem, const float4 *fac, float f, float base, uint64_t seen,
                                         uint32_t *p, uint64_t *l) {
  uint32_t q[NT / 2];
  uint64_t sum = *l;
  const float mx = weigh_pass<NT, true>(s_tmem, fac, f, base, seen, q, sum);
#pragma unroll
  for (int i = 0; i < NT / 2; ++i) p[i] = q[i];
  *l = sum;
  return mx;
}

// The row's maximum raised by the scores of this tile's NT tokens from t0 on (y
// = s * kf * f + the value's exponent) where they are above it by more than the
// lag, and O of the tiles before rescaled to it; returns the new maximum and what
// it is above the old one, negated.  Zero values' factors become those of
// kZeroExp, for every quad of rows: whether another one takes this tile's weights
// before or after that, its maximum is raised by the same values (hence by the
// lag and a half: whatever is above that has a weight above kMost).
template <int DP, int NT>
__device__ __noinline__ float2 raise_max(const TreeArgs &a, TileShared *sh, uint32_t s_tmem, uint32_t o_tmem,
                                         const float4 *fac, float f, uint64_t seen, float m, int t0, bool sums) {
  const int quad = (threadIdx.x >> 5) & 3, part = threadIdx.x >> 7, r_own = threadIdx.x & 127, lane = threadIdx.x & 31;
  const int D = a.head_dim;
  if (lane < NT && t0 + lane < sh->seg.total) {  // a lane a token, whose first codes mostly tell
    const uint4 *v = reinterpret_cast<const uint4 *>(
        a.v_codes + (((size_t)sh->seg.b * a.max_seq + t0 + lane) * a.kv_heads + sh->seg.kvh) * D);
    bool zero = true;
    for (int i = 0; zero && i < D / 16; ++i) {
      const uint4 x = __ldg(v + i);
      zero = ((x.x | x.y | x.z | x.w) & 0x7f7f7f7fu) == 0;
    }
    if (zero) const_cast<float *>(&fac[lane >> 1].z)[lane & 1] = pow2i((int)kZeroExp - kSpread);
  }
  __syncwarp();
  float mx = -INFINITY;
#pragma unroll 1
  for (int c = 0; c < NT / 16; ++c) {
    uint32_t r[16];
    tmem_ld16(s_tmem + c * 16, r);
    tmem_ld_wait(r);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float4 ft = fac[(c * 16 + e) / 2];
      const float v = (float)((int)(__float_as_uint(e & 1 ? ft.w : ft.z) >> 23) - 127 + kSpread);
      const float y = fmaf(__uint_as_float(r[e]) * (e & 1 ? ft.y : ft.x), f, v);
      if (seen >> (c * 16 + e) & 1) mx = fmaxf(mx, y);
    }
  }
  sh->red[part][r_own] = mx;
  quad_sync(quad);
  float mn = m;  // (a row that has seen nothing yet keeps its floor)
#pragma unroll
  for (int i = 0; i < kParts; ++i) mn = fmaxf(mn, sh->red[i][r_own]);
  if (mn <= m + (kLag + 0.5f)) mn = m;
  const float old = exp2_approx(m - mn);
  if (sums) {
#pragma unroll 1
    for (int d = 16 * part; d < D; d += 16 * kParts) {
      uint32_t r[16];
      tmem_ld16(o_tmem + d, r);
      tmem_ld_wait(r);
#pragma unroll
      for (int i = 0; i < 16; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * old);
      tmem_st16(o_tmem + d, r);
    }
    tmem_st_wait();
  }
  quad_sync(quad);  // red is read
  return make_float2(mn, m - mn);
}

// Columns [d, d + 16) of the row r_own's result: NaN where a value that it sees
// in the segment's open tiles holds one.  (Past a NaN the block does this for each
// of its segments.)
__device__ __noinline__ void put_nan(const TreeArgs &a, const TileShared *sh, int BT, int r_own, int d, uint32_t *r) {
  const Segment &s = sh->seg;
  const uint64_t sight = sh->sight[r_own];
  for (int t = max(s.j0, s.pos / BT) * BT; t < min(s.j1 * BT, s.total); ++t) {
    if (!Sight{(int)sight, sight}.sees(t, s.pos, a.parents != nullptr)) continue;
    const uint4 v = __ldg(reinterpret_cast<const uint4 *>(
        a.v_codes + (((size_t)s.b * a.max_seq + t) * a.kv_heads + s.kvh) * a.head_dim + d));
    const uint32_t w[4] = {not_numbers(v.x), not_numbers(v.y), not_numbers(v.z), not_numbers(v.w)};
    for (int i = 0; i < 16; ++i)
      if (w[i >> 2] >> (8 * (i & 3)) & 1) r[i] = 0x7fc00000u;
  }
}

// O of a row tile's share to its slot: four columns of 128 rows lie together, so
// that a warp stores 512 bytes.
__device__ __noinline__ void write_part(const TreeArgs &a, const TileShared *sh, int BT, size_t slot, uint32_t o_tmem) {
  const int part = threadIdx.x >> 7, r_own = threadIdx.x & 127, D = a.head_dim;
  float4 *o = reinterpret_cast<float4 *>(a.part) + slot * (kTileRows * (size_t)D / 4) + r_own;
  for (int d = 16 * part; d < D; d += 16 * kParts) {
    uint32_t r[16];
    tmem_ld16(o_tmem + d, r);
    tmem_ld_wait(r);
    if (sh->nan) {
      uint32_t x[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = r[i];
      put_nan(a, sh, BT, r_own, d, x);
#pragma unroll
      for (int i = 0; i < 16; ++i) r[i] = x[i];
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; ++i)
      o[(size_t)(d / 4 + i) * kTileRows] = make_float4(__uint_as_float(r[4 * i]), __uint_as_float(r[4 * i + 1]),
                                                       __uint_as_float(r[4 * i + 2]), __uint_as_float(r[4 * i + 3]));
  }
}

// The same to `out`, divided by the row's sum, with the gate.
__device__ __noinline__ void write_rows(const TreeArgs &a, const TileShared *sh, int BT, uint32_t o_tmem) {
  const int part = threadIdx.x >> 7, r_own = threadIdx.x & 127, D = a.head_dim;
  const int row = sh->seg.rt * kTileRows + r_own, n = row / a.group, h = sh->seg.kvh * a.group + row % a.group;
  const size_t node = (size_t)sh->seg.b * a.nodes + n;
  const bool live = n < a.nodes, there = sh->sight[r_own] != 0;
  float l = 0.0f;
#pragma unroll
  for (int i = 0; i < kParts; ++i) l += sh->red[i][r_own];
  const float inv = kSumBack / l;
  __nv_bfloat16 *o = a.out + (node * a.q_heads + h) * D;
  const float *gate = a.gate ? a.gate + node * a.gate_pitch + (size_t)h * a.gate_head : nullptr;
#pragma unroll 1
  for (int d = 16 * part; d < D; d += 16 * kParts) {
    uint32_t r[16];
    tmem_ld16(o_tmem + d, r);
    tmem_ld_wait(r);
    if (sh->nan) {
      uint32_t y[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) y[i] = r[i];
      put_nan(a, sh, BT, r_own, d, y);
#pragma unroll
      for (int i = 0; i < 16; ++i) r[i] = y[i];
    }
    __syncwarp();
    if (live) {
      float x[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        x[i] = there ? __uint_as_float(r[i]) * inv : 0.0f;
        if (there && gate) x[i] /= 1.0f + expf(-gate[d + i]);
      }
      uint4 *to = reinterpret_cast<uint4 *>(o + d);
      to[0] = make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
      to[1] = make_uint4(pack_bf16x2(x[8], x[9]), pack_bf16x2(x[10], x[11]), pack_bf16x2(x[12], x[13]),
                         pack_bf16x2(x[14], x[15]));
    }
    __syncwarp();
  }
}

// What the tile kernel reads at its start, made by blocks of 32 rows of a row
// tile (eight warps): the queries as f16 in the order of its TMEM stores
// [item][eight columns][128 rows], each row scaled by a power of two into f16's
// range, with the factor of its scores; what each node sees (a block a session).
// A kernel of its own since several blocks read a row's queries (here once, 128
// KB a row tile), and a row's factor needs all of its columns: 2 us, most of it
// hidden behind the tile kernel's own start.
constexpr int kPrepRows = 32;
__global__ void __launch_bounds__(256) tree_attn_prep_kernel(const __grid_constant__ TreeArgs a) {
  pdl_enter();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, D = a.head_dim;
  const int rows = a.nodes * a.group, row_tiles = (rows + kTileRows - 1) / kTileRows, items = a.kv_heads * row_tiles;
  if ((int)blockIdx.x >= a.batch * items * (kTileRows / kPrepRows)) {  // the blocks past the rows': a session's sights
    if (warp >= kTreeMaxNodes / 32) return;
    const int b = blockIdx.x - a.batch * items * (kTileRows / kPrepRows), n = warp * 32 + lane, pos = a.positions[b];
    if (a.parents) {
      const Sight s = sight_of(a, b, n, pos);
      if (n < a.nodes) a.sights[(size_t)b * kTreeMaxNodes + n] = s.bits;
    } else if (n == 0 && (pos < 0 || pos > a.max_seq - a.nodes) && a.error) {
      atomicCAS(a.error, 0, kErrPosition);
    }
    return;
  }
  const int item = blockIdx.x / (kTileRows / kPrepRows), r0 = blockIdx.x % (kTileRows / kPrepRows) * kPrepRows + warp * 4;
  const int b = item / items, kvh = item % items / row_tiles, row0 = item % row_tiles * kTileRows + r0;
  const int col = lane * 8;
  float x[4][8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = row0 + i, n = row / a.group;
#pragma unroll
    for (int k = 0; k < 8; ++k) x[i][k] = 0.0f;
    if (row >= rows || col >= D) continue;
    load_q8(a, ((size_t)b * a.nodes + n) * a.q_pitch + (size_t)(kvh * a.group + row - n * a.group) * a.q_head + col, x[i]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float amax = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k) amax = fmaxf(amax, fabsf(x[i][k]));
    const int e = q_exponent(warp_max(amax));
    const float f = pow2i(-e);
    if (col < D)
      a.q16[((size_t)item * (D / 8) + lane) * kTileRows + r0 + i] =
          make_uint4(pack_f16x2(x[i][0] * f, x[i][1] * f), pack_f16x2(x[i][2] * f, x[i][3] * f),
                     pack_f16x2(x[i][4] * f, x[i][5] * f), pack_f16x2(x[i][6] * f, x[i][7] * f));
    if (lane == 0)  // (queries past 2^114 end at the largest f32: their scores are apart by far more than the weights' range)
      a.q_fac[(size_t)item * kTileRows + r0 + i] = fminf(fmaxf(pow2i(e) * (a.scale_log2 / kKeyShift), -FLT_MAX), FLT_MAX);
  }
}

// This block's share of the units, one warp.
__device__ __noinline__ void share_out(const TreeArgs &a, TileShared *sh, int BT) {
  const int lane = threadIdx.x & 31, row_tiles = (a.nodes * a.group + kTileRows - 1) / kTileRows;
  const int items = a.kv_heads * row_tiles;
  int all = 0;
  for (int i = lane; i < a.batch; i += 32) all += session_units(a, i, BT);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
  const int units = all * items, blocks = min((int)gridDim.x, units);
  int u0 = 0, u1 = 0;
  if ((int)blockIdx.x < blocks) {
    u0 = (int)((long long)units * blockIdx.x / blocks);
    u1 = (int)((long long)units * (blockIdx.x + 1) / blocks);
  }
  int s = 0, before = 0;  // the session that holds unit u0, and the units before it
  if (u1 > u0)
    for (int i0 = 0; i0 < a.batch; i0 += 32) {
      const int n = i0 + lane < a.batch ? session_units(a, i0 + lane, BT) * items : 0;
      int sum = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += v;
      }
      const unsigned past = __ballot_sync(0xffffffffu, before + sum > u0);
      const int k = past ? __ffs(past) - 1 : 31;
      before += __shfl_sync(0xffffffffu, past ? sum - n : sum, k);
      if (past) {
        s = i0 + k;
        break;
      }
    }
  if (lane == 0)
    sh->walk = sh->soft_walk = Walk{s, u1 > u0 ? session_units(a, s, BT) : 1, row_tiles, u0 - before, u1 - u0};
}

template <int DP>
__global__ void __launch_bounds__(kTileThreads, 1)
    tree_attn_tile_kernel(const __grid_constant__ TreeArgs a, const __grid_constant__ CUtensorMap k_map,
                          const __grid_constant__ CUtensorMap v_map) {
  using Sh = TileShape<DP>;
  constexpr int BT = Sh::BT, ST = Sh::ST, RAW = Sh::RAW, META = Sh::META;
  extern __shared__ __align__(1024) uint8_t raw_sm[];
  TileShared *const sh = reinterpret_cast<TileShared *>(raw_sm);
  uint8_t *const sK = raw_sm + (sizeof(TileShared) + 1023) / 1024 * 1024, *const sV = sK + ST * Sh::kBytes;
  uint8_t *const rK = sV + ST * Sh::kBytes, *const rV = rK + RAW * Sh::kRawBytes;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const bool tree = a.parents != nullptr;
  // The tile kernel starts beside the prep kernel, which has by then waited
  // for whatever came before: only what the prep kernel itself writes is waited
  // for, by the softmax.
  asm volatile("griddepcontrol.launch_dependents;");
  if (warp == 0) {
    share_out(a, sh, BT);
  } else if (warp == kMmaWarp) {
    if (lane == 0) {
      for (int i = 0; i < 2; ++i) {
        mbar_init(&sh->kfull[i], kConvWarps);
        mbar_init(&sh->vfull[i], kConvWarps);
        mbar_init(&sh->kempty[i], 1);
        mbar_init(&sh->vempty[i], 1);
        mbar_init(&sh->rkfull[i], 1);
        mbar_init(&sh->rvfull[i], 1);
        mbar_init(&sh->rkempty[i], kConvWarps);
        mbar_init(&sh->rvempty[i], kConvWarps);
        mbar_init(&sh->sfull[i], 1);
        mbar_init(&sh->pready[i], kSoftWarps);
      }
      for (int i = 0; i < META; ++i) mbar_init(&sh->metafull[i], 1);
      mbar_init(&sh->qready, kSoftWarps);
      mbar_init(&sh->drain, 1);
      sh->abort = sh->never = sh->nan = 0;
      fence_barrier_init();
    }
    __syncwarp();
    tmem_alloc(&sh->tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  volatile int *const abort_s = &sh->abort;
  // (an allocation of all of TMEM's columns begins at 0, and this block's
  // shared memory on 1024 bytes: the addresses below are then constants)
  if (sh->tmem != 0 || (smem_u32(raw_sm) & 1023)) {
    if (tid == 0) give_up(a.error, abort_s);
    __syncthreads();
    if (warp == kMmaWarp) tmem_dealloc(sh->tmem, 512);
    return;
  }

  if (warp < kSoftWarps) {
    // ---- softmax ----
    constexpr int NT = BT / kParts;
    const int quad = warp & 3, part = warp >> 2, r_own = quad * 32 + lane;
    const uint32_t my = (uint32_t)(quad * 32) << 16;
    uint32_t g = 0;  // tiles so far
    // After a wait that ran out this role goes on to its end without waiting
    // (the results are void): its warps meet at barriers.
    bool ok = true;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    // The walk, and what a segment needs once, lie in shared memory: the loop
    // over its tiles wants the registers.
    for (int seg = 0;; ++seg) {
      if (tid == 0) {
        Walk w = sh->soft_walk;
        Segment next;
        sh->more = w.next(a, BT, next);
        sh->soft_walk = w;
        sh->seg = next;
      }
      soft_sync();
      if (!sh->more) break;
      const int j0 = sh->seg.j0, j1 = sh->seg.j1, pos = sh->seg.pos;
      // Only a segment with tiles takes up queries: what it then waits for (its
      // last product) shows that the MMA warp has seen this phase of qready, and
      // so the next may complete.  Nothing would wait in one without (what a
      // block has of a row tile may lie in its take-up or past its last row).
      const bool tiles = j1 > j0;
      const float f = tiles ? a.q_fac[(size_t)sh->seg.item * kTileRows + r_own] : 0.0f;
      uint64_t sight = 0;
      if (part == 0) {
        const int n = (sh->seg.rt * kTileRows + r_own) / a.group;
        if (tree)
          sight = n < a.nodes ? a.sights[(size_t)sh->seg.b * kTreeMaxNodes + n] : 0;
        else if (n < a.nodes && pos >= 0 && pos < a.max_seq - n)
          sight = n + 1;
      }
      if (tiles) {
        // 16 columns of the row at a time; a warp's loads are 512 bytes together
        const uint4 *q = a.q16 + (size_t)sh->seg.item * (a.head_dim / 8) * kTileRows + r_own;
        constexpr int kQ = DP / 16 / kParts;
        uint4 v[kQ][2];
#pragma unroll
        for (int i = 0; i < kQ; ++i)
#pragma unroll
          for (int k = 0; k < 2; ++k)
            v[i][k] = (i * kParts + part) * 16 < a.head_dim ? q[(size_t)((i * kParts + part) * 2 + k) * kTileRows]
                                                            : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < kQ; ++i) {
          const uint32_t w[8] = {v[i][0].x, v[i][0].y, v[i][0].z, v[i][0].w, v[i][1].x, v[i][1].y, v[i][1].z, v[i][1].w};
          tmem_st8(my + Sh::kTmemQ + (i * kParts + part) * 8, w);
        }
      }
      if (part == 0) sh->sight[r_own] = sight;
      tmem_st_wait();
      quad_sync(quad);
      if (tiles && lane == 0) mbar_arrive(&sh->qready);
      float m = kLowest;
      uint64_t l2 = 0;
      for (int j = j0; j < j1; ++j, ++g) {
        if (ok)
          ok = mbar_wait(&sh->sfull[g & 1], (g >> 1) & 1, abort_s) &&
               mbar_wait(&sh->metafull[g % META], (g / META) & 1, abort_s);
        if (!ok) give_up(a.error, abort_s);
        __syncwarp();
        tc_fence_after();
        const uint32_t s_tmem = my + Sh::kTmemS + (g & 1) * BT + part * NT;
        const float4 *fac = sh->fac[g % META] + part * NT / 2;
        const bool open = (j + 1) * BT > pos;
        uint64_t seen = ~0ull;
        if (open) {
          const uint64_t b = sh->sight[r_own];
          seen = Sight{(int)b, b}.seen64(j * BT + part * NT, pos, tree);
        }
        // With the maximum so far; where a weight has outgrown it (and for a
        // segment's first tile) the maximum is raised and the weights taken
        // again, once.
        uint32_t p[NT / 2];
        uint64_t l_new;
        for (bool raise = j == j0;;) {
          if (raise) {
            if (j > j0) {
              if (ok) ok = mbar_wait(&sh->vempty[(g - 1) % ST], ((g - 1) / ST) & 1, abort_s);
              if (!ok) give_up(a.error, abort_s);
              __syncwarp();
              tc_fence_after();
            }
            const float2 r = raise_max<DP, NT>(a, sh, s_tmem, my + Sh::kTmemO, fac, f, seen, m, j * BT + part * NT, j > j0);
            m = r.x;
            const float half = exp2_approx(0.5f * r.y);  // (as sum_to)
            l2 = mul2(mul2(l2, pack2(half, half)), pack2(half, half));
          }
          l_new = l2;
          float mx;
          if (open) {
            uint32_t q[NT / 2];
            uint64_t l = l2;
            mx = weigh_open<NT>(s_tmem, fac, f, kHead + kSpread - m, seen, q, &l);
#pragma unroll
            for (int i = 0; i < NT / 2; ++i) p[i] = q[i];
            l_new = l;
          } else {
            mx = weigh_pass<NT, false>(s_tmem, fac, f, kHead + kSpread - m, seen, p, l_new);
          }
          const bool more = quad_any(quad, mx > kMost);
          if (raise || !more) break;
          raise = true;
        }
        l2 = l_new;
        // P goes over the S that all of the quad's parts have read, by the barrier above
        const uint32_t p_tmem = my + Sh::kTmemS + (g & 1) * BT + part * (NT / 2);
        if constexpr (NT == 32)
          tmem_st16(p_tmem, p);
        else
          tmem_st8(p_tmem, p);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->pready[g & 1]);
      }
      float l0, l1;
      unpack2(l2, l0, l1);
      // A row tile that this block has whole is finished here.  Of the others a
      // block has two at most: the end of one (slot 0) and the start of another.
      const bool whole = sh->seg.starts && sh->seg.ends;
      const size_t slot = (size_t)blockIdx.x * 2 + (seg ? 1 : 0);
      sh->red[part][r_own] = l0 + l1;
      quad_sync(quad);
      if (part == 0 && !whole) {
        float l = 0.0f;
#pragma unroll
        for (int i = 0; i < kParts; ++i) l += sh->red[i][r_own];
        a.part_ml[slot * kTileRows + r_own] = make_float2(tiles ? m : -INFINITY, l);
      }
      if (tid == 0) {  // whose slots hold the row tile: from its first block's to its last's
        if (sh->seg.starts) a.shares[sh->seg.item].x = whole ? -1 : (int)slot;
        if (sh->seg.ends) a.shares[sh->seg.item].y = (int)blockIdx.x;
      }
      if (tiles) {
        if (ok) ok = mbar_wait(&sh->vempty[(g - 1) % ST], ((g - 1) / ST) & 1, abort_s);
        if (!ok) give_up(a.error, abort_s);
        __syncwarp();
        tc_fence_after();
        if (whole)
          write_rows(a, sh, BT, my + Sh::kTmemO);
        else
          write_part(a, sh, BT, slot, my + Sh::kTmemO);
      }
      soft_sync();  // O, red and the segment are read: the next may overwrite them
    }
  } else if (warp == kMmaWarp) {
    // ---- MMA issue ----
    // The whole warp keeps the loop, so that what it computes is known to be
    // the warp's; one lane issues.
    const bool leader = elect_one();
    const int D = a.head_dim;
    const uint32_t idesc_s = idesc_f16(128, BT, false), idesc_o = idesc_f16(128, D, true);
    Walk walk = sh->walk;
    Segment sg;
    uint32_t g = 0;
    bool ok = true;
    auto scores = [&](uint32_t i) {
      const uint32_t st = i % ST;
      ok = ok && mbar_wait(&sh->kfull[st], (i / ST) & 1, abort_s);
      // S of tile i lies where P of tile i - 2 was: its product is done
      if (ok && i >= 2) ok = mbar_wait(&sh->vempty[(i - 2) % ST], ((i - 2) / ST) & 1, abort_s);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) return;
      tc_fence_after();
      const uint64_t desc = smem_desc(smem_u32(sK) + st * Sh::kBytes, 16, 1024, 2);
      const uint32_t to = Sh::kTmemS + (i & 1) * BT;
      if (leader) {
#pragma unroll
        for (int k = 0; k < DP / 16; ++k)
          if (16 * k < D)
            mma_f16_ts(to, Sh::kTmemQ + 8 * k, desc + (((k >> 2) * (BT * 128) + (k & 3) * 32) >> 4), idesc_s, k > 0);
        tc_commit(&sh->sfull[i & 1]);
        tc_commit(&sh->kempty[st]);
      }
      __syncwarp();
    };
    for (uint32_t taken = 0; ok && walk.next(a, BT, sg);) {
      if (sg.j1 <= sg.j0) continue;
      ok = __all_sync(0xffffffffu, mbar_wait(&sh->qready, taken++ & 1, abort_s));
      if (!ok) break;
      tc_fence_after();
      const uint32_t g0 = g, g1 = g + (sg.j1 - sg.j0);
      scores(g0);
      for (; ok && g < g1; ++g) {
        if (g + 1 < g1) scores(g + 1);
        const uint32_t st = g % ST;
        ok = ok && mbar_wait(&sh->vfull[st], (g / ST) & 1, abort_s) &&
             mbar_wait(&sh->pready[g & 1], (g >> 1) & 1, abort_s);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        const uint64_t desc = smem_desc(smem_u32(sV) + st * Sh::kBytes, BT * 128, 1024, 2);
        const uint32_t from = Sh::kTmemS + (g & 1) * BT;
        if (leader) {
#pragma unroll
          for (int k = 0; k < BT / 16; ++k)
            mma_f16_ts(Sh::kTmemO, from + 8 * k, desc + (k * 2048 >> 4), idesc_o, g > g0 || k > 0);
          tc_commit(&sh->vempty[st]);
        }
        __syncwarp();
      }
    }
    if (!ok) {  // what was issued ends before its TMEM is given back
      if (leader) {
        give_up(a.error, abort_s);
        tc_commit(&sh->drain);
      }
      __syncwarp();
      mbar_wait(&sh->drain, 0, &sh->never);
    }
    __syncwarp();
  } else if (warp == kLoadWarp) {
    // ---- codes to shared memory ----
    if (lane == 0) {
      Walk walk = sh->walk;
      Segment sg;
      uint32_t g = 0;
      bool ok = true;
      const int boxes = (a.head_dim + Sh::kBox - 1) / Sh::kBox;
      while (ok && walk.next(a, BT, sg)) {
        for (int j = sg.j0; ok && j < sg.j1; ++j, ++g) {
          const int st = g % RAW;
          auto fetch = [&](const CUtensorMap *map, uint8_t *to, uint64_t *full, uint64_t *empty) {
            if (g >= RAW && ok) ok = mbar_wait(empty, ((g / RAW) - 1) & 1, abort_s);
            if (!ok) return;
            mbar_arrive_expect_tx(full, (uint32_t)boxes * (BT * Sh::kBox));
            for (int x = 0; x < boxes; ++x)
              tma_load_4d(to + x * (BT * Sh::kBox), map, x * Sh::kBox, sg.kvh, j * BT, sg.b, full);
          };
          fetch(&k_map, rK + st * Sh::kRawBytes, &sh->rkfull[st], &sh->rkempty[st]);
          fetch(&v_map, rV + st * Sh::kRawBytes, &sh->rvfull[st], &sh->rvempty[st]);
        }
      }
      if (!ok) give_up(a.error, abort_s);
      // the copies in flight land before the block ends
      for (uint32_t i = g > RAW ? g - RAW : 0; i < g; ++i) {
        mbar_wait(&sh->rkfull[i % RAW], (i / RAW) & 1, &sh->never);
        mbar_wait(&sh->rvfull[i % RAW], (i / RAW) & 1, &sh->never);
      }
    }
    __syncwarp();
  } else {
    // ---- codes to f16 tiles ----
    // A warp takes 64 bytes of eight tokens at a time (lane % 8 the token, lane
    // / 8 the 16-byte piece): eight lanes' 16-byte accesses then fall on all
    // banks on both sides, and a thread's pieces lie at one distance.
    const int cw = warp - kConvWarp;
    constexpr int P = Sh::kPieces, X = BT / 32, kStep = BT / P;
    const int ch = (cw % (DP / 64)) * 4 + (lane >> 3), t_own = cw / (DP / 64) * 8 + (lane & 7);
    const uint32_t src = DP == 64 ? t_own * 64 + ((ch ^ ((t_own >> 1) & 3)) * 16)
                                  : (ch >> 3) * (BT * 128) + t_own * 128 + (((ch & 7) ^ (t_own & 7)) * 16);
    const uint32_t dst = (ch >> 2) * (BT * 128) + t_own * 128 + (((2 * (ch & 3)) ^ (t_own & 7)) * 16);
    Walk walk = sh->walk;
    Segment sg;
    bool more = false;
    int j = 0;
    auto enter = [&]() {  // the next segment that is not empty
      do more = walk.next(a, BT, sg);
      while (more && sg.j1 <= sg.j0);
      j = more ? sg.j0 : 0;
    };
    enter();
    uint32_t xk[X], xv[X];
    auto load_exps = [&]() {
      const size_t row = ((size_t)sg.b * a.max_seq + (size_t)j * BT) * a.kv_heads + sg.kvh;
      const int live = sg.total - j * BT;
#pragma unroll
      for (int i = 0; i < X; ++i) {
        const int t = lane + 32 * i;
        xk[i] = t < live ? a.k_exp[row + (size_t)t * a.kv_heads] : 127;
        xv[i] = t < live ? a.v_exp[row + (size_t)t * a.kv_heads] : 127;
      }
    };
    auto fetch = [&](const uint8_t *stage, uint4(&v)[P]) {
#pragma unroll
      for (int i = 0; i < P; ++i)
        v[i] = *reinterpret_cast<const uint4 *>(stage + src + i * kStep * (DP == 64 ? 64 : 128));
    };
    // (one tile's pieces are held at a time: with both, spilled registers cost 4 x
    // 61 at 30011 188 us instead of 177)
    auto store = [&](uint8_t *stage, const uint4(&v)[P]) {
      uint8_t *to = stage + dst, *and_to = stage + (dst ^ 16);
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
        uint32_t o[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          o[2 * k] = e4m3x2_to_f16x2((uint16_t)w[k]);
          o[2 * k + 1] = e4m3x2_to_f16x2((uint16_t)(w[k] >> 16));
        }
        *reinterpret_cast<uint4 *>(to + i * kStep * 128) = make_uint4(o[0], o[1], o[2], o[3]);
        *reinterpret_cast<uint4 *>(and_to + i * kStep * 128) = make_uint4(o[4], o[5], o[6], o[7]);
      }
      fence_proxy_async_smem();
      __syncwarp();
    };
    if (more && cw == 0) load_exps();
    // After a wait that ran out this role goes on to its end without waiting
    // (the results are void): its warps meet at a barrier in open tiles.
    bool ok = true;
    auto wait = [&](uint64_t *bar, uint32_t phase) {
      if (ok) ok = mbar_wait(bar, phase & 1, abort_s);
      if (!ok) give_up(a.error, abort_s);
      __syncwarp();
    };
    for (uint32_t g = 0; more; ++g) {
      const int st = g % ST, rs = g % RAW;
      const bool open = (j + 1) * BT > sg.pos;
      float *ft = reinterpret_cast<float *>(sh->fac[g % META]);
      uint4 cb[P];
      wait(&sh->rkfull[rs], g / RAW);
      if (cw == 0) {
#pragma unroll
        for (int i = 0; i < X; ++i) {
          const int t = lane + 32 * i;
          ft[(t >> 1) * 4 + (t & 1)] = kv8_factor(xk[i]) * kKeyShift;
          ft[(t >> 1) * 4 + 2 + (t & 1)] = pow2i((int)kv8_value_exponent(xv[i]) - kSpread);
        }
      }
      if (open) {  // values that are not a number: zero in the product, and told to the softmax ahead of the tile
        wait(&sh->rvfull[rs], g / RAW);
#pragma unroll 1
        for (int i = 0; i < P; ++i) {
          const uint4 v = *reinterpret_cast<const uint4 *>(rV + rs * Sh::kRawBytes + src + i * kStep * (DP == 64 ? 64 : 128));
          if (not_numbers(v.x) | not_numbers(v.y) | not_numbers(v.z) | not_numbers(v.w)) sh->nan = 1;
        }
        conv_sync();
      }
      __syncwarp();
      if (cw == 0 && lane == 0) mbar_arrive(&sh->metafull[g % META]);
      fetch(rK + rs * Sh::kRawBytes, cb);
      if (g >= ST) wait(&sh->kempty[st], g / ST - 1);
      store(sK + st * Sh::kBytes, cb);
      if (lane == 0) {
        mbar_arrive(&sh->kfull[st]);
        mbar_arrive(&sh->rkempty[rs]);
      }
      if (!open) wait(&sh->rvfull[rs], g / RAW);
      fetch(rV + rs * Sh::kRawBytes, cb);
      if (open) {
#pragma unroll
        for (int i = 0; i < P; ++i) {
          cb[i].x &= ~not_numbers(cb[i].x);
          cb[i].y &= ~not_numbers(cb[i].y);
          cb[i].z &= ~not_numbers(cb[i].z);
          cb[i].w &= ~not_numbers(cb[i].w);
        }
      }
      if (++j >= sg.j1) enter();
      if (more && cw == 0) load_exps();
      if (g >= ST) wait(&sh->vempty[st], g / ST - 1);
      store(sV + st * Sh::kBytes, cb);
      if (lane == 0) {
        mbar_arrive(&sh->vfull[st]);
        mbar_arrive(&sh->rvempty[rs]);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(sh->tmem, 512);
  }
  // (a block without a share too: when this grid has ended, so has the prep grid)
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// The blocks that share a row tile's tokens meet, in order, with the gate:
// block (16 rows of a row tile, blockDim.x / 2 columns); thread (row, eight
// columns, share of the blocks).  Rows of nodes that are not there become zeros,
// and those of sessions that no block has.  What the tile kernel does not write
// is read before it is waited for.  Bound by the latency of two reads in a row
// (whose slots, then their values, in L2): 5 us for 21 MB of 148 blocks.
constexpr int kMergeThreads = 1024;
__global__ void __launch_bounds__(kMergeThreads, 1) tree_attn_tile_merge_kernel(const __grid_constant__ TreeArgs a, int BT) {
  __shared__ float4 acc_s[2][kMergeThreads];
  __shared__ float2 ml_s[kMergeThreads];
  const int t = threadIdx.x, share = threadIdx.y, D = a.head_dim;
  const int rows = a.nodes * a.group, row_tiles = (rows + kTileRows - 1) / kTileRows, items = a.kv_heads * row_tiles;
  const int item = blockIdx.x / (kTileRows / 16), r = blockIdx.x % (kTileRows / 16) * 16 + (t & 15);
  const int b = item / items, kvh = item % items / row_tiles, row = item % row_tiles * kTileRows + r;
  asm volatile("griddepcontrol.launch_dependents;");
  if (item % row_tiles * kTileRows + (r & ~15) >= rows) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    return;
  }
  const int d = blockIdx.y * (blockDim.x / 2) + 8 * (t >> 4);
  const bool live = row < rows && d < D;
  const int n = row / a.group, h = kvh * a.group + row % a.group, pos = a.positions[b];
  const size_t node = (size_t)b * a.nodes + n;
  const bool some = session_tiles(a, b, BT) > 0;
  float gate[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) gate[i] = 1.0f;
  if (live && a.gate && share == 0) {
    const float *g = a.gate + node * a.gate_pitch + (size_t)h * a.gate_head + d;
#pragma unroll
    for (int i = 0; i < 8; ++i) gate[i] = 1.0f + expf(-g[i]);
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  float m = -INFINITY, l = 0.0f;
  float acc[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = 0.0f;
  auto add = [&](float2 v, float4 x, float4 y) {
    const float mn = fmaxf(m, v.x), fo = exp2_approx(m - mn), fn = exp2_approx(v.x - mn);
    const float z[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
    l = sum_to(l, m - mn) + sum_to(v.y, v.x - mn);
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = acc[i] * fo + z[i] * fn;
    m = mn;
  };
  const int2 from = some ? a.shares[item] : make_int2(0, -1);  // its first slot, its last block
  if (from.x < 0) return;                                      // one block had it whole
  if (some) {
    const float4 *part = reinterpret_cast<const float4 *>(a.part) + (size_t)(live ? d / 4 : 0) * kTileRows + r;
    const int c0 = from.x >> 1;
#pragma unroll 4
    for (int c = c0 + share; c <= from.y; c += blockDim.y) {
      const size_t slot = c == c0 ? from.x : c * 2;
      const float2 v = a.part_ml[slot * kTileRows + r];
      const float4 *p = part + slot * (kTileRows * (size_t)D / 4);
      const float4 x = p[0], y = p[kTileRows];
      if (v.x != -INFINITY) add(v, x, y);
    }
  }
  if (blockDim.y > 1) {
    const int at = share * blockDim.x + t;
    if (share > 0) {
      acc_s[0][at] = make_float4(acc[0], acc[1], acc[2], acc[3]);
      acc_s[1][at] = make_float4(acc[4], acc[5], acc[6], acc[7]);
      ml_s[at] = make_float2(m, l);
    }
    __syncthreads();
    if (share > 0) return;
    for (int i = at + blockDim.x; i < (int)(blockDim.x * blockDim.y); i += blockDim.x)
      if (ml_s[i].x != -INFINITY) add(ml_s[i], acc_s[0][i], acc_s[1][i]);
  }
  if (!live) return;
  const bool there = some && (a.parents ? a.sights[(size_t)b * kTreeMaxNodes + n] != 0 : pos >= 0 && pos < a.max_seq - n);
  const float inv = kSumBack / l;
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = there ? acc[i] * inv / gate[i] : 0.0f;
  *reinterpret_cast<uint4 *>(a.out + (node * a.q_heads + h) * D + d) =
      make_uint4(pack_bf16x2(acc[0], acc[1]), pack_bf16x2(acc[2], acc[3]), pack_bf16x2(acc[4], acc[5]),
                 pack_bf16x2(acc[6], acc[7]));
}

template <int DP>
int launch(const TreeArgs &a, const TilePlan &p, cudaStream_t s) {
  using Sh = TileShape<DP>;
  constexpr size_t smem =
      (sizeof(TileShared) + 1023) / 1024 * 1024 + 2 * (size_t)Sh::ST * Sh::kBytes + 2 * (size_t)Sh::RAW * Sh::kRawBytes;
  static_assert(smem <= 227 * 1024);
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
  CUtensorMap k_map, v_map;
  if (int st = encode_cache_u8(&k_map, a.k_codes, a.batch, a.max_seq, a.kv_heads, a.head_dim, Sh::kBox, Sh::BT))
    return st;
  if (int st = encode_cache_u8(&v_map, a.v_codes, a.batch, a.max_seq, a.kv_heads, a.head_dim, Sh::kBox, Sh::BT))
    return st;
  cudaError_t e = launch_pdl(tree_attn_prep_kernel, dim3((unsigned)(p.items * (kTileRows / kPrepRows) + p.batch)), 256, 0, s, a);
  if (e != cudaSuccess) return cuda_fail(e, "tree_attn_prep_kernel");
  FPB_LAUNCH_CHECK("tree_attn_prep_kernel");
  e =
      launch_pdl(tree_attn_tile_kernel<DP>, dim3((unsigned)p.blocks), kTileThreads, smem, s, a, k_map, v_map);
  if (e != cudaSuccess) return cuda_fail(e, "tree_attn_tile_kernel");
  FPB_LAUNCH_CHECK("tree_attn_tile_kernel");
  // A row tile's blocks in one thread's loop while they are few, else shared, by
  // narrower blocks of more shares where they are many and the row tiles few
  // (whole calls; 74 blocks a row tile: 16 shares 22.4 us, 4 shares 31, none 66;
  // 18: 4 shares 57 us, 16 shares 69, none 65; 9: 2 shares 65 us, 4 shares 67,
  // none 68; 4: none 202 us, 2 shares 205, 4 shares 211).
  const size_t each = p.blocks / p.items;
  const unsigned shares = each > 32 ? 16 : each > 16 ? 4 : each > 8 ? 2 : 1, cols = shares == 16 ? 32 : 128;
  e = launch_pdl(tree_attn_tile_merge_kernel,
                 dim3((unsigned)(p.items * (kTileRows / 16)), (unsigned)((a.head_dim + cols - 1) / cols)),
                 dim3(2 * cols, shares), 0, s, a, p.BT);
  if (e != cudaSuccess) return cuda_fail(e, "tree_attn_tile_merge_kernel");
  FPB_LAUNCH_CHECK("tree_attn_tile_merge_kernel");
  return FPB_OK;
}

}  // namespace

TilePlan tile_plan(size_t batch, size_t nodes, size_t q_heads, size_t kv_heads, size_t head_dim, size_t max_seq) {
  TilePlan p;
  p.BT = head_dim > 128 ? 64 : 128;
  p.batch = batch;
  p.items = batch * kv_heads * ((nodes * (q_heads / kv_heads) + kTileRows - 1) / kTileRows);
  p.units = p.items * ((max_seq + p.BT - 1) / p.BT + kTakeUp / p.BT);
  p.blocks = (int)std::min<size_t>(sm_count(), p.items * ((max_seq + p.BT - 1) / p.BT));
  return p;
}

// The workspace: queries, partial results, sums, sights, factors, items' shares.
static size_t lay_out(TreeArgs *a, const TilePlan &p, size_t head_dim, void *workspace) {
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 15) / 16 * 16;
    return static_cast<uint8_t *>(workspace) + here;
  };
  TreeArgs unused{};
  if (!a) a = &unused;
  const size_t slots = (size_t)p.blocks * 2 * kTileRows;
  a->q16 = reinterpret_cast<uint4 *>(take(p.items * kTileRows * head_dim * 2));
  a->part = reinterpret_cast<float *>(take(slots * head_dim * 4));
  a->part_ml = reinterpret_cast<float2 *>(take(slots * sizeof(float2)));
  a->sights = reinterpret_cast<uint64_t *>(take(p.batch * kTreeMaxNodes * 8));
  a->q_fac = reinterpret_cast<float *>(take(p.items * kTileRows * 4));
  a->shares = reinterpret_cast<int2 *>(take(p.items * sizeof(int2)));
  return at;
}

size_t tile_workspace_bytes(const TilePlan &p, size_t head_dim) { return lay_out(nullptr, p, head_dim, nullptr); }

int run_tree_tiles(TreeArgs a, const TilePlan &p, void *workspace, cudaStream_t s) {
  lay_out(&a, p, a.head_dim, workspace);
  return a.head_dim <= 64 ? launch<64>(a, p, s) : a.head_dim <= 128 ? launch<128>(a, p, s) : launch<256>(a, p, s);
}

}  // namespace fpb
