// Attention of one new token a session over the paged cache (paged.cuh).
//
// Session b's query heads see the tokens t < lengths[b].  With s_t = scale q . k_t:
//   out = sum_t softmax(s)_t v_t, times sigmoid(gate) where a gate is given.
// One pass over the tokens: a warp holds its rows' running maximum m, sum of weights l
// and numerators, all f32, and two such parts meet as l1 2^(m1 - m) + l2 2^(m2 - m).
//
// Bound by the pages' bytes, each read once: 200 ragged sessions (1.65 GB) 253 us, 6.5
// TB/s; 3 x 100003 tokens x 4 heads of 128, bf16, 103 us, 5.5; 16 x 8192 x 2 heads of
// 256 47.6 us, 5.0; 8 x 2304 of f32 25.0 us.  About 10 us of a call do not depend on the
// bytes: the launch, the cut into shares, the first copies' way and the shares' meeting
// (1 x 777 tokens 10.6 us).
// A warp takes steps of 16 tokens (f32: 8) through a ring of TMA copies that it alone
// waits for, so that the block meets only at the end.  The products go by mma.sync: a
// kv head has up to 16 rows of queries, which would leave most of a tcgen05 tile's 128
// empty, and the copies are what takes the time.
// Products keep f32's precision: over bf16 pages f32 queries, and the weights beside
// them, are three bf16 parts, exact in their products (with two, 2^-16 of a factor, 16 x
// 8192 tokens were 5.3e-6 off in relative 2-norm, so 1.1e-6, where f32 arithmetic is 1.7e-6.
// Two and three: 16 x 8192 tokens 47.2 and 47.6 us, 1 x 777 10.2 and 10.6; where 16 rows
// make the products the bound 53 and 60, 40 x 4000 x 4 heads of 128 85 and 101).  Beside bf16
// queries, which are exact, weights are two (2^-16 of themselves).  Over f32 pages products
// are good to 2^-20: every factor is two parts of 11 bits, and the parts' small product is
// left out.  Sums are f32.
#include <algorithm>
#include <atomic>
#include <chrono>
#include <cmath>
#include <mutex>
#include <vector>

#include "paged.cuh"
#include "sm100.cuh"
#include "tma_host.cuh"

namespace fpb {
namespace {

using namespace sm100;

struct PagedArgs {
  const void *q, *k, *v;
  const float *gate;
  const int32_t *table, *lengths;
  long long q_pitch, q_head, gate_pitch, gate_head, table_pitch;  // elements
  long long page_pitch, row_pitch, head_pitch;                    // of k and v
  int batch, q_heads, kv_heads, group, head_dim, max_pages, pages, page_size, q_bf16, q_vec;
  int box;     // tokens of a copy: the largest power of two that divides the page size, up to a step's
  int whole;   // a copy takes all of a head vector's 128-byte pieces (else one: the last is not whole)
  int tiles;   // row tiles of a kv head's query heads
  int tok;     // tokens of a step
  int least;   // steps of a share, at least
  int slots;   // blocks that the GPU has room for
  int waves;   // 0: no more blocks than that; else shares of 1 / (waves * slots) of the steps
  float scale_log2;  // scale * log2(e): scores and maxima are held in powers of two
  void *out;
  int out_bf16;
  float *part;      // [slot][row][head_dim] the share's own outputs
  float2 *part_ml;  // [slot][row] maximum, sum of weights
  unsigned long long *flags, token;  // [slot]: `token`, this call's own, where the share's results are there
  int *error;
};

constexpr int kPagedMaxBatch = 4096, kPagedWaves = 2;
constexpr int kErrPagedWait = 503;
// The maximum may lag by kLag (powers of two) before the sums are rescaled: weights
// are 2^(y - m), up to 2^8, so that values down to the smallest normal number give
// normal numerators, and weights down to 2^-126 count.
constexpr float kLag = 8.0f;
// Outputs of a share over f32 pages below this (or not finite ones over any) are found again
// by plain_share(): the tensor cores hold the low parts of numbers below 2^-116 to 2^-136.
// (bf16 parts are whole down to 2^-133 of a sum.)
constexpr float kSmall = 1.9259299e-34f;  // 2^-112

__device__ __forceinline__ float pow2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two f32 sums at once.
__device__ __forceinline__ void add2(float &x, float &y, float u, float v) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(r)
      : "l"((uint64_t)__float_as_uint(y) << 32 | __float_as_uint(x)), "l"((uint64_t)__float_as_uint(v) << 32 | __float_as_uint(u)));
  x = __uint_as_float((uint32_t)r);
  y = __uint_as_float((uint32_t)(r >> 32));
}

__device__ __forceinline__ void mma_tf32(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// An f32 as what the tensor cores take of it (11 bits) and the rest of it, of which
// they take 11 more.  Cut: 2^-20 is lost at most, and 2^-10 the rest's size;
// nearest: 2^-21 and 2^-11.
__device__ __forceinline__ void split_cut(uint32_t x, uint32_t *hi, uint32_t *lo) {
  *hi = x & 0xffffe000u;
  *lo = __float_as_uint(__uint_as_float(x) - __uint_as_float(*hi));
}
__device__ __forceinline__ void split_nearest(float x, uint32_t *hi, uint32_t *lo) {
  const uint32_t h = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
  *hi = h;
  *lo = __float_as_uint(x - __uint_as_float(h));
}

__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Four 8 x 8 matrices of bf16, transposed; lane 8 i + r holds the address of row r of matrix i.
__device__ __forceinline__ void load_transposed(uint32_t (&x)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3])
               : "r"(addr)
               : "memory");
}

// An 8 x 8 matrix of 16-bit pairs (lane 4 r + c: row r, columns 2 c and 2 c + 1), transposed.
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// (lo, hi) as bf16 pairs, and what the rounding left of them in further ones.
template <int N>
__device__ __forceinline__ void split_bf16x2(float lo, float hi, uint32_t (&parts)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    parts[i] = pack_bf16x2(lo, hi);
    lo -= __uint_as_float(parts[i] << 16);
    hi -= __uint_as_float(parts[i] & 0xffff0000u);
  }
}

__device__ __forceinline__ float load_q(const PagedArgs &a, int b, int h, int d) {
  const size_t at = (size_t)b * a.q_pitch + (size_t)h * a.q_head + d;
  return a.q_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16 *>(a.q)[at]) : static_cast<const float *>(a.q)[at];
}

// Eight elements of a query from column d on (a multiple of 8); zeros where `there` is false.
__device__ __forceinline__ void load_q8(const PagedArgs &a, int b, int h, int d, bool there, float (&x)[8]) {
#pragma unroll
  for (int k = 0; k < 8; ++k) x[k] = 0.0f;
  if (!there) return;
  const size_t at = (size_t)b * a.q_pitch + (size_t)h * a.q_head + d;
  if (!a.q_vec) {
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = load_q(a, b, h, d + k);
  } else if (a.q_bf16) {
    const uint4 v = *reinterpret_cast<const uint4 *>(static_cast<const __nv_bfloat16 *>(a.q) + at);
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      x[2 * k] = __uint_as_float(u[k] << 16);
      x[2 * k + 1] = __uint_as_float(u[k] & 0xffff0000u);
    }
  } else {
    const float4 *p = reinterpret_cast<const float4 *>(static_cast<const float *>(a.q) + at);
    const float4 u = p[0], v = p[1];
    x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w;
    x[4] = v.x; x[5] = v.y; x[6] = v.z; x[7] = v.w;
  }
}

// N columns of head h from d on: the outputs x, times the gate's sigmoid where there is
// one.  No weights (their sum l is 0): zeros.
template <int N>
__device__ __forceinline__ void store_out(const PagedArgs &a, int b, int h, int d, const float (&x)[N], float l,
                                          const float (&gate)[N]) {
  const size_t at = ((size_t)b * a.q_heads + h) * a.head_dim + d;
  float o[N];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    o[k] = l != 0.0f ? x[k] : 0.0f;
    if (a.gate && l != 0.0f) o[k] /= 1.0f + expf(-gate[k]);
  }
#pragma unroll
  for (int k = 0; k < N; k += 2) {
    if (a.out_bf16)
      *reinterpret_cast<uint32_t *>(static_cast<__nv_bfloat16 *>(a.out) + at + k) = pack_bf16x2(o[k], o[k + 1]);
    else
      *reinterpret_cast<float2 *>(static_cast<float *>(a.out) + at + k) = make_float2(o[k], o[k + 1]);
  }
}

// What a block does: steps [first, first + count) of a session's kv head and row tile.
struct PagedShare {
  int b, kvh, tile, length, first, count, part, parts, slot;
};

// Two columns of a share's row r: its output where the session is whole, else for the join.
__device__ __forceinline__ void keep_out(const PagedArgs &a, const PagedShare &me, int rows, int r, int h, int d, float2 o,
                                         float sum) {
  if (me.parts > 1) {
    *reinterpret_cast<float2 *>(a.part + ((size_t)me.slot * rows + r) * a.head_dim + d) = o;
    return;
  }
  const float *g = a.gate ? a.gate + (size_t)me.b * a.gate_pitch + (size_t)h * a.gate_head + d : nullptr;
  const float x[2] = {o.x, o.y}, gate[2] = {g ? g[0] : 0.0f, g ? g[1] : 0.0f};
  store_out<2>(a, me.b, h, d, x, sum, gate);
}

// Operand row i of eight is token token_at(i) of its eight: a quarter of a warp
// then reads 16 bytes from all of the banks.  For f32 the values' rows are read by
// pairs of them too.
template <typename T>
__device__ __forceinline__ int token_at(int i) {
  return sizeof(T) == 2 ? (i >> 1) | (i & 1) << 2 : i & 1 ? ((i - 1) ^ 4) | 1 : i;
}

// Blocks of W warps.  Where the calls' blocks are all there at once there is one an
// SM, of 8 or 12 warps: smaller ones, two or three an SM, leave registers that do
// not lie together when the kernel before is still there, and an SM then takes one
// block less (3 x 100003 tokens behind another call 172 us, alone 106).  Where they
// come one after another small blocks overlap their beginnings and ends.
constexpr int warps_of(int DP, bool f32, bool once) { return !once ? 4 : DP == 256 && !f32 ? 8 : 12; }
constexpr int blocks_of(int DP, bool once) { return once ? 1 : DP == 256 ? 2 : 3; }

// QF: f32 queries (over f32 pages always: what there is of bf16 ones is converted).
template <typename T, int DP, int NR, bool ONCE, bool QF>
struct PagedShape {
  static constexpr bool kHalf = sizeof(T) == 2;
  static constexpr int W = warps_of(DP, !kHalf, ONCE), kThreads = 32 * W, kBlocks = blocks_of(DP, ONCE);
  static constexpr int kTok = kHalf ? 16 : 8;                       // tokens of a step
  static constexpr int kCols = 128 / (int)sizeof(T), kBoxes = DP / kCols;  // a copy's columns; copies side by side
  static constexpr uint32_t kPart = kTok * DP * sizeof(T);          // a step's keys, or its values
  static constexpr int kParts = (DP == 256 ? (kHalf ? 3 : 2) : DP == 128 ? 4 : 6) -
                                (!ONCE && (NR == 16 || (!kHalf && DP == 128)));  // of a warp's ring
  static constexpr bool kQShared = NR == 16 && DP >= 128;           // too many registers of queries beside those of sums
  static constexpr int kQPitch = DP + (kHalf ? 32 : 16);            // elements: 16-byte reads of eight rows on distinct banks
  static constexpr int kEndPitch = DP + 4;
  static constexpr size_t kRing = (size_t)W * kParts * kPart;
  static constexpr size_t kEnd = (size_t)W * NR * kEndPitch * 4;  // the warps' results, over the ring
  static constexpr size_t kPlan = (size_t)kPagedMaxBatch * 4;     // the sessions' steps, over the ring
  static constexpr size_t kOver = kRing > kEnd ? kRing : kEnd;
  static constexpr int kQParts = !kHalf ? 2 : QF ? 3 : 1, kPParts = QF ? 3 : 2;  // of the queries, of the weights over bf16 pages
  static constexpr size_t kQueries = (size_t)kQParts * NR * kQPitch * sizeof(T);
  static constexpr size_t smem = 1023 + kOver + kQueries;
  static_assert(kPlan <= kOver && kBlocks * (smem + 3 * 1024) <= 228 * 1024);
};

// The sessions' steps are cut into shares of S, each session's evenly, and the
// shares numbered in order of session, kv head, part and row tile.  Every block
// finds its own: false where there is none.  `steps` [batch] in shared memory.
// Where the GPU has room for an item a block: the smallest S whose shares it has room
// for at once, total / slots or else among 32 between that, which is below it, and total
// / (slots - items), whose shares fit (each item rounds up by less than one).  Shares
// that may come one after another: total / (waves * slots); but where that is less than
// a share's least, a few blocks more than there is room for would take as long as all of
// them, so one wave then, too, with heads of up to 128 (us for two waves and one: f32
// pages, 20 x 2000 tokens x 8 heads of 128 85 and 67, 55 x 600 73 and 53; longer ones want
// the finer shares, 37 x 9000 492 and 579, and so do 110 x 2000 x 2 heads of 256, 51 and
// 58).

// Lane 0 lo, lane 31 hi, the others between them, in even ratios but for rounding.
__device__ __forceinline__ int between(int lo, int hi) {
  const int lane = threadIdx.x & 31;
  const float ratio = __log2f((float)hi / (float)lo) * (1.0f / 31.0f);
  return lane == 31 ? hi : min(hi, (int)((float)lo * exp2f(ratio * lane)));
}

// Up to 32 sessions: every warp finds the shares on its own, a session a lane.
struct FewPlan {
  int length, steps, parts;   // of the lane's session
  int blocks0, slots0;        // blocks, and slots of sessions that are cut, before it
};

// From the lane's session's length.
__device__ __noinline__ FewPlan few_plan(const PagedArgs &a, int n) {
  const int lane = threadIdx.x & 31, heads = a.kv_heads * a.tiles;
  FewPlan p{};
  if (n < 0 || n > (long long)a.max_pages * a.page_size) n = 0;
  p.length = n;
  p.steps = n / a.tok + (n % a.tok != 0);
  const uint32_t alive = __ballot_sync(0xffffffffu, p.steps > 0);
  unsigned long long work = p.steps;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) work += __shfl_xor_sync(0xffffffffu, work, o);
  work *= heads;
  if (work == 0) return p;
  // ceil(work / n); 64-bit quotients take a few hundred cycles
  auto over = [&](uint32_t n) { return work >> 31 ? (int)min((work + n - 1) / n, 0x7fffffffull) : (int)(((uint32_t)work + n - 1) / n); };
  const uint32_t items = __popc(alive) * heads;
  int S = over((uint32_t)max(1, a.waves) * a.slots);
  const bool one = items < (uint32_t)a.slots && (!a.waves || (a.head_dim <= 128 && S < a.least));
  S = max(a.least, one ? over(a.slots) : S);
  if (one && __reduce_add_sync(0xffffffffu, ((uint32_t)p.steps + S - 1) / S) * heads > (uint32_t)a.slots) {
    const int lo = over(a.slots), hi = over(a.slots - items);
    const uint32_t trial = max(a.least, between(lo, hi));
    uint32_t blocks = 0;
#pragma unroll 4
    for (int b = 0; b < a.batch; ++b) blocks += ((uint32_t)__shfl_sync(0xffffffffu, p.steps, b) + trial - 1) / trial;
    const uint32_t fits = __ballot_sync(0xffffffffu, blocks * heads <= a.slots);
    S = __shfl_sync(0xffffffffu, (int)trial, __ffs(fits) - 1);
  }
  p.parts = (int)(((uint32_t)p.steps + S - 1) / S);
  const int blocks = p.parts * heads, slots = p.parts > 1 ? blocks : 0;
  int x = blocks, y = slots;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, x, o), v = __shfl_up_sync(0xffffffffu, y, o);
    if (lane >= o) {
      x += u;
      y += v;
    }
  }
  p.blocks0 = x - blocks;
  p.slots0 = y - slots;
  return p;
}

__device__ __forceinline__ bool paged_share_few(const PagedArgs &a, int length, uint32_t *empty, PagedShare *out) {
  const FewPlan p = few_plan(a, length);
  *empty = __ballot_sync(0xffffffffu, (int)(threadIdx.x & 31) < a.batch && p.steps == 0);
  const int x = (int)blockIdx.x - p.blocks0;
  const uint32_t mine = __ballot_sync(0xffffffffu, x >= 0 && x < p.parts * a.kv_heads * a.tiles);
  if (!mine) return false;
  const int b = __ffs(mine) - 1, P = __shfl_sync(0xffffffffu, p.parts, b), total = __shfl_sync(0xffffffffu, p.steps, b);
  const int at = __shfl_sync(0xffffffffu, x, b);
  out->b = b;
  out->tile = at % a.tiles;
  out->part = at / a.tiles % P;
  out->parts = P;
  out->kvh = at / a.tiles / P;
  out->length = __shfl_sync(0xffffffffu, p.length, b);
  out->first = (int)((long long)total * out->part / P);
  out->count = (int)((long long)total * (out->part + 1) / P) - out->first;
  out->slot = __shfl_sync(0xffffffffu, p.slots0, b) + (out->kvh * a.tiles + out->tile) * P + out->part;
  return true;
}

template <int TOK, int W>
__device__ __forceinline__ bool paged_share(const PagedArgs &a, int *steps, PagedShare *out) {
  constexpr int kThreads = 32 * W;
  __shared__ unsigned long long sum_s[W];
  __shared__ int alive_s[W], blocks_s[W][32], found_s[4];
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const long long most = (long long)a.max_pages * a.page_size;
  unsigned long long sum = 0;
  int alive = 0;
  for (int b = tid; b < a.batch; b += kThreads) {
    int n = a.lengths[b];
    if (n < 0 || n > most) {
      if (blockIdx.x == 0 && a.error) atomicCAS(a.error, 0, kErrLength);
      n = 0;
    }
    const int s = n / TOK + (n % TOK != 0);
    steps[b] = s;
    sum += s;
    alive += s > 0;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    alive += __shfl_xor_sync(0xffffffffu, alive, o);
  }
  if (lane == 0) {
    sum_s[w] = sum;
    alive_s[w] = alive;
  }
  if (tid == 0) found_s[0] = -1;
  __syncthreads();
  sum = 0;
  alive = 0;
#pragma unroll
  for (int i = 0; i < W; ++i) {
    sum += sum_s[i];
    alive += alive_s[i];
  }
  const int heads = a.kv_heads * a.tiles;
  const unsigned long long work = sum * heads;
  if (work == 0) return false;
  const uint32_t items = alive * heads;
  auto over = [&](uint32_t n) { return (int)min((work + n - 1) / n, 0x7fffffffull); };
  int S = over((uint32_t)max(1, a.waves) * a.slots);
  const bool one = items < (uint32_t)a.slots && (!a.waves || (a.head_dim <= 128 && S < a.least));
  S = max(a.least, one ? over(a.slots) : S);
  bool fit = true;
  if (one) {  // whether the blocks of that many steps each do
    uint32_t n = 0;
    for (int b = tid; b < a.batch; b += kThreads) n += ((uint32_t)steps[b] + S - 1) / S;
    n = __reduce_add_sync(0xffffffffu, n);
    if (lane == 0) blocks_s[w][0] = (int)n;
    __syncthreads();
    n = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) n += blocks_s[i][0];
    fit = n * heads <= (uint32_t)a.slots;
    __syncthreads();
  }
  if (!fit) {
    const int lo = over(a.slots), hi = over(a.slots - items);
    const uint32_t trial = max(a.least, between(lo, hi));
    uint32_t n = 0;
    for (int b = w; b < a.batch; b += W) n += ((uint32_t)steps[b] + trial - 1) / trial;
    blocks_s[w][lane] = (int)n;
    __syncthreads();
    n = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) n += blocks_s[i][lane];
    const uint32_t fits = __ballot_sync(0xffffffffu, n * heads <= (uint32_t)a.slots);
    S = __shfl_sync(0xffffffffu, (int)trial, __ffs(fits) - 1);
  }
  // the session of this block, and the slots of split sessions before it
  int blocks0 = 0, slots0 = 0;
  for (int b0 = 0; b0 < a.batch; b0 += kThreads) {
    const int b = b0 + tid, n = b < a.batch ? (int)(((uint32_t)steps[b] + S - 1) / S) : 0;
    int blocks = n * heads, slots = n > 1 ? blocks : 0, x = blocks, y = slots;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, x, o), v = __shfl_up_sync(0xffffffffu, y, o);
      if (lane >= o) {
        x += u;
        y += v;
      }
    }
    __syncthreads();  // (the words below are read)
    if (lane == 31) {
      blocks_s[w][0] = x;
      blocks_s[w][1] = y;
    }
    __syncthreads();
    int before = blocks0, slots_before = slots0;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      if (i < w) {
        before += blocks_s[i][0];
        slots_before += blocks_s[i][1];
      }
      blocks0 += blocks_s[i][0];
      slots0 += blocks_s[i][1];
    }
    before += x - blocks;
    slots_before += y - slots;
    if ((int)blockIdx.x >= before && (int)blockIdx.x < before + blocks) {
      found_s[0] = b;
      found_s[1] = before;
      found_s[2] = slots_before;
      found_s[3] = n;
    }
    __syncthreads();
    if (found_s[0] >= 0 || (int)blockIdx.x < blocks0) break;
  }
  const int b = found_s[0];
  if (b < 0) return false;
  const int n = found_s[3], at = (int)blockIdx.x - found_s[1], tile = at % a.tiles, part = at / a.tiles % n;
  out->b = b;
  out->tile = tile;
  out->part = part;
  out->parts = n;
  out->kvh = at / a.tiles / n;
  out->length = a.lengths[b];
  const int total = steps[b];
  out->first = (int)((long long)total * part / n);
  out->count = (int)((long long)total * (part + 1) / n) - out->first;
  out->slot = found_s[2] + (out->kvh * a.tiles + tile) * n + part;
  fence_proxy_async_smem();  // the words in `steps` lie where the first copies go
  __syncthreads();
  return true;
}

// Whether a share's output is one that the tensor cores' products may have wrong.
template <typename T>
__device__ __forceinline__ bool unusual(float x) {
  return !(fabsf(x) <= 3.402823466e38f) || (sizeof(T) == 4 && fabsf(x) < kSmall && x != 0.0f);
}

// The block's share again, where some of its outputs are unusual(): the whole block calls
// this, with the warps' numerators, maxima and sums in sm, m_s and l_s.  Outputs that a NaN
// among the inputs makes NaN are to be that, so NaN is looked for first.  Other outputs mean
// that the share is done again: scores in 64 bits, weights and values in f32, straight from
// the pages, a token at a time (a warp takes every W-th).  Two passes, of which the first
// finds a row's maximum and the power of two at or above its sum, so that weights add up to
// 1 at most: whatever the values are, their numerators stay within f32.  An infinite value
// counts whole however small its weight is: only a score of -inf has one of 0.
// (16 x 8192 tokens x 2 heads of 256, with one NaN or one a page: 249 and 279 us for 47;
// twenty times that where everything is done again.)
// Queries are taken from the block's own parts of them: where the output goes over them,
// the first one has been stored.
template <typename T, int DP, int NR, typename Sh>
__device__ __noinline__ void plain_share(const PagedArgs &a, PagedShare me, int rows, int head0, float *sm,
                                         float (*m_s)[NR], float (*l_s)[NR]) {
  constexpr int kTok = Sh::kTok, W = Sh::W, PITCH = Sh::kEndPitch;
  __shared__ uint32_t nan_columns[32], nan_rows;  // outputs that are to be NaN: eight columns a word, or whole rows
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, col = lane * 8, D = a.head_dim;
  // (without a sign: a step past the last token may pass 2^31)
  const uint32_t first = (uint32_t)me.first * kTok + w, end = min((uint32_t)me.length, (uint32_t)(me.first + me.count) * kTok);
  const int32_t *table = a.table + me.b * a.table_pitch;
  // where the lane's columns of token t lie, in elements; -1: its page is none
  auto place = [&](uint32_t t) {
    const int row = (int)(t % (uint32_t)a.page_size), page = table[t / (uint32_t)a.page_size];
    return page >= 0 && page < a.pages ? page * a.page_pitch + row * a.row_pitch + me.kvh * a.head_pitch + col : -1ll;
  };
  auto load8 = [&](const void *base, long long at, float (&x)[8]) {
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = col < D ? static_cast<float>(static_cast<const T *>(base)[at + k]) : 0.0f;
  };
  // the lane's columns of row r's query: its parts are exact, but for an infinite one's rest
  auto query8 = [&](int r, float (&x)[8]) {
    const uint8_t *const qs = reinterpret_cast<const uint8_t *>(sm) + Sh::kOver;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      x[k] = 0.0f;
      for (int part = Sh::kQParts - 1; part >= 0 && col < DP; --part) {
        const float y = static_cast<float>(reinterpret_cast<const T *>(qs)[(part * NR + r) * Sh::kQPitch + col + k]);
        x[k] = part == 0 && isinf(y) ? y : x[k] + y;
      }
    }
  };
  auto score = [&](const float (&q)[8], const float (&k)[8]) {
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < 8; ++i) s = fma((double)q[i], (double)k[i], s);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return (float)(s * (double)a.scale_log2);
  };
  // row r's maximum over the warps, and sum over that
  auto sum_of = [&](int r, float *top) {
    float sum = 0.0f;
    *top = -INFINITY;
    for (int x = 0; x < W; ++x) *top = fmaxf(*top, m_s[x][r]);
    for (int x = 0; x < W; ++x) sum += l_s[x][r] * (m_s[x][r] == -INFINITY ? 0.0f : pow2(m_s[x][r] - *top));
    return sum;
  };
  // f(r, d, o, sum) for two columns of each row, as the warps' results have them; the top and sum of each row
  auto meet = [&](auto f, auto end_of_row) {
    for (int r = w; r < rows; r += W) {
      float top;
      const float sum = sum_of(r, &top), inv = sum != 0.0f ? 1.0f / sum : 0.0f;
      for (int d = lane * 2; d < D; d += 64) {
        float2 o = make_float2(0.0f, 0.0f);
        for (int x = 0; x < W; ++x) {
          const float g = m_s[x][r] == -INFINITY ? 0.0f : pow2(m_s[x][r] - top) * inv;
          const float2 v = *reinterpret_cast<const float2 *>(sm + (x * NR + r) * PITCH + d);
          o.x = fmaf(v.x, g, o.x);
          o.y = fmaf(v.y, g, o.y);
        }
        f(r, d, o, sum);
      }
      end_of_row(r, top, sum);
    }
  };
  if (w == 0) nan_columns[lane] = 0;
  if (threadIdx.x == 0) nan_rows = 0;
  __syncthreads();
  uint32_t bits = 0, keys = 0;
#pragma unroll 4
  for (uint32_t t = first; t < end; t += W) {
    const long long at = place(t);
    if (at < 0) continue;
    float k8[8], v8[8];
    load8(a.k, at, k8);
    load8(a.v, at, v8);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      keys |= isnan(k8[k]);
      bits |= (uint32_t)isnan(v8[k]) << k;
    }
  }
  if (__any_sync(0xffffffffu, keys)) bits = 0xff;  // a score of NaN is the whole row
  if (bits) atomicOr(nan_columns + lane, bits);
  for (int r = w; r < rows; r += W) {
    float q[8];
    query8(r, q);
    bool none = false;
#pragma unroll
    for (int k = 0; k < 8; ++k) none |= isnan(q[k]);
    if (__any_sync(0xffffffffu, none) && lane == 0) atomicOr(&nan_rows, 1u << r);
  }
  __syncthreads();
  bool again = false;
  auto doubtful = [&](float x, int r, int d) {
    return unusual<T>(x) && !(isnan(x) && ((nan_columns[d >> 3] >> (d & 7) | nan_rows >> r) & 1));
  };
  meet([&](int r, int d, float2 o, float) { again |= doubtful(o.x, r, d) | doubtful(o.y, r, d + 1); }, [](int, float, float) {});
  if (!__syncthreads_or(again)) return;
  for (int r = 0; r < rows; ++r) {
    float q[8], x[8], m = -INFINITY, l = 0.0f;
    query8(r, q);
    for (uint32_t t = first; t < end; t += W) {
      const long long at = place(t);
      if (at < 0) continue;
      load8(a.k, at, x);
      const float y = score(q, x);
      if (y == -INFINITY) continue;
      if (y > m) {
        l = m == -INFINITY ? l : l * pow2(m - y);
        m = y;
      }
      l += pow2(y - m);
    }
    if (lane == 0) {
      m_s[w][r] = m;
      l_s[w][r] = l;
    }
  }
  __syncthreads();
  float my_l = 0.0f, my_base = -INFINITY;  // of row `lane`
  for (int r = 0; r < rows; ++r) {
    float q[8], x[8], acc[8], l = 0.0f, top;
    const float sum = sum_of(r, &top), base = sum == 0.0f ? 0.0f : top + ceilf(log2f(sum));
    query8(r, q);
#pragma unroll
    for (int k = 0; k < 8; ++k) acc[k] = 0.0f;
    for (uint32_t t = first; t < end; t += W) {
      const long long at = place(t);
      if (at < 0) continue;
      load8(a.k, at, x);
      const float y = score(q, x), p = pow2(y - base);
      load8(a.v, at, x);
      l += p;
#pragma unroll
      for (int k = 0; k < 8; ++k) acc[k] = isinf(x[k]) && y > -INFINITY ? acc[k] + x[k] : fmaf(p, x[k], acc[k]);
    }
    if (col < D) {
#pragma unroll
      for (int k = 0; k < 8; ++k) sm[(w * NR + r) * PITCH + col + k] = acc[k];
    }
    if (lane == r) {
      my_l = l;
      if (sum != 0.0f) my_base = base;
    }
  }
  __syncthreads();
  if (lane < rows) {
    m_s[w][lane] = my_base;
    l_s[w][lane] = my_l;
  }
  __syncthreads();
  meet([&](int r, int d, float2 o, float sum) { keep_out(a, me, NR, r, head0 + r, d, o, sum); },
       [&](int r, float top, float sum) {
         if (me.parts > 1 && lane == 0) a.part_ml[(size_t)me.slot * NR + r] = make_float2(top, sum);
       });
}

// The join of an item's shares for the thread's columns again, where infinite outputs of
// shares whose weights are nothing beside another's made NaN: as in plain_share(),
// infinities count whole.
template <int NR>
__device__ __noinline__ void plain_join(const PagedArgs &a, PagedShare me, int rows, int head0) {
  const int D = a.head_dim, slot0 = me.slot - me.part;
  for (int i = threadIdx.x; i < rows * D / 4; i += blockDim.x) {
    const int row = i / (D / 4), col = (i - row * (D / 4)) * 4;
    const float2 *ml = a.part_ml + (size_t)slot0 * NR + row;
    const float *part = a.part + ((size_t)slot0 * NR + row) * D + col;
    float top = -INFINITY, sum = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f}, gate[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int x = 0; x < me.parts; ++x) top = fmaxf(top, __ldcg(ml + (size_t)x * NR).x);
    auto weight = [&](float2 y) { return y.y * (y.x == -INFINITY ? 0.0f : pow2(y.x - top)); };
    for (int x = 0; x < me.parts; ++x) sum += weight(__ldcg(ml + (size_t)x * NR));
    for (int x = 0; x < me.parts; ++x) {
      const float2 y = __ldcg(ml + (size_t)x * NR);
      const float4 v = __ldcg(reinterpret_cast<const float4 *>(part + (size_t)x * NR * D));
      const float u[4] = {v.x, v.y, v.z, v.w}, f = weight(y) / sum;
#pragma unroll
      for (int k = 0; k < 4; ++k) o[k] = isinf(u[k]) && y.y > 0.0f ? o[k] + u[k] : fmaf(u[k], f, o[k]);
    }
    if (a.gate) {
      const float *g = a.gate + (size_t)me.b * a.gate_pitch + (size_t)(head0 + row) * a.gate_head + col;
#pragma unroll
      for (int k = 0; k < 4; ++k) gate[k] = g[k];
    }
    store_out<4>(a, me.b, head0 + row, col, o, sum, gate);
  }
}

template <typename T, int DP, int NR, bool ONCE, bool QF>
__global__ void __launch_bounds__((PagedShape<T, DP, NR, ONCE, QF>::kThreads), (PagedShape<T, DP, NR, ONCE, QF>::kBlocks))
    paged_attn_kernel(const __grid_constant__ PagedArgs a, const __grid_constant__ CUtensorMap k_map,
                      const __grid_constant__ CUtensorMap v_map) {
  using Sh = PagedShape<T, DP, NR, ONCE, QF>;
  constexpr int W = Sh::W, kTok = Sh::kTok, kParts = Sh::kParts, kNT = NR / 8;
  extern __shared__ uint8_t raw_sm[];
  uint8_t *const ring = raw_sm + (-smem_u32(raw_sm) & 1023);  // the swizzle goes by the address
  float *const sm = reinterpret_cast<float *>(ring);          // at the end: the warps' results
  __shared__ uint64_t full[W][kParts];
  __shared__ int abort_s;
  __shared__ PagedShare me_s;
  __shared__ float m_s[W][NR], l_s[W][NR];
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, D = a.head_dim;
  if (lane == 0) {
    for (int i = 0; i < kParts; ++i) mbar_init(&full[w][i], 1);
    if (w == 0) abort_s = 0;
    fence_barrier_init();
  }
  __syncwarp();
  if (tid == 0) {
    prefetch_tensormap(&k_map);
    prefetch_tensormap(&v_map);
  }
  // A warp takes steps w, w + W, ... of the share; part 2 i of its ring's sequence is
  // its i-th step's keys, part 2 i + 1 its values.  A step has copies one below
  // another: lane i's begins at token i * box.
  PagedShare me;
  int count = 0;
  const int32_t *table = a.table;
  const int boxes = kTok / a.box;
  auto token0 = [&](int i) { return (me.first + w + i * W) * kTok; };
  auto look_up = [&](int i) {  // the page of the lane's copy in step i
    const int t = token0(i) + lane * a.box;
    return lane < boxes && i < count && t < me.length ? __ldcg(table + t / a.page_size) : -1;
  };
  auto begin = [&]() {
    count = w < me.count ? (me.count - w + W - 1) / W : 0;
    table = a.table + me.b * a.table_pitch;
  };
  // Up to 32 sessions: the share is found while the kernel ahead still runs.  What
  // that one may have changed since is read again behind it, past L1, and the share
  // found anew if a length is another.
  const bool few = a.batch <= 32;
  uint32_t empty = 0;  // sessions without tokens, of up to 32
  bool any = false;
  int early = 0, page = -1, next_page = -1;
  if (few) {
    early = lane < a.batch ? __ldcg(a.lengths + lane) : 0;
    any = paged_share_few(a, early, &empty, &me);
    if (any) {
      begin();
      const int t = token0(0) + lane * a.box;
      if (lane < boxes && t < me.length) asm volatile("prefetch.global.L2 [%0];" ::"l"(table + t / a.page_size));
    }
  }
  pdl_enter();
  if (few) {
    const int length = lane < a.batch ? __ldcg(a.lengths + lane) : 0;
    if (any) next_page = look_up(0);
    if (blockIdx.x == 0 && w == 0 && (length < 0 || length > (long long)a.max_pages * a.page_size) && a.error)
      atomicCAS(a.error, 0, kErrLength);
    if (__any_sync(0xffffffffu, length != early)) {
      any = paged_share_few(a, length, &empty, &me);
      if (any) {
        begin();
        next_page = look_up(0);
      }
    }
  } else if ((any = paged_share<kTok, W>(a, reinterpret_cast<int *>(ring), &me))) {
    begin();
    next_page = look_up(0);
  }
  // sessions without tokens: block b writes session b's zeros, and those a grid on
  for (int b = blockIdx.x; b < a.batch; b += gridDim.x)
    if (few ? empty >> b & 1 : a.lengths[b] <= 0 || a.lengths[b] > (long long)a.max_pages * a.page_size)
      for (int i = tid; i < a.q_heads * D / 2; i += Sh::kThreads) {
        const float zeros[2] = {0.0f, 0.0f};
        store_out<2>(a, b, 0, 2 * i, zeros, 0.0f, zeros);
      }
  if (!any) return;
  uint8_t *const mine = ring + (size_t)w * kParts * Sh::kPart;
  bool wrong = false;  // a page outside the pool was met
  auto fetch = [&](int j) {
    const int i = j >> 1, t = token0(i) + lane * a.box;
    if (!(j & 1)) {
      page = next_page;
      next_page = look_up(i + 1);
    }
    const bool there = lane < boxes && t < me.length, good = there && page >= 0 && page < a.pages;
    const uint32_t all = __ballot_sync(0xffffffffu, good);
    if (__any_sync(0xffffffffu, there && !good)) {
      wrong = true;
      if (lane == 0 && a.error) atomicCAS(a.error, 0, kErrPage);
    }
    uint64_t *bar = &full[w][j % kParts];
    if (lane == 0) mbar_arrive_expect_tx(bar, __popc(all) * a.box * 128 * Sh::kBoxes);
    __syncwarp();
    if (good) {
      uint8_t *to = mine + (j % kParts) * Sh::kPart + lane * a.box * 128;
      const CUtensorMap *map = j & 1 ? &v_map : &k_map;
      const int row = t % a.page_size;
      if (a.whole) {
        tma_load_5d(to, map, 0, row, 0, me.kvh, page, bar);
      } else {
#pragma unroll
        for (int x = 0; x < Sh::kBoxes; ++x)
          tma_load_5d(to + x * (kTok * 128), map, x * Sh::kCols, row, 0, me.kvh, page, bar);
      }
    }
    __syncwarp();
  };
  // The queries, eight columns a lane and a row a warp, are asked for ahead of the
  // first copies (behind them, which take the memory a few microseconds, they came
  // 3 us later); the gates come to L2 meanwhile.
  int head0 = me.kvh * a.group + me.tile * NR, rows = min(NR, a.group - me.tile * NR);
  if (tid == 0) me_s = me;
  constexpr int kMine = (NR + W - 1) / W;
  float x[kMine][8];
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    const int r = w + i * W, col = lane * 8;
    load_q8(a, me.b, head0 + r, col, r < rows && col < D, x[i]);
    if (a.gate && r < rows && col < D)
      asm volatile("prefetch.global.L2 [%0];" ::"l"(a.gate + (size_t)me.b * a.gate_pitch + (size_t)(head0 + r) * a.gate_head + col));
  }
  for (int j = 0; j < min(2 * count, kParts); ++j) fetch(j);

  bool ok = true;
  auto wait = [&](int j) {
    if (ok) ok = mbar_wait(&full[w][j % kParts], (j / kParts) & 1, &abort_s);
    if (!ok) {  // (a wait that ran out: the results are void, but the loop ends)
      *(volatile int *)&abort_s = 1;
      if (a.error) atomicCAS(a.error, 0, kErrPagedWait);
    }
    __syncwarp();
    ok = __all_sync(0xffffffffu, ok);
  };
  int asked = min(2 * count, kParts);
  auto done = [&](int j) {  // part j is read: its place takes a later one
    __syncwarp();
    if (ok && j + kParts < 2 * count) {
      fetch(j + kParts);
      asked = j + kParts + 1;
    }
  };
  // whether token t of the session is one, with its page in the pool
  auto token_there = [&](int t) {
    if (t >= me.length) return false;
    if (!wrong) return true;
    const int p = table[t / a.page_size];
    return p >= 0 && p < a.pages;
  };
  // tokens of a step that are not there: their values become zeros, since a
  // weight of 0 does not hide a NaN
  auto clear_values = [&](uint8_t *part, int t0) {
    for (int r = 0; r < kTok; ++r) {
      if (token_there(t0 + r)) continue;
      for (int i = lane; i < Sh::kBoxes * 8; i += 32)
        *reinterpret_cast<uint4 *>(part + (i >> 3) * (kTok * 128) + r * 128 + (i & 7) * 16) = make_uint4(0, 0, 0, 0);
    }
    fence_proxy_async_smem();  // (the next copy into it comes behind these)
    __syncwarp();
  };

  // copies still in flight land before their memory is used otherwise
  auto finish = [&]() {
    if (!ok)
      for (int j = max(0, asked - kParts); j < asked; ++j) {
        int never = 0;
        mbar_wait(&full[w][j % kParts], (j / kParts) & 1, &never);
      }
    __syncthreads();
  };

  if constexpr (Sh::kHalf) {
    const int g = lane >> 2, c = lane & 3, own = token_at<T>(g);
    __nv_bfloat16 *const qs = reinterpret_cast<__nv_bfloat16 *>(ring + Sh::kOver);  // [part][row][kQPitch]
    // (of three parts the last is read where it is used, beside the registers of the others; a
    // sum of the first parts is kept apart from what the others add, which it would cut)
    constexpr int kPieces = DP / 32, kMT = DP / 16, kChains = !QF ? 2 : NR == 8 ? 4 : 3, kQP = Sh::kQParts, kPP = Sh::kPParts;
    constexpr int kHeld = Sh::kQShared ? 0 : kQP < 2 ? kQP : 2;
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int r = w + i * W, col = lane * 8;
      if (col < DP && r < NR) {
        uint32_t u[4][kQP];
#pragma unroll
        for (int k = 0; k < 4; ++k) split_bf16x2(x[i][2 * k], x[i][2 * k + 1], u[k]);
#pragma unroll
        for (int part = 0; part < kQP; ++part)
          *reinterpret_cast<uint4 *>(qs + (part * NR + r) * Sh::kQPitch + col) =
              make_uint4(u[0][part], u[1][part], u[2][part], u[3][part]);
      }
    }
    __syncthreads();
    // Q operands of piece p: row g (+ 8 i)'s dimensions 32 p + 8 c + [0, 8)
    auto stored = [&](int part, int i, int p) {
      return *reinterpret_cast<const uint4 *>(qs + (part * NR + g + 8 * i) * Sh::kQPitch + 32 * p + 8 * c);
    };
    uint4 qr[kHeld ? kHeld * kNT * kPieces : 1];
#pragma unroll
    for (int part = 0; part < kHeld; ++part)
#pragma unroll
      for (int i = 0; i < kNT; ++i)
#pragma unroll
        for (int p = 0; p < kPieces; ++p) qr[(part * kNT + i) * kPieces + p] = stored(part, i, p);
    auto query = [&](int part, int i, int p) {
      return part < kHeld ? qr[part < kHeld ? (part * kNT + i) * kPieces + p : 0] : stored(part, i, p);
    };
    float acc[kMT][kNT][4], m[kNT][2], l[kNT][2];
#pragma unroll
    for (int i = 0; i < kNT; ++i) {
#pragma unroll
      for (int k = 0; k < kMT; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[k][i][e] = 0.0f;
      m[i][0] = m[i][1] = -INFINITY;
      l[i][0] = l[i][1] = 0.0f;
    }
    for (int at = 0; at < count; ++at) {
      const int t0 = token0(at);
      const uint8_t *kst = mine + (2 * at) % kParts * Sh::kPart;
      wait(2 * at);
      // scores of 16 tokens: s[i][.][2 h + e] token own + 8 h, row 2 c + e + 8 i, in sums
      // that do not wait for one another
      float s[kNT][kChains][4];
#pragma unroll
      for (int i = 0; i < kNT; ++i)
#pragma unroll
        for (int u = 0; u < kChains; ++u)
#pragma unroll
          for (int k = 0; k < 4; ++k) s[i][u][k] = 0.0f;
#pragma unroll
      for (int p = 0; p < kPieces; ++p) {
        const uint8_t *row = kst + (p >> 1) * (kTok * 128) + own * 128 + ((4 * (p & 1) + c) ^ own) * 16;
        const uint4 u = *reinterpret_cast<const uint4 *>(row), v = *reinterpret_cast<const uint4 *>(row + 8 * 128);
#pragma unroll
        for (int i = 0; i < kNT; ++i) {
#pragma unroll
          for (int part = 0; part < kQP; ++part) {
            const uint4 q = query(part, i, p);
            mma_bf16(s[i][part ? (kChains == 4 ? 2 : kChains - 1) : 0], u.x, v.x, u.y, v.y, q.x, q.y);
            mma_bf16(s[i][part ? kChains - 1 : 1], u.z, v.z, u.w, v.w, q.z, q.w);
          }
        }
      }
      done(2 * at);
      const bool open = t0 + kTok > me.length || wrong;
      float y[kNT][2][2];  // scores: row, token
      bool grow = false;
#pragma unroll
      for (int i = 0; i < kNT; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float x = s[i][0][2 * h + e] + s[i][1][2 * h + e];
            if (kChains == 3) x += s[i][kChains - 1][2 * h + e];
            if (kChains == 4) x += s[i][kChains - 2][2 * h + e] + s[i][kChains - 1][2 * h + e];
            y[i][e][h] = x * a.scale_log2;
            if (open && !token_there(t0 + own + 8 * h)) y[i][e][h] = -INFINITY;
          }
          grow |= fmaxf(y[i][e][0], y[i][e][1]) > m[i][e] + kLag;
        }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int i = 0; i < kNT; ++i)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float mn = fmaxf(m[i][e], fmaxf(y[i][e][0], y[i][e][1]));
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
            const float old = m[i][e] == -INFINITY ? 0.0f : pow2(m[i][e] - mn);
            l[i][e] *= old;
            m[i][e] = mn;
#pragma unroll
            for (int k = 0; k < kMT; ++k) {
              acc[k][i][e] *= old;
              acc[k][i][2 + e] *= old;
            }
          }
      }
      uint32_t pp[kPP][kNT][2];
#pragma unroll
      for (int i = 0; i < kNT; ++i) {
        const float base[2] = {m[i][0] == -INFINITY ? 0.0f : -m[i][0], m[i][1] == -INFINITY ? 0.0f : -m[i][1]};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float p0 = pow2(y[i][0][h] + base[0]), p1 = pow2(y[i][1][h] + base[1]);
          l[i][0] += p0;
          l[i][1] += p1;
          uint32_t u[kPP];
          split_bf16x2(p0, p1, u);
#pragma unroll
          for (int part = 0; part < kPP; ++part) pp[part][i][h] = transposed(u[part]);
        }
      }
      uint8_t *vst = mine + (2 * at + 1) % kParts * Sh::kPart;
      wait(2 * at + 1);
      if (open) clear_values(vst, t0);
      const int vrow = token_at<T>(lane & 7), half = (lane >> 3) & 1;
      const uint32_t v0 = smem_u32(vst) + (vrow + 8 * (lane >> 4)) * 128;
#pragma unroll
      for (int k = 0; k < kMT; ++k) {
        uint32_t x[4];
        load_transposed(x, v0 + (k >> 2) * (kTok * 128) + ((2 * (k & 3) + half) ^ vrow) * 16);
#pragma unroll
        for (int i = 0; i < kNT; ++i)
#pragma unroll
          for (int part = 0; part < kPP; ++part)
            mma_bf16(acc[k][i], x[0], x[1], x[2], x[3], pp[part][i][0], pp[part][i][1]);
      }
      done(2 * at + 1);
    }
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
    finish();
    float *mine_f = sm + (size_t)w * NR * Sh::kEndPitch;
#pragma unroll
    for (int k = 0; k < kMT; ++k)
#pragma unroll
      for (int i = 0; i < kNT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          mine_f[(8 * i + 2 * c + (e & 1)) * Sh::kEndPitch + 16 * k + g + 8 * (e >> 1)] = acc[k][i][e];
  } else {
    // A product of parts is three of the tensor cores' (two parts each, without the small
    // ones'), and takes the time that the copies do (8 x 18432 tokens of 256: with f32
    // fma 111 us, so 102, 5.9 TB/s).  Of the scores' operand rows 8 to 15 are zeros.
    // S = Q K^T with the rows as M (eight of sixteen), eight tokens as N; O^T = V^T P^T
    // with the dimensions as M, the rows as N: S's result is P^T's operand as it lies.
    const int g = lane >> 2, c = lane & 3, own = token_at<T>(g);
    uint32_t *const qs = reinterpret_cast<uint32_t *>(ring + Sh::kOver);  // [high, low][row][kQPitch]
    constexpr int kBoxes = Sh::kBoxes, kMT = DP / 16;
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int r = w + i * W, col = lane * 8;
      if (col < DP && r < NR) {
        uint32_t hi[8], lo[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) split_nearest(x[i][k], &hi[k], &lo[k]);
#pragma unroll
        for (int k = 0; k < 8; k += 4) {
          *reinterpret_cast<uint4 *>(qs + r * Sh::kQPitch + col + k) = make_uint4(hi[k], hi[k + 1], hi[k + 2], hi[k + 3]);
          *reinterpret_cast<uint4 *>(qs + (NR + r) * Sh::kQPitch + col + k) = make_uint4(lo[k], lo[k + 1], lo[k + 2], lo[k + 3]);
        }
      }
    }
    __syncthreads();
    float acc[kMT][4], m = -INFINITY, l = 0.0f;  // the row g's maximum and sum
#pragma unroll
    for (int k = 0; k < kMT; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[k][e] = 0.0f;
    const int v0 = token_at<T>(2 * c), v1 = token_at<T>(2 * c + 1);
    for (int at = 0; at < count; ++at) {
      const int t0 = token0(at);
      const uint8_t *kst = mine + (2 * at) % kParts * Sh::kPart;
      wait(2 * at);
      // scores of eight tokens, row g: s[.][0] token v0, s[.][1] v1, in sums that do not
      // wait for one another
      float s[4][4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int k = 0; k < 4; ++k) s[u][k] = 0.0f;
      // (whole, twelve warps at their own places in it wait for its instructions: 8 x 2304
      // tokens 25.3 us, so 24.3; of four pieces 64 x 600 48.6, so 46.4)
#pragma unroll 8
      for (int p = 0; p < 2 * kBoxes; ++p) {  // sixteen dimensions: the lane's four, 16 p + 4 c
        const uint4 x = *reinterpret_cast<const uint4 *>(kst + (p >> 1) * (kTok * 128) + own * 128 +
                                                         ((4 * (p & 1) + c) ^ own) * 16);
        const uint4 qh = *reinterpret_cast<const uint4 *>(qs + g * Sh::kQPitch + 16 * p + 4 * c);
        const uint4 ql = *reinterpret_cast<const uint4 *>(qs + (NR + g) * Sh::kQPitch + 16 * p + 4 * c);
        uint4 hi, lo;
        split_cut(x.x, &hi.x, &lo.x);
        split_cut(x.y, &hi.y, &lo.y);
        split_cut(x.z, &hi.z, &lo.z);
        split_cut(x.w, &hi.w, &lo.w);
        mma_tf32(s[0], qh.x, 0, qh.y, 0, hi.x, hi.y);
        mma_tf32(s[1], qh.z, 0, qh.w, 0, hi.z, hi.w);
        mma_tf32(s[2], qh.x, 0, qh.y, 0, lo.x, lo.y);
        mma_tf32(s[3], ql.x, 0, ql.y, 0, hi.x, hi.y);
        mma_tf32(s[2], qh.z, 0, qh.w, 0, lo.z, lo.w);
        mma_tf32(s[3], ql.z, 0, ql.w, 0, hi.z, hi.w);
      }
      done(2 * at);
      const bool open = t0 + kTok > me.length || wrong;
      float y[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        y[u] = ((s[0][u] + s[1][u]) + (s[2][u] + s[3][u])) * a.scale_log2;
        if (open && !token_there(t0 + (u ? v1 : v0))) y[u] = -INFINITY;
      }
      if (__any_sync(0xffffffffu, fmaxf(y[0], y[1]) > m + kLag)) {
        float mn = fmaxf(m, fmaxf(y[0], y[1]));
        mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, 1));
        mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, 2));
        const float old = m == -INFINITY ? 0.0f : pow2(m - mn);
        l *= old;
        m = mn;
        const float f0 = __shfl_sync(0xffffffffu, old, 8 * c), f1 = __shfl_sync(0xffffffffu, old, 8 * c + 4);  // rows 2 c, 2 c + 1
#pragma unroll
        for (int k = 0; k < kMT; ++k) {
          acc[k][0] *= f0;
          acc[k][1] *= f1;
          acc[k][2] *= f0;
          acc[k][3] *= f1;
        }
      }
      const float base = m == -INFINITY ? 0.0f : -m;
      const float p0 = pow2(y[0] + base), p1 = pow2(y[1] + base);
      l += p0 + p1;
      uint32_t ph[2], pl[2];
      split_nearest(p0, &ph[0], &pl[0]);
      split_nearest(p1, &ph[1], &pl[1]);
      uint8_t *vst = mine + (2 * at + 1) % kParts * Sh::kPart;
      wait(2 * at + 1);
      if (open) clear_values(vst, t0);
      // (the sums over the steps are kept apart: the tensor cores' own cut what they add)
#pragma unroll
      for (int x = 0; x < kBoxes; ++x) {  // 32 dimensions: the lane's four, 32 x + 4 g
        const uint8_t *box = vst + x * (kTok * 128);
        const uint4 u = *reinterpret_cast<const uint4 *>(box + v0 * 128 + (g ^ v0) * 16);
        const uint4 v = *reinterpret_cast<const uint4 *>(box + v1 * 128 + (g ^ v1) * 16);
        uint4 uh, ul, vh, vl;
        split_cut(u.x, &uh.x, &ul.x);
        split_cut(u.y, &uh.y, &ul.y);
        split_cut(u.z, &uh.z, &ul.z);
        split_cut(u.w, &uh.w, &ul.w);
        split_cut(v.x, &vh.x, &vl.x);
        split_cut(v.y, &vh.y, &vl.y);
        split_cut(v.z, &vh.z, &vl.z);
        split_cut(v.w, &vh.w, &vl.w);
        float d[4] = {0.0f, 0.0f, 0.0f, 0.0f}, e[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        mma_tf32(d, uh.x, uh.y, vh.x, vh.y, ph[0], ph[1]);
        mma_tf32(e, uh.z, uh.w, vh.z, vh.w, ph[0], ph[1]);
        mma_tf32(d, ul.x, ul.y, vl.x, vl.y, ph[0], ph[1]);
        mma_tf32(e, ul.z, ul.w, vl.z, vl.w, ph[0], ph[1]);
        mma_tf32(d, uh.x, uh.y, vh.x, vh.y, pl[0], pl[1]);
        mma_tf32(e, uh.z, uh.w, vh.z, vh.w, pl[0], pl[1]);
        add2(acc[2 * x][0], acc[2 * x][1], d[0], d[1]);
        add2(acc[2 * x][2], acc[2 * x][3], d[2], d[3]);
        add2(acc[2 * x + 1][0], acc[2 * x + 1][1], e[0], e[1]);
        add2(acc[2 * x + 1][2], acc[2 * x + 1][3], e[2], e[3]);
      }
      done(2 * at + 1);
    }
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    if (c == 0) {
      m_s[w][g] = m;
      l_s[w][g] = l;
    }
    finish();
    float *mine_f = sm + (size_t)w * NR * Sh::kEndPitch;
    // tile 2 x + h of 16 dimensions: row i < 8 of it is dimension 32 x + 4 i + 2 h, row i + 8 the one after it
#pragma unroll
    for (int k = 0; k < kMT; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        mine_f[(2 * c + (e & 1)) * Sh::kEndPitch + 32 * (k >> 1) + 4 * g + 2 * (k & 1) + (e >> 1)] = acc[k][e];
  }
  __syncthreads();
  // (what only the end needs of it takes no registers meanwhile: 3 x 100003 tokens 112 us, so 103)
  me = me_s;
  head0 = me.kvh * a.group + me.tile * NR;
  rows = min(NR, a.group - me.tile * NR);
  // The warps' results meet: maxima, then sums over one maximum in warp order; weights
  // over their sum, so that no sum passes the values it is of.
  bool again = false;
  for (int r = w; r < rows; r += W) {
    float top = -INFINITY, f[W], sum = 0.0f;
#pragma unroll
    for (int x = 0; x < W; ++x) top = fmaxf(top, m_s[x][r]);
#pragma unroll
    for (int x = 0; x < W; ++x) {
      f[x] = m_s[x][r] == -INFINITY ? 0.0f : pow2(m_s[x][r] - top);
      sum = fmaf(l_s[x][r], f[x], sum);
    }
    const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
#pragma unroll
    for (int x = 0; x < W; ++x) f[x] *= inv;
    for (int d = lane * 2; d < D; d += 64) {
      float2 o = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int x = 0; x < W; ++x) {
        const float2 v = *reinterpret_cast<const float2 *>(sm + ((size_t)x * NR + r) * Sh::kEndPitch + d);
        o.x = fmaf(v.x, f[x], o.x);
        o.y = fmaf(v.y, f[x], o.y);
      }
      again |= unusual<T>(o.x) | unusual<T>(o.y);
      keep_out(a, me, NR, r, head0 + r, d, o, sum);
    }
    if (me.parts > 1 && lane == 0) a.part_ml[(size_t)me.slot * NR + r] = make_float2(top, sum);
  }
  if (__syncthreads_or(again)) plain_share<T, DP, NR, Sh>(a, me, rows, head0, sm, m_s, l_s);
  if (me.parts == 1) return;
  // The shares of an item meet in the block that finds all of them there: each says
  // so by its flag and then looks at the others', so that the last one does find
  // them (another that does as well writes the same).  What a flag says is the
  // call's own number, whatever lay there before; they are cleared for the next use.
  // (A kernel behind this one for it: 16 x 1000 tokens 17.9 us, so 16.0.)
  __shared__ int last_s;
  const int slot0 = me.slot - me.part;
  __syncthreads();
  if (w == 0) {
    if (lane == 0) {
      __threadfence();
      *reinterpret_cast<volatile unsigned long long *>(a.flags + me.slot) = a.token;
      __threadfence();
    }
    __syncwarp();
    bool all = true;
    for (int i = lane; i < me.parts; i += 32)
      all &= *reinterpret_cast<volatile unsigned long long *>(a.flags + slot0 + i) == a.token;
    all = __all_sync(0xffffffffu, all);
    __threadfence();
    if (lane == 0) last_s = all;
  }
  __syncthreads();
  if (!last_s) return;
  const float2 *ml = a.part_ml + (size_t)slot0 * NR;
  const float *part = a.part + (size_t)slot0 * NR * D;
  // (a thread's fours of columns, of a few shares at once, are asked for together, and the gates with them)
  constexpr int kItems = (NR * DP / 4 + Sh::kThreads - 1) / Sh::kThreads, kAtOnce = kItems >= 8 ? 2 : kItems >= 4 ? 4 : kItems == 2 ? 10 : 12;
  float4 o[kItems], gate[kItems];
  float top[kItems], sum[kItems];
  int row[kItems], col[kItems];
#pragma unroll
  for (int j = 0; j < kItems; ++j) {
    const int i = tid + j * Sh::kThreads;
    row[j] = i / (D / 4);
    col[j] = (i - row[j] * (D / 4)) * 4;
    o[j] = gate[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    top[j] = -INFINITY;
    sum[j] = 0.0f;
    if (a.gate && row[j] < rows) {
      const float *g = a.gate + (size_t)me.b * a.gate_pitch + (size_t)(head0 + row[j]) * a.gate_head + col[j];
      gate[j] = make_float4(g[0], g[1], g[2], g[3]);
    }
  }
#pragma unroll 1
  for (int x0 = 0; x0 < me.parts; x0 += kAtOnce) {
    float4 v[kItems][kAtOnce];
    float2 y[kItems][kAtOnce];
#pragma unroll
    for (int j = 0; j < kItems; ++j)
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        const bool in = x0 + k < me.parts && row[j] < rows;
        const size_t at = (size_t)(x0 + k) * NR + row[j];
        v[j][k] = in ? __ldcg(reinterpret_cast<const float4 *>(part + at * D + col[j])) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        y[j][k] = in ? __ldcg(ml + at) : make_float2(-INFINITY, 0.0f);
      }
#pragma unroll
    for (int j = 0; j < kItems; ++j) {
      float high = top[j];
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) high = fmaxf(high, y[j][k].x);
      float old = top[j] == -INFINITY ? 0.0f : sum[j] * pow2(top[j] - high);
      top[j] = high;
      sum[j] = old;
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        y[j][k].y *= y[j][k].x == -INFINITY ? 0.0f : pow2(y[j][k].x - high);
        sum[j] += y[j][k].y;
      }
      const float inv = sum[j] != 0.0f ? 1.0f / sum[j] : 0.0f;
      old *= inv;
      o[j].x *= old;
      o[j].y *= old;
      o[j].z *= old;
      o[j].w *= old;
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        const float f = y[j][k].y * inv;
        o[j].x = fmaf(v[j][k].x, f, o[j].x);
        o[j].y = fmaf(v[j][k].y, f, o[j].y);
        o[j].z = fmaf(v[j][k].z, f, o[j].z);
        o[j].w = fmaf(v[j][k].w, f, o[j].w);
      }
    }
  }
  bool odd = false;
#pragma unroll
  for (int j = 0; j < kItems; ++j) {
    if (row[j] >= rows) continue;
    odd |= isnan(o[j].x + o[j].y + o[j].z + o[j].w);
    const float x[4] = {o[j].x, o[j].y, o[j].z, o[j].w}, g[4] = {gate[j].x, gate[j].y, gate[j].z, gate[j].w};
    store_out<4>(a, me.b, head0 + row[j], col[j], x, sum[j], g);
  }
  if (odd) plain_join<NR>(a, me, rows, head0);
  for (int i = tid; i < me.parts; i += Sh::kThreads) a.flags[slot0 + i] = 0;
}

// How a call is cut.
struct Plan {
  int rows, tiles, slots, waves, least;
  size_t blocks, parts;
};

template <typename T, int DP, int NR, bool ONCE, bool QF>
int run_shape(const PagedArgs &a, const Plan &p, const CUtensorMap &k_map, const CUtensorMap &v_map, cudaStream_t s) {
  using Sh = PagedShape<T, DP, NR, ONCE, QF>;
  {
    static std::mutex mu;
    static std::vector<int> done;
    int dev = 0;
    FPB_CUDA_TRY(cudaGetDevice(&dev));
    std::lock_guard<std::mutex> lock(mu);
    if (std::find(done.begin(), done.end(), dev) == done.end()) {
      FPB_CUDA_TRY(cudaFuncSetAttribute(paged_attn_kernel<T, DP, NR, ONCE, QF>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        (int)Sh::smem));
      done.push_back(dev);
    }
  }
  cudaError_t e = launch_pdl(paged_attn_kernel<T, DP, NR, ONCE, QF>, (unsigned)p.blocks, Sh::kThreads, Sh::smem, s, a, k_map,
                             v_map);
  if (e != cudaSuccess) return cuda_fail(e, "paged_attn_kernel");
  FPB_LAUNCH_CHECK("paged_attn_kernel");
  return FPB_OK;
}

template <typename T, int DP, int NR>
int run_paged(const PagedArgs &a, const Plan &p, const CUtensorMap &k_map, const CUtensorMap &v_map, cudaStream_t s) {
  if constexpr (sizeof(T) == 2)
    if (a.q_bf16)
      return p.waves ? run_shape<T, DP, NR, false, false>(a, p, k_map, v_map, s)
                     : run_shape<T, DP, NR, true, false>(a, p, k_map, v_map, s);
  return p.waves ? run_shape<T, DP, NR, false, true>(a, p, k_map, v_map, s)
                 : run_shape<T, DP, NR, true, true>(a, p, k_map, v_map, s);
}

Plan plan_for(size_t batch, size_t q_heads, size_t kv_heads, size_t head_dim, bool f32) {
  Plan p{};
  const size_t group = q_heads / kv_heads;
  p.rows = group <= 8 || f32 ? 8 : 16;
  p.tiles = (int)((group + p.rows - 1) / p.rows);
  const size_t items = batch * kv_heads * p.tiles;
  // One wave, where every item has a block then.  Sessions of different lengths leave
  // some of those short; with heads of more than 128 that costs more than the blocks'
  // coming and going where more than half of the blocks can be (us for one wave and two:
  // 16 x 2000 tokens x 8 kv heads of 128, bf16, 27 and 35, 16 x 9000 92 and 117, 10 x
  // 9000 77 and 73; 50 x 2000 x 2 heads of 256 44 and 44, 66 x 9000 142 and 127).
  p.waves = (head_dim <= 128 ? items < (size_t)sm_count() : 2 * items <= (size_t)sm_count()) ? 0 : kPagedWaves;
  // (64 steps at least where blocks follow one another: of 24 20 x 5000 tokens x 8 heads
  // 89 us, so 76, 20 x 600 18 and 24; in one wave the SMs are empty otherwise: 1 x 777
  // tokens with 32 15.5 us, with 8 10.2.  Shares of two waves: of four 200 ragged sessions
  // take 276 us, so 255, of one as long.)
  p.least = p.waves ? 64 : 8;
  p.slots = sm_count() * blocks_of(head_dim > 128 ? 256 : 128, !p.waves);
  // an item that is cut has more than S steps, so at most twice its steps / S shares
  p.blocks = p.waves ? (size_t)p.waves * p.slots + items : p.slots;
  p.parts = p.waves ? (size_t)2 * p.waves * p.slots : p.slots;
  return p;
}

// A number that no other call has: mixed, so that nothing that happens to lie in a
// workspace is likely to be it (the mixing is that of splitmix64).
unsigned long long call_number() {
  static std::atomic<unsigned long long> calls{(unsigned long long)std::chrono::steady_clock::now().time_since_epoch().count()};
  unsigned long long x = calls.fetch_add(0x9e3779b97f4a7c15ull);
  x = (x ^ x >> 30) * 0xbf58476d1ce4e5b9ull;
  x = (x ^ x >> 27) * 0x94d049bb133111ebull;
  x ^= x >> 31;
  return x ? x : 1;
}

size_t workspace_for(const Plan &p, size_t head_dim) {
  return p.parts * (p.rows * (head_dim + 2) * sizeof(float) + sizeof(unsigned long long));
}

}  // namespace
}  // namespace fpb

using namespace fpb;

extern "C" size_t fpb_paged_attn_workspace_bytes(size_t batch, size_t q_heads, size_t kv_heads, size_t head_dim) {
  if (batch == 0 || kv_heads == 0 || q_heads == 0 || q_heads % kv_heads) return 16;
  const size_t a = workspace_for(plan_for(batch, q_heads, kv_heads, head_dim, false), head_dim),
               b = workspace_for(plan_for(batch, q_heads, kv_heads, head_dim, true), head_dim);
  return std::max(a, b);
}

extern "C" int fpb_paged_attn(const void *q, int q_dtype, size_t q_pitch, size_t q_head_pitch, const void *k_pages,
                              const void *v_pages, int page_dtype, size_t pages, size_t page_size, size_t page_pitch,
                              size_t row_pitch, size_t head_pitch, const int32_t *table, size_t table_pitch,
                              size_t max_pages, const int32_t *lengths, const float *gate, size_t gate_pitch,
                              size_t gate_head_pitch, size_t batch, size_t q_heads, size_t kv_heads, size_t head_dim,
                              float scale, void *workspace, size_t workspace_bytes, void *out, int out_dtype,
                              void *stream) {
  if (!q || !table || !lengths || !workspace || !out)
    return fail(FPB_ERR_INVALID_ARGUMENT, "fpb_paged_attn: null pointer");
  if ((q_dtype != FPB_F32 && q_dtype != FPB_BF16) || (out_dtype != FPB_F32 && out_dtype != FPB_BF16))
    return fail(FPB_ERR_INVALID_ARGUMENT, "fpb_paged_attn: dtype");
  if (int st = check_pages("fpb_paged_attn", k_pages, v_pages, page_dtype, pages, page_size, page_pitch, row_pitch,
                           head_pitch, kv_heads, head_dim))
    return st;
  if (batch == 0 || batch > (size_t)kPagedMaxBatch || q_heads == 0 || q_heads % kv_heads || q_heads > 65535 || max_pages == 0 ||
      max_pages > 0x7fffffffu / page_size || table_pitch < max_pages || table_pitch >> 38)
    return fail(FPB_ERR_SHAPE, "fpb_paged_attn: batch %zu (at most %d), heads %zu / %zu, tables of %zu pages (pitch "
                "%zu)", batch, kPagedMaxBatch, q_heads, kv_heads, max_pages, table_pitch);
  if (q_head_pitch < head_dim || (gate && gate_head_pitch < head_dim) || !std::isfinite(scale))
    return fail(FPB_ERR_SHAPE, "fpb_paged_attn: pitches or scale");
  if (!aligned_to(workspace, 16) || !aligned_to(out, 16) || !aligned_to(q, q_dtype == FPB_F32 ? 4 : 2) ||
      !aligned_to(gate, 4))
    return fail(FPB_ERR_INVALID_ARGUMENT, "fpb_paged_attn: alignment (workspace and out: 16 bytes)");
  const size_t need = fpb_paged_attn_workspace_bytes(batch, q_heads, kv_heads, head_dim);
  if (workspace_bytes < need)
    return fail(FPB_ERR_WORKSPACE, "fpb_paged_attn: workspace %zu < %zu bytes", workspace_bytes, need);
  {
    // The head vectors x [batch rows of pitch, q_heads of head] against the output, which is one piece
    const char *o = static_cast<const char *>(out), *end = o + batch * q_heads * head_dim * (out_dtype == FPB_F32 ? 4 : 2);
    auto meets = [&](const void *x, size_t pitch, size_t head, size_t el) {
      const char *v = static_cast<const char *>(x);
      if (!x || v >= end || v + ((batch - 1) * pitch + (q_heads - 1) * head + head_dim) * el <= o) return false;
      for (size_t b = 0; b < batch; ++b)
        for (size_t h = 0; h < q_heads; ++h)
          if (const char *u = v + (b * pitch + h * head) * el; u < end && u + head_dim * el > o) return true;
      return false;
    };
    const bool in_place = q == out && q_dtype == out_dtype && (q_heads == 1 || q_head_pitch == head_dim) &&
                          (batch == 1 || q_pitch == q_heads * head_dim);
    if ((!in_place && meets(q, q_pitch, q_head_pitch, q_dtype == FPB_F32 ? 4 : 2)) ||
        meets(gate, gate_pitch, gate_head_pitch, 4))
      return fail(FPB_ERR_INVALID_ARGUMENT, "fpb_paged_attn: out overlaps the gate, or q otherwise than in its place");
  }
  const bool f32 = page_dtype == FPB_F32;
  Plan p = plan_for(batch, q_heads, kv_heads, head_dim, f32);
  {  // no more blocks than the tables' tokens can have shares
    const size_t tok = f32 ? 8 : 16, steps = (max_pages * page_size + tok - 1) / tok;
    p.blocks = std::min(p.blocks, batch * kv_heads * p.tiles * ((steps + p.least - 1) / p.least));
  }
  if (p.blocks > 0x7fffffff) return fail(FPB_ERR_SHAPE, "fpb_paged_attn: %zu blocks", p.blocks);
  PagedArgs a{};
  a.q = q;
  a.k = k_pages;
  a.v = v_pages;
  a.page_pitch = (long long)page_pitch;
  a.row_pitch = (long long)row_pitch;
  a.head_pitch = (long long)head_pitch;
  a.gate = gate;
  a.table = table;
  a.lengths = lengths;
  a.q_pitch = (long long)q_pitch;
  a.q_head = (long long)q_head_pitch;
  a.gate_pitch = (long long)gate_pitch;
  a.gate_head = (long long)gate_head_pitch;
  a.table_pitch = (long long)table_pitch;
  a.batch = (int)batch;
  a.q_heads = (int)q_heads;
  a.kv_heads = (int)kv_heads;
  a.group = (int)(q_heads / kv_heads);
  a.head_dim = (int)head_dim;
  a.max_pages = (int)max_pages;
  a.pages = (int)pages;
  a.page_size = (int)page_size;
  a.q_bf16 = q_dtype == FPB_BF16;
  a.q_vec = aligned_to(q, 16) && (q_pitch | q_head_pitch) * (a.q_bf16 ? 2 : 4) % 16 == 0;
  a.box = f32 ? 8 : 16;
  while (page_size % a.box) a.box /= 2;
  a.whole = head_dim % (f32 ? 32 : 64) == 0 && a.box == (f32 ? 8 : 16);
  a.tiles = p.tiles;
  a.tok = f32 ? 8 : 16;
  a.least = p.least;
  a.slots = p.slots;
  a.waves = p.waves;
  a.scale_log2 = (float)((double)scale * 1.4426950408889634);
  a.out = out;
  a.out_bf16 = out_dtype == FPB_BF16;
  a.part = static_cast<float *>(workspace);
  a.part_ml = reinterpret_cast<float2 *>(a.part + p.parts * p.rows * head_dim);
  a.flags = reinterpret_cast<unsigned long long *>(a.part_ml + p.parts * p.rows);
  a.token = call_number();
  a.error = device_error_ptr();
  CUtensorMap k_map, v_map;
  if (int st = encode_pages(&k_map, k_pages, !f32, head_dim, kv_heads, page_size, pages, head_pitch, row_pitch,
                            page_pitch, (uint32_t)a.box, a.whole ? (head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256) / (f32 ? 32 : 64) : 1))
    return st;
  if (int st = encode_pages(&v_map, v_pages, !f32, head_dim, kv_heads, page_size, pages, head_pitch, row_pitch,
                            page_pitch, (uint32_t)a.box, a.whole ? (head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256) / (f32 ? 32 : 64) : 1))
    return st;
  cudaStream_t s = as_stream(stream);
  using bf = __nv_bfloat16;
  const bool few = p.rows == 8;
  int st;
  if (f32)
    st = head_dim <= 64    ? run_paged<float, 64, 8>(a, p, k_map, v_map, s)
         : head_dim <= 128 ? run_paged<float, 128, 8>(a, p, k_map, v_map, s)
                           : run_paged<float, 256, 8>(a, p, k_map, v_map, s);
  else
    st = head_dim <= 64    ? (few ? run_paged<bf, 64, 8>(a, p, k_map, v_map, s) : run_paged<bf, 64, 16>(a, p, k_map, v_map, s))
         : head_dim <= 128 ? (few ? run_paged<bf, 128, 8>(a, p, k_map, v_map, s) : run_paged<bf, 128, 16>(a, p, k_map, v_map, s))
                           : (few ? run_paged<bf, 256, 8>(a, p, k_map, v_map, s) : run_paged<bf, 256, 16>(a, p, k_map, v_map, s));
  return st;
}
