// The 8-bit key/value cache of speculative decoding: the step that norms,
// rotates and quantises new tokens into it, its read-back, and the move of an
// accepted path's rows.  The formats are in kv8.cuh.
#include <algorithm>
#include <cmath>

#include "kv8.cuh"

namespace fpb {
namespace {

constexpr int kAppendThreads = 128, kMaxHalf = 128, kMaxSpan = 2;

struct AppendArgs {
  const void *q, *k, *v;
  long long q_pitch, q_head, k_pitch, v_pitch;  // elements
  const float *q_gamma, *k_gamma;
  const int32_t *positions, *parents;
  int rows, span, nodes, q_heads, kv_heads, head_dim, rotary_dim, max_seq, vec;
  float inv_d, eps;
  void *q_out;
  int q_out_bf16;
  uint8_t *k_codes, *v_codes, *k_exp, *v_exp;
  int *error;
  uint64_t turn[kMaxHalf];  // theta^(-i / half) / (2 pi) of a turn, in units of 2^-64
};

// Eight consecutive elements as they lie; their f32 values.
template <typename T>
struct Eight {
  uint4 w[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T *p, bool vec) {
    if (vec) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = __ldg(reinterpret_cast<const uint4 *>(p) + i);
    } else {
      uint32_t *o = reinterpret_cast<uint32_t *>(w);
      if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = __float_as_uint(p[i]);
      } else {
        const uint16_t *h = reinterpret_cast<const uint16_t *>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = h[2 * i] | (uint32_t)h[2 * i + 1] << 16;
      }
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ void values(float (&x)[8]) const {
    const uint32_t *o = reinterpret_cast<const uint32_t *>(w);
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(o[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(o[i] << 16);
        x[2 * i + 1] = __uint_as_float(o[i] & 0xffff0000u);
      }
    }
  }
};

// Two values -> two e4m3 codes (RNE, satfinite; NaN stays NaN), a in the low byte.
__device__ __forceinline__ uint32_t e4m3x2(float a, float b) {
  uint16_t out;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(out) : "f"(b), "f"(a));
  return out;
}

// Some tokens' heads: block (x, part) takes the `span` rows from x * span on
// (row b * nodes + n: a token) and of their heads every gridDim.y-th group, LG
// lanes a head vector, two pieces of eight elements a lane (LG * 16 >= head_dim).
// Where the rotated dimensions' halves come in eights, a lane's second piece
// holds the partners of its first.
//  norm    x * rsqrt(mean x^2 + eps) * gamma, f32
//  rotate  dimensions i and i + half by (position + depth) * theta^(-i/half).
//          The turn is taken as a 64-bit fraction, an exact product of whole
//          numbers, and reduced before it is rounded to f32: an f32 product
//          is off by position * 2^-24 radians, 0.002 at position 32768.
//          The token's cosines and sines are made once for its heads.
//  write   q' as given, k' and v as codes and exponents at row position + n
// A decode step is bound by latency (loads of the positions, then sines: 3.5 us
// for 8 x 1 x 20 heads x 256), a prompt by instructions and their latency: 2 x
// 4096 x 48 heads x 128, bf16, takes 48 us for 185 MB (3.9 TB/s).  Sixteen
// elements a lane, not eight: a vector's sums, addresses and index take as many
// instructions for either (71 us), and partners in one lane need no shuffles.
// Blocks of four warps, seven an SM (of eight warps 56 us; eight an SM 50, fewer
// than seven 49).
template <typename T, int LG>
__global__ void __launch_bounds__(kAppendThreads, 7) kv8_append_kernel(const __grid_constant__ AppendArgs a) {
  pdl_enter();
  __shared__ float2 turn_s[kMaxSpan][kMaxHalf];  // cosine, sine
  __shared__ float xs[kAppendThreads / LG][LG * 16];
  __shared__ int depth_s[kMaxSpan], pos_s[kMaxSpan];
  __shared__ size_t to_s[kMaxSpan];  // the rows' places in the cache, in rows
  const int tid = threadIdx.x, lane = tid % LG, item = tid / LG;
  constexpr int kItems = kAppendThreads / LG;
  const int row0 = blockIdx.x * a.span, span = min(a.span, a.rows - row0);
  const int D = a.head_dim, heads = a.q_heads + 2 * a.kv_heads, half = a.rotary_dim / 2;
  const int turning = half % 8 == 0 ? half / 8 : 0;  // lanes whose pieces are partners
  const bool turns = lane < turning;
  const int c0 = turns ? 8 * lane : 16 * lane, col[2] = {c0, turns ? c0 + half : c0 + 8};  // (16 turning = 2 half)
  // a head's elements are asked for one head ahead, the first before the sines
  Eight<T> raw[2];
  auto ask = [&](int rl, int h) {
    raw[0].zero();
    raw[1].zero();
    if (rl >= span || c0 >= D) return;
    const size_t row = row0 + rl;
    const bool is_q = h < a.q_heads, is_k = !is_q && h < a.q_heads + a.kv_heads;
    const T *src = is_q   ? static_cast<const T *>(a.q) + row * a.q_pitch + (size_t)h * a.q_head
                   : is_k ? static_cast<const T *>(a.k) + row * a.k_pitch + (size_t)(h - a.q_heads) * D
                          : static_cast<const T *>(a.v) + row * a.v_pitch + (size_t)(h - a.q_heads - a.kv_heads) * D;
    raw[0].load(src + col[0], a.vec);
    raw[1].load(src + col[1], a.vec);
  };
  int rl = 0, h = blockIdx.y * kItems + item;
  while (h >= heads) {
    h -= heads;
    ++rl;
  }
  ask(rl, h);
  if (tid < span) {
    const int row = row0 + tid, b = row / a.nodes, n = row - b * a.nodes, pos = a.positions[b];
    bool bad = false;
    int depth = tree_depth(a.parents ? a.parents + (size_t)b * a.nodes : nullptr, n, &bad);
    if (bad && a.error) atomicCAS(a.error, 0, kErrParent);
    if (depth >= 0 && (pos < 0 || pos >= a.max_seq - n)) {
      if (a.error) atomicCAS(a.error, 0, kErrPosition);
      depth = -1;
    }
    depth_s[tid] = depth;
    pos_s[tid] = pos;
    to_s[tid] = (size_t)b * a.max_seq + pos + n;
  }
  __syncthreads();
  if (half > 0) {
    for (int i = tid; i < span * half; i += kAppendThreads) {
      const int r = i / half, c = i - r * half;
      const uint64_t turn = a.turn[c] * (uint64_t)(uint32_t)(pos_s[r] + max(depth_s[r], 0));
      const float t = (float)(int32_t)(uint32_t)(turn >> 32) * 0x1p-31f;  // half turns, in [-1, 1]
      float2 cs;
      sincospif(t, &cs.y, &cs.x);
      turn_s[r][c] = cs;
    }
    __syncthreads();
  }
  int turned = -1;  // the row whose cosines and sines the lane holds: they serve all of its heads
  float cs[8], sn[8];
  // (the loop ends together for the whole block: its warps' lanes shuffle)
  const int total = span * heads;
  for (int i0 = blockIdx.y * kItems; i0 < total; i0 += gridDim.y * kItems) {
    const int depth = rl < span ? depth_s[rl] : -1;
    const size_t row = row0 + rl;
    const bool live = rl < span && c0 < D;
    const bool is_q = h < a.q_heads, is_k = !is_q && h < a.q_heads + a.kv_heads;
    const int kvh = is_q ? 0 : h - a.q_heads - (is_k ? 0 : a.kv_heads), here = h, at = min(rl, span - 1);
    float x[2][8];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if (depth < 0) raw[j].zero();  // rows of nodes that are not there: zeros
      raw[j].values(x[j]);
    }
    h += gridDim.y * kItems;
    while (h >= heads) {
      h -= heads;
      ++rl;
    }
    ask(rl, h);
    const float *gamma = is_q ? a.q_gamma : is_k ? a.k_gamma : nullptr;
    float ss = 0.0f;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = fmaf(x[j][i], x[j][i], ss);
#pragma unroll
    for (int o = LG / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (gamma && live && depth >= 0) {  // (a norm of zeros with eps 0 would be NaN)
      const float scale = __frsqrt_rn(fmaf(ss, a.inv_d, a.eps));
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float4 g0 = __ldg(reinterpret_cast<const float4 *>(gamma + col[j])),
                     g1 = __ldg(reinterpret_cast<const float4 *>(gamma + col[j]) + 1);
        const float g[8] = {g0.x, g0.y, g0.z, g0.w, g1.x, g1.y, g1.z, g1.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) x[j][i] = x[j][i] * scale * g[i];
      }
    }
    if (turning) {
      if (turns && (is_q || is_k)) {
        if (at != turned) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            cs[i] = turn_s[at][c0 + i].x;
            sn[i] = turn_s[at][c0 + i].y;
          }
          turned = at;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float u = x[0][i], v = x[1][i];
          x[0][i] = fmaf(-v, sn[i], u * cs[i]);
          x[1][i] = fmaf(u, sn[i], v * cs[i]);
        }
      }
    } else if (half > 0) {
      const bool rotates = live && (is_q || is_k) && c0 < 2 * half;
      if (rotates) {
#pragma unroll
        for (int i = 0; i < 16; ++i) xs[item][c0 + i] = x[i >> 3][i & 7];
      }
      __syncwarp();
      if (rotates) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int c = c0 + i;
          float &v = x[i >> 3][i & 7];
          if (c < half)
            v = v * turn_s[at][c].x - xs[item][c + half] * turn_s[at][c].y;
          else if (c < 2 * half)
            v = v * turn_s[at][c - half].x + xs[item][c - half] * turn_s[at][c - half].y;
        }
      }
      __syncwarp();
    }
    float amax = 0.0f;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(x[j][i]));
#pragma unroll
    for (int o = LG / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if (!live) continue;
    if (is_q) {
      const size_t head = (row * a.q_heads + here) * D;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const size_t o = head + col[j];
        const float *y = x[j];
        if (a.q_out_bf16) {
          *reinterpret_cast<uint4 *>(static_cast<__nv_bfloat16 *>(a.q_out) + o) =
              make_uint4(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]), pack_bf16x2(y[4], y[5]),
                         pack_bf16x2(y[6], y[7]));
        } else {
          float4 *dst = reinterpret_cast<float4 *>(static_cast<float *>(a.q_out) + o);
          dst[0] = make_float4(y[0], y[1], y[2], y[3]);
          dst[1] = make_float4(y[4], y[5], y[6], y[7]);
        }
      }
    } else if (depth >= 0) {
      const int e = kv8_exponent(amax);
      const float inv = pow2i(-e);
      const size_t vec = to_s[at] * a.kv_heads + kvh;
      uint8_t *codes = (is_k ? a.k_codes : a.v_codes) + vec * D;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float *y = x[j];
        uint2 w;
        w.x = e4m3x2(y[0] * inv, y[1] * inv) | e4m3x2(y[2] * inv, y[3] * inv) << 16;
        w.y = e4m3x2(y[4] * inv, y[5] * inv) | e4m3x2(y[6] * inv, y[7] * inv) << 16;
        *reinterpret_cast<uint2 *>(codes + col[j]) = w;
      }
      if (lane == 0) (is_k ? a.k_exp : a.v_exp)[vec] = (uint8_t)(e + 127);
    }
  }
}

// Sixteen codes a thread; a session's rows are one contiguous range, K and V
// in grid z.  Bound by its bytes: one code read, one value written (8 x 8192 x 2
// heads x 256 to bf16: 33 us, 6.1 TB/s).
template <bool BF16>
__global__ void __launch_bounds__(256) kv8_read_kernel(const uint8_t *k_codes, const uint8_t *v_codes,
                                                       const uint8_t *k_exp, const uint8_t *v_exp,
                                                       const int32_t *begins, int begin, int count, int kv_heads,
                                                       int head_dim, int max_seq, void *k_out, void *v_out,
                                                       int *error) {
  pdl_enter();
  const int b = blockIdx.y;
  const bool is_v = blockIdx.z != 0;
  const int per = head_dim / 16;
  const uint32_t pieces = (uint32_t)count * (uint32_t)kv_heads * (uint32_t)per;
  const int t0 = begins ? begins[b] : begin;
  const bool bad = t0 < 0 || t0 > max_seq - count;
  if (bad && threadIdx.x == 0 && blockIdx.x == 0 && error) atomicCAS(error, 0, kErrPosition);
  const size_t first = ((size_t)b * max_seq + (bad ? 0 : t0)) * kv_heads;
  const uint4 *codes = reinterpret_cast<const uint4 *>(is_v ? v_codes : k_codes) + first * per;
  const uint8_t *exps = (is_v ? v_exp : k_exp) + first;
  void *out = is_v ? v_out : k_out;
  const size_t base = (size_t)b * pieces;
  for (uint32_t i = blockIdx.x * blockDim.x + threadIdx.x; i < pieces; i += gridDim.x * blockDim.x) {
    uint4 c = make_uint4(0, 0, 0, 0);
    float f = 0.0f;
    if (!bad) {
      c = __ldg(codes + i);
      f = kv8_factor(exps[i / (uint32_t)per]);
    }
    const uint32_t w[4] = {c.x, c.y, c.z, c.w};
    float x[16];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t h = e4m3x2_to_f16x2((uint16_t)(w[j / 2] >> (16 * (j & 1))));
      const float2 p = __half22float2(*reinterpret_cast<const __half2 *>(&h));
      x[2 * j] = p.x * f;
      x[2 * j + 1] = p.y * f;
    }
    if (BF16) {
      uint4 *dst = reinterpret_cast<uint4 *>(out) + (base + i) * 2;
#pragma unroll
      for (int j = 0; j < 2; ++j)
        dst[j] = make_uint4(pack_bf16x2(x[8 * j], x[8 * j + 1]), pack_bf16x2(x[8 * j + 2], x[8 * j + 3]),
                            pack_bf16x2(x[8 * j + 4], x[8 * j + 5]), pack_bf16x2(x[8 * j + 6], x[8 * j + 7]));
    } else {
      float4 *dst = reinterpret_cast<float4 *>(out) + (base + i) * 4;
#pragma unroll
      for (int j = 0; j < 4; ++j) dst[j] = make_float4(x[4 * j], x[4 * j + 1], x[4 * j + 2], x[4 * j + 3]);
    }
  }
}

// Row position + d becomes a copy of row position + path[d].  Ancestors come
// before their descendants, so path[d] >= d and the sources ascend: a thread
// that moves its own sixteen columns row by row, d ascending, never writes
// what it still has to read, and no two threads share a byte.  Bound by latency:
// a row is read once the one before has been written (16 sessions x 2 heads x
// 256: three rows moved 3.0 us, five 4.2).
__global__ void __launch_bounds__(256) kv8_keep_kernel(uint8_t *k_codes, uint8_t *v_codes, uint8_t *k_exp,
                                                       uint8_t *v_exp, const int32_t *positions, const int32_t *path,
                                                       int nodes, int kv_heads, int head_dim, int max_seq,
                                                       int *error) {
  pdl_enter();
  const int b = blockIdx.y, per = head_dim / 16, wide = kv_heads * per;
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= 2 * (wide + kv_heads)) return;
  const int pos = positions[b];
  const int32_t *p = path + (size_t)b * nodes;
  const size_t row0 = (size_t)b * max_seq + pos;
  int before = -1;
  for (int d = 0; d < nodes; ++d) {
    const int s = p[d];
    if (s < 0) break;
    if (s <= before || s >= nodes || pos < 0 || pos >= max_seq - s) {  // not an ascending path inside the cache
      if (error) atomicCAS(error, 0, s <= before || s >= nodes ? kErrParent : kErrPosition);
      return;
    }
    before = s;
    if (s == d) continue;
    const int j = i % (wide + kv_heads);
    const bool is_v = i >= wide + kv_heads;
    if (j < wide) {
      uint4 *c = reinterpret_cast<uint4 *>(is_v ? v_codes : k_codes);
      c[(row0 + d) * wide + j] = c[(row0 + s) * wide + j];
    } else {
      uint8_t *e = is_v ? v_exp : k_exp;
      e[(row0 + d) * kv_heads + j - wide] = e[(row0 + s) * kv_heads + j - wide];
    }
  }
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int check_cache(const char *name, const void *kc, const void *vc, const void *ke, const void *ve, size_t batch,
                size_t kv_heads, size_t head_dim, size_t max_seq) {
  if (!kc || !vc || !ke || !ve) return fail(FPB_ERR_INVALID_ARGUMENT, "%s: null cache", name);
  if (!aligned16(kc) || !aligned16(vc)) return fail(FPB_ERR_INVALID_ARGUMENT, "%s: codes not 16-byte aligned", name);
  if (batch == 0 || batch > 65535 || kv_heads == 0 || kv_heads > 4096 || head_dim == 0 || head_dim > 256 ||
      head_dim % 16 || max_seq == 0 || max_seq > (1u << 30))
    return fail(FPB_ERR_SHAPE, "%s: cache shape (batch %zu, max_seq %zu, kv_heads %zu, head_dim %zu: a multiple of "
                "16 up to 256)", name, batch, max_seq, kv_heads, head_dim);
  return FPB_OK;
}

template <typename T>
int run_append(AppendArgs a, size_t rows, cudaStream_t s) {
  const int lanes = a.head_dim / 16;
  const int lg = lanes <= 4 ? 4 : lanes <= 8 ? 8 : 16;
  const int heads = a.q_heads + 2 * a.kv_heads, per = kAppendThreads / lg;
  // Few rows: one group of heads a block (8 rows of 20 heads x 256 3.4 us, with
  // all heads in a block 4.8).  Beyond eight blocks an SM a block takes all of a
  // row's heads (1024 rows of 48 heads x 128 10.6 us, with a group a block 12),
  // and of two rows from sixteen rows an SM on: the rows' positions and sines are
  // then made for both at once (8192 rows 49 us, with one row a block 53, with
  // four 52; 2048 rows 17 with one, 18 with two).
  const int parts = (heads + per - 1) / per;
  a.span = rows >= (size_t)sm_count() * 16 ? kMaxSpan : 1;
  const size_t want = std::min<size_t>(parts, std::max<size_t>(1, (size_t)sm_count() * 8 / rows));
  const dim3 grid((unsigned)((rows + a.span - 1) / a.span), (unsigned)want);
  cudaError_t e = lg == 4   ? launch_pdl(kv8_append_kernel<T, 4>, grid, kAppendThreads, 0, s, a)
                  : lg == 8 ? launch_pdl(kv8_append_kernel<T, 8>, grid, kAppendThreads, 0, s, a)
                            : launch_pdl(kv8_append_kernel<T, 16>, grid, kAppendThreads, 0, s, a);
  if (e != cudaSuccess) return cuda_fail(e, "kv8_append_kernel");
  FPB_LAUNCH_CHECK("kv8_append_kernel");
  return FPB_OK;
}

}  // namespace
}  // namespace fpb

using namespace fpb;

extern "C" int fpb_kv8_append(const void *q, size_t q_pitch, size_t q_head_pitch, const void *k, size_t k_pitch,
                              const void *v, size_t v_pitch, int dtype, const float *q_gamma, const float *k_gamma,
                              const int32_t *positions, const int32_t *parents, size_t batch, size_t nodes,
                              size_t q_heads, size_t kv_heads, size_t head_dim, size_t rotary_dim, float theta,
                              float eps, size_t max_seq, void *q_out, int q_out_dtype, uint8_t *k_codes,
                              uint8_t *v_codes, uint8_t *k_exp, uint8_t *v_exp, void *stream) {
  if (!k || !v || !positions || (q_heads != 0) != (q != nullptr) || (q != nullptr) != (q_out != nullptr))
    return fail(FPB_ERR_INVALID_ARGUMENT, "fpb_kv8_append: null pointer (q, q_out and q_heads go together)");
  if (int st = check_cache("fpb_kv8_append", k_codes, v_codes, k_exp, v_exp, batch, kv_heads, head_dim, max_seq))
    return st;
  if ((dtype != FPB_F32 && dtype != FPB_BF16) || (q && q_out_dtype != FPB_F32 && q_out_dtype != FPB_BF16))
    return fail(FPB_ERR_INVALID_ARGUMENT, "fpb_kv8_append: dtype");
  if (nodes == 0 || nodes > max_seq || batch * nodes > 0x7fffffff || q_heads > 65535 ||
      (parents && nodes > (size_t)kTreeMaxNodes))
    return fail(FPB_ERR_SHAPE, "fpb_kv8_append: nodes %zu (a tree has at most %d)", nodes, kTreeMaxNodes);
  if (rotary_dim % 2 || rotary_dim > head_dim || (rotary_dim && !(theta >= 1.0f && std::isfinite(theta))))
    return fail(FPB_ERR_SHAPE, "fpb_kv8_append: rotary_dim %zu (even, at most head_dim), theta %g (at least 1)",
                rotary_dim, (double)theta);
  if (k_pitch < kv_heads * head_dim || v_pitch < kv_heads * head_dim || (q && q_head_pitch < head_dim))
    return fail(FPB_ERR_SHAPE, "fpb_kv8_append: pitch");
  const size_t el = dtype == FPB_F32 ? 4 : 2;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) % el ||
      (q && !aligned16(q_out)) || (q_gamma && !aligned16(q_gamma)) || (k_gamma && !aligned16(k_gamma)))
    return fail(FPB_ERR_INVALID_ARGUMENT, "fpb_kv8_append: alignment (q_out and the gammas: 16 bytes)");
  AppendArgs a{};
  a.q = q;
  a.k = k;
  a.v = v;
  a.q_pitch = (long long)q_pitch;
  a.q_head = (long long)q_head_pitch;
  a.k_pitch = (long long)k_pitch;
  a.v_pitch = (long long)v_pitch;
  a.q_gamma = q_gamma;
  a.k_gamma = k_gamma;
  a.positions = positions;
  a.parents = parents;
  a.rows = (int)(batch * nodes);
  a.nodes = (int)nodes;
  a.q_heads = (int)q_heads;
  a.kv_heads = (int)kv_heads;
  a.head_dim = (int)head_dim;
  a.rotary_dim = (int)rotary_dim;
  a.max_seq = (int)max_seq;
  a.vec = aligned16(q) && aligned16(k) && aligned16(v) && (q_pitch | q_head_pitch | k_pitch | v_pitch) * el % 16 == 0;
  a.inv_d = 1.0f / (float)head_dim;
  a.eps = eps;
  a.q_out = q_out;
  a.q_out_bf16 = q_out_dtype == FPB_BF16;
  a.k_codes = k_codes;
  a.v_codes = v_codes;
  a.k_exp = k_exp;
  a.v_exp = v_exp;
  a.error = device_error_ptr();
  const int half = (int)rotary_dim / 2;
  // theta^(-i / half) by products of 64-bit mantissas: off by i * 2^-63 of itself at most
  const long double ratio = half ? powl((long double)theta, -1.0L / half) : 0.0L;
  long double turn = 0x1p64L / (2.0L * M_PIl);
  for (int i = 0; i < half; ++i, turn *= ratio) a.turn[i] = (uint64_t)turn;
  cudaStream_t s = as_stream(stream);
  return dtype == FPB_F32 ? run_append<float>(a, batch * nodes, s) : run_append<__nv_bfloat16>(a, batch * nodes, s);
}

extern "C" int fpb_kv8_read(const uint8_t *k_codes, const uint8_t *v_codes, const uint8_t *k_exp,
                            const uint8_t *v_exp, size_t batch, size_t max_seq, size_t kv_heads, size_t head_dim,
                            const int32_t *begins, size_t begin, size_t count, void *k_out, void *v_out,
                            int out_dtype, void *stream) {
  if (int st = check_cache("fpb_kv8_read", k_codes, v_codes, k_exp, v_exp, batch, kv_heads, head_dim, max_seq))
    return st;
  if (!k_out || !v_out || !aligned16(k_out) || !aligned16(v_out))
    return fail(FPB_ERR_INVALID_ARGUMENT, "fpb_kv8_read: outputs null or not 16-byte aligned");
  if (out_dtype != FPB_F32 && out_dtype != FPB_BF16) return fail(FPB_ERR_INVALID_ARGUMENT, "fpb_kv8_read: dtype");
  if (count == 0 || count > max_seq || (!begins && begin > max_seq - count) ||
      count * kv_heads * (head_dim / 16) > 0x7fffffff)
    return fail(FPB_ERR_SHAPE, "fpb_kv8_read: rows [%zu, +%zu) of %zu", begin, count, max_seq);
  const size_t pieces = count * kv_heads * (head_dim / 16);
  // (32 blocks an SM for the keys, as many for the values: 33 us at 8 x 8192 x 2 x
  // 256 to bf16; eight 41, no limit 34)
  const size_t most = std::max<size_t>(1, (size_t)sm_count() * 32 / batch);
  const dim3 grid((unsigned)std::min((pieces + 255) / 256, most), (unsigned)batch, 2);
  auto go = [&](auto kernel) {
    cudaError_t e = launch_pdl(kernel, grid, 256, 0, as_stream(stream), k_codes, v_codes, k_exp, v_exp, begins,
                               (int)begin, (int)count, (int)kv_heads, (int)head_dim, (int)max_seq, k_out, v_out,
                               device_error_ptr());
    if (e != cudaSuccess) return cuda_fail(e, "kv8_read_kernel");
    FPB_LAUNCH_CHECK("kv8_read_kernel");
    return (int)FPB_OK;
  };
  return out_dtype == FPB_BF16 ? go(kv8_read_kernel<true>) : go(kv8_read_kernel<false>);
}

extern "C" int fpb_kv8_keep(uint8_t *k_codes, uint8_t *v_codes, uint8_t *k_exp, uint8_t *v_exp, size_t batch,
                            size_t max_seq, size_t kv_heads, size_t head_dim, const int32_t *positions,
                            const int32_t *path, size_t nodes, void *stream) {
  if (int st = check_cache("fpb_kv8_keep", k_codes, v_codes, k_exp, v_exp, batch, kv_heads, head_dim, max_seq))
    return st;
  if (!positions || !path) return fail(FPB_ERR_INVALID_ARGUMENT, "fpb_kv8_keep: null pointer");
  if (nodes == 0 || nodes > max_seq) return fail(FPB_ERR_SHAPE, "fpb_kv8_keep: nodes %zu", nodes);
  const size_t threads = 2 * kv_heads * (head_dim / 16 + 1);
  cudaError_t e = launch_pdl(kv8_keep_kernel, dim3((unsigned)((threads + 255) / 256), (unsigned)batch), 256, 0,
                             as_stream(stream), k_codes, v_codes, k_exp, v_exp, positions, path, (int)nodes,
                             (int)kv_heads, (int)head_dim, (int)max_seq, device_error_ptr());
  if (e != cudaSuccess) return cuda_fail(e, "kv8_keep_kernel");
  FPB_LAUNCH_CHECK("kv8_keep_kernel");
  return FPB_OK;
}
