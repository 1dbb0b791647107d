// The next tokens from the logits: temperature, top-k, top-p and min-p of each
// row, from given exponential variates.
//
// With w_i = exp((l_i - max l) / T), a row's tokens are ordered by l, falling,
// ties by index.  Each filter keeps a first part of that order:
//   top-k   the first k
//   top-p   the shortest part whose weights reach p of what top-k kept
//   min-p   those with w >= min_p
// The token is argmax w_i / e_i over what is kept: with exponential e it is
// distributed as w.
//
// The bytes are a row's logits, and of its noise what is kept (0.6 MB each for 151936
// f32, under 1 us at the memory's rate for eight rows); what takes the time is one
// dependent step behind another, each of 1 to 4 us for passes over a slice, meetings of
// the cluster's CTAs and a sort: 8 rows of 151936 f32 take 4 us greedily, 10 with top-k
// (one list), 10 with every token in the race, 30 where top-p ends among tens of
// thousands of tokens.  A row's slices stay in shared memory between the steps.
#include <algorithm>
#include <cmath>
#include <mutex>
#include <vector>

#include "common.cuh"

namespace fpb {
namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kMaxSlice = 49152;  // logits of a CTA in shared memory, f32: 192 KB
constexpr int kMaxVocab = 8 * kMaxSlice;
constexpr size_t kPairSlice = 100 * 1024;  // bytes of a slice of which two fit an SM
constexpr int kBatch = 5;         // 16-byte loads a thread has under way (f32 logits: twice as many)
constexpr int kBins = 256;        // bins of a histogram
constexpr int kList = kThreads;   // tokens that one CTA orders
constexpr int kLargest = 128;     // groups of a cluster's threads, each with its largest logit
// What the k-th largest of the groups' 128 largest logits reaches is, with logits in
// no order, -128 ln(1 - k / 128) tokens: for 120 of them 355, for 96 177.
constexpr int kDirect = 120, kDirectSum = 96;
constexpr int kLists = 16;  // at most: one, and for each of two filters one and 32 / 8 finer ones

constexpr float kLowest = -3.402823466e38f;

struct SampleArgs {
  const void *logits;
  const float *temperature, *top_p, *min_p, *noise;
  const int32_t *top_k;
  long long logits_pitch, noise_pitch;  // elements between rows
  int vocab, slice, vec, noise_vec;     // vec: every slice begins on 16 bytes
  int32_t *tokens;
  float *logprobs;
};

struct Best {
  float v;
  int i;
};
__device__ __forceinline__ Best better(Best a, Best b) { return b.v > a.v || (b.v == a.v && b.i < a.i) ? b : a; }

__device__ __forceinline__ float pow2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float inverse(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Order of f32 values as that of whole numbers (the zeros are one), and back.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t u) {
  return __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u);
}

// [*lo, *hi], so ordered, without its ends that are no value of the type: -0 is none
// (0 is its equal), and bf16 values lie 2^16 apart.  (Some value lies within.)
template <typename T>
__device__ __forceinline__ void to_values(uint32_t *lo, uint32_t *hi) {
  constexpr uint32_t kNone = 0x7fffffffu;
  uint32_t l = *lo, h = *hi - (*hi == kNone);
  if (sizeof(T) == 2) {
    l = l > kNone ? (l + 0xffffu) & 0xffff0000u : l | 0xffffu;
    h = h > kNone ? h & 0xffff0000u : ((h + 1) & 0xffff0000u) - 1;
  }
  *lo = l + (l == kNone);
  *hi = h;
}

__device__ __forceinline__ uint32_t peer_address(const void *p, unsigned rank) {
  const uint32_t local = (uint32_t)__cvta_generic_to_shared(p);
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(rank));
  return remote;
}
__device__ __forceinline__ void peer_store(const void *p, unsigned rank, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(peer_address(p, rank)), "r"(v) : "memory");
}
__device__ __forceinline__ unsigned long long peer_load(const unsigned long long *p, unsigned rank) {
  unsigned long long v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(peer_address(p, rank)) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t peer_load(const uint32_t *p, unsigned rank) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(peer_address(p, rank)) : "memory");
  return v;
}
// cluster_sync() behind code that lanes may leave apart: its barrier counts whole warps.
__device__ __forceinline__ void meet() {
  __syncwarp();
  cluster_sync();
}
// *p += v in shared memory where `ok`.
__device__ __forceinline__ void add_if(bool ok, uint32_t *p, uint32_t v) {
  asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t@q red.shared.add.u32 [%0], %1;\n\t}" ::"r"(
                   (uint32_t)__cvta_generic_to_shared(p)),
               "r"(v), "r"((int)ok)
               : "memory");
}

template <typename V>
__device__ __forceinline__ V warp_total(V v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <int C>
struct Shared {
  unsigned long long list[kList];  // tokens to be ordered, (falling logit, index) as one number
  uint32_t hist[kBins];            // tokens, or their weights
  // what the CTAs tell one another; the halves alternate, so that one exchange's
  // reads may overlap the next one's stores
  uint32_t got[2][5][C];
  float maxima[kLargest], group[kLargest / C];  // the cluster's, the CTA's own
  double sums[kWarps];
  uint32_t counts[kWarps];
  Best best[kWarps];
  int border;  // where a histogram reaches its target: the bin, tokens or weights before it
  uint32_t n_before, n_in;  // n_in: tokens in it, or about as many
  double s_before;
  uint32_t listed[kLists];  // tokens in the list, each time anew
  float cut;
  int cut_index;
  uint32_t bound;
  float last_sum[kWarps], last_x[kWarps];
};

// The block's n (<= kList) numbers x, one a thread, in order: the tid-th, or ~0 past
// them.  All threads.  Bitonic, neighbours up to 16 apart through registers.
template <int C>
__device__ __noinline__ unsigned long long sorted(Shared<C> &sh, int n, unsigned long long x) {
  const int tid = threadIdx.x;
  int size = 32;
  while (size < n) size *= 2;
  for (int run = 2; run <= size; run *= 2) {
    const bool up = (tid & run) == 0;
    int step = run / 2;
    for (; step >= 32; step /= 2) {
      __syncthreads();
      if (tid < size) sh.list[tid] = x;
      __syncthreads();
      if (tid < size) {
        const unsigned long long y = sh.list[tid ^ step];
        x = (x < y) == (((tid & step) == 0) == up) ? x : y;
      }
    }
    if (tid < size)
      for (; step > 0; step /= 2) {
        const unsigned long long y = __shfl_xor_sync(0xffffffffu, x, step);
        x = (x < y) == (((tid & step) == 0) == up) ? x : y;
      }
  }
  __syncthreads();
  return x;
}

// Over the cluster's histograms: the first bin at which the running count (from n0
// on), or weight (from s0 on; bin i's numbers times `unit` and 2^-(i * step)),
// reaches the target (-1: none), with what lies before it.  Every CTA finds the
// same.  Two threads a bin, half of the CTAs' each.
template <int C>
__device__ __noinline__ int find_border(Shared<C> &sh, bool weigh, double target, uint32_t n0, double s0, double unit,
                                        float step) {
  static_assert(kThreads == 2 * kBins);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, bin = tid >> 1, from = C / 2 * (tid & 1);
  unsigned long long f = 0;
#pragma unroll
  for (int r = 0; r < C / 2; ++r) f += peer_load(&sh.hist[bin], from + r);
  f += __shfl_xor_sync(0xffffffffu, f, 1);
  uint32_t c = weigh ? 0 : (uint32_t)f;
  const bool one = (tid & 1) == 0;
  if (!one) c = 0;
  const double v = weigh && one ? (double)f * unit * (double)pow2(-(float)bin * step) : 0.0;
  // running count and sum over the bins
  uint32_t n = c;
  double run = v;
#pragma unroll
  for (int o = 2; o < 32; o <<= 1) {
    const uint32_t u = __shfl_up_sync(0xffffffffu, n, o);
    const double w = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o && one) {
      n += u;
      run += w;
    }
  }
  if (lane == 30) {
    sh.counts[warp] = n;
    sh.sums[warp] = run;
  }
  if (tid == 0) sh.border = kBins;
  __syncthreads();
  for (int i = 0; i < warp; ++i) {
    n0 += sh.counts[i];
    s0 += sh.sums[i];
  }
  if (one && f > 0 && (weigh ? s0 + run >= target : n0 + n >= (uint32_t)target)) atomicMin(&sh.border, bin);
  __syncthreads();
  const int border = sh.border;
  if (one && bin == border) {
    sh.n_before = n0 + n - c;
    sh.n_in = weigh ? (uint32_t)((double)f * unit) : c;  // (a weight relative to its bin's is about 1)
    sh.s_before = s0 + run - v;
  }
  __syncthreads();
  return border < kBins ? border : -1;
}

// A cluster of C CTAs a row: CTA `rank` keeps the vocabulary's slice [rank
// * slice, +slice) in shared memory, so that the row is read once.
//  1. The largest logit of each of 128 groups of threads goes to every CTA: the row's largest, and with the
//     k-th largest of the 128 (all of them for top-p alone) a bound that at least k
//     tokens reach.
//  2. What reaches it (a few times k tokens) goes to the first CTA's list, which is
//     put in order; there the filters are running sums.  top-p alone: if the list's
//     weights make p of the row's.
//  3. Where they do not, or k is larger, the border that a filter leaves is found by
//     a histogram over the cluster, and in the border's bin by the list, or by finer
//     histograms until the tokens there fit it, or are equal.  What is kept races
//     where it lies.
template <typename T, int C>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const __grid_constant__ SampleArgs a) {
  // every CTA of the cluster runs, before its shared memory is stored to
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  pdl_enter();
  extern __shared__ __align__(16) uint8_t xs_raw[];
  T *const xs = reinterpret_cast<T *>(xs_raw);  // the slice's logits
  __shared__ Shared<C> sh;
  const unsigned rank = cluster_ctarank();
  const int b = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int v0 = (int)rank * a.slice, len = max(0, min(a.vocab - v0, a.slice)), padded = (len + 3) / 4 * 4;
  const T *row = static_cast<const T *>(a.logits) + (size_t)b * a.logits_pitch + v0;
  const float *noise = a.noise + (size_t)b * a.noise_pitch + v0;
  const float t = a.temperature ? a.temperature[b] : 1.0f;
  const int k = a.top_k ? a.top_k[b] : 0;
  const float p = a.top_p ? a.top_p[b] : 1.0f, m = a.min_p ? a.min_p[b] : 0.0f;
  const bool greedy = !(t > 0.0f), by_k = k > 0 && k < a.vocab, by_p = p < 1.0f;
  const float least = m > 0.0f ? fminf(m, 1.0f) : 0.0f;
  const bool plain = !by_k && !by_p && least == 0.0f;
  const float temp = fminf(fmaxf(t, 1e-6f), 1e6f), per = 1.4426950408889634f / temp;
  auto want_noise = [&]() {  // all of the slice's, to L2
    if (a.noise_vec && tid == 0 && len >= 4)
      asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(noise), "r"(len / 4 * 16) : "memory");
  };
  if (!greedy && plain) want_noise();
  if (tid < kLists) sh.listed[tid] = 0;
  if (tid == 0) sh.bound = 0xffffffffu;

  auto get4 = [&](int i) {  // four of them
    if constexpr (sizeof(T) == 4) {
      return *reinterpret_cast<const float4 *>(xs + i);
    } else {
      const uint2 u = *reinterpret_cast<const uint2 *>(xs + i);
      return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                         __uint_as_float(u.y & 0xffff0000u));
    }
  };

  // The slice to shared memory, and its largest logit: the first of the first four
  // that hold one.
  Best top{-INFINITY, 0x7fffffff};
  {
    constexpr int N = 16 / sizeof(T), kLoads = sizeof(T) == 4 ? 2 * kBatch : kBatch;
    auto finite = [](float x) { return fabsf(x) <= 3.402823466e38f ? x : -INFINITY; };
    auto take = [&](float x0, float x1, float x2, float x3, int i) {
      const float4 y = make_float4(finite(x0), finite(x1), finite(x2), finite(x3));
      if constexpr (sizeof(T) == 4)
        *reinterpret_cast<float4 *>(xs + i) = y;
      else
        *reinterpret_cast<uint2 *>(xs + i) = make_uint2(pack_bf16x2(y.x, y.y), pack_bf16x2(y.z, y.w));
      const float most = fmaxf(fmaxf(y.x, y.y), fmaxf(y.z, y.w));
      if (most > top.v) top = Best{most, i};
    };
    const int whole = a.vec ? len / N * N : 0;
    for (int i0 = tid * N; i0 < whole; i0 += kLoads * kThreads * N) {
      uint4 v[kLoads];
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        const int i = i0 + j * kThreads * N;
        v[j] = i < whole ? __ldg(reinterpret_cast<const uint4 *>(row + i)) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        const int i = i0 + j * kThreads * N;
        if (i >= whole) break;
        if constexpr (N == 4) {
          take(__uint_as_float(v[j].x), __uint_as_float(v[j].y), __uint_as_float(v[j].z), __uint_as_float(v[j].w), i);
        } else {
          take(__uint_as_float(v[j].x << 16), __uint_as_float(v[j].x & 0xffff0000u), __uint_as_float(v[j].y << 16),
               __uint_as_float(v[j].y & 0xffff0000u), i);
          take(__uint_as_float(v[j].z << 16), __uint_as_float(v[j].z & 0xffff0000u), __uint_as_float(v[j].w << 16),
               __uint_as_float(v[j].w & 0xffff0000u), i + 4);
        }
      }
    }
    for (int i = whole + tid * 4; i < padded; i += kThreads * 4) {
      float x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = i + j < len ? static_cast<float>(row[i + j]) : -INFINITY;
      take(x[0], x[1], x[2], x[3], i);
    }
    if (top.i != 0x7fffffff) {  // which of the four
      const float4 y = get4(top.i);
      top.i += v0 + (y.x == top.v ? 0 : y.y == top.v ? 1 : y.z == top.v ? 2 : 3);
    }
  }
  constexpr int kLanes = kThreads * C / kLargest;  // of a group
  static_assert(kLanes <= 32);
  auto block_best = [&](Best x, bool groups) {  // (the groups' own to sh.group)
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      if (groups && o == kLanes && lane % kLanes == 0) sh.group[tid / kLanes] = x.v;
      x = better(x, Best{__shfl_xor_sync(0xffffffffu, x.v, o), __shfl_xor_sync(0xffffffffu, x.i, o)});
    }
    if (groups && kLanes == 32 && lane == 0) sh.group[warp] = x.v;
    if (lane == 0) sh.best[warp] = x;
    __syncthreads();
    x = sh.best[lane % kWarps];
#pragma unroll
    for (int o = kWarps / 2; o > 0; o >>= 1)
      x = better(x, Best{__shfl_xor_sync(0xffffffffu, x.v, o), __shfl_xor_sync(0xffffffffu, x.i, o)});
    return x;
  };
  // Sum over the block: a warp's in f32, those in 64 bits.
  auto block_sum = [&](float v) {
    v = warp_total(v);
    __syncthreads();  // (the sums before are read)
    if (lane == 0) sh.sums[warp] = v;
    __syncthreads();
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) s += sh.sums[i];
    return s;
  };
  int flip = 0;
  auto tell = [&](uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3, uint32_t w4) {
    if (tid < 5 * C) {
      const int word = tid / C;
      peer_store(&sh.got[flip][word][rank], tid % C,
                 word == 0 ? w0 : word == 1 ? w1 : word == 2 ? w2 : word == 3 ? w3 : w4);
    }
    meet();
    flip ^= 1;
  };
  // (words 0, 1: a logit and its token; 2, 3: a sum; 4: a number)
  auto tell_best = [&](Best x, double sum, uint32_t n) {
    const unsigned long long u = __double_as_longlong(sum);
    tell(__float_as_uint(x.v), (uint32_t)x.i, (uint32_t)u, (uint32_t)(u >> 32), n);
  };
  auto heard = [&](int word, int from) { return sh.got[flip ^ 1][word][from]; };
  auto heard_double = [&](int from) {
    return __longlong_as_double((unsigned long long)heard(3, from) << 32 | heard(2, from));
  };
  auto over_ctas = [&](double s) {  // each lane with CTA lane % 8's: every lane gets the same
#pragma unroll
    for (int o = C / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return s;
  };
  auto heard_sum = [&]() { return over_ctas(heard_double(lane % C)); };
  auto heard_count = [&]() {
    uint32_t n = 0;
    for (int r = 0; r < C; ++r) n += heard(4, r);
    return n;
  };
  auto best_of_all = [&]() {
    Best x{__uint_as_float(heard(0, lane % C)), (int)heard(1, lane % C)};
#pragma unroll
    for (int o = C / 2; o > 0; o >>= 1)
      x = better(x, Best{__shfl_xor_sync(0xffffffffu, x.v, o), __shfl_xor_sync(0xffffffffu, x.i, o)});
    return x;
  };
  top = block_best(top, true);
  // for top-p alone: the slice's weights over its largest logit
  double slice_sum = 0.0;
  if (by_p && !by_k && !greedy) {
    const float over = fmaxf(top.v, kLowest);  // (a slice may have no finite logit)
    float part = 0.0f;
#pragma unroll 5
    for (int i = tid * 4; i < len; i += kThreads * 4) {
      const float4 x = get4(i);
      part += (pow2((x.x - over) * per) + pow2((x.y - over) * per)) + (pow2((x.z - over) * per) + pow2((x.w - over) * per));
    }
    slice_sum = block_sum(part);
  }
  __syncwarp();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  static_assert(kLargest <= kThreads);
  if (tid < kLargest)
    peer_store(&sh.maxima[rank * (kLargest / C) + tid / C], tid % C, __float_as_uint(sh.group[tid / C]));
  tell_best(top, slice_sum, 0);
  top = best_of_all();
  if (greedy || top.i == 0x7fffffff) {
    if (rank == 0 && tid == 0) {
      a.tokens[b] = top.i == 0x7fffffff ? -1 : top.i;
      if (a.logprobs) a.logprobs[b] = top.i == 0x7fffffff ? -INFINITY : 0.0f;
    }
    return;
  }
  const float largest = top.v;
  auto depth = [&](float x) { return (largest - x) * per; };  // w = 2^-depth
  double whole;  // the weights' sum, for top-p alone
  {
    const float theirs = fmaxf(__uint_as_float(heard(0, lane % C)), kLowest);
    whole = over_ctas(heard_double(lane % C) * (double)pow2(-depth(theirs)));
  }
  // What is kept so far: logits above `cut`, and those equal to it up to the slice's
  // token `cut_index`.
  float cut = -INFINITY, above_cut = -INFINITY;
  int cut_index = -1;
  auto set_cut = [&](float x, int token) {
    cut = x;
    above_cut = unordered(ordered(x) + 1);
    cut_index = token - v0;
  };
  auto kept = [&](float x, int i) { return x > cut || (x == cut && i <= cut_index); };
  // four of the slice's logits; -inf where they are not kept
  auto load4 = [&](int i) {
    float4 y = get4(i);
    if (cut > -INFINITY) {
      const float from = i <= cut_index ? cut : above_cut;
      y.x = y.x >= from ? y.x : -INFINITY;
      y.y = y.y >= from ? y.y : -INFINITY;
      y.z = y.z >= from ? y.z : -INFINITY;
      y.w = y.w >= from ? y.w : -INFINITY;
      if (i <= cut_index && cut_index < i + 3) {
        if (i + 1 > cut_index && y.y == cut) y.y = -INFINITY;
        if (i + 2 > cut_index && y.z == cut) y.z = -INFINITY;
        if (y.w == cut) y.w = -INFINITY;
      }
    }
    return y;
  };
  // f(x, i) for the slice's kept logits x[0, 4) from i on where one is `bound`
  // (finite) or above
  auto for_above = [&](float bound, auto f) {
#pragma unroll 2
    for (int i = tid * 4; i < len; i += kThreads * 4) {
      const float4 y = load4(i);
      const float x[4] = {y.x, y.y, y.z, y.w};
      if (fmaxf(fmaxf(y.x, y.y), fmaxf(y.z, y.w)) >= bound) f(x, i);
    }
  };
  // the row's token and its log probability, of weights that sum to s
  auto answer = [&](int token, float x, double s) {
    a.tokens[b] = token;
    if (a.logprobs) a.logprobs[b] = (float)(((double)x - (double)largest) / (double)temp - log(s));
  };
  // Lists the slice's logits from `bound` up that are wanted(x, i), as long as there
  // is room; returns how many the cluster has, with the sum of the weights of this
  // CTA's told where it is asked for.
  int lists = 0;
  auto gather = [&](float bound, bool weigh, auto wanted) {
    float in = 0.0f;
    for_above(bound, [&](const float (&x)[4], int i) {
      uint32_t hits = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) hits |= (uint32_t)((x[j] >= bound) & wanted(x[j], i + j)) << j;
      if (!hits) return;
      uint32_t at = atomicAdd(&sh.listed[lists], (uint32_t)__popc(hits));
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (hits >> j & 1) {
          if (at < (uint32_t)kList) sh.list[at] = (unsigned long long)~ordered(x[j]) << 32 | (uint32_t)(v0 + i + j);
          ++at;
          asm volatile("prefetch.global.L2 [%0];" ::"l"(noise + i + j));
          if (weigh) in += pow2(-depth(x[j]));
        }
    });
    const double mine = weigh ? block_sum(in) : 0.0;
    __syncthreads();
    tell_best(Best{0.0f, 0}, mine, sh.listed[lists]);
    ++lists;
    return heard_count();
  };
  // The lists of the cluster, n in all: its tid-th token, in order of CTA (the first
  // CTA's threads).
  auto listed = [&](int n) {
    int r = 0, at = tid;
    while (r < C - 1 && at >= (int)heard(4, r)) at -= (int)heard(4, r++);
    return tid < n ? peer_load(&sh.list[at], r) : ~0ull;
  };
  // The running sum of the weights w of the ordered list, without the thread's own.
  auto before_in_list = [&](float w) {
    double run = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double y = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += y;
    }
    __syncthreads();
    if (lane == 31) sh.sums[warp] = run;
    __syncthreads();
    double before = run - w;
    for (int i = 0; i < warp; ++i) before += sh.sums[i];
    return before;
  };

  if (by_k ? k <= kDirect : by_p) {
    const int wanted = by_k ? k : kDirectSum;
    {  // The smallest of the groups' largest that fewer than `wanted` of them are above:
       // four threads each, a quarter of the others.
      static_assert(kThreads == 4 * kLargest);
      const float mine = sh.maxima[tid / 4];
      int above = 0;
#pragma unroll
      for (int j = 0; j < kLargest / 16; ++j) {
        const float4 x = *reinterpret_cast<const float4 *>(sh.maxima + 4 * (4 * j + tid % 4));
        above += (x.x > mine) + (x.y > mine) + (x.z > mine) + (x.w > mine);
      }
      above += __shfl_xor_sync(0xffffffffu, above, 1);
      above += __shfl_xor_sync(0xffffffffu, above, 2);
      const uint32_t low = __reduce_min_sync(0xffffffffu, above < wanted ? ordered(mine) : 0xffffffffu);
      if (lane == 0) atomicMin(&sh.bound, low);
    }
    __syncthreads();
    const uint32_t n = gather(fmaxf(unordered(sh.bound), kLowest), !by_k, [](float, int) { return true; });
    // (a list whose weights make p of the row's but for rounding might be a token short)
    if (n <= (uint32_t)kList && (by_k || heard_sum() >= (double)p * whole * (1.0 + 1e-6))) {
      unsigned long long mine = rank == 0 ? listed((int)n) : 0;
      __syncwarp();
      asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // the lists are read
      if (rank != 0) {
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        return;
      }
      const int most = by_k ? min((int)n, k) : (int)n;
      mine = sorted(sh, (int)n, mine);
      const int token = (int)(uint32_t)mine;
      const float x = tid < most ? unordered(~(uint32_t)(mine >> 32)) : -INFINITY, w = pow2(-depth(x));
      const float e = tid < most ? __ldg(a.noise + (size_t)b * a.noise_pitch + token) : 1.0f;
      const double before = by_p ? before_in_list(w) : 0.0;
      if (by_k && by_p) whole = block_sum(w);
      const bool in = tid < most && (tid == 0 || !by_p || before < (double)p * whole) && w >= least;
      // (a number that is none, of a noise of none or a weight of 0 over a noise of 0, wins no race)
      const Best pick = block_best(in ? Best{fmaxf(w * inverse(e), 0.0f), token} : Best{0.0f, top.i}, false);
      const double s = block_sum(in ? w : 0.0f);
      if (tid < most && token == pick.i) answer(token, x, s);
      __syncwarp();
      asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
      return;
    }
  }

  // Weights go to a histogram as whole numbers, relative to their bin's, so that
  // their sum does not depend on the order: as many bits as leave room for the whole
  // slice in a word (17 for 151936 tokens: off by 2^-18 of themselves at most, so
  // that top-p's border is to within that of the row's sum).  A bin is a nearest
  // whole number: added to 1.5 * 2^23 it lies in the low bits, as the weight does
  // added to 2^23 (conversions take as long as a power, and a word's atomic longer
  // than the rest: with two words 22 bits are kept and a flat row takes 5 us more).
  constexpr float kRound = 12582912.0f;
  const float units = fminf(3.5e9f / (float)a.slice, 4.0e6f);
  auto count_in = [&](bool ok, int bin, float u, bool weigh) {
    add_if(ok, &sh.hist[bin], weigh ? __float_as_uint(fmaf(u, units, 8388608.0f)) & 0x7fffffu : 1u);
  };
  auto clear_hist = [&]() {
    if (tid < kBins) sh.hist[tid] = 0;
    __syncthreads();
  };
  if (by_p) want_noise();  // much of it: more is kept than fits the list

  for (int which = 0; which < 2; ++which) {
    const bool weigh = which == 1;
    if (!(weigh ? by_p : by_k)) continue;
    float bound = kLowest, octave = 8.0f;  // bins an octave
    if (weigh) {
      if (by_k) {  // of what top-k kept
        float part = 0.0f;
        for_above(kLowest, [&](const float (&x)[4], int) {
          part += (pow2(-depth(x[0])) + pow2(-depth(x[1]))) + (pow2(-depth(x[2])) + pow2(-depth(x[3])));
        });
        tell_best(top, block_sum(part), 0);
        whole = heard_sum();
      }
      // Tokens this far down can be no part of top-p's: all of them together, each
      // below (1 - p) / vocab of the sum, are less than 1 - p of it.
      const float deepest = log2f((float)a.vocab / ((1.0f - fmaxf(p, 0.0f)) * (float)whole)) + 1.0f;
      bound = fmaxf(largest - deepest / per, kLowest);
      octave = (float)(kBins - 1) / fmaxf(deepest, 1.0f);
    }
    const float step = 1.0f / octave;
    auto bin_of = [&](float x, float *nearest) {
      const float r = fminf(depth(x) * octave, (float)(kBins - 1)) + kRound;
      *nearest = r - kRound;
      return (int)(__float_as_uint(r) & 0x3ffu);
    };
    clear_hist();
    for_above(bound, [&](const float (&x)[4], int) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float nearest;
        const int bin = bin_of(x[j], &nearest);
        count_in(x[j] >= bound, bin, weigh ? pow2(fmaf(nearest, step, -depth(x[j]))) : 0.0f, weigh);
      }
    });
    meet();
    const double target = weigh ? (double)fmaxf(p, 0.0f) * whole : (double)k;
    const int border = find_border(sh, weigh, target, 0, 0.0, 1.0 / (double)units, step);
    if (border < 0) {  // all that is there is kept
      meet();  // the histograms are read
      continue;
    }
    uint32_t n_before = sh.n_before;
    double s_before = sh.s_before;
    // The logits [lo, hi] of the border's bin, ordered: a bin is a step of a falling
    // function, whose ends a warp finds 32 at a time.
    auto first_below = [&](int end) {  // the lowest ordered logit whose bin is below `end`
      // (it lies near the bins' border, or at an end; in [at, above])
      const float near = largest - ((float)end - 0.5f) * step / per, slack = fabsf(near) * 1e-6f + fabsf(largest) * 1e-6f;
      uint32_t at = ordered(bound), above = ordered(largest) + 1;
      float nearest;
      const uint32_t low = ordered(fminf(fmaxf(near - slack, bound), largest)), high = ordered(fminf(fmaxf(near + slack, bound), largest));
      if (bin_of(unordered(low), &nearest) >= end) at = low; else above = low;
      if (high >= at && high < above) {
        if (bin_of(unordered(high), &nearest) >= end) at = high; else above = high;
      }
      while (at < above) {
        const uint32_t part = ((above - at) >> 5) + 1, mine = at + lane * part;
        const bool in = mine < above && bin_of(unordered(mine), &nearest) >= end;
        const int n = __popc(__ballot_sync(0xffffffffu, in));  // the lanes' first n
        if (n < 32 && at + n * part < above) above = at + n * part;
        if (n > 0) at = at + (n - 1) * part + 1;
      }
      return at;
    };
    uint32_t lo = first_below(border + 1), hi = first_below(border) - 1;
    // By ever finer histograms, until the tokens there fit the list or are equal.
    bool all_of_it = false;
    uint32_t n_in = sh.n_in;
    while (true) {
      to_values<T>(&lo, &hi);
      if (lo == hi) break;
      const float low = unordered(lo), high = unordered(hi);
      if (n_in <= (uint32_t)kList) {
        n_in = gather(low, false, [&](float x, int) { return x <= high; });  // (meets: the histograms are read)
        if (n_in <= (uint32_t)kList) break;
      } else {
        meet();
      }
      const int shift = max(0, 32 - __clz((int)(hi - lo)) - 8);
      const float d0 = depth(high);
      clear_hist();
      for_above(low, [&](const float (&x)[4], int) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          count_in(x[j] >= low && x[j] <= high, (int)(min(hi - ordered(x[j]), hi - lo) >> shift),
                   weigh ? pow2(d0 - depth(x[j])) : 0.0f, weigh);
      });
      meet();
      const double scale = (double)pow2(-d0);
      const int finer = find_border(sh, weigh, weigh ? (target - s_before) / scale : target, weigh ? 0 : n_before, 0.0,
                                    1.0 / (double)units, 0.0f);
      if (finer < 0) {  // (rounding has the whole bin short of the target)
        all_of_it = true;
        break;
      }
      n_before = sh.n_before;
      n_in = sh.n_in;
      s_before += weigh ? sh.s_before * scale : 0.0;
      hi -= (uint32_t)finer << shift;
      if (hi - lo >= 1u << shift) lo = hi - ((1u << shift) - 1);
    }
    if (all_of_it) {
      set_cut(unordered(lo), 0x7fffffff);
    } else if (lo != hi) {
      if (rank == 0) {
        const unsigned long long mine = sorted(sh, (int)n_in, listed((int)n_in));
        const bool in = tid < (int)n_in;
        const float x = unordered(~(uint32_t)(mine >> 32)), w = in ? pow2(-depth(x)) : 0.0f;
        if (tid == 0) sh.border = weigh ? (int)n_in - 1 : min((int)n_in, k - (int)n_before) - 1;
        const double run = s_before + before_in_list(w) + w;  // (meets)
        if (weigh && in && run >= target) atomicMin(&sh.border, tid);
        __syncthreads();
        if (tid == max(0, sh.border))
          for (int r = 0; r < C; ++r) {
            peer_store(&sh.cut, r, __float_as_uint(x));
            peer_store(&sh.cut_index, r, (uint32_t)mine);
          }
      }
      meet();
      set_cut(sh.cut, sh.cut_index);
    } else {
      // equal logits: as many of them as are wanted, by index.  A warp counts those of
      // its own part of the slice, and the one that has the last goes through it again.
      const float equal = unordered(lo);
      const int quads = (len + 3) / 4, part = (quads + kWarps - 1) / kWarps, q1 = min(quads, (warp + 1) * part);
      auto count4 = [&](int q) {  // a bit for each of the four that is one of them
        if (q >= q1) return 0u;
        const int i = 4 * q;
        const float4 x = get4(i);
        return (uint32_t)((x.x == equal) & kept(equal, i)) | (uint32_t)((x.y == equal) & kept(equal, i + 1)) << 1 |
               (uint32_t)((x.z == equal) & kept(equal, i + 2)) << 2 | (uint32_t)((x.w == equal) & kept(equal, i + 3)) << 3;
      };
      int mine = 0;
#pragma unroll 4
      for (int q = warp * part + lane; q < q1; q += 32) mine += __popc(count4(q));
      mine = __reduce_add_sync(0xffffffffu, mine);
      __syncthreads();
      if (lane == 0) sh.counts[warp] = mine;
      __syncthreads();
      int before = 0, all = 0;
      for (int i = 0; i < kWarps; ++i) {
        if (i < warp) before += sh.counts[i];
        all += sh.counts[i];
      }
      tell((uint32_t)all, 0, 0, 0, 0);  // (meets: the histograms are read)
      int total = 0;
      for (int r = 0; r < C; ++r) {
        if (r < (int)rank) before += heard(0, r);
        total += heard(0, r);
      }
      const double each = (double)pow2(-depth(equal));
      int wanted = weigh ? (int)fmin(fmax(ceil((target - s_before) / each), 1.0), (double)total) : k - (int)n_before;
      wanted = max(1, min(wanted, total)) - before;  // the warp's
      if (wanted >= 1 && wanted <= mine) {
        for (int q = warp * part + lane;; q += 32) {
          uint32_t bits = count4(q);
          int run = __popc(bits);
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, run, o);
            if (lane >= o) run += y;
          }
          const int there = __shfl_sync(0xffffffffu, run, 31), skip = wanted - 1 - (run - __popc(bits));
          if (there >= wanted) {
            if (skip >= 0 && skip < __popc(bits)) {
              for (int n = 0; n < skip; ++n) bits &= bits - 1;
              for (int r = 0; r < C; ++r) peer_store(&sh.cut_index, r, (uint32_t)(v0 + 4 * q + __ffs(bits) - 1));
            }
            break;
          }
          wanted -= there;
        }
      }
      meet();
      set_cut(equal, sh.cut_index);
    }
    meet();  // what the CTAs told one another here is read
  }

  // The race over what is kept: the best of four tokens at a time, and in the end
  // which of a thread's best four it was.
  float best = 0.0f, part = 0.0f;
  int at = -1;
  const float deep = least > 0.0f ? -log2f(least) : INFINITY;
  const float bound = fmaxf(fmaxf(cut, largest - deep / per * 1.0001f - fabsf(largest) * 1e-6f), kLowest);
  auto weight = [&](float x) {  // 0: not kept
    const float w = pow2(-depth(x));
    return w >= least ? w : 0.0f;
  };
  constexpr int kFew = 3;
  for (int i0 = tid * 4; i0 - lane * 4 < len; i0 += kFew * kThreads * 4) {
    float4 x[kFew], e[kFew];
    bool any = false;
#pragma unroll
    for (int j = 0; j < kFew; ++j) {
      const int i = i0 + j * kThreads * 4;
      x[j] = i < len ? load4(i) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
      const bool hit = fmaxf(fmaxf(x[j].x, x[j].y), fmaxf(x[j].z, x[j].w)) >= bound;
      any |= hit;
      e[j] = make_float4(1.0f, 1.0f, 1.0f, 1.0f);
      if (hit && a.noise_vec && i + 4 <= len) {
        e[j] = __ldg(reinterpret_cast<const float4 *>(noise + i));
      } else if (hit) {
        e[j].x = __ldg(noise + i);
        if (i + 1 < len) e[j].y = __ldg(noise + i + 1);
        if (i + 2 < len) e[j].z = __ldg(noise + i + 2);
        if (i + 3 < len) e[j].w = __ldg(noise + i + 3);
      }
    }
    if (!__any_sync(0xffffffffu, any)) continue;
#pragma unroll
    for (int j = 0; j < kFew; ++j) {
      const int i = i0 + j * kThreads * 4;
      const float w[4] = {weight(x[j].x), weight(x[j].y), weight(x[j].z), weight(x[j].w)};
      part += (w[0] + w[1]) + (w[2] + w[3]);
      const float v = fmaxf(fmaxf(w[0] * inverse(e[j].x), w[1] * inverse(e[j].y)),
                            fmaxf(w[2] * inverse(e[j].z), w[3] * inverse(e[j].w)));
      if (v > best) {
        best = v;
        at = i;
      }
    }
  }
  Best pick{0.0f, top.i};
  float pick_x = largest;
  if (at >= 0) {
    pick.v = -1.0f;
    const float4 y = load4(at);
    const float x[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float w = weight(x[j]), v = w > 0.0f ? w * inverse(__ldg(noise + at + j)) : -1.0f;
      if (v > pick.v) {
        pick = Best{v, v0 + at + j};
        pick_x = x[j];
      }
    }
  }
  // the warps' best, with its logit, and sums meet
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const Best y{__shfl_xor_sync(0xffffffffu, pick.v, o), __shfl_xor_sync(0xffffffffu, pick.i, o)};
    const float y_x = __shfl_xor_sync(0xffffffffu, pick_x, o);
    const Best z = better(pick, y);
    if (z.i != pick.i) pick_x = y_x;
    pick = z;
  }
  part = warp_total(part);
  __syncthreads();
  if (lane == 0) {
    sh.best[warp] = pick;
    sh.last_x[warp] = pick_x;
    sh.last_sum[warp] = part;
  }
  __syncthreads();
  double mine_s = 0.0;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) {
    const Best z = better(pick, sh.best[i]);
    if (z.i != pick.i) pick_x = sh.last_x[i];
    pick = z;
    mine_s += sh.last_sum[i];
  }
  tell_best(pick, mine_s, __float_as_uint(pick_x));
  pick = best_of_all();
  const double all = heard_sum();
  if (rank == 0 && tid == 0) {
    float x = 0.0f;
    for (int r = 0; r < C; ++r)
      if ((int)heard(1, r) == pick.i) x = __uint_as_float(heard(4, r));
    answer(pick.i, x, all);
  }
}

template <typename T, int C>
int run_sample(const SampleArgs &a, size_t batch, cudaStream_t s) {
  {
    static std::mutex mu;
    static std::vector<int> done;
    int dev = 0;
    FPB_CUDA_TRY(cudaGetDevice(&dev));
    std::lock_guard<std::mutex> lock(mu);
    if (std::find(done.begin(), done.end(), dev) == done.end()) {
      FPB_CUDA_TRY(cudaFuncSetAttribute(sample_kernel<T, C>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        (int)std::max(kMaxSlice * sizeof(T), kPairSlice)));
      done.push_back(dev);
    }
  }
  cudaError_t e = launch_pdl_cluster(sample_kernel<T, C>, dim3(C, (unsigned)batch), kThreads,
                                     (size_t)a.slice * sizeof(T), s, C, a);
  if (e != cudaSuccess) return cuda_fail(e, "sample_kernel");
  FPB_LAUNCH_CHECK("sample_kernel");
  return FPB_OK;
}

}  // namespace
}  // namespace fpb

using namespace fpb;

extern "C" int fpb_sample(const void *logits, int logits_dtype, size_t logits_pitch, const float *temperature,
                          const int32_t *top_k, const float *top_p, const float *min_p, const float *noise,
                          size_t noise_pitch, size_t batch, size_t vocab, int32_t *tokens, float *logprobs,
                          void *stream) {
  if (!logits || !noise || !tokens) return fail(FPB_ERR_INVALID_ARGUMENT, "fpb_sample: null pointer");
  if (logits_dtype != FPB_F32 && logits_dtype != FPB_BF16)
    return fail(FPB_ERR_INVALID_ARGUMENT, "fpb_sample: dtype");
  if (batch == 0 || batch > 65535 || vocab == 0 || vocab > (size_t)kMaxVocab || logits_pitch < vocab || noise_pitch < vocab ||
      (logits_pitch | noise_pitch) >> 38)
    return fail(FPB_ERR_SHAPE, "fpb_sample: batch %zu, vocab %zu (at most %d), pitches", batch, vocab, kMaxVocab);
  if (reinterpret_cast<uintptr_t>(logits) % (logits_dtype == FPB_F32 ? 4 : 2) ||
      reinterpret_cast<uintptr_t>(noise) % 4)
    return fail(FPB_ERR_INVALID_ARGUMENT, "fpb_sample: alignment");
  SampleArgs a{};
  a.logits = logits;
  a.temperature = temperature;
  a.top_k = top_k;
  a.top_p = top_p;
  a.min_p = min_p;
  a.noise = noise;
  a.logits_pitch = (long long)logits_pitch;
  a.noise_pitch = (long long)noise_pitch;
  a.vocab = (int)vocab;
  a.tokens = tokens;
  a.logprobs = logprobs;
  // Two CTAs an SM: about 32 rows are there at once in clusters of eight, and most of a
  // row's time goes by in its exchanges, so that many rows take fewer CTAs each, as long
  // as two slices fit an SM (us for C = 8 / 4 / 2, each row with filters of its own:
  // 250 x 151936 bf16 113 / 95 / -, 100 of them 59 / 59, 40 of them 35 / 45; 250 x 32000
  // bf16 76 / 51 / 41, 100 of them 39 / 30 / 29, 56 of them 26 / 24 / 26, 24 of them 20 /
  // 21 / 25; 150 x 100000 f32 70 / 63 / -, 72 of them 43 / 42).
  const size_t el = logits_dtype == FPB_F32 ? 4 : 2, sms = sm_count();
  auto slice = [&](size_t c) { return ((vocab + c - 1) / c + 7) / 8 * 8; };
  const int C = batch * 8 > 5 * sms && slice(2) <= 16384 ? 2
                : batch * 16 > 5 * sms && slice(4) <= 16384 ? 4
                : batch * 8 > 5 * sms && slice(4) * el <= kPairSlice ? 4
                    : 8;
  a.slice = (int)slice(C);
  auto lies = [](const void *p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && bytes % 16 == 0; };
  a.vec = lies(logits, logits_pitch * el);
  a.noise_vec = lies(noise, noise_pitch * 4);
  cudaStream_t st = as_stream(stream);
  auto run = [&](auto t) {
    using T = decltype(t);
    return C == 2 ? run_sample<T, 2>(a, batch, st) : C == 4 ? run_sample<T, 4>(a, batch, st) : run_sample<T, 8>(a, batch, st);
  };
  return logits_dtype == FPB_F32 ? run(0.0f) : run(__nv_bfloat16());
}
