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
#include <algorithm>
#include <cmath>
#include <mutex>
#include <vector>

#include "common.cuh"

namespace fpb {
namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32, kCluster = 8;
constexpr int kMaxSlice = 49152;  // f32 of shared memory a CTA: 192 KB
constexpr int kBatch = 5;         // 16-byte loads a thread has under way
constexpr int kBins = 256, kPerOctave = 8;  // bins of a histogram: an eighth of a power of two each, the last one the rest
constexpr int kList = 2048;       // tokens that one CTA orders

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

// Order of f32 values as that of whole numbers, and back.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t u) {
  return __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u);
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
__device__ __forceinline__ void peer_store(const void *p, unsigned rank, unsigned long long v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(peer_address(p, rank)), "l"(v) : "memory");
}
__device__ __forceinline__ uint32_t peer_load(const uint32_t *p, unsigned rank) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(peer_address(p, rank)) : "memory");
  return v;
}

template <typename V>
__device__ __forceinline__ V warp_total(V v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

struct Shared {
  unsigned long long list[kList];  // of the first CTA: tokens to be ordered, (falling logit, index) as one number
  uint32_t hist[3][kBins];         // tokens; their weights' sum, low and high part
  // what the CTAs tell one another; the halves alternate, so that one exchange's
  // reads may overlap the next one's stores
  uint32_t got[2][5][kCluster];
  float maxima[kCluster * kWarps];  // every warp's largest logit
  double sums[kWarps];
  uint32_t counts[kWarps];
  Best best[kWarps];
  int border, n_before, n_in;  // where a histogram reaches its target: the bin, tokens before and in it
  double s_before;
  int gathered[3];  // of the first CTA: tokens in the list, each time anew
  int sent;         // this CTA's part of the first ones
  uint32_t cut, cut_index;
  float bound, pick_x;
};

// A cluster of kCluster CTAs a row: CTA `rank` keeps the vocabulary's slice [rank
// * slice, +slice) in shared memory, so that the row is read once.
//  1. Every warp's largest logit goes to every CTA: the row's largest, and with the
//     k-th largest of the 128 (all of them for top-p alone) a bound that at least k
//     tokens reach.
//  2. What reaches it (a few times k tokens) goes to the first CTA's list, which is
//     put in order; there the filters are running sums.  top-p alone: if the list's
//     weights make p of the row's.
//  3. Where they do not, or k is larger, the border that a filter leaves is found by
//     a histogram over the cluster, and in the border's bin by the list, or by finer
//     histograms until the tokens there fit it, or are equal.  What is kept races
//     where it lies.
template <typename T>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const __grid_constant__ SampleArgs a) {
  // every CTA of the cluster runs, before its shared memory is stored to
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  pdl_enter();
  extern __shared__ __align__(16) float xs[];  // the slice's logits
  __shared__ Shared sh;
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
  if (!greedy && plain && a.noise_vec && tid == 0 && len >= 4)  // all of its noise is wanted
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(noise), "r"(len / 4 * 16) : "memory");
  if (tid < 3) sh.gathered[tid] = 0;
  if (tid == 3) sh.sent = 0;

  // the slice to shared memory, and its first largest logit
  Best top{-INFINITY, 0x7fffffff};
  auto take = [&](float x, int i) {
    x = fabsf(x) <= 3.402823466e38f ? x : -INFINITY;
    if (x > top.v) top = Best{x, v0 + i};
    return x;
  };
  {
    constexpr int N = 16 / sizeof(T);
    const int whole = a.vec ? len / N * N : 0;
    for (int i0 = tid * N; i0 < whole; i0 += kBatch * kThreads * N) {
      uint4 v[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int i = i0 + j * kThreads * N;
        v[j] = i < whole ? __ldg(reinterpret_cast<const uint4 *>(row + i)) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int i = i0 + j * kThreads * N;
        if (i >= whole) break;
        const uint32_t w[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
        if constexpr (N == 4) {
          float4 y;
          y.x = take(__uint_as_float(w[0]), i);
          y.y = take(__uint_as_float(w[1]), i + 1);
          y.z = take(__uint_as_float(w[2]), i + 2);
          y.w = take(__uint_as_float(w[3]), i + 3);
          *reinterpret_cast<float4 *>(xs + i) = y;
        } else {
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            float4 y;
            y.x = take(__uint_as_float(w[2 * q] << 16), i + 4 * q);
            y.y = take(__uint_as_float(w[2 * q] & 0xffff0000u), i + 4 * q + 1);
            y.z = take(__uint_as_float(w[2 * q + 1] << 16), i + 4 * q + 2);
            y.w = take(__uint_as_float(w[2 * q + 1] & 0xffff0000u), i + 4 * q + 3);
            *reinterpret_cast<float4 *>(xs + i + 4 * q) = y;
          }
        }
      }
    }
    for (int i = whole + tid; i < padded; i += kThreads) xs[i] = i < len ? take(static_cast<float>(row[i]), i) : -INFINITY;
  }
  auto block_best = [&](Best x) {  // (the warps' own are left in sh.best)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
      x = better(x, Best{__shfl_xor_sync(0xffffffffu, x.v, o), __shfl_xor_sync(0xffffffffu, x.i, o)});
    if (lane == 0) sh.best[warp] = x;
    __syncthreads();
    x = sh.best[lane % kWarps];
#pragma unroll
    for (int o = kWarps / 2; o > 0; o >>= 1)
      x = better(x, Best{__shfl_xor_sync(0xffffffffu, x.v, o), __shfl_xor_sync(0xffffffffu, x.i, o)});
    return x;
  };
  auto block_sum = [&](double v) {
    v = warp_total(v);
    __syncthreads();  // (the sums before are read)
    if (lane == 0) sh.sums[warp] = v;
    __syncthreads();
    v = sh.sums[lane % kWarps];
#pragma unroll
    for (int o = kWarps / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  };
  int flip = 0;
  auto tell = [&](uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3, uint32_t w4 = 0) {
    if (tid < kCluster) {
      peer_store(&sh.got[flip][4][rank], tid, w4);
      peer_store(&sh.got[flip][0][rank], tid, w0);
      peer_store(&sh.got[flip][1][rank], tid, w1);
      peer_store(&sh.got[flip][2][rank], tid, w2);
      peer_store(&sh.got[flip][3][rank], tid, w3);
    }
    cluster_sync();
    flip ^= 1;
  };
  auto tell_sums = [&](double x, double y, uint32_t n = 0) {
    const unsigned long long u = __double_as_longlong(x), v = __double_as_longlong(y);
    tell((uint32_t)u, (uint32_t)(u >> 32), (uint32_t)v, (uint32_t)(v >> 32), n);
  };
  auto heard = [&](int word, int from) { return sh.got[flip ^ 1][word][from]; };
  auto heard_sum = [&](int word) {  // over the CTAs, in order
    double s = 0.0;
    for (int r = 0; r < kCluster; ++r)
      s += __longlong_as_double((unsigned long long)heard(word + 1, r) << 32 | heard(word, r));
    return s;
  };
  auto best_of_all = [&]() {
    Best x{__uint_as_float(heard(0, lane % kCluster)), (int)heard(1, lane % kCluster)};
#pragma unroll
    for (int o = kCluster / 2; o > 0; o >>= 1)
      x = better(x, Best{__shfl_xor_sync(0xffffffffu, x.v, o), __shfl_xor_sync(0xffffffffu, x.i, o)});
    return x;
  };
  top = block_best(top);
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  static_assert(kWarps * kCluster <= kThreads);
  if (tid < kWarps * kCluster)
    peer_store(&sh.maxima[rank * kWarps + tid / kCluster], tid % kCluster, __float_as_uint(sh.best[tid / kCluster].v));
  tell(__float_as_uint(top.v), (uint32_t)top.i, 0, 0);
  top = best_of_all();
  if (greedy || top.i == 0x7fffffff) {
    if (rank == 0 && tid == 0) {
      a.tokens[b] = top.i == 0x7fffffff ? -1 : top.i;
      if (a.logprobs) a.logprobs[b] = top.i == 0x7fffffff ? -INFINITY : 0.0f;
    }
    return;
  }
  const float temp = fminf(fmaxf(t, 1e-6f), 1e6f), per = 1.4426950408889634f / temp, largest = top.v;
  auto depth = [&](float x) { return (largest - x) * per; };  // w = 2^-depth
  // What is kept so far: logits above `cut` (ordered), and those of it up to index
  // `cut_index`.
  uint32_t cut = 0, cut_index = 0;
  auto kept = [&](float x, int i) {
    const uint32_t u = ordered(x);
    return u > cut || (u == cut && (uint32_t)(v0 + i) <= cut_index);
  };
  // f(x, i) for the slice's logits from `bound` (finite) up
  auto for_above = [&](float bound, auto f) {
#pragma unroll 2
    for (int i = tid * 4; i < len; i += kThreads * 4) {
      const float4 x = *reinterpret_cast<const float4 *>(xs + i);
      if (fmaxf(fmaxf(x.x, x.y), fmaxf(x.z, x.w)) >= bound) {
        if (x.x >= bound) f(x.x, i);
        if (x.y >= bound) f(x.y, i + 1);
        if (x.z >= bound) f(x.z, i + 2);
        if (x.w >= bound) f(x.w, i + 3);
      }
    }
  };
  constexpr float kLowest = -3.402823466e38f;
  // the row's token and its log probability, of weights that sum to s
  auto answer = [&](int token, float x, double s) {
    a.tokens[b] = token;
    if (a.logprobs) a.logprobs[b] = (float)(((double)x - (double)largest) / (double)temp - log(s));
  };
  // A token of the slice to the first CTA's list, if it has room.
  auto gather = [&](float x, int i, int counter) {
    uint32_t at;
    asm volatile("atom.shared::cluster.add.u32 %0, [%1], 1;"
                 : "=r"(at)
                 : "r"(peer_address(&sh.gathered[counter], 0))
                 : "memory");
    if (at < (uint32_t)kList) peer_store(&sh.list[at], 0, (unsigned long long)~ordered(x) << 32 | (uint32_t)(v0 + i));
  };
  // The first n of the list in order (the first CTA).
  auto sort_list = [&](int n) {
    if (n <= kThreads) {  // a token a thread; neighbours through registers
      int size = 32;
      while (size < n) size *= 2;
      unsigned long long x = tid < n ? sh.list[tid] : ~0ull;
      for (int run = 2; run <= size; run *= 2) {
        const bool up = (tid & run) == 0;
        for (int step = run / 2; step > 0; step /= 2) {
          unsigned long long y;
          if (step >= 32) {
            __syncthreads();
            if (tid < size) sh.list[tid] = x;
            __syncthreads();
            y = tid < size ? sh.list[tid ^ step] : x;
          } else {
            y = __shfl_xor_sync(0xffffffffu, x, step);
          }
          const bool low = (tid & step) == 0;
          x = (x < y) == (low == up) ? x : y;
        }
      }
      __syncthreads();
      if (tid < size) sh.list[tid] = x;
      __syncthreads();
      return;
    }
    int size = 2 * kThreads, bits;
    while (size < n) size *= 2;
    for (int i = n + tid; i < size; i += kThreads) sh.list[i] = ~0ull;
    __syncthreads();
    for (int run = 2; run <= size; run *= 2)
      for (bits = 30 - __clz(run); bits >= 0; --bits) {
        const int step = 1 << bits;
        for (int i = tid; i < size / 2; i += kThreads) {
          const int lo = (i >> bits) << (bits + 1) | (i & (step - 1)), hi = lo + step;
          const unsigned long long x = sh.list[lo], y = sh.list[hi];
          if ((x > y) == ((lo & run) == 0)) {
            sh.list[lo] = y;
            sh.list[hi] = x;
          }
        }
        __syncthreads();
      }
  };
  constexpr int kMine = kList / kThreads;
  // Four of the ordered list a thread: their logits and weights, and the weights'
  // sum before the first of them.
  auto list_sums = [&](int n, float (&x)[kMine], float (&w)[kMine]) {
    double mine = 0.0;
#pragma unroll
    for (int j = 0; j < kMine; ++j) {
      const int i = tid * kMine + j;
      x[j] = i < n ? unordered(~(uint32_t)(sh.list[i] >> 32)) : -INFINITY;
      w[j] = i < n ? pow2(-depth(x[j])) : 0.0f;
      mine += w[j];
    }
    double run = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double y = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += y;
    }
    __syncthreads();
    if (lane == 31) sh.sums[warp] = run;
    __syncthreads();
    double before = run - mine;
    for (int i = 0; i < warp; ++i) before += sh.sums[i];
    return before;
  };
  // The answer from a list of n that holds all that may be kept: the first `most` of
  // it, of them what makes p of `sum` (0: of their own weights).
  auto finish_list = [&](int n, int most, double sum) {
    sort_list(n);
    float x[kMine], w[kMine];
    double before = list_sums(n, x, w);
    if (sum == 0.0 && by_p) {
      double s = 0.0;
#pragma unroll
      for (int j = 0; j < kMine; ++j) s += tid * kMine + j < most ? w[j] : 0.0f;
      sum = block_sum(s);
    }
    Best pick{0.0f, top.i};
    double s = 0.0;
#pragma unroll
    for (int j = 0; j < kMine; ++j) {
      const int i = tid * kMine + j;
      if (i < most && (i == 0 || !by_p || before < (double)p * sum) && w[j] >= least) {
        const int token = (int)(uint32_t)sh.list[i];
        s += w[j];
        pick = better(pick, Best{__fdividef(w[j], a.noise[(size_t)b * a.noise_pitch + token]), token});
      }
      before += w[j];
    }
    s = block_sum(s);
    pick = block_best(pick);
#pragma unroll
    for (int j = 0; j < kMine; ++j) {
      const int i = tid * kMine + j;
      if (i < most && (int)(uint32_t)sh.list[i] == pick.i) answer(pick.i, x[j], s);
    }
  };

  double whole = 0.0;  // the row's weights, where they are known
  if (by_k ? k <= kWarps * kCluster : by_p) {
    const int wanted = by_k ? k : kWarps * kCluster;
    if (tid < kWarps * kCluster) {
      const float mine = sh.maxima[tid];
      int above = 0;
#pragma unroll 8
      for (int i = 0; i < kWarps * kCluster; ++i) {
        const float x = sh.maxima[i];
        above += x > mine || (x == mine && i < tid);
      }
      if (above == wanted - 1) sh.bound = fmaxf(mine, kLowest);
    }
    __syncthreads();
    const float bound = sh.bound;
    auto candidate = [&](float x, int i) {
      gather(x, i, 0);
      atomicAdd(&sh.sent, 1);
      asm volatile("prefetch.global.L2 [%0];" ::"l"(noise + i));
    };
    if (by_k) {
      for_above(bound, candidate);
      __syncthreads();
      tell_sums(0.0, 0.0, (uint32_t)sh.sent);
    } else {
      float part = 0.0f, in = 0.0f;
      for (int i = tid * 4; i < len; i += kThreads * 4) {
        const float4 x = *reinterpret_cast<const float4 *>(xs + i);
        const float w[4] = {pow2(-depth(x.x)), pow2(-depth(x.y)), pow2(-depth(x.z)), pow2(-depth(x.w))};
        part += (w[0] + w[1]) + (w[2] + w[3]);
        if (fmaxf(fmaxf(x.x, x.y), fmaxf(x.z, x.w)) >= bound) {
          const float y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (y[j] >= bound) {
              candidate(y[j], i + j);
              in += w[j];
            }
        }
      }
      const double mine = block_sum((double)part), mine_in = block_sum((double)in);
      tell_sums(mine, mine_in, (uint32_t)sh.sent);
      whole = heard_sum(0);
    }
    int n = 0;
    for (int r = 0; r < kCluster; ++r) n += (int)heard(4, r);
    // (a list whose weights make p of the row's but for rounding might be a token short)
    if (n <= kList && (by_k || heard_sum(2) >= (double)p * whole * (1.0 + 1e-6))) {
      if (rank == 0) finish_list(n, by_k ? min(n, k) : n, whole);
      return;
    }
  }

  // Weights go to a histogram as whole numbers, relative to the bin's largest, so
  // that their sum does not depend on the order: 31 bits in two parts of 16 and 15
  // (49152 of them fit 32 bits).
  auto count_in = [&](int bin, float u, bool weigh) {
    atomicAdd(&sh.hist[0][bin], 1u);
    if (weigh) {
      const uint32_t f = (uint32_t)__float2uint_rn(u * 0x1p31f);
      atomicAdd(&sh.hist[1][bin], f & 0xffffu);
      atomicAdd(&sh.hist[2][bin], f >> 16);
    }
  };
  auto clear_hist = [&]() {
    for (int i = tid; i < 3 * kBins; i += kThreads) (&sh.hist[0][0])[i] = 0;
    __syncthreads();
  };
  auto bin_of = [&](float x) { return (int)fminf(depth(x) * kPerOctave, (float)(kBins - 1)); };
  // Over the cluster's histograms (scale(bin): what a bin's weights are relative
  // to): the first bin at which the running count, or sum, from n0 and s0 on, reaches
  // the target (-1: none), with what lies before it.  Every CTA finds the same.
  auto find_border = [&](bool weigh, double target, double n0, double s0, auto scale) {
    uint32_t c = 0;
    unsigned long long s = 0;
    if (tid < kBins) {
#pragma unroll
      for (int r = 0; r < kCluster; ++r) {
        c += peer_load(&sh.hist[0][tid], r);
        if (weigh) s += peer_load(&sh.hist[1][tid], r) + ((unsigned long long)peer_load(&sh.hist[2][tid], r) << 16);
      }
    }
    const double v = weigh && tid < kBins ? (double)s * 0x1p-31 * scale(tid) : 0.0;
    // running count and sum over the bins
    uint32_t n = c;
    double run = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t x = __shfl_up_sync(0xffffffffu, n, o);
      const double y = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) {
        n += x;
        run += y;
      }
    }
    __syncthreads();
    if (lane == 31) {
      sh.counts[warp] = n;
      sh.sums[warp] = run;
    }
    if (tid == 0) sh.border = -1;
    __syncthreads();
    double s_at = s0;
    uint32_t n_at = 0;
#pragma unroll
    for (int i = 0; i < kBins / 32; ++i)
      if (i < warp) {
        n_at += sh.counts[i];
        s_at += sh.sums[i];
      }
    if (tid < kBins && c > 0 && (weigh ? s_at + run : n0 + n_at + n) >= target)
      atomicMax(&sh.border, kBins - 1 - tid);  // the first of them
    __syncthreads();
    const int border = sh.border < 0 ? -1 : kBins - 1 - sh.border;
    if (tid == border) {
      sh.n_before = (int)(n_at + n - c);
      sh.n_in = (int)c;
      sh.s_before = s_at + run - v;
    }
    __syncthreads();
    return border;
  };

  for (int which = 0; which < 2; ++which) {
    const bool weigh = which == 1;
    if (!(weigh ? by_p : by_k)) continue;
    float bound = kLowest;
    if (weigh) {
      if (whole == 0.0 || cut) {  // of what top-k kept
        float part = 0.0f;
        for_above(kLowest, [&](float x, int i) { part += kept(x, i) ? pow2(-depth(x)) : 0.0f; });
        tell_sums(block_sum((double)part), 0.0);
        whole = heard_sum(0);
      }
      // Tokens this far down can be no part of top-p's: all of them together, each
      // below (1 - p) / vocab of the sum, are less than 1 - p of it.
      const float deepest = log2f((float)a.vocab / ((1.0f - fmaxf(p, 0.0f)) * (float)whole)) + 1.0f;
      bound = fmaxf(largest - deepest / per, kLowest);
    }
    clear_hist();
    for_above(bound, [&](float x, int i) {
      if (!kept(x, i)) return;
      const int bin = bin_of(x);
      count_in(bin, weigh ? pow2((float)bin / kPerOctave - depth(x)) : 0.0f, weigh);
    });
    cluster_sync();
    const double target = weigh ? (double)fmaxf(p, 0.0f) * whole : (double)k;
    int border = find_border(weigh, target, 0.0, 0.0, [&](int bin) { return exp2(-(double)bin / kPerOctave); });
    if (border < 0) {  // all that is there is kept
      cluster_sync();  // the histograms are read
      continue;
    }
    int n_before = sh.n_before, n_in = sh.n_in;
    double s_before = sh.s_before;
    // (no logit of the border's bin is below this: the bin's own end, less rounding)
    const float deep = border == kBins - 1 ? INFINITY : (float)(border + 1) / kPerOctave;
    const float near = fmaxf(bound, fmaxf(largest - deep / per * 1.0001f - fabsf(largest) * 1e-6f, kLowest));
    if (n_before + n_in <= kList) {
      // what may be kept fits one CTA, which does the rest
      const int n = n_before + n_in;
      for_above(near, [&](float x, int i) {
        if (kept(x, i) && bin_of(x) <= border) gather(x, i, 1 + which);
      });
      cluster_sync();
      if (rank == 0) finish_list(n, weigh ? n : min(n, k), weigh ? whole : 0.0);
      return;
    }
    // Else the border itself is found, in the border's bin alone: by ever finer
    // histograms of the ordered logits until its tokens fit the list or are equal.
    uint32_t lo = 0xffffffffu, hi = 0;
    for_above(near, [&](float x, int i) {
      if (!kept(x, i) || bin_of(x) != border) return;
      lo = min(lo, ordered(x));
      hi = max(hi, ordered(x));
    });
    lo = __reduce_min_sync(0xffffffffu, lo);
    hi = __reduce_max_sync(0xffffffffu, hi);
    __syncthreads();
    if (lane == 0) {
      sh.counts[warp] = lo;
      sh.best[warp].i = (int)hi;
    }
    __syncthreads();
    lo = __reduce_min_sync(0xffffffffu, sh.counts[lane % kWarps]);
    hi = __reduce_max_sync(0xffffffffu, (uint32_t)sh.best[lane % kWarps].i);
    tell(lo, hi, 0, 0);
    lo = __reduce_min_sync(0xffffffffu, heard(0, lane % kCluster));
    hi = __reduce_max_sync(0xffffffffu, heard(1, lane % kCluster));
    while (n_in > kList && lo < hi) {
      const int shift = max(0, 32 - __clz((int)(hi - lo)) - 8);
      const float d0 = depth(unordered(hi));
      cluster_sync();  // the histograms are read
      clear_hist();
      for_above(near, [&](float x, int i) {
        const uint32_t u = ordered(x);
        if (u < lo || u > hi || !kept(x, i)) return;
        count_in((int)((hi - u) >> shift), weigh ? pow2(d0 - depth(x)) : 0.0f, weigh);
      });
      cluster_sync();
      const double scale = exp2(-(double)d0);
      border = find_border(weigh, target, (double)n_before, s_before, [&](int) { return scale; });
      if (border < 0) {  // (rounding has the whole bin short of the target: it is kept whole)
        hi = lo;
        n_in = 0;
        break;
      }
      n_before += sh.n_before;
      n_in = sh.n_in;
      s_before = sh.s_before;
      hi -= (uint32_t)border << shift;
      if (hi - lo >= 1u << shift) lo = hi - ((1u << shift) - 1);
    }
    if (n_in == 0) {
      cut = lo;
      cut_index = 0xffffffffu;
    } else if (n_in <= kList) {
      for_above(near, [&](float x, int i) {
        const uint32_t u = ordered(x);
        if (u >= lo && u <= hi && kept(x, i)) gather(x, i, 1 + which);
      });
      cluster_sync();
      if (rank == 0) {
        sort_list(n_in);
        float x[kMine], w[kMine];
        double run = s_before + list_sums(n_in, x, w);
        if (tid == 0) sh.border = weigh ? n_in - 1 : min(n_in - 1, k - 1 - n_before);
        __syncthreads();
        if (weigh) {
#pragma unroll
          for (int j = 0; j < kMine; ++j) {
            run += w[j];
            if (tid * kMine + j < n_in && run >= target) atomicMin(&sh.border, tid * kMine + j);
          }
          __syncthreads();
        }
        const unsigned long long last = sh.list[sh.border];
        if (tid < kCluster) {
          peer_store(&sh.cut, tid, ~(uint32_t)(last >> 32));
          peer_store(&sh.cut_index, tid, (uint32_t)last);
        }
      }
      cluster_sync();
      cut = sh.cut;
      cut_index = sh.cut_index;
    } else {
      // equal logits: as many of them as are wanted, by index
      const double each = (double)pow2(-depth(unordered(lo)));
      int wanted = weigh ? (int)fmin(fmax(ceil((target - s_before) / each), 1.0), (double)n_in) : k - n_before;
      wanted = max(1, min(wanted, n_in));
      const int chunk = (len + kThreads - 1) / kThreads, i0 = min(len, tid * chunk), i1 = min(len, i0 + chunk);
      int mine = 0;
      for (int i = i0; i < i1; ++i) mine += ordered(xs[i]) == lo && kept(xs[i], i);
      int run = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, run, o);
        if (lane >= o) run += y;
      }
      __syncthreads();
      if (lane == 31) sh.counts[warp] = run;
      __syncthreads();
      int before = run - mine, all = 0;
      for (int i = 0; i < kWarps; ++i) {
        if (i < warp) before += sh.counts[i];
        all += sh.counts[i];
      }
      tell((uint32_t)all, 0, 0, 0);
      for (int r = 0; r < (int)rank; ++r) before += heard(0, r);
      if (before < wanted && before + mine >= wanted) {
        int n = before, i = i0;
        for (;; ++i)
          if (ordered(xs[i]) == lo && kept(xs[i], i) && ++n == wanted) break;
        for (int r = 0; r < kCluster; ++r) peer_store(&sh.cut_index, r, (uint32_t)(v0 + i));
      }
      cluster_sync();
      cut = lo;
      cut_index = sh.cut_index;
    }
    cluster_sync();  // what the CTAs told one another here is read
  }

  // The race over what is kept: the best of four tokens at a time, and in the end
  // which of a thread's best four it was.
  float best = 0.0f, part = 0.0f;
  int at = -1;
  if (plain && a.noise_vec) {
#pragma unroll 2
    for (int i = tid * 4; i < len; i += kThreads * 4) {
      const float4 x = *reinterpret_cast<const float4 *>(xs + i);
      float4 e = make_float4(1.0f, 1.0f, 1.0f, 1.0f);
      if (i + 4 <= len) {
        e = __ldg(reinterpret_cast<const float4 *>(noise + i));
      } else {
        e.x = __ldg(noise + i);
        if (i + 1 < len) e.y = __ldg(noise + i + 1);
        if (i + 2 < len) e.z = __ldg(noise + i + 2);
      }
      const float w[4] = {pow2(-depth(x.x)), pow2(-depth(x.y)), pow2(-depth(x.z)), pow2(-depth(x.w))};
      part += (w[0] + w[1]) + (w[2] + w[3]);
      const float v = fmaxf(fmaxf(__fdividef(w[0], e.x), __fdividef(w[1], e.y)),
                            fmaxf(__fdividef(w[2], e.z), __fdividef(w[3], e.w)));
      if (v > best) {
        best = v;
        at = i;
      }
    }
  } else {
    const float deep = least > 0.0f ? -log2f(least) : INFINITY;
    const float bound = fmaxf(fmaxf(cut ? unordered(cut) : kLowest, largest - deep / per * 1.0001f - fabsf(largest) * 1e-6f),
                              kLowest);
    for_above(bound, [&](float x, int i) {
      const float w = pow2(-depth(x));
      if (w < least || !kept(x, i)) return;
      part += w;
      const float v = __fdividef(w, __ldg(noise + i));
      if (v > best) {
        best = v;
        at = i & ~3;
      }
    });
  }
  Best pick{0.0f, top.i};
  float pick_x = largest;
  if (at >= 0) {
    pick = Best{-1.0f, 0};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = at + j;
      const float x = i < len ? xs[i] : -INFINITY, w = pow2(-depth(x));
      if (x == -INFINITY || w < least || !kept(x, i)) continue;
      const float v = __fdividef(w, __ldg(noise + i));
      if (v > pick.v) {
        pick = Best{v, v0 + i};
        pick_x = x;
      }
    }
  }
  const double mine_s = block_sum((double)part);
  const Best mine = pick;
  pick = block_best(pick);
  if (mine.i == pick.i) sh.pick_x = pick_x;
  __syncthreads();
  const unsigned long long bits = __double_as_longlong(mine_s);
  if (tid < kCluster) peer_store(&sh.list[rank], tid, bits);
  tell(__float_as_uint(pick.v), (uint32_t)pick.i, __float_as_uint(sh.pick_x), 0);
  pick = best_of_all();
  if (rank == 0 && tid == 0) {
    double s = 0.0;
    float x = 0.0f;
    for (int r = 0; r < kCluster; ++r) {
      s += __longlong_as_double(sh.list[r]);
      if ((int)heard(1, r) == pick.i) x = __uint_as_float(heard(2, r));
    }
    answer(pick.i, x, s);
  }
}

template <typename T>
int run_sample(const SampleArgs &a, size_t batch, cudaStream_t s) {
  {
    static std::mutex mu;
    static std::vector<int> done;
    int dev = 0;
    FPB_CUDA_TRY(cudaGetDevice(&dev));
    std::lock_guard<std::mutex> lock(mu);
    if (std::find(done.begin(), done.end(), dev) == done.end()) {
      FPB_CUDA_TRY(cudaFuncSetAttribute(sample_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        (int)(kMaxSlice * sizeof(float))));
      done.push_back(dev);
    }
  }
  cudaError_t e = launch_pdl_cluster(sample_kernel<T>, dim3(kCluster, (unsigned)batch), kThreads,
                                     (size_t)a.slice * sizeof(float), s, kCluster, a);
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
  if (batch == 0 || batch > 65535 || vocab == 0 || vocab > (size_t)kMaxSlice * kCluster || logits_pitch < vocab || noise_pitch < vocab ||
      (logits_pitch | noise_pitch) >> 38)
    return fail(FPB_ERR_SHAPE, "fpb_sample: batch %zu, vocab %zu (at most %d), pitches", batch, vocab, kMaxSlice * kCluster);
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
  a.slice = (int)((vocab + kCluster - 1) / kCluster + 7) / 8 * 8;
  auto lies = [](const void *p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && bytes % 16 == 0; };
  a.vec = lies(logits, logits_pitch * (logits_dtype == FPB_F32 ? 4 : 2));
  a.noise_vec = lies(noise, noise_pitch * 4);
  return logits_dtype == FPB_F32 ? run_sample<float>(a, batch, as_stream(stream))
                                 : run_sample<__nv_bfloat16>(a, batch, as_stream(stream));
}
