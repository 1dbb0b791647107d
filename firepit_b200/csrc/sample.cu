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

#include "common.cuh"

namespace fpb {
namespace {

constexpr int kSampleThreads = 1024, kSampleWarps = kSampleThreads / 32;

struct SampleArgs {
  const void *logits;
  const float *temperature, *top_p, *min_p, *noise;
  const int32_t *top_k;
  long long logits_pitch, noise_pitch;  // elements between rows
  int vocab;
  int32_t *tokens;
  float *logprobs;
};

// Order of f32 values as that of whole numbers (-inf above 0).
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

template <typename V>
__device__ __forceinline__ V block_sum(V v, V *red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if (lane == 0) red[warp] = v;
  __syncthreads();
  V t = red[lane];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  return t;
}

struct Pick {
  double v;
  int i;
};

__device__ __forceinline__ Pick block_best(Pick x, Pick *red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto meet = [&]() {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const double v = __shfl_xor_sync(0xffffffffu, x.v, o);
      const int i = __shfl_xor_sync(0xffffffffu, x.i, o);
      if (v > x.v || (v == x.v && i < x.i)) x = Pick{v, i};
    }
  };
  meet();
  __syncthreads();
  if (lane == 0) red[warp] = x;
  __syncthreads();
  x = red[lane];
  meet();
  return x;
}

// One block a row.  What is kept is {key above `key`} and, at `key`, the indices
// up to `last`; both are found bit by bit, a pass over the row each.
template <typename T>
__global__ void __launch_bounds__(kSampleThreads) sample_kernel(const __grid_constant__ SampleArgs a) {
  pdl_enter();
  __shared__ double red[kSampleWarps];
  __shared__ Pick red_p[kSampleWarps];
  const int b = blockIdx.x, tid = threadIdx.x;
  const T *row = static_cast<const T *>(a.logits) + (size_t)b * a.logits_pitch;
  const float *noise = a.noise + (size_t)b * a.noise_pitch;
  auto logit = [&](int i) {
    const float x = static_cast<float>(row[i]);
    return fabsf(x) <= 3.402823466e38f ? x : -INFINITY;
  };
  Pick top{-INFINITY, 0x7fffffff};
  for (int i = tid; i < a.vocab; i += kSampleThreads) {
    const float x = logit(i);
    if (x > top.v) top = Pick{x, i};
  }
  top = block_best(top, red_p);
  const float t = a.temperature ? a.temperature[b] : 1.0f;
  if (top.i == 0x7fffffff || !(t > 0.0f)) {
    if (tid == 0) {
      a.tokens[b] = top.i == 0x7fffffff ? -1 : top.i;
      if (a.logprobs) a.logprobs[b] = top.i == 0x7fffffff ? -INFINITY : 0.0f;
    }
    return;
  }
  const double inv = 1.0 / (double)fminf(fmaxf(t, 1e-6f), 1e6f), best = top.v;
  uint32_t key = ordered(-INFINITY);  // (not kept itself)
  int last = -1;
  auto weight = [&](float x) { return exp(((double)x - best) * inv); };
  auto kept = [&](float x, int i) {
    const uint32_t u = ordered(x);
    return u > key || (u == key && i <= last);
  };
  // Shortens what is kept to the first part whose sum of f reaches `target`.
  auto cut = [&](double target, auto f) {
    uint32_t k = 0;
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t trial = k | 1u << bit;
      double s = 0.0;
      for (int i = tid; i < a.vocab; i += kSampleThreads) {
        const float x = logit(i);
        if (ordered(x) >= trial && kept(x, i)) s += f(x);
      }
      if (block_sum(s, red) >= target) k = trial;
    }
    int lo = 0, hi = a.vocab - 1;  // the first index at which the sum is reached
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      double s = 0.0;
      for (int i = tid; i < a.vocab; i += kSampleThreads) {
        const float x = logit(i);
        const uint32_t u = ordered(x);
        if ((u > k || (u == k && i <= mid)) && kept(x, i)) s += f(x);
      }
      if (block_sum(s, red) >= target)
        hi = mid;
      else
        lo = mid + 1;
    }
    key = k;
    last = lo;
  };
  const int k = a.top_k ? a.top_k[b] : 0;
  if (k > 0 && k < a.vocab) {
    double n = 0.0;
    for (int i = tid; i < a.vocab; i += kSampleThreads) n += kept(logit(i), i);
    if (block_sum(n, red) > k) cut((double)k, [](float) { return 1.0; });
  }
  const float p = a.top_p ? a.top_p[b] : 1.0f;
  if (p < 1.0f) {
    double s = 0.0;
    for (int i = tid; i < a.vocab; i += kSampleThreads) {
      const float x = logit(i);
      if (kept(x, i)) s += weight(x);
    }
    s = block_sum(s, red);
    cut(fmax((double)p * s, 1e-300), weight);
  }
  const float m = a.min_p ? a.min_p[b] : 0.0f;
  const double floor_w = m > 0.0f ? (double)fminf(m, 1.0f) : 0.0;
  Pick pick{-INFINITY, 0x7fffffff};
  double s = 0.0;
  for (int i = tid; i < a.vocab; i += kSampleThreads) {
    const float x = logit(i);
    const double w = weight(x);
    if (!kept(x, i) || w < floor_w) continue;
    s += w;
    const double v = w / (double)noise[i];
    if (v > pick.v) pick = Pick{v, i};
  }
  s = block_sum(s, red);
  pick = block_best(pick, red_p);
  if (tid == 0) {
    a.tokens[b] = pick.i;
    if (a.logprobs) a.logprobs[b] = (float)(((double)logit(pick.i) - best) * inv - log(s));
  }
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
  if (batch == 0 || batch > 65535 || vocab == 0 || vocab > 442368 || logits_pitch < vocab || noise_pitch < vocab ||
      (logits_pitch | noise_pitch) >> 38)
    return fail(FPB_ERR_SHAPE, "fpb_sample: batch %zu, vocab %zu (at most 442368), pitches", batch, vocab);
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
  cudaError_t e = logits_dtype == FPB_F32
                      ? launch_pdl(sample_kernel<float>, (unsigned)batch, kSampleThreads, 0, as_stream(stream), a)
                      : launch_pdl(sample_kernel<__nv_bfloat16>, (unsigned)batch, kSampleThreads, 0, as_stream(stream), a);
  if (e != cudaSuccess) return cuda_fail(e, "sample_kernel");
  FPB_LAUNCH_CHECK("sample_kernel");
  return FPB_OK;
}
