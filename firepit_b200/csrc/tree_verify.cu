// Verification of a tree of drafted tokens against the target's
// probabilities, from given random numbers.
//
// The walk starts at node 0.  At a node with logits l, r = softmax(l / T) is
// what the next token has to be distributed as.  The node's children are
// tried in order; child x with accept number u is taken when u < r(x) / q(x).
// Where it is refused, r becomes what the child leaves over:
//   drawn drafts (q the draft's probabilities)  r <- max(r - q, 0) / its sum
//   certain drafts (q = 1 at x)                 r(x) <- 0, then / its sum
// A taken child is the next node; where no child is taken the next token is
// argmax r(v) / noise(v) with exponential noise, which draws from r.  So each
// emitted token is distributed as the target's, whatever the drafts were.
// T = 0: a child is taken when it is the target's argmax.
#include <algorithm>
#include <cmath>
#include <mutex>
#include <vector>

#include "kv8.cuh"

namespace fpb {
namespace {

constexpr int kVerifyThreads = 512, kVerifyWarps = kVerifyThreads / 32, kVerifyCluster = 8;
constexpr int kVerifyMaxSlice = 55296;  // f32 of shared memory a CTA: 216 KB
constexpr int kBatch = 5;               // 16-byte loads a thread has under way
constexpr int kHold = 40;               // logits a thread keeps in registers between a slice's maximum and its powers

struct VerifyArgs {
  const void *logits;
  const float *draft, *accept, *noise;
  const int32_t *tokens, *parents;
  long long logits_pitch, draft_pitch, noise_pitch;  // elements between rows
  int nodes, vocab, slice, vec;  // vec: every row and slice begins on 16 bytes
  float scale_log2;  // log2(e) / temperature; 0: greedy
  int32_t *path, *count, *next;
  int *error;
};

struct Best {
  float v;
  int i;
};
__device__ __forceinline__ Best better(Best a, Best b) { return b.v > a.v || (b.v == a.v && b.i < a.i) ? b : a; }

// Stores v at this CTA's shared-memory address p, in cluster CTA `rank`.
__device__ __forceinline__ void dsmem_store(float *p, unsigned rank, float v) {
  unsigned local = (unsigned)__cvta_generic_to_shared(p), remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(rank));
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(remote), "f"(v) : "memory");
}

// Over the cluster, each lane holding CTA lane % 8's value (every lane gets the
// same bits: the pairs are added alike everywhere).
static_assert(kVerifyCluster == 8);
__device__ __forceinline__ float over_ctas_sum(float v) {
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ Best over_ctas_best(Best x) {
#pragma unroll
  for (int o = 4; o > 0; o >>= 1)
    x = better(x, Best{__shfl_xor_sync(0xffffffffu, x.v, o), __shfl_xor_sync(0xffffffffu, x.i, o)});
  return x;
}

__device__ __forceinline__ float pow2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Calls f(x, r) for every element x of row[0, len) with its r (read before and
// written back after where KEEP): loads in batches, shared memory 16 bytes at a
// time; the tail, and rows that do not begin on 16 bytes, element by element.
// The element's index is passed third.
template <bool KEEP, typename T, typename F>
__device__ __forceinline__ void for_row(const T *row, int len, bool vec, float *r, F f) {
  constexpr int N = 16 / sizeof(T);
  const int whole = vec ? len / N * N : 0;
  for (int i0 = threadIdx.x * N; i0 < whole; i0 += kBatch * kVerifyThreads * N) {
    uint4 v[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int i = i0 + k * kVerifyThreads * N;
      v[k] = i < whole ? __ldg(reinterpret_cast<const uint4 *>(row + i)) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int i = i0 + k * kVerifyThreads * N;
      if (i >= whole) break;
      const uint32_t w[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
      float x[N];
      if constexpr (N == 4) {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = __uint_as_float(w[j]);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          x[2 * j] = __uint_as_float(w[j] << 16);
          x[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
        }
      }
#pragma unroll
      for (int j = 0; j < N; j += 4) {
        float4 *at = reinterpret_cast<float4 *>(r + i + j);
        float4 y = r ? *at : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        f(x[j], y.x, i + j);
        f(x[j + 1], y.y, i + j + 1);
        f(x[j + 2], y.z, i + j + 2);
        f(x[j + 3], y.w, i + j + 3);
        if (KEEP && r) *at = y;
      }
    }
  }
  for (int i = whole + threadIdx.x; i < len; i += kVerifyThreads) {
    float y = r ? r[i] : 0.0f;
    f(static_cast<float>(row[i]), y, i);
    if (KEEP && r) r[i] = y;
  }
}

// `bytes` from p on (a row's slice, both multiples of 16) to L2.
__device__ __forceinline__ void to_l2(const void *p, int bytes) {
  if (bytes > 0) asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p), "r"(bytes) : "memory");
}

// Bytes: the visited nodes' logits once, once more per refused draft the draft's
// row, the noise.  Measured, 151936 tokens: 16 sessions x 9 drafts drawn, bf16
// logits, 33 to 39 us by its walks (83 MB at 2.1 to 2.5 TB/s), 8 x 32 tree 15 us,
// 2 x 5 greedy 14 to 16.  A step takes 4 us: maximum 1.6, powers 0.7, sums 0.3,
// the cluster's barrier 0.8, decisions 0.5; a greedy one 3.
// Block (cluster of kVerifyCluster CTAs) per session: CTA `rank` owns the
// vocabulary's slice [rank * slice, +slice) and keeps what is left of the
// node's distribution there in shared memory, so that a refused child's pass
// over the vocabulary does not go to memory for it again.  Every CTA takes the
// same walk: each pushes what a decision needs (its slice's maximum and sum,
// the children's weights that it owns) into every CTA's shared memory, and one
// cluster barrier a step makes it known.  The walk is bound by the latency of
// its steps: the rows that the next step may want (the children's logits, at
// the start the noise) are sent to L2 while the node's own is worked on.  (The
// node's draft row as well: 62 us instead of 59 where drafts are refused.)  Two
// CTAs an SM, since a cluster's eight have to lie in one part of the GPU: with
// one, 16 clusters do not run at once (16 sessions of 9 drafts, all taken,
// 151936 tokens: 79 us, with two 57).
template <typename T>
__global__ void __launch_bounds__(kVerifyThreads, 2) tree_verify_kernel(const __grid_constant__ VerifyArgs a) {
  pdl_enter();
  extern __shared__ __align__(16) float r[];  // [slice]: 2^((l - slice's maximum) scale), or what is left of it
  __shared__ int par[kTreeMaxNodes], tok[kTreeMaxNodes], owner[kTreeMaxNodes], refused[kTreeMaxNodes];
  __shared__ float acc[kTreeMaxNodes], q_tok[kTreeMaxNodes], red[kVerifyWarps], red2[kVerifyWarps];
  __shared__ int red_i[kVerifyWarps];
  // what the CTAs tell one another; the halves alternate, so that one step's
  // reads may overlap the next one's stores
  __shared__ float got_v[2][kVerifyCluster], got_i[2][kVerifyCluster], got_s[2][kVerifyCluster],
      got_r[2][kTreeMaxNodes];
  const unsigned rank = cluster_ctarank(), peer = threadIdx.x % kVerifyCluster;
  const int b = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int v0 = (int)rank * a.slice, len = max(0, min(a.vocab - v0, a.slice));
  const bool greedy = a.scale_log2 == 0.0f;
  auto logits_of = [&](int n) { return static_cast<const T *>(a.logits) + ((size_t)b * a.nodes + n) * a.logits_pitch + v0; };
  const float *noise = greedy ? nullptr : a.noise + (size_t)b * a.noise_pitch + v0;
  const int l_bytes = a.vec ? len * (int)sizeof(T) / 16 * 16 : 0, f_bytes = a.vec ? len / 4 * 16 : 0;
  for (int i = tid; i < a.nodes; i += kVerifyThreads) {
    const int p = a.parents ? a.parents[(size_t)b * a.nodes + i] : i - 1, x = a.tokens[(size_t)b * a.nodes + i];
    par[i] = p;
    tok[i] = x;
    owner[i] = x / a.slice;
    acc[i] = a.accept ? a.accept[(size_t)b * a.nodes + i] : 0.0f;
    q_tok[i] = a.draft && p >= 0 && p < i && x >= 0 && x < a.vocab
                   ? a.draft[((size_t)b * a.nodes + p) * a.draft_pitch + x] : 1.0f;
    if (rank == 0) a.path[(size_t)b * a.nodes + i] = -1;
    if (rank == 0 && a.error && i > 0 && p >= i) atomicCAS(a.error, 0, kErrParent);
  }
  __syncthreads();
  if (par[0] != -1) {  // no tree in this session
    if (rank == 0 && tid == 0) {
      a.count[b] = 0;
      a.next[b] = -1;
    }
    return;
  }
  cluster_sync();  // every CTA of the cluster runs: its shared memory may be stored to
  if (tid == 0 && !greedy) to_l2(noise, f_bytes);
  int flip = 0;
  auto block_sum = [&](float v) {  // of the block, for every thread; all threads meet (and in `tell` before the next)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (lane == 0) red2[warp] = v;
    __syncthreads();
    float t = red2[lane % kVerifyWarps];
#pragma unroll
    for (int o = kVerifyWarps / 2; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    return t;
  };
  auto block_best = [&](Best x) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
      x = better(x, Best{__shfl_xor_sync(0xffffffffu, x.v, o), __shfl_xor_sync(0xffffffffu, x.i, o)});
    if (lane == 0) {
      red[warp] = x.v;
      red_i[warp] = x.i;
    }
    __syncthreads();
    x = Best{red[lane % kVerifyWarps], red_i[lane % kVerifyWarps]};
#pragma unroll
    for (int o = kVerifyWarps / 2; o > 0; o >>= 1)
      x = better(x, Best{__shfl_xor_sync(0xffffffffu, x.v, o), __shfl_xor_sync(0xffffffffu, x.i, o)});
    return x;
  };
  // To every CTA: this slice's maximum and sum, and of the children of `node`
  // past `from` the weights that lie here (thread (child, peer); r complete).
  auto tell = [&](int node, int from, Best top, float s) {
    if (tid < kVerifyCluster) {
      dsmem_store(&got_v[flip][rank], peer, top.v);
      dsmem_store(&got_i[flip][rank], peer, __int_as_float(top.i));
      dsmem_store(&got_s[flip][rank], peer, s);
    }
    const int c = tid / kVerifyCluster;
    if (!greedy && c > from && c < a.nodes && par[c] == node) {
      const int x = tok[c] - v0;
      if (x >= 0 && x < len) dsmem_store(&got_r[flip][c], peer, r[x]);
    }
    cluster_sync();
    flip ^= 1;
  };
  static_assert(kTreeMaxNodes * kVerifyCluster <= kVerifyThreads);
  int node = 0, taken = 0, next = 0;
  while (true) {
    if (rank == 0 && tid == 0) a.path[(size_t)b * a.nodes + taken] = node;
    ++taken;
    auto prefetch = [&]() {  // what the next step may want (by the last warp, with its own loads under way)
      if (!a.vec || warp != kVerifyWarps - 1) return;
      for (int c = node + 1 + lane; c < a.nodes; c += 32)
        if (par[c] == node) to_l2(logits_of(c), l_bytes);
    };
    // the slice's maximum (of finite logits), then powers by it and their sum
    Best top{-INFINITY, 0x7fffffff};
    float s = 0.0f;
    constexpr int N = 16 / sizeof(T), kLoads = kHold / N;
    // The slice is read at once, and stays in registers between the two, where it
    // fills at least half of them; else it is read in batches and goes through
    // shared memory (12 sessions, 9 drafts taken, f32: 96000 tokens 36 us in
    // registers, 41 else; 32000 29 and 28; greedy, 16 x 9 and 151936 40.5 and 42).
    constexpr int kAll = kHold * kVerifyThreads;
    if (a.vec && len % N == 0 && a.slice <= kAll && a.slice * 2 >= kAll) {
      const T *row = logits_of(node);
      uint4 v[kLoads];
      float m = -INFINITY;
#pragma unroll
      for (int k = 0; k < kLoads; ++k) {
        const int i = (k * kVerifyThreads + tid) * N;
        // past the slice: NaN, which counts as -inf
        v[k] = i < len ? __ldg(reinterpret_cast<const uint4 *>(row + i)) : make_uint4(~0u, ~0u, ~0u, ~0u);
      }
      prefetch();
      auto value = [&](int k, int j) {
        const uint32_t w = N == 4 ? (j == 0 ? v[k].x : j == 1 ? v[k].y : j == 2 ? v[k].z : v[k].w)
                                  : (j < 2 ? v[k].x : j < 4 ? v[k].y : j < 6 ? v[k].z : v[k].w);
        const float x = __uint_as_float(N == 4 ? w : j & 1 ? w & 0xffff0000u : w << 16);
        return fabsf(x) <= 3.402823466e38f ? x : -INFINITY;
      };
      if (greedy) {
#pragma unroll
        for (int k = 0; k < kLoads; ++k)
#pragma unroll
          for (int j = 0; j < N; ++j) {
            const float x = value(k, j);
            if (x > top.v) top = Best{x, v0 + (k * kVerifyThreads + tid) * N + j};
          }
      } else {
#pragma unroll
        for (int k = 0; k < kLoads; ++k)
#pragma unroll
          for (int j = 0; j < N; ++j) m = fmaxf(m, value(k, j));
        top.v = m;
      }
      top = block_best(top);
      const float bias = top.v == -INFINITY ? 0.0f : -top.v * a.scale_log2;
      if (!greedy) {
#pragma unroll
        for (int k = 0; k < kLoads; ++k) {
          const int i = (k * kVerifyThreads + tid) * N;
          if (i >= len) break;
#pragma unroll
          for (int j = 0; j < N; j += 4) {
            float4 e;
            e.x = pow2(fmaf(value(k, j), a.scale_log2, bias));
            e.y = pow2(fmaf(value(k, j + 1), a.scale_log2, bias));
            e.z = pow2(fmaf(value(k, j + 2), a.scale_log2, bias));
            e.w = pow2(fmaf(value(k, j + 3), a.scale_log2, bias));
            s += (e.x + e.y) + (e.z + e.w);
            *reinterpret_cast<float4 *>(r + i + j) = e;
          }
        }
        s = block_sum(s);
      }
    } else {
      prefetch();
      for_row<true>(logits_of(node), len, a.vec, greedy ? nullptr : r, [&](float x, float &y, int i) {
        y = isfinite(x) ? x : -INFINITY;
        if (y > top.v) top = Best{y, v0 + i};
      });
      top = block_best(top);
      if (!greedy) {
        const float bias = top.v == -INFINITY ? 0.0f : -top.v * a.scale_log2;
#pragma unroll 4
        for (int i = tid; i < len; i += kVerifyThreads) {
          const float e = pow2(fmaf(r[i], a.scale_log2, bias));
          r[i] = e;
          s += e;
        }
        s = block_sum(s);
      }
    }
    tell(node, node, top, s);
    // the slices' factors to one maximum, and the whole sum
    float left = 0.0f, factor = 0.0f;  // of CTA `peer`'s r
    const float mc = got_v[flip ^ 1][peer];
    const Best all = over_ctas_best(Best{mc, __float_as_int(got_i[flip ^ 1][peer])});
    if (!greedy) {
      factor = mc == -INFINITY ? 0.0f : pow2((mc - all.v) * a.scale_log2);
      left = over_ctas_sum(got_s[flip ^ 1][peer] * factor);
    }
    int child = -1, rejected = 0;
    const float *q = a.draft ? a.draft + ((size_t)b * a.nodes + node) * a.draft_pitch + v0 : nullptr;
    for (int c = node + 1; c < a.nodes; ++c) {
      if (par[c] != node) continue;
      const int x = tok[c];
      if (x < 0 || x >= a.vocab) {
        if (rank == 0 && tid == 0 && a.error) atomicCAS(a.error, 0, kErrToken);
        continue;
      }
      if (greedy) {
        if (x == all.i) {
          child = c;
          break;
        }
        continue;
      }
      float rx = fmaxf(got_r[flip ^ 1][c], 0.0f) * __shfl_sync(0xffffffffu, factor, owner[c]);
      if (q) {
        if (acc[c] * q_tok[c] * left < rx) {
          child = c;
          break;
        }
        // What is left over, with its sign: whoever reads r takes it as at
        // least 0, and what it was can be had back.
        const float inv = __shfl_sync(0xffffffffu, factor, rank) / left;
        float z = 0.0f;
        for_row<true>(q, len, a.vec, r, [&](float x, float &y, int) {
          y = fmaf(fmaxf(y, 0.0f), inv, -x);
          z += fmaxf(y, 0.0f);
        });
        tell(node, c, top, block_sum(z));
        z = over_ctas_sum(got_s[flip ^ 1][peer]);
        left = z;
        if (!(z > 0.0f)) {  // the draft covers all that was left: it stays
          for_row<true>(q, len, a.vec, r, [&](float x, float &y, int) { y += x; });
          __syncthreads();
          tell(node, c, top, 0.0f);
          left = 1.0f;
        }
        factor = 1.0f;
      } else {
        for (int j = 0; j < rejected; ++j)
          if (refused[j] == x) rx = 0.0f;
        if (acc[c] * left < rx) {
          child = c;
          break;
        }
        left -= rx;
        __syncthreads();  // the list's readers are done
        if (tid == 0) refused[rejected] = x;
        ++rejected;
        __syncthreads();
      }
    }
    if (child >= 0) {
      node = child;
      __syncthreads();  // r is read
      continue;
    }
    if (greedy) {
      next = all.i == 0x7fffffff ? 0 : all.i;
      break;
    }
    for (int j = tid; j < rejected; j += kVerifyThreads)
      if (refused[j] >= v0 && refused[j] < v0 + len) r[refused[j] - v0] = 0.0f;
    __syncthreads();
    Best pick{-1.0f, 0x7fffffff};
    const float own = __shfl_sync(0xffffffffu, factor, rank);
    for_row<false>(noise, len, a.vec, r, [&](float e, float &y, int i) {
      const float w = __fdividef(fmaxf(y, 0.0f) * own, e);
      if (w > pick.v) pick = Best{w, v0 + i};
    });
    tell(a.nodes, a.nodes, block_best(pick), 0.0f);
    pick = over_ctas_best(Best{got_v[flip ^ 1][peer], __float_as_int(got_i[flip ^ 1][peer])});
    next = pick.i == 0x7fffffff ? 0 : pick.i;
    break;
  }
  // (nothing is stored to another CTA after its last barrier)
  if (rank == 0 && tid == 0) {
    a.count[b] = taken;
    a.next[b] = next;
  }
}

template <typename T>
int run_verify(const VerifyArgs &a, size_t batch, size_t smem, cudaStream_t s) {
  if (smem > 40 * 1024) {  // raised once a device, to the most any call needs
    static std::mutex mu;
    static std::vector<int> done;
    int dev = 0;
    FPB_CUDA_TRY(cudaGetDevice(&dev));
    std::lock_guard<std::mutex> lock(mu);
    if (std::find(done.begin(), done.end(), dev) == done.end()) {
      FPB_CUDA_TRY(cudaFuncSetAttribute(tree_verify_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        (int)(kVerifyMaxSlice * sizeof(float))));
      done.push_back(dev);
    }
  }
  cudaError_t e = launch_pdl_cluster(tree_verify_kernel<T>, dim3(kVerifyCluster, (unsigned)batch), kVerifyThreads,
                                     smem, s, kVerifyCluster, a);
  if (e != cudaSuccess) return cuda_fail(e, "tree_verify_kernel");
  FPB_LAUNCH_CHECK("tree_verify_kernel");
  return FPB_OK;
}

}  // namespace
}  // namespace fpb

using namespace fpb;

extern "C" int fpb_tree_verify(const void *logits, int logits_dtype, size_t logits_pitch, const float *draft,
                               size_t draft_pitch, const int32_t *tokens, const int32_t *parents,
                               const float *accept, const float *noise, size_t noise_pitch, size_t batch,
                               size_t nodes, size_t vocab, float temperature, int32_t *path, int32_t *count,
                               int32_t *next, void *stream) {
  if (!logits || !tokens || !path || !count || !next)
    return fail(FPB_ERR_INVALID_ARGUMENT, "fpb_tree_verify: null pointer");
  if (logits_dtype != FPB_F32 && logits_dtype != FPB_BF16)
    return fail(FPB_ERR_INVALID_ARGUMENT, "fpb_tree_verify: dtype");
  if (temperature != 0.0f && !(temperature >= 1e-6f && temperature <= 1e6f))
    return fail(FPB_ERR_INVALID_ARGUMENT, "fpb_tree_verify: temperature %g (0, or within [1e-6, 1e6])",
                (double)temperature);
  const bool greedy = temperature == 0.0f;
  if (!greedy && (!accept || !noise))
    return fail(FPB_ERR_INVALID_ARGUMENT, "fpb_tree_verify: a temperature above 0 needs accept and noise");
  if (batch == 0 || batch > 65535 || nodes == 0 || nodes > (size_t)kTreeMaxNodes || vocab == 0 ||
      logits_pitch < vocab || (!greedy && (noise_pitch < vocab || (draft && draft_pitch < vocab))))
    return fail(FPB_ERR_SHAPE, "fpb_tree_verify: batch %zu, nodes %zu (at most %d), vocab %zu, pitches", batch, nodes,
                kTreeMaxNodes, vocab);
  if (vocab > (size_t)kVerifyMaxSlice * kVerifyCluster)
    return fail(FPB_ERR_UNSUPPORTED, "fpb_tree_verify: vocab %zu > %d", vocab, kVerifyMaxSlice * kVerifyCluster);
  VerifyArgs a{};
  a.logits = logits;
  a.draft = greedy ? nullptr : draft;
  a.accept = greedy ? nullptr : accept;
  a.noise = noise;
  a.tokens = tokens;
  a.parents = parents;
  a.logits_pitch = (long long)logits_pitch;
  a.draft_pitch = (long long)draft_pitch;
  a.noise_pitch = (long long)noise_pitch;
  a.nodes = (int)nodes;
  a.vocab = (int)vocab;
  a.slice = (int)((vocab + kVerifyCluster - 1) / kVerifyCluster + 7) / 8 * 8;
  a.scale_log2 = greedy ? 0.0f : (float)(1.4426950408889634 / (double)temperature);
  a.path = path;
  a.count = count;
  a.next = next;
  a.error = device_error_ptr();
  const size_t el = logits_dtype == FPB_F32 ? 4 : 2;
  auto lies = [](const void *p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && bytes % 16 == 0; };
  a.vec = lies(logits, logits_pitch * el) && (greedy || lies(noise, noise_pitch * 4)) &&
          (!a.draft || lies(draft, draft_pitch * 4));
  const size_t smem = greedy ? 0 : (size_t)a.slice * sizeof(float);
  return logits_dtype == FPB_F32 ? run_verify<float>(a, batch, smem, as_stream(stream))
                                 : run_verify<__nv_bfloat16>(a, batch, smem, as_stream(stream));
}
