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

struct VerifyArgs {
  const void *logits;
  const float *draft, *accept, *noise;
  const int32_t *tokens, *parents;
  long long logits_pitch, draft_pitch, noise_pitch;  // elements between rows
  int nodes, vocab, slice;
  float temperature;
  int32_t *path, *count, *next;
  int *error;
};

struct Best {
  float v;
  int i;
};
__device__ __forceinline__ Best better(Best a, Best b) { return b.v > a.v || (b.v == a.v && b.i < a.i) ? b : a; }

__device__ __forceinline__ int dsmem_load_int(const int *p, unsigned rank) {
  return __float_as_int(dsmem_load(reinterpret_cast<const float *>(p), rank));
}

// Block (cluster of kVerifyCluster CTAs) per session: CTA `rank` owns the
// vocabulary's slice [rank * slice, +slice) and keeps what is left of the
// node's distribution there in shared memory, so that a refused child's pass
// over the vocabulary does not go to memory for it again, and rows of nodes
// off the path are never read.  Every CTA takes the same walk: the values a
// decision needs come through distributed shared memory.
template <typename T>
__global__ void __launch_bounds__(kVerifyThreads) tree_verify_kernel(const __grid_constant__ VerifyArgs a) {
  pdl_enter();
  extern __shared__ float r[];  // [slice]: exp(l / T - max), or what is left of it
  __shared__ int par[kTreeMaxNodes], tok[kTreeMaxNodes], refused[kTreeMaxNodes];
  __shared__ float acc[kTreeMaxNodes], red[kVerifyWarps], out_v[2];
  __shared__ int red_i[kVerifyWarps], out_i[2];
  const unsigned rank = cluster_ctarank(), ctas = cluster_nctarank();
  const int b = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int v0 = (int)rank * a.slice, len = max(0, min(a.vocab - v0, a.slice));
  for (int i = tid; i < a.nodes; i += kVerifyThreads) {
    par[i] = a.parents ? a.parents[(size_t)b * a.nodes + i] : i - 1;
    tok[i] = a.tokens[(size_t)b * a.nodes + i];
    acc[i] = a.accept ? a.accept[(size_t)b * a.nodes + i] : 0.0f;
    if (rank == 0) a.path[(size_t)b * a.nodes + i] = -1;
    if (rank == 0 && a.error && i > 0 && par[i] >= i) atomicCAS(a.error, 0, kErrParent);
  }
  __syncthreads();
  if (par[0] != -1) {  // no tree in this session
    if (rank == 0 && tid == 0) {
      a.count[b] = 0;
      a.next[b] = -1;
    }
    return;
  }
  int flip = 0;
  // Sum, or best, over the cluster; the slots alternate, so that one round's
  // reads may overlap the next round's write.
  auto cluster_sum = [&](float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if (lane == 0) red[warp] = v;
    __syncthreads();
    if (tid == 0) {
      float t = 0.0f;
      for (int w = 0; w < kVerifyWarps; ++w) t += red[w];
      out_v[flip] = t;
    }
    cluster_sync();
    float t = 0.0f;
    for (unsigned c = 0; c < ctas; ++c) t += dsmem_load(&out_v[flip], c);
    flip ^= 1;
    return t;
  };
  auto cluster_best = [&](Best x) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      Best y{__shfl_xor_sync(0xffffffffu, x.v, o), __shfl_xor_sync(0xffffffffu, x.i, o)};
      x = better(x, y);
    }
    __syncthreads();
    if (lane == 0) {
      red[warp] = x.v;
      red_i[warp] = x.i;
    }
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < kVerifyWarps; ++w) x = better(x, Best{red[w], red_i[w]});
      out_v[flip] = x.v;
      out_i[flip] = x.i;
    }
    cluster_sync();
    Best t{-INFINITY, 0x7fffffff};
    for (unsigned c = 0; c < ctas; ++c)
      t = better(t, Best{dsmem_load(&out_v[flip], c), dsmem_load_int(&out_i[flip], c)});
    flip ^= 1;
    return t;
  };
  const bool greedy = a.temperature == 0.0f;
  int node = 0, taken = 0, next = 0;
  while (true) {
    if (rank == 0 && tid == 0) a.path[(size_t)b * a.nodes + taken] = node;
    ++taken;
    // the node's row: maximum (of finite logits), then exponentials and their sum
    const T *row = static_cast<const T *>(a.logits) + ((size_t)b * a.nodes + node) * a.logits_pitch + v0;
    Best top{-INFINITY, 0x7fffffff};
    for (int i = tid; i < len; i += kVerifyThreads) {
      const float l = static_cast<float>(row[i]);
      const float x = isfinite(l) ? l : -INFINITY;
      if (!greedy) r[i] = x / a.temperature;
      if (x > top.v) top = Best{x, v0 + i};
    }
    top = cluster_best(top);
    float left = 0.0f;
    if (!greedy) {
      const float m = top.v / a.temperature;
      float s = 0.0f;
      for (int i = tid; i < len; i += kVerifyThreads) {
        const float e = r[i] == -INFINITY ? 0.0f : expf(r[i] - m);
        r[i] = e;
        s += e;
      }
      left = cluster_sum(s);
    }
    int child = -1, rejected = 0;
    const float *q = a.draft ? a.draft + ((size_t)b * a.nodes + node) * a.draft_pitch : nullptr;
    for (int c = node + 1; c < a.nodes; ++c) {
      if (par[c] != node) continue;
      const int x = tok[c];
      if (x < 0 || x >= a.vocab) {
        if (rank == 0 && tid == 0 && a.error) atomicCAS(a.error, 0, kErrToken);
        continue;
      }
      if (greedy) {
        if (x == top.i) {
          child = c;
          break;
        }
        continue;
      }
      float rx = dsmem_load(&r[x % a.slice], (unsigned)(x / a.slice));
      if (q) {
        if (acc[c] * q[x] * left < rx) {
          child = c;
          break;
        }
        cluster_sync();  // every CTA has read rx
        const float inv = 1.0f / left;
        float s = 0.0f;
        for (int i = tid; i < len; i += kVerifyThreads) s += fmaxf(r[i] * inv - q[v0 + i], 0.0f);
        s = cluster_sum(s);
        if (s > 0.0f) {  // else the draft covers all that was left: it stays
          for (int i = tid; i < len; i += kVerifyThreads) r[i] = fmaxf(r[i] * inv - q[v0 + i], 0.0f);
          left = s;
          cluster_sync();  // the new values are there for the next child
        }
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
      cluster_sync();  // reads of r are done before the next row overwrites it
      node = child;
      continue;
    }
    if (greedy) {
      next = top.i == 0x7fffffff ? 0 : top.i;
      break;
    }
    cluster_sync();
    for (int j = tid; j < rejected; j += kVerifyThreads)
      if (refused[j] >= v0 && refused[j] < v0 + len) r[refused[j] - v0] = 0.0f;
    __syncthreads();
    Best pick{-1.0f, 0x7fffffff};
    const float *e = a.noise + (size_t)b * a.noise_pitch + v0;
    for (int i = tid; i < len; i += kVerifyThreads) {
      const float w = r[i] / e[i];
      if (w > pick.v) pick = Best{w, v0 + i};
    }
    pick = cluster_best(pick);
    next = pick.i == 0x7fffffff ? 0 : pick.i;
    break;
  }
  if (rank == 0 && tid == 0) {
    a.count[b] = taken;
    a.next[b] = next;
  }
  cluster_sync();  // no CTA leaves while its slots may still be read
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
  a.temperature = temperature;
  a.path = path;
  a.count = count;
  a.next = next;
  a.error = device_error_ptr();
  const size_t smem = greedy ? 0 : (size_t)a.slice * sizeof(float);
  return logits_dtype == FPB_F32 ? run_verify<float>(a, batch, smem, as_stream(stream))
                                 : run_verify<__nv_bfloat16>(a, batch, smem, as_stream(stream));
}
