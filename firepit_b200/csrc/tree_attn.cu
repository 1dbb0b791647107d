// Attention of a tree of drafted tokens over the 8-bit cache (kv8.cuh).
//
// Node i of session b sees the cache rows before position[b], its ancestors'
// rows and its own (row position + j of node j).  With s_t = scale q . k_t:
//   out = sum_t softmax(s)_t v_t, times sigmoid(gate) where a gate is given.
#include <algorithm>
#include <cmath>

#include "kv8.cuh"

namespace fpb {
namespace {

struct TreeArgs {
  const void *q;
  const float *gate;
  const uint8_t *k_codes, *v_codes, *k_exp, *v_exp;
  const int32_t *positions, *parents;
  long long q_pitch, q_head, gate_pitch, gate_head;  // elements
  int nodes, q_heads, kv_heads, head_dim, max_seq, q_bf16;
  float scale;
  __nv_bfloat16 *out;
  int *error;
};

// One warp per (session, node, query head): eight columns a lane, the running
// maximum and sum of the softmax over the rows one by one.
__global__ void __launch_bounds__(256) tree_attn_kernel(const __grid_constant__ TreeArgs a) {
  pdl_enter();
  const int lane = threadIdx.x & 31, D = a.head_dim, c0 = lane * 8;
  const int h = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (h >= a.q_heads) return;
  const int b = blockIdx.y / a.nodes, n = blockIdx.y % a.nodes;
  const int kvh = h / (a.q_heads / a.kv_heads);
  const int32_t *par = a.parents ? a.parents + (size_t)b * a.nodes : nullptr;
  const int pos = a.positions[b];
  bool bad = false;
  int depth = tree_depth(par, n, &bad);
  if (depth >= 0 && (pos < 0 || pos >= a.max_seq - n)) {
    depth = -1;
    if (a.error) atomicCAS(a.error, 0, kErrPosition);
  }
  if (bad && a.error) atomicCAS(a.error, 0, kErrParent);
  float q[8], acc[8];
  const size_t row = (size_t)b * a.nodes + n;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const size_t at = row * a.q_pitch + (size_t)h * a.q_head + c0 + i;
    q[i] = c0 >= D ? 0.0f
           : a.q_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16 *>(a.q)[at])
                      : static_cast<const float *>(a.q)[at];
    acc[i] = 0.0f;
  }
  float m = -INFINITY, l = 0.0f;
  auto visit = [&](int t) {
    const size_t vec = ((size_t)b * a.max_seq + t) * a.kv_heads + kvh;
    uint2 kw = make_uint2(0, 0), vw = make_uint2(0, 0);
    if (c0 < D) {
      kw = *reinterpret_cast<const uint2 *>(a.k_codes + vec * D + c0);
      vw = *reinterpret_cast<const uint2 *>(a.v_codes + vec * D + c0);
    }
    const uint64_t k8 = (uint64_t)kw.y << 32 | kw.x, v8 = (uint64_t)vw.y << 32 | vw.x;
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s = fmaf(q[i], e4m3_to_f32((uint8_t)(k8 >> (8 * i))), s);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    s *= kv8_factor(a.k_exp[vec]) * a.scale;
    const float mn = fmaxf(m, s), old = m == -INFINITY ? 0.0f : expf(m - mn), p = expf(s - mn);
    const float f = p * kv8_factor(a.v_exp[vec]);
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = fmaf(f, e4m3_to_f32((uint8_t)(v8 >> (8 * i))), acc[i] * old);
    l = l * old + p;
    m = mn;
  };
  if (depth >= 0) {
    for (int t = 0; t < pos; ++t) visit(t);
    if (par)
      for (int j = n; j >= 0; j = par[j]) visit(pos + j);
    else
      for (int j = 0; j <= n; ++j) visit(pos + j);
  }
  if (c0 >= D) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float o = depth >= 0 ? acc[i] / l : 0.0f;
    if (a.gate && depth >= 0)
      o /= 1.0f + expf(-a.gate[row * a.gate_pitch + (size_t)h * a.gate_head + c0 + i]);
    a.out[(row * a.q_heads + h) * D + c0 + i] = __float2bfloat16_rn(o);
  }
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace fpb

using namespace fpb;

extern "C" size_t fpb_tree_attn_workspace_bytes(size_t batch, size_t nodes, size_t q_heads, size_t kv_heads,
                                                size_t head_dim, size_t max_seq) {
  (void)batch, (void)nodes, (void)q_heads, (void)kv_heads, (void)head_dim, (void)max_seq;
  return 16;
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
  a.nodes = (int)nodes;
  a.q_heads = (int)q_heads;
  a.kv_heads = (int)kv_heads;
  a.head_dim = (int)head_dim;
  a.max_seq = (int)max_seq;
  a.q_bf16 = q_dtype == FPB_BF16;
  a.scale = scale;
  a.out = static_cast<__nv_bfloat16 *>(out_bf16);
  a.error = device_error_ptr();
  cudaError_t e = launch_pdl(tree_attn_kernel, dim3((unsigned)((q_heads + 7) / 8), (unsigned)(batch * nodes)), 256, 0,
                             as_stream(stream), a);
  if (e != cudaSuccess) return cuda_fail(e, "tree_attn_kernel");
  FPB_LAUNCH_CHECK("tree_attn_kernel");
  return FPB_OK;
}
