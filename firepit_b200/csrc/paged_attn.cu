// Attention of one new token a session over the paged cache (paged.cuh).
//
// Session b's query heads see the tokens t < lengths[b].  With s_t = scale q . k_t:
//   out = sum_t softmax(s)_t v_t, times sigmoid(gate) where a gate is given.
#include <algorithm>
#include <cmath>

#include "paged.cuh"

namespace fpb {
namespace {

struct PagedArgs {
  const void *q, *k, *v;
  const float *gate;
  const int32_t *table, *lengths;
  long long q_pitch, q_head, gate_pitch, gate_head, table_pitch;  // elements
  PageShape page;
  int batch, q_heads, kv_heads, group, head_dim, max_pages, q_bf16;
  float scale_log2;  // scale * log2(e): scores and maxima are held in powers of two
  void *out;
  int out_bf16;
  int *error;
};

template <typename T>
__device__ __forceinline__ float value(const T *p, size_t i) {
  if constexpr (sizeof(T) == 4)
    return p[i];
  else
    return __bfloat162float(p[i]);
}

// One warp a query head: the tokens one by one, the maximum and sum running.
template <typename T>
__global__ void __launch_bounds__(128) paged_attn_kernel(const __grid_constant__ PagedArgs a) {
  pdl_enter();
  const int lane = threadIdx.x & 31, item = blockIdx.x * 4 + (threadIdx.x >> 5), D = a.head_dim;
  if (item >= a.batch * a.q_heads) return;
  const int b = item / a.q_heads, h = item % a.q_heads, kvh = h / a.group;
  int n = a.lengths[b];
  const long long most = (long long)a.max_pages * a.page.page_size;
  if (n < 0 || n > most) {
    if (lane == 0 && a.error) atomicCAS(a.error, 0, kErrLength);
    n = 0;
  }
  float q[8], acc[8], m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int d = lane + 32 * i;
    const size_t at = (size_t)b * a.q_pitch + (size_t)h * a.q_head + d;
    q[i] = d < D ? (a.q_bf16 ? value(static_cast<const __nv_bfloat16 *>(a.q), at) : value(static_cast<const float *>(a.q), at))
                 : 0.0f;
    acc[i] = 0.0f;
  }
  for (int t = 0; t < n; ++t) {
    const int p = t / a.page.page_size, page = a.table[b * a.table_pitch + p];
    if (page < 0 || page >= a.page.pages) {
      if (lane == 0 && a.error) atomicCAS(a.error, 0, kErrPage);
      continue;
    }
    const size_t at = page * a.page.page_pitch + (t - p * a.page.page_size) * a.page.row_pitch + kvh * a.page.head_pitch;
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (lane + 32 * i < D) s = fmaf(q[i], value(static_cast<const T *>(a.k), at + lane + 32 * i), s);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    s *= a.scale_log2;
    const float mn = fmaxf(m, s), old = m == -INFINITY ? 0.0f : exp2f(m - mn), w = exp2f(s - (mn == -INFINITY ? 0.0f : mn));
    m = mn;
    l = fmaf(l, old, w);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (lane + 32 * i < D) acc[i] = fmaf(acc[i], old, w * value(static_cast<const T *>(a.v), at + lane + 32 * i));
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int d = lane + 32 * i;
    if (d >= D) break;
    float o = l != 0.0f ? acc[i] / l : 0.0f;
    if (a.gate && n > 0) o /= 1.0f + expf(-a.gate[(size_t)b * a.gate_pitch + (size_t)h * a.gate_head + d]);
    const size_t at = ((size_t)b * a.q_heads + h) * D + d;
    if (a.out_bf16)
      static_cast<__nv_bfloat16 *>(a.out)[at] = __float2bfloat16_rn(o);
    else
      static_cast<float *>(a.out)[at] = o;
  }
}

}  // namespace
}  // namespace fpb

using namespace fpb;

extern "C" size_t fpb_paged_attn_workspace_bytes(size_t batch, size_t q_heads, size_t kv_heads, size_t head_dim) {
  (void)batch; (void)q_heads; (void)kv_heads; (void)head_dim;
  return 16;
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
  if (batch == 0 || batch > 16384 || q_heads == 0 || q_heads % kv_heads || q_heads > 65535 || max_pages == 0 ||
      max_pages > 0x7fffffffu / page_size || table_pitch < max_pages || table_pitch >> 38)
    return fail(FPB_ERR_SHAPE, "fpb_paged_attn: batch %zu (at most 16384), heads %zu / %zu, tables of %zu pages (pitch "
                "%zu)", batch, q_heads, kv_heads, max_pages, table_pitch);
  if (q_head_pitch < head_dim || (gate && gate_head_pitch < head_dim) || !std::isfinite(scale))
    return fail(FPB_ERR_SHAPE, "fpb_paged_attn: pitches or scale");
  if (!aligned_to(workspace, 16) || !aligned_to(out, 16) || !aligned_to(q, q_dtype == FPB_F32 ? 4 : 2) ||
      !aligned_to(gate, 4))
    return fail(FPB_ERR_INVALID_ARGUMENT, "fpb_paged_attn: alignment (workspace and out: 16 bytes)");
  const size_t need = fpb_paged_attn_workspace_bytes(batch, q_heads, kv_heads, head_dim);
  if (workspace_bytes < need)
    return fail(FPB_ERR_WORKSPACE, "fpb_paged_attn: workspace %zu < %zu bytes", workspace_bytes, need);
  PagedArgs a{};
  a.q = q;
  a.k = k_pages;
  a.v = v_pages;
  a.gate = gate;
  a.table = table;
  a.lengths = lengths;
  a.q_pitch = (long long)q_pitch;
  a.q_head = (long long)q_head_pitch;
  a.gate_pitch = (long long)gate_pitch;
  a.gate_head = (long long)gate_head_pitch;
  a.table_pitch = (long long)table_pitch;
  a.page = PageShape{(int)pages, (int)page_size, (long long)page_pitch, (long long)row_pitch, (long long)head_pitch};
  a.batch = (int)batch;
  a.q_heads = (int)q_heads;
  a.kv_heads = (int)kv_heads;
  a.group = (int)(q_heads / kv_heads);
  a.head_dim = (int)head_dim;
  a.max_pages = (int)max_pages;
  a.q_bf16 = q_dtype == FPB_BF16;
  a.scale_log2 = (float)((double)scale * 1.4426950408889634);
  a.out = out;
  a.out_bf16 = out_dtype == FPB_BF16;
  a.error = device_error_ptr();
  const unsigned blocks = (unsigned)((batch * q_heads + 3) / 4);
  cudaError_t e = page_dtype == FPB_F32 ? launch_pdl(paged_attn_kernel<float>, blocks, 128, 0, as_stream(stream), a)
                                        : launch_pdl(paged_attn_kernel<__nv_bfloat16>, blocks, 128, 0, as_stream(stream), a);
  if (e != cudaSuccess) return cuda_fail(e, "paged_attn_kernel");
  FPB_LAUNCH_CHECK("paged_attn_kernel");
  return FPB_OK;
}
