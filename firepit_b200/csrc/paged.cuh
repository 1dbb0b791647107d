// The paged key/value cache, as the kernels that plan (paged.cu), write (kv8.cu)
// and read (paged_attn.cu) it agree on it.
//
// Token t of request b lies in row t % page_size of page table[b][t / page_size];
// its slot is page * page_size + row.
#pragma once
#include "common.cuh"

namespace fpb {

// Where a slot's head vectors lie, in elements from the first page's.
struct PageShape {
  int pages, page_size;
  long long page_pitch, row_pitch, head_pitch;
};

// Device error codes of these operators (fpb_device_error).
constexpr int kErrPage = 506, kErrLength = 507;

inline bool aligned_to(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// Checks of the pages that every entry point makes; `el` bytes an element.
inline int check_pages(const char *name, const void *k, const void *v, int dtype, size_t pages, size_t page_size,
                       size_t page_pitch, size_t row_pitch, size_t head_pitch, size_t kv_heads, size_t head_dim) {
  if (!k || !v) return fail(FPB_ERR_INVALID_ARGUMENT, "%s: null pages", name);
  if (dtype != FPB_F32 && dtype != FPB_BF16) return fail(FPB_ERR_INVALID_ARGUMENT, "%s: dtype of the pages", name);
  const size_t el = dtype == FPB_F32 ? 4 : 2;
  if (pages == 0 || page_size == 0 || pages > 0x7fffffffu / page_size || kv_heads == 0 || kv_heads > 4096 ||
      head_dim == 0 || head_dim > 256 || head_dim % 16)
    return fail(FPB_ERR_SHAPE, "%s: pages (%zu x %zu rows, fewer than 2^31; kv_heads %zu; head_dim %zu: a multiple of "
                "16 up to 256)", name, pages, page_size, kv_heads, head_dim);
  if (head_pitch < head_dim || row_pitch < head_dim || page_pitch < head_dim ||
      (head_pitch | row_pitch | page_pitch) >> 38)
    return fail(FPB_ERR_SHAPE, "%s: pitches of the pages", name);
  if (!aligned_to(k, 16) || !aligned_to(v, 16) || (head_pitch | row_pitch | page_pitch) * el % 16)
    return fail(FPB_ERR_INVALID_ARGUMENT, "%s: pages and their pitches have to lie on 16 bytes", name);
  return FPB_OK;
}

}  // namespace fpb
