// Host-side helpers shared by the tensor-core GEMMs (defined in gemm_nvfp4.cu).
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <cstddef>
#include <cstdint>

namespace fpb {
// 2-D byte tensor [rows, row_bytes] read in boxes of 128 bytes x box_rows with
// 128-byte swizzle; out-of-range elements read as zero.  FPB status.
int encode_rows_u8(CUtensorMap *map, const void *base, uint64_t rows, uint64_t row_bytes, uint32_t box_rows);

// 8-bit cache codes [batch, max_seq, kv_heads, head_dim] read in boxes of
// box_bytes (64 or 128, swizzled over as many) x 1 head x box_rows tokens;
// out-of-range elements read as zero.  FPB status.
int encode_cache_u8(CUtensorMap *map, const void *base, uint64_t batch, uint64_t max_seq, uint64_t kv_heads,
                    uint64_t head_dim, uint32_t box_bytes, uint32_t box_rows);

// Pages of a cache [pages, page_size, kv_heads, head_dim] bf16 or f32 (pitches in
// elements) as (column, row, piece, head, page), read in boxes of 128 bytes x
// box_rows tokens x `pieces` 128-byte pieces of a head vector x 1 head with 128-byte
// swizzle; out-of-range elements read as zero.  pieces 1: head_dim columns and one
// piece; else head_dim is whole pieces.  FPB status.
int encode_pages(CUtensorMap *map, const void *base, bool bf16, uint64_t head_dim, uint64_t kv_heads,
                 uint64_t page_size, uint64_t pages, uint64_t head_pitch, uint64_t row_pitch, uint64_t page_pitch,
                 uint32_t box_rows, uint32_t pieces);

// Output map for the GEMM epilogues' tiled stores: y [rows, cols] (bf16 or
// f32, row pitch ld elements), boxes of box_cols x box_rows (box_cols 0: 128
// bytes); 128-byte boxes use the 128-byte swizzle, narrower ones none.
// Returns false (no error recorded) when y cannot be stored that way (base or
// pitch not 16-byte aligned); the caller then stores directly.
bool encode_store_map(CUtensorMap *map, void *y, bool bf16, uint64_t rows, uint64_t cols, uint64_t ld,
                      uint32_t box_rows, uint32_t box_cols);

// A GEMM on bf16 operands through the persistent tcgen05 kernel's bf16 mode:
// y [m, n] = b_globals[n] * sum over passes j of A_{a_sel[j]} . B_{b_sel[j]}^T
// (A [m, k], B [n, k] bf16 row-major, k % 8 == 0; b_globals null = 1).
struct F16Gemm {
  size_t m, n, k;
  const void *a[2];
  const void *b[2];
  int passes;
  int a_sel[3], b_sel[3];
  const float *b_globals;
  void *y;
  int y_bf16;
};
int run_f16_gemm(const F16Gemm &g, cudaStream_t s);
// Activations of the bf16 mode (bf16 x in place; f32 x split into bf16 hi
// and lo in `ws`, `used` bytes) and the workspace that split needs.
int hilo_activations(const void *x, int x_dtype, size_t m, size_t k, uint8_t *ws, const void **hi,
                     const void **lo, size_t *used, cudaStream_t s);
size_t hilo_workspace_bytes(size_t m, size_t k, int x_dtype);
}  // namespace fpb
