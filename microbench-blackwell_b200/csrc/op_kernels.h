// op_kernels.h -- internal interface between the C entries of the operators around the
// linear layer (op_api.cu) and their kernels.  Not part of the public ABI.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace b2g {

// Microscaled casts (block_quant.cu).  in: rows x cols, ld_in elements apart.  codes /
// sf: one row of kp = cols rounded up to 32 elements per input row; codes_t / sf_t: one
// row of tp = rows rounded up to 32 per input column.  Either pair may be null.
struct BlockQuantArgs {
  const void* in;
  int64_t ld_in;
  int64_t rows, cols;
  int64_t kp, tp;
  uint8_t *codes, *sf;
  uint8_t *codes_t, *sf_t;
  const uint8_t* rand;  // rows x cols bytes, ld_rand apart; null: nearest even
  int64_t ld_rand;
  float scale;
  int in_vec;    // every row of `in` starts on 16 bytes
  int rand_vec;  // every row of `rand` starts on 8 bytes
};
// fmt: BlockFmt; type: b2g_dtype; pow2: scale is a power of two, 2^100 at most
cudaError_t launch_block_quant(int fmt, int type, bool pow2, const BlockQuantArgs& a,
                               cudaStream_t s);

struct BlockDequantArgs {
  const uint8_t *codes, *sf;
  int64_t rows, cols, kp;
  void* out;
  int64_t ld_out;
  float scale;
  int out_vec;  // every row of `out` starts on 16 bytes
};
cudaError_t launch_block_dequant(int fmt, int type, const BlockDequantArgs& a, cudaStream_t s);

// Norms around a block (residual_norm.cu).
struct ResidualNormArgs {
  int64_t rows, cols;
  const void *x, *y, *gate, *w_post, *w_pre;
  int64_t ld_x, ld_y, ld_x_out, ld_h;
  int64_t rows_per_gate;
  void *x_out, *h;
  uint8_t *codes, *sf;
  int64_t kp;
  float *rstd_post, *rstd_pre;
  float eps, alpha, beta;
  int vec;  // all rows of all 16- or 32-bit operands start on 16 bytes
};
constexpr int64_t kNormMaxCols = 32768;
// h_fmt: -1 none, else BlockFmt of codes / sf
cudaError_t launch_residual_norm(int type, int h_fmt, const ResidualNormArgs& a, int sm_count,
                                 cudaStream_t s);

struct ResidualNormGradArgs {
  int64_t rows, cols;
  const void *dh, *dx_out, *v, *y, *gate, *w_post, *w_pre;
  const float *rstd_post, *rstd_pre;
  int64_t ld_dh, ld_dx_out, ld_v, ld_y, ld_dx, ld_dy;
  int64_t rows_per_gate;
  void *dx, *dy;
  float *dgate, *dw_post, *dw_pre;
  float alpha, beta;
  int vec;        // as above
  int dgate_vec;  // dgate starts on 16 bytes
  uint32_t* err;  // the handle's error word
  void* ws;  // norm_grad_ws_bytes() bytes
};
size_t norm_grad_ws_bytes(int type, const ResidualNormGradArgs& a, int sm_count);
cudaError_t launch_residual_norm_grad(int type, const ResidualNormGradArgs& a, int sm_count,
                                      cudaStream_t s);

// Few-token product with microscaled weights (few_linear.cu).
constexpr int kFewMaxTokens = 65536;
constexpr int kFewMaxExtent = 1 << 24;  // N and K: indexes within a matrix's edge are 32 bits
constexpr int kFewTokens = 8;           // at most in few_linear.cu
// Bytes of x in a CTA there: with the warps' rings (up to 72 KB) and their sums (8 KB) two
// CTAs fit an SM.
constexpr int kFewXBytes = 32768;
struct FewLinearArgs {
  int64_t T, N, K, kp;
  const void* x;
  int64_t ld_x;
  const uint8_t *w, *sf;
  void* out;
  int64_t ld_out;
  float alpha;
  int x_vec;  // every row of `x` starts on 16 bytes
  void* ws;   // few_linear_ws_bytes() or few_tiles_ws_bytes() bytes
  uint32_t* count;  // ..._counters() words, zero before and after
  uint32_t* err;    // the handle's error word
  uint64_t wait_ns; // limit of bounded waits (0: default)
};
size_t few_linear_ws_bytes(int fmt, const FewLinearArgs& a, int sm_count);
size_t few_linear_counters(int fmt, const FewLinearArgs& a, int sm_count);
// Its tensor-core form (few_tiles.cu): map_w over the codes' bytes [N][row bytes], map_x over
// fp16 [T][x_cols] at the start of the workspace, boxes as few_tiles_maps() says, both with
// the 128-byte swizzle.
struct FewTilesMaps {
  uint64_t w_row_bytes, x_cols;
  uint32_t w_box_bytes, w_box_rows, x_box_cols, x_box_rows;
};
void few_tiles_maps(int fmt, const FewLinearArgs& a, int sm_count, FewTilesMaps* m);
size_t few_tiles_ws_bytes(int fmt, const FewLinearArgs& a, int sm_count);
size_t few_tiles_counters(int fmt, const FewLinearArgs& a, int sm_count);
cudaError_t launch_few_tiles(int fmt, int type, const FewLinearArgs& a, const CUtensorMap& map_w,
                             const CUtensorMap& map_x, int sm_count, cudaStream_t s);
cudaError_t launch_few_linear(int fmt, int type, const FewLinearArgs& a, int sm_count,
                              cudaStream_t s);

}  // namespace b2g
