// op_api.cu -- C entries of the operators around the linear layer (declared in
// include/b2g.h): checks of arguments, workspaces and dispatch.
#include <cuda_runtime.h>
#include <string.h>

#include "b2g.h"
#include "b2g_handle.h"
#include "op_common.cuh"
#include "op_kernels.h"

using namespace b2g;

namespace {

bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

size_t type_bytes(int type) { return type == B2G_F32 ? 4 : 2; }

bool type_ok(int type) { return type == B2G_F32 || type == B2G_BF16 || type == B2G_F16; }

// Formats with one scale per block, as BlockFmt; -1 for the others.
int block_fmt(int format) {
  switch (format) {
    case B2G_FMT_NVFP4: return BF_NVFP4;
    case B2G_FMT_MXF4: return BF_MXF4;
    case B2G_FMT_MXF8: return BF_MXF8;
    default: return -1;
  }
}

int64_t up32(int64_t n) { return (n + 31) / 32 * 32; }

// Sizes a call may have: no product of two of them leaves int64.
constexpr int64_t kMaxExtent = int64_t(1) << 31;

// A row-major operand: element-aligned, rows no closer than their extent.
bool matrix_ok(const void* p, int type, int64_t cols, int64_t ld) {
  return p && aligned(p, type_bytes(type)) && ld >= cols && ld < kMaxExtent;
}

// Whether every row starts on `bytes` bytes.
bool rows_aligned(const void* p, int64_t ld, size_t elem, size_t bytes) {
  return aligned(p, bytes) && ((size_t)ld * elem) % bytes == 0;
}

// 128-byte swizzled map of a row-major matrix whose rows follow one another.
b2g_status tensor_map(b2g_handle* h, CUtensorMap* map, CUtensorMapDataType type, int elem,
                      const void* base, uint64_t cols, uint64_t rows, uint32_t box_cols,
                      uint32_t box_rows) {
  const cuuint64_t dims[2] = {cols, rows}, strides[1] = {cols * (uint64_t)elem};
  const cuuint32_t box[2] = {box_cols, box_rows}, one[2] = {1, 1};
  const CUresult r = h->encode_tiled(map, type, 2, const_cast<void*>(base), dims, strides, box, one,
                                     CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                     CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(h, B2G_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d) dims=%llu x %llu", (int)r,
                (unsigned long long)cols, (unsigned long long)rows);
  return B2G_OK;
}

// b2g_linear's form.  Nine tokens and more (the other one's limit is eight) take the tensor
// cores' (few_tiles.cu), fewer the registers' (few_linear.cu) unless x does not fit one CTA and
// the weights are many.  Measured (us, registers / tensor cores, 8 tokens): all of x in a CTA
// 2048 x 2048 4.8 / 7.5, 16384 x 2048 8.2 / 9.7; beyond, 2048 x 8192 9.3 / 10.4, 8192 x 8192
// 17.5 / 16.4, 16384 x 8192 29.2 / 22.6 (NVFP4), 8192 x 8192 22.8 / 21.8 (MXFP8).
bool linear_tiles(const FewLinearArgs& a) {
  return a.T > kFewTokens || (2 * a.T * a.kp > kFewXBytes && a.N * a.kp >= (int64_t)1 << 26);
}

}  // namespace

extern "C" {

b2g_status b2g_block_quantize(b2g_handle* h, const b2g_block_quant_desc* d, void* stream) {
  if (!h || !d) return B2G_ERR_INVALID;
  h->last_error[0] = 0;
  const int fmt = block_fmt(d->format);
  if (fmt < 0)
    return fail(h, B2G_ERR_UNSUPPORTED, "b2g_block_quantize: format %d (NVFP4, MXFP4 or MXFP8)",
                d->format);
  if (!type_ok(d->in_type)) return fail(h, B2G_ERR_INVALID, "b2g_block_quantize: in_type %d", d->in_type);
  if (d->rows < 0 || d->cols < 0 || d->rows >= kMaxExtent || d->cols >= kMaxExtent)
    return fail(h, B2G_ERR_INVALID, "b2g_block_quantize: rows or cols out of range");
  if (!(d->scale > 0.0f) || d->scale > 3.0e38f)
    return fail(h, B2G_ERR_INVALID, "b2g_block_quantize: scale must be positive and finite");
  if (d->rows == 0 || d->cols == 0) return B2G_OK;  // pointers of empty buffers may be null
  if ((d->codes == nullptr) != (d->sf == nullptr) || (d->codes_t == nullptr) != (d->sf_t == nullptr))
    return fail(h, B2G_ERR_INVALID, "b2g_block_quantize: codes need their scales");
  if (!d->codes && !d->codes_t) return fail(h, B2G_ERR_INVALID, "b2g_block_quantize: no output");
  if (!matrix_ok(d->in, d->in_type, d->cols, d->ld_in))
    return fail(h, B2G_ERR_INVALID, "b2g_block_quantize: input null, misaligned or ld_in < cols");
  if (d->rand && (d->ld_rand < d->cols || d->ld_rand >= kMaxExtent))
    return fail(h, B2G_ERR_INVALID, "b2g_block_quantize: ld_rand < cols");
  if (!aligned(d->codes, 16) || !aligned(d->codes_t, 16))
    return fail(h, B2G_ERR_INVALID, "b2g_block_quantize: codes must be 16-byte aligned");
  BlockQuantArgs a;
  memset(&a, 0, sizeof(a));
  const size_t es = type_bytes(d->in_type);
  a.in = d->in;
  a.ld_in = d->ld_in;
  a.rows = d->rows;
  a.cols = d->cols;
  a.kp = up32(d->cols);
  a.tp = up32(d->rows);
  a.codes = static_cast<uint8_t*>(d->codes);
  a.sf = static_cast<uint8_t*>(d->sf);
  a.codes_t = static_cast<uint8_t*>(d->codes_t);
  a.sf_t = static_cast<uint8_t*>(d->sf_t);
  a.rand = static_cast<const uint8_t*>(d->rand);
  a.ld_rand = d->ld_rand;
  a.scale = d->scale;
  a.in_vec = rows_aligned(d->in, d->ld_in, es, 16);
  a.rand_vec = d->rand && rows_aligned(d->rand, d->ld_rand, 1, 8);
  uint32_t bits;
  memcpy(&bits, &d->scale, 4);
  // a power of two that an NVFP4 scale's reciprocal, at most 2^9, can take in and stay finite
  const bool pow2 = (bits & 0x7FFFFFu) == 0 && (bits >> 23) != 0 && d->scale <= 0x1p100f;
  DeviceGuard g(h->device);
  B2G_CUDA(h, launch_block_quant(fmt, d->in_type, pow2, a, reinterpret_cast<cudaStream_t>(stream)));
  return B2G_OK;
}

b2g_status b2g_block_dequantize(b2g_handle* h, int format, const void* d_codes, const void* d_sf,
                                int64_t rows, int64_t cols, int out_type, void* d_out,
                                int64_t ld_out, float scale, void* stream) {
  if (!h) return B2G_ERR_INVALID;
  h->last_error[0] = 0;
  const int fmt = block_fmt(format);
  if (fmt < 0)
    return fail(h, B2G_ERR_UNSUPPORTED, "b2g_block_dequantize: format %d (NVFP4, MXFP4 or MXFP8)",
                format);
  if (!type_ok(out_type)) return fail(h, B2G_ERR_INVALID, "b2g_block_dequantize: out_type %d", out_type);
  if (rows < 0 || cols < 0 || rows >= kMaxExtent || cols >= kMaxExtent)
    return fail(h, B2G_ERR_INVALID, "b2g_block_dequantize: rows or cols out of range");
  if (rows == 0 || cols == 0) return B2G_OK;
  if (!d_codes || !d_sf || !aligned(d_codes, 16) || !matrix_ok(d_out, out_type, cols, ld_out))
    return fail(h, B2G_ERR_INVALID,
                "b2g_block_dequantize: null or misaligned buffers, or ld_out < cols");
  BlockDequantArgs a;
  a.codes = static_cast<const uint8_t*>(d_codes);
  a.sf = static_cast<const uint8_t*>(d_sf);
  a.rows = rows;
  a.cols = cols;
  a.kp = up32(cols);
  a.out = d_out;
  a.ld_out = ld_out;
  a.scale = scale;
  a.out_vec = rows_aligned(d_out, ld_out, type_bytes(out_type), 16);
  DeviceGuard g(h->device);
  B2G_CUDA(h, launch_block_dequant(fmt, out_type, a, reinterpret_cast<cudaStream_t>(stream)));
  return B2G_OK;
}

b2g_status b2g_residual_norm(b2g_handle* h, const b2g_residual_norm_desc* d, void* stream) {
  if (!h || !d) return B2G_ERR_INVALID;
  h->last_error[0] = 0;
  const int type = d->type;
  if (!type_ok(type)) return fail(h, B2G_ERR_INVALID, "b2g_residual_norm: type %d", type);
  if (d->rows < 0 || d->cols < 1 || d->rows >= kMaxExtent || d->cols >= kMaxExtent)
    return fail(h, B2G_ERR_INVALID, "b2g_residual_norm: rows or cols out of range");
  if (d->cols > kNormMaxCols)
    return fail(h, B2G_ERR_UNSUPPORTED, "b2g_residual_norm: cols > %lld", (long long)kNormMaxCols);
  if (!(d->eps >= 0.0f)) return fail(h, B2G_ERR_INVALID, "b2g_residual_norm: eps < 0");
  if (d->rows == 0) return B2G_OK;  // pointers of empty buffers may be null
  int h_fmt = -1;
  if (d->codes || d->sf) {
    h_fmt = block_fmt(d->h_format);
    if (h_fmt < 0)
      return fail(h, B2G_ERR_UNSUPPORTED, "b2g_residual_norm: h_format %d (NVFP4, MXFP4 or MXFP8)",
                  d->h_format);
    if (!d->codes || !d->sf || !aligned(d->codes, 16))
      return fail(h, B2G_ERR_INVALID, "b2g_residual_norm: codes (16-byte aligned) need their scales");
  }
  if (!d->y && (d->gate || d->w_post || d->rstd_post))
    return fail(h, B2G_ERR_INVALID, "b2g_residual_norm: gate, w_post and rstd_post belong to y");
  if (!d->w_post && d->rstd_post)
    return fail(h, B2G_ERR_INVALID, "b2g_residual_norm: rstd_post belongs to w_post");
  if (!d->w_pre && (d->h || d->codes || d->rstd_pre))
    return fail(h, B2G_ERR_INVALID, "b2g_residual_norm: h, codes and rstd_pre need w_pre");
  if (!d->x_out && !d->h && !d->codes)
    return fail(h, B2G_ERR_INVALID, "b2g_residual_norm: no output");
  if (d->gate && d->rows_per_gate < 1)
    return fail(h, B2G_ERR_INVALID, "b2g_residual_norm: rows_per_gate < 1");
  const size_t es = type_bytes(type);
  if (!matrix_ok(d->x, type, d->cols, d->ld_x) ||
      (d->y && !matrix_ok(d->y, type, d->cols, d->ld_y)) ||
      (d->x_out && !matrix_ok(d->x_out, type, d->cols, d->ld_x_out)) ||
      (d->h && !matrix_ok(d->h, type, d->cols, d->ld_h)) || !aligned(d->gate, es) ||
      !aligned(d->w_post, es) || !aligned(d->w_pre, es) || !aligned(d->rstd_post, 4) ||
      !aligned(d->rstd_pre, 4))
    return fail(h, B2G_ERR_INVALID,
                "b2g_residual_norm: null or misaligned buffers, or a leading dimension < cols");
  ResidualNormArgs a;
  a.rows = d->rows;
  a.cols = d->cols;
  a.x = d->x;
  a.y = d->y;
  a.gate = d->gate;
  a.w_post = d->w_post;
  a.w_pre = d->w_pre;
  a.ld_x = d->ld_x;
  a.ld_y = d->ld_y;
  a.ld_x_out = d->ld_x_out;
  a.ld_h = d->ld_h;
  a.rows_per_gate = d->gate ? d->rows_per_gate : 1;
  a.x_out = d->x_out;
  a.h = d->h;
  a.codes = static_cast<uint8_t*>(d->codes);
  a.sf = static_cast<uint8_t*>(d->sf);
  a.kp = up32(d->cols);
  a.rstd_post = d->rstd_post;
  a.rstd_pre = d->rstd_pre;
  a.eps = d->eps;
  a.alpha = d->alpha;
  a.beta = d->beta;
  auto fits = [&](size_t bytes) {
    auto ok = [&](const void* p, int64_t ld) { return !p || rows_aligned(p, ld, es, bytes); };
    return ok(d->x, d->ld_x) && ok(d->y, d->ld_y) && ok(d->x_out, d->ld_x_out) && ok(d->h, d->ld_h) &&
           ok(d->gate, d->cols) && aligned(d->w_post, bytes) && aligned(d->w_pre, bytes);
  };
  a.vec = fits(16);
  DeviceGuard g(h->device);
  B2G_CUDA(h, launch_residual_norm(type, h_fmt, a, h->sm_count,
                                   reinterpret_cast<cudaStream_t>(stream)));
  return B2G_OK;
}

b2g_status b2g_residual_norm_backward(b2g_handle* h, const b2g_residual_norm_grad_desc* d,
                                      void* stream) {
  if (!h || !d) return B2G_ERR_INVALID;
  h->last_error[0] = 0;
  const int type = d->type;
  if (!type_ok(type)) return fail(h, B2G_ERR_INVALID, "b2g_residual_norm_backward: type %d", type);
  if (d->rows < 0 || d->cols < 1 || d->rows >= kMaxExtent || d->cols >= kMaxExtent)
    return fail(h, B2G_ERR_INVALID, "b2g_residual_norm_backward: rows or cols out of range");
  if (d->cols > kNormMaxCols)
    return fail(h, B2G_ERR_UNSUPPORTED, "b2g_residual_norm_backward: cols > %lld",
                (long long)kNormMaxCols);
  if (!aligned(d->dgate, 4) || !aligned(d->dw_post, 4) || !aligned(d->dw_pre, 4))
    return fail(h, B2G_ERR_INVALID, "b2g_residual_norm_backward: misaligned fp32 gradient");
  const size_t es = type_bytes(type);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  DeviceGuard g(h->device);
  if (d->rows == 0) {  // sums over no rows; pointers of empty buffers may be null
    if (d->dw_post) B2G_CUDA(h, cudaMemsetAsync(d->dw_post, 0, d->cols * sizeof(float), s));
    if (d->dw_pre) B2G_CUDA(h, cudaMemsetAsync(d->dw_pre, 0, d->cols * sizeof(float), s));
    return B2G_OK;
  }
  if (!d->dh && !d->dx_out)
    return fail(h, B2G_ERR_INVALID, "b2g_residual_norm_backward: neither dh nor dx_out");
  if (d->dh && (!d->x_out || !d->w_pre || !d->rstd_pre))
    return fail(h, B2G_ERR_INVALID, "b2g_residual_norm_backward: dh needs x_out, w_pre and rstd_pre");
  if (!d->dh && d->dw_pre)
    return fail(h, B2G_ERR_INVALID, "b2g_residual_norm_backward: dw_pre needs dh");
  if (!d->y && (d->gate || d->w_post || d->dy || d->dgate || d->dw_post))
    return fail(h, B2G_ERR_INVALID,
                "b2g_residual_norm_backward: gate, w_post and their gradients belong to y");
  if ((d->w_post == nullptr) != (d->rstd_post == nullptr) || (d->dw_post && !d->w_post))
    return fail(h, B2G_ERR_INVALID,
                "b2g_residual_norm_backward: w_post, rstd_post and dw_post belong together");
  if (d->dgate && !d->gate)
    return fail(h, B2G_ERR_INVALID, "b2g_residual_norm_backward: dgate needs gate");
  if (!d->dx && !d->dy && !d->dgate && !d->dw_post && !d->dw_pre)
    return fail(h, B2G_ERR_INVALID, "b2g_residual_norm_backward: no output");
  if (d->gate && d->rows_per_gate < 1)
    return fail(h, B2G_ERR_INVALID, "b2g_residual_norm_backward: rows_per_gate < 1");
  if ((d->dh && !matrix_ok(d->dh, type, d->cols, d->ld_dh)) ||
      (d->dx_out && !matrix_ok(d->dx_out, type, d->cols, d->ld_dx_out)) ||
      (d->dh && !matrix_ok(d->x_out, type, d->cols, d->ld_x_out)) ||
      (d->y && !matrix_ok(d->y, type, d->cols, d->ld_y)) ||
      (d->dx && !matrix_ok(d->dx, type, d->cols, d->ld_dx)) ||
      (d->dy && !matrix_ok(d->dy, type, d->cols, d->ld_dy)) || !aligned(d->gate, es) ||
      !aligned(d->w_post, es) || !aligned(d->w_pre, es) || !aligned(d->rstd_post, 4) ||
      !aligned(d->rstd_pre, 4))
    return fail(h, B2G_ERR_INVALID,
                "b2g_residual_norm_backward: null or misaligned buffers, or a leading dimension < cols");
  ResidualNormGradArgs a;
  memset(&a, 0, sizeof(a));
  a.rows = d->rows;
  a.cols = d->cols;
  a.dh = d->dh;
  a.dx_out = d->dx_out;
  a.v = d->x_out;
  a.y = d->y;
  a.gate = d->gate;
  a.w_post = d->w_post;
  a.w_pre = d->w_pre;
  a.rstd_post = d->rstd_post;
  a.rstd_pre = d->rstd_pre;
  a.ld_dh = d->ld_dh;
  a.ld_dx_out = d->ld_dx_out;
  a.ld_v = d->ld_x_out;
  a.ld_y = d->ld_y;
  a.ld_dx = d->ld_dx;
  a.ld_dy = d->ld_dy;
  a.rows_per_gate = d->gate ? d->rows_per_gate : 1;
  a.dx = d->dx;
  a.dy = d->dy;
  a.dgate = d->dgate;
  a.dw_post = d->dw_post;
  a.dw_pre = d->dw_pre;
  a.alpha = d->alpha;
  a.beta = d->beta;
  auto fits = [&](size_t bytes) {
    auto ok = [&](const void* p, int64_t ld) { return !p || rows_aligned(p, ld, es, bytes); };
    return ok(d->dh, d->ld_dh) && ok(d->dx_out, d->ld_dx_out) && (!d->dh || ok(d->x_out, d->ld_x_out)) &&
           ok(d->y, d->ld_y) && ok(d->dx, d->ld_dx) && ok(d->dy, d->ld_dy) && ok(d->gate, d->cols) &&
           aligned(d->w_post, bytes) && aligned(d->w_pre, bytes);
  };
  a.vec = fits(16);
  a.dgate_vec = aligned(d->dgate, 16);
  a.err = h->d_err;
  const b2g_status st = reserve(h, &h->op_ws, norm_grad_ws_bytes(type, a, h->sm_count), false, s);
  if (st != B2G_OK) return st;
  a.ws = h->op_ws.p;
  B2G_CUDA(h, launch_residual_norm_grad(type, a, h->sm_count, s));
  return B2G_OK;
}

b2g_status b2g_linear(b2g_handle* h, const b2g_linear_desc* d, void* stream) {
  if (!h || !d) return B2G_ERR_INVALID;
  h->last_error[0] = 0;
  const int fmt = block_fmt(d->format);
  if (fmt < 0)
    return fail(h, B2G_ERR_UNSUPPORTED, "b2g_linear: format %d (NVFP4, MXFP4 or MXFP8)", d->format);
  if (d->type == B2G_F32)
    return fail(h, B2G_ERR_UNSUPPORTED, "b2g_linear: x must be bf16 or fp16");
  if (!type_ok(d->type)) return fail(h, B2G_ERR_INVALID, "b2g_linear: type %d", d->type);
  if (d->T < 0 || d->N < 0 || d->K < 1 || d->T > kFewMaxTokens || d->N > kFewMaxExtent ||
      d->K > kFewMaxExtent)
    return fail(h, B2G_ERR_INVALID, "b2g_linear: T, N or K out of range (T up to %d, N and K to %d)",
                kFewMaxTokens, kFewMaxExtent);
  if (d->T == 0 || d->N == 0) return B2G_OK;
  if (!matrix_ok(d->x, d->type, d->K, d->ld_x) || !matrix_ok(d->out, d->type, d->N, d->ld_out) ||
      !d->w || !d->sfw || !aligned(d->w, 16) || !aligned(d->sfw, 2))
    return fail(h, B2G_ERR_INVALID,
                "b2g_linear: null or misaligned buffers (w 16, sfw 2 bytes), or a leading "
                "dimension too small");
  FewLinearArgs a;
  memset(&a, 0, sizeof(a));
  a.T = d->T;
  a.N = d->N;
  a.K = d->K;
  a.kp = up32(d->K);
  a.x = d->x;
  a.ld_x = d->ld_x;
  a.w = static_cast<const uint8_t*>(d->w);
  a.sf = static_cast<const uint8_t*>(d->sfw);
  a.out = d->out;
  a.ld_out = d->ld_out;
  a.alpha = d->alpha;
  a.x_vec = rows_aligned(d->x, d->ld_x, 2, 16);
  DeviceGuard g(h->device);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  a.err = h->d_err;
  a.wait_ns = h->wait_ns;
  const bool tiles = linear_tiles(a);
  b2g_status st = reserve(h, &h->op_ws, tiles ? few_tiles_ws_bytes(fmt, a, h->sm_count)
                                              : few_linear_ws_bytes(fmt, a, h->sm_count), false, s);
  if (st != B2G_OK) return st;
  const size_t counters = tiles ? few_tiles_counters(fmt, a, h->sm_count)
                                : few_linear_counters(fmt, a, h->sm_count);
  st = reserve(h, &h->op_count, counters * sizeof(uint32_t), true, s);
  if (st != B2G_OK) return st;
  a.ws = h->op_ws.p;
  a.count = static_cast<uint32_t*>(h->op_count.p);
  if (!tiles) {
    B2G_CUDA(h, launch_few_linear(fmt, d->type, a, h->sm_count, s));
    return B2G_OK;
  }
  FewTilesMaps m;
  few_tiles_maps(fmt, a, h->sm_count, &m);
  CUtensorMap map_w, map_x;
  b2g_status mt = tensor_map(h, &map_w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, d->w, m.w_row_bytes,
                             (uint64_t)d->N, m.w_box_bytes, m.w_box_rows);
  if (mt != B2G_OK) return mt;
  mt = tensor_map(h, &map_x, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, a.ws, m.x_cols, (uint64_t)d->T,
                  m.x_box_cols, m.x_box_rows);
  if (mt != B2G_OK) return mt;
  B2G_CUDA(h, launch_few_tiles(fmt, d->type, a, map_w, map_x, h->sm_count, s));
  return B2G_OK;
}

}  // extern "C"
