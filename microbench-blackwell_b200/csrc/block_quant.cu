// block_quant.cu -- microscaled casts of activations, weights and gradients, along the
// rows and the columns of a matrix in one pass, and their read-back.
//
// The reference fills its operands with byte patterns and its scales with constants
// (tcgen05_sparse_mma/tcgen05_sparse_mma.cu:246-256,320-325); a training step casts
// each operand twice, because the products of forward and backward run along different
// dimensions and a block's scale lies along the product's.
#include "b2g.h"
#include "op_common.cuh"
#include "op_kernels.h"

namespace b2g {
namespace {

constexpr int kThreads = 256;

// eight random bytes, zeros from the n-th on
__device__ __forceinline__ uint2 load_rand8(const uint8_t* p, int n, bool vec) {
  if (vec && n >= 8) return __ldg(reinterpret_cast<const uint2*>(p));
  uint32_t w[2] = {0u, 0u};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n) w[i >> 2] |= (uint32_t)__ldg(p + i) << (8 * (i & 3));
  return make_uint2(w[0], w[1]);
}

// Codes and scale of eight elements held by one thread; the threads of a block (2 for
// 16 elements, 4 for 32) are neighbours and share the largest magnitude.
template <int FMT, int QM, bool SR>
__device__ __forceinline__ void encode_row8(float (&x)[8], float scale, uint2 rnd,
                                            uint8_t* codes, uint8_t* sf, bool write) {
  float amax = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = __fmul_rn(x[i], scale);
    amax = max_nan(amax, fabsf(x[i]));
  }
  amax = max_nan(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 1));
  if constexpr (bf_block(FMT) == 32) amax = max_nan(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 2));
  const BlockScale s = block_scale<FMT>(amax);
  uint32_t w[2];
  encode8<FMT, QM, SR>(x, s, rnd, w);
  if (!write) return;
  if constexpr (FMT == BF_MXF8)
    *reinterpret_cast<uint2*>(codes) = make_uint2(w[0], w[1]);
  else
    *reinterpret_cast<uint32_t*>(codes) = w[0];
  if ((threadIdx.x & (bf_block(FMT) / 8 - 1)) == 0) *sf = (uint8_t)s.byte;
}

// Rows only: eight elements per thread.  blockDim.x threads along a row, blockDim.y rows.
template <typename T, int FMT, int QM, bool SR>
__global__ void __launch_bounds__(kThreads) quant_rows_kernel(const BlockQuantArgs a) {
  constexpr int bits = bf_bits(FMT), blk = bf_block(FMT);
  const int64_t c = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) * 8;
  const bool in_row = c < a.kp;
  const int n = c >= a.cols ? 0 : (int)(a.cols - c < 8 ? a.cols - c : 8);
  const int64_t step = (int64_t)gridDim.y * blockDim.y;
  // two rows at a time: both loads are in flight before the first is used
  for (int64_t r = (int64_t)blockIdx.y * blockDim.y + threadIdx.y; __any_sync(0xFFFFFFFFu, r < a.rows);
       r += 2 * step) {
    const bool ok0 = in_row && r < a.rows, ok1 = in_row && r + step < a.rows;
    const T* p = static_cast<const T*>(a.in) + r * a.ld_in + c;
    const Raw8<T> raw0 = load8(p, ok0 ? n : 0, a.in_vec);
    const Raw8<T> raw1 = load8(p + step * a.ld_in, ok1 ? n : 0, a.in_vec);
    uint2 rnd0 = make_uint2(0, 0), rnd1 = rnd0;
    if constexpr (SR) {
      const uint8_t* q = a.rand + r * a.ld_rand + c;
      rnd0 = load_rand8(q, ok0 ? n : 0, a.rand_vec);
      rnd1 = load_rand8(q + step * a.ld_rand, ok1 ? n : 0, a.rand_vec);
    }
    float x[8];
    unpack8(raw0, x);
    encode_row8<FMT, QM, SR>(x, a.scale, rnd0, a.codes + (r * a.kp + c) * bits / 8,
                             a.sf + (r * a.kp + c) / blk, ok0);
    unpack8(raw1, x);
    encode_row8<FMT, QM, SR>(x, a.scale, rnd1, a.codes + ((r + step) * a.kp + c) * bits / 8,
                             a.sf + ((r + step) * a.kp + c) / blk, ok1);
  }
}

// Rows and columns: one CTA takes a tile of 128 rows x 128 bytes, casts it along the
// rows on the way into shared memory (where it is kept unscaled in its own type) and
// along the columns out of it.  A thread of the column pass reads 16 rows of one
// 32-bit word (two 16-bit columns or one fp32 column), eight threads side by side down
// the rows, so that a warp writes 64 (e2m1) or 128 (e4m3) contiguous bytes per column.
// 16-byte chunk c of row r lies at chunk c ^ (r / 16 % 8): the eight threads of one
// column word then read different banks.
constexpr int kTileRows = 128;

template <typename T, int FMT, int QM, bool SR, bool ROWS>
__global__ void __launch_bounds__(kThreads) quant_both_kernel(const BlockQuantArgs a) {
  constexpr int bits = bf_bits(FMT), blk = bf_block(FMT);
  constexpr int kCols = 128 / (int)sizeof(T);    // columns of a tile
  constexpr int kVec = kCols / 8;                // eights of a row
  constexpr int kPer = 4 / (int)sizeof(T);       // columns of a 32-bit word
  __shared__ __align__(16) uint32_t tile[kTileRows * 32];
  __shared__ __align__(16) uint8_t rnd_tile[SR ? kTileRows * kCols : 16];
  const int tid = threadIdx.x;
  const unsigned col_tiles = (unsigned)((a.kp + kCols - 1) / kCols);
  const int64_t r0 = (int64_t)(blockIdx.x / col_tiles) * kTileRows;
  const int64_t c0 = (int64_t)(blockIdx.x % col_tiles) * kCols;

#pragma unroll
  for (int i = 0; i < kTileRows * kVec / kThreads; ++i) {
    const int item = i * kThreads + tid, v = item % kVec, lr = item / kVec;
    const int64_t r = r0 + lr, c = c0 + v * 8;
    const int n = r >= a.rows || c >= a.cols ? 0 : (int)(a.cols - c < 8 ? a.cols - c : 8);
    const Raw8<T> raw = load8(static_cast<const T*>(a.in) + r * a.ld_in + c, n, a.in_vec);
    uint2 rnd = make_uint2(0, 0);
    const int g = (lr >> 4) & 7;
    if constexpr (SR) {
      rnd = load_rand8(a.rand + r * a.ld_rand + c, n, a.rand_vec);
      // 32-bit word q of a row lies at q ^ 2 g (fp32 tiles: half as many words)
      uint32_t* q = reinterpret_cast<uint32_t*>(rnd_tile) + lr * (kCols / 4);
      const int at = (2 * v) ^ ((2 * g) & (kCols / 4 - 1));
      *reinterpret_cast<uint2*>(q + at) = rnd;
    }
    uint4* row = reinterpret_cast<uint4*>(tile) + lr * 8;
    if constexpr (sizeof(T) == 4) {
      row[(2 * v) ^ g] = raw.w[0];
      row[(2 * v + 1) ^ g] = raw.w[1];
    } else {
      row[v ^ g] = raw.w[0];
    }
    if constexpr (ROWS) {
      float x[8];
      unpack8(raw, x);
      encode_row8<FMT, QM, SR>(x, a.scale, rnd, a.codes + (r * a.kp + c) * bits / 8,
                               a.sf + (r * a.kp + c) / blk, r < a.rows && c < a.kp);
    }
  }
  __syncthreads();

  const int g = tid & 7, w = tid >> 3;  // 16-row group, 32-bit word of the row
  uint32_t raw[16];
#pragma unroll
  for (int i = 0; i < 16; ++i)
    raw[i] = tile[(g * 16 + i) * 32 + ((((w >> 2) ^ g) << 2) | (w & 3))];
  const int64_t r = r0 + g * 16;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int64_t c = c0 + w * kPer + j;
    float x[2][8];
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float f;
      if constexpr (sizeof(T) == 4) {
        f = __uint_as_float(raw[i]);
      } else {
        const float2 p = pair_f32<T>(raw[i]);
        f = j ? p.y : p.x;
      }
      f = __fmul_rn(f, a.scale);
      x[i >> 3][i & 7] = f;
      amax = max_nan(amax, fabsf(f));
    }
    if constexpr (blk == 32) amax = max_nan(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 1));
    const BlockScale s = block_scale<FMT>(amax);
    uint2 rnd[2] = {make_uint2(0, 0), make_uint2(0, 0)};
    if constexpr (SR) {
      uint32_t b[4] = {0u, 0u, 0u, 0u};
      const int byte = w * kPer + j;
      const int at = (((byte >> 2) ^ ((2 * g) & (kCols / 4 - 1))) << 2) | (byte & 3);
#pragma unroll
      for (int i = 0; i < 16; ++i)
        b[i >> 2] |= (uint32_t)rnd_tile[(g * 16 + i) * kCols + at] << (8 * (i & 3));
      rnd[0] = make_uint2(b[0], b[1]);
      rnd[1] = make_uint2(b[2], b[3]);
    }
    uint32_t lo[2], hi[2];
    encode8<FMT, QM, SR>(x[0], s, rnd[0], lo);
    encode8<FMT, QM, SR>(x[1], s, rnd[1], hi);
    if (c < a.cols && r < a.tp) {
      uint8_t* dst = a.codes_t + (c * a.tp + r) * bits / 8;
      if constexpr (FMT == BF_MXF8)
        *reinterpret_cast<uint4*>(dst) = make_uint4(lo[0], lo[1], hi[0], hi[1]);
      else
        *reinterpret_cast<uint2*>(dst) = make_uint2(lo[0], hi[0]);
      if (blk == 16 || (g & 1) == 0) a.sf_t[(c * a.tp + r) / blk] = (uint8_t)s.byte;
    }
  }
}

// Read-back: eight codes per thread.
template <typename T, int FMT>
__global__ void __launch_bounds__(kThreads) dequant_kernel(const BlockDequantArgs a) {
  constexpr int bits = bf_bits(FMT), blk = bf_block(FMT);
  const int64_t c = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) * 8;
  if (c >= a.cols) return;
  const int n = (int)(a.cols - c < 8 ? a.cols - c : 8);
  for (int64_t r = (int64_t)blockIdx.y * blockDim.y + threadIdx.y; r < a.rows;
       r += (int64_t)gridDim.y * blockDim.y) {
    const int64_t e = r * a.kp + c;
    const uint32_t sb = __ldg(a.sf + e / blk);
    float s;
    if constexpr (FMT == BF_NVFP4)
      s = e4m3_pair(sb).x;
    else
      s = e8m0_value(sb);
    float v[8];
    if constexpr (FMT == BF_MXF8) {
      const uint2 w = __ldg(reinterpret_cast<const uint2*>(a.codes + e));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 p = e4m3_pair((i < 2 ? w.x : w.y) >> (16 * (i & 1)));
        v[2 * i] = p.x;
        v[2 * i + 1] = p.y;
      }
    } else {
      const uint32_t w = __ldg(reinterpret_cast<const uint32_t*>(a.codes + e * bits / 8));
      uint32_t h[4];
      e2m1x8_pairs(w, h);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
        v[2 * i] = p.x;
        v[2 * i + 1] = p.y;
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __fmul_rn(__fmul_rn(v[i], s), a.scale);
    store8(static_cast<T*>(a.out) + r * a.ld_out + c, v, n, a.out_vec);
  }
}

// blockDim.x threads of eight elements along a row of `cols`, the rest along the rows
void row_shape(int64_t rows, int64_t cols, dim3* grid, dim3* block) {
  const int64_t v = (cols + 7) / 8;
  int bx = 4;
  while (bx < kThreads && bx < v) bx *= 2;
  const int by = kThreads / bx;
  const int64_t gx = (v + bx - 1) / bx;
  int64_t gy = (rows + by - 1) / by;
  *block = dim3(bx, by);
  *grid = dim3((unsigned)gx, (unsigned)(gy < 65535 ? gy : 65535));
}

template <typename T, int FMT, int QM, bool SR>
cudaError_t quant_launch(const BlockQuantArgs& a, cudaStream_t s) {
  if (!a.codes_t) {
    dim3 grid, block;
    row_shape((a.rows + 1) / 2, a.kp, &grid, &block);
    quant_rows_kernel<T, FMT, QM, SR><<<grid, block, 0, s>>>(a);
    return cudaGetLastError();
  }
  constexpr int kCols = 128 / (int)sizeof(T);
  const int64_t tiles = ((a.tp + kTileRows - 1) / kTileRows) * ((a.kp + kCols - 1) / kCols);
  if (tiles > 0x7FFFFFFF) return cudaErrorInvalidValue;
  const unsigned grid = (unsigned)tiles;
  if (a.codes)
    quant_both_kernel<T, FMT, QM, SR, true><<<grid, kThreads, 0, s>>>(a);
  else
    quant_both_kernel<T, FMT, QM, SR, false><<<grid, kThreads, 0, s>>>(a);
  return cudaGetLastError();
}

template <typename T, int FMT, int QM>
cudaError_t quant_sr(const BlockQuantArgs& a, cudaStream_t s) {
  return a.rand ? quant_launch<T, FMT, QM, true>(a, s) : quant_launch<T, FMT, QM, false>(a, s);
}

template <typename T>
cudaError_t quant_fmt(int fmt, bool pow2, const BlockQuantArgs& a, cudaStream_t s) {
  if (fmt == BF_MXF8) return quant_sr<T, BF_MXF8, Q_EXACT>(a, s);
  if (fmt == BF_MXF4) return quant_sr<T, BF_MXF4, Q_EXACT>(a, s);
  // the short quotient holds for inputs of at most 11 significant bits
  if constexpr (sizeof(T) == 2)
    if (pow2) return quant_sr<T, BF_NVFP4, Q_SNAP>(a, s);
  return quant_sr<T, BF_NVFP4, Q_DIVIDE>(a, s);
}

template <typename T>
cudaError_t dequant_fmt(int fmt, const BlockDequantArgs& a, cudaStream_t s) {
  dim3 grid, block;
  row_shape(a.rows, a.cols, &grid, &block);
  if (fmt == BF_MXF8)
    dequant_kernel<T, BF_MXF8><<<grid, block, 0, s>>>(a);
  else if (fmt == BF_MXF4)
    dequant_kernel<T, BF_MXF4><<<grid, block, 0, s>>>(a);
  else
    dequant_kernel<T, BF_NVFP4><<<grid, block, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_block_quant(int fmt, int type, bool pow2, const BlockQuantArgs& a,
                               cudaStream_t s) {
  if (type == B2G_F32) return quant_fmt<float>(fmt, pow2, a, s);
  if (type == B2G_BF16) return quant_fmt<__nv_bfloat16>(fmt, pow2, a, s);
  return quant_fmt<__half>(fmt, pow2, a, s);
}

cudaError_t launch_block_dequant(int fmt, int type, const BlockDequantArgs& a, cudaStream_t s) {
  if (type == B2G_F32) return dequant_fmt<float>(fmt, a, s);
  if (type == B2G_BF16) return dequant_fmt<__nv_bfloat16>(fmt, a, s);
  return dequant_fmt<__half>(fmt, a, s);
}

}  // namespace b2g
