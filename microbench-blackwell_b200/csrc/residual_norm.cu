// residual_norm.cu -- norms before and after a block, fused with its gate and residual
// scale.
//
//   z = y * rstd(y) * w_post            (z = y without w_post)
//   v = alpha * x + beta * gate * z     (v = alpha * x without y)
//   x_out = v,  h = v * rstd(v) * w_pre,  rstd(a) = 1 / sqrt(mean(a^2) + eps)
//
// All sums and the row v are fp32; x_out and h are rounded once.  h is formed from the
// unrounded v.
#include <string.h>

#include <type_traits>

#include "b2g.h"
#include "b2g_gemm.h"
#include "b2g_ptx.cuh"
#include "op_common.cuh"
#include "op_kernels.h"

namespace b2g {
namespace {

// One row per blockDim.x threads, held in registers: NV times eight elements a thread.  Each
// element is read once and written once, so bytes bound it: 16384 x 8192 bf16 with norm after,
// gate and norm before 168 us, 6.4 of the 6.5 TB/s that a copy measures; into MXFP8 codes 176 us
// (82 %: the casts); 4095 x 5000 fp16 39 us (64 %) and one row 3.8 us: waits for memory and
// barriers.
// ANY: operands of any alignment, read and written as the aligned words that cover them:
// 16384 x 8191 bf16 397 us, bound by the shifting (974 us element by element).
template <typename T, int NV, int HF, bool ANY>
__global__ void __launch_bounds__(1024) residual_norm_kernel(const ResidualNormArgs a) {
  // Weights and gate are asked for before the row's sums meet, where registers allow (16-bit
  // types: w_pre; one eight a thread: all three): 1000 x 4096 10.0 -> 9.3 us, 300 x 1024 3.5 ->
  // 3.1 us; all three with four eights a thread 168 -> 224 us at 16384 x 8192, in spills.
  constexpr bool kEarlyPre = sizeof(T) == 2, kEarlyPost = kEarlyPre && NV == 1;
  __shared__ float red[2][32];
  const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  if (row >= a.rows) return;  // whole warps: blockDim.y > 1 only with one warp per row
  extern __shared__ __align__(16) uint4 stores[];  // ANY: one buffer a warp
  uint4* buf = stores + (threadIdx.y * blockDim.x + threadIdx.x) / 32 * (2 * sizeof(T) * 8 + 1);
  const T* x = static_cast<const T*>(a.x) + row * a.ld_x;
  const T* y = static_cast<const T*>(a.y) + row * a.ld_y;
  Raw8<T> rx[NV], ry[NV];
  const int cols = (int)a.cols;
  int col[NV], n[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    col[j] = (j * (int)blockDim.x + (int)threadIdx.x) * 8;
    const int left = cols - col[j];
    n[j] = left < 0 ? 0 : left < 8 ? left : 8;
  }
  // eight elements of row r of an operand that has `rows` rows
  auto get = [&](const T* at, int64_t r, int64_t rows, int j) {
    return load8_any<T, ANY>(at + col[j], n[j], cols >= 16 && r > 0 && r < rows - 1);
  };
  auto put = [&](void* p, int64_t ld, int j, const float2(&f)[4]) {
    const int left = cols - (col[j] - (int)(threadIdx.x & 31) * 8);
    const float o[8] = {f[0].x, f[0].y, f[1].x, f[1].y, f[2].x, f[2].y, f[3].x, f[3].y};
    store8_any<T, ANY>(static_cast<T*>(p) + row * ld + col[j], o, n[j],
                       left < 0 ? 0 : left < 256 ? left : 256, buf);
  };
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    rx[j] = get(x, row, a.rows, j);
    if (a.y) ry[j] = get(y, row, a.rows, j);
  }
  float2 v[NV][4];
  if (a.y) {
    const int64_t gate_row = row / a.rows_per_gate, last_gate = (a.rows - 1) / a.rows_per_gate;
    const T* gate = a.gate ? static_cast<const T*>(a.gate) + gate_row * a.cols : nullptr;
    Raw8<T> wp[NV], gp[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (kEarlyPost && a.w_post) wp[j] = get(static_cast<const T*>(a.w_post), 0, 1, j);
      if (kEarlyPost && gate) gp[j] = get(gate, gate_row, last_gate + 1, j);
    }
    float r1 = 1.0f;
    if (a.w_post) {
      float2 sum = both(0.0f);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        float2 f[4];
        unpack4x2(ry[j], f);
#pragma unroll
        for (int i = 0; i < 4; ++i) sum = fma2(f[i], f[i], sum);
      }
      float ss[1] = {sum.x + sum.y};
      row_sum(ss, red[0]);
      r1 = 1.0f / sqrtf(ss[0] / (float)a.cols + a.eps);
      if (a.rstd_post && threadIdx.x == 0) a.rstd_post[row] = r1;
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float2 fx[4], fy[4];
      unpack4x2(rx[j], fx);
      unpack4x2(ry[j], fy);
      if (a.w_post) {
        float2 w[4];
        unpack4x2(kEarlyPost ? wp[j] : get(static_cast<const T*>(a.w_post), 0, 1, j), w);
#pragma unroll
        for (int i = 0; i < 4; ++i) fy[i] = mul2(mul2(fy[i], both(r1)), w[i]);
      }
      if (gate) {
        float2 g[4];
        unpack4x2(kEarlyPost ? gp[j] : get(gate, gate_row, last_gate + 1, j), g);
#pragma unroll
        for (int i = 0; i < 4; ++i) fy[i] = mul2(fy[i], g[i]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) v[j][i] = fma2(both(a.beta), fy[i], mul2(both(a.alpha), fx[i]));
    }
  } else {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      unpack4x2(rx[j], v[j]);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[j][i] = mul2(v[j][i], both(a.alpha));
    }
  }
  if (a.x_out) {
#pragma unroll
    for (int j = 0; j < NV; ++j) put(a.x_out, a.ld_x_out, j, v[j]);
  }
  if (!a.w_pre) return;
  float2 sum = both(0.0f);
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) sum = fma2(v[j][i], v[j][i], sum);
  Raw8<T> wq[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j)
    if (kEarlyPre) wq[j] = get(static_cast<const T*>(a.w_pre), 0, 1, j);
  float ss[1] = {sum.x + sum.y};
  row_sum(ss, red[1]);
  const float r2 = 1.0f / sqrtf(ss[0] / (float)a.cols + a.eps);
  if (a.rstd_pre && threadIdx.x == 0) a.rstd_pre[row] = r2;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    float2 w[4];
    unpack4x2(kEarlyPre ? wq[j] : get(static_cast<const T*>(a.w_pre), 0, 1, j), w);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[j][i] = mul2(mul2(v[j][i], both(r2)), w[i]);
    if (a.h) put(a.h, a.ld_h, j, v[j]);
    if constexpr (HF >= 0) {
      constexpr int blk = bf_block(HF), bits = bf_bits(HF);
      constexpr int mode = HF == BF_NVFP4 ? Q_DIVIDE : Q_EXACT;
      float amax = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) amax = max_nan(amax, max_nan(fabsf(v[j][i].x), fabsf(v[j][i].y)));
      amax = max_nan(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 1));
      if constexpr (blk == 32) amax = max_nan(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 2));
      const BlockScale s = block_scale<HF, mode>(amax);
      uint32_t q[2];
      encode8<HF, mode, false, false>(v[j], s, 1.0f, make_uint2(0, 0), q);
      if (col[j] < a.kp) {
        const int64_t e = row * a.kp + col[j];
        if constexpr (HF == BF_MXF8)
          *reinterpret_cast<uint2*>(a.codes + e) = make_uint2(q[0], q[1]);
        else
          *reinterpret_cast<uint32_t*>(a.codes + e * bits / 8) = q[0];
        if ((threadIdx.x & (blk / 8 - 1)) == 0) a.sf[e / blk] = (uint8_t)s.byte;
      }
    }
  }
}

template <typename T, int HF, bool ANY>
cudaError_t norm_launch(const ResidualNormArgs& a, int sm_count, cudaStream_t s) {
  const int64_t v = ((HF < 0 ? a.cols : a.kp) + 7) / 8;
  // Few rows, or a few thousand short ones: as many threads to a row as it has eights, for
  // latency.  Many: four eights a thread, which keeps eight 16-byte loads in flight in each,
  // or one warp's share of a short row.  Measured (bf16, us, one eight a thread / four):
  // 1 x 8192 4.1 / 5.7, 300 x 2048 3.8 / 6.2, 4000 x 2048 18.3 / 20.4, 16384 x 2048 59.9 /
  // 49.7, 4000 x 4096 33.4 / 30.8, 16384 x 8192 255 / 171; 20000 x 256 12.7 / 31.0.
  const int nv = v <= 32 || (a.rows < 2 * sm_count && v <= 1024) || (v <= 256 && a.rows * v <= 1 << 20) ? 1
                 : v <= 64 ? 2
                           : 4;
  int64_t tpr = ((v + nv - 1) / nv + 31) / 32 * 32;
  const int rpc = tpr == 32 ? 4 : 1;
  const dim3 block((unsigned)tpr, rpc);
  const unsigned grid = (unsigned)((a.rows + rpc - 1) / rpc);
  const size_t smem = ANY ? tpr * rpc / 32 * (2 * sizeof(T) * 8 + 1) * sizeof(uint4) : 0;
  if (nv == 1)
    residual_norm_kernel<T, 1, HF, ANY><<<grid, block, smem, s>>>(a);
  else if (nv == 2)
    residual_norm_kernel<T, 2, HF, ANY><<<grid, block, smem, s>>>(a);
  else
    residual_norm_kernel<T, 4, HF, ANY><<<grid, block, smem, s>>>(a);
  return cudaGetLastError();
}

template <typename T>
cudaError_t norm_fmt(int h_fmt, const ResidualNormArgs& a, int sm_count, cudaStream_t s) {
  switch (h_fmt) {
    case BF_NVFP4: return a.vec ? norm_launch<T, BF_NVFP4, false>(a, sm_count, s) : norm_launch<T, BF_NVFP4, true>(a, sm_count, s);
    case BF_MXF4: return a.vec ? norm_launch<T, BF_MXF4, false>(a, sm_count, s) : norm_launch<T, BF_MXF4, true>(a, sm_count, s);
    case BF_MXF8: return a.vec ? norm_launch<T, BF_MXF8, false>(a, sm_count, s) : norm_launch<T, BF_MXF8, true>(a, sm_count, s);
    default: return a.vec ? norm_launch<T, -1, false>(a, sm_count, s) : norm_launch<T, -1, true>(a, sm_count, s);
  }
}

}  // namespace

cudaError_t launch_residual_norm(int type, int h_fmt, const ResidualNormArgs& a, int sm_count,
                                 cudaStream_t s) {
  if (type == B2G_F32) return norm_fmt<float>(h_fmt, a, sm_count, s);
  if (type == B2G_BF16) return norm_fmt<__nv_bfloat16>(h_fmt, a, sm_count, s);
  return norm_fmt<__half>(h_fmt, a, sm_count, s);
}

}  // namespace b2g
