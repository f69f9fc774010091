// residual_norm_grad.cu -- gradient of the norms before and after a block with its gate and
// residual scale (residual_norm.cu).
#include <string.h>

#include <type_traits>

#include "b2g.h"
#include "b2g_gemm.h"
#include "b2g_ptx.cuh"
#include "op_common.cuh"
#include "op_kernels.h"

namespace b2g {
namespace {

// ------------------------------------------------------------------ gradient
// With v^ = v r2, y^ = y r1, p = w_pre dh, q = beta w_post g:
//   dv = dx_out + r2 (p - v^ mean(p v^)),  dx = alpha dv,  dw_pre = sum dh v^
//   dy = r1 (q dv - y^ mean(q dv y^)),  dgate = beta sum z dv,  dw_post = sum beta g dv y^
// mean(q dv y^) follows from sums that need no dv: with A = sum p v^, B = sum q y^
// (dx_out + r2 p), C = sum q y^ v^ it is (B - r2 (A / D) C) / D.  So one reduction per
// row gives both means.  Every product is taken with v^ and y^, never with a power of r2 or
// r1 by itself: a row's gradients then have the range of the formula, whatever its size.

// Rows of up to 8192 columns go through grad_rows_kernel in one pass; wider ones, which do not
// fit a CTA's registers and shared memory, through a pass for the means and one down the
// columns (16384 x 8192 bf16: 352 us in one pass, 905 us in two).

// One pass: a CTA owns a run of rows and all columns, NV times eight a thread, with the
// sums over its rows in registers.  Each thread copies its own part of the next rows into
// shared memory while it works on one, so a row costs one barrier, for the means.
// Reads 4 and writes 2 elements for each; 16384 x 8192 bf16 352 us, 4.6 TB/s of the 6.5 that a
// copy measures: with the column sums 128 registers a thread leave 16 warps an SM, and a row's
// barrier and two chains of sums are not hidden by them all.  Bulk copies in place of each
// thread's own took 364 us, 1024 threads of 64 registers 440 us.
constexpr int kRowStages = 3;

struct GradRows {
  int threads, max_threads, nv, stages, ctas;
  bool any;
  bool gate_rows;   // a gate row per few rows: it is copied along with the row
  size_t smem;
};

// Shared memory of a CTA: slots for a row's four or five tensors; any alignment: 32 bytes more a
// tensor, and a buffer for each warp's stores.
constexpr size_t kGradRoom = 224 * 1024;
constexpr size_t grad_stage(int max_threads, int nv, int elem, bool few) {
  return (size_t)max_threads * nv * (few ? 5 : 4) * 8 * elem;
}
constexpr size_t grad_smem(int stages, size_t stage, int max_threads, bool any) {
  return stages * (stage + (any ? 5 * 32 : 0)) + (any ? max_threads / 32 * 65 * 16 : 0);
}

// What is summed over rows that more than one CTA has: part[cta][2][cols] (dw_pre, dw_post)
// and slots[2 cta + (0: the gate the CTA starts in, 1: the one it ends in)][cols].
__device__ __host__ __forceinline__ int64_t first_row(int64_t cta, int64_t rows, int64_t ctas) {
  return cta * rows / ctas;
}

// While the gate stays, dgate and dw_post are one sum Z = sum y^ dv away: dgate = beta
// w_post Z, dw_post = beta g Z.  So a row adds to two sums (dw_pre and Z), and gate *
// w_post is kept as one product; both are renewed when the gate changes.
// MAXT: bound of the CTA's threads and their stride in shared memory.  ALL: dh, dx_out, y,
// w_post, dx and dy are there, so that the common pass is free of tests for them (16384 x 8192
// 352 us, with the tests 372).  FEW: a gate has few rows; its values come through the ring and
// dw_post stays in registers, where otherwise it is added up in `part` (a gate a row 522 us,
// without 700; a gate per 16 rows of 4096 258 us, without 246).
// ANY: operands of any alignment (16384 x 8191 887 us, in two passes 1346; 803 with
// the powers of r in the row's scalars, which leave fp32's range).  Rows are copied as the aligned words that cover them and
// shifted on the way out of shared memory; an element may then lie in a neighbour's copy,
// so a row's copies have landed, for all, by the barrier of the row before, and its slot
// is filled again after the barrier of the row behind.
template <typename T, int NV, int MAXT, bool ALL, bool FEW, bool ANY>
__global__ void __launch_bounds__(MAXT, 512 / MAXT)
grad_rows_kernel(const ResidualNormGradArgs a, const GradRows plan, float* part, float* slots) {
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ float red[2][3 * 32];
  constexpr int W = (int)sizeof(T) / 2;          // 16-byte words of eight elements
  constexpr bool kKeep = sizeof(T) == 2;         // weights stay in registers
  const int tid = threadIdx.x, nt = blockDim.x;
  const int64_t r0 = first_row(blockIdx.x, a.rows, gridDim.x);
  const int64_t r1 = first_row(blockIdx.x + 1, a.rows, gridDim.x);
  const bool has_h = ALL || a.dh, has_y = ALL || a.y, has_x = ALL || a.dx_out;
  const bool norm_y = ALL || a.w_post, out_x = ALL || a.dx, out_y = ALL || a.dy;
  const int cols = (int)a.cols;
  const int64_t pitch = ((int64_t)cols + 7) / 8 * 8;  // of part and slots
  uint32_t col[NV];
  int n[NV];    // this thread's columns, 0 .. 8
  bool on[NV];  // it takes part (ANY: its warp does)
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    col[j] = (uint32_t)(j * nt + tid) * 8;
    const int left = cols - (int)col[j];
    n[j] = left < 0 ? 0 : left < 8 ? left : 8;
    on[j] = ANY ? left + (tid & 31) * 8 > 0 : left > 0;
  }
  auto live = [&](int j) { return ANY ? n[j] > 0 : on[j]; };
  // tensors of a row: dh, v, dx_out, y, gate (FEW); a slot holds [tensor][j][word][thread],
  // or (ANY) [tensor][covering words]
  constexpr uint32_t kStride = MAXT * 16, kTensor = NV * W * kStride + (ANY ? 32 : 0);
  constexpr uint32_t slot_bytes = (FEW ? 5 : 4) * kTensor;
  const uint32_t base = smem_u32(ring) + (ANY ? 0 : tid * 16);
  // ANY: what store8_any() needs, behind the slots
  uint4* const stores = reinterpret_cast<uint4*>(ring + kRowStages * slot_bytes) + tid / 32 * 65;
  auto put = [&](auto* row, int j, const float2(&f)[4]) {
    if constexpr (ANY) {
      const float o[8] = {f[0].x, f[0].y, f[1].x, f[1].y, f[2].x, f[2].y, f[3].x, f[3].y};
      const int count = cols - ((int)col[j] - (tid & 31) * 8);
      store8_any<std::remove_reference_t<decltype(*row)>, true>(row + col[j], o, n[j],
                                                                count < 256 ? count : 256, stores);
    } else {
      store4x2(row + col[j], f, true);
    }
  };
  auto get = [&](const void* p, int64_t r, int64_t rows, int j) {  // of row r, cols apart
    return load8_any<T, ANY>(static_cast<const T*>(p) + r * cols + col[j], ANY ? n[j] : on[j] ? 8 : 0,
                             cols >= 16 && r > 0 && r < rows - 1);
  };
  // row r of a tensor with leading dimension ld: the same for the CTA, columns are added
  auto row_of = [](auto* p, int64_t ld, int64_t r) { return p + r * ld; };
  auto copy = [&](uint32_t slot, int tensor, const T* p, int64_t ld, int64_t r, int64_t rows) {
    const T* row = row_of(p, ld, r);
    if constexpr (ANY) {
      const uintptr_t at = reinterpret_cast<uintptr_t>(row), first = at & ~(uintptr_t)15;
      const int words = (int)((at - first) + cols * sizeof(T) + 15) / 16;
      const uintptr_t lo = reinterpret_cast<uintptr_t>(p),
                      hi = reinterpret_cast<uintptr_t>(p + ((rows - 1) * ld + cols));
      // with rows before and behind, all words are the operand's
      const bool inside = cols >= 16 && r > 0 && r < rows - 1;
      for (int k = tid; k < words; k += nt) {
        const uintptr_t q = first + 16 * (uintptr_t)k;
        const uint32_t to = slot + tensor * kTensor + 16 * k;
        if (inside || (q >= lo && q + 16 <= hi)) {
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(q) : "memory");
        } else {  // an end of the operand: its elements alone
          for (int i = 0; i < 16; i += (int)sizeof(T))
            if (q + i >= lo && q + i + sizeof(T) <= hi)
              *reinterpret_cast<T*>(ring + (to - base) + i) = *reinterpret_cast<const T*>(q + i);
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (on[j]) {
#pragma unroll
          for (int w = 0; w < W; ++w)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                             slot + tensor * kTensor + (j * W + w) * kStride),
                         "l"(reinterpret_cast<const uint4*>(row + col[j]) + w)
                         : "memory");
        }
    }
  };
  const T *pdh = static_cast<const T*>(a.dh), *pv = static_cast<const T*>(a.v);
  const T *px = static_cast<const T*>(a.dx_out), *py = static_cast<const T*>(a.y);
  const T* const pg = static_cast<const T*>(a.gate);
  const int64_t gates = a.gate ? (a.rows - 1) / a.rows_per_gate + 1 : 0;
  auto ask = [&](uint32_t slot, int64_t r) {
    if (r < r1) {
      if (has_h) {
        copy(slot, 0, pdh, a.ld_dh, r, a.rows);
        copy(slot, 1, pv, a.ld_v, r, a.rows);
      }
      if (has_x) copy(slot, 2, px, a.ld_dx_out, r, a.rows);
      if (has_y) copy(slot, 3, py, a.ld_y, r, a.rows);
      if (FEW) copy(slot, 4, pg, a.cols, r / a.rows_per_gate, gates);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  uint32_t off[FEW ? 5 : 4];  // ANY: bytes of the row at hand past an aligned word
  auto fetch = [&](uint32_t slot, int tensor, int j, float2 (&f)[4]) {
    Raw8<T> r;
    if constexpr (ANY) {
      const uint4* q = reinterpret_cast<const uint4*>(ring + (slot - base) + tensor * kTensor) +
                       (j * nt + tid) * W;
      uint4 w[W + 1];
#pragma unroll
      for (int i = 0; i <= W; ++i) w[i] = q[i];
#pragma unroll
      for (int i = 0; i < W; ++i) r.w[i] = shift16(w[i], w[i + 1], off[tensor]);
    } else {
#pragma unroll
      for (int w = 0; w < W; ++w)
        r.w[w] = *static_cast<const uint4*>(
            __cvta_shared_to_generic(slot + tensor * kTensor + (j * W + w) * kStride));
    }
    unpack4x2(r, f);
    if (ANY && n[j] < 8) {  // past the row's end: zeros
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (2 * i >= n[j]) f[i].x = 0.0f;
        if (2 * i + 1 >= n[j]) f[i].y = 0.0f;
      }
    }
  };
  for (int s = 0; s < plan.stages; ++s) ask(base + s * slot_bytes, r0 + s);
  if (ANY) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kRowStages - 1) : "memory");
    __syncthreads();
  }

  Raw8<T> wq[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j)
    if (kKeep && has_h) wq[j] = get(a.w_pre, 0, 1, j);
  float2 dwq[NV][4], dwp[NV][4], z[NV][4], gw[NV][4];
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) dwq[j][i] = dwp[j][i] = z[j][i] = both(0.0f);

  const float mean = 1.0f / (float)a.cols;
  const int64_t first_gate = a.gate ? r0 / a.rows_per_gate : 0;
  int64_t gate = first_gate - 1, next_gate = r0;  // the row that starts the next gate
  float* const my_part = part + (int64_t)blockIdx.x * 2 * pitch;
  bool again = false;  // dw_post has a part already
  // eight values of w_post, of a gate's row: ones where there is none
  auto ones = [](float2 (&f)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = both(1.0f);
  };
  auto post_of = [&](int j, float2 (&f)[4]) {
    ones(f);
    if (norm_y) unpack4x2(get(a.w_post, 0, 1, j), f);
  };
  auto gate_of = [&](int64_t g, int j, float2 (&f)[4]) {
    ones(f);
    if (a.gate) unpack4x2(get(a.gate, g, gates, j), f);
  };
  // gradients of the gate that ends before row r (its last row here is r - 1)
  auto leave_gate = [&](int64_t r) {
    const bool whole = a.gate && gate * a.rows_per_gate >= r0 &&
                       (r == a.rows || (gate + 1) * a.rows_per_gate <= r);
    float* slot_at = slots + (2 * (int64_t)blockIdx.x + (gate == first_gate ? 0 : 1)) * pitch;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (!on[j]) continue;
      float2 f[4];
      if (a.dgate) {
        post_of(j, f);
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = mul2(mul2(f[i], both(a.beta)), z[j][i]);
        if (!whole) {
          if (live(j)) store4x2(slot_at + col[j], f, true);
        } else if (ANY) {
          put(a.dgate + gate * a.cols, j, f);
        } else {
          store4x2(a.dgate + gate * a.cols + col[j], f, a.dgate_vec);
        }
      }
      if (a.dw_post) {
        gate_of(gate, j, f);
        if (!FEW && again) {
          Raw8<float> old;
          old = load8(my_part + pitch + col[j], 0, true);
          if (live(j)) {
            old.w[0] = reinterpret_cast<const uint4*>(my_part + pitch + col[j])[0];
            old.w[1] = reinterpret_cast<const uint4*>(my_part + pitch + col[j])[1];
          }
          unpack4x2(old, dwp[j]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) dwp[j][i] = fma2(mul2(f[i], both(a.beta)), z[j][i], dwp[j][i]);
        if (!FEW && live(j)) store4x2(my_part + pitch + col[j], dwp[j], true);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) z[j][i] = both(0.0f);
    }
    again = true;
  };
  uint32_t slot = base, before = base;
  const uint32_t last_slot = base + (plan.stages - 1) * slot_bytes;
  float next_r2 = has_h && r0 < r1 ? __ldg(a.rstd_pre + r0) : 0.0f;
  float next_rp = norm_y && r0 < r1 ? __ldg(a.rstd_post + r0) : 1.0f;
  for (int64_t r = r0; r < r1; ++r) {
    const float r2 = next_r2, rp = next_rp;
    if (r + 1 < r1) {
      if (has_h) next_r2 = __ldg(a.rstd_pre + r + 1);
      if (norm_y) next_rp = __ldg(a.rstd_post + r + 1);
    }
    const bool renew = has_y && r == next_gate;
    if (renew) {
      if (r > r0) leave_gate(r);
      ++gate;
      next_gate = a.gate ? (gate + 1) * a.rows_per_gate : r1;
    }
    if (renew && !FEW) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (!on[j]) continue;
        float2 g[4];
        post_of(j, gw[j]);
        gate_of(gate, j, g);
#pragma unroll
        for (int i = 0; i < 4; ++i) gw[j][i] = mul2(gw[j][i], g[i]);
      }
    }
    if (ANY) {
      auto past = [&](const T* p, int64_t ld, int64_t row) {
        return (uint32_t)reinterpret_cast<uintptr_t>(row_of(p, ld, row)) & 15u;
      };
      off[0] = past(pdh, a.ld_dh, r);
      off[1] = past(pv, a.ld_v, r);
      off[2] = past(px, a.ld_dx_out, r);
      off[3] = past(py, a.ld_y, r);
      if (FEW) off[4] = past(pg, a.cols, r / a.rows_per_gate);
    } else if (plan.stages == kRowStages) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kRowStages - 1) : "memory");
    } else {
      asm volatile("cp.async.wait_group 1;" ::: "memory");
    }
    if (renew && FEW) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (!on[j]) continue;
        float2 g[4];
        post_of(j, gw[j]);
        fetch(slot, 4, j, g);
#pragma unroll
        for (int i = 0; i < 4; ++i) gw[j][i] = mul2(gw[j][i], g[i]);
      }
    }
    // u: dv without the mean's part, dx_out + r2 p
    float2 sum[3] = {both(0.0f), both(0.0f), both(0.0f)}, u[NV][4];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float2 v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) u[j][i] = v[i] = both(0.0f);
      if (!on[j]) continue;
      if (has_x) fetch(slot, 2, j, u[j]);
      if (has_h) {
        float2 p[4], w[4];
        fetch(slot, 0, j, p);
        fetch(slot, 1, j, v);
        unpack4x2(kKeep ? wq[j] : get(a.w_pre, 0, 1, j), w);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[i] = mul2(v[i], both(r2));
          dwq[j][i] = fma2(p[i], v[i], dwq[j][i]);
          p[i] = mul2(p[i], w[i]);
          sum[0] = fma2(p[i], v[i], sum[0]);
          u[j][i] = fma2(p[i], both(r2), u[j][i]);
        }
      }
      if (norm_y) {
        float2 y[4];
        fetch(slot, 3, j, y);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 qy = mul2(gw[j][i], mul2(y[i], both(rp)));
          sum[1] = fma2(qy, u[j][i], sum[1]);
          sum[2] = fma2(qy, v[i], sum[2]);
        }
      }
    }
    float s[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) s[k] = sum[k].x + sum[k].y;
    if (ANY) {
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      row_sum_cta(s, red[(r - r0) & 1]);
      if (r > r0) ask(before, r - 1 + kRowStages);
    } else if (has_h || norm_y) {
      row_sum(s, red[(r - r0) & 1]);
    }
    // of v^ and of y^
    const float c2 = r2 * (s[0] * mean);
    const float c1 = rp * ((s[1] - c2 * s[2]) * mean * a.beta), rb = rp * a.beta;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (!on[j]) continue;
      float2(&dv)[4] = u[j];
      float2 o[4];
      if (has_h) {
        float2 v[4];
        fetch(slot, 1, j, v);
#pragma unroll
        for (int i = 0; i < 4; ++i) dv[i] = fma2(mul2(v[i], both(r2)), both(-c2), dv[i]);
      }
      if (out_x) {
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = mul2(dv[i], both(a.alpha));
        put(row_of(static_cast<T*>(a.dx), a.ld_dx, r), j, o);
      }
      if (has_y) {
        float2 y[4];
        fetch(slot, 3, j, y);
        // dy = beta r1 g w dv - y^ c1
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          y[i] = mul2(y[i], both(rp));
          z[j][i] = fma2(y[i], dv[i], z[j][i]);
          o[i] = mul2(gw[j][i], mul2(dv[i], both(rb)));
          if (norm_y) o[i] = fma2(y[i], both(-c1), o[i]);
        }
        if (out_y) put(row_of(static_cast<T*>(a.dy), a.ld_dy, r), j, o);
      }
    }
    if (!ANY) ask(slot, r + plan.stages);
    before = slot;
    slot = slot == last_slot ? base : slot + slot_bytes;
  }
  if (has_y && r1 > r0) leave_gate(r1);
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    if (!live(j)) continue;
    if (a.dw_pre) store4x2(my_part + col[j], dwq[j], true);
    if (a.dw_post && (FEW || r1 == r0)) store4x2(my_part + pitch + col[j], dwp[j], true);
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// Adds what grad_rows_kernel left in parts, 32 columns a CTA: blockIdx.y 0 dw_pre, 1
// dw_post, 2 + b the gate that CTA b is the first of several to have.
__global__ void __launch_bounds__(512) grad_rows_sum_kernel(const ResidualNormGradArgs a, int64_t ctas,
                                                            const float* part, const float* slots) {
  __shared__ float red[16][32];
  const int64_t c = (int64_t)blockIdx.x * 32 + threadIdx.x;
  const float* src;
  float* out;
  const int64_t pitch = (a.cols + 7) / 8 * 8;
  int64_t first = 0, count = ctas;
  bool odd_first = false;  // the first term lies in the first CTA's second slot
  if (blockIdx.y < 2) {
    out = blockIdx.y == 0 ? a.dw_pre : a.dw_post;
    src = part + blockIdx.y * pitch;
    if (!out) return;
  } else {
    const int64_t b = blockIdx.y - 2, per = a.rows_per_gate;
    const int64_t r0 = first_row(b, a.rows, ctas), r1 = first_row(b + 1, a.rows, ctas);
    if (r0 == r1) return;
    const int64_t g = (r1 - 1) / per, end = (g + 1) * per < a.rows ? (g + 1) * per : a.rows;
    if (end <= r1 || g * per < r0) return;  // the CTA has all of it, or not its start
    first = b;
    count = (end * ctas - 1) / a.rows - b + 1;
    odd_first = g != r0 / per;
    out = a.dgate + g * a.cols;
    src = slots;
  }
  float s = 0.0f;
  if (c < a.cols) {
#pragma unroll 4
    for (int64_t i = threadIdx.y; i < count; i += 16)
      s += __ldcg(src + (first + i) * 2 * pitch + (odd_first && i == 0 ? pitch : 0) + c);
  }
  red[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && c < a.cols) {
#pragma unroll
    for (int i = 1; i < 16; ++i) s += red[i][threadIdx.x];
    out[c] = s;
  }
}

// The launch of grad_rows_kernel, or threads 0 where the two passes serve: rows so wide that
// enough of them do not fit a CTA's shared memory or its registers.
GradRows grad_rows(int type, const ResidualNormGradArgs& a, int sm_count) {
  GradRows p;
  memset(&p, 0, sizeof(p));
  const int64_t v = (a.cols + 7) / 8;
  if (v > 1024) return p;
  p.any = !a.vec || a.cols % 8;
  const int es = type == B2G_F32 ? 4 : 2;
  // sixteen columns a thread only where eight do not do: 32768 x 4096 354 us with sixteen, 339
  // with eight, 65536 x 2048 431 and 316
  p.nv = v > 512 ? 2 : 1;
  const int threads = ((int)((v + p.nv - 1) / p.nv) + 31) / 32 * 32;
  p.max_threads = threads > 256 ? 512 : threads > 128 ? 256 : 128;
  // FEW; a gate per 4 rows of 8192 485 us so, 559 without, per 7 of 4096 265 and 259
  p.gate_rows = a.gate && a.rows_per_gate < 8 && a.rows_per_gate < a.rows;
  const size_t stage = grad_stage(p.max_threads, p.nv, es, p.gate_rows);
  // CTAs on an SM: by registers (128 a thread) and shared memory
  int on_sm = 512 / p.max_threads;
  p.stages = kRowStages;
  if (!p.any && p.stages * stage * on_sm > kGradRoom) p.stages = 2;
  p.smem = grad_smem(p.stages, stage, p.max_threads, p.any);
  while (on_sm > 1 && p.smem * on_sm > kGradRoom) --on_sm;
  if (p.smem > kGradRoom) return p;
  const int64_t most = (int64_t)on_sm * sm_count;
  // at least two rows a CTA: each costs its sums' way through memory
  const int64_t want = (a.rows + 1) / 2;
  p.ctas = (int)(want < most ? want : most);
  p.threads = threads;
  return p;
}

template <typename T, int NV, int MAXT, bool ALL, bool FEW, bool ANY>
cudaError_t grad_rows_main(const ResidualNormGradArgs& a, const GradRows& p, float* part, float* slots,
                           cudaStream_t s) {
  // grad_rows() chooses no form whose slots do not fit
  constexpr size_t least =
      grad_smem(ANY ? kRowStages : 2, grad_stage(MAXT, NV, sizeof(T), FEW), MAXT, ANY);
  if constexpr (least > kGradRoom) {
    return cudaErrorInvalidConfiguration;
  } else {
    static std::atomic<int> seen[16];
    const cudaError_t e = allow_smem(grad_rows_kernel<T, NV, MAXT, ALL, FEW, ANY>, (int)p.smem, seen);
    if (e != cudaSuccess) return e;
    grad_rows_kernel<T, NV, MAXT, ALL, FEW, ANY><<<p.ctas, p.threads, p.smem, s>>>(a, p, part, slots);
    return cudaGetLastError();
  }
}

template <typename T, bool ALL, bool FEW, bool ANY>
cudaError_t grad_rows_shape(const ResidualNormGradArgs& a, const GradRows& p, float* part, float* slots,
                            cudaStream_t s) {
  if (p.nv == 2) return grad_rows_main<T, 2, 512, ALL, FEW, ANY>(a, p, part, slots, s);
  if (p.max_threads == 128) return grad_rows_main<T, 1, 128, ALL, FEW, ANY>(a, p, part, slots, s);
  if (p.max_threads == 256) return grad_rows_main<T, 1, 256, ALL, FEW, ANY>(a, p, part, slots, s);
  return grad_rows_main<T, 1, 512, ALL, FEW, ANY>(a, p, part, slots, s);
}

template <typename T, bool ALL, bool FEW>
cudaError_t grad_rows_any(const ResidualNormGradArgs& a, const GradRows& p, float* part, float* slots,
                          cudaStream_t s) {
  return p.any ? grad_rows_shape<T, ALL, FEW, true>(a, p, part, slots, s)
               : grad_rows_shape<T, ALL, FEW, false>(a, p, part, slots, s);
}

template <typename T>
cudaError_t grad_rows_launch(const ResidualNormGradArgs& a, const GradRows& p, cudaStream_t s) {
  float* part = static_cast<float*>(a.ws);
  float* slots = part + (size_t)p.ctas * 2 * ((a.cols + 7) / 8 * 8);
  const bool all = a.dh && a.dx_out && a.y && a.w_post && a.dx && a.dy;
  cudaError_t e;
  if (p.gate_rows)
    e = all ? grad_rows_any<T, true, true>(a, p, part, slots, s)
            : grad_rows_any<T, false, true>(a, p, part, slots, s);
  else
    e = all ? grad_rows_any<T, true, false>(a, p, part, slots, s)
            : grad_rows_any<T, false, false>(a, p, part, slots, s);
  if (e != cudaSuccess) return e;
  // gates of one row never meet two CTAs
  const unsigned gates = a.dgate && a.rows_per_gate > 1 ? (unsigned)p.ctas : 0u;
  if (a.dw_pre || a.dw_post || gates)
    grad_rows_sum_kernel<<<dim3((unsigned)((a.cols + 31) / 32), 2 + gates), dim3(32, 16), 0, s>>>(
        a, p.ctas, part, slots);
  return cudaGetLastError();
}

// Row means: stat[row] = {r2 A / D, beta r1 (B - r2 (A / D) C) / D}, which multiply v^ and y^
// (the second is 0 without w_post).
template <typename T, bool ANY>
__global__ void __launch_bounds__(256) grad_stat_kernel(const ResidualNormGradArgs a, float2* stat) {
  __shared__ float red[3 * 32];
  const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  if (row >= a.rows) return;
  const int span = blockDim.x;
  const float r2 = a.dh ? a.rstd_pre[row] : 0.0f;
  const float r1 = a.w_post ? a.rstd_post[row] : 0.0f;
  float s[3] = {0.0f, 0.0f, 0.0f};
  const int cols = (int)a.cols;
  for (int c = threadIdx.x * 8; c < cols; c += span * 8) {
    const int n = cols - c < 8 ? cols - c : 8;
    // columns c .. of row r of an operand with `rows` rows, ld apart
    auto get = [&](const void* p, int64_t r, int64_t ld, int64_t rows, float (&f)[8]) {
      unpack8(load8_any<T, ANY>(static_cast<const T*>(p) + r * ld + c, n,
                                cols >= 16 && r > 0 && r < rows - 1), f);
    };
    float p[8] = {0, 0, 0, 0, 0, 0, 0, 0}, v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (a.dh) {
      float w[8];
      get(a.dh, row, a.ld_dh, a.rows, p);
      get(a.v, row, a.ld_v, a.rows, v);
      get(a.w_pre, 0, 0, 1, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        p[i] *= w[i];
        v[i] *= r2;
        s[0] = fmaf(p[i], v[i], s[0]);
      }
    }
    if (a.w_post) {
      float y[8], w[8], d[8] = {0, 0, 0, 0, 0, 0, 0, 0};
      get(a.y, row, a.ld_y, a.rows, y);
      get(a.w_post, 0, 0, 1, w);
      if (a.dx_out) get(a.dx_out, row, a.ld_dx_out, a.rows, d);
      if (a.gate) {
        float g[8];
        get(a.gate, row / a.rows_per_gate, a.cols, (a.rows - 1) / a.rows_per_gate + 1, g);
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] *= g[i];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float qy = w[i] * (y[i] * r1);
        s[1] = fmaf(qy, fmaf(r2, p[i], d[i]), s[1]);
        s[2] = fmaf(qy, v[i], s[2]);
      }
    }
  }
  row_sum(s, red);
  if (threadIdx.x == 0) {
    const float m = 1.0f / (float)a.cols;
    const float c2 = r2 * (s[0] * m);
    stat[row] = make_float2(c2, r1 * ((s[1] - c2 * s[2]) * m * a.beta));
  }
}

// How the column pass cuts the rows: a chunk of whole gates (their dgate rows are then
// written directly) where a gate has few rows, else chunks within one gate.
struct GradChunks {
  bool whole;         // a chunk holds whole gates
  int64_t per;        // rows of a gate (all rows without one)
  int64_t gates;
  int64_t rows;       // rows of a chunk (whole: a multiple of per)
  int64_t per_gate;   // chunks of a gate (whole: unused)
  int64_t chunks;
};
constexpr int kLanes = 8;       // rows a column CTA works on at once
constexpr int kGradCols = 256;  // columns of a column CTA

GradChunks grad_chunks(const ResidualNormGradArgs& a, int sm_count) {
  GradChunks c;
  c.per = a.gate && a.rows_per_gate < a.rows ? a.rows_per_gate : a.rows;
  c.gates = (a.rows + c.per - 1) / c.per;
  // chunks of 16 to 128 rows, about four CTAs an SM
  const int64_t col_tiles = (a.cols + kGradCols - 1) / kGradCols;
  int64_t r = a.rows * col_tiles / (4 * (int64_t)sm_count);
  r = r < 16 ? 16 : r > 128 ? 128 : r;
  c.whole = c.gates > 1 && c.per <= r;
  if (c.whole) {
    c.rows = r / c.per * c.per;
    c.per_gate = 0;
    c.chunks = (a.rows + c.rows - 1) / c.rows;
  } else {
    c.rows = r;
    c.per_gate = (c.per + r - 1) / r;
    c.chunks = c.gates * c.per_gate;
  }
  return c;
}

// Column pass: 256 columns (eight a thread) of one chunk of rows, a row per warp.  Sums
// over the chunk go to part[chunk][3][cols] (dw_pre, dw_post, dgate).
template <typename T, bool ANY>
__global__ void __launch_bounds__(256) grad_cols_kernel(const ResidualNormGradArgs a, GradChunks ck,
                                                        const float2* stat, float* part) {
  __shared__ float red[kLanes][kGradCols];
  const int lane = threadIdx.x, ry = threadIdx.y;
  const int64_t chunk = blockIdx.x;
  __shared__ uint4 gate_stores[kLanes][65];
  __shared__ uint4 stores[ANY ? kLanes : 1][2 * sizeof(T) * 8 + 1];
  const int cols = (int)a.cols, c0 = (int)blockIdx.y * kGradCols, c = c0 + lane * 8;
  const int n = c >= cols ? 0 : cols - c < 8 ? cols - c : 8;
  const int count = cols - c0 < 256 ? cols - c0 : 256;
  // columns c .. of row r of an operand with `rows` rows, ld apart
  auto get = [&](const void* p, int64_t r, int64_t ld, int64_t rows, float (&f)[8]) {
    unpack8(load8_any<T, ANY>(static_cast<const T*>(p) + r * ld + c, n,
                              cols >= 16 && r > 0 && r < rows - 1), f);
  };
  auto put = [&](void* p, int64_t r, int64_t ld, const float(&f)[8]) {
    store8_any<T, ANY>(static_cast<T*>(p) + r * ld + c, f, n, count, stores[ANY ? ry : 0]);
  };
  int64_t r0, r1;
  if (ck.whole) {
    r0 = chunk * ck.rows;
    r1 = r0 + ck.rows;
  } else {
    const int64_t g = chunk / ck.per_gate;
    r0 = g * ck.per + chunk % ck.per_gate * ck.rows;
    r1 = r0 + ck.rows < (g + 1) * ck.per ? r0 + ck.rows : (g + 1) * ck.per;
  }
  if (r1 > a.rows) r1 = a.rows;
  float wq[8], wp[8], g[8];
  if (a.w_post) get(a.w_post, 0, 0, 1, wp);
  if (a.dh) get(a.w_pre, 0, 0, 1, wq);
  float dwq[8], dwp[8], dg[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    dwq[i] = dwp[i] = dg[i] = 0.0f;
    g[i] = 1.0f;
    if (!a.w_post) wp[i] = 1.0f;
    if (!a.dh) wq[i] = 0.0f;
  }
  // rows of this thread: whole gates in turn, or every kLanes-th row of the chunk
  const int64_t run = ck.whole ? ck.per : 1;
  for (int64_t rb = r0 + ry * run; rb < r1; rb += kLanes * run) {
    const int64_t re = rb + run < r1 ? rb + run : r1;
    if (a.gate && (ck.whole || rb == r0 + ry * run))
      get(a.gate, rb / ck.per, a.cols, ck.gates, g);
    for (int64_t r = rb; r < re; ++r) {
      const float2 st = stat[r];
      float dv[8] = {0, 0, 0, 0, 0, 0, 0, 0};
      if (a.dx_out) get(a.dx_out, r, a.ld_dx_out, a.rows, dv);
      if (a.dh) {
        const float r2 = a.rstd_pre[r];
        float dh[8], v[8];
        get(a.dh, r, a.ld_dh, a.rows, dh);
        get(a.v, r, a.ld_v, a.rows, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          v[i] *= r2;
          dv[i] += r2 * (wq[i] * dh[i]) - v[i] * st.x;
          dwq[i] = fmaf(dh[i], v[i], dwq[i]);
        }
      }
      float o[8];
      if (a.dx) {
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = a.alpha * dv[i];
        put(a.dx, r, a.ld_dx, o);
      }
      if (a.y) {
        const float r1s = a.w_post ? a.rstd_post[r] : 1.0f;
        float y[8];
        get(a.y, r, a.ld_y, a.rows, y);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float bd = a.beta * dv[i], yh = y[i] * r1s, dz = bd * g[i];
          dg[i] = fmaf(bd * wp[i], yh, dg[i]);
          dwp[i] = fmaf(dz, yh, dwp[i]);
          o[i] = r1s * wp[i] * dz - yh * st.y;
        }
        if (a.dy) put(a.dy, r, a.ld_dy, o);
      }
    }
    if (ck.whole && a.dgate) {
      store8_any<float, true>(a.dgate + rb / ck.per * a.cols + c, dg, n, count, gate_stores[ry]);
#pragma unroll
      for (int i = 0; i < 8; ++i) dg[i] = 0.0f;
    }
  }
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    const float(&acc)[8] = k == 0 ? dwq : k == 1 ? dwp : dg;
    const bool on = k == 0 ? a.dw_pre != nullptr : k == 1 ? a.dw_post != nullptr
                                                          : a.dgate != nullptr && !ck.whole;
    if (!on) continue;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) red[ry][lane * 8 + i] = acc[i];
    __syncthreads();
    const int t = ry * 32 + lane;
    float sum = 0.0f;
#pragma unroll
    for (int l = 0; l < kLanes; ++l) sum += red[l][t];
    const int64_t cc = (int64_t)blockIdx.y * kGradCols + t;
    if (cc < a.cols) part[(chunk * 3 + k) * a.cols + cc] = sum;
  }
}

// out[g][c] = sum of count rows of part (stride row_stride floats) from row first + g *
// count on, for 32 columns of one g: 32 threads along the columns, 8 down the rows.
__global__ void __launch_bounds__(256) grad_sum_kernel(const float* part, int64_t row_stride,
                                                       int64_t count, int64_t cols, float* out) {
  __shared__ float red[8][32];
  const int64_t c = (int64_t)blockIdx.y * 32 + threadIdx.x, g = blockIdx.x;
  float s = 0.0f;
  if (c < cols)
    for (int64_t i = threadIdx.y; i < count; i += 8) s += part[(g * count + i) * row_stride + c];
  red[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && c < cols) {
#pragma unroll
    for (int i = 1; i < 8; ++i) s += red[i][threadIdx.x];
    out[g * cols + c] = s;
  }
}

template <typename T>
cudaError_t grad_launch(int type, const ResidualNormGradArgs& a, int sm_count, cudaStream_t s) {
  const GradRows p = grad_rows(type, a, sm_count);
  if (p.threads) return grad_rows_launch<T>(a, p, s);
  const GradChunks ck = grad_chunks(a, sm_count);
  float2* stat = static_cast<float2*>(a.ws);
  float* part = reinterpret_cast<float*>(stat + (a.rows + 15) / 16 * 16);
  const int64_t v = (a.cols + 7) / 8;
  const int tpr = v <= 32 ? 32 : v <= 64 ? 64 : v <= 128 ? 128 : 256;
  const int rpc = tpr == 32 ? 4 : 1;
  const unsigned stat_grid = (unsigned)((a.rows + rpc - 1) / rpc);
  const unsigned col_tiles = (unsigned)((a.cols + kGradCols - 1) / kGradCols);
  const dim3 cols_grid((unsigned)ck.chunks, col_tiles), cols_block(32, kLanes);
  if (a.vec) {
    grad_stat_kernel<T, false><<<stat_grid, dim3(tpr, rpc), 0, s>>>(a, stat);
    grad_cols_kernel<T, false><<<cols_grid, cols_block, 0, s>>>(a, ck, stat, part);
  } else {
    grad_stat_kernel<T, true><<<stat_grid, dim3(tpr, rpc), 0, s>>>(a, stat);
    grad_cols_kernel<T, true><<<cols_grid, cols_block, 0, s>>>(a, ck, stat, part);
  }
  const unsigned sums = (unsigned)((a.cols + 31) / 32);
  if (a.dw_pre)
    grad_sum_kernel<<<dim3(1, sums), dim3(32, 8), 0, s>>>(part, 3 * a.cols, ck.chunks, a.cols, a.dw_pre);
  if (a.dw_post)
    grad_sum_kernel<<<dim3(1, sums), dim3(32, 8), 0, s>>>(part + a.cols, 3 * a.cols, ck.chunks, a.cols,
                                                          a.dw_post);
  if (a.dgate && !ck.whole)
    grad_sum_kernel<<<dim3((unsigned)ck.gates, sums), dim3(32, 8), 0, s>>>(
        part + 2 * a.cols, 3 * a.cols, ck.per_gate, a.cols, a.dgate);
  return cudaGetLastError();
}

}  // namespace

size_t norm_grad_ws_bytes(int type, const ResidualNormGradArgs& a, int sm_count) {
  const GradRows p = grad_rows(type, a, sm_count);
  if (p.threads) return (size_t)p.ctas * 4 * (size_t)((a.cols + 7) / 8 * 8) * sizeof(float);
  const GradChunks ck = grad_chunks(a, sm_count);
  return (size_t)(a.rows + 15) / 16 * 16 * sizeof(float2) +
         (size_t)ck.chunks * 3 * (size_t)a.cols * sizeof(float);
}

cudaError_t launch_residual_norm_grad(int type, const ResidualNormGradArgs& a, int sm_count,
                                      cudaStream_t s) {
  if (type == B2G_F32) return grad_launch<float>(type, a, sm_count, s);
  if (type == B2G_BF16) return grad_launch<__nv_bfloat16>(type, a, sm_count, s);
  return grad_launch<__half>(type, a, sm_count, s);
}

}  // namespace b2g
