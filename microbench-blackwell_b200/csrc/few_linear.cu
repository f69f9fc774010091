// few_linear.cu -- y = alpha * x . W^T of a few tokens (16-bit x) with microscaled
// weights, for decoding: every weight is read once and used a handful of times, so the
// kernel is bound by the weights' bytes.
//
// Codes become fp16 pairs in registers and go into mma.sync m16n8k16 with the weights
// as the 16-row operand and up to 8 tokens as the 8 columns: tcgen05 takes its operands
// from shared or tensor memory, so a decoded weight would have to be stored first, for
// products whose own time does not count at this many tokens.  e2m1 and e4m3 values and
// e2m1 * ue4m3 products are exact in fp16; sums are fp32.  x becomes fp16 in a first
// kernel: fp16 as it is, bf16 scaled per token by the power of two that brings its
// largest value to 2^14 .. 2^15, which is exact for values down to 2^-28 of the largest
// (below that the error is at most 2^-40 of the largest).
#include "b2g.h"
#include "op_common.cuh"
#include "op_kernels.h"

namespace b2g {
namespace {

constexpr int kWarps = 8;

// k-order inside the kernel: a thread takes 16 bytes of codes of a row at a time
// (kSpan elements), the four threads of a quad 4 * kSpan neighbouring elements (a
// group); MMA step j of a group multiplies elements 4 j .. 4 j + 3 of each thread.  Any
// order of k serves as long as both operands use it, so no code is moved between
// threads.
__host__ __device__ constexpr int few_span(int fmt) { return 128 / bf_bits(fmt); }

// x as fp16 B fragments: [group][token tile][step pair][lane] of 16 bytes, the lane's
// four elements of two steps; xs[token] = the power of two to undo.  One CTA per token
// of the padded tiles (zeros past T).
template <typename T, int FMT>
__global__ void __launch_bounds__(512) few_prepare_kernel(const FewLinearArgs a, uint4* frag,
                                                          float* xs, int tiles) {
  __shared__ float red[16];
  constexpr int span = few_span(FMT);
  const int token = blockIdx.x, tile = token >> 3;
  const int64_t vecs = (a.kp + 4 * span - 1) / (4 * span) * (4 * span) / 8;
  const T* x = static_cast<const T*>(a.x) + (int64_t)token * a.ld_x;
  const bool on = token < a.T;
  float scale = 1.0f;
  if constexpr (sizeof(T) == 2 && !__is_same(T, __half)) {
    float amax = 0.0f;
    for (int64_t v = threadIdx.x; v < vecs; v += blockDim.x) {
      const int64_t c = v * 8, left = a.K - c;
      float f[8];
      unpack8(load8(x + c, !on || left < 0 ? 0 : left < 8 ? (int)left : 8, a.x_vec), f);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float m = fabsf(f[i]);
        amax = fmaxf(amax, m < __uint_as_float(0x7F800000u) ? m : 0.0f);  // of the finite ones
      }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, o));
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = amax;
    __syncthreads();
    amax = red[0];
    for (int i = 1; i < (int)(blockDim.x >> 5); ++i) amax = fmaxf(amax, red[i]);
    // exponent field of 2^(14 - floor(log2 amax)), at most 2^126
    int e = 127 + 14 - ((int)(__float_as_uint(amax) >> 23) - 127);
    e = e > 253 ? 253 : e;
    scale = amax > 0.0f ? __uint_as_float((uint32_t)e << 23) : 1.0f;
  }
  if (threadIdx.x == 0) xs[token] = 1.0f / scale;
  for (int64_t v = threadIdx.x; v < vecs; v += blockDim.x) {
    const int64_t c = v * 8, left = a.K - c;
    float f[8];
    unpack8(load8(x + c, !on || left < 0 ? 0 : left < 8 ? (int)left : 8, a.x_vec), f);
    // eight elements: one step pair of one thread
    const int64_t group = c / (4 * span);
    const int in = (int)(c % (4 * span)), t = in / span, jp = in % span / 8;
    const int lane = (token & 7) * 4 + t;
    uint4 w;
    w.x = pack2<__half>(f[0] * scale, f[1] * scale);
    w.y = pack2<__half>(f[2] * scale, f[3] * scale);
    w.z = pack2<__half>(f[4] * scale, f[5] * scale);
    w.w = pack2<__half>(f[6] * scale, f[7] * scale);
    frag[((group * tiles + tile) * (span / 8) + jp) * 32 + lane] = w;
  }
}

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                        uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t mul_h2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

__device__ __forceinline__ uint32_t word_of(const uint4& v, int i) {
  return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
}

// fp16 pairs of the eight elements of steps 2 jp and 2 jp + 1 of 16 bytes of codes
template <int FMT>
__device__ __forceinline__ void decode_steps(const uint4& codes, int jp, uint32_t (&p)[4]) {
  if constexpr (FMT == BF_MXF8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint16_t w = (uint16_t)(word_of(codes, 2 * jp + (i >> 1)) >> (16 * (i & 1)));
      asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(p[i]) : "h"(w));
    }
  } else {
    e2m1x8_pairs(word_of(codes, jp), p);
  }
}

// Codes and scale bytes of one group: rows g and g + 8 of the warp's 16.
struct GroupData {
  uint4 w[2];
  uint32_t s[2];
};

template <int FMT>
__device__ __forceinline__ void load_group(const FewLinearArgs& a, const uint8_t* const (&w)[2],
                                           const uint8_t* const (&sf)[2], int64_t group, int t,
                                           bool on, GroupData& d) {
  constexpr int span = few_span(FMT);
  const int64_t k = group * 4 * span + t * span;
  on = on && k < a.kp;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    d.w[i] = make_uint4(0, 0, 0, 0);
    d.s[i] = 0;
    if (on) {
      d.w[i] = __ldcs(reinterpret_cast<const uint4*>(w[i] + k * bf_bits(FMT) / 8));
      if constexpr (FMT == BF_NVFP4)
        d.s[i] = __ldg(reinterpret_cast<const uint16_t*>(sf[i] + k / 16));
      else
        d.s[i] = __ldg(sf[i] + k / 32);
    }
  }
}

// 2^d as two fp16, d from -14 to 0
__device__ __forceinline__ uint32_t pow2_h2(int d) {
  return (uint32_t)(15 + d) * 0x04000400u;
}

// acc += (decoded, scaled codes of one group) . x
template <int FMT, int NT>
__device__ __forceinline__ void group_mma(const GroupData& d, const uint4* xf, float (&acc)[NT][4]) {
  constexpr int steps = few_span(FMT) / 4;
  const int lane = threadIdx.x & 31;
  if constexpr (FMT == BF_NVFP4) {
    // two scales a row, one for each 16 elements
    uint32_t h[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
      asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h[i]) : "h"((uint16_t)d.s[i]));
#pragma unroll
    for (int jp = 0; jp < steps / 2; ++jp) {
      uint32_t m[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) m[i] = __byte_perm(h[i], 0, jp < steps / 4 ? 0x1010 : 0x3232);
      uint32_t f[2][4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t p[4];
        decode_steps<FMT>(d.w[i], jp, p);
#pragma unroll
        for (int k = 0; k < 4; ++k) f[k >> 1][i + 2 * (k & 1)] = mul_h2(p[k], m[i]);
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const uint4 b = __ldg(xf + (n * (steps / 2) + jp) * 32 + lane);
        mma_f16(acc[n], f[0], b.x, b.y);
        mma_f16(acc[n], f[1], b.z, b.w);
      }
    }
  } else {
    // E8M0 scales have more range than fp16: within the group each row's codes are
    // scaled by 2^(s - ref) with ref the largest scale of the row's four threads, exact
    // down to 2^-14, and the sum by 2^ref in fp32.  A group with a wider range (blocks of
    // zeros apart, which are exact with any scale) is multiplied one thread's blocks
    // at a time, each with its own scale as ref.
    const int t = lane & 3;
    int s[2], ref[2];
    bool wide = false;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      s[i] = (int)d.s[i];
      ref[i] = max(s[i], __shfl_xor_sync(0xFFFFFFFFu, s[i], 1));
      ref[i] = max(ref[i], __shfl_xor_sync(0xFFFFFFFFu, ref[i], 2));
      wide |= s[i] < ref[i] - 14;
    }
    bool slow = __any_sync(0xFFFFFFFFu, wide);
    if (slow) {
      wide = false;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t any = (d.w[i].x | d.w[i].y | d.w[i].z | d.w[i].w) &
                             (FMT == BF_MXF8 ? 0x7F7F7F7Fu : 0x77777777u);
        if (!any) s[i] = max(s[i], ref[i] - 14);
        wide |= s[i] < ref[i] - 14;
      }
      slow = __any_sync(0xFFFFFFFFu, wide);
    }
#pragma unroll 1
    for (int p = 0; p < (slow ? 4 : 1); ++p) {
      uint32_t m[2];
      float f32s[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = slow ? __shfl_sync(0xFFFFFFFFu, s[i], (lane & ~3) + p) : ref[i];
        m[i] = slow ? (t == p ? 0x3C003C00u : 0u) : pow2_h2(s[i] - r);
        f32s[i] = e8m0_value((uint32_t)r);
      }
      float c[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) c[n][i] = 0.0f;
#pragma unroll
      for (int jp = 0; jp < steps / 2; ++jp) {
        uint32_t f[2][4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint32_t p[4];
          decode_steps<FMT>(d.w[i], jp, p);
#pragma unroll
          for (int k = 0; k < 4; ++k) f[k >> 1][i + 2 * (k & 1)] = mul_h2(p[k], m[i]);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const uint4 b = __ldg(xf + (n * (steps / 2) + jp) * 32 + lane);
          mma_f16(c[n], f[0], b.x, b.y);
          mma_f16(c[n], f[1], b.z, b.w);
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        acc[n][0] = fmaf(f32s[0], c[n][0], acc[n][0]);
        acc[n][1] = fmaf(f32s[0], c[n][1], acc[n][1]);
        acc[n][2] = fmaf(f32s[1], c[n][2], acc[n][2]);
        acc[n][3] = fmaf(f32s[1], c[n][3], acc[n][3]);
      }
    }
  }
}

// blockIdx: x row blocks of 16 * (kWarps / wk), y slices of K, z groups of 8 * NT tokens.
// The CTA's warps are wk slices of its K range by kWarps / wk row blocks.
struct FewShape {
  int wk, slices, tiles, groups, z;
};

template <typename T, int FMT, int NT>
__global__ void __launch_bounds__(kWarps * 32) few_linear_kernel(const FewLinearArgs a,
                                                                 const FewShape sh,
                                                                 const uint4* frag, const float* xs,
                                                                 float* part) {
  constexpr int span = few_span(FMT);
  __shared__ float red[kWarps][NT][128];
  __shared__ bool last;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int wr = kWarps / sh.wk;
  const int ks = blockIdx.y * sh.wk + warp % sh.wk;  // K slice of this warp
  const int nks = sh.slices * sh.wk;
  const int64_t row0 = ((int64_t)blockIdx.x * wr + warp / sh.wk) * 16;
  const uint8_t *w[2], *sf[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    int64_t r = row0 + g + 8 * i;
    r = r < a.N ? r : a.N - 1;  // rows past N repeat the last one and are not stored
    w[i] = a.w + r * a.kp * bf_bits(FMT) / 8;
    sf[i] = a.sf + r * a.kp / bf_block(FMT);
  }
  const int64_t gb = (int64_t)sh.groups * ks / nks, ge = (int64_t)sh.groups * (ks + 1) / nks;
  const int tile0 = blockIdx.z * NT;
  const uint4* xf = frag + (gb * sh.tiles + tile0) * (span / 8) * 32;
  const int64_t xstep = (int64_t)sh.tiles * (span / 8) * 32;
  float acc[NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[n][i] = 0.0f;

  // two groups at a time, the next two on their way
  GroupData cur[2], nxt[2];
  load_group<FMT>(a, w, sf, gb, t, gb < ge, cur[0]);
  load_group<FMT>(a, w, sf, gb + 1, t, gb + 1 < ge, cur[1]);
  for (int64_t gi = gb; gi < ge; gi += 2) {
    load_group<FMT>(a, w, sf, gi + 2, t, gi + 2 < ge, nxt[0]);
    load_group<FMT>(a, w, sf, gi + 3, t, gi + 3 < ge, nxt[1]);
    group_mma<FMT, NT>(cur[0], xf, acc);
    if (gi + 1 < ge) group_mma<FMT, NT>(cur[1], xf + xstep, acc);
    xf += 2 * xstep;
    cur[0] = nxt[0];
    cur[1] = nxt[1];
  }

  // accumulator i of lane (g, t): row g + 8 (i / 2), token 2 t + i % 2
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) red[warp][n][(2 * t + (i & 1)) * 16 + g + 8 * (i >> 1)] = acc[n][i];
  __syncthreads();
  const int64_t items = (int64_t)wr * NT * 128;
  float* mine = part + (((int64_t)blockIdx.z * gridDim.x + blockIdx.x) * sh.slices + blockIdx.y) * items;
  auto put = [&](int64_t item, float sum) {
    const int rb = (int)(item / (NT * 128)), e = (int)(item % (NT * 128));
    const int64_t token = (int64_t)(tile0 + e / 128) * 8 + e % 128 / 16;
    const int64_t row = ((int64_t)blockIdx.x * wr + rb) * 16 + e % 16;
    if (token < a.T && row < a.N)
      static_cast<T*>(a.out)[token * a.ld_out + row] = from_f32<T>(a.alpha * (sum * xs[token]));
  };
  for (int item = threadIdx.x; item < items; item += kWarps * 32) {
    const int rb = item / (NT * 128), e = item % (NT * 128);
    float sum = 0.0f;
    for (int k = 0; k < sh.wk; ++k) sum += red[rb * sh.wk + k][e / 128][e % 128];
    if (sh.slices == 1)
      put(item, sum);
    else
      mine[item] = sum;
  }
  if (sh.slices == 1) return;
  // the CTA that arrives last adds the slices, always in the same order
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) {
    uint32_t* c = a.count + (int64_t)blockIdx.z * gridDim.x + blockIdx.x;
    last = atomicAdd(c, 1u) == (uint32_t)sh.slices - 1u;
    if (last) *c = 0u;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  const float* all = part + ((int64_t)blockIdx.z * gridDim.x + blockIdx.x) * sh.slices * items;
  for (int item = threadIdx.x; item < items; item += kWarps * 32) {
    float sum = 0.0f;
    for (int k = 0; k < sh.slices; ++k) sum += __ldcg(all + k * items + item);
    put(item, sum);
  }
}

int few_nt(int64_t T) { return T <= 8 ? 1 : T <= 16 ? 2 : T <= 32 ? 4 : 8; }

FewShape few_shape(int fmt, const FewLinearArgs& a, int sm_count) {
  FewShape s;
  const int nt = few_nt(a.T), span = few_span(fmt);
  s.groups = (int)((a.kp + 4 * span - 1) / (4 * span));
  s.z = (int)((a.T + 8 * nt - 1) / (8 * nt));
  s.tiles = s.z * nt;
  s.wk = nt == 1 ? 8 : nt == 2 ? 4 : 1;
  const int64_t rb = (a.N + 16 * (kWarps / s.wk) - 1) / (16 * (kWarps / s.wk));
  // K slices across CTAs: three CTAs an SM, at least four groups for each warp
  int64_t want = (3 * (int64_t)sm_count + rb - 1) / rb;
  const int64_t most = s.groups / (4 * s.wk);
  s.slices = (int)(want < most ? want : most);
  if (s.slices < 1) s.slices = 1;
  return s;
}

size_t up256(size_t n) { return (n + 255) / 256 * 256; }

size_t frag_bytes(int fmt, const FewShape& s) {
  return up256((size_t)s.groups * s.tiles * (few_span(fmt) / 8) * 32 * sizeof(uint4));
}

template <typename T, int FMT, int NT>
cudaError_t few_launch(const FewLinearArgs& a, const FewShape& sh, cudaStream_t s) {
  uint4* frag = static_cast<uint4*>(a.ws);
  float* xs = reinterpret_cast<float*>(static_cast<char*>(a.ws) + frag_bytes(FMT, sh));
  float* part = xs + up256(sh.tiles * 8 * sizeof(float)) / sizeof(float);
  few_prepare_kernel<T, FMT><<<sh.tiles * 8, 512, 0, s>>>(a, frag, xs, sh.tiles);
  const int rows = 16 * (kWarps / sh.wk);
  const dim3 grid((unsigned)((a.N + rows - 1) / rows), sh.slices, sh.z);
  few_linear_kernel<T, FMT, NT><<<grid, kWarps * 32, 0, s>>>(a, sh, frag, xs, part);
  return cudaGetLastError();
}

template <typename T, int FMT>
cudaError_t few_nt_launch(const FewLinearArgs& a, int sm_count, cudaStream_t s) {
  const FewShape sh = few_shape(FMT, a, sm_count);
  switch (few_nt(a.T)) {
    case 1: return few_launch<T, FMT, 1>(a, sh, s);
    case 2: return few_launch<T, FMT, 2>(a, sh, s);
    case 4: return few_launch<T, FMT, 4>(a, sh, s);
    default: return few_launch<T, FMT, 8>(a, sh, s);
  }
}

template <typename T>
cudaError_t few_fmt_launch(int fmt, const FewLinearArgs& a, int sm_count, cudaStream_t s) {
  if (fmt == BF_NVFP4) return few_nt_launch<T, BF_NVFP4>(a, sm_count, s);
  if (fmt == BF_MXF4) return few_nt_launch<T, BF_MXF4>(a, sm_count, s);
  return few_nt_launch<T, BF_MXF8>(a, sm_count, s);
}

}  // namespace

size_t few_linear_ws_bytes(int fmt, const FewLinearArgs& a, int sm_count) {
  const FewShape s = few_shape(fmt, a, sm_count);
  const int nt = few_nt(a.T), wr = kWarps / s.wk;
  const int64_t rb = (a.N + 16 * wr - 1) / (16 * wr);
  const size_t part = s.slices > 1 ? (size_t)s.z * rb * s.slices * wr * nt * 128 * sizeof(float) : 0;
  return frag_bytes(fmt, s) + up256(s.tiles * 8 * sizeof(float)) + part;
}

size_t few_linear_counters(int fmt, const FewLinearArgs& a, int sm_count) {
  const FewShape s = few_shape(fmt, a, sm_count);
  const int wr = kWarps / s.wk;
  return s.slices > 1 ? (size_t)s.z * ((a.N + 16 * wr - 1) / (16 * wr)) : 0;
}

cudaError_t launch_few_linear(int fmt, int type, const FewLinearArgs& a, int sm_count,
                              cudaStream_t s) {
  if (type == B2G_BF16) return few_fmt_launch<__nv_bfloat16>(fmt, a, sm_count, s);
  return few_fmt_launch<__half>(fmt, a, sm_count, s);
}

}  // namespace b2g
