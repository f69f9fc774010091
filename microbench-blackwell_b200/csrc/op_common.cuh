// op_common.cuh -- device helpers of the operators around the linear layer: eight
// elements at a time from 16- or 32-bit rows, and microscaled 4- and 8-bit codes.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <mutex>

namespace b2g {

// Lets a kernel use `bytes` of dynamic shared memory on the current device.  The attribute
// is set once for each kernel, device and size above the last (`seen`: one word per device,
// the kernel's own), by one host thread at a time: a smaller size may not come behind a larger.
template <typename K>
inline cudaError_t allow_smem(K kernel, int bytes, std::atomic<int> (&seen)[16]) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 16 && seen[dev].load(std::memory_order_acquire) >= bytes) return cudaSuccess;
  static std::mutex one;
  std::lock_guard<std::mutex> lock(one);
  if (dev < 16 && seen[dev].load(std::memory_order_relaxed) >= bytes) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && dev < 16) seen[dev].store(bytes, std::memory_order_release);
  return e;
}

// Eight consecutive elements of a row as they lie in memory: one 16-byte word for
// 16-bit types, two for fp32.
template <typename T>
struct Raw8 {
  uint4 w[sizeof(T) == 4 ? 2 : 1];
};

template <typename T>
__device__ __forceinline__ float to_f32(T x);
template <>
__device__ __forceinline__ float to_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) {
  return __bfloat162float(x);
}
template <>
__device__ __forceinline__ float to_f32<__half>(__half x) { return __half2float(x); }

template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }

// Elements [0, n) of the eight at p, zeros after them; `vec`: p is 16-byte aligned.
template <typename T>
__device__ __forceinline__ Raw8<T> load8(const T* p, int n, bool vec) {
  Raw8<T> r;
  constexpr int W = sizeof(T) == 4 ? 2 : 1;
  if (vec && n >= 8) {
#pragma unroll
    for (int i = 0; i < W; ++i) r.w[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
    return r;
  }
  uint32_t u[4 * W];
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      u[i] = i < n ? __ldg(reinterpret_cast<const uint32_t*>(p) + i) : 0u;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint16_t* q = reinterpret_cast<const uint16_t*>(p);
      const uint32_t lo = 2 * i < n ? __ldg(q + 2 * i) : 0u;
      const uint32_t hi = 2 * i + 1 < n ? __ldg(q + 2 * i + 1) : 0u;
      u[i] = lo | (hi << 16);
    }
  }
#pragma unroll
  for (int i = 0; i < W; ++i)
    r.w[i] = make_uint4(u[4 * i], u[4 * i + 1], u[4 * i + 2], u[4 * i + 3]);
  return r;
}

// The 32 bytes at p, which has the alignment of its elements only: three aligned 16-byte
// words, all within [lo, hi), shifted together.  False where they are not within.
__device__ __forceinline__ bool load32_any(const void* p, const void* lo, const void* hi,
                                           uint32_t (&u)[8]) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(p), m = at & 15;
  const uint4* a = reinterpret_cast<const uint4*>(at - m);
  if (a < lo || a + 3 > hi) return false;
  const uint4 x = __ldg(a), y = __ldg(a + 1), z = __ldg(a + 2);
  uint32_t w[12] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w, z.x, z.y, z.z, z.w};
  if (m & 8)
#pragma unroll
    for (int i = 0; i < 10; ++i) w[i] = w[i + 2];
  if (m & 4)
#pragma unroll
    for (int i = 0; i < 9; ++i) w[i] = w[i + 1];
  const uint32_t bits = (uint32_t)(m & 3) * 8;
#pragma unroll
  for (int i = 0; i < 8; ++i) u[i] = __funnelshift_r(w[i], w[i + 1], bits);
  return true;
}

template <typename T>
__device__ __forceinline__ float2 pair_f32(uint32_t w);
template <>
__device__ __forceinline__ float2 pair_f32<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
template <>
__device__ __forceinline__ float2 pair_f32<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

template <typename T>
__device__ __forceinline__ void unpack8(const Raw8<T>& r, float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    const uint32_t u[8] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w,
                           r.w[1].x, r.w[1].y, r.w[1].z, r.w[1].w};
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(u[i]);
  } else {
    const uint32_t u[4] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = pair_f32<T>(u[i]);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
}

// Two fp32 in one register pair: one instruction for both.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n\t.reg .b64 a, b, c, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 a, b, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "mul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 a, b, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 both(float a) { return make_float2(a, a); }

// the same as four pairs
template <typename T>
__device__ __forceinline__ void unpack4x2(const Raw8<T>& r, float2 (&v)[4]) {
  if constexpr (sizeof(T) == 4) {
    v[0] = make_float2(__uint_as_float(r.w[0].x), __uint_as_float(r.w[0].y));
    v[1] = make_float2(__uint_as_float(r.w[0].z), __uint_as_float(r.w[0].w));
    v[2] = make_float2(__uint_as_float(r.w[1].x), __uint_as_float(r.w[1].y));
    v[3] = make_float2(__uint_as_float(r.w[1].z), __uint_as_float(r.w[1].w));
  } else {
    v[0] = pair_f32<T>(r.w[0].x);
    v[1] = pair_f32<T>(r.w[0].y);
    v[2] = pair_f32<T>(r.w[0].z);
    v[3] = pair_f32<T>(r.w[0].w);
  }
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&b);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 b = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&b);
}

// Stores the first n of eight values at p; `vec`: p is 16-byte aligned.
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8], int n, bool vec) {
  if (vec && n >= 8) {
    if constexpr (sizeof(T) == 4) {
      reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      *reinterpret_cast<uint4*>(p) = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]),
                                                pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n) p[i] = from_f32<T>(v[i]);
}

// Bytes m .. m + 15 of two 16-byte words, m even and below 16.
__device__ __forceinline__ uint4 shift16(const uint4& x, const uint4& y, uint32_t m) {
  uint32_t w[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
  if (m & 8)
#pragma unroll
    for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
  if (m & 4)
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
  const uint32_t bits = (m & 2) * 8;
  return make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits),
                    __funnelshift_r(w[2], w[3], bits), __funnelshift_r(w[3], w[4], bits));
}

// load8 for rows of any alignment (ANY; else every p is 16-byte aligned): aligned words
// shifted together where they lie within the operand, else element by element.  `inside`:
// the row has others of 16 elements or more before and behind it, so they do.
template <typename T, bool ANY>
__device__ __forceinline__ Raw8<T> load8_any(const T* p, int n, bool inside) {
  if constexpr (ANY) {
    const uint32_t m = (uint32_t)reinterpret_cast<uintptr_t>(p) & 15u;
    if (m && n >= 8) {
      if (inside) {
        Raw8<T> r;
        const uint4* q = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(p) - m);
        uint4 w[sizeof(T) / 2 + 1];
#pragma unroll
        for (int i = 0; i <= (int)sizeof(T) / 2; ++i) w[i] = __ldg(q + i);
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.w[i] = shift16(w[i], w[i + 1], m);
        return r;
      }
      return load8(p, n, false);
    }
    return load8(p, n, m == 0);
  } else {
    return load8(p, n, true);
  }
}

// store8 of a whole warp for rows of any alignment (ANY): p is lane 0's place plus eight
// elements a lane, `count` the warp's elements in the row.  The values go through `buf`
// (the warp's own, (8 * sizeof(T)) * 32 + 16 bytes) and out as aligned 16-byte words, with
// single elements at the ends.
template <typename T, bool ANY>
__device__ __forceinline__ void store8_any(T* p, const float (&v)[8], int n, int count, uint4* buf) {
  if constexpr (!ANY) {
    store8(p, v, n, true);
  } else {
    constexpr int W = (int)sizeof(T) / 2;  // 16-byte words of eight elements
    const int lane = threadIdx.x & 31;
    T* first = p - lane * 8;
    const uint32_t m = (uint32_t)reinterpret_cast<uintptr_t>(first) & 15u;
    if (m == 0) {
      store8(p, v, n, true);
      return;
    }
    if constexpr (sizeof(T) == 4) {
      buf[lane * 2] = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]),
                                 __float_as_uint(v[3]));
      buf[lane * 2 + 1] = make_uint4(__float_as_uint(v[4]), __float_as_uint(v[5]),
                                     __float_as_uint(v[6]), __float_as_uint(v[7]));
    } else {
      buf[lane] = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]),
                             pack2<T>(v[6], v[7]));
    }
    __syncwarp();
    const int bytes = count * (int)sizeof(T);
    int head = 16 - (int)m;
    head = head < bytes ? head : bytes;
    const int full = (bytes - head) / 16;
    char* dst = reinterpret_cast<char*>(first);
#pragma unroll
    for (int k = 0; k < W; ++k) {
      const int i = k * 32 + lane;
      if (i < full)
        *reinterpret_cast<uint4*>(dst + head + 16 * i) = shift16(buf[i], buf[i + 1], 16 - m);
    }
    // elements before the first word and after the last
    const int tail = head + 16 * full, heads = head / (int)sizeof(T);
    const int rest = (bytes - tail) / (int)sizeof(T);
    const T* e = reinterpret_cast<const T*>(buf);
    if (lane < heads) first[lane] = e[lane];
    if (lane >= 16 && lane - 16 < rest)
      first[tail / (int)sizeof(T) + lane - 16] = e[tail / (int)sizeof(T) + lane - 16];
    __syncwarp();
  }
}

template <typename T>
__device__ __forceinline__ void store4x2(T* p, const float2 (&v)[4], bool vec) {
  const float f[8] = {v[0].x, v[0].y, v[1].x, v[1].y, v[2].x, v[2].y, v[3].x, v[3].y};
  store8(p, f, 8, vec);
}

// ---------------------------------------------------------------- microscaled codes
// Element formats with one scale per block (the numbers of BlockFmt are internal):
//   NVFP4  e2m1, ue4m3 scale per 16:  s = e4m3(amax / 6)
//   MXFP4  e2m1, E8M0 scale per 32:   s = 2^(floor(log2 amax) - 2)
//   MXFP8  e4m3, E8M0 scale per 32:   s = 2^(floor(log2 amax) - 8)
// codes = element(x / s), to nearest even and saturating.  A block that holds an
// infinity or a NaN gets a NaN scale and so reads back as NaN: an overflow upstream
// stays visible.
enum BlockFmt : int { BF_NVFP4 = 0, BF_MXF4 = 1, BF_MXF8 = 2 };
__host__ __device__ constexpr int bf_block(int f) { return f == BF_NVFP4 ? 16 : 32; }
__host__ __device__ constexpr int bf_bits(int f) { return f == BF_MXF8 ? 8 : 4; }

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// eight e2m1 codes, element i in bits [4i, 4i + 4)
__device__ __forceinline__ uint32_t e2m1x8(const float2 (&x)[4]) {
  uint32_t r;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(r)
      : "f"(x[0].x), "f"(x[0].y), "f"(x[1].x), "f"(x[1].y), "f"(x[2].x), "f"(x[2].y),
        "f"(x[3].x), "f"(x[3].y));
  return r;
}

// values of eight e2m1 codes as fp16 pairs
__device__ __forceinline__ void e2m1x8_pairs(uint32_t w, uint32_t (&h)[4]) {
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(w));
}

// value of the two e4m3 codes in the low bytes of w
__device__ __forceinline__ float2 e4m3_pair(uint32_t w) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)w));
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// 2^(byte - 127), the value of an E8M0 byte (255: NaN)
__device__ __forceinline__ float e8m0_value(uint32_t byte) {
  return __uint_as_float(byte == 0u ? 0x00400000u : byte == 255u ? 0x7FFFFFFFu : byte << 23);
}

// Largest magnitudes of the halves of two words of 16-bit elements, NaN if one is.
template <typename T>
__device__ __forceinline__ uint32_t absmax_pair(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (__is_same(T, __half))
    asm("{\n\t.reg .b32 x, y;\n\tabs.f16x2 x, %1;\n\tabs.f16x2 y, %2;\n\t"
        "max.NaN.f16x2 %0, x, y;\n\t}"
        : "=r"(r)
        : "r"(a), "r"(b));
  else
    asm("{\n\t.reg .b32 x, y;\n\tabs.bf16x2 x, %1;\n\tabs.bf16x2 y, %2;\n\t"
        "max.NaN.bf16x2 %0, x, y;\n\t}"
        : "=r"(r)
        : "r"(a), "r"(b));
  return r;
}

// How x / s is formed.  MX scales are powers of two: x * (1 / s) is exact.  NVFP4:
//   Q_DIVIDE  x / s rounded to fp32, right for any x;
//   Q_SNAP    for x with at most 11 significant bits (16-bit inputs times a power of
//             two).  The boundaries of e2m1 have at most 3 bits and s has 4, so x / s
//             either lies on a boundary or at least 2^-13 beside it.  fma(x, 1/s, 48)
//             - 48 rounds the quotient to a multiple of 2^-18: a quotient on a boundary
//             comes out on it and no other crosses one, for two instructions (two
//             elements each) where the division takes about ten.  In the same way amax / 6
//             comes from a product rounded to 16 bits: the boundaries of e4m3 have 5.
enum QuotientMode : int { Q_EXACT = 0, Q_DIVIDE = 1, Q_SNAP = 2 };

// The scale of a block from its largest magnitude: the stored byte, its value and the
// reciprocal of the value (0 where all codes shall be 0), rounded up.
struct BlockScale {
  uint32_t byte;
  float value, inv;
};

template <int FMT, int QM>
__device__ __forceinline__ BlockScale block_scale(float amax) {
  BlockScale s;
  const bool finite = amax < __uint_as_float(0x7F800000u);  // false for NaN too
  if constexpr (FMT == BF_NVFP4) {
    const float sixth =
        QM == Q_SNAP ? __uint_as_float((__float_as_uint(amax * (1.0f / 6.0f)) + 0x80u) & ~0xFFu)
                     : amax / 6.0f;
    s.byte = e4m3x2(sixth, 0.0f) & 0xFFu;
    s.value = e4m3_pair(s.byte).x;
    s.inv = s.byte ? __frcp_ru(s.value) : 0.0f;
    if (!finite) s = {0x7Fu, 0.0f, 0.0f};
  } else {
    constexpr int emax = FMT == BF_MXF8 ? 8 : 2;
    // exponent field of amax (0 for 0 and subnormals: their scale is clamped anyway)
    const int e = (int)(__float_as_uint(amax) >> 23) - emax;
    s.byte = e > 0 ? (uint32_t)e : 0u;
    s.value = e8m0_value(s.byte);
    s.inv = __uint_as_float((254u - s.byte) << 23);
    if (!finite) s = {0xFFu, 0.0f, 0.0f};
  }
  return s;
}

// Stochastic rounding with a given byte r: |x / s| in steps of the element format goes up
// when its fraction and (r + 1/2) / 256 together reach the next step.  |x / s| is scaled so
// that the format's lowest binade becomes the lowest normal one of fp32: the bits of the
// result then are the magnitude code with the fraction below it, subnormal codes included,
// and (r + 1/2) / 256 of a step is added to them as an integer.  x: the quotient already
// (Q_DIVIDE: the element).  Q_SNAP: a fraction that with r reaches the step exactly must not
// come out below; 1 / s is rounded up, and the product then does not fall below a threshold
// that x / s reaches.  No other quotient lies that near: the thresholds have 12 bits.
// The shift rounds towards zero: what it drops below a subnormal code's 22 (20) bits of
// fraction must not lift an fp32 quotient to a threshold that it lies under.
template <int FMT, int QM>
__device__ __forceinline__ float round_stochastic(float x, const BlockScale& s,
                                                  uint32_t word, int byte) {
  constexpr float down = FMT == BF_MXF8 ? 0x1p-120f : 0x1p-126f;
  constexpr float up = FMT == BF_MXF8 ? 0x1p120f : 0x1p126f;
  constexpr int frac = FMT == BF_MXF8 ? 20 : 22;  // bits below the code
  uint32_t bits;
  if constexpr (QM == Q_DIVIDE)
    bits = __float_as_uint(s.inv != 0.0f ? __fmul_rz(fabsf(x / s.value), down) : 0.0f);
  else
    bits = __float_as_uint(__fmul_rz(fabsf(x), down));  // x is the quotient already
  // 256 r + 128: the byte above a half, one permutation
  const uint32_t r = __byte_perm(word, 0x80u, 0x5504u | (uint32_t)(byte << 4));
  bits = (r * (1u << (frac - 16)) + bits) & (0xFFFFFFFFu << frac);
  return __uint_as_float(bits) * __uint_as_float((__float_as_uint(x) & 0x80000000u) | __float_as_uint(up));
}

// Codes of eight elements of one block (times `fold`, a power of two, where FOLD): 32 bits
// (e2m1) in w[0] or 64 (e4m3) in w[0..1].  rnd: eight random bytes, used when SR.
template <int FMT, int QM, bool SR, bool FOLD>
__device__ __forceinline__ void encode8(const float2 (&in)[4], const BlockScale& s, float fold,
                                        uint2 rnd, uint32_t (&w)[2]) {
  float2 q[4];
  float mult = FOLD ? s.inv * fold : s.inv;
  float2 x[4] = {in[0], in[1], in[2], in[3]};
  // MX: fold / s leaves fp32's range in a block of zeros, or one so small that its scale is the
  // least or next to it.  fold then goes into the elements first: 0 * infinity would be NaN.
  // (Both ways, 8192 x 8192 bf16: 50 and 53 us; without this test 47 and 52.)
  if (FOLD && QM == Q_EXACT && mult > 0x1.fffffep127f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = mul2(x[i], both(fold));
    mult = s.inv;
  }
  if constexpr (SR) {
    // 1 / s and the format's shift are two products: as one it may leave fp32's range (MX), or
    // be subnormal and lose bits (NVFP4)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (QM != Q_DIVIDE) x[i] = mul2(x[i], both(mult));
      const uint32_t word = i < 2 ? rnd.x : rnd.y;
      q[i].x = round_stochastic<FMT, QM>(x[i].x, s, word, 2 * (i & 1));
      q[i].y = round_stochastic<FMT, QM>(x[i].y, s, word, 2 * (i & 1) + 1);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (QM == Q_DIVIDE) {
        q[i].x = s.inv != 0.0f ? x[i].x / s.value : 0.0f;
        q[i].y = s.inv != 0.0f ? x[i].y / s.value : 0.0f;
      } else if constexpr (QM == Q_SNAP) {
        q[i] = add2(fma2(x[i], both(mult), both(48.0f)), both(-48.0f));
      } else {
        q[i] = mul2(x[i], both(mult));
      }
    }
  }
  if constexpr (FMT == BF_MXF8) {
    w[0] = e4m3x2(q[0].x, q[0].y) | (e4m3x2(q[1].x, q[1].y) << 16);
    w[1] = e4m3x2(q[2].x, q[2].y) | (e4m3x2(q[3].x, q[3].y) << 16);
  } else {
    w[0] = e2m1x8(q);
    w[1] = 0u;
  }
}

// ---------------------------------------------------------------- sums
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}

// Sums of K values over the CTA's row of threads (blockDim.x of them; one warp per row
// where blockDim.x is 32).  `red`: K * 32 floats, not in use by an earlier call.
template <int K>
__device__ __forceinline__ void row_sum(float (&v)[K], float* red) {
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = warp_sum(v[k]);
  if (blockDim.x == 32) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  if (lane == 0)
#pragma unroll
    for (int k = 0; k < K; ++k) red[k * 32 + warp] = v[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = warp_sum(lane < warps ? red[k * 32 + lane] : 0.0f);
}

// The same over a CTA of any number of warps, always with its barrier.
template <int K>
__device__ __forceinline__ void row_sum_cta(float (&v)[K], float* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = warp_sum(v[k]);
  if (lane == 0)
#pragma unroll
    for (int k = 0; k < K; ++k) red[k * 32 + warp] = v[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = warp_sum(lane < warps ? red[k * 32 + lane] : 0.0f);
}

}  // namespace b2g
