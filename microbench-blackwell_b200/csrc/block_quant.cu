// block_quant.cu -- microscaled casts of activations, weights and gradients, along the
// rows and the columns of a matrix in one pass, and their read-back.
//
// The reference fills its operands with byte patterns and its scales with constants
// (tcgen05_sparse_mma/tcgen05_sparse_mma.cu:246-256,320-325); a training step casts
// each operand twice, because the products of forward and backward run along different
// dimensions and a block's scale lies along the product's.
//
// Bound by bytes along the rows: 8192 x 8192 bf16 into NVFP4 27 us (6.3 TB/s of 6.5 measured
// by a copy), MXFP4 27, MXFP8 31, read back 34 to 38.  Both ways in one pass 50, 50 and 53 us
// (rows alone and columns alone 64, 64 and 69) and rounded by given bytes 83, 82 and 86: there
// the conversions bound it.  Rows off 16 bytes (8190 columns) 37, 37 and 39 us along the rows.
#include "b2g.h"
#include "op_common.cuh"
#include "op_kernels.h"

namespace b2g {
namespace {

constexpr int kThreads = 256;

// eight random bytes, zeros from the n-th on
__device__ __forceinline__ uint2 load_rand8(const uint8_t* p, int n, bool vec, const uint8_t* lo,
                                            const uint8_t* hi) {
  if (vec && n >= 8) return __ldg(reinterpret_cast<const uint2*>(p));
  if (n >= 8) {
    // off 8 bytes: two aligned words, both within [lo, hi), shifted together
    const uintptr_t at = reinterpret_cast<uintptr_t>(p), m = at & 7;
    const uint2* q = reinterpret_cast<const uint2*>(at - m);
    if (q >= static_cast<const void*>(lo) && q + 2 <= static_cast<const void*>(hi)) {
      const uint2 x = __ldg(q), y = __ldg(q + 1);
      const uint32_t a = m & 4 ? x.y : x.x, b = m & 4 ? y.x : x.y, c = m & 4 ? y.y : y.x;
      const uint32_t bits = (uint32_t)(m & 3) * 8;
      return make_uint2(__funnelshift_r(a, b, bits), __funnelshift_r(b, c, bits));
    }
  }
  uint32_t w[2] = {0u, 0u};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n) w[i >> 2] |= (uint32_t)__ldg(p + i) << (8 * (i & 3));
  return make_uint2(w[0], w[1]);
}

// A thread's 16 elements of a row: a block of NVFP4, half of an MX block (its neighbour has
// the other half).
template <typename T>
struct Raw16 {
  Raw8<T> h[2];
};

// 16 random bytes, zeros from the n-th on
struct Rand16 {
  uint2 h[2];
};

// Elements [0, n) of the 16 at p.  Rows off 16 bytes are read in aligned words where
// those lie within the matrix, [a.in, its last element].
template <typename T>
__device__ __forceinline__ Raw16<T> load16(const BlockQuantArgs& a, const T* p, int n) {
  Raw16<T> r;
  if (!a.in_vec && n == 16) {
    const T* lo = static_cast<const T*>(a.in);
    const T* hi = lo + ((a.rows - 1) * a.ld_in + a.cols);
    uint32_t u[8], v[8];
    if constexpr (sizeof(T) == 2) {
      if (load32_any(p, lo, hi, u)) {
        r.h[0].w[0] = make_uint4(u[0], u[1], u[2], u[3]);
        r.h[1].w[0] = make_uint4(u[4], u[5], u[6], u[7]);
        return r;
      }
    } else {
      if (load32_any(p, lo, hi, u) && load32_any(p + 8, lo, hi, v)) {
        r.h[0].w[0] = make_uint4(u[0], u[1], u[2], u[3]);
        r.h[0].w[1] = make_uint4(u[4], u[5], u[6], u[7]);
        r.h[1].w[0] = make_uint4(v[0], v[1], v[2], v[3]);
        r.h[1].w[1] = make_uint4(v[4], v[5], v[6], v[7]);
        return r;
      }
    }
  }
  r.h[0] = load8(p, n < 8 ? n : 8, a.in_vec);
  r.h[1] = load8(p + 8, n < 8 ? 0 : n - 8, a.in_vec);
  return r;
}

__device__ __forceinline__ Rand16 load_rand16(const BlockQuantArgs& a, const uint8_t* p, int n) {
  Rand16 r;
  const uint8_t* hi = a.rand + ((a.rows - 1) * a.ld_rand + a.cols);
  r.h[0] = load_rand8(p, n < 8 ? n : 8, a.rand_vec, a.rand, hi);
  r.h[1] = load_rand8(p + 8, n < 8 ? 0 : n - 8, a.rand_vec, a.rand, hi);
  return r;
}

template <int FMT, int QM, bool SR, bool FOLD>
__device__ __forceinline__ void store_row16(const float2 (&x)[2][4], const BlockScale& s, float fold,
                                            const Rand16& rnd, uint8_t* codes, uint8_t* sf) {
  uint32_t lo[2], hi[2];
  encode8<FMT, QM, SR, FOLD>(x[0], s, fold, rnd.h[0], lo);
  encode8<FMT, QM, SR, FOLD>(x[1], s, fold, rnd.h[1], hi);
  if constexpr (FMT == BF_MXF8)
    *reinterpret_cast<uint4*>(codes) = make_uint4(lo[0], lo[1], hi[0], hi[1]);
  else
    *reinterpret_cast<uint2*>(codes) = make_uint2(lo[0], hi[0]);
  if (bf_block(FMT) == 16 || (threadIdx.x & 1) == 0) *sf = (uint8_t)s.byte;
}

// Codes and scale of 16 elements of a row.  All lanes of a warp take part.
template <typename T, int FMT, int QM, bool SR, bool PRE>
__device__ __forceinline__ void encode_row16(const Raw16<T>& raw, float scale, const Rand16& rnd,
                                             uint8_t* codes, uint8_t* sf, bool write) {
  float2 x[2][4];
  float amax;
  if constexpr (PRE) {
    amax = 0.0f;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      unpack4x2(raw.h[k], x[k]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[k][i] = mul2(x[k][i], both(scale));
        amax = max_nan(amax, max_nan(fabsf(x[k][i].x), fabsf(x[k][i].y)));
      }
    }
  } else {
    const uint4 a = raw.h[0].w[0], b = raw.h[1].w[0];
    const uint32_t m = absmax_pair<T>(
        absmax_pair<T>(absmax_pair<T>(a.x, a.y), absmax_pair<T>(a.z, a.w)),
        absmax_pair<T>(absmax_pair<T>(b.x, b.y), absmax_pair<T>(b.z, b.w)));
    const float2 f = pair_f32<T>(m);
    amax = max_nan(f.x, f.y) * scale;
    unpack4x2(raw.h[0], x[0]);
    unpack4x2(raw.h[1], x[1]);
  }
  if constexpr (bf_block(FMT) == 32) amax = max_nan(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 1));
  const BlockScale s = block_scale<FMT, QM>(amax);
  if (write) store_row16<FMT, QM, SR, !PRE>(x, s, scale, rnd, codes, sf);
}

// Rows only: 16 elements per thread (a block of NVFP4, so that its scale needs no other lane;
// eight a thread took 45 us where this took 29).  blockDim.x threads along a row, blockDim.y
// rows.
template <typename T, int FMT, int QM, bool SR, bool PRE>
__global__ void __launch_bounds__(kThreads) quant_rows_kernel(const BlockQuantArgs a) {
  constexpr int bits = bf_bits(FMT), blk = bf_block(FMT);
  const int64_t c = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) * 16;
  const bool in_row = c < a.kp;
  const int n = c >= a.cols ? 0 : (int)(a.cols - c < 16 ? a.cols - c : 16);
  const int64_t step = (int64_t)gridDim.y * blockDim.y;
  // two rows at a time: the loads of both are in flight before the first is used
  for (int64_t r = (int64_t)blockIdx.y * blockDim.y + threadIdx.y; __any_sync(0xFFFFFFFFu, r < a.rows);
       r += 2 * step) {
    const bool ok0 = in_row && r < a.rows, ok1 = in_row && r + step < a.rows;
    const T* p = static_cast<const T*>(a.in) + r * a.ld_in + c;
    const Raw16<T> raw0 = load16(a, p, ok0 ? n : 0);
    const Raw16<T> raw1 = load16(a, p + step * a.ld_in, ok1 ? n : 0);
    Rand16 rnd0, rnd1;
    if constexpr (SR) {
      const uint8_t* q = a.rand + r * a.ld_rand + c;
      rnd0 = load_rand16(a, q, ok0 ? n : 0);
      rnd1 = load_rand16(a, q + step * a.ld_rand, ok1 ? n : 0);
    }
    encode_row16<T, FMT, QM, SR, PRE>(raw0, a.scale, rnd0, a.codes + (r * a.kp + c) * bits / 8,
                                      a.sf + (r * a.kp + c) / blk, ok0);
    encode_row16<T, FMT, QM, SR, PRE>(raw1, a.scale, rnd1,
                                      a.codes + ((r + step) * a.kp + c) * bits / 8,
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

template <typename T, int FMT, int QM, bool SR, bool PRE, bool ROWS>
__global__ void __launch_bounds__(kThreads) quant_both_kernel(const BlockQuantArgs a) {
  constexpr int bits = bf_bits(FMT), blk = bf_block(FMT);
  constexpr int kCols = 128 / (int)sizeof(T);    // columns of a tile
  constexpr int kVec = kCols / 16;               // sixteens of a row
  constexpr int kPer = 4 / (int)sizeof(T);       // columns of a 32-bit word
  constexpr int kRandWords = kCols / 4;          // words of a row of random bytes
  __shared__ __align__(16) uint32_t tile[kTileRows * 32];
  __shared__ __align__(16) uint32_t rnd_tile[SR ? kTileRows * kRandWords : 4];
  const int tid = threadIdx.x;
  const unsigned col_tiles = (unsigned)((a.kp + kCols - 1) / kCols);
  const int64_t r0 = (int64_t)(blockIdx.x / col_tiles) * kTileRows;
  const int64_t c0 = (int64_t)(blockIdx.x % col_tiles) * kCols;

  constexpr int kItems = kTileRows * kVec / kThreads;
  Raw16<T> raw[kItems];
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    const int item = i * kThreads + tid;
    const int64_t r = r0 + item / kVec, c = c0 + item % kVec * 16;
    const int n = r >= a.rows || c >= a.cols ? 0 : (int)(a.cols - c < 16 ? a.cols - c : 16);
    raw[i] = load16(a, static_cast<const T*>(a.in) + r * a.ld_in + c, n);
  }
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    const int item = i * kThreads + tid, v = item % kVec, lr = item / kVec;
    const int64_t r = r0 + lr, c = c0 + v * 16;
    const int g = (lr >> 4) & 7;
    Rand16 rnd;
    if constexpr (SR) {
      const int n = r >= a.rows || c >= a.cols ? 0 : (int)(a.cols - c < 16 ? a.cols - c : 16);
      rnd = load_rand16(a, a.rand + r * a.ld_rand + c, n);
      // pair p of 32-bit words of a row lies at p ^ g (fp32 tiles: half as many pairs)
      uint2* q = reinterpret_cast<uint2*>(rnd_tile) + lr * (kRandWords / 2);
      q[(2 * v) ^ (g & (kRandWords / 2 - 1))] = rnd.h[0];
      q[(2 * v + 1) ^ (g & (kRandWords / 2 - 1))] = rnd.h[1];
    }
    uint4* row = reinterpret_cast<uint4*>(tile) + lr * 8;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int k = 0; k < 4; ++k) row[(4 * v + k) ^ g] = raw[i].h[k >> 1].w[k & 1];
    } else {
      row[(2 * v) ^ g] = raw[i].h[0].w[0];
      row[(2 * v + 1) ^ g] = raw[i].h[1].w[0];
    }
    if constexpr (ROWS)
      encode_row16<T, FMT, QM, SR, PRE>(raw[i], a.scale, rnd, a.codes + (r * a.kp + c) * bits / 8,
                                        a.sf + (r * a.kp + c) / blk, r < a.rows && c < a.kp);
  }
  __syncthreads();

  const int g = tid & 7, w = tid >> 3;  // 16-row group, 32-bit word of the row
  uint32_t word[16];
#pragma unroll
  for (int i = 0; i < 16; ++i)
    word[i] = tile[(g * 16 + i) * 32 + ((((w >> 2) ^ g) << 2) | (w & 3))];
  const int64_t r = r0 + g * 16;
  // the word's columns side by side: largest magnitudes of both at a time
  float2 amax;
  float2 x[16];
  if constexpr (sizeof(T) == 2) {
    if constexpr (PRE) {
      amax = both(0.0f);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        x[i] = mul2(pair_f32<T>(word[i]), both(a.scale));
        amax = make_float2(max_nan(amax.x, fabsf(x[i].x)), max_nan(amax.y, fabsf(x[i].y)));
      }
    } else {
      uint32_t m = absmax_pair<T>(word[0], word[1]);
#pragma unroll
      for (int i = 2; i < 16; ++i) m = absmax_pair<T>(m, word[i]);
      amax = mul2(pair_f32<T>(m), both(a.scale));
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = pair_f32<T>(word[i]);
    }
  } else {
    amax = both(0.0f);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      x[i] = make_float2(__fmul_rn(__uint_as_float(word[i]), a.scale), 0.0f);
      amax.x = max_nan(amax.x, fabsf(x[i].x));
    }
  }
  if constexpr (blk == 32) {
    amax.x = max_nan(amax.x, __shfl_xor_sync(0xFFFFFFFFu, amax.x, 1));
    if constexpr (kPer == 2) amax.y = max_nan(amax.y, __shfl_xor_sync(0xFFFFFFFFu, amax.y, 1));
  }
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int64_t c = c0 + w * kPer + j;
    const BlockScale s = block_scale<FMT, QM>(j ? amax.y : amax.x);
    float2 y[2][4];
#pragma unroll
    for (int i = 0; i < 16; i += 2)
      y[i >> 3][(i & 7) >> 1] = j ? make_float2(x[i].y, x[i + 1].y) : make_float2(x[i].x, x[i + 1].x);
    uint2 rnd[2] = {make_uint2(0, 0), make_uint2(0, 0)};
    if constexpr (SR) {
      // byte w * kPer + j of each of the 16 rows, gathered into four words
      const int byte = w * kPer + j, pair = byte >> 3;
      const int at = ((pair ^ (g & (kRandWords / 2 - 1))) << 1) | ((byte >> 2) & 1);
      uint32_t b[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint32_t q[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) q[i] = rnd_tile[(g * 16 + 4 * k + i) * kRandWords + at];
        const uint32_t sel = (byte & 3) | (((byte & 3) + 4) << 4);
        b[k] = __byte_perm(__byte_perm(q[0], q[1], sel), __byte_perm(q[2], q[3], sel), 0x5410);
      }
      rnd[0] = make_uint2(b[0], b[1]);
      rnd[1] = make_uint2(b[2], b[3]);
    }
    uint32_t lo[2], hi[2];
    encode8<FMT, QM, SR, !PRE>(y[0], s, a.scale, rnd[0], lo);
    encode8<FMT, QM, SR, !PRE>(y[1], s, a.scale, rnd[1], hi);
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

// Read-back: eight codes per thread, of four rows at a time so that their loads are in
// flight together.  SHIFT: rows of `out` off 16 bytes (5000 x 4099 MXFP4 60 us with single
// elements, 20 us so); a thread then takes the eight
// elements of an aligned place in the row, whose codes are shifted out of two words and
// which may meet two blocks.
template <typename T, int FMT, bool SHIFT>
__global__ void __launch_bounds__(kThreads) dequant_kernel(const BlockDequantArgs a) {
  constexpr int blk = bf_block(FMT), kRows = 4, kWords = bf_bits(FMT) / 4;  // words of eight codes
  const int64_t v = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int64_t step = (int64_t)gridDim.y * blockDim.y, last = a.kp / 8 - 1;
  for (int64_t r0 = (int64_t)blockIdx.y * blockDim.y + threadIdx.y; r0 < a.rows; r0 += kRows * step) {
    uint32_t w[kRows][SHIFT ? 2 * kWords : kWords];
    uint32_t sb[kRows][SHIFT ? 2 : 1];
    int64_t c[kRows];
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      const int64_t r = r0 + k * step < a.rows ? r0 + k * step : r0;
      c[k] = v * 8;
      if constexpr (SHIFT) {
        // elements of the row before its first aligned place
        const uintptr_t at = reinterpret_cast<uintptr_t>(static_cast<T*>(a.out) + r * a.ld_out);
        const int lead = (int)((16 - (at & 15)) & 15) / (int)sizeof(T);
        c[k] = lead ? v * 8 + lead - 8 : v * 8;
      }
      // eights of codes: the one c lies in (or the row's ends where there is none), the next
      int64_t e = c[k] < 0 ? 0 : c[k] / 8;
      e = e < last ? e : last;
      const uint32_t* p = reinterpret_cast<const uint32_t*>(a.codes) + (r * (a.kp / 8) + e) * kWords;
      const uint8_t* sf = a.sf + r * (a.kp / blk);
      const int next = e < last ? 1 : 0;
      if constexpr (kWords == 2) {
        const uint2 x = __ldg(reinterpret_cast<const uint2*>(p));
        w[k][0] = x.x;
        w[k][1] = x.y;
        if constexpr (SHIFT) {
          const uint2 y = __ldg(reinterpret_cast<const uint2*>(p) + next);
          w[k][2] = y.x;
          w[k][3] = y.y;
        }
      } else {
        w[k][0] = __ldg(p);
        if constexpr (SHIFT) w[k][1] = __ldg(p + next);
      }
      sb[k][0] = __ldg(sf + e * 8 / blk);
      if constexpr (SHIFT) sb[k][1] = __ldg(sf + (e + next) * 8 / blk);
    }
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      const int64_t r = r0 + k * step;
      if (r >= a.rows || c[k] >= a.cols) continue;
      auto scale_of = [](uint32_t b) { return FMT == BF_NVFP4 ? e4m3_pair(b).x : e8m0_value(b); };
      const float s0 = scale_of(sb[k][0]);
      // codes from c[k] on: c[k] < 0 starts before the row, with places that are not stored
      int part = 0;  // elements of the first eight that come before
      uint32_t u[kWords];
#pragma unroll
      for (int i = 0; i < kWords; ++i) u[i] = w[k][i];
      float s1 = s0;
      if constexpr (SHIFT) {
        part = (int)(c[k] & 7);
        s1 = scale_of(sb[k][1]);
        if (c[k] < 0) {  // the first eight stand where the second would
#pragma unroll
          for (int i = 0; i < kWords; ++i) {
            w[k][i + kWords] = w[k][i];
            w[k][i] = 0u;
          }
          s1 = s0;
        }
        if constexpr (kWords == 1) {
          u[0] = __funnelshift_r(w[k][0], w[k][1], 4 * part);
        } else {
          const uint32_t x = part & 4 ? w[k][1] : w[k][0], y = part & 4 ? w[k][2] : w[k][1],
                         z = part & 4 ? w[k][3] : w[k][2];
          u[0] = __funnelshift_r(x, y, 8 * (part & 3));
          u[1] = __funnelshift_r(y, z, 8 * (part & 3));
        }
      }
      float2 f[4];
      if constexpr (FMT == BF_MXF8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = e4m3_pair(u[i >> 1] >> (16 * (i & 1)));
      } else {
        uint32_t h[4];
        e2m1x8_pairs(u[0], h);
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
      }
      // code * s is exact
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f[i] = mul2(f[i], make_float2(2 * i + part < 8 ? s0 : s1, 2 * i + 1 + part < 8 ? s0 : s1));
        if (a.scale != 1.0f) f[i] = mul2(f[i], both(a.scale));
      }
      const float o[8] = {f[0].x, f[0].y, f[1].x, f[1].y, f[2].x, f[2].y, f[3].x, f[3].y};
      T* dst = static_cast<T*>(a.out) + r * a.ld_out + c[k];
      const int64_t left = a.cols - c[k];
      if (SHIFT && c[k] < 0) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (c[k] + i >= 0 && i < left) dst[i] = from_f32<T>(o[i]);
      } else {
        store8(dst, o, left < 8 ? (int)left : 8, true);
      }
    }
  }
}

// blockDim.x threads of `per` elements along a row of `cols`, the rest along the rows: whole
// warps, and with more than 128 threads to a row as few idle ones as 32 allow
void row_shape(int64_t rows, int64_t cols, int per, dim3* grid, dim3* block) {
  const int64_t v = (cols + per - 1) / per;
  const int64_t gx = (v + kThreads - 1) / kThreads;
  int bx = 4;
  while (bx < v && bx < 128) bx *= 2;
  if (v > 128) bx = (int)((v + gx - 1) / gx + 31) / 32 * 32;
  const int by = kThreads / bx;
  int64_t gy = (rows + by - 1) / by;
  *block = dim3(bx, by);
  *grid = dim3((unsigned)gx, (unsigned)(gy < 65535 ? gy : 65535));
}

template <typename T, int FMT, int QM, bool SR, bool PRE>
cudaError_t quant_launch(const BlockQuantArgs& a, cudaStream_t s) {
  if (!a.codes_t) {
    dim3 grid, block;
    row_shape((a.rows + 1) / 2, a.kp, 16, &grid, &block);
    quant_rows_kernel<T, FMT, QM, SR, PRE><<<grid, block, 0, s>>>(a);
    return cudaGetLastError();
  }
  constexpr int kCols = 128 / (int)sizeof(T);
  const int64_t tiles = ((a.tp + kTileRows - 1) / kTileRows) * ((a.kp + kCols - 1) / kCols);
  if (tiles > 0x7FFFFFFF) return cudaErrorInvalidValue;
  if (a.codes)
    quant_both_kernel<T, FMT, QM, SR, PRE, true><<<(unsigned)tiles, kThreads, 0, s>>>(a);
  else
    quant_both_kernel<T, FMT, QM, SR, PRE, false><<<(unsigned)tiles, kThreads, 0, s>>>(a);
  return cudaGetLastError();
}

template <typename T, int FMT, int QM, bool PRE>
cudaError_t quant_sr(const BlockQuantArgs& a, cudaStream_t s) {
  return a.rand ? quant_launch<T, FMT, QM, true, PRE>(a, s)
                : quant_launch<T, FMT, QM, false, PRE>(a, s);
}

// PRE: each element is multiplied by `scale` first.  16-bit inputs with a power of two need
// not: it goes into the reciprocal of the block's scale, and NVFP4 quotients are then found
// without a division (8192 x 8192 bf16 into NVFP4 along the rows: scale 1 27 us, scale 3 48 us;
// both ways 50 and 100 us).
template <typename T>
cudaError_t quant_fmt(int fmt, bool pow2, const BlockQuantArgs& a, cudaStream_t s) {
  if constexpr (sizeof(T) == 2) {
    if (pow2) {
      if (fmt == BF_MXF8) return quant_sr<T, BF_MXF8, Q_EXACT, false>(a, s);
      if (fmt == BF_MXF4) return quant_sr<T, BF_MXF4, Q_EXACT, false>(a, s);
      return quant_sr<T, BF_NVFP4, Q_SNAP, false>(a, s);
    }
  }
  if (fmt == BF_MXF8) return quant_sr<T, BF_MXF8, Q_EXACT, true>(a, s);
  if (fmt == BF_MXF4) return quant_sr<T, BF_MXF4, Q_EXACT, true>(a, s);
  return quant_sr<T, BF_NVFP4, Q_DIVIDE, true>(a, s);
}

template <typename T, bool SHIFT>
cudaError_t dequant_fmt(int fmt, const BlockDequantArgs& a, cudaStream_t s) {
  dim3 grid, block;
  // SHIFT: a row may begin before an aligned place
  row_shape((a.rows + 3) / 4, a.cols + (SHIFT ? 7 : 0), 8, &grid, &block);
  if (fmt == BF_MXF8)
    dequant_kernel<T, BF_MXF8, SHIFT><<<grid, block, 0, s>>>(a);
  else if (fmt == BF_MXF4)
    dequant_kernel<T, BF_MXF4, SHIFT><<<grid, block, 0, s>>>(a);
  else
    dequant_kernel<T, BF_NVFP4, SHIFT><<<grid, block, 0, s>>>(a);
  return cudaGetLastError();
}

template <typename T>
cudaError_t dequant_rows(int fmt, const BlockDequantArgs& a, cudaStream_t s) {
  return a.out_vec ? dequant_fmt<T, false>(fmt, a, s) : dequant_fmt<T, true>(fmt, a, s);
}

}  // namespace

cudaError_t launch_block_quant(int fmt, int type, bool pow2, const BlockQuantArgs& a,
                               cudaStream_t s) {
  if (type == B2G_F32) return quant_fmt<float>(fmt, pow2, a, s);
  if (type == B2G_BF16) return quant_fmt<__nv_bfloat16>(fmt, pow2, a, s);
  return quant_fmt<__half>(fmt, pow2, a, s);
}

cudaError_t launch_block_dequant(int fmt, int type, const BlockDequantArgs& a, cudaStream_t s) {
  if (type == B2G_F32) return dequant_rows<float>(fmt, a, s);
  if (type == B2G_BF16) return dequant_rows<__nv_bfloat16>(fmt, a, s);
  return dequant_rows<__half>(fmt, a, s);
}

}  // namespace b2g
