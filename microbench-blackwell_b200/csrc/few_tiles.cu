// few_tiles.cu -- y = alpha * x . W^T of some tens of tokens with microscaled weights: the
// tensor-core form of b2g_linear (few_linear.cu has the form for a handful).
//
// The weights are the 128-row operand A of tcgen05.mma kind::f16, taken from tensor memory:
// sixteen warps decode codes to fp16 (exact, as in few_linear.cu) and write them there, a row
// a thread, so that decoded weights never pass through shared memory.  x, laid out as fp16
// by a first kernel, is operand B, up to 128 tokens of it; sums stay in tensor memory until
// the end.  A decoded weight then serves all tokens for one instruction's issue.
//
// Measured, 16384 x 8192, 16 tokens: NVFP4 21.4 us, MXFP4 23.3, MXFP8 34.0; 64 tokens 25.5,
// 28.3, 37.1; 128 tokens 43.0, 46.0, 46.9 (x is read from L2 by every CTA, 64 KB for each
// 16 KB of codes); 2048 x 2048, 16 tokens 8 to 9 us.  Of MXFP4's 16 tokens about 6 us pass
// before the first step is decoded (x's layout, launch, first copies) and 2 after the last;
// between, a step of 256 elements x 128 rows takes 0.43 us, 4.9 TB/s of weights, MXFP8's, of half
// as many elements, 6 TB/s.  Tensor pipe (11 % busy), issue slots (53 %) and memory (70 % in the
// loop) are none of them full: it is the chain copy, decoding, products, and neither more
// buffers nor more ring slots shortened it.
#include <cuda.h>

#include "b2g.h"
#include "b2g_desc.h"
#include "b2g_gemm.h"
#include "b2g_ptx.cuh"
#include "op_common.cuh"
#include "op_kernels.h"

namespace b2g {
namespace {

constexpr int kRows = 128;            // weight rows of a CTA
// Two groups of eight decoding warps take every other step each; four of them cover the rows,
// twice, for the halves of a step.  (Eight warps in all: 16384 x 8192 NVFP4 44 us, 16 tokens.)
constexpr int kGroups = 2, kHalves = 2;
constexpr int kQuads = kGroups * kHalves;  // sets of four warps
constexpr int kDecodeWarps = 4 * kQuads;
constexpr int kThreads = (kDecodeWarps + 2) * 32;
constexpr int kCodeBytes = 128;       // of a row in a step
constexpr int kMaxStages = 6;          // MXFP8 16384 x 8192 34.0 us with six, 38.1 with four
constexpr int kMaxBuffers = 4;        // of decoded steps in tensor memory
constexpr int kScaleBytes = 2048;     // of a ring slot: 16, 8 or 4 bytes a row

__host__ __device__ constexpr int step_k(int fmt) { return kCodeBytes * 8 / bf_bits(fmt); }

struct TileShape {
  int tokens;    // of a CTA, a multiple of 16 up to 128
  int steps;     // of K in all
  int slices;    // of K, one a CTA
  int row_tiles, z;
  int stages;
  int words;     // a row's scales of a step are one aligned word, copied into the ring
  int smem;
};

// x as fp16 [T][steps * step_k], zero past K, times a power of two for each token (bf16)
// that brings its largest value to 2^14 .. 2^15; xs[token] undoes it.
template <typename T>
__global__ void __launch_bounds__(512) tiles_prepare_kernel(const FewLinearArgs a, int64_t kq,
                                                            __half* x16, float* xs) {
  __shared__ float red[16];
  const int64_t token = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + token * a.ld_x;
  // the product kernel may start; it waits for this one to end before it reads x
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  float scale = 1.0f;
  auto eight = [&](int64_t v) {
    const int64_t left = a.K - v * 8;
    return load8(x + v * 8, left < 0 ? 0 : left < 8 ? (int)left : 8, a.x_vec);
  };
  if constexpr (__is_same(T, __nv_bfloat16)) {
    float amax = 0.0f;
    for (int64_t v = threadIdx.x; v * 8 < a.K; v += 512) {
      float f[8];
      unpack8(eight(v), f);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float m = fabsf(f[i]);
        amax = fmaxf(amax, m < __uint_as_float(0x7F800000u) ? m : 0.0f);  // of the finite ones
      }
    }
    const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(amax));
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = __uint_as_float(top);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 16; ++i) amax = fmaxf(amax, red[i]);
    int e = 127 + 14 - ((int)(__float_as_uint(amax) >> 23) - 127);
    e = e > 253 ? 253 : e;
    scale = amax > 0.0f ? __uint_as_float((uint32_t)e << 23) : 1.0f;
  }
  if (threadIdx.x == 0) xs[token] = 1.0f / scale;
  for (int64_t v = threadIdx.x; v * 8 < kq; v += 512) {
    const Raw8<T> r = eight(v);
    uint4 w = r.w[0];
    if constexpr (__is_same(T, __nv_bfloat16)) {
      float f[8];
      unpack8(r, f);
      w = make_uint4(pack2<__half>(f[0] * scale, f[1] * scale), pack2<__half>(f[2] * scale, f[3] * scale),
                     pack2<__half>(f[4] * scale, f[5] * scale), pack2<__half>(f[6] * scale, f[7] * scale));
    }
    *reinterpret_cast<uint4*>(x16 + token * kq + v * 8) = w;
  }
}

// 32 lanes x 16 columns of 32 bits: lane i of the warp writes TMEM lane (its quarter * 32 + i)
__device__ __forceinline__ void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

__device__ __forceinline__ void tmem_st_wait() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ uint32_t mul_h2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// N scale bytes of a row of `count`; zeros past its end.
template <int N>
__device__ __forceinline__ uint32_t load_scales(const uint8_t* row, int first, int count) {
  uint32_t s = 0u;
#pragma unroll
  for (int i = 0; i < N; ++i) s |= (first + i < count ? (uint32_t)__ldg(row + first + i) : 0u) << (8 * i);
  return s;
}

// MX: the scales of a row within a CTA's K slice are taken relative to one of them, the
// largest of a few samples: 2^(s - ref) times an element is exact and finite in fp16 for s
// - ref from -14 to 13 (e2m1) or 7 (e4m3).  Blocks outside (and not all zeros) are left out
// of the tensor product.
template <int FMT>
constexpr uint32_t kAbove = FMT == BF_MXF8 ? 7 : 13;

template <int FMT>
__device__ __forceinline__ bool any_code(const uint32_t (&c)[bf_bits(FMT)]) {
  uint32_t any = 0u;
#pragma unroll
  for (int i = 0; i < bf_bits(FMT); ++i) any |= c[i];
  return (any & (FMT == BF_MXF8 ? 0x7F7F7F7Fu : 0x77777777u)) != 0u;
}

// The products of a row's blocks that were left out, in fp32 and from global memory:
// far[j * kDecodeWarps * 32] of the j-th of `count` tokens, whose x starts at x16.
template <int FMT>
__device__ __noinline__ void far_blocks(const FewLinearArgs& a, const __half* x16, int64_t kq, int row,
                                        int k_begin, int k_end, uint32_t ref, int count, float* far) {
  for (int j = 0; j < count; ++j) far[j * kDecodeWarps * 32] = 0.0f;
  const int64_t kp = a.kp;
  for (int k0 = k_begin; k0 < k_end; k0 += 32) {
    const uint32_t s = __ldg(a.sf + (row * kp + k0) / 32);
    if (s == 255u || s - ref + 14u <= 14u + kAbove<FMT>) continue;
    const uint32_t* codes = reinterpret_cast<const uint32_t*>(a.w + (row * kp + k0) * bf_bits(FMT) / 8);
    uint32_t c[bf_bits(FMT)];
    for (int i = 0; i < bf_bits(FMT); ++i) c[i] = __ldg(codes + i);
    if (!any_code<FMT>(c)) continue;
    for (int j = 0; j < count; ++j) {
      const __half* x = x16 + j * kq + k0;
      float dot = 0.0f;
      for (int i = 0; i < 32; ++i) {
        const uint32_t word = __ldg(codes + i * bf_bits(FMT) / 32) >> (i * bf_bits(FMT) % 32);
        float v;
        if constexpr (FMT == BF_MXF8) {
          v = e4m3_pair(word & 0xFFu).x;
        } else {
          uint32_t q[4];
          e2m1x8_pairs(word & 15u, q);
          v = __half2float(__ushort_as_half((unsigned short)(q[0] & 0xFFFFu)));
        }
        dot = fmaf(v, __half2float(x[i]), dot);
      }
      far[j * kDecodeWarps * 32] = fmaf(e8m0_value(s), dot, far[j * kDecodeWarps * 32]);
    }
  }
}

template <typename T, int FMT>
__global__ void __launch_bounds__(kThreads, 1)
few_tiles_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                 const FewLinearArgs a, const TileShape sh, const __half* x16, const float* xs,
                 float* part) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  // ring slots (codes, x, scales) start on 1024 bytes
  const uint32_t ring = (smem_u32(smem_raw) + 1023u) & ~1023u;
  __shared__ __align__(8) uint64_t bars[2 * kMaxStages + 2 * kMaxBuffers + 1];
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int aborted;
  __shared__ bool last;
  __shared__ uint32_t row_ref[kRows];
  __shared__ float token_scale[128];
  __shared__ uint8_t has_far[kQuads][kRows];
  constexpr int sk = step_k(FMT);
  constexpr uint32_t a_cols = sk / 2;               // TMEM columns of a decoded step
  // Of them, and of ring slots, an even number: each is then always filled or read by the same
  // group, which has waited for every one of its barriers' phases and cannot take one for the
  // next but one.
  constexpr int buffers = FMT == BF_MXF8 ? 4 : 2;
  static_assert(buffers % kGroups == 0 && buffers <= kMaxBuffers && 128 + buffers * a_cols <= 512,
                "buffers");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tile = (int)blockIdx.x / sh.slices, slice = (int)blockIdx.x % sh.slices;
  const int s0 = (int)((unsigned)sh.steps * (unsigned)slice / (unsigned)sh.slices);
  const int s1 = (int)((unsigned)sh.steps * (slice + 1u) / (unsigned)sh.slices);
  const int row0 = tile * kRows, token0 = (int)blockIdx.y * 128;
  const int cols = (int)(a.T - token0 < 128 ? a.T - token0 : 128);
  const uint32_t x_bytes = (uint32_t)sh.tokens * sk * 2, slot_bytes = kRows * kCodeBytes + x_bytes + kScaleBytes;
  auto full = [&](int s) { return smem_u32(&bars[s]); };
  auto empty = [&](int s) { return smem_u32(&bars[kMaxStages + s]); };
  auto a_full = [&](int b) { return smem_u32(&bars[2 * kMaxStages + b]); };
  auto a_empty = [&](int b) { return smem_u32(&bars[2 * kMaxStages + kMaxBuffers + b]); };
  const uint32_t done = smem_u32(&bars[2 * kMaxStages + 2 * kMaxBuffers]);

  if (threadIdx.x < kRows) row_ref[threadIdx.x] = 0u;
  if (threadIdx.x == 0) {
    aborted = 0;
    for (int s = 0; s < kMaxStages; ++s) {
      mbar_init(full(s), 1 + 32);  // the copies' byte count, and a lane's scales each
      mbar_init(empty(s), 1);
    }
    for (int b = 0; b < buffers; ++b) {
      mbar_init(a_full(b), 4 * kHalves);
      mbar_init(a_empty(b), 1);
    }
    mbar_init(done, 1);
    fence_mbar_init();
  }
  if (warp == kDecodeWarps) {
    tmem_alloc<1>(smem_u32(&tmem_slot), 512);
    tmem_relinquish<1>();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot, tmem_a = tmem + 128;  // sums, then decoded steps

  if (warp == kDecodeWarps + 1) {
    // ---- copies: codes and scales at once, x when the first kernel has laid it out
    const bool one = elect_one();
    const uint64_t once = l2_policy_evict_normal(), keep = l2_policy_evict_last();
    constexpr int n = sk / bf_block(FMT);  // scale bytes of a row in a step
    const int scales = (int)a.kp / bf_block(FMT);
    auto ask_codes = [&](int step, int stage) {
      if (one) {
        mbar_arrive_expect_tx(full(stage), kRows * kCodeBytes + x_bytes);
        tma_load_2d(ring + stage * slot_bytes, &map_w, step * kCodeBytes, row0, full(stage), once);
      }
      if (sh.words) {
        const uint32_t to = ring + stage * slot_bytes + kRows * kCodeBytes + x_bytes;
        const bool on = step * n < scales;
#pragma unroll
        for (int k = 0; k < kRows / 32; ++k) {
          const int r = k * 32 + lane, row = row0 + r < (int)a.N ? row0 + r : (int)a.N - 1;
          const uint8_t* src = a.sf + (int64_t)row * scales + (on ? step * n : 0);
          if constexpr (n == 16)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + r * n), "l"(src),
                         "r"(on ? n : 0)
                         : "memory");
          else
            asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(to + r * n), "l"(src),
                         "n"(n), "r"(on ? n : 0)
                         : "memory");
        }
      }
      asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(full(stage)) : "memory");
    };
    auto ask_x = [&](int step, int stage) {
      const uint32_t at = ring + stage * slot_bytes + kRows * kCodeBytes;
      if (one)
        for (int i = 0; i < sk / 64; ++i)
          tma_load_2d(at + i * sh.tokens * 128, &map_x, step * sk + i * 64, token0, full(stage), keep);
    };
    const int first = s1 - s0 < sh.stages ? s1 - s0 : sh.stages;
    for (int i = 0; i < first; ++i) ask_codes(s0 + i, i);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    for (int i = 0; i < first; ++i) ask_x(s0 + i, i);
    int stage = 0;
    uint32_t round = 0;
    int asked = first;
    for (int i = first; i < s1 - s0; ++i) {
      const bool ok = mbar_wait(empty(stage), round, &aborted, a.err, ERRW_TIMEOUT_PRODUCER, a.wait_ns);
      if (!__all_sync(0xFFFFFFFFu, ok)) break;
      ask_codes(s0 + i, stage);
      ask_x(s0 + i, stage);
      ++asked;
      if (++stage == sh.stages) {
        stage = 0;
        round ^= 1u;
      }
    }
    // every copy lands before the CTA ends, however short the caller's limit is
    int none = 0;
    for (int i = asked > sh.stages ? asked - sh.stages : 0; i < asked; ++i)
      mbar_wait(full(i % sh.stages), (uint32_t)(i / sh.stages) & 1u, &none, nullptr, 0, 0);
    __syncwarp();
  } else if (warp == kDecodeWarps) {
    // ---- products
    const uint32_t idesc = encode_idesc(KIND_F16, 0, 0, 128, sh.tokens, 0, 0);
    const uint32_t on = elect_one() ? 1u : 0u;
    int stage = 0, b = 0;
    uint32_t turn = 0;
    for (int i = 0; i < s1 - s0; ++i) {
      // the decoding warps waited for the slot, x included, before they arrived here
      const bool ok = mbar_wait(a_full(b), turn, &aborted, a.err, ERRW_TIMEOUT_MMA, a.wait_ns);
      if (!__all_sync(0xFFFFFFFFu, ok)) break;
      tc_fence_after();
      const uint32_t x = ring + stage * slot_bytes + kRows * kCodeBytes;
      // further descriptors differ in their low bits, by addresses in units of 16 bytes
      const uint64_t bd0 = encode_smem_desc(x, 16, 1024, SWZ_128B);
#pragma unroll
      for (int k = 0; k < sk / 16; ++k) {
        const uint64_t bd = bd0 + (uint32_t)(k / 4 * sh.tokens * 8 + k % 4 * 2);
        mma_ts<1, KIND_F16>(tmem, tmem_a + b * a_cols + 8 * k, bd, idesc, (i | k) != 0 ? 1u : 0u, on);
      }
      tc_commit<1>(a_empty(b), on);
      tc_commit<1>(empty(stage), on);
      __syncwarp();
      if (++b == buffers) {
        b = 0;
        turn ^= 1u;
      }
      if (++stage == sh.stages) stage = 0;
    }
    tc_commit<1>(done, on);
    // nothing of this warp is in flight when tensor memory is given back
    int none = 0;
    if (!mbar_wait(done, 0, &none, nullptr, 0, 0) && on) {
      aborted = 1;
      if (a.err) atomicOr(a.err, ERRW_TIMEOUT_MMA);
    }
    __syncwarp();
  } else {
    // ---- decoding: row `r`, one half of every other step
    const int quad = warp >> 2, group = quad / kHalves, half = quad % kHalves, r = (warp & 3) * 32 + lane;
    const int row = row0 + r < (int)a.N ? row0 + r : (int)a.N - 1;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const int scales = (int)a.kp / bf_block(FMT);             // of a row
    constexpr int per_step = sk / bf_block(FMT);
    const uint8_t* sf = a.sf + (int64_t)row * scales;
    uint32_t ref = 0;
    if constexpr (FMT != BF_NVFP4) {
      // the largest scale of eight steps spread over the slice, two of them a quad's; a NaN
      // scale says nothing of the others
#pragma unroll
      for (int q = 2 * quad; q < 2 * quad + 2; ++q) {
        const int first = (s0 + (s1 - s0) * q / 8) * per_step;
        uint32_t w[per_step / 4];
        if (sh.words) {
          if constexpr (per_step == 8) {
            const uint2 v = __ldg(reinterpret_cast<const uint2*>(sf + first));
            w[0] = v.x, w[1] = v.y;
          } else {
            w[0] = __ldg(reinterpret_cast<const uint32_t*>(sf + first));
          }
        } else {
#pragma unroll
          for (int i = 0; i < per_step / 4; ++i) w[i] = load_scales<4>(sf, first + 4 * i, scales);
        }
#pragma unroll
        for (int i = 0; i < per_step; ++i) {
          const uint32_t s = (w[i / 4] >> (8 * (i % 4))) & 0xFFu;
          ref = s > ref && s != 255u ? s : ref;
        }
      }
      atomicMax(&row_ref[r], ref);
      asm volatile("bar.sync 1, %0;" ::"n"(kDecodeWarps * 32) : "memory");
      ref = row_ref[r];
    }
    int stage = group, b = group;
    uint32_t round = 0, turn = 1;
    bool any_far = false;
    constexpr int mine_n = per_step / kHalves;  // scale bytes of a half: 8, 4 or 2
    constexpr int units = sk / kHalves / 32;    // of 32 elements
    const uint32_t to0 = tmem_a + lanes + half * (units * 16);
    for (int i = group; i < s1 - s0; i += kGroups) {
      bool ok = mbar_wait(full(stage), round, &aborted, a.err, ERRW_TIMEOUT_OTHER, a.wait_ns);
      ok = ok && (i < buffers || mbar_wait(a_empty(b), turn, &aborted, a.err, ERRW_TIMEOUT_OTHER, a.wait_ns));
      ok = __all_sync(0xFFFFFFFFu, ok);
      if (!ok) break;
      tc_fence_after();
      const uint32_t slot = ring + stage * slot_bytes, to = to0 + b * a_cols;
      uint32_t now[2] = {0u, 0u};
      if (sh.words) {
        const uint32_t at = slot + kRows * kCodeBytes + x_bytes + r * per_step + half * mine_n;
        if constexpr (mine_n == 8) {
          asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(now[0]), "=r"(now[1]) : "r"(at) : "memory");
        } else if constexpr (mine_n == 4) {
          asm volatile("ld.shared.u32 %0, [%1];" : "=r"(now[0]) : "r"(at) : "memory");
        } else {
          uint16_t h;
          asm volatile("ld.shared.u16 %0, [%1];" : "=h"(h) : "r"(at) : "memory");
          now[0] = h;
        }
      } else {
        const int first = (s0 + i) * per_step + half * mine_n;
#pragma unroll
        for (int k = 0; k < (mine_n + 3) / 4; ++k)
          now[k] = load_scales<mine_n < 4 ? mine_n : 4>(sf, first + 4 * k, scales);
      }
#pragma unroll
      for (int u = 0; u < units; ++u) {
        constexpr int pieces = bf_bits(FMT) / 4;  // of 16 bytes in a unit
        uint32_t c[4 * pieces];
#pragma unroll
        for (int p = 0; p < pieces; ++p)
          asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(c[4 * p]), "=r"(c[4 * p + 1]), "=r"(c[4 * p + 2]), "=r"(c[4 * p + 3])
                       : "r"(slot + r * kCodeBytes + ((((half * units + u) * pieces + p) ^ (r & 7)) << 4))
                       : "memory");
        // multipliers of the unit's halves
        uint32_t m[2];
        if constexpr (FMT == BF_NVFP4) {
          uint32_t h;
          asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)(now[u / 2] >> (16 * (u % 2)))));
          m[0] = __byte_perm(h, 0, 0x1010);
          m[1] = __byte_perm(h, 0, 0x3232);
        } else {
          const uint32_t s = (now[0] >> (8 * u)) & 0xFFu, e = s - ref + 15u;  // fp16's exponent
          m[0] = e * 0x04000400u;
          if (e - 1u > 14u + kAbove<FMT> || s == 255u) {
            m[0] = s == 255u ? 0x7E007E00u : 0u;
            any_far |= s != 255u && any_code<FMT>(c);
          }
          m[1] = m[0];
        }
        uint32_t f[16];
        if constexpr (FMT == BF_MXF8) {
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(f[k]) : "h"((uint16_t)(c[k >> 1] >> (16 * (k & 1)))));
            f[k] = mul_h2(f[k], m[0]);
          }
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint32_t q[4];
            e2m1x8_pairs(c[k], q);
#pragma unroll
            for (int j = 0; j < 4; ++j) f[4 * k + j] = mul_h2(q[j], m[k >> 1]);
          }
        }
        __syncwarp();
        tmem_st_32x32b_x16(to + u * 16, f);
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(a_full(b));
      b += kGroups;
      if (b >= buffers) {
        b -= buffers;
        turn ^= 1u;
      }
      stage += kGroups;
      if (stage >= sh.stages) {
        stage -= sh.stages;
        round ^= 1u;
      }
    }
    if constexpr (FMT != BF_NVFP4) has_far[quad][r] = any_far;
  }

  asm volatile("griddepcontrol.wait;" ::: "memory");  // over long since: xs and x16 are read now
  if (threadIdx.x < cols) token_scale[threadIdx.x] = __ldcg(xs + token0 + threadIdx.x);
  tc_fence_before();
  __syncthreads();  // the products are done and the copies landed (their warps waited for them)
  tc_fence_after();
  const int n = (int)a.N;
  const int64_t at = (int64_t)blockIdx.y * sh.row_tiles + tile;
  float* mine = part + (at * sh.slices + slice) * ((int64_t)sh.tokens * kRows);
  if (warp < kDecodeWarps && !aborted) {
    const int quad = warp >> 2, r = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const int first = quad * (sh.tokens / kQuads);  // of this thread's tokens
    float scale = 1.0f;
    bool any_far = false;
    // the ring is free: 64 KB of it for 32 tokens a thread
    float* far = static_cast<float*>(__cvta_shared_to_generic(ring)) + threadIdx.x;
    if constexpr (FMT != BF_NVFP4) {
      scale = e8m0_value(row_ref[r]);
#pragma unroll
      for (int q = 0; q < kQuads; ++q) any_far |= has_far[q][r] != 0;
      const int left = cols - first, count = left < sh.tokens / kQuads ? left : sh.tokens / kQuads;
      if (any_far)
        far_blocks<FMT>(a, x16 + (int64_t)(token0 + first) * sh.steps * sk, (int64_t)sh.steps * sk,
                        row0 + r < n ? row0 + r : n - 1, s0 * sk, min(s1 * sk, (int)a.kp), row_ref[r], count,
                        far);
      __syncwarp();
    }
    for (int j = 0; j < sh.tokens / kQuads; j += 4) {
      float v[4];
      asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0, %1, %2, %3}, [%4];"
                   : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3])
                   : "r"(tmem + lanes + first + j));
      tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int t = first + j + i;
        if (t >= cols) break;
        float sum = FMT == BF_NVFP4 || v[i] == 0.0f ? v[i] : v[i] * scale;
        if constexpr (FMT != BF_NVFP4) {
          if (any_far) sum += far[(j + i) * kDecodeWarps * 32];
        }
        if (sh.slices > 1)
          __stcg(mine + t * kRows + r, sum);
        else if (row0 + r < n)
          static_cast<T*>(a.out)[(int64_t)(token0 + t) * a.ld_out + row0 + r] =
              from_f32<T>(a.alpha * (sum * token_scale[t]));
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kDecodeWarps) tmem_dealloc<1>(tmem, 512);
  if (sh.slices == 1) return;
  // the CTA that arrives last adds the slices, always in the same order
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) {
    last = atomicAdd(a.count + at, 1u) == (uint32_t)sh.slices - 1u;
    if (last) a.count[at] = 0u;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  const float* all = part + at * sh.slices * ((int64_t)sh.tokens * kRows);
  // four rows of a token at a time
  const int64_t stride = (int64_t)sh.tokens * kRows / 4;
#pragma unroll 2
  for (int e = threadIdx.x; e < cols * (kRows / 4); e += kThreads) {
    const int t = e / (kRows / 4), r = e % (kRows / 4) * 4;
    const float4* p = reinterpret_cast<const float4*>(all) + e;
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
    for (int k = 0; k < sh.slices; ++k) {
      const float4 q = __ldcg(p + k * stride);
      sum.x += q.x;
      sum.y += q.y;
      sum.z += q.z;
      sum.w += q.w;
    }
    const float s = token_scale[t], v[4] = {sum.x, sum.y, sum.z, sum.w};
    T* dst = static_cast<T*>(a.out) + (int64_t)(token0 + t) * a.ld_out + row0 + r;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (row0 + r + i < n) dst[i] = from_f32<T>(a.alpha * (v[i] * s));
  }
}

TileShape tile_shape(int fmt, const FewLinearArgs& a, int sm_count) {
  TileShape s;
  const int64_t t = a.T < 128 ? a.T : 128;
  s.tokens = (int)((t + 15) / 16 * 16);
  s.z = (int)((a.T + 127) / 128);
  s.steps = (int)((a.kp + step_k(fmt) - 1) / step_k(fmt));
  s.row_tiles = (int)((a.N + kRows - 1) / kRows);
  const int scales = step_k(fmt) / bf_block(fmt);  // of a row in a step
  s.words = a.kp / bf_block(fmt) % scales == 0 && (reinterpret_cast<uintptr_t>(a.sf) % scales) == 0;
  // one CTA an SM; K is cut as far as there are SMs left and each CTA keeps two steps
  int n = sm_count / (s.row_tiles * s.z);
  n = n < s.steps / 2 ? n : s.steps / 2;
  s.slices = n < 1 ? 1 : n;
  const int slot = kRows * kCodeBytes + s.tokens * step_k(fmt) * 2 + kScaleBytes;
  s.stages = (220 * 1024) / slot < kMaxStages ? (220 * 1024) / slot / kGroups * kGroups : kMaxStages;
  s.smem = s.stages * slot + 1024;
  // tensor memory is taken whole: one CTA an SM
  if (s.smem < 120 * 1024) s.smem = 120 * 1024;
  return s;
}

size_t up256(size_t n) { return (n + 255) / 256 * 256; }

struct TileWs {
  size_t x16, xs, part, total;
};

TileWs tile_ws(int fmt, const FewLinearArgs& a, const TileShape& s) {
  TileWs w;
  w.x16 = 0;
  w.xs = up256((size_t)a.T * s.steps * step_k(fmt) * 2);
  w.part = w.xs + up256((size_t)a.T * sizeof(float));
  const size_t ctas = (size_t)s.row_tiles * s.slices * s.z;
  w.total = w.part + (s.slices > 1 ? ctas * s.tokens * kRows * sizeof(float) : 0);
  return w;
}

template <typename T, int FMT>
cudaError_t tiles_launch(const FewLinearArgs& a, const TileShape& sh, const CUtensorMap& mw,
                         const CUtensorMap& mx, const TileWs& w, cudaStream_t s) {
  char* ws = static_cast<char*>(a.ws);
  float* xs = reinterpret_cast<float*>(ws + w.xs);
  tiles_prepare_kernel<T><<<(unsigned)a.T, 512, 0, s>>>(a, (int64_t)sh.steps * step_k(FMT),
                                                        reinterpret_cast<__half*>(ws + w.x16), xs);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  static std::atomic<int> seen[16];
  e = allow_smem(few_tiles_kernel<T, FMT>, sh.smem, seen);
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(sh.row_tiles * sh.slices), (unsigned)sh.z);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = (size_t)sh.smem;
  cfg.stream = s;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, few_tiles_kernel<T, FMT>, mw, mx, a, sh,
                            reinterpret_cast<const __half*>(ws + w.x16), static_cast<const float*>(xs),
                            reinterpret_cast<float*>(ws + w.part));
}

}  // namespace

size_t few_tiles_ws_bytes(int fmt, const FewLinearArgs& a, int sm_count) {
  return tile_ws(fmt, a, tile_shape(fmt, a, sm_count)).total;
}

size_t few_tiles_counters(int fmt, const FewLinearArgs& a, int sm_count) {
  const TileShape s = tile_shape(fmt, a, sm_count);
  return s.slices > 1 ? (size_t)s.row_tiles * s.z : 0;
}

void few_tiles_maps(int fmt, const FewLinearArgs& a, int sm_count, FewTilesMaps* m) {
  const TileShape s = tile_shape(fmt, a, sm_count);
  m->w_row_bytes = (uint64_t)(a.kp * bf_bits(fmt) / 8);
  m->w_box_bytes = kCodeBytes;
  m->w_box_rows = kRows;
  m->x_cols = (uint64_t)s.steps * step_k(fmt);
  m->x_box_cols = 64;
  m->x_box_rows = (uint32_t)s.tokens;
}

cudaError_t launch_few_tiles(int fmt, int type, const FewLinearArgs& a, const CUtensorMap& map_w,
                             const CUtensorMap& map_x, int sm_count, cudaStream_t s) {
  const TileShape sh = tile_shape(fmt, a, sm_count);
  const TileWs w = tile_ws(fmt, a, sh);
  if (type == B2G_BF16) {
    if (fmt == BF_NVFP4) return tiles_launch<__nv_bfloat16, BF_NVFP4>(a, sh, map_w, map_x, w, s);
    if (fmt == BF_MXF4) return tiles_launch<__nv_bfloat16, BF_MXF4>(a, sh, map_w, map_x, w, s);
    return tiles_launch<__nv_bfloat16, BF_MXF8>(a, sh, map_w, map_x, w, s);
  }
  if (fmt == BF_NVFP4) return tiles_launch<__half, BF_NVFP4>(a, sh, map_w, map_x, w, s);
  if (fmt == BF_MXF4) return tiles_launch<__half, BF_MXF4>(a, sh, map_w, map_x, w, s);
  return tiles_launch<__half, BF_MXF8>(a, sh, map_w, map_x, w, s);
}

}  // namespace b2g
