// few_linear.cu -- y = alpha * x . W^T of one to eight tokens (16-bit x) with microscaled
// weights, for decoding: every weight is read once and used a handful of times, so the
// weights' bytes are the floor.
//
// Codes become fp16 pairs in registers and go into mma.sync m16n8k16 with the weights
// as the 16-row operand and the tokens as the 8 columns: tcgen05 takes its operands
// from shared or tensor memory, so a decoded weight would have to be stored first, for
// products whose own time does not count at this many tokens.  e2m1 and e4m3 values and
// e2m1 * ue4m3 products are exact in fp16; sums are fp32.  A first kernel lays x out as
// fp16: fp16 as it is, bf16 scaled per token by the power of two that brings its largest
// value to 2^14 .. 2^15, which is exact for values down to 2^-28 of the largest (below
// that the error is at most 2^-40 of the largest).  The second one starts along with it
// and has its first weights on their way by the time x is laid out.  (Every CTA laying all of
// x out for itself, without a first kernel: 2048 x 2048 3.8 for 4.5 us, but 8192 x 8192 14.5
// for 13.4 us.)
//
// Measured, one token: 8192 x 8192 NVFP4 13.4 us, MXFP4 13.4, MXFP8 18.2; 16384 x 8192 22.5,
// 23.4, 30.4 (2.9 to 4.6 TB/s); 2048 x 2048 4.5 to 4.8 us.  About 4 us of it are the two
// launches' latencies; beyond, instructions: 2.4 an element and lane, at 16 warps an SM.
#include "b2g.h"
#include "op_common.cuh"
#include "op_kernels.h"

namespace b2g {
namespace {

constexpr int kWarps = 8;

// k-order inside the kernel: a thread takes 32 neighbouring elements of a row (16 or 32
// bytes of codes), the four threads of a quad a group of 128; MMA step j of a group
// multiplies elements 4 j .. 4 j + 3 of each thread.  Any order of k serves as long as
// both operands use it, so no code is moved between threads.
constexpr int kSpan = 32, kGroup = 128;
constexpr int kPairs = kSpan / 8;  // step pairs of a group

// A warp asks for 128 bytes of codes of each of its 16 rows at a time, whole cache lines:
// a step of 256 (4 bits) or 128 (8 bits) elements.
__host__ __device__ constexpr int few_groups(int fmt) { return 8 / bf_bits(fmt); }  // of a step
__host__ __device__ constexpr int few_step(int fmt) { return few_groups(fmt) * kGroup; }

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

// fp16 pairs of the eight elements of steps 2 jp and 2 jp + 1
template <int FMT>
__device__ __forceinline__ void decode_steps(const uint32_t (&w)[bf_bits(FMT)], int jp,
                                             uint32_t (&p)[4]) {
  if constexpr (FMT == BF_MXF8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint16_t h = (uint16_t)(w[2 * jp + (i >> 1)] >> (16 * (i & 1)));
      asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(p[i]) : "h"(h));
    }
  } else {
    e2m1x8_pairs(w[jp], p);
  }
}

// A thread's codes of one group (rows g and g + 8 of the warp's 16) and their scale
// bytes: two of NVFP4, one of MX.
template <int FMT>
struct GroupData {
  uint32_t w[2][bf_bits(FMT)];
  uint32_t s[2];
};

template <typename V>
__device__ __forceinline__ V shared_at(uint32_t address) {
  return *static_cast<const V*>(__cvta_shared_to_generic(address));
}

__device__ __forceinline__ void cp_async16(uint32_t smem, const void* src, bool on) {
  const int n = on ? 16 : 0;  // 0: zeros, src is not read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem), "l"(src), "r"(n)
               : "memory");
}

__device__ __forceinline__ void cp_async4(uint32_t smem, const void* src, bool on) {
  const int n = on ? 4 : 0;
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem), "l"(src), "r"(n)
               : "memory");
}

// A warp's ring of steps in shared memory, filled asynchronously.  A slot holds the codes
// as [row][8 pieces of 16 bytes] and the scales as [row][bytes].  In odd rows the pieces
// are exchanged (4 bits: the halves, 8 bits: neighbours), so that the eight lanes of two
// rows that read 16 bytes each at a time meet different banks.
template <int FMT>
struct Ring {
  static constexpr int kScale = few_step(FMT) / bf_block(FMT);  // scale bytes of a row
  static constexpr int kWords = kScale / 4;
  static constexpr int kSlot = 2048 + 16 * kScale;              // bytes
  static constexpr int kSwap = FMT == BF_MXF8 ? 1 : 4;

  uint32_t base;          // shared address
  int lane, kp;
  bool words;             // scales are copied in 4-byte words
  const uint8_t* w;       // codes of row lane / 8 at piece lane % 8 of a step
  const uint8_t* sf;      // first scale of the 16 rows
  int pitch;              // bytes between rows of codes
  int last_row;           // rows past N repeat this one and are not stored

  // the 16 rows from row0 on
  __device__ __forceinline__ void rows(const FewLinearArgs& a, int row0) {
    last_row = (int)a.N - 1 - row0;
    w = a.w + (int64_t)row0 * pitch + lane % 8 * 16;
    sf = a.sf + (int64_t)row0 * (kp / bf_block(FMT));
  }

  __device__ __forceinline__ void fill(int slot, int step) const {
    const uint32_t at = base + slot * kSlot;
    const int k = step * few_step(FMT);
    const bool on = k + lane % 8 * (128 / bf_bits(FMT)) < kp;
    const uint8_t* src = w + (on ? (uint32_t)step * 128u : 0u);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = i * 4 + lane / 8;
      cp_async16(at + row * 128 + ((lane % 8) ^ (row & 1 ? kSwap : 0)) * 16,
                 src + (int64_t)min(row, last_row) * pitch, on);
    }
    const uint32_t st = at + 2048;
    const int b = k / bf_block(FMT), end = kp / bf_block(FMT);  // scale bytes of a row
    if (words) {
#pragma unroll
      for (int i = 0; i < (16 * kWords + 31) / 32; ++i) {
        const int word = i * 32 + lane;
        if (word < 16 * kWords) {
          const bool in = b + word % kWords * 4 < end;
          cp_async4(st + word * 4,
                    sf + (int64_t)min(word / kWords, last_row) * end + (in ? b + word % kWords * 4 : 0), in);
        }
      }
    } else {
      // rows of scales off 4 bytes: one byte at a time, past the end the last one
      for (int i = lane; i < 16 * kScale; i += 32) {
        const int c = min(b + i % kScale, end - 1);
        const uint32_t s = __ldg(sf + (int64_t)min(i / kScale, last_row) * end + c);
        asm volatile("st.shared.u8 [%0], %1;" ::"r"(st + i), "r"(s) : "memory");
      }
    }
  }

  // group `part` of the step in `slot`
  __device__ __forceinline__ void read(int slot, int part, GroupData<FMT>& d) const {
    const uint32_t at = base + slot * kSlot;
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < bf_bits(FMT) / 4; ++j) {
        const int piece = FMT == BF_MXF8 ? 2 * t + j : part * 4 + t;
        const uint4 v = shared_at<uint4>(at + (g + 8 * i) * 128 + (piece ^ (g & 1 ? kSwap : 0)) * 16);
        d.w[i][4 * j] = v.x;
        d.w[i][4 * j + 1] = v.y;
        d.w[i][4 * j + 2] = v.z;
        d.w[i][4 * j + 3] = v.w;
      }
    const uint32_t st = at + 2048;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if constexpr (FMT == BF_NVFP4)
        d.s[i] = shared_at<uint16_t>(st + (g + 8 * i) * kScale + part * 8 + t * 2);
      else
        d.s[i] = shared_at<uint8_t>(st + (g + 8 * i) * kScale + part * 4 + t);
    }
  }
};

// c += codes of one group, times the fp16 pairs m, times x.  m[i]: multipliers of row
// g + 8 i for the first and the second half of the thread's elements.  xf: shared address
// of the lane's fragments, one step pair `step` bytes after the other, their 16-byte place
// xor'ed with the step pair where swz is set.
template <int FMT>
__device__ __forceinline__ void codes_mma(const GroupData<FMT>& d, const uint32_t (&m)[2][2],
                                          uint32_t xf, uint32_t step, uint32_t swz, float (&c)[4]) {
#pragma unroll
  for (int jp = 0; jp < kPairs; ++jp) {
    uint32_t f[2][4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t p[4];
      decode_steps<FMT>(d.w[i], jp, p);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        f[k >> 1][i + 2 * (k & 1)] = mul_h2(p[k], m[i][jp < kPairs / 2 ? 0 : 1]);
    }
    const uint4 b = shared_at<uint4>((xf ^ (swz & (16u * jp))) + jp * step);
    mma_f16(c, f[0], b.x, b.y);
    mma_f16(c, f[1], b.z, b.w);
  }
}

// Sums of a warp.  NVFP4: scales are multiplied into the codes, sums are final.  MX: an
// E8M0 scale has more range than fp16, so codes are multiplied by 2^(s - ref) with one
// ref for each row, and the sum by 2^ref in fp32 when ref changes and at the end.
template <int FMT>
struct Sums {
  float c[4];
  float total[4];  // MX: what earlier refs summed up
  int ref[2];      // MX: of rows g and g + 8, the same in a quad

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = total[i] = 0.0f;
    ref[0] = ref[1] = 127;
  }

  // total += c * 2^ref, c = 0
  __device__ __forceinline__ void flush() {
    const float s0 = e8m0_value((uint32_t)ref[0]), s1 = e8m0_value((uint32_t)ref[1]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // a sum that is still zero stays zero, whatever its ref
      if (c[i] != 0.0f) total[i] = fmaf(i < 2 ? s0 : s1, c[i], total[i]);
      c[i] = 0.0f;
    }
  }

  // d = s - ref of a scale that keeps 2^d times any element normal and finite in fp16:
  // -14 .. 13 (e2m1, at most 6) or 7 (e4m3, at most 448)
  static constexpr unsigned kSpread = 14 + (FMT == BF_MXF8 ? 7 : 13);

  // whether a scale of the group does not fit its row's ref
  __device__ __forceinline__ bool far(const GroupData<FMT>& d) const {
    if constexpr (FMT == BF_NVFP4) return false;
    return (unsigned)((int)d.s[0] - ref[0] + 14) > kSpread ||
           (unsigned)((int)d.s[1] - ref[1] + 14) > kSpread;
  }

  // a group whose scales fit
  __device__ __forceinline__ void add(const GroupData<FMT>& d, uint32_t xf, uint32_t step, uint32_t swz) {
    uint32_t m[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if constexpr (FMT == BF_NVFP4) {
        uint32_t h;
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)d.s[i]));
        m[i][0] = __byte_perm(h, 0, 0x1010);
        m[i][1] = __byte_perm(h, 0, 0x3232);
      } else {
        m[i][0] = m[i][1] = (uint32_t)((int)d.s[i] - ref[i] + 15) * 0x04000400u;
      }
    }
    codes_mma<FMT>(d, m, xf, step, swz, c);
  }

  // Any group: the largest scale of each row's four threads becomes ref.  Blocks of zeros
  // fit any.  If the four are too far apart, they are multiplied one thread's blocks at a
  // time, each with its own scale as ref.  A NaN scale (255) makes its multiplier NaN.
  __device__ __forceinline__ void add_any(const GroupData<FMT>& d, uint32_t xf, uint32_t step, uint32_t swz) {
    const int lane = threadIdx.x & 31, t = lane & 3;
    int s[2], top[2];
    bool wide = false;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t any = 0u;
#pragma unroll
      for (int k = 0; k < bf_bits(FMT); ++k) any |= d.w[i][k];
      const bool zero = (any & (FMT == BF_MXF8 ? 0x7F7F7F7Fu : 0x77777777u)) == 0u;
      s[i] = zero && d.s[i] != 255u ? 0 : (int)d.s[i];
      top[i] = max(s[i], __shfl_xor_sync(0xFFFFFFFFu, s[i], 1));
      top[i] = max(top[i], __shfl_xor_sync(0xFFFFFFFFu, top[i], 2));
      wide |= !zero && s[i] < top[i] - 14;
    }
    wide = __any_sync(0xFFFFFFFFu, wide || top[0] == 255 || top[1] == 255);
#pragma unroll 1
    for (int p = 0; p < (wide ? 4 : 1); ++p) {
      flush();
      uint32_t m[2][2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int one = __shfl_sync(0xFFFFFFFFu, s[i], (lane & ~3) + p);
        ref[i] = wide ? one : top[i];
        const uint32_t e = (uint32_t)(max(s[i] - top[i], -14) + 15) * 0x04000400u;
        m[i][0] = m[i][1] = !wide ? e : t != p ? 0u : s[i] == 255 ? 0x7E007E00u : 0x3C003C00u;
      }
      codes_mma<FMT>(d, m, xf, step, swz, c);
    }
  }
};

// Work of a launch.  K is cut into `slices`; CTA c keeps slice c % slices and has that part
// of x in shared memory.  k_split 1: each warp takes row blocks of 16 by itself, every
// (rows_ctas * kWarps)-th one.  k_split kWarps: the warps of a CTA share a row block and
// cut its K among them.
struct FewShape {
  int steps, slices, rows_ctas, k_split;
  int groups;      // of 128 elements, whole steps
  int words;       // rows of scales start on 4 bytes
  int x_bytes;     // shared memory of a CTA's part of x
};

// Steps of weights a warp has on their way: at two CTAs an SM 4 x 2 KB x 16 = 128 KB, which
// covers the memory's latency at its rate.  Measured: 8192 x 8192, one token, NVFP4 13.4 us; 6
// steps, which leave one CTA an SM, 17.0 us; 3 steps and three CTAs 15.1 us.
constexpr int kAhead = 4;

// x as fp16 B fragments: [group][step pair][4 threads][token] of 16 bytes, the four
// elements of two steps; xs[token] = the power of two to undo.  Of eight tokens column c of thread t and pair jp lies at c ^ (jp + 4 (t % 2)): the lanes that
// read it, and the eight neighbours that write one column, meet different banks.  Zero past
// K up to the end of the last group.  One CTA per token.
template <typename T>
__global__ void __launch_bounds__(512) few_prepare_kernel(const FewLinearArgs a, const FewShape sh,
                                                          uint4* frag, float* xs) {
  __shared__ float red[16];
  const int token = blockIdx.x, tokens = (int)a.T;
  const int vecs = sh.groups * (kGroup / 8);
  const T* x = static_cast<const T*>(a.x) + (int64_t)token * a.ld_x;
  // the product kernel may start and load weights; it waits for this one to end before
  // it reads x
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  float scale = 1.0f;
  constexpr int kHold = 4;  // eights a thread keeps between the two passes
  Raw8<T> raw[kHold];
#pragma unroll
  for (int i = 0; i < kHold; ++i) {
    const int v = threadIdx.x + i * 512;
    const int64_t left = a.K - (int64_t)v * 8;
    raw[i] = load8(x + (int64_t)v * 8, left < 0 ? 0 : left < 8 ? (int)left : 8, a.x_vec);
  }
  auto at = [&](int v, int i) {
    if (i < kHold) return raw[i];
    const int64_t left = a.K - (int64_t)v * 8;
    return load8(x + (int64_t)v * 8, left < 0 ? 0 : left < 8 ? (int)left : 8, a.x_vec);
  };
  if constexpr (__is_same(T, __nv_bfloat16)) {
    float amax = 0.0f;
    auto take = [&](const Raw8<T>& r) {
      float f[8];
      unpack8(r, f);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float m = fabsf(f[i]);
        amax = fmaxf(amax, m < __uint_as_float(0x7F800000u) ? m : 0.0f);  // of the finite ones
      }
    };
#pragma unroll
    for (int i = 0; i < kHold; ++i) take(raw[i]);
    for (int i = kHold, v = threadIdx.x + kHold * 512; v < vecs; ++i, v += 512) take(at(v, i));
    const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(amax));
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = __uint_as_float(top);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 16; ++i) amax = fmaxf(amax, red[i]);
    // exponent field of 2^(14 - floor(log2 amax)), at most 2^126
    int e = 127 + 14 - ((int)(__float_as_uint(amax) >> 23) - 127);
    e = e > 253 ? 253 : e;
    scale = amax > 0.0f ? __uint_as_float((uint32_t)e << 23) : 1.0f;
  }
  if (threadIdx.x == 0) xs[token] = 1.0f / scale;
  auto put = [&](int v, const Raw8<T>& r) {
    // eight elements: one step pair of one thread
    const int in = v % (kGroup / 8), jp = in % kPairs, t = in / kPairs;
    uint4 w = r.w[0];
    if constexpr (__is_same(T, __nv_bfloat16)) {
      float f[8];
      unpack8(r, f);
      w.x = pack2<__half>(f[0] * scale, f[1] * scale);
      w.y = pack2<__half>(f[2] * scale, f[3] * scale);
      w.z = pack2<__half>(f[4] * scale, f[5] * scale);
      w.w = pack2<__half>(f[6] * scale, f[7] * scale);
    }
    const int place = tokens == 8 ? token ^ (jp | (t & 1) << 2) : token;
    frag[((v / (kGroup / 8) * kPairs + jp) * 4 + t) * tokens + place] = w;
  };
#pragma unroll
  for (int i = 0; i < kHold; ++i) {
    const int v = threadIdx.x + i * 512;
    if (v < vecs) put(v, raw[i]);
  }
  for (int i = kHold, v = threadIdx.x + kHold * 512; v < vecs; ++i, v += 512) put(v, at(v, i));
}

template <typename T, int FMT>
__global__ void __launch_bounds__(kWarps * 32, 2)
few_linear_kernel(const FewLinearArgs a, const FewShape sh, const uint4* frag, const float* xs,
                  float* part) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float red[2][kWarps][128];  // k_split: sums of the warps
  constexpr int kSlots = kAhead;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const bool split = sh.k_split > 1;
  const int slice = (int)blockIdx.x % sh.slices;
  // steps of this CTA and of this warp
  const int cb = (int)((unsigned)sh.steps * (unsigned)slice / (unsigned)sh.slices);
  const int ce = (int)((unsigned)sh.steps * (slice + 1u) / (unsigned)sh.slices);
  const int gb = split ? cb + (ce - cb) * warp / kWarps : cb;
  const int ge = split ? cb + (ce - cb) * (warp + 1) / kWarps : ce;
  const int row_blocks = ((int)a.N + 15) / 16;
  const int rb_step = split ? sh.rows_ctas : sh.rows_ctas * kWarps;
  const int rb0 = split ? (int)blockIdx.x / sh.slices : (int)blockIdx.x / sh.slices * kWarps + warp;

  // position of the next step to ask for
  Ring<FMT> ring;
  ring.kp = (int)a.kp;
  ring.pitch = (int)(a.kp * bf_bits(FMT) / 8);
  ring.lane = lane;
  ring.base = (uint32_t)__cvta_generic_to_shared(smem) + sh.x_bytes + warp * kSlots * Ring<FMT>::kSlot;
  ring.words = sh.words;
  int ask_rb = gb < ge ? rb0 : row_blocks, ask_g = gb;
  if (ask_rb < row_blocks) ring.rows(a, ask_rb * 16);
  auto ask = [&](int slot) {
    if (ask_rb < row_blocks) {
      ring.fill(slot, ask_g);
      if (++ask_g == ge) {
        ask_g = gb;
        ask_rb += rb_step;
        if (ask_rb < row_blocks) ring.rows(a, ask_rb * 16);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll 1
  for (int u = 0; u < kSlots; ++u) ask(u);

  const int cols = (int)a.T;
  const uint32_t step = 64 * cols;  // bytes of an MMA step pair
  const uint32_t group_bytes = kPairs * step;
  constexpr int kParts = few_groups(FMT);
  const uint32_t x_smem = (uint32_t)__cvta_generic_to_shared(smem);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  {
    const uint32_t bytes = (uint32_t)(ce - cb) * kParts * group_bytes;
    const uint8_t* src = reinterpret_cast<const uint8_t*>(frag) + (int64_t)cb * kParts * group_bytes;
    for (uint32_t i = threadIdx.x * 16; i < bytes; i += kWarps * 32 * 16)
      cp_async16(x_smem + i, src + i, true);
    asm volatile("cp.async.commit_group;" ::: "memory");
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
  }

  // columns past T repeat another one's or hold anything, and are not stored
  const uint32_t swz = cols == 8 ? 0x70u : 0u;
  const uint32_t xf0 = x_smem + (uint32_t)(gb - cb) * kParts * group_bytes +
                       (t * cols + (cols == 8 ? g ^ (t & 1) << 2 : g < cols ? g : 0)) * 16;
  int slot = 0, turn = 0;
#pragma unroll 1
  for (int rb = rb0; rb < row_blocks; rb += rb_step, turn ^= 1) {
    Sums<FMT> sums;
    sums.clear();
    uint32_t xf = xf0;
#pragma unroll 1
    for (int gi = gb; gi < ge; ++gi) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kSlots - 1) : "memory");
      __syncwarp();  // rows come from several lanes' copies
      GroupData<FMT> d[kParts];
#pragma unroll
      for (int k = 0; k < kParts; ++k) ring.read(slot, k, d[k]);
      __syncwarp();
      ask(slot);
      slot = slot == kSlots - 1 ? 0 : slot + 1;
#pragma unroll
      for (int k = 0; k < kParts; ++k) {
        if (FMT != BF_NVFP4 && __any_sync(0xFFFFFFFFu, sums.far(d[k])))
          sums.add_any(d[k], xf, step, swz);
        else
          sums.add(d[k], xf, step, swz);
        xf += group_bytes;
      }
    }
    if constexpr (FMT != BF_NVFP4) sums.flush();

    // accumulator i of lane (g, t): row g + 8 (i / 2), token 2 t + i % 2
    const float(&sum)[4] = FMT == BF_NVFP4 ? sums.c : sums.total;
    float* mine = part + ((int64_t)rb * sh.slices + slice) * 128;
    auto put = [&](int token, int row, float s) {
      if (token < cols && row < (int)a.N)
        static_cast<T*>(a.out)[token * a.ld_out + row] = from_f32<T>(a.alpha * s);
    };
    if (split) {
      // two buffers: a warp writes one again only after the barrier of the other
#pragma unroll
      for (int i = 0; i < 4; ++i)
        red[turn][warp][(2 * t + (i & 1)) * 16 + g + 8 * (i >> 1)] = sum[i];
      __syncthreads();
      const int e = threadIdx.x;
      if (e < cols * 16) {
        float s = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) s += red[turn][w][e];
        s *= xs[e / 16];
        if (sh.slices == 1)
          put(e / 16, rb * 16 + e % 16, s);
        else
          __stcg(mine + e, s);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int token = 2 * t + (i & 1), r = g + 8 * (i >> 1);
        if (token >= cols) continue;
        const float s = sum[i] * xs[token];
        if (sh.slices == 1)
          put(token, rb * 16 + r, s);
        else
          __stcg(mine + token * 16 + r, s);
      }
    }
    if (sh.slices == 1) continue;
    // the warp (k_split: the CTA's first warps, one after the other) that arrives last at
    // the row block adds the slices, always in the same order; part: [row
    // block][slice][token][16 rows]
    if (split) {
      if (warp * 32 >= cols * 16) continue;
    }
    __threadfence();
    __syncwarp();
    const uint32_t arrivals = (uint32_t)sh.slices * (split ? (cols * 16 + 31) / 32 : 1);
    uint32_t before = 0;
    if (lane == 0) before = atomicAdd(a.count + rb, 1u);
    before = __shfl_sync(0xFFFFFFFFu, before, 0);
    if (before != arrivals - 1u) continue;
    if (lane == 0) a.count[rb] = 0u;
    __threadfence();
    const float* all = part + (int64_t)rb * sh.slices * 128;
    // four rows of one token at a time
    for (int e = lane * 4; e < cols * 16; e += 128) {
      float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
      for (int k = 0; k < sh.slices; ++k) {
        const float4 p = __ldcg(reinterpret_cast<const float4*>(all + k * 128 + e));
        s.x += p.x;
        s.y += p.y;
        s.z += p.z;
        s.w += p.w;
      }
      const int row = rb * 16 + e % 16;
      put(e / 16, row, s.x);
      put(e / 16, row + 1, s.y);
      put(e / 16, row + 2, s.z);
      put(e / 16, row + 3, s.w);
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

FewShape few_shape(int fmt, const FewLinearArgs& a, int sm_count) {
  FewShape s;
  const int cols = (int)a.T;
  s.steps = (int)((a.kp + few_step(fmt) - 1) / few_step(fmt));
  s.groups = s.steps * few_groups(fmt);
  s.words = a.kp / bf_block(fmt) % 4 == 0 && (reinterpret_cast<uintptr_t>(a.sf) & 3) == 0;
  // All of x in a CTA: its warps share the row blocks, and no sums pass through global memory
  // (NVFP4, one by one / shared: 2048 x 2048 7.2 / 4.6 us of one token, 7.3 / 4.8 us of eight).
  // Not with parts of x: 8192 x 8192 of eight tokens 17.5 / 41 us, with many ends of row blocks.
  const int64_t x_all = (int64_t)s.groups * cols * kGroup * 2;
  s.k_split = x_all <= kFewXBytes ? kWarps : 1;
  const int ctas = 2 * sm_count;  // that run at a time
  const int64_t row_blocks = (a.N + 15) / 16, per_cta = kWarps / s.k_split;
  // a warp has at least two steps of a row block; between the bounds, the cut that leaves
  // the busiest warp the least work
  const int least = (int)((x_all + kFewXBytes - 1) / kFewXBytes);
  const int most = s.steps / (2 * s.k_split) > least ? s.steps / (2 * s.k_split) : least;
  int64_t best = INT64_MAX;
  s.slices = least;
  s.rows_ctas = 1;
  for (int n = least; n <= most && n <= ctas; ++n) {
    const int rows_ctas = ctas / n;
    const int64_t per = (row_blocks + rows_ctas * per_cta - 1) / (rows_ctas * per_cta);
    // in halves of a step, with about one for ending a row block and another for adding slices
    const int64_t work = per * (2 * ((s.steps + n * s.k_split - 1) / (n * s.k_split)) + (n > 1 ? 2 : 1));
    if (work < best) {
      best = work;
      s.slices = n;
      s.rows_ctas = rows_ctas;
    }
  }
  // no more CTAs than row blocks need
  const int64_t need = (row_blocks + per_cta - 1) / per_cta;
  if (s.rows_ctas > need) s.rows_ctas = (int)need;
  s.x_bytes = (s.steps + s.slices - 1) / s.slices * few_groups(fmt) * cols * kGroup * 2;
  return s;
}

size_t up256(size_t n) { return (n + 255) / 256 * 256; }

size_t frag_bytes(const FewShape& s, int64_t T) { return up256((size_t)s.groups * kPairs * 64 * T); }

template <typename T, int FMT>
cudaError_t few_launch(const FewLinearArgs& a, int sm_count, cudaStream_t s) {
  const FewShape sh = few_shape(FMT, a, sm_count);
  uint4* frag = static_cast<uint4*>(a.ws);
  float* xs = reinterpret_cast<float*>(static_cast<char*>(a.ws) + frag_bytes(sh, a.T));
  float* part = xs + up256(a.T * sizeof(float)) / sizeof(float);
  few_prepare_kernel<T><<<(unsigned)a.T, 512, 0, s>>>(a, sh, frag, xs);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  const int smem = sh.x_bytes + kWarps * kAhead * Ring<FMT>::kSlot;
  static std::atomic<int> seen[16];
  e = allow_smem(few_linear_kernel<T, FMT>, smem, seen);
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(sh.slices * sh.rows_ctas));
  cfg.blockDim = dim3(kWarps * 32);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = s;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, few_linear_kernel<T, FMT>, a, sh,
                            static_cast<const uint4*>(frag), static_cast<const float*>(xs), part);
}

template <typename T>
cudaError_t few_fmt_launch(int fmt, const FewLinearArgs& a, int sm_count, cudaStream_t s) {
  if (fmt == BF_NVFP4) return few_launch<T, BF_NVFP4>(a, sm_count, s);
  if (fmt == BF_MXF4) return few_launch<T, BF_MXF4>(a, sm_count, s);
  return few_launch<T, BF_MXF8>(a, sm_count, s);
}

}  // namespace

size_t few_linear_ws_bytes(int fmt, const FewLinearArgs& a, int sm_count) {
  const FewShape s = few_shape(fmt, a, sm_count);
  const size_t part = s.slices == 1 ? 0 : (size_t)((a.N + 15) / 16) * s.slices * 128 * sizeof(float);
  return frag_bytes(s, a.T) + up256(a.T * sizeof(float)) + part;
}

size_t few_linear_counters(int fmt, const FewLinearArgs& a, int sm_count) {
  const FewShape s = few_shape(fmt, a, sm_count);
  return s.slices > 1 ? (size_t)((a.N + 15) / 16) : 0;
}

cudaError_t launch_few_linear(int fmt, int type, const FewLinearArgs& a, int sm_count,
                              cudaStream_t s) {
  if (type == B2G_BF16) return few_fmt_launch<__nv_bfloat16>(fmt, a, sm_count, s);
  return few_fmt_launch<__half>(fmt, a, sm_count, s);
}

}  // namespace b2g
