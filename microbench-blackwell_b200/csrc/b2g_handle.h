// b2g_handle.h -- the handle behind the C ABI and what its entry points share.  Not
// part of the public ABI.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

#include <new>

#include "b2g.h"

typedef CUresult (*PFN_encodeTiled_t)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                      const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                      const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                      CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// b2g_gemm_host splits M into at most kHostChunks row chunks and N into at most
// kHostColChunks column chunks
constexpr int kHostChunks = 4;
constexpr int kHostColChunks = 4;

// A device buffer of the handle that grows on demand (reserve()).
struct DeviceWs {
  void* p;
  size_t bytes;
  bool in_graph;  // a captured graph may hold its address
};

// A buffer that was replaced while a captured graph may still use it; freed with the handle.
struct RetiredWs {
  void* p;
  RetiredWs* next;
};

struct b2g_handle {
  int device;
  int sm_count;
  int clock_khz;
  int cc_major, cc_minor;
  uint32_t* d_err;
  PFN_encodeTiled_t encode_tiled;
  void* ws;                // device workspace of b2g_gemm_host
  size_t ws_bytes;
  DeviceWs meta_ws;        // scratch: engine-layout 2:4 metadata of the last sparse call
  DeviceWs sf_ws;          // scratch: engine-layout scale factors of the last call
  void* d_probe;           // b2g_probe_mma result words
  DeviceWs part_ws;        // split tail: fp32 partial tiles
  DeviceWs flag_ws;        // split tail: per-warp stamps (zeroed when allocated)
  uint32_t epoch;          // stamp of the last split-tail launch
  uint64_t wait_ns;        // limit of the kernel-side bounded waits (0: kWaitLimitNs)
  // b2g_gemm_host pipeline: copy-in and copy-out streams, events per row chunk
  cudaStream_t s_in, s_out;
  cudaEvent_t ev_start, ev_out, ev_c, ev_a[kHostChunks], ev_b[kHostColChunks];
  bool pipe_ready;
  uint32_t* trace_host;    // host-mapped progress trace (nullable)
  uint32_t* trace_dev;
  int trace_ctas;
  // co-resident cluster pairs per kernel instance and shared-memory size (the
  // occupancy query of cta_group::2 launches), kept after the first query
  struct OccEntry {
    uint32_t key;
    int smem, clusters;
  } occ[16];
  int n_occ;
  // operators around the linear layer (op_api.cu): fp32 partial sums and laid-out
  // operands of one call, and arrival counters that every launch leaves at zero
  DeviceWs op_ws, op_count;
  RetiredWs* retired;
  char last_error[512];
};

inline b2g_status fail(b2g_handle* h, b2g_status s, const char* fmt, ...) {
  if (h) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(h->last_error, sizeof(h->last_error), fmt, ap);
    va_end(ap);
  }
  return s;
}

#define B2G_CUDA(h, expr)                                                                  \
  do {                                                                                     \
    cudaError_t e__ = (expr);                                                              \
    if (e__ != cudaSuccess)                                                                \
      return fail((h), B2G_ERR_CUDA, "%s failed: %s", #expr, cudaGetErrorString(e__));     \
  } while (0)

// Make the handle's device current for the duration of a call.
struct DeviceGuard {
  int prev = -1;
  explicit DeviceGuard(int dev) {
    if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
    if (prev != dev) cudaSetDevice(dev);
  }
  ~DeviceGuard() {
    int cur;
    if (prev >= 0 && cudaGetDevice(&cur) == cudaSuccess && cur != prev) cudaSetDevice(prev);
  }
};

// Lets the calling thread allocate while a stream is being captured.
struct AllowInCapture {
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  AllowInCapture() { cudaThreadExchangeStreamCaptureMode(&mode); }
  ~AllowInCapture() { cudaThreadExchangeStreamCaptureMode(&mode); }
};

// Makes w hold `bytes` bytes for a call on stream s; new ones are zeros where `zeroed`.  A
// buffer that a captured graph may use is not freed before the handle: the graph is replayed
// with its address.  Within a capture a larger one is allocated and zeroed at once, beside the
// graph; outside, s is waited for, since earlier calls may still use the old one.
inline b2g_status reserve(b2g_handle* h, DeviceWs* w, size_t bytes, bool zeroed, cudaStream_t s) {
  if (bytes == 0) return B2G_OK;
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  B2G_CUDA(h, cudaStreamIsCapturing(s, &status));
  const bool capturing = status != cudaStreamCaptureStatusNone;
  if (w->bytes < bytes) {
    AllowInCapture allow;
    if (!capturing) B2G_CUDA(h, cudaStreamSynchronize(s));
    if (w->p && (capturing || w->in_graph)) {
      RetiredWs* old = new (std::nothrow) RetiredWs{w->p, h->retired};
      if (!old) return fail(h, B2G_ERR_CUDA, "out of host memory");
      h->retired = old;
    } else if (w->p) {
      cudaFree(w->p);
    }
    *w = DeviceWs{};
    void* p = nullptr;
    B2G_CUDA(h, cudaMalloc(&p, bytes));
    cudaError_t e = cudaSuccess;
    if (zeroed && capturing) {
      cudaStream_t beside;
      e = cudaStreamCreateWithFlags(&beside, cudaStreamNonBlocking);
      if (e == cudaSuccess) {
        e = cudaMemsetAsync(p, 0, bytes, beside);
        const cudaError_t done = cudaStreamSynchronize(beside);
        if (e == cudaSuccess) e = done;
        cudaStreamDestroy(beside);
      }
    } else if (zeroed) {
      // on the call's stream: nothing orders another one before its kernel
      e = cudaMemsetAsync(p, 0, bytes, s);
    }
    if (e != cudaSuccess) {
      cudaFree(p);
      return fail(h, B2G_ERR_CUDA, "zeroing a workspace failed: %s", cudaGetErrorString(e));
    }
    w->p = p;
    w->bytes = bytes;
  }
  w->in_graph |= capturing;
  return B2G_OK;
}
