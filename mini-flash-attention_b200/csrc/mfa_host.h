// Host-side services shared by the translation units of libmfa_b200.so (those that are not here are
// defined in mfa_capi.cu): errors, the per-device set-up, pointer checks, launches and tensor maps.
// Every function that returns int returns an MFA_* code and leaves its message for
// mfa_last_error_string().
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>
#include <mutex>
#include <string>

#include "../../include/mfa_b200.h"

namespace mfa {
namespace host {

int fail(int code, const std::string& msg);
int fail_cuda(cudaError_t e, const char* what);

constexpr int kMaxDevices = 64;

// A device's one-time set-up: `run` is called, by one thread at a time, until it has returned
// MFA_OK. A failure is the calling entry's own, the next one tries again. The process's first
// call may be one that is captured: nothing in a set-up belongs to the stream, so for its time the
// thread may make the calls that a capture forbids by default (kernel attributes, symbol
// addresses, a memory pool).
class SetUp {
 public:
  template <class F>
  int operator()(F&& run) {
    if (done_.load(std::memory_order_acquire)) return MFA_OK;
    const std::lock_guard<std::mutex> lock(mu_);
    if (done_.load(std::memory_order_relaxed)) return MFA_OK;
    const Relaxed relaxed;
    const int rc = run();
    if (rc == MFA_OK) done_.store(true, std::memory_order_release);
    return rc;
  }

 private:
  // The thread's capture mode, relaxed while this lives.
  struct Relaxed {
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    const bool changed = cudaThreadExchangeStreamCaptureMode(&mode) == cudaSuccess;
    ~Relaxed() {
      if (changed) cudaThreadExchangeStreamCaptureMode(&mode);
    }
  };
  std::mutex mu_;
  std::atomic<bool> done_{false};
};

// The current device after its one-time set-up.
struct Device {
  int index;
  int sms;
  int* status;             // device status word
  cudaMemPool_t pool;      // the library's stream-ordered pool
  unsigned long long timeout_ns;
};
int open_device(Device* out);

// `p` must be memory that device `dev` addresses directly.
int check_pointer(const void* p, const char* name, int dev);

// Null and misaligned pointers; with a device (dev >= 0), also those that are not its memory.
struct Pointer {
  const void* p;
  const char* name;
  uintptr_t align;
};
inline int check_pointers(const Pointer* ptrs, int count, int dev) {
  for (int i = 0; i < count; ++i) {
    const Pointer& x = ptrs[i];
    if (!x.p) return fail(MFA_ERR_INVALID_ARGUMENT, std::string("null ") + x.name);
    if (reinterpret_cast<uintptr_t>(x.p) & (x.align - 1))
      return fail(MFA_ERR_INVALID_ARGUMENT, std::string(x.name) + " must be " +
                                                std::to_string(x.align) + "-byte aligned");
    const int rc = dev < 0 ? MFA_OK : check_pointer(x.p, x.name, dev);
    if (rc != MFA_OK) return rc;
  }
  return MFA_OK;
}

// Launches a kernel that waits for the stream's earlier work itself (griddepcontrol.wait) and may be
// set up while that work ends; in clusters of `cluster` CTAs.
struct Grid {
  int64_t ctas;
  int threads, smem;
  cudaStream_t stream;
  int cluster = 1;
};
template <class... Params, class... Args>
cudaError_t launch(const Grid& g, void (*kernel)(Params...), const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(g.ctas));
  cfg.blockDim = dim3(static_cast<unsigned>(g.threads));
  cfg.dynamicSmemBytes = static_cast<size_t>(g.smem);
  cfg.stream = g.stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(g.cluster);
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = g.cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// Element strides of a contiguous tensor in `layout`.
struct Strides {
  int64_t n, h, b;
};
Strides strides_of(int layout, int64_t heads, int64_t n, int64_t d);

// 4-D map {D, N, H, B} of a tensor, box of 128 rows and min(D, 64) columns.
int encode_heads(CUtensorMap* map, const void* base, int64_t batch, int64_t heads, int64_t n,
                 int64_t d, const Strides& strides, bool bf16);

// A map of 16-bit elements with 64-column boxes in the 128-byte swizzle; rank - 1 strides.
int encode_map(CUtensorMap* map, const void* base, int rank, const uint64_t* dims,
               const uint64_t* stride_bytes, const uint32_t* box, bool bf16);

}  // namespace host
}  // namespace mfa
