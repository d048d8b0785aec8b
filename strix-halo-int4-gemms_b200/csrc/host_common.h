// What the C entry points of every translation unit share: the thread's error message, the device of a call and
// the outermost layer of an entry point, through which no C++ exception passes.
#pragma once

#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>
#include <string>

namespace b200 {

// Sets the calling thread's message (b200_int4_gemms_last_error) and returns 1.
int host_fail(std::string msg);
int host_fail_cuda(const char* what, cudaError_t err);
void host_clear_error();

// Selects the device of a call for its duration; the caller's current device is restored at the end.
class DeviceScope {
 public:
  // 0 and the device's SM count, or 1 with a message (index out of range, no sm_100a device).
  int enter(int device_index, int* sm_count);
  ~DeviceScope();

 private:
  int previous_ = -1;
  bool changed_ = false;
};

template <typename Fn>
int guarded(Fn&& fn) noexcept {
  try {
    host_clear_error();
    return fn();
  } catch (...) {  // std::bad_alloc of a message at most
    return 1;
  }
}

// Allows a kernel its dynamic shared memory (with the static part it may pass the 48 KB that need no permission), once
// for each device: the attribute stays with the device's context.  Internal linkage: a static of an inline function would be
// one object for every copy of this library that a process loads, while each copy's kernels need the permission themselves.
template <auto Kernel>
static int allow_shared_memory(int smem_bytes) {
  static std::atomic<uint64_t> done{0};
  int device = 0;
  if (const cudaError_t err = cudaGetDevice(&device); err != cudaSuccess) return host_fail_cuda("cudaGetDevice", err);
  const uint64_t bit = uint64_t{1} << (device & 63);
  if (done.load(std::memory_order_acquire) & bit) return 0;
  const cudaError_t err = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes);
  if (err != cudaSuccess) return host_fail_cuda("cudaFuncSetAttribute(max dynamic shared memory)", err);
  done.fetch_or(bit, std::memory_order_release);
  return 0;
}

inline bool is_aligned(const void* p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

}  // namespace b200
