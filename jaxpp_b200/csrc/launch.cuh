// What a launcher asks the runtime for again and again, kept per device: a call of a few microseconds of work should not spend
// one on questions.
#pragma once

#include <cuda_runtime.h>

#include <atomic>
#include <mutex>

namespace jpb {

constexpr int MAX_DEVICES = 64;

inline int current_device() {
  int dev = 0;
  cudaGetDevice(&dev);
  return dev >= 0 && dev < MAX_DEVICES ? dev : 0;
}
// The code of a launch, and no error left behind for the next question about one: the caller raises it.
inline int launch_result(cudaError_t e) {
  const cudaError_t last = cudaGetLastError();
  return int(e != cudaSuccess ? e : last);
}
inline int sm_count_of_device() {
  static std::atomic<int> sms[MAX_DEVICES];
  const int dev = current_device();
  int n = sms[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) return 148;
    sms[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}
// The largest dynamic shared memory that a kernel was allowed so far (one object per kernel).  Without asking, a CTA has 48 KB of
// both kinds together: 32 KB leave room for any kernel's static part.
// Asked for under a lock, and only ever raised: a second thread must not set a smaller limit between the first one's question and
// its launch.
struct SmemLimit {
  std::atomic<int> bytes[MAX_DEVICES];
  std::mutex lock;
  template <typename Kernel>
  int allow(Kernel kernel, int want) {
    const int dev = current_device();
    if (want <= 32 * 1024 || want <= bytes[dev].load(std::memory_order_acquire)) return 0;
    std::lock_guard<std::mutex> held(lock);
    if (want <= bytes[dev].load(std::memory_order_relaxed)) return 0;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, want);
    if (e != cudaSuccess) return launch_result(e);
    bytes[dev].store(want, std::memory_order_release);
    return 0;
  }
};

}  // namespace jpb
