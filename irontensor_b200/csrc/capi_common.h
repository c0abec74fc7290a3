// What the translation units of the C ABI share: the context and stream objects, error texts, launches.
#pragma once
#include "../../include/irontensor_b200.h"

#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>
#include <memory>
#include <mutex>
#include <utility>
#include <vector>

// Records the calling thread's error text (it_last_error) and returns `code`.
__attribute__((visibility("hidden"), format(printf, 2, 3))) it_status fail(it_status code, const char* fmt, ...);

#define IT_CUDA(expr)                                                                              \
  do {                                                                                             \
    cudaError_t e_ = (expr);                                                                       \
    if (e_ != cudaSuccess) return fail(IT_ERR_CUDA, "%s: %s", #expr, cudaGetErrorString(e_));      \
  } while (0)

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// The counters of captured launches.  A graph gives its launches' back when it and the executable graphs made from it are
// gone, possibly after the context and from a thread of the driver's: hence shared ownership.
struct CaptureSlots {
  struct Held {   // what a graph holds
    std::shared_ptr<CaptureSlots> slots;
    int i = 0;
    Held* next = nullptr;
  };
  std::mutex mutex;
  int next = 0;
  Held *oldest = nullptr, *newest = nullptr;   // given back: reused oldest first, and only once every one has been out
  ~CaptureSlots() {
    while (oldest != nullptr) {
      Held* h = oldest;
      oldest = h->next;
      delete h;
    }
  }
};
struct it_ctx {
  int device = 0;
  int sm_count = 0;
  int* d_status = nullptr;      // two device status words: of kernels whose waits run out, and of lengths outside a quantised cache
  int* h_status = nullptr;      // pinned mirror
  int* range_status() const { return d_status + 1; }   // kernels do not stop for this one
  cudaStream_t status_stream = nullptr;   // reads the status word without touching a caller's stream
  std::mutex status_mutex;      // h_status and status_stream are shared by every thread using the context
  EncodeTiledFn encode = nullptr;
  int timing = 0;               // events around: 1 the backward main kernel; 2 the forward kernel too; 3 the backward's prepare and finish passes too
  // [forward | backward main | backward prepare | backward finish][start | stop]; the prepare pass starts where the
  // previous timer stopped only in time, not in events: three pairs share the boundaries prepare|main|finish
  cudaEvent_t ev[4][2] = {};
  bool ev_valid[4] = {false, false, false, false};
  std::atomic<uint64_t> launches{0};
  // Work-item counters of the forward kernel that walks its items in a loop: a pair of ints per live stream object (launches
  // on one stream run one after the other, so a stream needs one pair), handed out from a pool allocated with the
  // context so that wrapping a stream calls nothing a stream capture forbids; and behind those one per captured launch.
  // Zeroed once, here; every launch leaves its pair at zero, also one that gave up.
  static constexpr int WORK_SLOTS = 4096, CAPTURE_SLOTS = 61440;
  static constexpr size_t WORK_BYTES = 2 * sizeof(int) * (WORK_SLOTS + CAPTURE_SLOTS);
  std::shared_ptr<CaptureSlots> captured;
  int* d_work_pool = nullptr;
  std::mutex work_mutex;
  std::vector<int> work_free;
  int work_next = 0;
};
struct it_stream {
  cudaStream_t s = nullptr;
  bool owned = false;
  int* d_work = nullptr;     // this stream's work-item counter; null when the pool ran out (the launcher then starts one CTA per item)
  bool work_used = false;    // a launch has drawn from the counter
};

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Launch with the programmatic-stream-serialization attribute: the kernel may be set up while the kernel in front of it
// in the stream still runs, and waits in griddepcontrol.wait for that kernel's completion before it touches its results.
// launch_cluster: in clusters of `cluster` CTAs along x (1: no clusters).
template <typename... KArgs, typename... Args>
cudaError_t launch_cluster(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t s, int cluster, Args&&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(std::forward<Args>(args))...);
}
template <typename... KArgs, typename... Args>
cudaError_t launch_dependent(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t s, Args&&... args) {
  return launch_cluster(kernel, grid, block, smem, s, 1, std::forward<Args>(args)...);
}
