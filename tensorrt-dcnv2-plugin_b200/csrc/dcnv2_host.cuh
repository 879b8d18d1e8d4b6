// dcnv2_host.cuh — host helpers shared by the entry points: per-device facts, the driver's
// tensor-map encoder and size arithmetic.
#pragma once
#include <atomic>
#include <cstddef>
#include <cstdint>
#include <mutex>

#include <cuda_runtime.h>
#include <cudaTypedefs.h>

namespace dcnv2 {

constexpr size_t kSmemLimit = 227 * 1024;     // opt-in dynamic shared memory per block
constexpr unsigned long long kDefaultTimeoutNs = 2000000000ull;  // 2 s per on-chip wait

struct DevInfo {
  int sm_count = 0;
  int major = 0;
  int minor = 0;
  bool ok = false;
  std::atomic<uint32_t> attr_set{0};
  std::atomic<int> pair_clusters[3] = {{0}, {0}, {0}};  // co-resident CTA pairs, per precision
};
constexpr int kMaxDevices = 64;
inline DevInfo g_dev[kMaxDevices];
inline std::once_flag g_dev_once[kMaxDevices];

inline DevInfo* device_info(int dev) {
  if (dev < 0 || dev >= kMaxDevices) return nullptr;
  std::call_once(g_dev_once[dev], [dev]() {
    DevInfo& d = g_dev[dev];
    if (cudaDeviceGetAttribute(&d.sm_count, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&d.major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&d.minor, cudaDevAttrComputeCapabilityMinor, dev) != cudaSuccess) {
      cudaGetLastError();
      d.ok = false;
      return;
    }
    d.ok = true;
  });
  return &g_dev[dev];
}

inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline size_t align_up(size_t v, size_t a) { return (v + a - 1) / a * a; }

// cuTensorMapEncodeTiled through the runtime's driver entry point (no libcuda link needed).
inline PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, []() {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault,
                                         &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
    cudaGetLastError();
  });
  return fn;
}

}  // namespace dcnv2
