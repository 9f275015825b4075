// dcn_launch.cu -- host-side launch helpers (see dcn_launch.h).
#include "dcn_launch.h"

#include <atomic>
#include <map>
#include <mutex>
#include <utility>

namespace dcn {

namespace {
std::mutex g_attr_mu;
std::map<std::pair<const void*, int>, int> g_smem_set;  // (kernel, device) -> bytes
constexpr int kMaxDevices = 64;
std::atomic<int> g_sms[kMaxDevices] = {};
std::atomic<int> g_cluster_slots[kMaxDevices][3] = {};
}  // namespace

cudaError_t ensure_dynamic_smem(const void* func, int bytes) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  std::lock_guard<std::mutex> lk(g_attr_mu);
  int& cur = g_smem_set[{func, dev}];
  if (bytes <= cur) return cudaSuccess;
  e = cudaFuncSetAttribute(func, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) cur = bytes;
  return e;
}

int device_sm_count() {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0) return 148;
  if (dev < kMaxDevices) {
    const int known = g_sms[dev].load(std::memory_order_relaxed);
    if (known > 0) return known;
  }
  int sms = 0;
  if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0)
    sms = 148;
  if (dev < kMaxDevices) g_sms[dev].store(sms, std::memory_order_relaxed);
  return sms;
}

int device_cluster_slots(const void* func, int threads, int smem, int size) {
  const int log = size >= 8 ? 2 : size >= 4 ? 1 : 0;
  int dev = 0;
  const bool known_device = cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < kMaxDevices;
  if (known_device) {
    const int known = g_cluster_slots[dev][log].load(std::memory_order_relaxed);
    if (known > 0) return known;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)size);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)size;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int slots = 0;
  if (cudaOccupancyMaxActiveClusters(&slots, func, &cfg) != cudaSuccess || slots <= 0) {
    (void)cudaGetLastError();
    return device_sm_count() / (2 * size);
  }
  if (known_device) g_cluster_slots[dev][log].store(slots, std::memory_order_relaxed);
  return slots;
}

}  // namespace dcn
