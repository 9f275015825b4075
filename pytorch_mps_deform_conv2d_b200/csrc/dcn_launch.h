// dcn_launch.h -- host-side launch helpers shared by the kernel files.
#pragma once

#include <cuda_runtime.h>

namespace dcn {

// cudaFuncSetAttribute(MaxDynamicSharedMemorySize) once per (kernel, device)
// and size: later calls with the same or a smaller size return at once.
cudaError_t ensure_dynamic_smem(const void* func, int bytes);

// Multiprocessor count of the current device (queried once per device).
int device_sm_count();

// Clusters of `size` (2, 4 or 8) CTAs that the current device holds at a time,
// one CTA an SM: how many SMs a group of them has left differs from chip to
// chip.  Asked for once per device and size, through `func` (whose dynamic
// shared memory has been allowed); half of what the SMs would hold if the
// question fails.
int device_cluster_slots(const void* func, int threads, int smem, int size);

}  // namespace dcn
