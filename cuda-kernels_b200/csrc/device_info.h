// What the library's other translation units need of a device's one-time
// set-up (b200_gemm.cu keeps it): one status word and one wait limit for all
// kernels of the library.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>
#include <cstdint>

namespace b200 {
struct DeviceInfo {
  int sm_count;
  uint32_t* status;     // device status word (DeviceStatus bits)
  uint64_t timeout_ns;  // limit of every device-side wait
  PFN_cuTensorMapEncodeTiled_v12000 encode;
};
// The current device's set-up, made on first use; a B200_* status code.
int device_info(DeviceInfo* out);
}  // namespace b200
