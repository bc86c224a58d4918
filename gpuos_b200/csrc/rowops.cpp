// The current device of this library's own CUDA runtime (it is linked
// statically, so torch's current device is not its own), for callers that take
// the device from a tensor.  Not part of the C ABI.
#include <cuda_runtime.h>

#include <cstdint>

// Makes `device` current; returns the device to go back to, or -1 where it was
// current already (or cannot be made so: the launch reports that).
extern "C" int32_t gpuos_rowops_enter(int32_t device) {
  int before = -1;
  if (cudaGetDevice(&before) != cudaSuccess || before == device) return -1;
  return cudaSetDevice(device) == cudaSuccess ? before : -1;
}

extern "C" void gpuos_rowops_leave(int32_t before) {
  if (before >= 0) cudaSetDevice(before);
}
