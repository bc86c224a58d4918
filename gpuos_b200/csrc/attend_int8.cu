// gpuos_attend's kernels for a cache of int8 codes.
#include "attend.cuh"
#include "attend_wide.cuh"

template void gpuos::rowops::attend::launch<gpuos::rowops::attend::kInt8>(const Plan&, const Args&, cudaStream_t);
template void gpuos::rowops::attend::launch_wide<gpuos::rowops::attend::kInt8>(const Args&, cudaStream_t);
