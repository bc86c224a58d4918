// gpuos_attend's kernels for a cache of e4m3 codes.
#include "attend.cuh"
#include "attend_wide.cuh"

template void gpuos::rowops::attend::launch<gpuos::rowops::attend::kE4M3>(const Plan&, const Args&, cudaStream_t);
template void gpuos::rowops::attend::launch_wide<gpuos::rowops::attend::kE4M3>(const Args&, cudaStream_t);
