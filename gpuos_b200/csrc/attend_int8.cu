// gpuos_attend's kernels for a cache of int8 codes.
#include "attend.cuh"

template void gpuos::rowops::attend::launch<gpuos::rowops::attend::kInt8>(const Plan&, const Args&, cudaStream_t);
