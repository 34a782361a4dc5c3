// A launch that may start while its predecessor in the stream still runs (device/pdl.cuh), in clusters of `cluster` CTAs.
#pragma once
#include <cuda_runtime.h>

namespace smr {

template <class... Params, class... Args>
int launch_pdl(void (*kernel)(Params...), dim3 grid, int threads, size_t smem, int cluster, cudaStream_t stream,
               const Args&... args) {
  if (smem > 0)
    if (int e = (int)cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem)) return e;
  cudaLaunchAttribute attrs[2] = {};
  attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[0].val.programmaticStreamSerializationAllowed = 1;
  attrs[1].id = cudaLaunchAttributeClusterDimension;
  attrs[1].val.clusterDim.x = cluster;
  attrs[1].val.clusterDim.y = attrs[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attrs;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return (int)cudaLaunchKernelEx(&cfg, kernel, Params(args)...);
}

}  // namespace smr
