// What the host sides of the library share: the text of the last CUDA error, and launches that may
// begin while the kernel before them in the stream still runs.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace leat {

// true, with the text kept for leat_sampler_last_cuda_error(), if `e` is an error
int cuda_failed(cudaError_t e, const char* what);

// A launch that may begin while the kernel before it in the stream still runs (programmatic
// dependent launch); the kernel itself waits, with grid_dependency_wait(), before it reads what
// that kernel writes.  cluster: blocks per cluster along x, 0 for none.
template <typename... Params, typename... Args>
cudaError_t launch_dependent_cluster(int cluster, void (*kernel)(Params...), dim3 grid, dim3 block, size_t shared,
                                     cudaStream_t stream, const Args&... args) {
  cudaLaunchConfig_t config = {};
  config.gridDim = grid;
  config.blockDim = block;
  config.dynamicSmemBytes = shared;
  config.stream = stream;
  cudaLaunchAttribute attribute[2];
  attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute[0].val.programmaticStreamSerializationAllowed = 1;
  attribute[1].id = cudaLaunchAttributeClusterDimension;
  attribute[1].val.clusterDim.x = cluster > 0 ? cluster : 1;
  attribute[1].val.clusterDim.y = 1;
  attribute[1].val.clusterDim.z = 1;
  config.attrs = attribute;
  config.numAttrs = cluster > 0 ? 2 : 1;
  return cudaLaunchKernelEx(&config, kernel, args...);
}

template <typename... Params, typename... Args>
cudaError_t launch_dependent(void (*kernel)(Params...), dim3 grid, dim3 block, size_t shared, cudaStream_t stream,
                             const Args&... args) {
  return launch_dependent_cluster(0, kernel, grid, block, shared, stream, args...);
}

inline bool aligned(const void* p, size_t a) { return ((uintptr_t)p % a) == 0; }

}  // namespace leat
