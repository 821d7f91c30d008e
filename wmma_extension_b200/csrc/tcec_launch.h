// Launches of kernels that may be set up while the kernel before them ends.
#pragma once
#include <cuda_runtime.h>

namespace tcec_host {

// Launches `kernel`, which waits for the kernel before it on the stream by itself (wait_for_launch_before), so that it may be set up
// while that one ends.
// cluster > 0: in clusters of so many CTAs.
template <class... Params, class... Args>
void launch_clusters(void (*kernel)(Params...), int cluster, dim3 grid, int threads, size_t smem, cudaStream_t stream,
                     const Args&... args) {
  cudaLaunchAttribute attrs[2] = {};
  attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[0].val.programmaticStreamSerializationAllowed = 1;
  attrs[1].id = cudaLaunchAttributeClusterDimension;
  attrs[1].val.clusterDim.x = cluster;
  attrs[1].val.clusterDim.y = attrs[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = grid;
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  config.attrs = attrs;
  config.numAttrs = cluster > 0 ? 2 : 1;
  cudaLaunchKernelEx(&config, kernel, Params(args)...);
}
template <class... Params, class... Args>
void launch_early(void (*kernel)(Params...), dim3 grid, int threads, size_t smem, cudaStream_t stream, const Args&... args) {
  launch_clusters(kernel, 0, grid, threads, smem, stream, args...);
}
// Launches a kernel that is not set up before the one in front of it has ended.
template <class... Params, class... Args>
void launch_late(void (*kernel)(Params...), dim3 grid, int threads, size_t smem, cudaStream_t stream, const Args&... args) {
  kernel<<<grid, threads, smem, stream>>>(Params(args)...);
}

}  // namespace tcec_host
