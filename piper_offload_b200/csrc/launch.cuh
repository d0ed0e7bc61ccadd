// launch.cuh - launches that may begin while the launch before them ends (programmatic stream serialization).
//
// A kernel launched so calls grid_launch_dependents(), which lets the next such launch set itself up, and grid_wait(), which
// ends when all launches before it have ended and their writes are visible. Memory that a launch of another call may have
// written is read after the wait. Before it, an INT8 product loads its weight and reads the ends of its groups, and a
// gradient those: they may, because the launch before each is the same call's (quantize_kernel, scale_kernel), which waits
// first and lets them begin after. A kernel that allocates tensor memory lets the next begin when it has it: the next may
// allocate before its own wait (the product of a few tokens does, 32 columns), and on an SM with a block that is still to
// have all 512 each would wait for the other. Registers and shared memory keep the two apart as they are now, no rule does.
// In a program's stream such launches take the start of a launch, 1.5 to 2.5 us, out of the time between two of them: 1 x
// 14336 x 4096 16.0 -> 13.3 us a call.
#pragma once
#include <cuda_runtime.h>

namespace piper {

template <class... Params, class... Args>
cudaError_t launch(void (*kernel)(Params...), int64_t blocks, int threads, size_t smem, int cluster, cudaStream_t stream, const Args&... args) {
  cudaLaunchAttribute attributes[2] = {};
  attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attributes[0].val.programmaticStreamSerializationAllowed = 1;
  attributes[1].id = cudaLaunchAttributeClusterDimension;
  attributes[1].val.clusterDim.x = static_cast<unsigned>(cluster);
  attributes[1].val.clusterDim.y = attributes[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(static_cast<unsigned>(blocks));
  config.blockDim = dim3(static_cast<unsigned>(threads));
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  config.attrs = attributes;
  config.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&config, kernel, args...);
}

}  // namespace piper
