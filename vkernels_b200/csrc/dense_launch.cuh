// dense_launch.cuh - how the kernels of the dense feed-forward operators follow one another on a stream.
#pragma once

#include "common.cuh"

namespace vkernels::kernels::cuda {

namespace {

// A kernel of these may be scheduled while the kernels before it on its stream still run (programmatic launch): its barriers
// and tensor memory are set up meanwhile. Nothing in memory is touched before this, which returns once all of them are done
// and their writes visible.
__device__ __forceinline__ void wait_for_earlier_kernels() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
void overlap_launch(cudaLaunchAttribute& a) {
  a.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  a.val.programmaticStreamSerializationAllowed = 1;
}

}  // namespace

}  // namespace vkernels::kernels::cuda
