// Launches that overlap the end of the kernel before them (programmatic dependent launch).
#pragma once

#include <cuda_runtime.h>

namespace fgs {

// Lets the kernel's programmatic dependent start (once every CTA has called it or ended), and waits for the kernel that
// this one depends on, whose writes are visible behind it. Both do nothing in a kernel that was launched in the ordinary way.
__device__ inline void allow_dependent() { asm volatile("griddepcontrol.launch_dependents;"); }
__device__ inline void wait_dependency() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// What a dependent kernel reads of its predecessor's writes is not const and __restrict__: that promises that nobody writes it
// while the kernel runs, and the read could be moved in front of the wait.

// Launches a kernel as the programmatic dependent of the one before it in the stream: it may start before that one has
// ended, and has to call wait_dependency() before it touches what that one, or any kernel before it, reads or writes.
template <typename... Params, typename... Args>
cudaError_t launch_dependent(void (*kernel)(Params...), dim3 grid, int threads, size_t smem, cudaStream_t s, Args&&... args) {
    cudaLaunchConfig_t config{};
    config.gridDim = grid;
    config.blockDim = dim3(static_cast<unsigned>(threads));
    config.dynamicSmemBytes = smem;
    config.stream = s;
    cudaLaunchAttribute attribute{};
    attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &attribute;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, kernel, static_cast<Params>(args)...);
}

}  // namespace fgs
