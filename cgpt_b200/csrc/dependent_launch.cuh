// Programmatic dependent launch of the later kernels of one operator: the launch is prepared, and its CTAs placed where there is
// room, while the kernel before it in the stream still runs. The first kernel calls launch_dependents() as soon as it starts, the
// later one wait_for_previous() before it touches anything the first one writes or reads: it returns when that kernel has
// finished and its writes are visible. To ordinary loads: a parameter that points to what the first kernel writes must not be
// `const __restrict__`, which allows loads that count on memory that stays as it is from the launch on. Kernels of other operators
// are launched normally, after all of this.
#pragma once

#include <utility>

#include "common.cuh"

namespace cgpt {

__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <typename... P, typename... A>
cudaError_t launch_after_previous(void (*kernel)(P...), dim3 grid, unsigned threads, std::size_t smem, cudaStream_t s, A&&... args) {
    cudaLaunchConfig_t config = {};
    config.gridDim = grid;
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = smem;
    config.stream = s;
    cudaLaunchAttribute attribute;
    attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &attribute;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, kernel, static_cast<P>(std::forward<A>(args))...);
}

}  // namespace cgpt
