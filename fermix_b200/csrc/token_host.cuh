// Launches of the operators on tokens.
#pragma once
#include "block_host.cuh"
#include "token_common.cuh"

namespace fxh {

// A launch that follows another of the same call and waits for it in the kernel (wait_for_last): its blocks come up while
// the last writes of the one before are still on their way to memory, without a gap between the two (65600 tokens over a
// table of 50001 x 1000 bf16, trained, 9 launches: 142 -> 127 us). No kernel lets the next one come earlier
// (griddepcontrol.launch_dependents): its blocks then fill the multiprocessors unevenly while the last wave of the one
// before still runs (4096 x 128 tokens over 512 x 128 f32, trained: 149 us with plain launches, 151 with the early start,
// 140 so).
template <typename... P, typename... A>
int launch_next(void (*kern)(P...), dim3 grid, unsigned threads, size_t smem, cudaStream_t s, const A&... args) {
  cudaLaunchAttribute overlap{};
  overlap.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  overlap.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t c{};
  c.gridDim = grid;
  c.blockDim = dim3(threads);
  c.dynamicSmemBytes = smem;
  c.stream = s;
  c.attrs = &overlap;
  c.numAttrs = 1;
  return cudaLaunchKernelEx(&c, kern, static_cast<P>(args)...) == cudaSuccess ? FX_OK : FX_ERR_CUDA;
}

}  // namespace fxh
