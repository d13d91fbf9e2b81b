// Several launches of one call that overlap one another.
#pragma once
#include "common.cuh"

namespace pgf {

// The launches of one call.  The first waits for what is in front of it in the stream, as any launch.  A later one
// (chained) may start as soon as all CTAs of the one before have begun, so that it fills the SMs which that one's
// last wave leaves idle (programmatic dependent launch).  What it must not read too early it waits for (wait: the
// launch before has ended); and one CTA of each waits for it at its own end, so that the end of the last launch
// is the end of all.  16 x 2048 tokens x 16 heads of 64: a backward's 256-CTA launches, each 1.7 waves, take 341 us
// so and 363 one after the other.  What a launch reads that one further in front has written it reads past the L1 cache.
struct Link {
  int chained, wait;
};
struct Chain {
  int n = 0, wait = 0;     // wait: the next launch reads what the one before writes
  Link next() {
    const Link l = {n++ > 0, wait};
    wait = 0;
    return l;
  }
};
__device__ __forceinline__ void chain_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void chain_begin(const Link& l) {
  if (l.wait) chain_wait();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void chain_end() {
  if (blockIdx.x == gridDim.x - 1 && threadIdx.x == 0) chain_wait();
}
template <class... P, class... A>
cudaError_t launch_link(const Link& l, void (*kernel)(P...), dim3 grid, unsigned threads, size_t smem, cudaStream_t s,
                        const A&... args) {
  cudaLaunchAttribute at = {};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = &at;
  cfg.numAttrs = l.chained ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace pgf
