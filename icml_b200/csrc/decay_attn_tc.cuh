// The tensor-core engine of the decay attention, as the entry points call it.
#pragma once
#include "decay_attn.cuh"
#include "tc_common.cuh"

namespace pgf {
namespace da {

constexpr int TC_CHUNK = 128;

// Whether a bf16 tensor can be read by the engine's TMA loads: 16-byte aligned base, pitches and width, at
// most 128 wide.
bool tc_fits(const Tensor& t, int64_t B, int64_t L);
// One F call, or only the pieces' own end states (into job.start).  job.seg_len: a multiple of TC_CHUNK.
int tc_walk(const Job& job, bool state_only, cudaStream_t s);

}  // namespace da
}  // namespace pgf
