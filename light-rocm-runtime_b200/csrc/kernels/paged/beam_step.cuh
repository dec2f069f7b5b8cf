// The bookkeeping of a beam search between its operators: what a step takes
// over from the fork of its pages, and what it leaves for the next one.
#ifndef LRRT_PAGED_BEAM_STEP_CUH_
#define LRRT_PAGED_BEAM_STEP_CUH_

#include "common.cuh"

namespace lrrt::ops {

// The forked table becomes the current one; each row's new token goes to the
// position after its last and is seen by the step's attention.
__device__ __forceinline__ void beam_begin(const BeamBeginArgs &args) {
  const uint32_t at = blockIdx.x * 256u + threadIdx.x;
  if (at < args.rows * args.columns) {
    args.table[at] = args.forked_table[at];
  }
  if (at < args.rows) {
    const int32_t length = args.forked_lengths[at];
    args.positions[at] = length;
    args.lengths[at] = length + 1;
  }
  if (at == 0 && args.status[0] > 0) {
    *args.missing_pages = static_cast<uint32_t>(args.status[0]);
  }
}

// The chosen tokens are the next inputs; tokens and parents are kept for the
// way back from the last step's beams.
__device__ __forceinline__ void beam_end(const BeamEndArgs &args) {
  const uint32_t step = *args.step;
  for (uint32_t row = threadIdx.x; row < args.rows; row += 256u) {
    const int32_t token = args.tokens[row];
    args.next_tokens[row] = token >= 0 ? static_cast<uint32_t>(token) : 0u;
    if (step < args.maximum_steps) {
      args.all_tokens[step * args.rows + row] = token;
      args.all_parents[step * args.rows + row] = args.parents[row];
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    *args.step = step + 1u;
  }
}

} // namespace lrrt::ops

#endif // LRRT_PAGED_BEAM_STEP_CUH_
