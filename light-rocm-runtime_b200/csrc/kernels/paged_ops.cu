// Module of the paged-cache operators (paged_ops.cubin; include/lrrt_ops.h):
// the entry points of the kernels in paged/*.cuh, one per element type and
// shape. The host library (csrc/ops/ops.cpp) picks them by name.
#include "paged/attention.cuh"
#include "paged/beam_select.cuh"
#include "paged/beam_step.cuh"
#include "paged/pages.cuh"
#include "paged/rope_append.cuh"

using namespace lrrt::ops;

#define LRRT_ROPE(name, type, width, copy_width)                                                  \
  extern "C" __global__ void __launch_bounds__(kRopeThreads)                                      \
      ops_rope_half_##name(const __grid_constant__ RopeAppendArgs args) {                         \
    wait_for_previous_launch();                                                                   \
    rope_append<type, width, copy_width, false>(args);                                            \
  }                                                                                               \
  extern "C" __global__ void __launch_bounds__(kRopeThreads)                                      \
      ops_rope_pairs_##name(const __grid_constant__ RopeAppendArgs args) {                        \
    wait_for_previous_launch();                                                                   \
    rope_append<type, width, copy_width, true>(args);                                             \
  }

LRRT_ROPE(f32_x4, float, 4, 4)
LRRT_ROPE(f32_x1, float, 1, 1)
LRRT_ROPE(bf16_x8, __nv_bfloat16, 8, 8)
LRRT_ROPE(bf16_x4x8, __nv_bfloat16, 4, 8)
LRRT_ROPE(bf16_x4, __nv_bfloat16, 4, 4)
LRRT_ROPE(bf16_x1, __nv_bfloat16, 1, 1)
LRRT_ROPE(f16_x8, __half, 8, 8)
LRRT_ROPE(f16_x4x8, __half, 4, 8)
LRRT_ROPE(f16_x4, __half, 4, 4)
LRRT_ROPE(f16_x1, __half, 1, 1)

#define LRRT_ATTENTION(name, type, dim, head_tiles, team)                                         \
  extern "C" __global__ void                                                                      \
      __launch_bounds__(PagedAttention<type, dim, head_tiles, team>::kThreads, 1)                 \
      ops_attention_##name(const __grid_constant__ PagedAttentionArgs args) {                     \
    extern __shared__ __align__(128) unsigned char shared[];                                      \
    wait_for_previous_launch();                                                                   \
    PagedAttention<type, dim, head_tiles, team>(args, shared).run();                              \
  }

LRRT_ATTENTION(f32_64x8, float, 64, 1, 1)
LRRT_ATTENTION(f32_64x16, float, 64, 2, 1)
LRRT_ATTENTION(f32_96x8, float, 96, 1, 1)
LRRT_ATTENTION(f32_96x16, float, 96, 1, 2)
LRRT_ATTENTION(f32_128x8, float, 128, 1, 1)
LRRT_ATTENTION(f32_128x16, float, 128, 1, 2)
LRRT_ATTENTION(bf16_64x8, __nv_bfloat16, 64, 1, 1)
LRRT_ATTENTION(bf16_64x16, __nv_bfloat16, 64, 2, 1)
LRRT_ATTENTION(bf16_96x8, __nv_bfloat16, 96, 1, 1)
LRRT_ATTENTION(bf16_96x16, __nv_bfloat16, 96, 2, 1)
LRRT_ATTENTION(bf16_128x8, __nv_bfloat16, 128, 1, 1)
LRRT_ATTENTION(bf16_128x16, __nv_bfloat16, 128, 2, 1)
LRRT_ATTENTION(bf16_256x8, __nv_bfloat16, 256, 1, 1)
LRRT_ATTENTION(bf16_256x16, __nv_bfloat16, 256, 1, 2)
LRRT_ATTENTION(f16_64x8, __half, 64, 1, 1)
LRRT_ATTENTION(f16_64x16, __half, 64, 2, 1)
LRRT_ATTENTION(f16_96x8, __half, 96, 1, 1)
LRRT_ATTENTION(f16_96x16, __half, 96, 2, 1)
LRRT_ATTENTION(f16_128x8, __half, 128, 1, 1)
LRRT_ATTENTION(f16_128x16, __half, 128, 2, 1)
LRRT_ATTENTION(f16_256x8, __half, 256, 1, 1)
LRRT_ATTENTION(f16_256x16, __half, 256, 1, 2)

#define LRRT_PLAN(name, args_type)                                                                \
  extern "C" __global__ void __cluster_dims__(kPlanBlocks, 1, 1) __launch_bounds__(kPlanThreads)  \
      ops_##name(const __grid_constant__ args_type args) {                                        \
    wait_for_previous_launch();                                                                   \
    let_next_launch_begin();                                                                      \
    name<Plan<true>>(args);                                                                       \
  }                                                                                               \
  extern "C" __global__ void __launch_bounds__(kPlanThreadsAlone)                                 \
      ops_##name##_alone(const __grid_constant__ args_type args) {                                \
    wait_for_previous_launch();                                                                   \
    let_next_launch_begin();                                                                      \
    name<Plan<false>>(args);                                                                      \
  }

LRRT_PLAN(fork_plan, ForkArgs)
LRRT_PLAN(compact_plan, CompactArgs)

#define LRRT_MOVE(bytes, type)                                                                    \
  extern "C" __global__ void __launch_bounds__(kMoveThreads)                                      \
      ops_move_pages_##bytes(const __grid_constant__ MoveArgs args) {                             \
    wait_for_previous_launch();                                                                   \
    move_pages<type>(args);                                                                       \
  }

LRRT_MOVE(16, uint4)
LRRT_MOVE(4, uint32_t)

#define LRRT_BEAM(name, type)                                                                     \
  extern "C" __global__ void __launch_bounds__(kBeamThreads, kBeamBlocksPerSm)                    \
      ops_beam_##name(const __grid_constant__ BeamArgs args) {                                    \
    wait_for_previous_launch();                                                                   \
    beam_select<type>(args);                                                                      \
  }

LRRT_BEAM(f32, float)
LRRT_BEAM(bf16, __nv_bfloat16)
LRRT_BEAM(f16, __half)

extern "C" __global__ void __launch_bounds__(256)
    ops_beam_begin(const __grid_constant__ BeamBeginArgs args) {
  wait_for_previous_launch();
  beam_begin(args);
}

extern "C" __global__ void __launch_bounds__(256)
    ops_beam_end(const __grid_constant__ BeamEndArgs args) {
  wait_for_previous_launch();
  beam_end(args);
}

extern "C" __global__ void __launch_bounds__(256)
    ops_zero(const __grid_constant__ ZeroArgs args) {
  wait_for_previous_launch();
  for (uint64_t i = uint64_t{blockIdx.x} * 256u + threadIdx.x; i < args.count;
       i += uint64_t{gridDim.x} * 256u) {
    args.words[i] = 0;
  }
}
