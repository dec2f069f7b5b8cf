// The best continuations over the beams of a group and the vocabulary.
//
// One pass over the logits: a block reads a chunk of a row into registers,
// takes the chunk's maximum m and sum of exp(x - m), and its `count` best
// elements; the last block of a row joins the chunks (sums by
// l1 e^(m1 - m) + l2 e^(m2 - m)), the last row of a group ranks the beams'
// candidates by score + logit - log sum. Bound by reading the logits once.
//
// Elements are compared as 64-bit keys, the value's order in the upper half
// and the complement of the index in the lower, so that no two are equal and
// the order of threads and blocks decides nothing.
#ifndef LRRT_PAGED_BEAM_SELECT_CUH_
#define LRRT_PAGED_BEAM_SELECT_CUH_

#include "common.cuh"

namespace lrrt::ops {

constexpr uint32_t kBeamWarps = kBeamThreads / 32u;
// Candidates that are ranked against one another at once.
constexpr uint32_t kBeamPool = 1024;

struct BeamShared {
  uint64_t pool[kBeamPool];
  uint64_t best[kBeamMaximumCount];
  uint64_t warp_keys[kBeamWarps];
  float warp_values[kBeamWarps];
  uint32_t pooled;
  uint32_t last;
};

// Order of floats as unsigned numbers; NaN like -infinity.
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t bits = __float_as_uint(x != x ? -INFINITY : x);
  // -0 and +0 are equal values: both become +0.
  const uint32_t plain = bits == 0x80000000u ? 0u : bits;
  return (plain >> 31) != 0 ? ~plain : plain | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t order) {
  return __uint_as_float((order >> 31) != 0 ? order & 0x7fffffffu : ~order);
}
__device__ __forceinline__ uint64_t key_of(float x, uint32_t index) {
  return uint64_t{order_of(x)} << 32 | ~index;
}
constexpr uint64_t kNoKey = 0; // below every key

__device__ __forceinline__ uint64_t larger(uint64_t a, uint64_t b) { return a > b ? a : b; }

// The `count` largest of the block's keys (Each per thread, in registers),
// in shared.best, falling; kNoKey where there are fewer.
//
// The block's threads are split into `count` rounded up to a power of two
// groups; the smallest of the groups' maxima is no larger than the count-th
// largest key, so only keys from there on are candidates: about
// count * (1 + 1/2 + ... + 1/count) of them when the order is random. They are
// ranked by counting the larger ones. Where more than kBeamPool pass, the best
// are taken one after another instead.
template <int Each>
__device__ __forceinline__ void block_best(const uint64_t (&keys)[Each], uint32_t count,
                                           BeamShared &shared) {
  const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5u;
  uint64_t mine = kNoKey;
#pragma unroll
  for (int i = 0; i < Each; ++i) {
    mine = larger(mine, keys[i]);
  }
  // Groups within a warp: 32 / (groups per warp) lanes each; with no more
  // groups than warps, whole warps.
  uint32_t groups = 1;
  while (groups < count) {
    groups <<= 1u;
  }
  const uint32_t lanes = groups <= kBeamWarps ? 32u : 32u * kBeamWarps / groups;
  uint64_t group_best = mine;
#pragma unroll
  for (uint32_t offset = 1; offset < 32u; offset <<= 1u) {
    const uint64_t other = __shfl_xor_sync(kAllLanes, group_best, offset);
    if (offset < lanes) {
      group_best = larger(group_best, other);
    }
  }
  uint64_t floor = group_best; // the smallest of the warp's groups
#pragma unroll
  for (uint32_t offset = 1; offset < 32u; offset <<= 1u) {
    const uint64_t other = __shfl_xor_sync(kAllLanes, floor, offset);
    floor = floor < other ? floor : other;
  }
  __syncthreads(); // shared is free
  if (lane == 0) {
    shared.warp_keys[warp] = floor;
  }
  if (threadIdx.x == 0) {
    shared.pooled = 0;
  }
  __syncthreads();
  floor = shared.warp_keys[0];
#pragma unroll
  for (uint32_t w = 1; w < kBeamWarps; ++w) {
    floor = floor < shared.warp_keys[w] ? floor : shared.warp_keys[w];
  }
  if (mine >= floor) {
#pragma unroll
    for (int i = 0; i < Each; ++i) {
      if (keys[i] >= floor && keys[i] != kNoKey) {
        const uint32_t at = atomicAdd(&shared.pooled, 1u);
        if (at < kBeamPool) {
          shared.pool[at] = keys[i];
        }
      }
    }
  }
  if (threadIdx.x < count) {
    shared.best[threadIdx.x] = kNoKey;
  }
  __syncthreads();
  const uint32_t pooled = shared.pooled;
  if (pooled <= kBeamPool) {
    for (uint32_t i = threadIdx.x; i < pooled; i += kBeamThreads) {
      const uint64_t key = shared.pool[i];
      uint32_t rank = 0;
      for (uint32_t j = 0; j < pooled; ++j) {
        rank += shared.pool[j] > key ? 1u : 0u;
      }
      if (rank < count) {
        shared.best[rank] = key;
      }
    }
    __syncthreads();
    return;
  }
  uint64_t bound = ~uint64_t{0};
  for (uint32_t rank = 0; rank < count; ++rank) {
    uint64_t best = kNoKey;
#pragma unroll
    for (int i = 0; i < Each; ++i) {
      best = keys[i] < bound ? larger(best, keys[i]) : best;
    }
#pragma unroll
    for (uint32_t offset = 16; offset != 0; offset >>= 1u) {
      best = larger(best, __shfl_xor_sync(kAllLanes, best, offset));
    }
    if (lane == 0) {
      shared.warp_keys[warp] = best;
    }
    __syncthreads();
    best = shared.warp_keys[0];
#pragma unroll
    for (uint32_t w = 1; w < kBeamWarps; ++w) {
      best = larger(best, shared.warp_keys[w]);
    }
    if (threadIdx.x == 0) {
      shared.best[rank] = best;
    }
    bound = best;
    __syncthreads();
  }
}

// As block_best, over `total` keys in global memory, 2048 at a time with the
// best so far among them.
__device__ __forceinline__ void block_best_of(const uint64_t *keys, uint32_t total, uint32_t count,
                                              BeamShared &shared) {
  constexpr int kEach = 8;
  constexpr uint32_t kRound = kBeamThreads * kEach;
  uint32_t done = 0;
  while (true) {
    uint64_t held[kEach];
    const uint32_t kept = done == 0 ? 0u : count;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const uint32_t at = i * kBeamThreads + threadIdx.x;
      if (at < kept) {
        held[i] = shared.best[at];
      } else {
        const uint64_t from = uint64_t{done} + at - kept;
        held[i] = from < total ? __ldcg(keys + from) : kNoKey;
      }
    }
    block_best(held, count, shared);
    done += kRound - kept;
    if (done >= total) {
      return;
    }
  }
}

__device__ __forceinline__ float block_max(float x, BeamShared &shared) {
  const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5u;
#pragma unroll
  for (uint32_t offset = 16; offset != 0; offset >>= 1u) {
    x = fmaxf(x, __shfl_xor_sync(kAllLanes, x, offset));
  }
  __syncthreads();
  if (lane == 0) {
    shared.warp_values[warp] = x;
  }
  __syncthreads();
  x = shared.warp_values[0];
#pragma unroll
  for (uint32_t w = 1; w < kBeamWarps; ++w) {
    x = fmaxf(x, shared.warp_values[w]);
  }
  return x;
}

__device__ __forceinline__ float block_sum(float x, BeamShared &shared) {
  const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5u;
#pragma unroll
  for (uint32_t offset = 16; offset != 0; offset >>= 1u) {
    x += __shfl_xor_sync(kAllLanes, x, offset);
  }
  __syncthreads();
  if (lane == 0) {
    shared.warp_values[warp] = x;
  }
  __syncthreads();
  x = shared.warp_values[0];
#pragma unroll
  for (uint32_t w = 1; w < kBeamWarps; ++w) {
    x += shared.warp_values[w];
  }
  return x;
}

// Whether this block is the last of `blocks` to get here; its reads then see
// what the others wrote before. The counter is zero again afterwards.
__device__ __forceinline__ bool arrive_last(uint32_t *counter, uint32_t blocks,
                                            BeamShared &shared) {
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) {
    const uint32_t before = atomicAdd(counter, 1u);
    shared.last = before + 1u == blocks ? 1u : 0u;
    if (shared.last != 0) {
      *counter = 0;
    }
  }
  __syncthreads();
  __threadfence();
  return shared.last != 0;
}

// The beams of a group against one another.
__device__ __forceinline__ void rank_beams(const BeamArgs &args, uint32_t group,
                                           BeamShared &shared) {
  constexpr int kEach = kBeamMaximumCandidates / kBeamThreads;
  const uint32_t candidates = args.beams * args.count;
  uint64_t keys[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const uint32_t at = i * kBeamThreads + threadIdx.x;
    keys[i] = kNoKey;
    if (at < candidates) {
      const uint32_t beam = at / args.count, rank = at - beam * args.count;
      const uint32_t row = group * args.beams + beam;
      float score = args.scores[row];
      if (args.finished == nullptr || args.finished[row] == 0) {
        const uint64_t key = __ldcg(args.row_keys + uint64_t{row} * args.count + rank);
        const float logit = value_of(static_cast<uint32_t>(key >> 32));
        score = key == kNoKey ? -INFINITY : score + (logit - __ldcg(args.row_log_sums + row));
      } else if (rank != 0) {
        score = -INFINITY;
      }
      keys[i] = score > -INFINITY ? key_of(score, at) : kNoKey; // NaN: no candidate
    }
  }
  block_best(keys, args.count, shared);
  if (threadIdx.x < args.count) {
    const uint64_t key = shared.best[threadIdx.x];
    const uint64_t out = uint64_t{group} * args.count + threadIdx.x;
    float score = -INFINITY;
    int32_t parent = -1, token = -1;
    bool finished = true;
    if (key != kNoKey) {
      const uint32_t at = ~static_cast<uint32_t>(key);
      const uint32_t beam = at / args.count, rank = at - beam * args.count;
      const uint32_t row = group * args.beams + beam;
      score = value_of(static_cast<uint32_t>(key >> 32));
      parent = static_cast<int32_t>(row);
      finished = args.finished != nullptr && args.finished[row] != 0;
      if (finished) {
        token = args.end_token;
      } else {
        const uint64_t from = __ldcg(args.row_keys + uint64_t{row} * args.count + rank);
        token = static_cast<int32_t>(~static_cast<uint32_t>(from));
        finished = token == args.end_token;
      }
    }
    shared.pool[threadIdx.x] = uint64_t{finished ? 1u : 0u};
    args.parents_out[out] = parent;
    args.tokens_out[out] = token;
    // scores_out may be scores: all of the group's were read before the
    // barriers above; finished_out is stored behind one more.
    args.scores_out[out] = score;
  }
  __syncthreads();
  if (threadIdx.x < args.count && args.finished_out != nullptr) {
    args.finished_out[uint64_t{group} * args.count + threadIdx.x] =
        static_cast<uint8_t>(shared.pool[threadIdx.x]);
  }
}

// grid (chunks, rows). Width elements a load, Loads of them per thread.
template <typename T, int Width, int Loads>
__device__ __forceinline__ void beam_select(const BeamArgs &args) {
  __shared__ BeamShared shared;
  constexpr int kEach = Width * Loads;
  constexpr uint32_t kChunk = kBeamThreads * kEach;
  const uint32_t chunk = blockIdx.x, row = blockIdx.y;
  const uint32_t group = row / args.beams;
  const bool going = args.finished == nullptr || args.finished[row] == 0;
  if (going) {
    const T *logits = static_cast<const T *>(args.logits) + row * args.logits_stride;
    const uint32_t begin = chunk * kChunk;
    float x[kEach];
#pragma unroll
    for (int load = 0; load < Loads; ++load) {
      const uint32_t at = begin + (load * kBeamThreads + threadIdx.x) * Width;
      if (at + Width <= args.vocab) {
        const auto v = *reinterpret_cast<const Vector<T, Width> *>(logits + at);
#pragma unroll
        for (int i = 0; i < Width; ++i) {
          x[load * Width + i] = to_float(v.at[i]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < Width; ++i) {
          x[load * Width + i] = at + i < args.vocab ? to_float(logits[at + i]) : -INFINITY;
        }
      }
    }
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      top = fmaxf(top, x[i]); // passes over NaN
    }
    top = block_max(top, shared);
    const float base = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const float e = exp2_fast((x[i] - base) * kLog2E);
      sum += x[i] != x[i] ? 0.0f : e;
    }
    sum = block_sum(sum, shared);
    uint64_t keys[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const uint32_t at = begin + ((i / Width) * kBeamThreads + threadIdx.x) * Width + i % Width;
      keys[i] = at < args.vocab ? key_of(x[i], at) : kNoKey;
    }
    block_best(keys, args.count, shared);
    const uint64_t slot = uint64_t{row} * args.chunks + chunk;
    if (threadIdx.x < args.count) {
      args.chunk_keys[slot * args.count + threadIdx.x] = shared.best[threadIdx.x];
    }
    if (threadIdx.x == 0) {
      args.chunk_sums[slot] = {top, sum};
    }
  }
  if (!arrive_last(args.row_arrivals + row, args.chunks, shared)) {
    return;
  }
  if (going) {
    const auto *sums =
        reinterpret_cast<const float2 *>(args.chunk_sums + uint64_t{row} * args.chunks);
    float top = -INFINITY;
    for (uint32_t i = threadIdx.x; i < args.chunks; i += kBeamThreads) {
      top = fmaxf(top, __ldcg(sums + i).x);
    }
    top = block_max(top, shared);
    float sum = 0.0f;
    for (uint32_t i = threadIdx.x; i < args.chunks; i += kBeamThreads) {
      const float2 s = __ldcg(sums + i);
      sum += s.x == -INFINITY ? 0.0f : s.y * exp2_fast((s.x - top) * kLog2E);
    }
    sum = block_sum(sum, shared);
    block_best_of(args.chunk_keys + uint64_t{row} * args.chunks * args.count,
                  args.chunks * args.count, args.count, shared);
    if (threadIdx.x < args.count) {
      args.row_keys[uint64_t{row} * args.count + threadIdx.x] = shared.best[threadIdx.x];
    }
    if (threadIdx.x == 0) {
      args.row_log_sums[row] = top + logf(sum);
    }
  }
  if (!arrive_last(args.group_arrivals + group, args.beams, shared)) {
    return;
  }
  rank_beams(args, group, shared);
}

} // namespace lrrt::ops

#endif // LRRT_PAGED_BEAM_SELECT_CUH_
