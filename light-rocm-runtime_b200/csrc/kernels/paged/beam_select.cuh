// The best continuations over the beams of a group and the vocabulary.
//
// One pass over the logits. A block reads a part of a row in rounds of 16 KB, four
// of them under way by cp.async; every thread has its own elements copied, so
// that rounds have no barriers. It keeps a running maximum and sum of
// exponentials (sums of disjoint elements join as l1 e^(m1 - m) + l2 e^(m2 - m)),
// and notes the maximum of each round. The threads' maxima give a floor that at
// least `count` elements reach and few others; those few are read once more
// (from the caches, and only where a noted maximum reaches the floor) and ranked.
// The last block of a row joins the parts, the last row of a group ranks the
// beams' candidates by score + logit - log sum.
//
// Bound by reading the logits once, by the exponentials (16 a clock and SM: 10 us
// for the two rows of 151936 that the fullest SM has of 256), and by the fixed
// work of a part (7 us to the end of the launch: floor, second reading, ranking,
// joining) where there are few rows. Measured: 256 rows of 151936 logits in bf16,
// 8 beams a group, 16 wanted, 23.6 us (3.3 TB/s; an earlier form with two rounds under
// way in registers 30.8 us, with the ring 24.3); 200 rows in f32 27.6 us (4.4 TB/s);
// 4 rows in f32, 9.9 us.
//
// Pooled elements are 64-bit keys, the value's order in the upper half and the
// complement of the index in the lower, so that no two are equal and the order
// of threads and blocks decides nothing.
#ifndef LRRT_PAGED_BEAM_SELECT_CUH_
#define LRRT_PAGED_BEAM_SELECT_CUH_

#include "common.cuh"

namespace lrrt::ops {

constexpr uint32_t kBeamWarps = kBeamThreads / 32u;
constexpr uint32_t kBeamShare = kBeamPool / kBeamWarps; // of the pool, for a warp
static_assert(kBeamShare == kBeamThreads && kBeamShare >= 2u * kBeamMaximumCount,
              "a thread takes one key of each share; a share holds the best of two sets");


struct BeamShared {
  union {
    uint4 ring[kBeamStages][kBeamRoundBytes / 16u]; // rounds under way
    uint64_t pool[kBeamPool];                       // after the last of them
  };
  float noted[kBeamNotedRounds + 1][kBeamThreads]; // maximum of each round and thread
  uint64_t best[kBeamMaximumCount]; // the pool's best, falling, when it was last ranked
  uint64_t floors[kBeamWarps][32];
  float2 sums[kBeamWarps];
  uint32_t pooled, listed, floor;
  uint32_t last;
};
static_assert(sizeof(BeamShared) <= kBeamSharedBytes, "shared memory of a block");

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
// What stands for no key in the pool, different at each place: below every
// key too, whose order is never 0.
__device__ __forceinline__ uint64_t key_or_place(uint64_t key, uint32_t place) {
  return key == kNoKey ? uint64_t{place} + 1u : key;
}
__device__ __forceinline__ uint64_t key_or_none(uint64_t key) {
  return key >> 32 != 0 ? key : kNoKey;
}

__device__ __forceinline__ uint64_t larger(uint64_t a, uint64_t b) { return a > b ? a : b; }

// A floor that at least `count` elements reach, whose threads' maxima are
// `mine`, and not many more: the threads form classes, at least four times
// `count` of them (or every thread one), and the floor is the count-th largest
// of the classes' maxima. With 4 count classes about
// 4 count ln(4 / 3) = 1.15 count elements reach it where their order is random.
// Two barriers.
__device__ __forceinline__ float count_floor(float mine, uint32_t count, BeamShared &shared) {
  float *values = reinterpret_cast<float *>(shared.floors);
  uint32_t each = 32; // neighbouring threads of a class
  while (each > 1u && kBeamThreads / each < 4u * count) {
    each >>= 1u;
  }
  const uint32_t classes = kBeamThreads / each;
#pragma unroll
  for (uint32_t offset = 1; offset < 32u; offset <<= 1u) {
    const float other = __shfl_xor_sync(kAllLanes, mine, offset);
    mine = offset < each ? fmaxf(mine, other) : mine;
  }
  if (threadIdx.x == 0) {
    shared.floor = ~0u;
  }
  if (threadIdx.x % each == 0) {
    values[threadIdx.x / each] = mine;
  }
  __syncthreads();
  if (threadIdx.x < classes) {
    mine = values[threadIdx.x];
    uint32_t larger_ones = 0;
#pragma unroll 2
    for (uint32_t j = 0; j < classes; j += 8u) {
      const float4 v = *reinterpret_cast<const float4 *>(values + j);
      const float4 w = *reinterpret_cast<const float4 *>(values + j + 4u);
      larger_ones += (v.x > mine ? 1u : 0u) + (v.y > mine ? 1u : 0u) + (v.z > mine ? 1u : 0u) +
                     (v.w > mine ? 1u : 0u) + (w.x > mine ? 1u : 0u) + (w.y > mine ? 1u : 0u) +
                     (w.z > mine ? 1u : 0u) + (w.w > mine ? 1u : 0u);
    }
    if (larger_ones < count) {
      atomicMin(&shared.floor, order_of(mine));
    }
  }
  __syncthreads();
  return value_of(shared.floor);
}

__device__ __forceinline__ uint64_t warp_largest(uint64_t key) {
#pragma unroll
  for (uint32_t offset = 16; offset != 0; offset >>= 1u) {
    key = larger(key, __shfl_xor_sync(kAllLanes, key, offset));
  }
  return key;
}

// Puts the `count` largest of the pool's first `total` keys into `best`, falling,
// kNoKey after the last: ranked by counting the larger ones. With more keys than
// threads, those below the count-th largest of the threads' maxima are dropped
// first: no more than `count` threads have keys that are left. The pool's
// contents are lost. Begins and ends with a barrier.
__device__ __noinline__ void rank_pool(uint32_t total, uint32_t count, BeamShared &shared) {
  const uint32_t thread = threadIdx.x;
  __syncthreads();
  if (total <= kBeamThreads) {
    // One, two or four threads for a key, each counting among as many others.
    const uint32_t shift = total <= kBeamThreads / 4u ? 2u : total <= kBeamThreads / 2u ? 1u : 0u;
    const uint32_t parts = 1u << shift, at = thread >> shift;
    const uint32_t of_warp = 32u >> shift; // keys
    if (thread / 32u * of_warp < total) {  // whole warps, the last one's surplus without keys
      const uint64_t key = at < total ? shared.pool[at] : kNoKey;
      uint32_t rank = 0;
#pragma unroll 8
      for (uint32_t j = thread & (parts - 1u); j < total; j += parts) {
        rank += shared.pool[j] > key ? 1u : 0u;
      }
      // The lanes' loops differ in length, so all of the warp's are waited for.
      rank += shift > 0u ? __shfl_xor_sync(kAllLanes, rank, 1) : 0u;
      rank += shift > 1u ? __shfl_xor_sync(kAllLanes, rank, 2) : 0u;
      if (at < total && rank < count) {
        shared.best[rank] = key_or_none(key);
      }
    }
    if (thread >= total && thread < count) {
      shared.best[thread] = kNoKey;
    }
    __syncthreads();
    return;
  }
  uint64_t keys[kBeamWarps];
  uint64_t mine = kNoKey;
#pragma unroll
  for (uint32_t i = 0; i < kBeamWarps; ++i) {
    const uint32_t at = i * kBeamThreads + thread;
    keys[i] = at < total ? shared.pool[at] : kNoKey;
    mine = larger(mine, keys[i]);
  }
  if (thread == 0) {
    shared.pooled = 0;
  }
  uint64_t *maxima = &shared.floors[0][0];
  maxima[thread] = mine;
  __syncthreads();
  uint32_t larger_ones = 0;
#pragma unroll 8
  for (uint32_t j = 0; j < kBeamThreads; ++j) {
    larger_ones += maxima[j] > mine ? 1u : 0u;
  }
  if (larger_ones + 1u == count) { // one thread: no two keys are equal
    shared.best[0] = mine;
  }
  __syncthreads();
  const uint64_t floor = shared.best[0];
  if (larger_ones < count) {
#pragma unroll
    for (uint32_t i = 0; i < kBeamWarps; ++i) {
      if (keys[i] >= floor) {
        shared.pool[atomicAdd(&shared.pooled, 1u)] = keys[i];
      }
    }
  }
  __syncthreads();
  total = shared.pooled; // at least `count`
#pragma unroll 1
  for (uint32_t at = thread; at < total; at += kBeamThreads) {
    const uint64_t key = shared.pool[at];
    uint32_t rank = 0;
#pragma unroll 8
    for (uint32_t j = 0; j < total; ++j) {
      rank += shared.pool[j] > key ? 1u : 0u;
    }
    if (rank < count) {
      shared.best[rank] = key_or_none(key);
    }
  }
  __syncthreads();
}

// The same for one warp's share, which it has alone: one largest after
// another. Returns the last of them.
__device__ __noinline__ uint64_t prune_share(uint64_t *share, uint32_t held, uint32_t count) {
  const uint32_t lane = threadIdx.x & 31u;
  constexpr uint32_t kEach = kBeamShare / 32u;
  uint64_t keys[kEach];
  __syncwarp();
#pragma unroll
  for (uint32_t i = 0; i < kEach; ++i) {
    keys[i] = i * 32u + lane < held ? share[i * 32u + lane] : kNoKey;
  }
  __syncwarp();
  uint64_t bound = ~uint64_t{0};
#pragma unroll 1
  for (uint32_t rank = 0; rank < count; ++rank) {
    uint64_t best = kNoKey;
#pragma unroll
    for (uint32_t i = 0; i < kEach; ++i) {
      best = keys[i] < bound ? larger(best, keys[i]) : best;
    }
    bound = warp_largest(best);
    if (lane == 0) {
      share[rank] = bound;
    }
  }
  __syncwarp();
  return bound;
}

// e^(x - base), 1 where they are equal at any size: rows may be masked throughout
// with a type's lowest value, whose product with log2 e leaves 32 bits. (x log2 e -
// base log2 e in one instruction took 22.7 us where this takes 23.6, 256 rows of 151936
// in bf16; it lost all of a sum above 1e10, and 8e-4 of its logarithm at 6e4.)
__device__ __forceinline__ float exp_above(float x, float base) {
  return exp2_fast((x - base) * kLog2E);
}

// Maximum and sum of a set of elements, and of two sets.
__device__ __forceinline__ float2 join_sums(float2 a, float2 b) {
  const float top = fmaxf(a.x, b.x);
  const float base = top == -INFINITY ? 0.0f : top;
  return make_float2(top, a.y * exp_above(a.x, base) + b.y * exp_above(b.x, base));
}
__device__ __forceinline__ float2 join_lanes(float2 mine) {
#pragma unroll
  for (uint32_t offset = 16; offset != 0; offset >>= 1u) {
    mine = join_sums(mine, make_float2(__shfl_xor_sync(kAllLanes, mine.x, offset),
                                       __shfl_xor_sync(kAllLanes, mine.y, offset)));
  }
  return mine;
}

// The logarithm of a row's sum, relative to its maximum. It goes into all scores of
// the row, so it is kept in 64 bits and scores are rounded once: without the sum's
// exponent log2f is below 1, and its last place as small. (In 32 bits scores were
// 1.1e-7 off, relative to their sizes; now 0.4e-7.)
__device__ __forceinline__ double log_of(float sum) {
  float whole = 0.0f, rest = sum;
  if (rest >= 1.0f && rest < INFINITY) {
    const uint32_t bits = __float_as_uint(rest);
    whole = static_cast<float>(static_cast<int32_t>(bits >> 23) - 127);
    rest = __uint_as_float((bits & 0x007fffffu) | 0x3f800000u);
  }
  return (double{whole} + double{log2f(rest)}) * 0.69314718055994531;
}

// Whether this block is the last of `blocks` to get here; its reads then see
// what the others wrote before. The counter is zero again afterwards.
__device__ __forceinline__ bool arrive_last(uint32_t *counter, uint32_t blocks,
                                            BeamShared &shared) {
  if (blocks == 1u) {
    __syncthreads();
    return true;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    shared.last = arrive(counter) + 1u == blocks ? 1u : 0u;
    if (shared.last != 0) {
      *counter = 0;
    }
  }
  __syncthreads();
  return shared.last != 0;
}

// The beams of a group against one another.
__device__ __forceinline__ void rank_beams(const BeamArgs &args, uint32_t group,
                                           BeamShared &shared) {
  const uint32_t candidates = args.beams * args.count;
#pragma unroll 1
  for (uint32_t at = threadIdx.x; at < candidates; at += kBeamThreads) {
    const uint32_t beam = at / args.count, rank = at - beam * args.count;
    const uint32_t row = group * args.beams + beam;
    float score = args.scores[row];
    if (args.finished == nullptr || args.finished[row] == 0) {
      const uint64_t key = __ldcg(args.row_keys + uint64_t{row} * args.count + rank);
      const float logit = value_of(static_cast<uint32_t>(key >> 32));
      const double above = double{logit} - __ldcg(args.row_tops + row); // exact, or nearly
      score = key == kNoKey ? -INFINITY
                            : static_cast<float>(double{score} +
                                                 (above - __ldcg(args.row_log_sums + row)));
    } else if (rank != 0) {
      score = -INFINITY;
    }
    const uint64_t key = score > -INFINITY ? key_of(score, at) : kNoKey; // NaN: no candidate
    shared.pool[at] = key_or_place(key, at);
  }
  rank_pool(candidates, args.count, shared);
  bool finished = true;
  const uint64_t out = uint64_t{group} * args.count + threadIdx.x;
  if (threadIdx.x < args.count) {
    const uint64_t key = shared.best[threadIdx.x];
    float score = -INFINITY;
    int32_t parent = -1, token = -1;
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
    args.parents_out[out] = parent;
    args.tokens_out[out] = token;
    args.scores_out[out] = score; // may be `scores`: all were read before the barriers above
  }
  __syncthreads(); // finished_out may be `finished`
  if (threadIdx.x < args.count && args.finished_out != nullptr) {
    args.finished_out[out] = finished ? 1u : 0u;
  }
}

// grid (parts, rows). Parts begin on 16 bytes; the elements of a row before the
// first such place, and after the last whole vector, are taken one by one.
template <typename T>
__device__ __forceinline__ void beam_select(const BeamArgs &args) {
  extern __shared__ __align__(16) unsigned char beam_memory[];
  BeamShared &shared = *reinterpret_cast<BeamShared *>(beam_memory);
  constexpr uint32_t kRound = beam_round(sizeof(T));
  constexpr int kEach = kRound / kBeamThreads; // elements of a thread and round
  constexpr int kPerWord = 4 / sizeof(T);
  constexpr int Width = 16 / sizeof(T); // elements of a vector
  constexpr int kWords = kEach / kPerWord;
  using W = Words<T>;
  const uint32_t part = blockIdx.x, row = blockIdx.y;
  const uint32_t group = row / args.beams;
  const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5u;
  const bool going = args.finished == nullptr || args.finished[row] == 0;
  if (going) {
    const T *logits = static_cast<const T *>(args.logits) + row * args.logits_stride;
    const uint32_t skew =
        min(static_cast<uint32_t>(-reinterpret_cast<uintptr_t>(logits) % 16u / sizeof(T)),
            args.vocab); // elements before the row's first vector
    const uint32_t begin = min(skew + part * args.part_elements, args.vocab);
    const uint32_t end = min(args.vocab - begin, args.part_elements) + begin;
    auto index_of = [&](uint32_t round, int i) {
      return round + ((i / Width) * kBeamThreads + threadIdx.x) * Width + i % Width;
    };
    // A thread's elements of a round, -infinity past the last whole vector.
    const uint32_t whole = end - (end - begin) % Width;
    auto load = [&](uint32_t stage, uint32_t round) {
#pragma unroll
      for (int i = 0; i < kEach; i += Width) {
        const uint32_t index = index_of(round, i);
        if (index < whole) {
          copy_16(shared_address(&shared.ring[stage][i / Width * kBeamThreads + threadIdx.x]),
                  reinterpret_cast<uint64_t>(logits + index), true);
        }
      }
    };
    auto read = [&](uint32_t(&to)[kWords], uint32_t stage, uint32_t round) {
#pragma unroll
      for (int i = 0; i < kEach; i += Width) {
        uint4 v = shared.ring[stage][i / Width * kBeamThreads + threadIdx.x];
        if (index_of(round, i) >= whole) {
          v = make_uint4(W::kLeast, W::kLeast, W::kLeast, W::kLeast);
        }
        to[i / kPerWord] = v.x;
        to[i / kPerWord + 1] = v.y;
        to[i / kPerWord + 2] = v.z;
        to[i / kPerWord + 3] = v.w;
      }
    };
    float top = -INFINITY, sum = 0.0f; // as join_sums takes them
    float largest = -INFINITY;
    auto take = [&](const uint32_t(&from)[kWords], uint32_t round, uint32_t number) {
      uint32_t larger_word = from[0];
#pragma unroll
      for (int k = 1; k < kWords; ++k) {
        larger_word = W::larger(larger_word, from[k]);
      }
      const float most = fmaxf(W::largest(larger_word), -INFINITY); // NaN counts as -infinity
      shared.noted[number][threadIdx.x] = most;
      largest = fmaxf(largest, most);
      const float now = fmaxf(top, most);
      const float base = now == -INFINITY ? 0.0f : now;
      float each[4] = {}; // four sums at a time
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        each[i % 4] += exp_above(W::value(from[i / kPerWord], i % kPerWord), base);
      }
      float terms = (each[0] + each[1]) + (each[2] + each[3]);
      if (terms != terms) { // there is a NaN
        terms = 0.0f;
#pragma unroll 1
        for (int i = 0; i < kEach; ++i) {
          const uint32_t index = index_of(round, i);
          const float y = index < whole ? to_float(logits[index]) : -INFINITY;
          terms += y == y ? exp_above(y, base) : 0.0f;
        }
      }
      sum = sum * exp_above(top, base) + terms;
      top = now;
    };
    // Each thread has its own elements copied, so that rounds need no barrier;
    // a stage is filled again once its elements are in registers.
    const uint32_t rounds = (whole - begin + kRound - 1u) / kRound;
#pragma unroll
    for (uint32_t i = 0; i < kBeamStages; ++i) {
      if (i < rounds) {
        load(i, begin + i * kRound);
      }
      commit_copies();
    }
    uint32_t stage = 0;
#pragma unroll 1
    for (uint32_t number = 0; number < rounds; ++number) {
      const uint32_t round = begin + number * kRound;
      uint32_t words[kWords];
      wait_copies<kBeamStages - 1>();
      read(words, stage, round);
      if (number + kBeamStages < rounds) {
        load(stage, round + kBeamStages * kRound);
      }
      commit_copies();
      take(words, round, number);
      stage = stage + 1u == kBeamStages ? 0u : stage + 1u;
    }

    // Elements before the first and past the last whole vector: one more round,
    // of an element for each of the first threads.
    auto odd_index = [&](uint32_t thread) -> uint32_t { // at `end` there is none
      if (thread < Width) {
        return part == 0 && thread < skew ? thread : end;
      }
      return min(whole + thread - Width, end);
    };
    float odd = -INFINITY;
    if (threadIdx.x < 2u * Width && odd_index(threadIdx.x) != end) {
      odd = to_float(logits[odd_index(threadIdx.x)]);
      odd = odd == odd ? odd : -INFINITY;
      largest = fmaxf(largest, odd);
      const float2 joined = join_sums(make_float2(top, sum), make_float2(odd, 1.0f));
      top = joined.x;
      sum = joined.y;
    }
    shared.noted[rounds][threadIdx.x] = odd;

    // What reaches the floor, into the pool: rounds of threads with such a
    // maximum are listed, and each is read again by a warp, an element a lane,
    // four such reads at a time.
    static_assert(kEach <= 32, "a lane per element");
    static_assert((kBeamNotedRounds + 1u) * kBeamThreads <= 65536u, "a listed round is 16 bits");
    static_assert(kBeamNotedRounds + 1u <= 64u, "a bit per round");
    constexpr uint32_t kListed = 2u * kBeamPool, kPooled = kBeamPool / 2u;
    auto *list = reinterpret_cast<uint16_t *>(shared.pool + kPooled); // the pool's other half
    if (threadIdx.x == 0) {
      shared.pooled = 0;
      shared.listed = 0;
    }
    float floor = count_floor(largest, args.count, shared);
    uint64_t least_key = uint64_t{order_of(floor)} << 32; // the lowest that enters
    uint64_t reaching = 0; // this thread's rounds
#pragma unroll 4
    for (uint32_t i = 0; i <= rounds; ++i) {
      reaching |= uint64_t{shared.noted[i][threadIdx.x] >= floor} << i;
    }
    if (reaching != 0) {
      uint32_t at = atomicAdd(&shared.listed, static_cast<uint32_t>(__popcll(reaching)));
#pragma unroll 1
      for (; reaching != 0; reaching &= reaching - 1u, ++at) {
        if (at < kListed) {
          list[at] = static_cast<uint16_t>((__ffsll(reaching) - 1) * kBeamThreads + threadIdx.x);
        }
      }
    }
    __syncthreads();
    // The key of this lane's element of a thread's round.
    auto key_at = [&](uint32_t i, uint32_t thread) -> uint64_t {
      uint32_t index =
          begin + i * kRound + (lane / Width * kBeamThreads + thread) * Width + lane % Width;
      bool there = lane < kEach && index < whole;
      if (i == rounds) {
        index = odd_index(thread);
        there = lane == 0 && index != end;
      }
      return there ? key_of(to_float(logits[index]), index) : kNoKey;
    };
    const uint32_t listed = shared.listed;
#pragma unroll 1
    for (uint32_t first = warp; first < min(listed, kListed); first += 4u * kBeamWarps) {
      uint64_t keys[4];
#pragma unroll
      for (uint32_t k = 0; k < 4u; ++k) {
        const uint32_t at = first + k * kBeamWarps;
        keys[k] = kNoKey;
        if (at < min(listed, kListed)) {
          keys[k] = key_at(list[at] / kBeamThreads, list[at] % kBeamThreads);
        }
      }
#pragma unroll
      for (uint32_t k = 0; k < 4u; ++k) {
        if (keys[k] >= least_key) {
          const uint32_t at = atomicAdd(&shared.pooled, 1u);
          if (at < kPooled) {
            shared.pool[at] = keys[k];
          }
        }
      }
    }
    __syncthreads();
    uint32_t total = shared.pooled;
    if (listed > kListed || total > kPooled) {
      // Equal values, or an order that defeats the floor: each warp keeps the
      // best of its threads' elements in its share of the pool, raising the
      // floor as it goes.
      __syncthreads();
      uint64_t *share = shared.pool + warp * kBeamShare;
      uint32_t held = 0;
#pragma unroll 1
      for (uint32_t i = 0; i <= rounds; ++i) {
        uint32_t looking = __ballot_sync(kAllLanes, shared.noted[i][threadIdx.x] >= floor);
#pragma unroll 1
        for (; looking != 0; looking &= looking - 1u) {
          const uint64_t key = key_at(i, warp * 32u + __ffs(looking) - 1u);
          const uint32_t entering = __ballot_sync(kAllLanes, key >= least_key);
          if (key >= least_key) {
            share[held + __popc(entering & ((1u << lane) - 1u))] = key;
          }
          held += __popc(entering);
          if (held + 32u > kBeamShare) {
            least_key = prune_share(share, held, args.count) + 1u;
            held = args.count;
            floor = value_of(static_cast<uint32_t>(least_key >> 32));
          }
        }
      }
      for (uint32_t at = held + lane; at < kBeamShare; at += 32u) {
        share[at] = key_or_place(kNoKey, warp * kBeamShare + at);
      }
      total = kBeamPool;
    }
    const float2 sums = join_lanes(make_float2(top, sum));
    if (lane == 0) {
      shared.sums[warp] = sums;
    }
    rank_pool(total, args.count, shared);
    const uint64_t slot = uint64_t{row} * args.parts + part;
    if (args.parts != 1u && threadIdx.x < args.count) {
      args.part_keys[slot * args.count + threadIdx.x] = shared.best[threadIdx.x];
    }
    if (threadIdx.x == 0) {
      float2 all = shared.sums[0];
#pragma unroll
      for (uint32_t w = 1; w < kBeamWarps; ++w) {
        all = join_sums(all, shared.sums[w]);
      }
      if (args.parts != 1u) {
        args.part_sums[slot] = {all.x, all.y};
      } else {
        args.row_tops[row] = all.x;
        args.row_log_sums[row] = log_of(all.y);
      }
    }
  }
  if (!arrive_last(args.row_arrivals + row, args.parts, shared)) {
    return;
  }
  if (going) {
    if (args.parts != 1u) {
      const uint64_t *keys = args.part_keys + uint64_t{row} * args.parts * args.count;
      const uint32_t total = args.parts * args.count;
#pragma unroll 2
      for (uint32_t at = threadIdx.x; at < total; at += kBeamThreads) {
        shared.pool[at] = key_or_place(__ldcg(keys + at), at);
      }
      if (warp == kBeamWarps - 1u) { // the last one: it has the fewest keys to bring
        const auto *sums =
            reinterpret_cast<const float2 *>(args.part_sums) + uint64_t{row} * args.parts;
        const float2 none = make_float2(-INFINITY, 0.0f);
        const float2 all =
            join_lanes(join_sums(lane < args.parts ? __ldcg(sums + lane) : none,
                                 lane + 32u < args.parts ? __ldcg(sums + lane + 32u) : none));
        if (lane == 0) {
          args.row_tops[row] = all.x;
          args.row_log_sums[row] = log_of(all.y);
        }
      }
      rank_pool(total, args.count, shared);
    }
    if (threadIdx.x < args.count) {
      args.row_keys[uint64_t{row} * args.count + threadIdx.x] = shared.best[threadIdx.x];
    }
  }
  if (!arrive_last(args.group_arrivals + group, args.beams, shared)) {
    return;
  }
  rank_beams(args, group, shared);
}

} // namespace lrrt::ops

#endif // LRRT_PAGED_BEAM_SELECT_CUH_
