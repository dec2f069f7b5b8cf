// Rotary positions of queries and keys, and the append of keys and values to
// their pages: (a, b) -> (a cos - b sin, b cos + a sin) for each pair, in 32
// bits, rounded once.
//
// Bound by memory: every input is read once and every output written once
// (the cosine and sine rows come from the caches, a token's heads share them).
// A thread takes a vector of each half of a head's pairs, or a vector that is
// copied (CopyWidth elements: wider where only the halves are odd), and has its loads under way before it knows the token's place.
// Neighbouring threads take neighbouring columns, so rows are read and written
// in whole lines. Value heads come after all query and key heads: blocks do
// one or the other. More vectors a thread (four heads' with the same angles) left
// fewer loads under way and took 124 us where this takes 72.
//
// Measured, 32 heads over 8 of 128 elements in bf16: 16384 tokens 72 us (5.7 TB/s);
// 14 heads over 2 of 64 in f32, one token for each of 32 sequences: 2.1 us, a
// launch's latency.
#ifndef LRRT_PAGED_ROPE_APPEND_CUH_
#define LRRT_PAGED_ROPE_APPEND_CUH_

#include "common.cuh"

namespace lrrt::ops {

// Where a token's rows of the cache are.
struct Place {
  uint32_t page, row;
  bool valid;
};

__device__ __forceinline__ Place place_of(const RopeAppendArgs &args, uint32_t token,
                                          int32_t position) {
  const int32_t sequence =
      args.sequences != nullptr ? args.sequences[token] : static_cast<int32_t>(token);
  Place place{0, 0, static_cast<uint32_t>(sequence) < args.table.rows &&
                        static_cast<uint32_t>(position) < args.table_positions}; // or negative
  if (place.valid) {
    const uint32_t column = args.cache.page.quotient(static_cast<uint32_t>(position));
    place.row = static_cast<uint32_t>(position) - column * args.cache.page.divisor;
    place.valid = column < args.table.columns;
    if (place.valid) {
      const int32_t page = args.table.pages[sequence * args.table.row_stride + column];
      place.page = static_cast<uint32_t>(page);
      place.valid = place.page < args.cache.page_count;
    }
  }
  return place;
}

template <typename T, int Width>
__device__ __forceinline__ void append_values(const RopeAppendArgs &args, uint32_t item) {
  const uint32_t token = args.values_per_token.quotient(item);
  const uint32_t in_token = item - token * args.values_per_token.divisor;
  const uint32_t head = args.values_per_head.quotient(in_token);
  const uint32_t at = (in_token - head * args.values_per_head.divisor) * Width;
  WordVector<T, Width> x;
  x.load(static_cast<const T *>(args.v.data) + args.v.offset(token, head) + at);
  const Place place = place_of(args, token, args.positions[token]);
  if (place.valid) {
    const Pages &values = args.cache.values;
    x.store(static_cast<T *>(values.data) + values.offset(place.page, place.row, head) + at);
  }
}

template <typename T, int Width, int CopyWidth, bool Interleaved>
__device__ __forceinline__ void rope_append(const RopeAppendArgs &args) {
  using V = WordVector<T, Width>;
  using W = Words<T>;
  constexpr int kPerWord = 4 / static_cast<int>(sizeof(T));
  const uint32_t turned_blocks = (args.items + kRopeThreads - 1u) / kRopeThreads;
  if (blockIdx.x >= turned_blocks) {
    const uint32_t item = (blockIdx.x - turned_blocks) * kRopeThreads + threadIdx.x;
    if (item < args.value_items) {
      append_values<T, CopyWidth>(args, item);
    }
    return;
  }
  const uint32_t item = blockIdx.x * kRopeThreads + threadIdx.x;
  if (item >= args.items) {
    return;
  }
  const uint32_t token = args.per_token.quotient(item);
  const uint32_t in_token = item - token * args.per_token.divisor;
  const int32_t position = args.positions[token];
  const uint32_t head = args.per_head.quotient(in_token);
  const uint32_t unit = in_token - head * args.per_head.divisor;
  const bool is_key = head >= args.heads;
  const uint32_t half = args.rotary_dim / 2u, turned = half / Width;
  const bool turns = unit < turned;
  const uint32_t pair = unit * Width; // first of the pairs
  // The elements: of the pairs' first and second halves, or past the pairs.
  uint32_t at = args.rotary_dim + (unit - turned) * CopyWidth, at_second = at;
  if (turns) {
    at = Interleaved ? 2u * pair : pair;
    at_second = Interleaved ? at + Width : at + half;
  }
  const T *from = is_key ? static_cast<const T *>(args.k.data) +
                               args.k.offset(token, head - args.heads)
                         : static_cast<const T *>(args.q.data) + args.q.offset(token, head);
  V x[2];
  WordVector<T, CopyWidth> copied;
  if (CopyWidth == Width || turns) {
    x[0].load(from + at);
  } else {
    copied.load(from + at);
  }
  if (turns) {
    x[1].load(from + at_second);
  }

  const Place place = place_of(args, token, position);
  T *to;
  if (is_key) {
    if (!place.valid) {
      return;
    }
    const Pages &keys = args.cache.keys;
    to = static_cast<T *>(keys.data) + keys.offset(place.page, place.row, head - args.heads);
  } else {
    to = static_cast<T *>(args.q_out.data) + args.q_out.offset(token, head);
    if (!place.valid) { // padding
      x[0] = V{};
      x[1] = V{};
      copied = {};
    }
  }
  if (turns && place.valid) {
    constexpr int kPart = Width < 4 ? Width : 4;
    const size_t angles = static_cast<size_t>(position) * half + pair;
    float c[Width], s[Width];
#pragma unroll
    for (int part = 0; part < Width; part += kPart) {
      WordVector<float, kPart> cos4, sin4;
      cos4.load(args.cos_table + angles + part);
      sin4.load(args.sin_table + angles + part);
#pragma unroll
      for (int i = 0; i < kPart; ++i) {
        c[part + i] = __uint_as_float(cos4.at[i]);
        s[part + i] = __uint_as_float(sin4.at[i]);
      }
    }
    auto turn = [&](int j, float &a, float &b) {
      const float first = a, second = b;
      a = first * c[j] - second * s[j];
      b = second * c[j] + first * s[j];
    };
    if constexpr (Interleaved && kPerWord == 2 && Width > 1) { // a pair is a word
#pragma unroll
      for (int j = 0; j < Width; ++j) {
        uint32_t &word = x[j / V::kWords].at[j % V::kWords];
        float a = W::value(word, 0), b = W::value(word, 1);
        turn(j, a, b);
        word = W::of(a, b);
      }
    } else if constexpr (Interleaved && Width > 1) { // two words
#pragma unroll
      for (int j = 0; j < Width; ++j) {
        uint32_t &low = x[2 * j / Width].at[2 * j % Width];
        uint32_t &high = x[(2 * j + 1) / Width].at[(2 * j + 1) % Width];
        float a = W::value(low, 0), b = W::value(high, 0);
        turn(j, a, b);
        low = W::of(a, 0.0f);
        high = W::of(b, 0.0f);
      }
    } else { // in the two vectors
#pragma unroll
      for (int k = 0; k < V::kWords; ++k) {
        uint32_t &low = x[0].at[k], &high = x[1].at[k];
        float a = W::value(low, 0), b = W::value(high, 0);
        float a_next = W::value(low, kPerWord - 1), b_next = W::value(high, kPerWord - 1);
        turn(Width > 1 ? k * kPerWord : 0, a, b);
        if constexpr (Width > 1 && kPerWord == 2) {
          turn(k * kPerWord + 1, a_next, b_next);
        }
        low = W::of(a, a_next);
        high = W::of(b, b_next);
      }
    }
  }
  if (CopyWidth == Width || turns) {
    x[0].store(to + at);
  } else {
    copied.store(to + at);
  }
  if (turns) {
    x[1].store(to + at_second);
  }
}

} // namespace lrrt::ops

#endif // LRRT_PAGED_ROPE_APPEND_CUH_
