// Rotary positions of queries and keys, and the append of keys and values to
// their pages: (a, b) -> (a cos - b sin, b cos + a sin) for each pair, in 32
// bits, rounded once.
//
// Bound by memory: every input is read once and every output written once
// (the cosine and sine rows come from the caches, a token's heads share them).
// A thread takes one item: a vector of each half of a head's pairs, or a
// vector that is copied. Items of a token are neighbours, so its rows are read
// and written in whole lines.
#ifndef LRRT_PAGED_ROPE_APPEND_CUH_
#define LRRT_PAGED_ROPE_APPEND_CUH_

#include "common.cuh"

namespace lrrt::ops {

template <typename T, int Width, bool Interleaved>
__device__ __forceinline__ void rope_append(const RopeAppendArgs &args) {
  using V = Vector<T, Width>;
  const uint64_t item = uint64_t{blockIdx.x} * kRopeThreads + threadIdx.x;
  if (item >= args.items) {
    return;
  }
  // Tokens below 2^31 / items_per_token are split by the multiplication.
  const uint32_t token = args.items < (uint64_t{1} << 31)
                             ? args.per_token.quotient(static_cast<uint32_t>(item))
                             : static_cast<uint32_t>(item / args.items_per_token);
  const uint32_t in_token =
      static_cast<uint32_t>(item - uint64_t{token} * args.items_per_token);
  const int32_t position = args.positions[token];
  const int32_t sequence =
      args.sequences != nullptr ? args.sequences[token] : static_cast<int32_t>(token);
  bool valid = sequence >= 0 && static_cast<uint32_t>(sequence) < args.table.rows &&
               position >= 0 && static_cast<uint32_t>(position) < args.table_positions;
  const uint32_t column = valid ? args.cache.page.quotient(static_cast<uint32_t>(position)) : 0;
  valid = valid && column < args.table.columns;
  int32_t page = -1;
  if (valid) {
    page = args.table.pages[sequence * args.table.row_stride + column];
    valid = page >= 0 && static_cast<uint32_t>(page) < args.cache.page_count;
  }
  const int64_t row = valid ? position - int64_t{column} * args.cache.page.divisor : 0;

  if (in_token >= args.turned_items) { // a vector of a value head
    if (!valid) {
      return;
    }
    const uint32_t in_values = in_token - args.turned_items;
    const uint32_t head = args.per_value_head.quotient(in_values);
    const uint32_t at = (in_values - head * args.per_value_head.divisor) * Width;
    const T *from = static_cast<const T *>(args.v.data) + token * args.v.row_stride +
                    head * args.v.head_stride + at;
    T *to = static_cast<T *>(args.cache.values) + page * args.cache.value_page +
            row * args.cache.value_token + head * args.cache.value_head + at;
    *reinterpret_cast<V *>(to) = *reinterpret_cast<const V *>(from);
    return;
  }
  const uint32_t head = args.per_head.quotient(in_token);
  const uint32_t unit = in_token - head * args.per_head.divisor;
  const bool is_key = head >= args.heads;
  if (is_key && !valid) {
    return;
  }
  const Rows &source = is_key ? args.k : args.q;
  const T *from = static_cast<const T *>(source.data) + token * source.row_stride +
                  (is_key ? head - args.heads : head) * source.head_stride;
  T *to = is_key ? static_cast<T *>(args.cache.keys) + page * args.cache.key_page +
                       row * args.cache.key_token + (head - args.heads) * args.cache.key_head
                 : static_cast<T *>(args.q_out.data) + token * args.q_out.row_stride +
                       head * args.q_out.head_stride;
  const uint32_t half = args.rotary_dim / 2u;
  const uint32_t turned = half / Width;
  if (unit >= turned) { // past the rotated columns
    const uint32_t at = args.rotary_dim + (unit - turned) * Width;
    V x = *reinterpret_cast<const V *>(from + at);
    if (!valid) {
      x = V{};
    }
    *reinterpret_cast<V *>(to + at) = x;
    return;
  }
  // Pairs first .. first + Width - 1, as two vectors.
  const uint32_t first = unit * Width;
  const uint32_t at[2] = {Interleaved ? 2u * first : first,
                          Interleaved ? 2u * first + Width : first + half};
  V x[2] = {*reinterpret_cast<const V *>(from + at[0]), *reinterpret_cast<const V *>(from + at[1])};
  if (!valid) {
    x[0] = V{};
    x[1] = V{};
  } else {
    using F = Vector<float, (Width < 4 ? Width : 4)>;
    constexpr int kParts = Width < 4 ? 1 : Width / 4;
    constexpr int kPart = Width < 4 ? Width : 4;
    const size_t angles = static_cast<size_t>(position) * half + first;
    float c[Width], s[Width];
#pragma unroll
    for (int part = 0; part < kParts; ++part) {
      const F cos4 = *reinterpret_cast<const F *>(args.cos_table + angles + part * kPart);
      const F sin4 = *reinterpret_cast<const F *>(args.sin_table + angles + part * kPart);
#pragma unroll
      for (int i = 0; i < kPart; ++i) {
        c[part * kPart + i] = cos4.at[i];
        s[part * kPart + i] = sin4.at[i];
      }
    }
#pragma unroll
    for (int i = 0; i < Width; ++i) {
      // Element of the first and of the second of pair first + i.
      T &low = Interleaved ? x[2 * i / Width].at[2 * i % Width] : x[0].at[i];
      T &high = Interleaved ? x[(2 * i + 1) / Width].at[(2 * i + 1) % Width] : x[1].at[i];
      const float a = to_float(low), b = to_float(high);
      low = from_float<T>(a * c[i] - b * s[i]);
      high = from_float<T>(b * c[i] + a * s[i]);
    }
  }
  *reinterpret_cast<V *>(to + at[0]) = x[0];
  *reinterpret_cast<V *>(to + at[1]) = x[1];
}

} // namespace lrrt::ops

#endif // LRRT_PAGED_ROPE_APPEND_CUH_
