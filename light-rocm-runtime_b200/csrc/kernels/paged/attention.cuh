// Attention of one query row per sequence over a paged cache.
//
// One pass over the keys and values with a running maximum m and sum l of
// exp(s - m), in base 2; states of disjoint keys join as m = max(m1, m2),
// l = l1 2^(m1 - m) + l2 2^(m2 - m), and the weighted values likewise.
//
// Bound by reading the cache once. What the layout does about that:
//  - Every unit (a warp, or two with 8 of 16 heads each where the states of all
//    would not fit a warp's registers) streams its own tiles (8 or 16 KB of keys
//    and values) through shared-memory stages filled by cp.async, so a block keeps
//    128 to 192 KB in flight without a barrier between its units. Rows are
//    gathered through the page table, whose entries are read one tile ahead.
//  - The query heads of one key-value head share each row that is read: scores
//    are computed transposed, S^T = K Q^T, with 16 keys as the rows of the
//    matrix product and 8 query heads as its columns, and so are the outputs,
//    O^T = V^T P^T. These shapes (m16n8) waste nothing of up to 8 heads, which
//    memory bounds. (A tcgen05 tile of 128 keys by 16 heads is not built; groups
//    of 9 to 16 heads, which issue slots bound, would be the ones to gain.) A
//    tile's products are summed by themselves and added in rounded 32 bits.
//    16-bit weights are split into two 16-bit parts, so that the probabilities
//    keep 16 bits (in f16 down to 2^-39 of a row's largest); 32-bit operands into
//    two TF32 parts (three products).
//  - The tiles of all sequences and heads form one sequence that is cut into
//    equal parts for the blocks, and each part into equal parts for the units,
//    whatever the lengths are. A row that lies within a unit's part is finished
//    by that unit; the pieces of others are joined in shared memory, and where
//    a row lies in several blocks through the workspace by the last of them to
//    arrive. Pieces are joined in their order, so that results do not depend on
//    timing.
//
// Measured (cache reads at 6.5 TB/s take the time in brackets): 64 ragged
// sequences of up to 8192 keys, 32 heads over 8 of 128 elements in bf16, 136 us
// (122), in pages of one token 162 us (133); two of about 123000 keys with capped
// scores 50 us (38); 128 heads over 8 in bf16 132 us (109), 16 over 4 of 128 in f32
// 180 us (132). Few keys are bound by latency (launch, lengths, page numbers, first
// tile, joining): 32 sequences of 1152, 14 heads over 2 of 64 in f32, 15.9 us
// (5.5); one of 160, 7.7 us.
#ifndef LRRT_PAGED_ATTENTION_CUH_
#define LRRT_PAGED_ATTENTION_CUH_

#include "common.cuh"

namespace lrrt::ops {

__device__ __forceinline__ void load_matrices(uint32_t (&r)[4], uint32_t address) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(address)
               : "memory");
}
__device__ __forceinline__ void load_matrices_transposed(uint32_t (&r)[4], uint32_t address) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(address)
               : "memory");
}
__device__ __forceinline__ uint32_t transpose_matrix(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t load_shared(uint32_t address) {
  uint32_t x;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(x) : "r"(address) : "memory");
  return x;
}

// c += a b for 16-bit elements (m16n8k16) and TF32 (m16n8k8).
__device__ __forceinline__ void multiply(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1, __nv_bfloat16) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, "
               "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void multiply(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1, __half) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, "
               "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void multiply(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1, float) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, "
               "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// c = a b.
__device__ __forceinline__ void multiply_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                               uint32_t b1, __nv_bfloat16) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, "
               "{%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
               : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ void multiply_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                               uint32_t b1, __half) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, "
               "{%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
               : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ void multiply_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                               uint32_t b1, float) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, "
               "{%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
               : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}

// x = high + low to about 21 bits, both TF32: high is x rounded to nearest
// (half away from zero) to 11 bits, low the first 11 bits of the exact rest.
__device__ __forceinline__ void split_tf32(uint32_t bits, uint32_t &high, uint32_t &low) {
  high = (bits + 0x1000u) & 0xffffe000u;
  low = __float_as_uint(__uint_as_float(bits) - __uint_as_float(high)) & 0xffffe000u;
}

// Weights and values are split so that infinite values go through: both parts of
// a weight are positive, so that an infinity times them is that infinity (0, and a
// negative rest, would make a NaN of it), and the second part of an infinite value
// is finite. Weights and values are cut off after their first part, not rounded: the
// rest has their sign, and NaN stays NaN. The rest is rounded to nearest.
__device__ __forceinline__ uint32_t rounded_tf32(float x) {
  return (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
}

// A weight as two TF32 numbers; 2^-126 is nothing beside any sum.
__device__ __forceinline__ void split_weight_tf32(uint32_t bits, uint32_t &high, uint32_t &low) {
  high = bits & 0xffffe000u;
  low = rounded_tf32(fmaxf(__uint_as_float(bits) - __uint_as_float(high), 0x1p-126f));
}

// A value: the rest's size is below 2^117, and stays below it where it is rounded, so
// that the largest numbers do not become infinities. That of an infinity is a NaN
// before the minimum. (Not rounded, and so not bounded from below, 171 us where this
// takes 180, 64 ragged sequences of 16 heads over 4 of 128, and errors of 3.6e-7
// where these are 2.5e-7.)
__device__ __forceinline__ void split_value_tf32(uint32_t bits, uint32_t &high, uint32_t &low) {
  high = bits & 0xffffe000u;
  const float rest = __uint_as_float(bits) - __uint_as_float(high);
  low = rounded_tf32(fmaxf(fminf(rest, 0x1.ffcp116f), -0x1.ffcp116f));
}

// Two weights as a pair of 16-bit numbers, and what they leave over as another. In
// f16 the least number, 2^-39 of the largest weight, stands for a first part of 0.
__device__ __forceinline__ void split_weights(float x, float y, uint32_t &high, uint32_t &low,
                                              __nv_bfloat16) {
  high = __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x7632);
  const __nv_bfloat162 rest = __floats2bfloat162_rn(x - __uint_as_float(high << 16),
                                                    y - __uint_as_float(high & 0xffff0000u));
  memcpy(&low, &rest, 4);
  asm("max.bf16x2 %0, %0, %1;" : "+r"(low) : "r"(0x00800080u)); // 2^-126
}
__device__ __forceinline__ void split_weights(float x, float y, uint32_t &high, uint32_t &low,
                                              __half) {
  asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(high) : "f"(y), "f"(x));
  __half2 first;
  memcpy(&first, &high, 4);
  const __half2 rest = __floats2half2_rn(x - __low2float(first), y - __high2float(first));
  memcpy(&low, &rest, 4);
  asm("max.f16x2 %0, %0, %1;" : "+r"(low) : "r"(0x00010001u));
  asm("max.NaN.f16x2 %0, %0, %1;" : "+r"(high) : "r"(0x00010001u));
}

// Weights are taken 2^kWeightBits times as large, and their sums with them, so that
// f16, which ends at 2^-24, holds those far below a row's largest one: its two
// parts then end at 2^-39 of it. Without, a key 17 below another in its score
// weighed nothing in the products and 4e-8 in the sum. (The largest is 2^15, and
// f16 goes on to 2^16.) bf16 has the exponents of 32 bits.
template <typename T> constexpr float kWeightBits = 0.0f;
template <> constexpr float kWeightBits<__half> = 15.0f;

// The keys of a sequence that a step sees.
struct Span {
  uint32_t begin, end;
};

__device__ __forceinline__ Span span_of(const PagedAttentionArgs &args, uint32_t sequence) {
  const int32_t length = args.lengths[sequence];
  const uint32_t end = length < 0 ? 0u : min(static_cast<uint32_t>(length), args.capacity);
  return {args.window != 0 && end > args.window ? end - args.window : 0u, end};
}

// A tile and its row: a sequence, and a kv head with a block of its query heads.
struct TileCursor {
  uint32_t sequence, row, tile; // row within the sequence; tile within the row
  uint32_t tiles;               // of the row
  Span span;
};

// Team: warps that share a unit's tiles, each with 8 * HeadTiles of the heads.
template <typename T, int Dim, int HeadTiles, int Team> class PagedAttention {
  static constexpr bool kWide = sizeof(T) == 4; // 32-bit elements
  static constexpr uint32_t kRowBytes = attention_row_bytes(Dim, sizeof(T)); // in a tile
  static constexpr uint32_t kHeads = 8u * HeadTiles * Team;
  static constexpr uint32_t kUnits = attention_units(Dim, kRowBytes, kHeads);
  static constexpr uint32_t kWarps = kUnits * Team;
  static constexpr uint32_t kKeys = attention_tile_keys(kRowBytes);
  static constexpr uint32_t kChunks = kRowBytes / 16u; // 16-byte chunks of a row
  static constexpr uint32_t kRowsPerPass = 32u / kChunks;
  static constexpr uint32_t kPasses = kKeys / kRowsPerPass / Team; // of one warp
  // Passes at once for tiles of several pages: all for large tiles (pages of 8
  // keys, 64 ragged sequences of up to 8192: f32 of 128, 16 heads over 4, 174 us,
  // 178 with four; of 96, 48 over 4, 189 and 199; bf16 of 256, 32 over 4, 164 and
  // 168), four where that code is in the way of the rest (pages of 64: bf16 of 128,
  // 128 over 8, 131 us instead of 133; of 256, 64 over 4, 146 instead of 149). Of the
  // large tiles f32 teams of 128 alone lose by it, 258 and 245 us.
  static constexpr int kScatteredPasses = kRowBytes > 256u && (kWide || Team == 1) ? 16 : 4;
  static constexpr uint32_t kKeyTiles = kKeys / 16u;
  static constexpr uint32_t kSteps = Dim * sizeof(T) / 32u; // of Q K^T (32 bytes of a row)
  static constexpr uint32_t kStages = attention_stages(Dim, kRowBytes, kHeads);
  static constexpr uint32_t kStageBytes = attention_tile_bytes(kRowBytes);
  static constexpr uint32_t kStateFloats = attention_state_floats(Dim, kHeads);
  static constexpr uint32_t kStateRow = Dim + 4u;           // floats of a head in a state
  static constexpr uint32_t kMaximaAt = kHeads * kStateRow; // then the sums
  static_assert(Team == attention_team(kRowBytes, kHeads), "warps of a unit");
  static_assert(kChunks >= 8 && kChunks <= 32 && kKeys >= 16 && kKeys <= 32, "tile shape");

  // A row's chunk c is stored at c xor (row & 7): eight rows of a chunk column
  // then lie in different banks.
  static __device__ __forceinline__ uint32_t swizzled(uint32_t row, uint32_t chunk) {
    return row * kRowBytes + ((chunk ^ (row & 7u)) << 4u);
  }

  struct Piece { // of a row that a unit leaves unfinished
    uint32_t row_begin, row_end; // the places of the row's tiles
    uint32_t sequence, row, present;
  };
  struct HeadBlock {
    uint32_t first, count; // query heads of a row
  };

  const PagedAttentionArgs &args_;
  const uint32_t lane_ = threadIdx.x & 31u, warp_ = threadIdx.x >> 5u;
  const uint32_t unit_ = warp_ / Team, member_ = warp_ % Team;
  uint32_t ring_;          // this unit's stages
  unsigned char *rings_;   // all units'; at the end, the states of their last pieces
  float *states_;          // shared: [kUnits] of the pieces that began before the unit's part
  Piece *firsts_, *lasts_; // [kUnits] of either kind
  uint32_t *starts_;       // [kThreads] places before each thread's share; where states will be
  uint32_t *seen_;         // [kStages] which keys of this unit's stages have a page
  uint32_t *flags_;        // [2] whether the block joins its first, its last row

  uint32_t query_[HeadTiles][kSteps][kWide ? 4 : 2];
  float out_[HeadTiles][Dim / 16][4];
  float maximum_[HeadTiles][2], sum_[HeadTiles][2];

  // The unit's warps.
  __device__ __forceinline__ void unit_sync() const {
    if constexpr (Team == 1) {
      __syncwarp();
    } else {
      asm volatile("barrier.sync %0, %1;" ::"r"(1u + unit_), "n"(32 * Team) : "memory");
    }
  }
  // A head of this warp's, among the block's.
  __device__ __forceinline__ uint32_t head_at(int n) const {
    return Team == 1 ? n * 8u : member_ * (8u * HeadTiles) + n * 8u;
  }

  __device__ __forceinline__ uint32_t tiles_of(const Span &span) const {
    return (span.end - span.begin + kKeys - 1u) / kKeys;
  }

  // The next sequence with tiles; the caller knows that there is one.
  __device__ __forceinline__ void enter_sequence(TileCursor &at) const {
    while (true) {
      at.span = span_of(args_, at.sequence);
      at.tiles = tiles_of(at.span);
      if (at.tiles != 0 || at.sequence + 1u >= args_.table.rows) {
        return;
      }
      ++at.sequence;
    }
  }
  __device__ __forceinline__ void next_row(TileCursor &at) const {
    at.tile = 0;
    if (++at.row == args_.rows_per_sequence) {
      at.row = 0;
      ++at.sequence;
      enter_sequence(at);
    }
  }

  __device__ __forceinline__ HeadBlock heads_of(uint32_t row) const {
    const uint32_t kv_head = row / args_.head_blocks;
    const uint32_t at = (row - kv_head * args_.head_blocks) * kHeads;
    return {kv_head * args_.group + at, min(kHeads, args_.group - at)};
  }

  // Where a tile's keys are, one per lane (twice over with 16 of them).
  struct Gather {
    int32_t page; // -1: none
    uint32_t row, head;
  };
  __device__ __forceinline__ Gather locate(const TileCursor &at) const {
    Gather gather{-1, 0, at.row / args_.head_blocks};
    const uint32_t key = at.span.begin + at.tile * kKeys + (lane_ & (kKeys - 1u));
    if (key < at.span.end) {
      const uint32_t column = args_.cache.page.quotient(key);
      gather.row = key - column * args_.cache.page.divisor;
      gather.page = args_.table.pages[at.sequence * args_.table.row_stride + column];
    }
    return gather;
  }

  // A pass copies kRowsPerPass rows of keys and values. Where a tile lies in one
  // page, rows are a stride apart; otherwise every lane works out the addresses
  // of its key and value, and passes take them from those lanes.
  __device__ __forceinline__ void issue(const Gather &gather, uint32_t stage) const {
    const bool present = static_cast<uint32_t>(gather.page) < args_.cache.page_count;
    const uint32_t seen = __ballot_sync(kAllLanes, present);
    if (lane_ == 0) {
      seen_[stage] = seen;
    }
    const uint32_t page = present ? gather.page : 0u; // nothing is read there, zeros are written
    const Pages &k = args_.cache.keys, &v = args_.cache.values;
    const uint32_t chunk = lane_ % kChunks;
    const uint32_t row_of_pass = lane_ / kChunks + member_ * (kPasses * kRowsPerPass);
    const bool inside = chunk * (16u / sizeof(T)) < args_.head_dim;
    const uint32_t offset = inside ? chunk * 16u : 0u;
    const uint32_t wanted = inside ? seen >> row_of_pass : 0u;
    const uint32_t to = ring_ + stage * kStageBytes;
    const uint32_t first_page = __shfl_sync(kAllLanes, page, 0);
    const uint32_t first_row = __shfl_sync(kAllLanes, gather.row, 0);
    const bool follows =
        page == first_page && gather.row == first_row + (lane_ & (kKeys - 1u));
    if (__all_sync(kAllLanes, follows || !present)) {
      const uint32_t row = first_row + row_of_pass;
      uint64_t key = reinterpret_cast<uint64_t>(static_cast<const T *>(k.data) +
                                                k.offset(first_page, row, gather.head)) + offset;
      uint64_t value = reinterpret_cast<uint64_t>(static_cast<const T *>(v.data) +
                                                  v.offset(first_page, row, gather.head)) + offset;
      const int64_t key_step = int64_t{k.token_stride} * (kRowsPerPass * sizeof(T));
      const int64_t value_step = int64_t{v.token_stride} * (kRowsPerPass * sizeof(T));
#pragma unroll
      for (uint32_t pass = 0; pass < kPasses; ++pass) {
        const uint32_t at = to + swizzled(pass * kRowsPerPass + row_of_pass, chunk);
        const bool valid = (wanted >> pass * kRowsPerPass & 1u) != 0;
        if (chunk < Dim * sizeof(T) / 16u) {
          copy_16(at, key, valid);
          copy_16(at + kStageBytes / 2u, value, valid);
        }
        key += key_step;
        value += value_step;
      }
    } else {
      const T *key = static_cast<const T *>(k.data) + k.offset(page, gather.row, gather.head);
      const T *value = static_cast<const T *>(v.data) + v.offset(page, gather.row, gather.head);
#pragma unroll kScatteredPasses
      for (uint32_t pass = 0; pass < kPasses; ++pass) {
        const uint32_t row = pass * kRowsPerPass + row_of_pass;
        const uint64_t key_row =
            __shfl_sync(kAllLanes, reinterpret_cast<uint64_t>(key), row) + offset;
        const uint64_t value_row =
            __shfl_sync(kAllLanes, reinterpret_cast<uint64_t>(value), row) + offset;
        const bool valid = (wanted >> pass * kRowsPerPass & 1u) != 0;
        const uint32_t at = to + swizzled(row, chunk);
        if (chunk < Dim * sizeof(T) / 16u) {
          copy_16(at, key_row, valid);
          copy_16(at + kStageBytes / 2u, value_row, valid);
        }
      }
    }
  }

  // The query heads of a row, as the products' second operand: of 16-bit
  // elements pairs, which may lie at odd places (`Paired` false).
  template <bool Paired>
  __device__ __forceinline__ void load_queries(uint32_t sequence, uint32_t first_head,
                                               uint32_t heads) {
#pragma unroll
    for (int n = 0; n < HeadTiles; ++n) {
      const uint32_t head = head_at(n) + lane_ / 4u;
      const T *q = static_cast<const T *>(args_.q.data) +
                   args_.q.offset(sequence, first_head + min(head, heads - 1u));
      const uint32_t limit = head < heads ? args_.head_dim : 0u;
#pragma unroll
      for (uint32_t k = 0; k < kSteps; ++k) {
#pragma unroll
        for (uint32_t half = 0; half < 2u; ++half) {
          if constexpr (kWide) {
            const uint32_t d = k * 8u + half * 4u + (lane_ & 3u);
            query_[n][k][half] = d < limit ? __float_as_uint(q[d]) : 0u;
          } else {
            const uint32_t d = k * 16u + half * 8u + (lane_ & 3u) * 2u;
            if constexpr (Paired) {
              query_[n][k][half] = d < limit ? *reinterpret_cast<const uint32_t *>(q + d) : 0u;
            } else {
              uint16_t low = 0, high = 0;
              if (d < limit) {
                memcpy(&low, q + d, 2);
                memcpy(&high, q + d + 1u, 2);
              }
              query_[n][k][half] = uint32_t{low} | uint32_t{high} << 16;
            }
          }
        }
      }
    }
    if constexpr (kWide) {
#pragma unroll
      for (int n = 0; n < HeadTiles; ++n) {
#pragma unroll
        for (uint32_t k = 0; k < kSteps; ++k) {
#pragma unroll
          for (uint32_t half = 0; half < 2u; ++half) {
            split_tf32(query_[n][k][half], query_[n][k][half], query_[n][k][2u + half]);
          }
        }
      }
    }
  }

  __device__ __forceinline__ void begin_row(uint32_t sequence, uint32_t first_head,
                                            uint32_t heads) {
    if (kWide || args_.paired_queries != 0) {
      load_queries<true>(sequence, first_head, heads);
    } else {
      load_queries<false>(sequence, first_head, heads);
    }
#pragma unroll
    for (int n = 0; n < HeadTiles; ++n) {
#pragma unroll
      for (int m = 0; m < Dim / 16; ++m) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          out_[n][m][i] = 0.0f;
        }
      }
      maximum_[n][0] = maximum_[n][1] = -INFINITY;
      sum_[n][0] = sum_[n][1] = 0.0f;
    }
  }

  // The product of a query and a key of the tile at `keys`, by 32-bit arithmetic.
  static __device__ __noinline__ float whole_score(const PagedAttentionArgs &args, uint32_t keys,
                                                   uint32_t key, uint32_t sequence,
                                                   uint32_t first_head, uint32_t head,
                                                   uint32_t heads) {
    float sum = 0.0f;
    if (head < heads) {
      const T *q =
          static_cast<const T *>(args.q.data) + args.q.offset(sequence, first_head + head);
#pragma unroll 1
      for (uint32_t d = 0; d < args.head_dim; ++d) {
        const uint32_t word = load_shared(keys + swizzled(key, d / 4u) + (d & 3u) * 4u);
        sum = fmaf(to_float(q[d]), __uint_as_float(word), sum);
      }
    }
    return sum;
  }

  // One tile of keys: scores, weights and weighted values. Score registers
  // i of a 16 x 8 tile: key lane / 4 + (i / 2) * 8, head (lane % 4) * 2 + i % 2.
  __device__ __forceinline__ void compute(uint32_t stage, uint32_t first_key, uint32_t end,
                                          uint32_t sequence, uint32_t first_head,
                                          uint32_t heads) {
    const uint32_t keys = ring_ + stage * kStageBytes;
    const uint32_t values = keys + kStageBytes / 2u;
    float slope[HeadTiles][2]; // under way before the products; 0 without a bias
#pragma unroll
    for (int n = 0; n < HeadTiles; ++n) {
#pragma unroll
      for (uint32_t i = 0; i < 2u; ++i) {
        const uint32_t head = head_at(n) + (lane_ & 3u) * 2u + i;
        slope[n][i] =
            args_.slopes != nullptr && head < heads ? args_.slopes[first_head + head] : 0.0f;
      }
    }
    float score[HeadTiles][kKeyTiles][4];
#pragma unroll
    for (uint32_t m = 0; m < kKeyTiles; ++m) {
#pragma unroll
      for (int n = 0; n < HeadTiles; ++n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          score[n][m][i] = 0.0f;
        }
      }
      const uint32_t row = m * 16u + (lane_ & 15u);
#pragma unroll
      for (uint32_t k = 0; k < kSteps; ++k) {
        uint32_t a[4];
        load_matrices(a, keys + swizzled(row, 2u * k + (lane_ >> 4u)));
        if constexpr (kWide) {
          uint32_t high[4], low[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            split_tf32(a[i], high[i], low[i]);
          }
          // The tensor cores' sums drop the bits below the larger operand's
          // last: each step's products are summed there, and the steps in
          // rounded 32 bits.
#pragma unroll
          for (int n = 0; n < HeadTiles; ++n) {
            float part[4];
            multiply_first(part, low, query_[n][k][0], query_[n][k][1], T());
            multiply(part, high, query_[n][k][2], query_[n][k][3], T());
            multiply(part, high, query_[n][k][0], query_[n][k][1], T());
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              score[n][m][i] += part[i];
            }
          }
        } else {
#pragma unroll
          for (int n = 0; n < HeadTiles; ++n) {
            multiply(score[n][m], a, query_[n][k][0], query_[n][k][1], T());
          }
        }
      }
    }
    if constexpr (kWide) {
      // The two parts of an infinity, or of a number that rounds to one, make a
      // NaN: such scores are summed anew from the numbers themselves.
      bool finite = true;
#pragma unroll
      for (int n = 0; n < HeadTiles; ++n) {
#pragma unroll
        for (uint32_t m = 0; m < kKeyTiles; ++m) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            finite = finite && fabsf(score[n][m][i]) < INFINITY;
          }
        }
      }
      if (!__all_sync(kAllLanes, finite)) {
#pragma unroll
        for (int n = 0; n < HeadTiles; ++n) {
#pragma unroll
          for (uint32_t m = 0; m < kKeyTiles; ++m) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              score[n][m][i] = whole_score(args_, keys, m * 16u + (i / 2) * 8u + lane_ / 4u,
                                           sequence, first_head,
                                           head_at(n) + (lane_ & 3u) * 2u + i % 2, heads);
            }
          }
        }
        __syncwarp();
      }
    }
    const uint32_t seen = seen_[stage];
    const bool capped = args_.softcap > 0.0f;
    const float to_base_2 = (capped ? args_.softcap : args_.scale) * kLog2E;
    const float to_cap = capped ? args_.scale / args_.softcap : 0.0f;
    if (capped) {
      // All types alike: 1 - 2 / (1 + e^2x) by one exponential took 97 us where this
      // takes 100 (64 ragged sequences of up to 4096 keys, 128 heads over 8 of 128
      // in f16), and lost what a cap far above the scores leaves of them.
#pragma unroll
      for (int n = 0; n < HeadTiles; ++n) {
#pragma unroll
        for (uint32_t m = 0; m < kKeyTiles; ++m) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            score[n][m][i] = tanhf(score[n][m][i] * to_cap);
          }
        }
      }
    }
#pragma unroll
    for (int n = 0; n < HeadTiles; ++n) {
      float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (uint32_t m = 0; m < kKeyTiles; ++m) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t key = m * 16u + (i / 2) * 8u + lane_ / 4u;
          float s = score[n][m][i] * to_base_2;
          if (args_.slopes != nullptr) {
            const int32_t distance = static_cast<int32_t>(end - 1u - first_key - key);
            s -= slope[n][i % 2] * kLog2E * static_cast<float>(distance);
          }
          s = (seen >> key & 1u) != 0 ? s : -INFINITY;
          score[n][m][i] = s;
          top[i % 2] = fmaxf(top[i % 2], s);
        }
      }
      bool rescale = false;
      float factor[2], base[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (uint32_t offset = 4; offset < 32u; offset <<= 1u) {
          top[i] = fmaxf(top[i], __shfl_xor_sync(kAllLanes, top[i], offset));
        }
        const float now = fmaxf(maximum_[n][i], top[i]);
        base[i] = now == -INFINITY ? 0.0f : now;
        factor[i] = exp2_fast(maximum_[n][i] - base[i]);
        rescale = rescale || now != maximum_[n][i];
        maximum_[n][i] = now;
      }
      if (__any_sync(kAllLanes, rescale)) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          sum_[n][i] *= factor[i];
        }
#pragma unroll
        for (int m = 0; m < Dim / 16; ++m) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            out_[n][m][i] *= factor[i % 2];
          }
        }
      }
#pragma unroll
      for (uint32_t m = 0; m < kKeyTiles; ++m) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float p = exp2_fast(score[n][m][i] - (base[i % 2] - kWeightBits<T>));
          score[n][m][i] = p;
          sum_[n][i % 2] += p;
        }
      }
    }
    // O^T += V^T P^T. The weights are transposed in registers: a lane then
    // holds head lane / 4 and keys (lane % 4) * 2, + 1 of eight. A tile's products
    // are summed by themselves, the tiles in rounded 32 bits: the tensor cores' sums
    // drop the bits below the last of the sum so far, and a row of 100000 keys
    // that one warp summed there came out 5e-4 too small.
    if constexpr (kWide) {
#pragma unroll
      for (uint32_t m = 0; m < kKeyTiles; ++m) {
#pragma unroll
        for (uint32_t part = 0; part < 2u; ++part) { // eight keys a product
          uint32_t weight[HeadTiles][4]; // high, high, low, low of the two keys
#pragma unroll
          for (int n = 0; n < HeadTiles; ++n) {
            const uint32_t x = __float_as_uint(score[n][m][2u * part]);
            const uint32_t y = __float_as_uint(score[n][m][2u * part + 1u]);
            const uint32_t lows = transpose_matrix(__byte_perm(x, y, 0x5410));
            const uint32_t highs = transpose_matrix(__byte_perm(x, y, 0x7632));
            split_weight_tf32(__byte_perm(lows, highs, 0x5410), weight[n][0], weight[n][2]);
            split_weight_tf32(__byte_perm(lows, highs, 0x7632), weight[n][1], weight[n][3]);
          }
          // Column k of the product is key 2 k, and column k + 4 key 2 k + 1.
          const uint32_t key = m * 16u + part * 8u + (lane_ & 3u) * 2u;
#pragma unroll
          for (int d = 0; d < Dim / 16; ++d) {
            uint32_t high[4], low[4];
#pragma unroll
            for (uint32_t i = 0; i < 4u; ++i) {
              const uint32_t column = d * 16u + (i & 1u) * 8u + lane_ / 4u;
              const uint32_t word = load_shared(values + swizzled(key + (i >> 1u), column / 4u) +
                                                (column & 3u) * 4u);
              split_value_tf32(word, high[i], low[i]);
            }
#pragma unroll
            for (int n = 0; n < HeadTiles; ++n) {
              float part[4];
              multiply_first(part, low, weight[n][0], weight[n][1], T());
              multiply(part, high, weight[n][2], weight[n][3], T());
              multiply(part, high, weight[n][0], weight[n][1], T());
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                out_[n][d][i] += part[i];
              }
            }
          }
        }
      }
    } else {
      uint32_t weight[kKeyTiles][HeadTiles][4]; // high of keys 0-7 and 8-15, low of them
#pragma unroll
      for (uint32_t m = 0; m < kKeyTiles; ++m) {
#pragma unroll
        for (int n = 0; n < HeadTiles; ++n) {
#pragma unroll
          for (uint32_t part = 0; part < 2u; ++part) {
            uint32_t high, low;
            split_weights(score[n][m][2u * part], score[n][m][2u * part + 1u], high, low, T());
            weight[m][n][part] = transpose_matrix(high);
            weight[m][n][2u + part] = transpose_matrix(low);
          }
        }
      }
      const uint32_t row = (lane_ >> 4u) * 8u + (lane_ & 7u);
#pragma unroll
      for (int d = 0; d < Dim / 16; ++d) {
        float part[HeadTiles][4];
#pragma unroll
        for (uint32_t m = 0; m < kKeyTiles; ++m) {
          uint32_t a[4];
          load_matrices_transposed(
              a, values + swizzled(m * 16u + row, 2u * d + (lane_ >> 3u & 1u)));
#pragma unroll
          for (int n = 0; n < HeadTiles; ++n) {
            if (m == 0) {
              multiply_first(part[n], a, weight[m][n][2], weight[m][n][3], T());
            } else {
              multiply(part[n], a, weight[m][n][2], weight[m][n][3], T());
            }
            multiply(part[n], a, weight[m][n][0], weight[m][n][1], T());
          }
        }
#pragma unroll
        for (int n = 0; n < HeadTiles; ++n) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            out_[n][d][i] += part[n][i];
          }
        }
      }
    }
  }

  // The sums over a warp's lanes; afterwards every lane has those of its heads.
  __device__ __forceinline__ void sum_lanes() {
#pragma unroll
    for (int n = 0; n < HeadTiles; ++n) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (uint32_t offset = 4; offset < 32u; offset <<= 1u) {
          sum_[n][i] += __shfl_xor_sync(kAllLanes, sum_[n][i], offset);
        }
      }
    }
  }

  // A sum of 0 is that of a row that sees no token: the largest weight is
  // 2^kWeightBits. Where all scores are NaN the maximum is -infinity too.
  __device__ __forceinline__ void write_lse(uint32_t sequence, uint32_t head, float top,
                                            float sum) const {
    if (args_.lse != nullptr) {
      args_.lse[uint64_t{sequence} * args_.heads + head] =
          sum == 0.0f ? -INFINITY : (top + (log2f(sum) - kWeightBits<T>)) * kLn2;
    }
  }

  // A row that this warp has all of.
  __device__ __forceinline__ void finish_row(uint32_t sequence, uint32_t first_head,
                                             uint32_t heads) const {
#pragma unroll
    for (int n = 0; n < HeadTiles; ++n) {
#pragma unroll
      for (uint32_t i = 0; i < 2u; ++i) {
        const uint32_t head = head_at(n) + (lane_ & 3u) * 2u + i;
        if (head >= heads) {
          continue;
        }
        const float top = maximum_[n][i];
        const float inverse = sum_[n][i] == 0.0f ? 0.0f : 1.0f / sum_[n][i];
        T *out = static_cast<T *>(args_.out.data) +
                 args_.out.offset(sequence, first_head + head);
#pragma unroll
        for (uint32_t d = 0; d < Dim / 16u; ++d) {
#pragma unroll
          for (uint32_t half = 0; half < 2u; ++half) {
            const uint32_t column = d * 16u + half * 8u + lane_ / 4u;
            if (column < args_.head_dim) {
              out[column] = from_float<T>(out_[n][d][2u * half + i] * inverse);
            }
          }
        }
        if (lane_ < 4u) {
          write_lse(sequence, first_head + head, top, sum_[n][i]);
        }
      }
    }
  }

  __device__ __forceinline__ void save_state(float *state) const {
#pragma unroll
    for (int n = 0; n < HeadTiles; ++n) {
#pragma unroll
      for (uint32_t i = 0; i < 4u; ++i) {
        const uint32_t head = head_at(n) + (lane_ & 3u) * 2u + (i & 1u);
#pragma unroll
        for (uint32_t d = 0; d < Dim / 16u; ++d) {
          state[head * kStateRow + d * 16u + (i >> 1u) * 8u + lane_ / 4u] = out_[n][d][i];
        }
        if (lane_ < 4u && i < 2u) {
          state[kMaximaAt + head] = maximum_[n][i];
          state[kMaximaAt + kHeads + head] = sum_[n][i];
        }
      }
    }
  }

  // Four columns of a head, joined from several states: unscaled, with their
  // maximum and sum.
  struct Joined {
    float4 x;
    float top, sum;

    __device__ __forceinline__ void add_state(const float *state, uint32_t head,
                                              uint32_t column) {
      const float other = state[kMaximaAt + head];
      const float other_sum = state[kMaximaAt + kHeads + head];
      const float4 y = *reinterpret_cast<const float4 *>(state + head * kStateRow + column);
      const float now = fmaxf(top, other);
      const float base = now == -INFINITY ? 0.0f : now;
      const float mine = exp2_fast(top - base), theirs = exp2_fast(other - base);
      x = {x.x * mine + y.x * theirs, x.y * mine + y.y * theirs, x.z * mine + y.z * theirs,
           x.w * mine + y.w * theirs};
      sum = sum * mine + other_sum * theirs;
      top = now;
    }
  };

  __device__ __forceinline__ void finish(uint32_t sequence, uint32_t head, uint32_t column,
                                         const Joined &joined) const {
    const float inverse = joined.sum == 0.0f ? 0.0f : 1.0f / joined.sum;
    T *out = static_cast<T *>(args_.out.data) + args_.out.offset(sequence, head);
    const float x[4] = {joined.x.x, joined.x.y, joined.x.z, joined.x.w};
#pragma unroll
    for (uint32_t i = 0; i < 4u; ++i) {
      if (column + i < args_.head_dim) {
        out[column + i] = from_float<T>(x[i] * inverse);
      }
    }
    if (column == 0) {
      write_lse(sequence, head, joined.top, joined.sum);
    }
  }

  // The pieces of one row that the block's units left, from `unit` on: its
  // last one, or its first for a row from before the block. A row that other
  // blocks have a part of goes to `part`. By `threads` threads, this one the
  // `thread`th.
  __device__ __forceinline__ void join_pieces(const Piece &piece, uint32_t unit, bool from_last,
                                              float *part, uint32_t thread, uint32_t threads) {
    uint32_t count = 1;
    while (unit + count < kUnits && firsts_[unit + count].present != 0 &&
           firsts_[unit + count].row_begin == piece.row_begin) {
      ++count;
    }
    const float *first_state =
        from_last ? reinterpret_cast<const float *>(rings_ + unit * kStages * kStageBytes)
                  : states_ + unit * kStateFloats;
    const HeadBlock heads = heads_of(piece.row);
#pragma unroll 1
    for (uint32_t at = thread * 4u; at < heads.count * Dim; at += threads * 4u) {
      const uint32_t head = at / Dim, column = at % Dim;
      Joined joined{{0.0f, 0.0f, 0.0f, 0.0f}, -INFINITY, 0.0f};
      const float *state = first_state;
#pragma unroll 2
      for (uint32_t i = 0; i < count; ++i) {
        joined.add_state(state, head, column);
        state = states_ + (unit + i + 1u) * kStateFloats;
      }
      if (part == nullptr) {
        finish(piece.sequence, heads.first + head, column, joined);
      } else {
        *reinterpret_cast<float4 *>(part + head * kStateRow + column) = joined.x;
        if (column == 0) {
          part[kMaximaAt + head] = joined.top;
          part[kMaximaAt + kHeads + head] = joined.sum;
        }
      }
    }
  }

  // The state that block `block` leaves of a row of several: its last where
  // the row begins in it, else its first.
  __device__ __forceinline__ float *part_of(uint32_t block, bool begins) const {
    return args_.states + (2u * size_t{block} + (begins ? 1u : 0u)) * kStateFloats;
  }

  __device__ __forceinline__ uint32_t parts_of(const Piece &piece, uint32_t per_block) const {
    return (piece.row_end - 1u) / per_block - piece.row_begin / per_block + 1u;
  }

  // The parts that the blocks left of a row, all of them there by now: brought
  // into the rings, which are free, as many at a time as these hold.
  __device__ __forceinline__ void join_parts(const Piece &piece, uint32_t per_block) const {
    const uint32_t first = piece.row_begin / per_block, count = parts_of(piece, per_block);
    const HeadBlock heads = heads_of(piece.row);
    constexpr uint32_t kRound = kUnits * kStages * kStageBytes / (4u * kStateFloats);
    constexpr uint32_t kItems = kHeads * Dim / 4u;
    constexpr uint32_t kEach = (kItems + kThreads - 1u) / kThreads;
    const float *staged = reinterpret_cast<const float *>(rings_);
    Joined joined[kEach];
#pragma unroll
    for (uint32_t j = 0; j < kEach; ++j) {
      joined[j] = {{0.0f, 0.0f, 0.0f, 0.0f}, -INFINITY, 0.0f};
    }
#pragma unroll 1
    for (uint32_t begin = 0; begin < count; begin += kRound) {
      const uint32_t now = min(kRound, count - begin);
#pragma unroll 1
      for (uint32_t i = warp_; i < now; i += kWarps) {
        const uint64_t from =
            reinterpret_cast<uint64_t>(part_of(first + begin + i, begin + i == 0));
        const uint32_t to = shared_address(staged + i * kStateFloats);
#pragma unroll 4
        for (uint32_t at = lane_; at < kStateFloats / 4u; at += 32u) {
          copy_16(to + at * 16u, from + at * 16u, true);
        }
      }
      commit_copies();
      wait_copies<0>();
      __syncthreads();
#pragma unroll
      for (uint32_t j = 0; j < kEach; ++j) {
        const uint32_t at = (threadIdx.x + j * kThreads) * 4u;
        if (at < heads.count * Dim) {
#pragma unroll 4
          for (uint32_t i = 0; i < now; ++i) {
            joined[j].add_state(staged + i * kStateFloats, at / Dim, at % Dim);
          }
        }
      }
      __syncthreads();
    }
#pragma unroll
    for (uint32_t j = 0; j < kEach; ++j) {
      const uint32_t at = (threadIdx.x + j * kThreads) * 4u;
      if (at < heads.count * Dim) {
        finish(piece.sequence, heads.first + at / Dim, at % Dim, joined[j]);
      }
    }
  }

  // Where unit u's tiles begin: equal parts, empty ones at the end alone.
  static __device__ __forceinline__ uint32_t unit_part(uint32_t begin, uint32_t count,
                                                       uint32_t u) {
    return begin + count / kUnits * u + min(u, count % kUnits);
  }

  // Places: the tiles of all rows one after another, each row's followed by
  // kAttentionRowCost places that stand for the work a row takes besides its
  // tiles. Blocks and units take equal numbers of places.
  __device__ __forceinline__ uint32_t places_of(uint32_t sequence) const {
    const uint32_t tiles = tiles_of(span_of(args_, sequence));
    return tiles == 0 ? 0u : (tiles + kAttentionRowCost) * args_.rows_per_sequence;
  }

  // The sequence of a place and the places before it, from the sums before
  // each thread's share (in shared memory, at the start). For whole warps.
  struct Start {
    uint32_t sequence, before;
  };
  __device__ __forceinline__ Start find(uint32_t place, uint32_t share) const {
    constexpr uint32_t kEach = kThreads / 32u;
    // The last thread with no more than `place` before it: a group of threads
    // per lane, then the group's threads.
    const uint32_t groups = __ballot_sync(kAllLanes, starts_[lane_ * kEach] <= place);
    const uint32_t group = 31u - __clz(groups);
    const uint32_t threads =
        __ballot_sync(kAllLanes, lane_ < kEach && starts_[group * kEach + lane_ % kEach] <= place);
    const uint32_t thread = group * kEach + 31u - __clz(threads);
    Start start{thread * share, starts_[thread]};
#pragma unroll 1
    while (true) {
      const uint32_t places = places_of(start.sequence);
      if (place - start.before < places) {
        return start;
      }
      start.before += places;
      ++start.sequence;
    }
  }

  // The place where the next row begins, or this one where it is one.
  __device__ __forceinline__ uint32_t row_boundary(uint32_t place, uint32_t total,
                                                   uint32_t share) const {
    if (place >= total) {
      return total;
    }
    const Start start = find(place, share);
    const uint32_t row = tiles_of(span_of(args_, start.sequence)) + kAttentionRowCost;
    return start.before + (place - start.before + row - 1u) / row * row;
  }

  // A unit's tiles, between the places begin and end, each loaded kStages - 1
  // steps ahead, and their page numbers two more.
  __device__ __forceinline__ void run_unit(uint32_t begin, uint32_t end, const Start &start) {
    TileCursor at; // the tile to compute
    at.sequence = start.sequence;
    at.span = span_of(args_, at.sequence);
    at.tiles = tiles_of(at.span);
    at.row = (begin - start.before) / (at.tiles + kAttentionRowCost);
    uint32_t row_begin = start.before + at.row * (at.tiles + kAttentionRowCost);
    at.tile = begin - row_begin;
    uint32_t tile = begin; // the place of the tile to compute
    if (at.tile >= at.tiles) { // past the row's last
      tile = row_begin = row_begin + at.tiles + kAttentionRowCost;
      if (tile >= end) {
        return;
      }
      next_row(at);
    }
    uint32_t row_end = row_begin + at.tiles;
    TileCursor load_at = at;
    Gather gather = locate(load_at), gather_after = gather;
    // The tile to load and the one to look up, `ahead` the place of the latter;
    // past the end there are none.
    uint32_t ahead = tile;
    bool load = true, load_after = true;
    auto look_up = [&]() {
      if (load_after) {
        ++ahead;
        if (++load_at.tile == load_at.tiles) {
          ahead += kAttentionRowCost;
          if (ahead < end) {
            next_row(load_at);
          }
        }
        load_after = ahead < end;
        if (load_after) {
          gather_after = locate(load_at);
        }
      }
    };
    look_up();
    uint32_t load_stage = 0, stage = 0;
    HeadBlock heads = heads_of(at.row);
    bool entered = false;
#pragma unroll 1
    for (uint32_t step = 0; tile < end; ++step) {
      if (!entered && step + 1u >= kStages) { // the first tiles are under way before
        begin_row(at.sequence, heads.first, heads.count);
        entered = true;
      }
      if (load) {
        issue(gather, load_stage);
        gather = gather_after;
        load = load_after;
        look_up();
      }
      commit_copies();
      load_stage = load_stage + 1u == kStages ? 0u : load_stage + 1u;
      if (step + 1u < kStages) {
        continue; // not all stages are under way yet
      }
      wait_copies<kStages - 1>();
      unit_sync();
      compute(stage, at.span.begin + (tile - row_begin) * kKeys, at.span.end, at.sequence,
              heads.first, heads.count);
      unit_sync(); // the stage is filled again by the next issue
      stage = stage + 1u == kStages ? 0u : stage + 1u;
      ++tile;
      if (tile != row_end && tile != end) {
        continue;
      }
      sum_lanes();
      if (row_begin >= begin && row_end <= end) {
        finish_row(at.sequence, heads.first, heads.count);
      } else {
        // A row from before the unit's part is its first; one that goes on
        // past it is its last, and nothing is left to load then.
        const bool is_first = row_begin < begin;
        if (!is_first) {
          wait_copies<0>();
          unit_sync();
        }
        save_state(is_first ? states_ + unit_ * kStateFloats
                            : reinterpret_cast<float *>(rings_ + unit_ * kStages * kStageBytes));
        if (lane_ == 0 && member_ == 0) {
          (is_first ? firsts_ : lasts_)[unit_] = {row_begin, row_end, at.sequence, at.row, 1u};
        }
      }
      if (tile != row_end) {
        break; // the row goes on past the end
      }
      tile = row_begin = row_end + kAttentionRowCost;
      if (tile < end) {
        next_row(at);
        row_end = row_begin + at.tiles;
        heads = heads_of(at.row);
        entered = false;
      }
    }
    wait_copies<0>();
  }

public:
  static constexpr uint32_t kThreads = 32u * kWarps;

  __device__ __forceinline__ PagedAttention(const PagedAttentionArgs &args, unsigned char *shared)
      : args_(args) {
    rings_ = shared;
    ring_ = shared_address(shared) + unit_ * kStages * kStageBytes;
    unsigned char *at = shared + kUnits * kStages * kStageBytes;
    states_ = reinterpret_cast<float *>(at);
    at += 4u * kUnits * kStateFloats;
    firsts_ = reinterpret_cast<Piece *>(at);
    lasts_ = firsts_ + kUnits;
    starts_ = reinterpret_cast<uint32_t *>(states_);
    seen_ = reinterpret_cast<uint32_t *>(lasts_ + kUnits) + unit_ * kStages;
    flags_ = reinterpret_cast<uint32_t *>(lasts_ + kUnits) + kUnits * kStages;
    static_assert(2u * sizeof(Piece) * kUnits + 4u * kStages * kUnits + 8u <= 1024u &&
                      kThreads + 2u * kWarps <= kUnits * kStateFloats,
                  "shared memory of the bookkeeping");
  }

  __device__ __forceinline__ void run() {
    // Places before each thread's share of the sequences, and all of them.
    const uint32_t share = (args_.table.rows + kThreads - 1u) / kThreads;
    const uint32_t mine_begin = min(threadIdx.x * share, args_.table.rows);
    const uint32_t mine_end = min(mine_begin + share, args_.table.rows);
    uint32_t mine = 0;
#pragma unroll 1
    for (uint32_t s = mine_begin; s < mine_end; ++s) {
      mine += places_of(s);
    }
    uint32_t upto = mine, most = mine; // inclusive sums; places of the sequence with most
#pragma unroll
    for (uint32_t offset = 1; offset < 32u; offset <<= 1u) {
      const uint32_t other = __shfl_up_sync(kAllLanes, upto, offset);
      upto += lane_ >= offset ? other : 0u;
      most = max(most, __shfl_xor_sync(kAllLanes, most, offset));
    }
    uint32_t *warp_sums = starts_ + kThreads;
    if (lane_ == 31u) {
      warp_sums[warp_] = upto;
      warp_sums[kWarps + warp_] = most;
      firsts_[unit_].present = 0;
      lasts_[unit_].present = 0;
    }
    __syncthreads();
    uint32_t before = upto - mine, total = 0;
#pragma unroll
    for (uint32_t w = 0; w < kWarps; ++w) {
      const uint32_t sum = warp_sums[w];
      before += w < warp_ ? sum : 0u;
      total += sum;
      most = max(most, warp_sums[kWarps + w]);
    }
    starts_[threadIdx.x] = before;
    __syncthreads();
    const uint32_t per_block =
        max((total + gridDim.x - 1u) / gridDim.x, kAttentionMinimumTiles);
    uint32_t begin = min(blockIdx.x * per_block, total);
    uint32_t end = min(begin + per_block, total);
    const uint32_t whole_tiles =
        2u * args_.table.rows * args_.rows_per_sequence >= gridDim.x ? kAttentionWholeTilesMany
                                                                     : kAttentionWholeTilesFew;
    if (share == 1u && most <= (whole_tiles + kAttentionRowCost) * args_.rows_per_sequence) {
      begin = row_boundary(begin, total, share);
      end = row_boundary(end, total, share);
    }
    const uint32_t count = end - begin;
    const uint32_t unit_begin = unit_part(begin, count, unit_);
    const uint32_t unit_end = unit_part(begin, count, unit_ + 1u);
    Start start{0, 0};
    if (unit_begin < unit_end) {
      start = find(unit_begin, share);
    }
    __syncthreads(); // the starts lie where states will
    if (unit_begin < unit_end) {
      run_unit(unit_begin, unit_end, start);
    }
    __syncthreads();
    // Rows from before the block (i = 0), then those that begin in unit i - 1:
    // one or two by all threads, more of them a warp each.
    const uint32_t present = __ballot_sync(
        kAllLanes, lane_ <= kUnits &&
                       (lane_ == 0 ? firsts_[0] : lasts_[lane_ - 1u]).present != 0);
    const bool by_warp = __popc(present) > 2;
    uint32_t go_on[2] = {kUnits + 1u, kUnits + 1u}; // those of other blocks too
    uint32_t turn = 0;
#pragma unroll 1
    for (uint32_t left = present; left != 0; left &= left - 1u, ++turn) {
      const uint32_t i = __ffs(left) - 1u;
      const Piece &piece = i == 0 ? firsts_[0] : lasts_[i - 1u];
      const bool begins = piece.row_begin >= begin;
      const bool whole = begins && piece.row_end <= end;
      if (!whole) {
        go_on[begins ? 1 : 0] = i;
      }
      if (!by_warp || turn % kWarps == warp_) {
        join_pieces(piece, i == 0 ? 0u : i - 1u, i != 0,
                    whole ? nullptr : part_of(blockIdx.x, begins),
                    by_warp ? lane_ : threadIdx.x, by_warp ? 32u : kThreads);
      }
    }
    // Where this block is the last to leave its part of a row, it joins them.
    __syncthreads();
    if (threadIdx.x < 2u) {
      const uint32_t i = threadIdx.x == 0 ? go_on[0] : go_on[1];
      uint32_t last = 0;
      if (i <= kUnits) {
        const Piece &piece = i == 0 ? firsts_[0] : lasts_[i - 1u];
        uint32_t *arrivals =
            args_.arrivals + size_t{piece.sequence} * args_.rows_per_sequence + piece.row;
        last = arrive(arrivals) + 1u == parts_of(piece, per_block) ? 1u : 0u;
        if (last != 0) {
          *arrivals = 0;
        }
      }
      flags_[threadIdx.x] = last;
    }
    __syncthreads();
#pragma unroll 1
    for (uint32_t which = 0; which < 2u; ++which) {
      if (flags_[which] != 0) {
        const uint32_t i = which == 0 ? go_on[0] : go_on[1];
        join_parts(i == 0 ? firsts_[0] : lasts_[i - 1u], per_block);
      }
    }
    // Rows of sequences that see nothing.
#pragma unroll 1
    for (uint32_t s = blockIdx.x; s < args_.table.rows; s += gridDim.x) {
      const Span span = span_of(args_, s);
      if (span.begin == span.end) {
        const Joined none{{0.0f, 0.0f, 0.0f, 0.0f}, -INFINITY, 0.0f};
#pragma unroll 1
        for (uint32_t at = threadIdx.x * 4u; at < args_.heads * Dim; at += kThreads * 4u) {
          finish(s, at / Dim, at % Dim, none);
        }
      }
    }
  }
};

} // namespace lrrt::ops

#endif // LRRT_PAGED_ATTENTION_CUH_
