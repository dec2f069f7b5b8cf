// Attention of one query row per sequence over a paged cache.
//
// One pass over the keys and values with a running maximum m and sum l of
// exp(s - m), in base 2; states of disjoint keys join as m = max(m1, m2),
// l = l1 2^(m1 - m) + l2 2^(m2 - m), and the weighted values likewise.
//
// Bound by reading the cache once. What the layout does about that:
//  - Every warp streams its own tiles (16 KB of keys and values) through three
//    shared-memory stages filled by cp.async, so a block's four warps keep
//    about 128 KB in flight without a barrier between them. Rows are gathered
//    through the page table, whose entries are read one tile ahead.
//  - The query heads of one key-value head share each row that is read: scores
//    are computed transposed, S^T = K Q^T, with 16 keys as the rows of the
//    matrix product and 8 query heads as its columns, and so are the outputs,
//    O^T = V^T P^T. One query row per head leaves nothing to fill the 128 rows
//    of a tcgen05 tile from the query side; these shapes (m16n8) waste none.
//    16-bit weights are split into two 16-bit parts, so that the probabilities
//    keep more than 16 bits; 32-bit operands into two TF32 parts (three
//    products).
//  - The tiles of all sequences and heads form one sequence that is cut into
//    equal parts for the blocks, whatever the lengths are. A block's first and
//    last row may be shared with its neighbours: it leaves its state in the
//    workspace, and the last block to arrive joins the states in the blocks'
//    order, so results do not depend on timing.
#ifndef LRRT_PAGED_ATTENTION_CUH_
#define LRRT_PAGED_ATTENTION_CUH_

#include "common.cuh"

namespace lrrt::ops {

__device__ __forceinline__ uint32_t shared_address(const void *pointer) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(pointer));
}

// 16 bytes from global to shared memory; zeros where `valid` is false.
__device__ __forceinline__ void copy_16(uint32_t to, const void *from, bool valid) {
  const uint32_t bytes = valid ? 16u : 0u;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void commit_copies() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int Pending> __device__ __forceinline__ void wait_copies() {
  asm volatile("cp.async.wait_group %0;" ::"n"(Pending) : "memory");
}

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

// x = high + low to about 22 bits, both TF32: high is x rounded to nearest
// (half away from zero) to 11 bits, low the exact rest, rounded likewise.
__device__ __forceinline__ void split_tf32(uint32_t bits, uint32_t &high, uint32_t &low) {
  high = (bits + 0x1000u) & 0xffffe000u;
  low = (__float_as_uint(__uint_as_float(bits) - __uint_as_float(high)) + 0x1000u) & 0xffffe000u;
}

// Two floats as a pair of 16-bit numbers, and what the rounding left over as
// another.
template <typename T>
__device__ __forceinline__ void split_16(float x, float y, uint32_t &high, uint32_t &low) {
  const T hx = from_float<T>(x), hy = from_float<T>(y);
  const T lx = from_float<T>(x - to_float(hx)), ly = from_float<T>(y - to_float(hy));
  uint16_t a, b;
  memcpy(&a, &hx, 2);
  memcpy(&b, &hy, 2);
  high = uint32_t{a} | uint32_t{b} << 16;
  memcpy(&a, &lx, 2);
  memcpy(&b, &ly, 2);
  low = uint32_t{a} | uint32_t{b} << 16;
}

// Which keys of a sequence a step sees, and in how many tiles.
struct Span {
  uint32_t begin, end;
};

__device__ __forceinline__ Span span_of(const PagedAttentionArgs &args, uint32_t sequence) {
  const int64_t capacity = int64_t{args.table.columns} * args.cache.page.divisor;
  int64_t end = args.lengths[sequence];
  end = end < 0 ? 0 : end > capacity ? capacity : end;
  const int64_t begin = args.window != 0 && end > args.window ? end - args.window : 0;
  return {static_cast<uint32_t>(begin), static_cast<uint32_t>(end)};
}

// A place in the sequence of tiles: rows (sequence, kv head, block of query
// heads) in order, each with the tiles of its sequence.
struct TileCursor {
  uint32_t sequence, row, tile; // row within the sequence; tile within the row
  uint32_t tiles;               // of the row
  Span span;
};

template <uint32_t KeysPerTile>
__device__ __forceinline__ void enter_sequence(const PagedAttentionArgs &args, TileCursor &at) {
  while (true) { // past empty sequences; the caller knows that tiles are left
    at.span = span_of(args, at.sequence);
    at.tiles = (at.span.end - at.span.begin + KeysPerTile - 1u) / KeysPerTile;
    if (at.tiles != 0 || at.sequence + 1u >= args.table.rows) {
      return;
    }
    ++at.sequence;
  }
}

template <uint32_t KeysPerTile>
__device__ __forceinline__ void advance(const PagedAttentionArgs &args, TileCursor &at,
                                        uint32_t tiles) {
  at.tile += tiles;
  while (at.tile >= at.tiles) {
    at.tile -= at.tiles;
    if (++at.row == args.rows_per_sequence) {
      at.row = 0;
      ++at.sequence;
      enter_sequence<KeysPerTile>(args, at);
    }
  }
}

template <typename T, int Dim, int HeadTiles> class PagedAttention {
  static constexpr bool kWide = sizeof(T) == 4; // 32-bit elements
  static constexpr uint32_t kRowBytes = Dim * sizeof(T);
  static constexpr uint32_t kWarps = attention_warps(kRowBytes);
  static constexpr uint32_t kKeys = attention_tile_keys(kRowBytes);
  static constexpr uint32_t kChunks = kRowBytes / 16u; // 16-byte chunks of a row
  static constexpr uint32_t kRowsPerPass = kChunks >= 32u ? 1u : 32u / kChunks;
  static constexpr uint32_t kKeyTiles = kKeys / 16u;
  static constexpr uint32_t kKeysPerLane = kKeys > 32u ? kKeys / 32u : 1u;
  static constexpr uint32_t kHeads = 8u * HeadTiles;
  static constexpr uint32_t kSteps = kRowBytes / 32u; // k steps of Q K^T (32 bytes of a row)
  static constexpr uint32_t kStages = kAttentionStages;
  static constexpr uint32_t kStageBytes = attention_tile_bytes(kRowBytes);
  static constexpr uint32_t kStateFloats = attention_state_floats(Dim, kHeads);
  static_assert(kChunks >= 8 && kChunks <= 32 && kKeys >= 16 && kKeys <= 64, "tile shape");

  // A row's chunk c is stored at c xor (row & 7): eight rows of a chunk column
  // then lie in different banks.
  static __device__ __forceinline__ uint32_t swizzled(uint32_t row, uint32_t chunk) {
    return row * kRowBytes + ((chunk ^ (row & 7u)) << 4u);
  }

  const PagedAttentionArgs &args_;
  const uint32_t lane_ = threadIdx.x & 31u, warp_ = threadIdx.x >> 5u;
  uint32_t ring_;           // this warp's stages
  uint64_t *seen_;          // [kStages] which keys of the stage have a page
  float *merge_;            // shared: states of 8 heads per warp
  float *merge_maxima_, *merge_sums_; // [warps][8]
  uint32_t *flag_;

  uint32_t query_[HeadTiles][kSteps][kWide ? 4 : 2];
  float out_[HeadTiles][Dim / 16][4];
  float maximum_[HeadTiles][2], sum_[HeadTiles][2];

  struct Gather {
    int64_t key[kKeysPerLane], value[kKeysPerLane]; // element offsets of a lane's keys
    bool valid[kKeysPerLane];
  };

  // Where the keys of a tile are, one or two of them per lane.
  __device__ __forceinline__ void locate(const TileCursor &at, Gather &gather) const {
    const uint32_t head = at.row / args_.head_blocks;
#pragma unroll
    for (uint32_t i = 0; i < kKeysPerLane; ++i) {
      const uint32_t key = at.span.begin + at.tile * kKeys + i * 32u + (lane_ & (kKeys - 1u));
      gather.valid[i] = key < at.span.end;
      gather.key[i] = 0;
      gather.value[i] = 0;
      if (gather.valid[i]) {
        const uint32_t column = args_.cache.page.quotient(key);
        const uint32_t row = key - column * args_.cache.page.divisor;
        const int32_t page = args_.table.pages[at.sequence * args_.table.row_stride + column];
        gather.valid[i] = page >= 0 && static_cast<uint32_t>(page) < args_.cache.page_count;
        if (gather.valid[i]) {
          gather.key[i] = page * args_.cache.key_page + row * args_.cache.key_token +
                          head * args_.cache.key_head;
          gather.value[i] = page * args_.cache.value_page + row * args_.cache.value_token +
                            head * args_.cache.value_head;
        }
      }
    }
  }

  __device__ __forceinline__ void issue(const Gather &gather, uint32_t stage) const {
    const uint32_t keys = ring_ + stage * kStageBytes;
    const uint32_t values = keys + kStageBytes / 2u;
    const uint32_t chunk = lane_ % kChunks;
    const bool inside = chunk * (16u / sizeof(T)) < args_.head_dim;
    const T *key_base = static_cast<const T *>(args_.cache.keys) + chunk * (16u / sizeof(T));
    const T *value_base = static_cast<const T *>(args_.cache.values) + chunk * (16u / sizeof(T));
    uint64_t seen = 0;
#pragma unroll
    for (uint32_t i = 0; i < kKeysPerLane; ++i) {
      seen |= uint64_t{__ballot_sync(kAllLanes, gather.valid[i])} << (32u * i);
    }
    if (lane_ == 0) {
      seen_[stage] = seen;
    }
#pragma unroll
    for (uint32_t pass = 0; pass < kKeys / kRowsPerPass; ++pass) {
      const uint32_t row = pass * kRowsPerPass + lane_ / kChunks;
      const uint32_t part = pass * kRowsPerPass / 32u; // which of a lane's keys
      const int64_t key = __shfl_sync(kAllLanes, gather.key[part], row & 31u);
      const int64_t value = __shfl_sync(kAllLanes, gather.value[part], row & 31u);
      const bool valid = inside && (seen >> row & 1u) != 0;
      const uint32_t at = swizzled(row, chunk);
      copy_16(keys + at, valid ? key_base + key : args_.cache.keys, valid);
      copy_16(values + at, valid ? value_base + value : args_.cache.values, valid);
    }
  }

  __device__ __forceinline__ void begin_row(uint32_t sequence, uint32_t first_head,
                                            uint32_t heads) {
#pragma unroll
    for (int n = 0; n < HeadTiles; ++n) {
      const uint32_t head = n * 8u + lane_ / 4u;
      const T *q = static_cast<const T *>(args_.q.data) + sequence * args_.q.row_stride +
                   (first_head + head) * args_.q.head_stride;
#pragma unroll
      for (uint32_t k = 0; k < kSteps; ++k) {
        if constexpr (kWide) {
#pragma unroll
          for (uint32_t half = 0; half < 2u; ++half) {
            const uint32_t d = k * 8u + half * 4u + (lane_ & 3u);
            const float x = head < heads && d < args_.head_dim ? q[d] : 0.0f;
            split_tf32(__float_as_uint(x), query_[n][k][half], query_[n][k][2u + half]);
          }
        } else {
#pragma unroll
          for (uint32_t half = 0; half < 2u; ++half) {
            const uint32_t d = k * 16u + half * 8u + (lane_ & 3u) * 2u;
            uint32_t pair = 0;
            if (head < heads && d < args_.head_dim) {
              uint16_t low, high;
              memcpy(&low, q + d, 2);
              memcpy(&high, q + d + 1u, 2);
              pair = uint32_t{low} | uint32_t{high} << 16;
            }
            query_[n][k][half] = pair;
          }
        }
      }
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

  // One tile of keys: scores, weights and weighted values. Score registers
  // i of a 16 x 8 tile: key lane / 4 + (i / 2) * 8, head (lane % 4) * 2 + i % 2.
  __device__ __forceinline__ void compute(uint32_t stage, uint32_t first_key, uint32_t end,
                                          uint32_t first_head, uint32_t heads) {
    const uint32_t keys = ring_ + stage * kStageBytes;
    const uint32_t values = keys + kStageBytes / 2u;
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
            float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            multiply(part, low, query_[n][k][0], query_[n][k][1], T());
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
    const uint64_t seen = seen_[stage];
    const float to_base_2 = args_.softcap > 0.0f ? args_.softcap * kLog2E : args_.scale * kLog2E;
    const float to_cap = args_.softcap > 0.0f ? args_.scale / args_.softcap : 0.0f;
#pragma unroll
    for (int n = 0; n < HeadTiles; ++n) {
      float slope[2] = {0.0f, 0.0f};
      if (args_.slopes != nullptr) {
#pragma unroll
        for (uint32_t i = 0; i < 2u; ++i) {
          const uint32_t head = n * 8u + (lane_ & 3u) * 2u + i;
          slope[i] = head < heads ? args_.slopes[first_head + head] * kLog2E : 0.0f;
        }
      }
      float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (uint32_t m = 0; m < kKeyTiles; ++m) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t key = m * 16u + (i / 2) * 8u + lane_ / 4u;
          float s = score[n][m][i];
          s = args_.softcap > 0.0f ? tanhf(s * to_cap) * to_base_2 : s * to_base_2;
          const int32_t distance = static_cast<int32_t>(end - 1u - first_key - key);
          s -= slope[i % 2] * static_cast<float>(distance);
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
          const float p = exp2_fast(score[n][m][i] - base[i % 2]);
          score[n][m][i] = p;
          sum_[n][i % 2] += p;
        }
      }
    }
    // O^T += V^T P^T. The weights are transposed in registers: a lane then
    // holds head lane / 4 and keys (lane % 4) * 2, + 1 of eight.
#pragma unroll
    for (uint32_t m = 0; m < kKeyTiles; ++m) {
      if constexpr (kWide) {
#pragma unroll
        for (uint32_t part = 0; part < 2u; ++part) { // eight keys a product
          uint32_t weight[HeadTiles][4]; // high, high, low, low of the two keys
#pragma unroll
          for (int n = 0; n < HeadTiles; ++n) {
            const uint32_t x = __float_as_uint(score[n][m][2u * part]);
            const uint32_t y = __float_as_uint(score[n][m][2u * part + 1u]);
            const uint32_t lows = transpose_matrix(__byte_perm(x, y, 0x5410));
            const uint32_t highs = transpose_matrix(__byte_perm(x, y, 0x7632));
            split_tf32(__byte_perm(lows, highs, 0x5410), weight[n][0], weight[n][2]);
            split_tf32(__byte_perm(lows, highs, 0x7632), weight[n][1], weight[n][3]);
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
              split_tf32(word, high[i], low[i]);
            }
#pragma unroll
            for (int n = 0; n < HeadTiles; ++n) {
              float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
              multiply(part, low, weight[n][0], weight[n][1], T());
              multiply(part, high, weight[n][2], weight[n][3], T());
              multiply(part, high, weight[n][0], weight[n][1], T());
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                out_[n][d][i] += part[i];
              }
            }
          }
        }
      } else {
        uint32_t weight[HeadTiles][4]; // high of keys 0-7 and 8-15, low of them
#pragma unroll
        for (int n = 0; n < HeadTiles; ++n) {
#pragma unroll
          for (uint32_t part = 0; part < 2u; ++part) {
            uint32_t high, low;
            split_16<T>(score[n][m][2u * part], score[n][m][2u * part + 1u], high, low);
            weight[n][part] = transpose_matrix(high);
            weight[n][2u + part] = transpose_matrix(low);
          }
        }
        const uint32_t row = m * 16u + (lane_ >> 4u) * 8u + (lane_ & 7u);
#pragma unroll
        for (int d = 0; d < Dim / 16; ++d) {
          uint32_t a[4];
          load_matrices_transposed(a, values + swizzled(row, 2u * d + (lane_ >> 3u & 1u)));
#pragma unroll
          for (int n = 0; n < HeadTiles; ++n) {
            multiply(out_[n][d], a, weight[n][2], weight[n][3], T());
            multiply(out_[n][d], a, weight[n][0], weight[n][1], T());
          }
        }
      }
    }
  }

  __device__ __forceinline__ void store(uint32_t sequence, uint32_t head, uint32_t d,
                                        float x) const {
    T *out = static_cast<T *>(args_.out.data) + sequence * args_.out.row_stride +
             head * args_.out.head_stride;
    out[d] = from_float<T>(x);
  }

  // The warps' states of a row joined, eight heads at a time: the result
  // where the block has the whole row (`state` null), else a partial state.
  __device__ __forceinline__ void end_row(uint32_t sequence, uint32_t first_head, uint32_t heads,
                                          float *state) {
#pragma unroll
    for (int n = 0; n < HeadTiles; ++n) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (uint32_t offset = 4; offset < 32u; offset <<= 1u) {
          sum_[n][i] += __shfl_xor_sync(kAllLanes, sum_[n][i], offset);
        }
        if (lane_ < 4u) {
          merge_maxima_[warp_ * 8u + lane_ * 2u + i] = maximum_[n][i];
          merge_sums_[warp_ * 8u + lane_ * 2u + i] = sum_[n][i];
        }
      }
#pragma unroll
      for (int d = 0; d < Dim / 16; ++d) {
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i) {
          const uint32_t head = (lane_ & 3u) * 2u + (i & 1u);
          const uint32_t column = d * 16u + (i >> 1u) * 8u + lane_ / 4u;
          merge_[(warp_ * 8u + head) * Dim + column] = out_[n][d][i];
        }
      }
      __syncthreads();
      for (uint32_t at = threadIdx.x; at < 8u * Dim; at += kThreads) {
        const uint32_t head = at / Dim, column = at % Dim;
        float top = -INFINITY;
#pragma unroll
        for (uint32_t w = 0; w < kWarps; ++w) {
          top = fmaxf(top, merge_maxima_[w * 8u + head]);
        }
        float sum = 0.0f, x = 0.0f;
        const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
        for (uint32_t w = 0; w < kWarps; ++w) {
          const float factor = exp2_fast(merge_maxima_[w * 8u + head] - base);
          sum += merge_sums_[w * 8u + head] * factor;
          x += merge_[(w * 8u + head) * Dim + column] * factor;
        }
        const uint32_t in_row = n * 8u + head;
        if (state != nullptr) {
          state[in_row * Dim + column] = x;
          if (column == 0) {
            state[kHeads * Dim + in_row] = top;
            state[kHeads * (Dim + 1u) + in_row] = sum;
          }
        } else if (in_row < heads) {
          finish(sequence, first_head + in_row, column, x, top, sum);
        }
      }
      __syncthreads();
    }
  }

  __device__ __forceinline__ void finish(uint32_t sequence, uint32_t head, uint32_t column, float x,
                                         float top, float sum) const {
    const bool empty = top == -INFINITY;
    if (column < args_.head_dim) {
      store(sequence, head, column, empty ? 0.0f : x / sum);
    }
    if (column == 0 && args_.lse != nullptr) {
      args_.lse[uint64_t{sequence} * args_.heads + head] =
          empty ? -INFINITY : (top + log2f(sum)) * kLn2;
    }
  }

  // The states that blocks first .. last left of a row, joined by the last of
  // them to get here. Block b left it as its last row where the row began in
  // it, else as its first.
  __device__ __forceinline__ void join(uint32_t sequence, uint32_t row, uint32_t first_head,
                                       uint32_t heads, uint32_t first, uint32_t last,
                                       uint64_t row_begin, uint64_t per_block) const {
    __threadfence();
    __syncthreads();
    uint32_t *arrivals = args_.arrivals + uint64_t{sequence} * args_.rows_per_sequence + row;
    if (threadIdx.x == 0) {
      const bool is_last = atomicAdd(arrivals, 1u) == last - first;
      *flag_ = is_last ? 1u : 0u;
      if (is_last) {
        *arrivals = 0;
      }
    }
    __syncthreads();
    if (*flag_ == 0) {
      __syncthreads(); // the flag may be written again
      return;
    }
    __threadfence();
    const uint32_t count = last - first + 1u;
    auto state_of = [&](uint32_t i) {
      const uint32_t block = first + i;
      const uint32_t slot = row_begin >= block * per_block ? 1u : 0u;
      return args_.states + (2u * uint64_t{block} + slot) * kStateFloats;
    };
    // Weights [head][state] in the merge area, as far as it reaches.
    float *weights = merge_;
    for (uint32_t at = threadIdx.x; at < kHeads * count; at += kThreads) {
      weights[at] = __ldcg(state_of(at % count) + kHeads * Dim + at / count);
    }
    __syncthreads();
    for (uint32_t at = threadIdx.x; at < heads * Dim; at += kThreads) {
      const uint32_t head = at / Dim;
      float top = -INFINITY;
      for (uint32_t i = 0; i < count; ++i) {
        top = fmaxf(top, weights[head * count + i]);
      }
      const float base = top == -INFINITY ? 0.0f : top;
      float x = 0.0f, sum = 0.0f;
#pragma unroll 8
      for (uint32_t i = 0; i < count; ++i) {
        const float *state = state_of(i);
        const float factor = exp2_fast(weights[head * count + i] - base);
        x += __ldcg(state + at) * factor;
        sum += __ldcg(state + kHeads * (Dim + 1u) + head) * factor;
      }
      finish(sequence, first_head + head, at % Dim, x, top, sum);
    }
    __syncthreads();
  }

public:
  static constexpr uint32_t kThreads = 32u * kWarps;

  __device__ __forceinline__ PagedAttention(const PagedAttentionArgs &args, unsigned char *shared)
      : args_(args) {
    ring_ = shared_address(shared) + warp_ * kStages * kStageBytes;
    unsigned char *at = shared + kWarps * kStages * kStageBytes;
    merge_ = reinterpret_cast<float *>(at);
    at += 4u * attention_merge_floats(Dim, kRowBytes);
    merge_maxima_ = reinterpret_cast<float *>(at);
    merge_sums_ = merge_maxima_ + kWarps * 8u;
    seen_ = reinterpret_cast<uint64_t *>(merge_sums_ + kWarps * 8u) + warp_ * kStages;
    at += 2u * 4u * kWarps * 8u + 8u * kWarps * kStages;
    flag_ = reinterpret_cast<uint32_t *>(at);
  }

  __device__ __forceinline__ void run() {
    // Tiles before each thread's share of the sequences, and of all of them.
    const uint32_t share = (args_.table.rows + kThreads - 1u) / kThreads;
    const uint32_t mine_begin = min(threadIdx.x * share, args_.table.rows);
    const uint32_t mine_end = min(mine_begin + share, args_.table.rows);
    uint64_t mine = 0;
    for (uint32_t s = mine_begin; s < mine_end; ++s) {
      const Span span = span_of(args_, s);
      mine += uint64_t{(span.end - span.begin + kKeys - 1u) / kKeys} * args_.rows_per_sequence;
    }
    uint64_t *sums = reinterpret_cast<uint64_t *>(merge_); // [warps], then the block's start
    uint64_t upto = mine;
#pragma unroll
    for (uint32_t offset = 1; offset < 32u; offset <<= 1u) {
      const uint64_t other = __shfl_up_sync(kAllLanes, upto, offset);
      upto += lane_ >= offset ? other : 0;
    }
    if (lane_ == 31u) {
      sums[warp_] = upto;
    }
    __syncthreads();
    uint64_t before = upto - mine, total = 0;
#pragma unroll
    for (uint32_t w = 0; w < kWarps; ++w) {
      before += w < warp_ ? sums[w] : 0;
      total += sums[w];
    }
    __syncthreads();
    uint64_t per_block = (total + gridDim.x - 1u) / gridDim.x;
    per_block = per_block < kAttentionMinimumTiles ? kAttentionMinimumTiles : per_block;
    const uint64_t begin = blockIdx.x * per_block;
    const uint64_t end = begin + per_block < total ? begin + per_block : total;
    if (begin < total && begin >= before && begin < before + mine) {
      uint32_t s = mine_begin;
      while (true) {
        const Span span = span_of(args_, s);
        const uint64_t tiles =
            uint64_t{(span.end - span.begin + kKeys - 1u) / kKeys} * args_.rows_per_sequence;
        if (begin < before + tiles) {
          break;
        }
        before += tiles;
        ++s;
      }
      sums[0] = s;
      sums[1] = before;
    }
    // Rows of sequences that see nothing.
    for (uint32_t s = blockIdx.x; s < args_.table.rows; s += gridDim.x) {
      const Span span = span_of(args_, s);
      if (span.begin == span.end) {
        for (uint32_t at = threadIdx.x; at < args_.heads * Dim; at += kThreads) {
          finish(s, at / Dim, at % Dim, 0.0f, -INFINITY, 0.0f);
        }
      }
    }
    __syncthreads();
    if (begin >= total) {
      return;
    }
    TileCursor row_at; // the row that the block is at; tile: where it begins
    row_at.sequence = static_cast<uint32_t>(sums[0]);
    const uint64_t before_sequence = sums[1];
    __syncthreads();
    enter_sequence<kKeys>(args_, row_at);
    row_at.row = static_cast<uint32_t>((begin - before_sequence) / row_at.tiles);
    row_at.tile = static_cast<uint32_t>((begin - before_sequence) % row_at.tiles);
    uint64_t row_begin = begin - row_at.tile;

    // This warp's tiles are begin + warp, + 4, ...: `next` is the one to load.
    TileCursor load_at = row_at;
    uint64_t next = begin + warp_;
    Gather gather;
    if (next < end) {
      advance<kKeys>(args_, load_at, warp_);
      locate(load_at, gather);
    }
    uint32_t load_stage = 0, stage = 0;
    auto issue_next = [&]() {
      if (next < end) {
        issue(gather, load_stage);
        next += kWarps;
        if (next < end) {
          advance<kKeys>(args_, load_at, kWarps);
          locate(load_at, gather);
        }
      }
      commit_copies();
      load_stage = load_stage + 1u == kStages ? 0u : load_stage + 1u;
    };
#pragma unroll
    for (uint32_t i = 0; i + 1u < kStages; ++i) {
      issue_next();
    }
    uint64_t tile = begin + warp_;
    while (true) {
      const uint64_t row_end = row_begin + row_at.tiles;
      const uint64_t stop = row_end < end ? row_end : end;
      const uint32_t kv_head = row_at.row / args_.head_blocks;
      const uint32_t block_head = (row_at.row - kv_head * args_.head_blocks) * kHeads;
      const uint32_t first_head = kv_head * args_.group + block_head;
      const uint32_t heads = min(kHeads, args_.group - block_head);
      begin_row(row_at.sequence, first_head, heads);
      for (; tile < stop; tile += kWarps) {
        issue_next();
        wait_copies<kStages - 1>();
        __syncwarp();
        compute(stage,
                row_at.span.begin + static_cast<uint32_t>(tile - row_begin) * kKeys,
                row_at.span.end, first_head, heads);
        __syncwarp(); // the stage is filled again by the next issue
        stage = stage + 1u == kStages ? 0u : stage + 1u;
      }
      const uint32_t first = static_cast<uint32_t>(row_begin / per_block);
      const uint32_t last = static_cast<uint32_t>((row_end - 1u) / per_block);
      if (first == last) {
        end_row(row_at.sequence, first_head, heads, nullptr);
      } else {
        const uint32_t slot = row_begin >= begin ? 1u : 0u;
        end_row(row_at.sequence, first_head, heads,
                args_.states + (2u * uint64_t{blockIdx.x} + slot) * kStateFloats);
        join(row_at.sequence, row_at.row, first_head, heads, first, last, row_begin, per_block);
      }
      if (row_end >= end) {
        break;
      }
      row_begin = row_end;
      row_at.tile = row_at.tiles;
      advance<kKeys>(args_, row_at, 0);
    }
    wait_copies<0>();
  }
};

} // namespace lrrt::ops

#endif // LRRT_PAGED_ATTENTION_CUH_
