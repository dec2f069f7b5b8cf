// Kernel arguments of the paged-cache operators' module (paged_ops.cubin),
// shared by the device code and the host library. Every kernel takes one of
// these structs by value; the host launches them through lr_launch* with the
// struct as the packed argument blob. The operators are described in
// include/lrrt_ops.h.
#ifndef LRRT_OPS_KERNELS_HPP_
#define LRRT_OPS_KERNELS_HPP_

#include <cstdint>

#if defined(__CUDACC__)
#define LRRT_OPS_HD __host__ __device__
#else
#define LRRT_OPS_HD
#endif

namespace lrrt::ops {

// n / divisor for n < 2^31 as one multiplication: with 2^(s-1) < d <= 2^s and
// m = ceil(2^(31+s) / d) < 2^32, n m = 2^(31+s) n / d + n e / d with e < d, and
// the excess n e / (d 2^(31+s)) < 2^-s <= 1 / d never reaches the next integer.
struct Divider {
  uint32_t divisor, multiplier, shift; // shift = s - 1; divisor 1 has none

  static Divider of(uint32_t d) {
    uint32_t s = 0;
    while ((uint64_t{1} << s) < d) {
      ++s;
    }
    const uint64_t m = ((uint64_t{1} << (31u + s)) + d - 1u) / d;
    return {d, static_cast<uint32_t>(m), s == 0 ? 0u : s - 1u};
  }
  LRRT_OPS_HD uint32_t quotient(uint32_t n) const {
    if (divisor == 1) {
      return n;
    }
#if defined(__CUDA_ARCH__)
    return __umulhi(n, multiplier) >> shift;
#else
    return static_cast<uint32_t>((uint64_t{n} * multiplier) >> 32) >> shift;
#endif
  }
};

// Strides are in elements and below 2^31, so that an offset is one 32-bit by
// 32-bit product of 64 bits.
struct Rows {
  void *data;
  int32_t row_stride, head_stride;

  LRRT_OPS_HD int64_t offset(uint32_t row, uint32_t head) const {
    return int64_t{row} * row_stride + int64_t{head} * head_stride;
  }
};

struct Pages {
  void *data;
  int32_t page_stride, token_stride, head_stride;

  LRRT_OPS_HD int64_t offset(uint32_t page, uint32_t token, uint32_t head) const {
    return int64_t{page} * page_stride + int64_t{token} * token_stride +
           int64_t{head} * head_stride;
  }
};

struct Cache {
  Pages keys, values;
  uint32_t page_count, kv_heads;
  Divider page;
};

struct Table {
  const int32_t *pages;
  int64_t row_stride;
  uint32_t rows, columns;
};

constexpr uint32_t kRopeThreads = 256;

struct RopeAppendArgs {
  Rows q, q_out, k, v;
  Cache cache;
  Table table;
  const int32_t *sequences, *positions;
  const float *cos_table, *sin_table;
  uint32_t items, value_items; // of all tokens' query and key heads, and value heads
  uint32_t heads, rotary_dim, table_positions;
  Divider per_token, per_head;             // items of a token, of a head
  Divider values_per_token, values_per_head;
};

// Shared memory of an attention block: a ring of tiles for each of its units,
// and a partial state for each. A unit is a warp, or two warps that share its
// tiles, with eight heads each, where the states of 16 heads of a long row
// would not fit one warp's registers. A tile is 16 keys and values, or 32 of the
// short rows of 128 bytes: 8 KB, and 16 KB for rows of 512 bytes. Eight units
// have three tiles each (two beside states of 16 heads); of the large tiles six
// have two (four with three: 216 us instead of 180 for 64 sequences of up to 8192
// keys, 16 heads over 4 of 128 in f32), four have three beside states of 256 elements, or
// as teams (two beside 16 heads of 256).
// Rows of 96 elements (for heads of 65 to 96) lie in the places of 128.
LRRT_OPS_HD constexpr uint32_t attention_row_bytes(uint32_t dim, uint32_t element_bytes) {
  return (dim == 96u ? 128u : dim) * element_bytes;
}
LRRT_OPS_HD constexpr uint32_t attention_tile_bytes(uint32_t row_bytes) {
  return row_bytes <= 256u ? 8192u : 16384u;
}
LRRT_OPS_HD constexpr uint32_t attention_tile_keys(uint32_t row_bytes) {
  return attention_tile_bytes(row_bytes) / (2u * row_bytes);
}
LRRT_OPS_HD constexpr uint32_t attention_team(uint32_t row_bytes, uint32_t heads) {
  return heads > 8u && row_bytes > 256u ? 2u : 1u;
}
LRRT_OPS_HD constexpr uint32_t attention_units(uint32_t dim, uint32_t row_bytes,
                                               uint32_t heads) {
  return row_bytes <= 256u ? 8u : attention_team(row_bytes, heads) == 1u && dim <= 128u ? 6u : 4u;
}
LRRT_OPS_HD constexpr uint32_t attention_threads(uint32_t dim, uint32_t row_bytes,
                                                 uint32_t heads) {
  return 32u * attention_units(dim, row_bytes, heads) * attention_team(row_bytes, heads);
}
LRRT_OPS_HD constexpr uint32_t attention_stages(uint32_t dim, uint32_t row_bytes,
                                                uint32_t heads) {
  return attention_units(dim, row_bytes, heads) == 4u ? (dim > 128u && heads > 8u ? 2u : 3u)
         : heads > 8u || row_bytes > 256u             ? 2u
                                                      : 3u;
}
// One partial state: the weighted values (rows padded against bank conflicts),
// the maxima and the sums of a block's heads.
LRRT_OPS_HD constexpr uint32_t attention_state_floats(uint32_t dim, uint32_t heads) {
  return heads * (dim + 6u);
}
LRRT_OPS_HD constexpr uint32_t attention_shared_bytes(uint32_t dim, uint32_t row_bytes,
                                                      uint32_t heads) {
  return attention_units(dim, row_bytes, heads) *
             (attention_stages(dim, row_bytes, heads) * attention_tile_bytes(row_bytes) +
              4u * attention_state_floats(dim, heads)) +
         1024u;
}
static_assert(attention_shared_bytes(128, 256, 8) <= 232448u &&
                  attention_shared_bytes(128, 256, 16) <= 232448u &&
                  attention_shared_bytes(64, 256, 16) <= 232448u &&
                  attention_shared_bytes(128, 512, 8) <= 232448u &&
                  attention_shared_bytes(128, 512, 16) <= 232448u &&
                  attention_shared_bytes(256, 512, 8) <= 232448u &&
                  attention_shared_bytes(256, 512, 16) <= 232448u,
              "a block's shared memory");
// Places that a block takes at least, so that a short row is not split into more
// partial states than its tiles are worth. Measured (2000 bf16 keys of 8 heads of
// 128, group of 4): at least 4, 8, 16 of them 8.9, 10.6, 10.9 us.
constexpr uint32_t kAttentionMinimumTiles = 4;
// Where no row has more tiles than this, blocks take whole rows, so that states
// are joined in shared memory only: the first of these with few rows, the
// second where there are at least half as many as blocks. Measured, whole rows
// and split ones: 8 rows of 10 tiles 7.4 and 8.5 us; 8 rows of 19 tiles 8.7 and
// 7.5 us; 128 rows of 31 tiles 11.7 and 13.3 us; 64 rows of 64 tiles 20.7 and
// 16.2 us.
constexpr uint32_t kAttentionWholeTilesFew = 16;
constexpr uint32_t kAttentionWholeTilesMany = 32;
// What a row costs a warp besides its tiles (its queries, and its end), in
// tiles. Measured with 0, 1, 3: 64 sequences of up to 900 keys 29.1, 23.0, 23.7
// us; of up to 8192 keys 137, 135, 135 us; 128 of up to 200 keys 21.6, 17.8, 18.6 us.
constexpr uint32_t kAttentionRowCost = 1;

struct PagedAttentionArgs {
  Rows q, out;
  Cache cache;
  Table table;
  const int32_t *lengths;
  const float *slopes; // null: no distance bias
  float *lse;          // null: not wanted
  float *states;       // [2 * grid][attention_state_floats]
  uint32_t *arrivals;  // [table.rows * rows_per_sequence], zero between launches
  uint32_t heads, group, head_dim, window;
  uint32_t capacity; // tokens that the table holds: columns * page size
  uint32_t paired_queries; // 16-bit q rows are multiples of 4 bytes
  uint32_t head_blocks, rows_per_sequence; // blocks of query heads per kv head; kv_heads * them
  float scale, softcap;
};

// `rows` rows of page `source` go to page `target`, which may be none (-1).
struct PageMove {
  int32_t source, target;
  uint32_t rows;
  uint32_t row; // of the new table that it is for
};

// What a row of a forked table takes from its parent, and gets anew.
struct ForkRow {
  int32_t parent, last; // -1: none; the parent's last, unfinished page
  uint32_t length, part; // tokens; those in the last page
  uint32_t have, need;   // pages that they fill; pages of the new row
  uint32_t copies;       // 1: the last page has to be copied
  uint32_t first_new;    // the first of its new pages among the free ones
};

constexpr uint32_t kPlanBlocks = 8; // one cluster
constexpr uint32_t kPlanThreads = 512;
constexpr uint32_t kPlanThreadsAlone = 1024; // of a block that plans by itself
constexpr uint32_t kPlanAloneBytes = 200u * 1024u; // of working arrays, in shared memory
constexpr uint32_t kPlanAloneEntries = 32768;      // of the table

// Working arrays of a plan: [row_count] rows (fork), and [page_count] marks,
// free pages and ranks (compact).
struct PlanArrays {
  ForkRow *rows;
  uint32_t *marks;
  int32_t *free_pages;
  uint32_t *ranks;
  uint32_t row_count;
};

struct ForkArgs {
  Table table;
  const int32_t *lengths, *parents;
  const uint8_t *held;
  int32_t *table_out;
  int64_t table_out_stride;
  int32_t *lengths_out, *status;
  uint32_t rows_out, room, page_count;
  uint32_t capacity; // tokens of a row of the table
  Divider page;
  PlanArrays arrays;
  PageMove *moves; // [rows_out]
  uint32_t *move_count;
};

struct CompactArgs {
  Table table;
  const uint8_t *held;
  int32_t *table_out;
  int64_t table_out_stride;
  int32_t *status;
  uint32_t page_count, page_size;
  PlanArrays arrays;
  PageMove *moves; // [page_count]
  uint32_t *move_count;
};

constexpr uint32_t kMoveThreads = 256;
constexpr uint32_t kMoveSliceVectors = 256; // vectors of one warp's slice: eight per lane

struct MoveArgs {
  void *keys, *values;
  int64_t layer_stride, page_stride; // bytes
  const PageMove *moves;             // null: sources and targets, whole pages
  const uint32_t *move_count;
  const int32_t *sources, *targets;
  uint32_t count; // without move_count
  uint32_t page_count, page_size, segments, row_bytes;
  Divider per_move;    // units of a move: layers * 2 * segments * slices
  Divider per_segment; // slices of a segment
  Divider segments_divider;
};

constexpr uint32_t kBeamThreads = 256;
constexpr uint32_t kBeamBlocksPerSm = 2;
constexpr uint32_t kBeamMaximumCount = 64;
constexpr uint32_t kBeamMaximumCandidates = 2048; // beams * count
// A block reads a round of elements at a time, with four rounds under way: two
// such blocks fill an SM's shared memory.
constexpr uint32_t kBeamRoundBytes = 16384;
constexpr uint32_t kBeamStages = 4;
LRRT_OPS_HD constexpr uint32_t beam_round(uint32_t element_bytes) {
  return kBeamRoundBytes / element_bytes;
}
constexpr uint32_t kBeamPool = 2048;              // candidates it holds
constexpr uint32_t kBeamMaximumParts = 64;        // of a row
constexpr uint32_t kBeamNotedRounds = 40;         // of a part
constexpr uint32_t kBeamMaximumVocab = 1u << 21;
static_assert(kBeamMaximumVocab <= kBeamNotedRounds * beam_round(4) *
                                       (kBeamPool / kBeamMaximumCount),
              "the parts of the longest row hold it");
constexpr uint32_t kBeamSharedBytes = 111616;
static_assert(kBeamMaximumCandidates <= kBeamPool, "a group's candidates fit the pool");

struct Pair {
  float x, y;
};

struct BeamArgs {
  const void *logits;
  int64_t logits_stride;
  const float *scores;
  const uint8_t *finished;
  float *scores_out;
  int32_t *parents_out, *tokens_out;
  uint8_t *finished_out;
  uint32_t groups, beams, vocab, count;
  uint32_t parts, part_elements; // of a row; elements a multiple of 8
  int32_t end_token;
  uint64_t *part_keys;    // [rows][parts][count]
  Pair *part_sums;        // [rows][parts] maximum, sum of exponentials above it
  uint64_t *row_keys;     // [rows][count]
  float *row_tops;        // [rows] maximum
  double *row_log_sums;   // [rows] logarithm of the sum above it
  uint32_t *row_arrivals; // [rows], zero between launches
  uint32_t *group_arrivals; // [groups], likewise
};

// A beam search's bookkeeping before and after the operators of a step.
struct BeamBeginArgs {
  const int32_t *forked_table, *forked_lengths, *status; // of lro_pages_fork
  int32_t *table;               // [rows][columns]
  int32_t *lengths, *positions; // [rows]
  uint32_t *missing_pages;
  uint32_t rows, columns;
};

struct BeamEndArgs {
  const int32_t *tokens, *parents;    // [rows], of lro_beam_select
  uint32_t *next_tokens;              // [rows]
  int32_t *all_tokens, *all_parents;  // [maximum_steps][rows]
  uint32_t *step;
  uint32_t rows, maximum_steps;
};

struct ZeroArgs {
  uint32_t *words;
  uint64_t count;
};

} // namespace lrrt::ops

#endif // LRRT_OPS_KERNELS_HPP_
