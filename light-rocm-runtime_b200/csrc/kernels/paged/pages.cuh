// Sharing, splitting, freeing and compacting the pages of a cache.
//
// A plan kernel works out the new tables and a list of page moves: one block
// with its working arrays in shared memory where they fit, else a cluster of
// eight with them in the workspace. A copy kernel over the whole GPU then moves
// the rows of every layer. Which pages are free follows from the tables alone, so no
// reference counts are kept that could drift from them. Every choice is the
// lowest number, so the results do not depend on the order of threads.
//
// The plan is bound by latency (a few dependent reads of small tables between
// barriers), the copy by memory bandwidth. Measured, both launches: forks of 32
// beams over 24 layers of 2 heads of 64 in f32 8.0 us (0.9 us of copies), of 128
// beams over 16 layers of 8 heads of 128 in bf16 24.5 us (15.5 of copies, 4.1
// TB/s over all); a compaction that moves 230 MB 77.5 us (5.9 TB/s).
#ifndef LRRT_PAGED_PAGES_CUH_
#define LRRT_PAGED_PAGES_CUH_

#include "common.cuh"

#include <cooperative_groups.h>

namespace lrrt::ops {

namespace cg = cooperative_groups;

constexpr uint32_t kNobody = 0xffffffffu; // mark of a page that no row holds

// A block alone, or the cluster: its threads, its barrier, and reads of what
// other threads of it wrote (past the L1 cache where they are of other SMs).
template <bool Clustered> struct Plan {
  static constexpr uint32_t kBlocks = Clustered ? kPlanBlocks : 1u;
  static constexpr uint32_t kThreads = Clustered ? kPlanThreads : kPlanThreadsAlone;
  static constexpr uint32_t kAll = kBlocks * kThreads;
  static constexpr uint32_t kWarps = kThreads / 32u;

  static __device__ __forceinline__ uint32_t rank() {
    return Clustered ? cg::this_cluster().block_rank() : 0u;
  }
  static __device__ __forceinline__ void sync() {
    if constexpr (Clustered) {
      cg::this_cluster().sync();
    } else {
      __syncthreads();
    }
  }
  template <typename T> static __device__ __forceinline__ T read(const T *from) {
    if constexpr (Clustered) {
      return __ldcg(from);
    } else {
      return *from;
    }
  }
  // Shared variables of every block of it.
  template <typename T> static __device__ __forceinline__ T *of_block(T *mine, uint32_t block) {
    if constexpr (Clustered) {
      return cg::this_cluster().map_shared_rank(mine, block);
    } else {
      return mine;
    }
  }
  // The contiguous share of [0, count) of one of its threads.
  static __device__ __forceinline__ void share(uint32_t count, uint32_t &begin, uint32_t &end) {
    const uint32_t each = (count + kAll - 1u) / kAll;
    const uint64_t first = uint64_t{blockIdx.x * kThreads + threadIdx.x} * each;
    begin = first < count ? static_cast<uint32_t>(first) : count;
    end = count - begin < each ? count : begin + each;
  }
};

// Two 32-bit counts in one.
__device__ __forceinline__ uint64_t pack_counts(uint32_t low, uint32_t high) {
  return uint64_t{high} << 32 | low;
}

// Exclusive prefix sums over the threads (rank, then thread) of two values, and
// their totals. Once per kernel.
struct PlanSums {
  uint64_t x, y;
};
template <typename P> struct PlanScan {
  PlanSums warps[P::kWarps];
  PlanSums blocks[P::kBlocks];
};

template <typename P>
__device__ __forceinline__ PlanSums plan_scan(PlanSums value, PlanScan<P> &scan,
                                              PlanSums &total) {
  const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5u;
  PlanSums sum = value;
#pragma unroll
  for (uint32_t offset = 1; offset < 32u; offset <<= 1u) {
    const uint64_t x = __shfl_up_sync(kAllLanes, sum.x, offset);
    const uint64_t y = __shfl_up_sync(kAllLanes, sum.y, offset);
    if (lane >= offset) {
      sum.x += x;
      sum.y += y;
    }
  }
  if (lane == 31u) {
    scan.warps[warp] = sum;
  }
  __syncthreads();
  PlanSums before{sum.x - value.x, sum.y - value.y}, block{0, 0};
#pragma unroll 4
  for (uint32_t w = 0; w < P::kWarps; ++w) {
    const PlanSums s = scan.warps[w];
    before.x += w < warp ? s.x : 0;
    before.y += w < warp ? s.y : 0;
    block.x += s.x;
    block.y += s.y;
  }
  if (threadIdx.x < P::kBlocks) {
    *P::of_block(&scan.blocks[P::rank()], threadIdx.x) = block;
  }
  P::sync();
  total = {0, 0};
#pragma unroll 4
  for (uint32_t b = 0; b < P::kBlocks; ++b) {
    const PlanSums s = scan.blocks[b];
    before.x += b < P::rank() ? s.x : 0;
    before.y += b < P::rank() ? s.y : 0;
    total.x += s.x;
    total.y += s.y;
  }
  return before;
}

// The working arrays: in shared memory for a block alone.
template <typename P>
__device__ __forceinline__ PlanArrays plan_arrays(const PlanArrays &arrays, uint32_t pages) {
  if constexpr (P::kBlocks != 1u) {
    return arrays;
  } else {
    extern __shared__ __align__(16) unsigned char plan_memory[];
    auto *rows = reinterpret_cast<ForkRow *>(plan_memory);
    auto *marks = reinterpret_cast<uint32_t *>(rows + arrays.row_count);
    return {rows, marks, reinterpret_cast<int32_t *>(marks + pages), marks + 2u * size_t{pages},
            arrays.row_count};
  }
}

// What a row of the new table takes from its parent.
__device__ __forceinline__ ForkRow fork_row(const ForkArgs &args, uint32_t row) {
  ForkRow r{-1, -1, 0, 0, 0, 0, 0, 0};
  const int32_t parent = args.parents[row];
  if (parent < 0 || static_cast<uint32_t>(parent) >= args.table.rows) {
    return r;
  }
  r.parent = parent;
  const int32_t length = args.lengths[parent];
  r.length = length < 0 ? 0u : min(static_cast<uint32_t>(length), args.capacity);
  const uint32_t full = args.page.quotient(r.length);
  const uint32_t part = r.length - full * args.page.divisor;
  r.have = full + (part != 0 ? 1u : 0u);
  const uint32_t later = r.length + min(args.room, args.capacity - r.length);
  const uint32_t pages = args.page.quotient(later);
  r.need = pages + (pages * args.page.divisor != later ? 1u : 0u);
  if (part != 0) {
    const int32_t page = args.table.pages[parent * args.table.row_stride + full];
    if (static_cast<uint32_t>(page) < args.page_count) {
      r.last = page;
      r.part = part;
    }
  }
  return r;
}

// owners[page]: kNobody free; 0 held whole by a row (or held outside); s + 1:
// the unfinished last page of row s, the lowest that has it.
template <typename P> __device__ __forceinline__ void fork_plan(const ForkArgs &args) {
  __shared__ PlanScan<P> scan;
  const PlanArrays arrays = plan_arrays<P>(args.arrays, args.page_count);
  uint32_t *owners = arrays.marks;
  const uint32_t thread = blockIdx.x * P::kThreads + threadIdx.x;
  const uint32_t lane = threadIdx.x & 31u;
  const uint32_t warp = thread >> 5u;
  uint32_t row_begin, row_end;
  P::share(args.rows_out, row_begin, row_end);
#pragma unroll 1
  for (uint32_t row = row_begin; row < row_end; ++row) {
    const ForkRow r = fork_row(args, row);
    arrays.rows[row] = r;
    args.lengths_out[row] = static_cast<int32_t>(r.length);
  }
#pragma unroll 4
  for (uint32_t page = thread; page < args.page_count; page += P::kAll) {
    owners[page] = args.held != nullptr && args.held[page] != 0 ? 0u : kNobody;
  }
  P::sync();
#pragma unroll 1
  for (uint32_t row = row_begin; row < row_end; ++row) {
    const int32_t last = arrays.rows[row].last;
    if (last >= 0) {
      atomicMin(owners + last, row + 1u);
    }
  }
#pragma unroll 1
  for (uint32_t row = warp; row < args.rows_out; row += P::kAll / 32u) {
    const ForkRow &r = arrays.rows[row];
    const int32_t parent = P::read(&r.parent);
    const uint32_t have = P::read(&r.have), length = P::read(&r.length);
    const int32_t *pages = args.table.pages + parent * args.table.row_stride;
    int32_t *out = args.table_out + row * args.table_out_stride;
    const uint32_t full = args.page.quotient(length);
#pragma unroll 2
    for (uint32_t column = lane; column < args.table.columns; column += 32u) {
      const int32_t page = column < have ? pages[column] : -1;
      const bool inside = static_cast<uint32_t>(page) < args.page_count;
      out[column] = inside ? page : -1;
      if (inside && column < full) {
        owners[page] = 0; // the lowest there is: no minimum can raise it
      }
    }
  }
  P::sync();
  // The free pages below a thread's share; the new pages and the copies that
  // the rows before its share want.
  uint32_t page_begin, page_end, free_here = 0, wanted = 0, copies = 0;
  P::share(args.page_count, page_begin, page_end);
#pragma unroll 4
  for (uint32_t page = page_begin; page < page_end; ++page) {
    free_here += P::read(owners + page) == kNobody ? 1u : 0u;
  }
#pragma unroll 1
  for (uint32_t row = row_begin; row < row_end; ++row) {
    const ForkRow r = arrays.rows[row];
    const uint32_t copy = r.last >= 0 && P::read(owners + r.last) != row + 1u ? 1u : 0u;
    arrays.rows[row].copies = copy;
    wanted += r.need - r.have + copy;
    copies += copy;
  }
  PlanSums totals;
  PlanSums before = plan_scan({free_here, pack_counts(wanted, copies)}, scan, totals);
#pragma unroll 4
  for (uint32_t page = page_begin; page < page_end; ++page) {
    if (P::read(owners + page) == kNobody) {
      arrays.free_pages[before.x++] = static_cast<int32_t>(page);
    }
  }
#pragma unroll 1
  for (uint32_t row = row_begin; row < row_end; ++row) {
    const ForkRow r = arrays.rows[row];
    arrays.rows[row].first_new = static_cast<uint32_t>(before.y);
    if (r.copies != 0) {
      args.moves[before.y >> 32] = {r.last, -1, r.part, row};
    }
    before.y += pack_counts(r.need - r.have + r.copies, r.copies);
  }
  P::sync();
  const uint32_t free_pages = static_cast<uint32_t>(totals.x);
#pragma unroll 1
  for (uint32_t row = warp; row < args.rows_out; row += P::kAll / 32u) {
    const ForkRow &r = arrays.rows[row];
    const uint32_t from = P::read(&r.have) - P::read(&r.copies), need = P::read(&r.need);
    const uint32_t first = P::read(&r.first_new);
    int32_t *out = args.table_out + row * args.table_out_stride;
#pragma unroll 1
    for (uint32_t column = from + lane; column < need; column += 32u) {
      const uint32_t at = first + column - from;
      out[column] = at < free_pages ? P::read(arrays.free_pages + at) : -1;
    }
  }
  const uint32_t copies_in_all = static_cast<uint32_t>(totals.y >> 32);
#pragma unroll 1
  for (uint32_t i = thread; i < copies_in_all; i += P::kAll) {
    // A row's copy is the first of its new pages; without one nothing moves.
    const uint32_t at = P::read(&arrays.rows[P::read(&args.moves[i].row)].first_new);
    args.moves[i].target = at < free_pages ? P::read(arrays.free_pages + at) : -1;
  }
  if (thread == 0) {
    const uint32_t all = static_cast<uint32_t>(totals.y);
    args.status[0] = static_cast<int32_t>(all > free_pages ? all - free_pages : 0u);
    args.status[1] = static_cast<int32_t>(all < free_pages ? free_pages - all : 0u);
    *args.move_count = copies_in_all;
  }
}

// marks[page]: kNobody free, 0 held outside, 1 live.
template <typename P> __device__ __forceinline__ void compact_plan(const CompactArgs &args) {
  __shared__ PlanScan<P> scan;
  const PlanArrays arrays = plan_arrays<P>(args.arrays, args.page_count);
  __shared__ uint32_t live_below; // of the live pages, those numbered below `used`
  const uint32_t thread = blockIdx.x * P::kThreads + threadIdx.x;
  const uint32_t lane = threadIdx.x & 31u;
  const uint32_t warp = thread >> 5u;
#pragma unroll 4
  for (uint32_t page = thread; page < args.page_count; page += P::kAll) {
    arrays.marks[page] = args.held != nullptr && args.held[page] != 0 ? 0u : kNobody;
  }
  P::sync();
#pragma unroll 1
  for (uint32_t row = warp; row < args.table.rows; row += P::kAll / 32u) {
    const int32_t *pages = args.table.pages + row * args.table.row_stride;
#pragma unroll 2
    for (uint32_t column = lane; column < args.table.columns; column += 32u) {
      const int32_t page = pages[column];
      if (static_cast<uint32_t>(page) < args.page_count &&
          (args.held == nullptr || args.held[page] == 0)) {
        arrays.marks[page] = 1u;
      }
    }
  }
  P::sync();
  uint32_t begin, end, used_here = 0, live_here = 0;
  P::share(args.page_count, begin, end);
#pragma unroll 4
  for (uint32_t page = begin; page < end; ++page) {
    const uint32_t mark = P::read(arrays.marks + page);
    used_here += mark != kNobody ? 1u : 0u;
    live_here += mark == 1u ? 1u : 0u;
  }
  PlanSums totals;
  PlanSums before = plan_scan({used_here, live_here}, scan, totals);
  const uint32_t used = static_cast<uint32_t>(totals.x), live = static_cast<uint32_t>(totals.y);
  // The live pages before each live page, and the free pages in their order: of
  // the pages below a free one all that are not used are free.
#pragma unroll 1
  for (uint32_t page = begin; page < end; ++page) {
    const uint32_t mark = P::read(arrays.marks + page);
    if (page == used) {
      for (uint32_t b = 0; b < P::kBlocks; ++b) {
        *P::of_block(&live_below, b) = static_cast<uint32_t>(before.y);
      }
    }
    if (mark == kNobody) {
      arrays.free_pages[page - before.x] = static_cast<int32_t>(page);
    } else {
      arrays.ranks[page] = static_cast<uint32_t>(before.y);
      ++before.x;
      before.y += mark == 1u ? 1u : 0u;
    }
  }
  if (used == args.page_count && threadIdx.x == 0) {
    live_below = live; // no page lies above
  }
  P::sync();
  // As many free pages lie below `used` as used ones lie above, so every
  // moved page has a place.
  const uint32_t below = live_below, moved = live - below;
  begin = max(begin, used);
#pragma unroll 1
  for (uint32_t page = begin; page < end; ++page) {
    if (P::read(arrays.marks + page) == 1u) {
      const uint32_t rank = arrays.ranks[page] - below;
      args.moves[rank] = {static_cast<int32_t>(page), P::read(arrays.free_pages + rank),
                          args.page_size, 0u};
    }
  }
#pragma unroll 1
  for (uint32_t row = warp; row < args.table.rows; row += P::kAll / 32u) {
    const int32_t *pages = args.table.pages + row * args.table.row_stride;
    int32_t *out = args.table_out + row * args.table_out_stride;
#pragma unroll 2
    for (uint32_t column = lane; column < args.table.columns; column += 32u) {
      int32_t page = pages[column];
      if (static_cast<uint32_t>(page) >= args.page_count) {
        page = -1;
      } else if (static_cast<uint32_t>(page) >= used && P::read(arrays.marks + page) == 1u) {
        page = P::read(arrays.free_pages + P::read(arrays.ranks + page) - below);
      }
      out[column] = page;
    }
  }
  if (thread == 0) {
    args.status[0] = static_cast<int32_t>(used);
    args.status[1] = static_cast<int32_t>(moved);
    *args.move_count = moved;
  }
}

// Units: (move, layer, keys or values, segment, slice), a warp each; a slice
// is kMoveSliceVectors vectors, eight loads in flight per lane.
template <typename V> __device__ __forceinline__ void move_pages(const MoveArgs &args) {
  const uint32_t moves = args.move_count != nullptr ? __ldcg(args.move_count) : args.count;
  const uint32_t lane = threadIdx.x & 31u;
  const uint32_t warp = (blockIdx.x * kMoveThreads + threadIdx.x) / 32u;
  const uint32_t warps = gridDim.x * (kMoveThreads / 32u);
  const uint32_t units = args.per_move.divisor;
  // The grid's warps are so many moves and units ahead of one another.
  const uint32_t moves_ahead = args.per_move.quotient(warps);
  const uint32_t units_ahead = warps - moves_ahead * units;
  uint32_t index = args.per_move.quotient(warp), in_move = warp - index * units;
#pragma unroll 1
  for (; index < moves;
       index += moves_ahead, in_move += units_ahead, index += in_move >= units ? 1u : 0u,
       in_move -= in_move >= units ? units : 0u) {
    const uint32_t segment_index = args.per_segment.quotient(in_move);
    const uint32_t slice = in_move - segment_index * args.per_segment.divisor;
    const uint32_t plane = args.segments_divider.quotient(segment_index);
    const uint32_t segment = segment_index - plane * args.segments;
    PageMove move;
    if (args.moves != nullptr) {
      move = args.moves[index];
    } else {
      move = {args.sources[index], args.targets[index], args.page_size, 0u};
    }
    if (move.source < 0 || static_cast<uint32_t>(move.source) >= args.page_count ||
        move.target < 0 || static_cast<uint32_t>(move.target) >= args.page_count) {
      continue;
    }
    const uint32_t vectors = move.rows * args.row_bytes / sizeof(V);
    const uint32_t begin = slice * kMoveSliceVectors + lane;
    if (slice * kMoveSliceVectors >= vectors) {
      continue;
    }
    char *pool = static_cast<char *>((plane & 1u) != 0 ? args.values : args.keys) +
                 (plane >> 1u) * args.layer_stride +
                 int64_t{segment} * args.page_size * args.row_bytes;
    const V *from = reinterpret_cast<const V *>(pool + move.source * args.page_stride);
    V *to = reinterpret_cast<V *>(pool + move.target * args.page_stride);
    V held[kMoveSliceVectors / 32u];
#pragma unroll
    for (uint32_t i = 0; i < kMoveSliceVectors / 32u; ++i) {
      if (begin + i * 32u < vectors) {
        held[i] = from[begin + i * 32u];
      }
    }
#pragma unroll
    for (uint32_t i = 0; i < kMoveSliceVectors / 32u; ++i) {
      if (begin + i * 32u < vectors) {
        to[begin + i * 32u] = held[i];
      }
    }
  }
}

} // namespace lrrt::ops

#endif // LRRT_PAGED_PAGES_CUH_
