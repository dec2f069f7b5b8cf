// Sharing, splitting, freeing and compacting the pages of a cache.
//
// A plan kernel (one cluster of eight blocks) works out the new tables and a
// list of page moves; a copy kernel over the whole GPU then moves the rows of
// every layer. Which pages are free follows from the tables alone, so no
// reference counts are kept that could drift from them. Every choice is the
// lowest number, so the results do not depend on the order of threads.
//
// The plan is bound by latency (a few dependent reads of small tables, joined
// by cluster barriers), the copy by memory bandwidth.
#ifndef LRRT_PAGED_PAGES_CUH_
#define LRRT_PAGED_PAGES_CUH_

#include "common.cuh"

#include <cooperative_groups.h>

namespace lrrt::ops {

namespace cg = cooperative_groups;

constexpr uint32_t kPlanAll = kPlanBlocks * kPlanThreads;
constexpr uint32_t kPlanWarps = kPlanThreads / 32u;
constexpr uint32_t kNobody = 0xffffffffu; // mark of a page that no row holds

// Exclusive prefix sums over the cluster's threads (rank, then thread) of two
// counts at once, and their totals. Two cluster barriers.
struct PlanScan {
  uint64_t warp_sums[kPlanWarps];
  uint64_t block_sums[kPlanBlocks];
};

__device__ __forceinline__ uint64_t pack_counts(uint32_t low, uint32_t high) {
  return uint64_t{high} << 32 | low;
}

__device__ __forceinline__ uint64_t plan_scan(uint64_t value, PlanScan &scan, uint64_t &total) {
  cg::cluster_group cluster = cg::this_cluster();
  const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5u;
  uint64_t sum = value;
#pragma unroll
  for (uint32_t offset = 1; offset < 32u; offset <<= 1u) {
    const uint64_t other = __shfl_up_sync(kAllLanes, sum, offset);
    if (lane >= offset) {
      sum += other;
    }
  }
  if (lane == 31u) {
    scan.warp_sums[warp] = sum;
  }
  __syncthreads();
  uint64_t before = 0, block = 0;
#pragma unroll
  for (uint32_t w = 0; w < kPlanWarps; ++w) {
    const uint64_t s = scan.warp_sums[w];
    before += w < warp ? s : 0;
    block += s;
  }
  if (threadIdx.x < kPlanBlocks) {
    *cluster.map_shared_rank(&scan.block_sums[cluster.block_rank()], threadIdx.x) = block;
  }
  cluster.sync();
  total = 0;
#pragma unroll
  for (uint32_t b = 0; b < kPlanBlocks; ++b) {
    const uint64_t s = scan.block_sums[b];
    before += b < cluster.block_rank() ? s : 0;
    total += s;
  }
  cluster.sync(); // the sums may be overwritten from here on
  return before + sum - value;
}

// The contiguous share of [0, count) of one of the cluster's threads.
__device__ __forceinline__ void plan_share(uint32_t count, uint32_t &begin, uint32_t &end) {
  const uint32_t share = (count + kPlanAll - 1u) / kPlanAll;
  const uint64_t first = uint64_t{blockIdx.x * kPlanThreads + threadIdx.x} * share;
  begin = first < count ? static_cast<uint32_t>(first) : count;
  end = count - begin < share ? count : begin + share;
}

// What a row of the new table takes from its parent.
struct ForkRow {
  const int32_t *pages; // the parent's
  uint32_t length, have, need; // tokens; pages they fill; pages of the new row
  uint32_t part;               // tokens in the last, unfinished page
  int32_t last;                // that page, -1: none
};

__device__ __forceinline__ ForkRow fork_row(const ForkArgs &args, uint32_t row) {
  ForkRow r{nullptr, 0, 0, 0, 0, -1};
  const int32_t parent = args.parents[row];
  if (parent < 0 || static_cast<uint32_t>(parent) >= args.table.rows) {
    return r;
  }
  r.pages = args.table.pages + parent * args.table.row_stride;
  const uint64_t capacity = uint64_t{args.table.columns} * args.page.divisor;
  const int32_t length = args.lengths[parent];
  r.length = length < 0 ? 0u
                        : static_cast<uint32_t>(
                              static_cast<uint64_t>(length) < capacity ? length : capacity);
  const uint32_t full = args.page.quotient(r.length);
  r.part = r.length - full * args.page.divisor;
  r.have = full + (r.part != 0 ? 1u : 0u);
  const uint64_t wanted =
      (uint64_t{r.length} + args.room + args.page.divisor - 1u) / args.page.divisor;
  r.need = wanted < args.table.columns ? static_cast<uint32_t>(wanted) : args.table.columns;
  if (r.part != 0) {
    const int32_t page = r.pages[full];
    r.last = page >= 0 && static_cast<uint32_t>(page) < args.page_count ? page : -1;
  }
  return r;
}

__device__ __forceinline__ bool fork_copies(const ForkArgs &args, const ForkRow &r, uint32_t row) {
  return r.last >= 0 && __ldcg(args.owners + r.last) != row + 1u;
}

// owners[page]: kNobody free; 0 held whole by a row (or held outside); s + 1:
// the unfinished last page of row s, the lowest that has it.
__device__ __forceinline__ void fork_plan(const ForkArgs &args) {
  __shared__ PlanScan scan;
  cg::cluster_group cluster = cg::this_cluster();
  const uint32_t thread = blockIdx.x * kPlanThreads + threadIdx.x;
  const uint32_t lane = threadIdx.x & 31u;
  const uint32_t warp = thread >> 5u;
  for (uint32_t page = thread; page < args.page_count; page += kPlanAll) {
    args.owners[page] = args.held != nullptr && args.held[page] != 0 ? 0u : kNobody;
  }
  cluster.sync();
  for (uint32_t row = warp; row < args.rows_out; row += kPlanAll / 32u) {
    const ForkRow r = fork_row(args, row);
    int32_t *out = args.table_out + row * args.table_out_stride;
    const uint32_t full = r.have - (r.part != 0 ? 1u : 0u);
    for (uint32_t column = lane; column < args.table.columns; column += 32u) {
      const int32_t page = column < r.have ? r.pages[column] : -1;
      const bool inside = page >= 0 && static_cast<uint32_t>(page) < args.page_count;
      out[column] = inside ? page : -1;
      if (inside && column < full) {
        args.owners[page] = 0; // the lowest there is: no minimum can raise it
      }
    }
    if (lane == 0) {
      args.lengths_out[row] = static_cast<int32_t>(r.length);
      if (r.last >= 0) {
        atomicMin(args.owners + r.last, row + 1u);
      }
    }
  }
  cluster.sync();
  // Numbers of the free pages below a thread's share, and of the new pages and
  // copies that the rows before its share want.
  uint32_t begin, end;
  plan_share(args.page_count, begin, end);
  uint32_t free_here = 0;
  for (uint32_t page = begin; page < end; ++page) {
    free_here += __ldcg(args.owners + page) == kNobody ? 1u : 0u;
  }
  uint64_t free_total;
  uint32_t rank = static_cast<uint32_t>(plan_scan(free_here, scan, free_total));
  for (uint32_t page = begin; page < end; ++page) {
    if (__ldcg(args.owners + page) == kNobody) {
      args.free_pages[rank++] = static_cast<int32_t>(page);
    }
  }
  plan_share(args.rows_out, begin, end);
  uint32_t wanted = 0, copies = 0;
  for (uint32_t row = begin; row < end; ++row) {
    const ForkRow r = fork_row(args, row);
    const uint32_t copy = fork_copies(args, r, row) ? 1u : 0u;
    wanted += r.need - r.have + copy;
    copies += copy;
  }
  uint64_t totals;
  uint64_t before = plan_scan(pack_counts(wanted, copies), scan, totals);
  for (uint32_t row = begin; row < end; ++row) {
    const ForkRow r = fork_row(args, row);
    const uint32_t copy = fork_copies(args, r, row) ? 1u : 0u;
    args.first_new[row] = static_cast<uint32_t>(before);
    args.first_copy[row] = static_cast<uint32_t>(before >> 32);
    before += pack_counts(r.need - r.have + copy, copy);
  }
  cluster.sync();
  const uint32_t free_pages = static_cast<uint32_t>(free_total);
  for (uint32_t row = warp; row < args.rows_out; row += kPlanAll / 32u) {
    const ForkRow r = fork_row(args, row);
    const bool copy = fork_copies(args, r, row);
    int32_t *out = args.table_out + row * args.table_out_stride;
    const uint32_t from = r.have - (copy ? 1u : 0u);
    const uint32_t first = __ldcg(args.first_new + row);
    for (uint32_t column = from + lane; column < r.need; column += 32u) {
      const uint32_t at = first + column - from;
      const int32_t page = at < free_pages ? __ldcg(args.free_pages + at) : -1;
      out[column] = page;
      if (copy && column == from) {
        args.moves[__ldcg(args.first_copy + row)] = {r.last, page, page >= 0 ? r.part : 0u, 0u};
      }
    }
  }
  if (thread == 0) {
    const uint32_t all = static_cast<uint32_t>(totals);
    args.status[0] = static_cast<int32_t>(all > free_pages ? all - free_pages : 0u);
    args.status[1] = static_cast<int32_t>(all < free_pages ? free_pages - all : 0u);
    *args.move_count = static_cast<uint32_t>(totals >> 32);
  }
}

// marks[page]: kNobody free, 0 held outside, 1 live.
__device__ __forceinline__ void compact_plan(const CompactArgs &args) {
  __shared__ PlanScan scan;
  cg::cluster_group cluster = cg::this_cluster();
  const uint32_t thread = blockIdx.x * kPlanThreads + threadIdx.x;
  const uint32_t lane = threadIdx.x & 31u;
  const uint32_t warp = thread >> 5u;
  for (uint32_t page = thread; page < args.page_count; page += kPlanAll) {
    args.marks[page] = args.held != nullptr && args.held[page] != 0 ? 0u : kNobody;
  }
  cluster.sync();
  for (uint32_t row = warp; row < args.table.rows; row += kPlanAll / 32u) {
    const int32_t *pages = args.table.pages + row * args.table.row_stride;
    for (uint32_t column = lane; column < args.table.columns; column += 32u) {
      const int32_t page = pages[column];
      if (page >= 0 && static_cast<uint32_t>(page) < args.page_count &&
          (args.held == nullptr || args.held[page] == 0)) {
        args.marks[page] = 1u;
      }
    }
  }
  cluster.sync();
  uint32_t begin, end;
  plan_share(args.page_count, begin, end);
  uint32_t used_here = 0;
  for (uint32_t page = begin; page < end; ++page) {
    used_here += __ldcg(args.marks + page) != kNobody ? 1u : 0u;
  }
  uint64_t total;
  plan_scan(used_here, scan, total);
  const uint32_t used = static_cast<uint32_t>(total);
  uint32_t high_here = 0, low_here = 0;
  for (uint32_t page = begin; page < end; ++page) {
    const uint32_t mark = __ldcg(args.marks + page);
    high_here += mark == 1u && page >= used ? 1u : 0u;
    low_here += mark == kNobody && page < used ? 1u : 0u;
  }
  uint64_t totals;
  const uint64_t before = plan_scan(pack_counts(high_here, low_here), scan, totals);
  uint32_t high = static_cast<uint32_t>(before), low = static_cast<uint32_t>(before >> 32);
  for (uint32_t page = begin; page < end; ++page) {
    const uint32_t mark = __ldcg(args.marks + page);
    if (mark == kNobody && page < used) {
      args.free_pages[low++] = static_cast<int32_t>(page);
    }
    if (mark == 1u && page >= used) {
      args.ranks[page] = high;
      args.moves[high++].source = static_cast<int32_t>(page);
    }
  }
  cluster.sync();
  // As many free pages lie below `used` as used ones lie above, so every
  // moved page has a place.
  const uint32_t moved = static_cast<uint32_t>(totals);
  for (uint32_t i = thread; i < moved; i += kPlanAll) {
    args.moves[i].target = __ldcg(args.free_pages + i);
    args.moves[i].rows = args.page_size;
  }
  for (uint32_t row = warp; row < args.table.rows; row += kPlanAll / 32u) {
    const int32_t *pages = args.table.pages + row * args.table.row_stride;
    int32_t *out = args.table_out + row * args.table_out_stride;
    for (uint32_t column = lane; column < args.table.columns; column += 32u) {
      int32_t page = pages[column];
      if (page < 0 || static_cast<uint32_t>(page) >= args.page_count) {
        page = -1;
      } else if (static_cast<uint32_t>(page) >= used && __ldcg(args.marks + page) == 1u) {
        page = __ldcg(args.free_pages + __ldcg(args.ranks + page));
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
  const uint64_t units = uint64_t{moves} * args.units_per_move;
  const uint32_t lane = threadIdx.x & 31u;
  const uint64_t warps = uint64_t{gridDim.x} * (kMoveThreads / 32u);
  for (uint64_t unit = (uint64_t{blockIdx.x} * kMoveThreads + threadIdx.x) / 32u; unit < units;
       unit += warps) {
    const uint32_t index = unit < (uint64_t{1} << 31)
                               ? args.per_move.quotient(static_cast<uint32_t>(unit))
                               : static_cast<uint32_t>(unit / args.units_per_move);
    const uint32_t in_move = static_cast<uint32_t>(unit - uint64_t{index} * args.units_per_move);
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
