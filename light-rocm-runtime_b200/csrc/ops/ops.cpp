// Host library of the paged-cache operators (include/lrrt_ops.h): checks of
// the arguments, the choice of kernels, the workspace and the launches. The
// device code is paged_ops.cubin (csrc/kernels/paged_ops.cu).
#include "lrrt_ops.h"

#include "lrrt/interop.h"
#include "lrrt/lrrt.hpp"
#include "lrrt/ops/kernels.hpp"

#include <algorithm>
#include <array>
#include <cmath>
#include <cstdlib>
#include <cstring>
#include <optional>
#include <stdexcept>
#include <string>
#include <unordered_map>
#include <utility>
#include <vector>

namespace {

using namespace lrrt::ops;

thread_local std::string t_last_error;

// The text of an error, or none where there is no memory for it.
template <typename... Parts> void set_error(const Parts &...parts) noexcept {
  try {
    std::string text;
    (text.append(parts), ...);
    t_last_error = std::move(text);
  } catch (...) {
    t_last_error.clear();
  }
}

template <typename Body> lr_status_t guarded(const char *what, Body body) noexcept {
  try {
    body();
    return LR_SUCCESS;
  } catch (const lrrt::Error &error) {
    char detail[512] = {};
    lr_last_error_detail(detail, sizeof(detail));
    const bool more = detail[0] != '\0';
    set_error(what, ": ", error.what(), more ? " [" : "", detail, more ? "]" : "");
    return error.status();
  } catch (const std::invalid_argument &error) {
    set_error(what, ": ", error.what());
    return LR_ERROR_INVALID_ARGUMENT;
  } catch (const std::exception &error) {
    set_error(what, ": ", error.what());
    return LR_ERROR_RUNTIME;
  } catch (...) {
    set_error(what, ": unknown failure");
    return LR_ERROR_RUNTIME;
  }
}

void require(bool condition, const char *text) {
  if (!condition) {
    throw std::invalid_argument(text);
  }
}

constexpr uint64_t ceil_div(uint64_t a, uint64_t b) { return (a + b - 1u) / b; }
constexpr size_t aligned(size_t bytes) { return (bytes + 255u) / 256u * 256u; }

bool multiple_of(const void *pointer, size_t bytes) {
  return reinterpret_cast<uintptr_t>(pointer) % bytes == 0;
}
bool multiple_of(int64_t elements, size_t element_bytes, size_t bytes) {
  return elements * static_cast<int64_t>(element_bytes) % static_cast<int64_t>(bytes) == 0;
}

size_t type_bytes(uint32_t type) {
  require(type <= LRO_F16, "unknown element type");
  return type == LRO_F32 ? 4u : 2u;
}
const char *type_name(uint32_t type) {
  return type == LRO_F32 ? "f32" : type == LRO_BF16 ? "bf16" : "f16";
}

constexpr uint64_t kMaximumTokens = uint64_t{1} << 31; // positions are int32

void check_cache(const lro_cache_t &cache) {
  type_bytes(cache.type);
  require(cache.keys != nullptr && cache.values != nullptr, "the cache has no keys or values");
  require(cache.page_count > 0 && cache.page_count <= 0x7fffffffu, "page_count out of range");
  require(cache.page_size > 0 && cache.page_size <= (1u << 20), "page_size must be 1 to 2^20");
  require(cache.kv_heads > 0 && cache.kv_heads <= 65536u, "kv_heads out of range");
  require(cache.head_dim > 0 && cache.head_dim <= 65536u, "head_dim out of range");
}

void check_table(const lro_table_t &table, uint32_t page_size) {
  require(table.pages != nullptr || table.rows == 0 || table.columns == 0,
          "the page table is missing");
  require(table.rows <= 0x7fffffffu, "the page table has too many rows");
  require(uint64_t{table.columns} * page_size < kMaximumTokens,
          "the page table holds 2^31 tokens or more");
}

int32_t stride_of(int64_t elements) {
  require(elements >= INT32_MIN && elements <= INT32_MAX,
          "strides must be less than 2^31 elements");
  return static_cast<int32_t>(elements);
}
Cache cache_of(const lro_cache_t &cache) {
  return {{cache.keys, stride_of(cache.key_page_stride), stride_of(cache.key_token_stride),
           stride_of(cache.key_head_stride)},
          {cache.values, stride_of(cache.value_page_stride), stride_of(cache.value_token_stride),
           stride_of(cache.value_head_stride)},
          cache.page_count,
          cache.kv_heads,
          Divider::of(cache.page_size)};
}
Rows rows_of(const lro_rows_t &rows) {
  return {rows.data, stride_of(rows.row_stride), stride_of(rows.head_stride)};
}
Table table_of(const lro_table_t &table) {
  return {table.pages, table.row_stride, table.rows, table.columns};
}

void check_rows(const lro_rows_t &rows, size_t bytes, const char *text) {
  require(rows.data != nullptr && multiple_of(rows.data, bytes), text);
}

// Refuses places of `width` neighbouring elements that are written to, `sizes` of
// them `strides` apart, unless each stride spans all that lies within it: others
// may share memory.
template <size_t N>
void require_apart(std::array<int64_t, N> strides, std::array<uint64_t, N> sizes, uint64_t width,
                   const char *text) {
  std::array<std::pair<uint64_t, uint64_t>, N> axes;
  for (size_t i = 0; i < N; ++i) {
    axes[i] = {static_cast<uint64_t>(std::abs(strides[i])), sizes[i]};
    if (sizes[i] == 0) {
      return;
    }
  }
  std::sort(axes.begin(), axes.end());
  for (const auto &[stride, size] : axes) {
    if (size > 1u) {
      require(stride >= width, text);
      width += stride * (size - 1u);
    }
  }
}

// Whether a new table's rows share memory with the table's: of the same stride
// each two of them that come near, else the extents of all.
bool tables_meet(const int32_t *out, int64_t out_stride, uint32_t out_rows,
                 const lro_table_t &table) {
  if (out_rows == 0 || table.rows == 0 || table.columns == 0) {
    return false;
  }
  const int64_t distance =
      reinterpret_cast<intptr_t>(table.pages) - reinterpret_cast<intptr_t>(out);
  const int64_t width = int64_t{table.columns} * 4, stride = 4 * table.row_stride;
  const int64_t out_last = 4 * out_stride * (int64_t{out_rows} - 1);
  const int64_t last = stride * (int64_t{table.rows} - 1);
  if (out_stride == table.row_stride && stride != 0) {
    // Row i of the table is `distance` + stride (i - j) past row j of the new one.
    const int64_t nearest = -distance / stride;
    for (int64_t k = nearest - 1; k <= nearest + 1; ++k) {
      if (k > -int64_t{out_rows} && k < int64_t{table.rows} &&
          std::abs(distance + stride * k) < width) {
        return true;
      }
    }
    return false;
  }
  return distance + std::min<int64_t>(last, 0) < std::max<int64_t>(out_last, 0) + width &&
         distance + std::max<int64_t>(last, 0) + width > std::min<int64_t>(out_last, 0);
}

// Whether vectors of `bytes` bytes fit rows of this layout.
bool rows_take(const lro_rows_t &rows, size_t element, size_t bytes) {
  return multiple_of(rows.data, bytes) && multiple_of(rows.row_stride, element, bytes) &&
         multiple_of(rows.head_stride, element, bytes);
}
bool cache_takes(const lro_cache_t &cache, size_t bytes) {
  const size_t element = type_bytes(cache.type);
  return multiple_of(cache.keys, bytes) && multiple_of(cache.values, bytes) &&
         multiple_of(cache.key_page_stride, element, bytes) &&
         multiple_of(cache.key_token_stride, element, bytes) &&
         multiple_of(cache.key_head_stride, element, bytes) &&
         multiple_of(cache.value_page_stride, element, bytes) &&
         multiple_of(cache.value_token_stride, element, bytes) &&
         multiple_of(cache.value_head_stride, element, bytes);
}

} // namespace

struct lro_context_t {
  lro_context_t(lr_device_t device_in, lr_queue_t *queue_in, const void *image, size_t size)
      : device(device_in), queue(queue_in), module(device_in, image, size) {
    sms = device.properties().compute_unit_count;
    reserve(size_t{8} << 20);
    reserve_counters(16384);
  }

  void reserve(size_t bytes) {
    if (!scratch || scratch->size() < bytes) {
      grow(scratch, bytes, false);
    }
  }

  // Counters are zero between calls: the kernels put them back.
  void reserve_counters(size_t count) {
    if (!counters || counters->size() < 4u * count) {
      grow(counters, 4u * count, true);
    }
  }

  // A larger buffer takes the place of one, which stays: work on the queue and
  // captured graphs may still use it. Sizes double at least, so that all that is
  // kept is no larger than what is in use.
  void grow(std::optional<lrrt::DeviceBuffer> &buffer, size_t bytes, bool zero) {
    uint32_t capturing = 0;
    lrrt::check(lr_queue_is_capturing(device.get(), queue, &capturing), "lr_queue_is_capturing");
    if (capturing != 0) {
      throw std::runtime_error("the workspace is too small for this call, and cannot grow while "
                               "its stream is captured: reserve it before");
    }
    outgrown.reserve(outgrown.size() + 1u);
    lrrt::DeviceBuffer larger(device,
                              aligned(std::max(bytes, buffer ? 2u * buffer->size() : size_t{0})));
    if (zero) {
      launch("ops_zero", 64, 256, 0,
             ZeroArgs{static_cast<uint32_t *>(larger.data()), larger.size() / 4u});
    }
    if (buffer) {
      outgrown.push_back(std::move(*buffer));
    }
    buffer.emplace(std::move(larger));
  }

  lr_kernel_t *kernel(const std::string &name) {
    const auto found = kernels.find(name);
    if (found != kernels.end()) {
      return found->second;
    }
    lr_kernel_t *handle = module.kernel(name.c_str()).get();
    lrrt::check(lr_kernel_set_overlapped(handle, 1), "lr_kernel_set_overlapped");
    kernels.emplace(name, handle);
    return handle;
  }

  template <typename Args>
  void launch(const std::string &name, uint64_t blocks_x, uint32_t threads, uint32_t shared,
              const Args &args, uint32_t blocks_y = 1) {
    require(blocks_x * threads <= 0xffffffffu, "the call is too large for one launch");
    const lr_launch_config_t config{{static_cast<uint32_t>(blocks_x * threads), blocks_y, 1},
                                    {threads, 1, 1},
                                    shared};
    lr_kernel_t *handle = kernel(name);
    if (queue != nullptr) {
      lrrt::check(lr_launch_on_queue(queue, handle, &config, &args, sizeof(args)), name.c_str());
    } else {
      lrrt::check(lr_launch(handle, &config, &args, sizeof(args)), name.c_str());
    }
  }

  lrrt::Device device;
  lr_queue_t *queue;
  lrrt::Module module;
  std::unordered_map<std::string, lr_kernel_t *> kernels;
  std::optional<lrrt::DeviceBuffer> scratch, counters;
  std::vector<lrrt::DeviceBuffer> outgrown;
  uint32_t sms = 0;
};

namespace {

void rope_append(lro_context_t &context, const lro_rope_append_t &a) {
  check_cache(a.cache);
  check_table(a.table, a.cache.page_size);
  const size_t element = type_bytes(a.cache.type);
  const uint32_t dim = a.cache.head_dim;
  require(a.heads > 0 && a.heads <= 65536u, "heads out of range");
  require(a.rotary_dim % 2u == 0 && a.rotary_dim <= dim,
          "rotary_dim must be even and at most head_dim");
  require(a.rotary_dim == 0 || a.table_positions <= 0x7fffffffu, "table_positions out of range");
  require(a.rotary_dim == 0 || (a.cos_table != nullptr && a.sin_table != nullptr &&
                                multiple_of(a.cos_table, 4) && multiple_of(a.sin_table, 4)),
          "the cos/sin tables are missing");
  if (a.tokens == 0) {
    return;
  }
  require(a.positions != nullptr, "positions are missing");
  check_rows(a.q, element, "q is missing or misaligned");
  check_rows(a.q_out, element, "q_out is missing or misaligned");
  check_rows(a.k, element, "k is missing or misaligned");
  check_rows(a.v, element, "v is missing or misaligned");
  require(cache_takes(a.cache, element), "the cache is misaligned");
  require_apart(std::array{a.q_out.row_stride, a.q_out.head_stride},
                std::array{uint64_t{a.tokens}, uint64_t{a.heads}}, dim,
                "rows of q_out share memory");
  const std::array cache_sizes{uint64_t{a.cache.page_count}, uint64_t{a.cache.page_size},
                               uint64_t{a.cache.kv_heads}};
  require_apart(std::array{a.cache.key_page_stride, a.cache.key_token_stride,
                           a.cache.key_head_stride},
                cache_sizes, dim, "rows of keys share memory");
  require_apart(std::array{a.cache.value_page_stride, a.cache.value_token_stride,
                           a.cache.value_head_stride},
                cache_sizes, dim, "rows of values share memory");

  // The widest vector that all rows and columns are made of: 16 bytes, 8 (for
  // 16-bit rows such as a half of 20 elements), or single elements. Measured with
  // 16384 tokens in bf16: 73, 109, 335 us.
  // What is copied (values, and what is not turned) may take wider ones than the
  // pairs: 6000 tokens of 56 heads over 8 of 80 elements in bf16, 40 of them turned,
  // 40 us, and 54 with the pairs' vectors for all.
  const uint32_t half = a.rotary_dim / 2u, rest = dim - a.rotary_dim;
  const auto rows_and_cache_take = [&](size_t bytes) {
    return rows_take(a.q, element, bytes) && rows_take(a.q_out, element, bytes) &&
           rows_take(a.k, element, bytes) && rows_take(a.v, element, bytes) &&
           cache_takes(a.cache, bytes);
  };
  uint32_t width = 1, copy_width = 1;
  for (const size_t bytes : {size_t{16}, size_t{8}}) {
    const uint32_t elements = static_cast<uint32_t>(bytes / element);
    const uint32_t angles = std::min(elements, 4u);
    if (elements < 4u || rest % elements != 0 || dim % elements != 0 ||
        !rows_and_cache_take(bytes)) {
      continue;
    }
    copy_width = std::max(copy_width, elements);
    if (half % elements == 0 && multiple_of(a.cos_table, 4u * angles) &&
        multiple_of(a.sin_table, 4u * angles)) {
      width = elements;
      break;
    }
  }
  if (width == 1) {
    copy_width = 1;
  }
  const uint32_t per_head = half / width + rest / copy_width, per_value_head = dim / copy_width;
  const uint64_t per_token = (uint64_t{a.heads} + a.cache.kv_heads) * per_head;
  const uint64_t values_per_token = uint64_t{a.cache.kv_heads} * per_value_head;
  require((per_token + values_per_token) * a.tokens < (uint64_t{1} << 31),
          "the tokens have too many elements");
  RopeAppendArgs args{};
  args.q = rows_of(a.q);
  args.q_out = rows_of(a.q_out);
  args.k = rows_of(a.k);
  args.v = rows_of(a.v);
  args.cache = cache_of(a.cache);
  args.table = table_of(a.table);
  args.sequences = a.sequences;
  args.positions = a.positions;
  args.cos_table = a.cos_table;
  args.sin_table = a.sin_table;
  args.items = static_cast<uint32_t>(per_token * a.tokens);
  args.value_items = static_cast<uint32_t>(values_per_token * a.tokens);
  args.heads = a.heads;
  args.rotary_dim = a.rotary_dim;
  args.table_positions = a.rotary_dim == 0 ? 0x7fffffffu : a.table_positions;
  args.per_token = Divider::of(static_cast<uint32_t>(per_token));
  args.per_head = Divider::of(per_head);
  args.values_per_token = Divider::of(static_cast<uint32_t>(values_per_token));
  args.values_per_head = Divider::of(per_value_head);
  context.launch(std::string("ops_rope_") + (a.interleaved != 0 ? "pairs_" : "half_") +
                     type_name(a.cache.type) + "_x" + std::to_string(width) +
                     (copy_width != width ? "x" + std::to_string(copy_width) : std::string()),
                 ceil_div(args.items, kRopeThreads) + ceil_div(args.value_items, kRopeThreads),
                 kRopeThreads, 0, args);
}

void paged_attention(lro_context_t &context, const lro_paged_attention_t &a) {
  check_cache(a.cache);
  check_table(a.table, a.cache.page_size);
  const size_t element = type_bytes(a.cache.type);
  const uint32_t limit = a.cache.type == LRO_F32 ? 128u : 256u;
  require(a.cache.head_dim % 8u == 0 && a.cache.head_dim <= limit,
          "head_dim must be a multiple of 8, at most 256 (128 in 32 bits)");
  require(a.heads > 0 && a.heads <= 65536u && a.heads % a.cache.kv_heads == 0,
          "heads must be a multiple of kv_heads");
  require(std::isfinite(a.scale), "scale must be finite");
  require(std::isfinite(a.softcap) && a.softcap >= 0.0f, "softcap must be finite, 0 or more");
  if (a.table.rows == 0) {
    return;
  }
  require(a.lengths != nullptr, "lengths are missing");
  check_rows(a.q, element, "q is missing or misaligned");
  check_rows(a.out, element, "out is missing or misaligned");
  require_apart(std::array{a.out.row_stride, a.out.head_stride},
                std::array{uint64_t{a.table.rows}, uint64_t{a.heads}}, a.cache.head_dim,
                "rows of out share memory");
  require(cache_takes(a.cache, 16),
          "cache pointers and strides must be multiples of 16 bytes");

  // The next of the kernels' widths: what lies past the head's elements are
  // products of zeros. Heads of 96 in f32 (8 over 1, 6 sequences of about 90000
  // keys) as 96 and as 128 elements: 98 and 115 us; of 80 in f16 (128 over 8, 8
  // sequences of 3900): 28 and 31 us.
  uint32_t dim = 256;
  for (const uint32_t width : {128u, 96u, 64u}) {
    dim = a.cache.head_dim <= width ? width : dim;
  }
  const uint32_t group = a.heads / a.cache.kv_heads;
  // Up to 16 query heads share a row that is read; blocks of them read it one
  // after another. Measured (64 ragged sequences of up to 8192 keys), blocks of 16
  // heads and of 8: bf16, 128 heads over 8, of 128 elements 132 and 228 us, of 64 85
  // and 158 us; 64 over 4 of 256 145 and 241 us; f32, 128 over 8 of 64 175 and 238 us,
  // 48 over 4 of 128 258 and 326 us.
  const uint32_t heads = group > 8u ? 16u : 8u;
  PagedAttentionArgs args{};
  args.q = rows_of(a.q);
  args.out = rows_of(a.out);
  args.cache = cache_of(a.cache);
  args.table = table_of(a.table);
  args.lengths = a.lengths;
  args.slopes = a.slopes;
  args.lse = a.lse;
  args.heads = a.heads;
  args.group = group;
  args.head_dim = a.cache.head_dim;
  args.window = a.window;
  args.paired_queries = rows_take(a.q, element, 4) ? 1u : 0u;
  args.head_blocks = static_cast<uint32_t>(ceil_div(group, heads));
  args.rows_per_sequence = a.cache.kv_heads * args.head_blocks;
  args.scale = a.scale;
  args.softcap = a.softcap;

  uint64_t tokens = uint64_t{a.table.columns} * a.cache.page_size;
  args.capacity = static_cast<uint32_t>(tokens);
  if (a.window != 0) {
    tokens = std::min<uint64_t>(tokens, a.window);
  }
  const uint64_t rows = uint64_t{a.table.rows} * args.rows_per_sequence;
  const uint32_t row_bytes = attention_row_bytes(dim, static_cast<uint32_t>(element));
  const uint32_t keys = attention_tile_keys(row_bytes);
  const uint64_t tiles = rows * (ceil_div(tokens, keys) + kAttentionRowCost);
  require(tiles < (uint64_t{1} << 31), "the table's tokens, times the kv heads, are too many");
  const uint32_t grid = static_cast<uint32_t>(
      std::clamp<uint64_t>(ceil_div(tiles, kAttentionMinimumTiles), 1u, context.sms));
  context.reserve(size_t{8} * grid * attention_state_floats(dim, heads));
  context.reserve_counters(rows);
  args.states = static_cast<float *>(context.scratch->data());
  args.arrivals = static_cast<uint32_t *>(context.counters->data());
  context.launch(std::string("ops_attention_") + type_name(a.cache.type) + "_" +
                     std::to_string(dim) + "x" + std::to_string(heads),
                 grid, attention_threads(dim, row_bytes, heads),
                 attention_shared_bytes(dim, row_bytes, heads), args);
}

// Checks the pool and fills what its moves share; returns whether 16-byte
// vectors fit it.
bool pool_moves(const lro_pool_t &pool, MoveArgs &args) {
  require(pool.keys != nullptr && pool.values != nullptr, "the pool has no keys or values");
  require(pool.page_count > 0 && pool.page_count <= 0x7fffffffu, "page_count out of range");
  require(pool.page_size > 0 && pool.page_size <= (1u << 20), "page_size must be 1 to 2^20");
  require(pool.layers > 0 && pool.segments > 0 && pool.row_bytes > 0,
          "layers, segments and row_bytes must be positive");
  const uint64_t run = uint64_t{pool.page_size} * pool.row_bytes;
  require(run < (uint64_t{1} << 31), "a page's run of rows must be less than 2 GB");
  const auto fits = [&](size_t bytes) {
    return multiple_of(pool.keys, bytes) && multiple_of(pool.values, bytes) &&
           multiple_of(pool.layer_stride_bytes, 1, bytes) &&
           multiple_of(pool.page_stride_bytes, 1, bytes) && pool.row_bytes % bytes == 0;
  };
  require(fits(4), "pool pointers, strides and row_bytes must be multiples of 4 bytes");
  require_apart(std::array{pool.layer_stride_bytes, pool.page_stride_bytes},
                std::array{uint64_t{pool.layers}, uint64_t{pool.page_count}}, run * pool.segments,
                "the pool's pages share memory");
  const bool wide = fits(16); // 4 bytes at a time: 86 us where 16 take 78
  const uint64_t slices = ceil_div(run, kMoveSliceVectors * (wide ? 16u : 4u));
  const uint64_t units = uint64_t{pool.layers} * 2u * pool.segments * slices;
  require(units < (uint64_t{1} << 31), "a page has too many parts");
  args.keys = pool.keys;
  args.values = pool.values;
  args.layer_stride = pool.layer_stride_bytes;
  args.page_stride = pool.page_stride_bytes;
  args.page_count = pool.page_count;
  args.page_size = pool.page_size;
  args.segments = pool.segments;
  args.row_bytes = pool.row_bytes;
  args.per_move = Divider::of(static_cast<uint32_t>(units));
  args.per_segment = Divider::of(static_cast<uint32_t>(slices));
  args.segments_divider = Divider::of(pool.segments);
  return wide;
}

// At most `most` moves, one warp per unit, at most eight blocks per SM.
void launch_moves(lro_context_t &context, const MoveArgs &args, bool wide, uint64_t most) {
  const uint64_t blocks = ceil_div(most * args.per_move.divisor, kMoveThreads / 32u);
  context.launch(wide ? "ops_move_pages_16" : "ops_move_pages_4",
                 std::min<uint64_t>(blocks, uint64_t{context.sms} * 8u), kMoveThreads, 0, args);
}

// Workspace of a plan: the number of moves, the moves, and the arrays.
void plan_memory(lro_context_t &context, size_t rows, size_t pages, size_t moves,
                 PlanArrays &arrays, PageMove *&list, uint32_t *&list_count) {
  const size_t rows_at = 256u + aligned(sizeof(PageMove) * moves),
               marks_at = rows_at + aligned(sizeof(ForkRow) * rows),
               free_at = marks_at + aligned(4u * pages), ranks_at = free_at + aligned(4u * pages);
  context.reserve(ranks_at + aligned(4u * pages));
  auto *scratch = static_cast<unsigned char *>(context.scratch->data());
  list_count = reinterpret_cast<uint32_t *>(scratch);
  list = reinterpret_cast<PageMove *>(scratch + 256);
  arrays = {reinterpret_cast<ForkRow *>(scratch + rows_at),
            reinterpret_cast<uint32_t *>(scratch + marks_at),
            reinterpret_cast<int32_t *>(scratch + free_at),
            reinterpret_cast<uint32_t *>(scratch + ranks_at), static_cast<uint32_t>(rows)};
}

// A block alone where its shared memory holds the arrays and the table is
// small, else the cluster. Measured, alone and clustered, with the moves: a fork
// of 32 beams 8.0 and 9.2 us, of 128 beams 24.4 and 26.1 us.
template <typename Args>
void launch_plan(lro_context_t &context, const std::string &what, size_t array_bytes,
                 uint64_t entries, const Args &args) {
  if (array_bytes <= kPlanAloneBytes && entries <= kPlanAloneEntries) {
    context.launch("ops_" + what + "_plan_alone", 1, kPlanThreadsAlone,
                   static_cast<uint32_t>(array_bytes), args);
  } else {
    context.launch("ops_" + what + "_plan", kPlanBlocks, kPlanThreads, 0, args);
  }
}

void pages_fork(lro_context_t &context, const lro_pages_fork_t &a) {
  MoveArgs moves{};
  const bool wide = pool_moves(a.pool, moves);
  check_table(a.table, a.pool.page_size);
  require(a.status != nullptr, "status is missing");
  require(a.rows_out == 0 || (a.parents != nullptr && a.lengths_out != nullptr &&
                              (a.lengths != nullptr || a.table.rows == 0) &&
                              (a.table_out != nullptr || a.table.columns == 0)),
          "lengths, parents or an output is missing");
  require(a.rows_out <= 0x7fffffffu &&
              uint64_t{a.rows_out} * (uint64_t{a.table.columns} + 1u) < (uint64_t{1} << 32),
          "the new table is too large");
  require(!tables_meet(a.table_out, a.table_out_row_stride, a.rows_out, a.table),
          "table_out must not be the table, nor share memory with it");
  require_apart(std::array{a.table_out_row_stride}, std::array{uint64_t{a.rows_out}},
                a.table.columns, "rows of table_out share memory");
  const size_t rows = a.rows_out, pages = a.pool.page_count;
  PlanArrays arrays{};
  PageMove *list = nullptr;
  uint32_t *list_count = nullptr;
  plan_memory(context, rows, pages, rows, arrays, list, list_count);
  ForkArgs args{};
  args.table = table_of(a.table);
  args.lengths = a.lengths;
  args.parents = a.parents;
  args.held = a.held;
  args.table_out = a.table_out;
  args.table_out_stride = a.table_out_row_stride;
  args.lengths_out = a.lengths_out;
  args.status = a.status;
  args.rows_out = a.rows_out;
  args.room = a.room;
  args.capacity = a.table.columns * a.pool.page_size;
  args.page_count = a.pool.page_count;
  args.page = Divider::of(a.pool.page_size);
  args.move_count = list_count;
  args.moves = list;
  args.arrays = arrays;
  launch_plan(context, "fork", sizeof(ForkRow) * rows + 8u * pages,
              uint64_t{a.rows_out} * a.table.columns, args);
  if (a.rows_out != 0 && a.pool.page_size > 1) { // pages of one token are never unfinished
    moves.moves = args.moves;
    moves.move_count = args.move_count;
    launch_moves(context, moves, wide, a.rows_out);
  }
}

void pages_compact(lro_context_t &context, const lro_pages_compact_t &a) {
  MoveArgs moves{};
  const bool wide = pool_moves(a.pool, moves);
  check_table(a.table, a.pool.page_size);
  require(a.status != nullptr, "status is missing");
  require(a.table_out != nullptr || a.table.rows == 0 || a.table.columns == 0,
          "table_out is missing");
  require((a.table_out == a.table.pages && a.table_out_row_stride == a.table.row_stride) ||
              !tables_meet(a.table_out, a.table_out_row_stride, a.table.rows, a.table),
          "table_out shares memory with the table and is not it");
  require_apart(std::array{a.table_out_row_stride}, std::array{uint64_t{a.table.rows}},
                a.table.columns, "rows of table_out share memory");
  const size_t pages = a.pool.page_count;
  PlanArrays arrays{};
  PageMove *list = nullptr;
  uint32_t *list_count = nullptr;
  plan_memory(context, 0, pages, pages, arrays, list, list_count);
  CompactArgs args{};
  args.table = table_of(a.table);
  args.held = a.held;
  args.table_out = a.table_out;
  args.table_out_stride = a.table_out_row_stride;
  args.status = a.status;
  args.page_count = a.pool.page_count;
  args.page_size = a.pool.page_size;
  args.move_count = list_count;
  args.moves = list;
  args.arrays = arrays;
  launch_plan(context, "compact", 12u * pages, uint64_t{a.table.rows} * a.table.columns, args);
  moves.moves = args.moves;
  moves.move_count = args.move_count;
  // A page moves only from above the live ones to below them: half the pool.
  launch_moves(context, moves, wide, std::max<uint64_t>(pages / 2u, 1u));
}

void pages_copy(lro_context_t &context, const lro_pages_copy_t &a) {
  MoveArgs moves{};
  const bool wide = pool_moves(a.pool, moves);
  if (a.count == 0) {
    return;
  }
  require(a.sources != nullptr && a.targets != nullptr, "sources or targets are missing");
  moves.sources = a.sources;
  moves.targets = a.targets;
  moves.count = a.count;
  launch_moves(context, moves, wide, a.count);
}

void beam_select(lro_context_t &context, const lro_beam_select_t &a) {
  const size_t element = type_bytes(a.type);
  require(a.beams >= 1 && a.beams <= kBeamMaximumCount && a.count >= 1 &&
              a.count <= kBeamMaximumCount && a.beams * a.count <= kBeamMaximumCandidates,
          "beams and count must be 1 to 64, their product at most 2048");
  require(a.vocab >= a.count && a.vocab <= kBeamMaximumVocab, "vocab must be count to 2^21");
  require(uint64_t{a.groups} * a.beams <= 65535u, "at most 65535 beams in all");
  if (a.groups == 0) {
    return;
  }
  require(a.logits != nullptr && multiple_of(a.logits, element),
          "logits are missing or misaligned");
  require(a.scores != nullptr && a.scores_out != nullptr && a.parents_out != nullptr &&
              a.tokens_out != nullptr,
          "scores or an output is missing");
  require(a.count == a.beams || (a.scores_out != a.scores &&
                                 (a.finished == nullptr || a.finished_out != a.finished)),
          "outputs may be inputs only where count = beams");
  const size_t rows = size_t{a.groups} * a.beams;
  // Parts of a row, by the time of the SM with most of them, in units of 10 ns. A
  // round of 16 KB takes a block 0.42 us of 16-bit elements and 0.3 us of 32-bit
  // ones where it has its SM alone, 0.7 and 0.48 us where two share it; a part's
  // fixed work (floor, ranking) 4.2 us alone and 4.8 us beside another; joining
  // a row's parts 2.5 us and a little for each. Measured, 151936 logits: 256 rows in
  // bf16 1, 2, 3 parts 24, 31, 37 us; 96 rows in f32 1, 2, 3, 4 parts 19, 19, 16.5,
  // 20 us; 32 rows in bf16 1, 2, 4, 5, 8 parts 15, 13, 11.2, 12.4, 11.5 us; 4 rows in
  // f32 4, 8, 20, 38 parts 11.8, 10.2, 9.9, 10.5 us.
  const uint32_t round = beam_round(static_cast<uint32_t>(element));
  const uint64_t rounds = ceil_div(a.vocab, round);
  const uint64_t most = std::min<uint64_t>({rounds, kBeamMaximumParts, kBeamPool / a.count});
  const uint64_t alone_round = element == 4u ? 30u : 42u, shared_round = element == 4u ? 48u : 70u;
  uint64_t parts = 1, least = ~uint64_t{0};
  for (uint64_t n = ceil_div(rounds, kBeamNotedRounds); n <= most; ++n) {
    const uint64_t blocks = ceil_div(rows * n, context.sms); // of the SM
    const uint64_t waves = ceil_div(blocks, kBeamBlocksPerSm);
    const uint64_t cost = waves * ((blocks > 1u ? shared_round : alone_round) * ceil_div(rounds, n) +
                                   (blocks > 1u ? 480u : 420u)) +
                          (n > 1u ? 250u + 4u * n : 0u);
    if (cost < least) {
      least = cost;
      parts = n;
    }
  }
  const uint64_t part_elements = (ceil_div(a.vocab, parts) + 7u) / 8u * 8u;
  parts = ceil_div(a.vocab, part_elements);
  const size_t sums_at = aligned(8u * rows * parts * a.count),
               row_keys_at = sums_at + aligned(8u * rows * parts),
               log_sums_at = row_keys_at + aligned(8u * rows * a.count),
               tops_at = log_sums_at + aligned(8u * rows);
  context.reserve(tops_at + aligned(4u * rows));
  context.reserve_counters(rows + a.groups);
  auto *scratch = static_cast<unsigned char *>(context.scratch->data());
  auto *counters = static_cast<uint32_t *>(context.counters->data());
  BeamArgs args{};
  args.logits = a.logits;
  args.logits_stride = a.logits_row_stride;
  args.scores = a.scores;
  args.finished = a.finished;
  args.scores_out = a.scores_out;
  args.parents_out = a.parents_out;
  args.tokens_out = a.tokens_out;
  args.finished_out = a.finished_out;
  args.groups = a.groups;
  args.beams = a.beams;
  args.vocab = a.vocab;
  args.count = a.count;
  args.parts = static_cast<uint32_t>(parts);
  args.part_elements = static_cast<uint32_t>(part_elements);
  args.end_token = a.end_token;
  args.part_keys = reinterpret_cast<uint64_t *>(scratch);
  args.part_sums = reinterpret_cast<Pair *>(scratch + sums_at);
  args.row_keys = reinterpret_cast<uint64_t *>(scratch + row_keys_at);
  args.row_tops = reinterpret_cast<float *>(scratch + tops_at);
  args.row_log_sums = reinterpret_cast<double *>(scratch + log_sums_at);
  args.row_arrivals = counters;
  args.group_arrivals = counters + rows;
  context.launch(std::string("ops_beam_") + type_name(a.type),
                 parts, kBeamThreads, kBeamSharedBytes, args, static_cast<uint32_t>(rows));
}

} // namespace

extern "C" {

LRRT_API lr_status_t lro_context_create(lr_device_t device, lr_queue_t *queue,
                                        const void *module_image, size_t module_image_size,
                                        lro_context_t **context) {
  return guarded("lro_context_create", [&] {
    require(module_image != nullptr && module_image_size != 0, "the module image is missing");
    require(context != nullptr, "context is null");
    *context = new lro_context_t(device, queue, module_image, module_image_size);
  });
}

LRRT_API lr_status_t lro_context_destroy(lro_context_t *context) {
  return guarded("lro_context_destroy", [&] {
    require(context != nullptr, "context is null");
    context->device.synchronize();
    delete context;
  });
}

LRRT_API lr_status_t lro_context_reserve(lro_context_t *context, size_t workspace_bytes) {
  return guarded("lro_context_reserve", [&] {
    require(context != nullptr, "context is null");
    context->reserve(workspace_bytes);
  });
}

LRRT_API lr_status_t lro_context_reserve_counters(lro_context_t *context, uint64_t counters) {
  return guarded("lro_context_reserve_counters", [&] {
    require(context != nullptr, "context is null");
    require(counters < (uint64_t{1} << 40), "too many counters");
    context->reserve_counters(counters);
  });
}

LRRT_API lr_status_t lro_rope_tables(uint32_t positions, uint32_t rotary_dim, double theta,
                                     double factor, double low_turns, double high_turns,
                                     double trained_positions, float *cos_table,
                                     float *sin_table) {
  return guarded("lro_rope_tables", [&] {
    require(rotary_dim != 0 && rotary_dim % 2u == 0, "rotary_dim must be even and positive");
    require(std::isfinite(theta) && theta > 0.0, "theta must be positive");
    require(std::isfinite(factor) && factor >= 1.0, "factor must be at least 1");
    require(std::isfinite(low_turns) && std::isfinite(high_turns) && low_turns >= 0.0 &&
                high_turns >= low_turns,
            "low_turns must be 0 to high_turns");
    require(std::isfinite(trained_positions) && (high_turns == 0.0 || trained_positions > 0.0),
            "trained_positions must be positive");
    require(cos_table != nullptr && sin_table != nullptr, "a table is null");
    const uint32_t half = rotary_dim / 2u;
    for (uint32_t i = 0; i < half; ++i) {
      double frequency = std::pow(theta, -2.0 * i / rotary_dim);
      if (factor > 1.0) {
        double keep = 0.0; // share of the frequency that is not scaled
        if (high_turns > 0.0) {
          const double turns = trained_positions * frequency / (2.0 * std::acos(-1.0));
          keep = high_turns > low_turns ? (turns - low_turns) / (high_turns - low_turns)
                                        : (turns >= high_turns ? 1.0 : 0.0);
          keep = std::clamp(keep, 0.0, 1.0);
        }
        frequency = frequency * keep + frequency / factor * (1.0 - keep);
      }
      for (uint32_t p = 0; p < positions; ++p) {
        cos_table[size_t{p} * half + i] = static_cast<float>(std::cos(p * frequency));
        sin_table[size_t{p} * half + i] = static_cast<float>(std::sin(p * frequency));
      }
    }
  });
}

#define LRRT_OPS_ENTRY(name, arguments_type, body)                                                \
  LRRT_API lr_status_t name(lro_context_t *context, const arguments_type *arguments) {            \
    return guarded(#name, [&] {                                                                   \
      require(context != nullptr && arguments != nullptr, "context or arguments are null");       \
      body(*context, *arguments);                                                                 \
    });                                                                                           \
  }

LRRT_OPS_ENTRY(lro_rope_append, lro_rope_append_t, rope_append)
LRRT_OPS_ENTRY(lro_paged_attention, lro_paged_attention_t, paged_attention)
LRRT_OPS_ENTRY(lro_pages_fork, lro_pages_fork_t, pages_fork)
LRRT_OPS_ENTRY(lro_pages_compact, lro_pages_compact_t, pages_compact)
LRRT_OPS_ENTRY(lro_pages_copy, lro_pages_copy_t, pages_copy)
LRRT_OPS_ENTRY(lro_beam_select, lro_beam_select_t, beam_select)

LRRT_API const char *lro_last_error(void) { return t_last_error.c_str(); }

} // extern "C"
