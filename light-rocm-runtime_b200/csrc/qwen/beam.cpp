// Beam search over a paged cache: buffers, the step's launch sequence, its CUDA
// graph, and the way back through the chosen tokens.
#include "beam.hpp"

#include "lrrt/ops/kernels.hpp"
#include "prefill_common.hpp"

#include <algorithm>
#include <cmath>

namespace lrrt::qwen::prefill {

using namespace detail;

namespace {

void check_cuda(cudaError_t status, const char *what) {
  if (status != cudaSuccess) {
    throw std::runtime_error(std::string(what) + ": " + cudaGetErrorString(status));
  }
}

void check_ops(lr_status_t status) {
  if (status != LR_SUCCESS) {
    throw std::runtime_error(lro_last_error());
  }
}

lro_context_t *open_ops(Device device, const void *image, size_t size) {
  lro_context_t *context = nullptr;
  check_ops(lro_context_create(device.get(), nullptr, image, size, &context));
  return context;
}

} // namespace

template <typename T>
T *BeamSearch::allocate(std::optional<DeviceBuffer> &buffer, size_t count) {
  buffer.emplace(prefill_.device_, std::max<size_t>(sizeof(T) * count, 16));
  return static_cast<T *>(buffer->data());
}

BeamSearch::BeamSearch(Prefill &prefill, const ModelView &model, const void *ops_image,
                       size_t ops_image_size, uint32_t groups, uint32_t beams, uint32_t capacity,
                       uint32_t page_size, uint32_t eos_token)
    : prefill_(prefill), module_(prefill.device_, ops_image, ops_image_size),
      begin_(module_.kernel("ops_beam_begin")), end_(module_.kernel("ops_beam_end")),
      ops_(open_ops(prefill.device_, ops_image, ops_image_size)), groups_(groups), beams_(beams),
      rows_(0), capacity_(capacity), page_size_(page_size),
      layers_(static_cast<uint32_t>(model.layers.size())), eos_token_(eos_token) {
  if (groups_ == 0 || beams_ == 0 || beams_ > 32u ||
      uint64_t{groups_} * beams_ > prefill_.max_chunk_tokens() || capacity_ == 0 ||
      capacity_ > model.capacity || page_size_ == 0 || page_size_ > 1024u ||
      beams_ > model.vocab) {
    throw std::invalid_argument("beam search needs groups * beams rows up to the prefill chunk, at "
                                "most 32 beams, capacity <= the model's RoPE rows and pages of 1 "
                                "to 1024 tokens");
  }
  rows_ = groups_ * beams_;
  columns_ = ceil_div(capacity_, page_size_);
  pages_ = rows_ * columns_; // every row with pages of its own
  for (const Kernel *kernel : {&begin_, &end_}) {
    check(lr_kernel_set_overlapped(kernel->get(), 1), "lr_kernel_set_overlapped");
  }
  const size_t pool = size_t{layers_} * pages_ * page_size_ * qd::kKvSize;
  keys_ = allocate<float>(keys_buffer_, pool);
  values_ = allocate<float>(values_buffer_, pool);
  table_ = allocate<int32_t>(table_buffer_, size_t{rows_} * columns_);
  forked_table_ = allocate<int32_t>(forked_table_buffer_, size_t{rows_} * columns_);
  lengths_ = allocate<int32_t>(lengths_buffer_, rows_);
  forked_lengths_ = allocate<int32_t>(forked_lengths_buffer_, rows_);
  positions_ = allocate<int32_t>(positions_buffer_, rows_);
  status_ = allocate<int32_t>(status_buffer_, 2);
  parents_ = allocate<int32_t>(parents_buffer_, rows_);
  tokens_ = allocate<int32_t>(tokens_buffer_, rows_);
  next_tokens_ = allocate<uint32_t>(next_tokens_buffer_, rows_);
  scores_ = allocate<float>(scores_buffer_, rows_);
  finished_ = allocate<uint8_t>(finished_buffer_, rows_);
  logits_ = allocate<float>(logits_buffer_, size_t{rows_} * model.vocab);
  attended_ = allocate<float>(attended_buffer_, size_t{rows_} * kHidden);
  history_ = allocate<uint32_t>(history_buffer_, 2);
  all_tokens_ = allocate<int32_t>(all_tokens_buffer_, size_t{capacity_} * rows_);
  all_parents_ = allocate<int32_t>(all_parents_buffer_, size_t{capacity_} * rows_);
  // Room for every step's operators, so that none of them allocates while the
  // step is captured.
  check_ops(lro_context_reserve(
      ops_.get(), (size_t{16} << 20) + size_t{rows_} * 64u * 8u * (beams_ + 1u) +
                      64u * (size_t{pages_} + rows_)));
}

BeamSearch::~BeamSearch() {
  if (graph_ != nullptr) {
    lr_synchronize(prefill_.device_.get());
    cudaGraphExecDestroy(graph_);
  }
}

float *BeamSearch::layer_pages(float *pool, uint32_t layer) const {
  return pool + size_t{layer} * pages_ * page_size_ * qd::kKvSize;
}

// One step of every row (enqueued on the device's default queue).
void BeamSearch::enqueue_step(const ModelView &model) {
  Prefill &p = prefill_;
  const uint32_t b = rows_;
  auto *hidden = static_cast<float *>(p.hidden_->data());
  auto *normalized = static_cast<float *>(p.normalized_->data());
  auto *normalized_lo = static_cast<float *>(p.normalized_lo_->data());
  auto *qkv = static_cast<float *>(p.qkv_->data());
  auto *attention = static_cast<float *>(p.attention_->data());
  auto *attention_lo = static_cast<float *>(p.attention_lo_->data());
  auto *activated = static_cast<float *>(p.activated_->data());
  auto *activated_lo = static_cast<float *>(p.activated_lo_->data());
  auto finish = [&](const PartialTiles &partials, const float *norm_weight) {
    launch(p.finish_rows_.get(), rows_config(b, row_threads(b), staged_bytes(partials, kHidden)),
           FinishArgs{partials, hidden, b, model.epsilon, norm_weight, normalized, normalized_lo});
  };

  // The beams chosen by the step before, each with a place for its token.
  const int64_t row = int64_t{qd::kKvSize}, page = row * page_size_;
  lro_pages_fork_t fork{};
  fork.pool = {keys_,
               values_,
               static_cast<int64_t>(sizeof(float)) * page * pages_,
               static_cast<int64_t>(sizeof(float)) * page,
               layers_,
               pages_,
               page_size_,
               1,
               static_cast<uint32_t>(sizeof(float) * row),
               0};
  fork.table = {table_, columns_, b, columns_};
  fork.lengths = lengths_;
  fork.parents = parents_;
  fork.table_out = forked_table_;
  fork.table_out_row_stride = columns_;
  fork.lengths_out = forked_lengths_;
  fork.status = status_;
  fork.rows_out = b;
  fork.room = 1;
  check_ops(lro_pages_fork(ops_.get(), &fork));
  launch(begin_.get(), rows_config(ceil_div(uint64_t{b} * columns_, 256), 256),
         ops::BeamBeginArgs{forked_table_, forked_lengths_, status_, table_, lengths_, positions_,
                            history_ + 1, b, columns_});
  launch(p.embed_.get(), rows_config(b, 256),
         EmbedArgs{next_tokens_, model.embeddings, hidden, b, model.vocab});
  launch(p.rmsnorm_.get(), rows_config(b, 256),
         NormArgs{hidden, model.layers[0].attention_norm, normalized, normalized_lo, b,
                  model.epsilon});
  for (uint32_t layer = 0; layer < layers_; ++layer) {
    const LayerView &w = model.layers[layer];
    const Prefill::LayerMaps &maps = p.layer_maps_[layer];
    const lro_cache_t cache{layer_pages(keys_, layer),
                            layer_pages(values_, layer),
                            page,
                            row,
                            qd::kHeadSize,
                            page,
                            row,
                            qd::kHeadSize,
                            LRO_F32,
                            pages_,
                            page_size_,
                            qd::kKvHeads,
                            qd::kHeadSize};
    const lro_table_t table{table_, columns_, b, columns_};
    p.tc_gemm(kQkvTile, p.normalized_maps_, maps.qkv, b, kQkv, kHidden, GemmEpilogue::bias, qkv,
              nullptr, kQkv, w.qkv_bias, false);
    lro_rope_append_t rope{};
    rope.q = rope.q_out = {qkv, kQkv, qd::kHeadSize};
    rope.k = {qkv + kHidden, kQkv, qd::kHeadSize};
    rope.v = {qkv + kHidden + qd::kKvSize, kQkv, qd::kHeadSize};
    rope.cache = cache;
    rope.table = table;
    rope.positions = positions_;
    rope.cos_table = model.rope_cos;
    rope.sin_table = model.rope_sin;
    rope.tokens = b;
    rope.heads = qd::kAttentionHeads;
    rope.rotary_dim = qd::kHeadSize;
    rope.table_positions = model.capacity;
    check_ops(lro_rope_append(ops_.get(), &rope));
    lro_paged_attention_t attend{};
    attend.q = {qkv, kQkv, qd::kHeadSize};
    attend.out = {attended_, kHidden, qd::kHeadSize};
    attend.cache = cache;
    attend.table = table;
    attend.lengths = lengths_;
    attend.heads = qd::kAttentionHeads;
    attend.scale = 1.0f / std::sqrt(static_cast<float>(qd::kHeadSize));
    check_ops(lro_paged_attention(ops_.get(), &attend));
    const uint64_t values = uint64_t{b} * kHidden;
    launch(p.split_.get(), rows_config(std::min<uint32_t>(ceil_div(values, 256), kSms * 8), 256),
           SplitArgs{attended_, attention, attention_lo, values});
    finish(p.tc_gemm(kHiddenTile, p.attention_maps_, maps.o, b, kHidden, kHidden,
                     GemmEpilogue::residual, hidden, nullptr, kHidden, nullptr, true),
           w.mlp_norm);
    p.tc_gemm(kGateUpTile, p.normalized_maps_, maps.gate_up, b, kIntermediate, kHidden,
              GemmEpilogue::swiglu, activated, activated_lo, kIntermediate, nullptr, false);
    finish(p.tc_gemm(kHiddenTile, p.activated_maps_, maps.down, b, kHidden, kIntermediate,
                     GemmEpilogue::residual, hidden, nullptr, kHidden, nullptr, true),
           layer + 1u < layers_ ? model.layers[layer + 1u].attention_norm : model.final_norm);
  }
  p.tc_gemm(kGateUpTile, p.normalized_maps_, p.tail_maps_, b, model.vocab, kHidden,
            GemmEpilogue::store, logits_, nullptr, model.vocab, nullptr, false);
  lro_beam_select_t select{};
  select.logits = logits_;
  select.logits_row_stride = model.vocab;
  select.scores = select.scores_out = scores_;
  select.finished = select.finished_out = finished_;
  select.parents_out = parents_;
  select.tokens_out = tokens_;
  select.type = LRO_F32;
  select.groups = groups_;
  select.beams = select.count = beams_;
  select.vocab = model.vocab;
  select.end_token = eos_token_ == UINT32_MAX ? -1 : static_cast<int32_t>(eos_token_);
  check_ops(lro_beam_select(ops_.get(), &select));
  launch(end_.get(), rows_config(1, 256),
         ops::BeamEndArgs{tokens_, parents_, next_tokens_, all_tokens_, all_parents_, history_, b,
                          capacity_});
}

void BeamSearch::capture_step(const ModelView &model) {
  check_cuda(cudaSetDevice(static_cast<int>(prefill_.device_.index())), "cudaSetDevice");
  void *native = nullptr;
  check(lr_queue_native_handle(prefill_.device_.get(), nullptr, &native),
        "lr_queue_native_handle");
  cudaStream_t stream = static_cast<cudaStream_t>(native);
  prefill_.device_.synchronize();
  check_cuda(cudaStreamBeginCapture(stream, cudaStreamCaptureModeThreadLocal),
             "cudaStreamBeginCapture");
  cudaGraph_t graph = nullptr;
  try {
    enqueue_step(model);
  } catch (...) {
    cudaStreamEndCapture(stream, &graph);
    if (graph != nullptr) {
      cudaGraphDestroy(graph);
    }
    throw;
  }
  check_cuda(cudaStreamEndCapture(stream, &graph), "cudaStreamEndCapture");
  const cudaError_t instantiated = cudaGraphInstantiate(&graph_, graph, 0);
  cudaGraphDestroy(graph);
  check_cuda(instantiated, "cudaGraphInstantiate");
}

void BeamSearch::search(const ModelView &model, const uint32_t *prompts, const uint32_t *counts,
                        uint32_t steps, Path path, uint64_t weights_generation, int32_t *tokens,
                        float *scores) {
  if (prompts == nullptr || counts == nullptr || tokens == nullptr || scores == nullptr ||
      steps == 0) {
    throw std::invalid_argument("beam search needs prompts, at least one step, and outputs");
  }
  size_t total = 0;
  for (uint32_t g = 0; g < groups_; ++g) {
    if (counts[g] == 0 || uint64_t{counts[g]} + steps > uint64_t{capacity_} + 1u) {
      throw std::invalid_argument("a prompt is empty, or it and the steps exceed the capacity");
    }
    total += counts[g];
  }
  for (size_t i = 0; i < total; ++i) {
    if (prompts[i] >= model.vocab) {
      throw std::invalid_argument("prompt token out of range");
    }
  }
  prefill_.device_.synchronize();
  prefill_.prepare_tensor_cores(model, weights_generation);
  prefill_.prepare_tail(model, weights_generation);

  // Group g's prompt fills pages g * columns and on, in order: a contiguous
  // cache. All its beams begin there; the first fork splits the last page, and
  // only the first beam has a score to go on from.
  std::vector<int32_t> table(size_t{rows_} * columns_, -1), lengths(rows_), parents(rows_);
  std::vector<uint32_t> next(rows_);
  std::vector<float> start(rows_, -INFINITY);
  const std::vector<uint8_t> going(rows_, 0);
  const uint32_t *prompt = prompts;
  for (uint32_t g = 0; g < groups_; ++g) {
    const uint32_t known = counts[g] - 1u;
    ModelView view = model;
    view.capacity = capacity_;
    for (uint32_t layer = 0; layer < layers_; ++layer) {
      const size_t at = size_t{g} * columns_ * page_size_ * qd::kKvSize;
      view.layers[layer].key_cache = layer_pages(keys_, layer) + at;
      view.layers[layer].value_cache = layer_pages(values_, layer) + at;
    }
    prefill_.run(view, prompt, known, 0, path, weights_generation);
    for (uint32_t k = 0; k < beams_; ++k) {
      const uint32_t row = g * beams_ + k;
      for (uint32_t column = 0; column < ceil_div(known, page_size_); ++column) {
        table[size_t{row} * columns_ + column] = static_cast<int32_t>(g * columns_ + column);
      }
      lengths[row] = static_cast<int32_t>(known);
      parents[row] = static_cast<int32_t>(row);
      next[row] = prompt[known];
    }
    start[size_t{g} * beams_] = 0.0f;
    prompt += counts[g];
  }
  copy_to_device(*table_buffer_, table.data(), sizeof(int32_t) * table.size());
  copy_to_device(*lengths_buffer_, lengths.data(), sizeof(int32_t) * rows_);
  copy_to_device(*parents_buffer_, parents.data(), sizeof(int32_t) * rows_);
  copy_to_device(*next_tokens_buffer_, next.data(), sizeof(uint32_t) * rows_);
  copy_to_device(*scores_buffer_, start.data(), sizeof(float) * rows_);
  copy_to_device(*finished_buffer_, going.data(), rows_);
  const uint32_t zeros[2] = {0, 0};
  copy_to_device(*history_buffer_, zeros, sizeof(zeros));
  check(lr_memcpy(prefill_.device_.get(), prefill_.error_->data(), zeros, sizeof(uint32_t),
                  LR_MEMCPY_HOST_TO_DEVICE),
        "lr_memcpy beam error");

  // The first step of all is launched as it is: it loads the kernels.
  uint32_t step = 0;
  if (graph_ == nullptr) {
    enqueue_step(model);
    ++step;
    if (step < steps) {
      capture_step(model);
    }
  }
  void *native = nullptr;
  check(lr_queue_native_handle(prefill_.device_.get(), nullptr, &native),
        "lr_queue_native_handle");
  for (; step < steps; ++step) {
    check_cuda(cudaGraphLaunch(graph_, static_cast<cudaStream_t>(native)), "cudaGraphLaunch");
  }
  prefill_.device_.synchronize();
  uint32_t error = 0, history[2] = {};
  check(lr_memcpy(prefill_.device_.get(), &error, prefill_.error_->data(), sizeof(error),
                  LR_MEMCPY_DEVICE_TO_HOST),
        "lr_memcpy beam error");
  copy_to_host(history, *history_buffer_, sizeof(history));
  if (error != 0) {
    throw std::runtime_error("beam search: tensor-core GEMM gave up waiting (code " +
                             std::to_string(error) + ")");
  }
  if (history[0] != steps || history[1] != 0) {
    throw std::runtime_error("beam search: " + std::to_string(history[0]) + " steps, " +
                             std::to_string(history[1]) + " pages missing");
  }
  std::vector<int32_t> chosen(size_t{steps} * rows_), from(chosen.size());
  copy_to_host(chosen.data(), *all_tokens_buffer_, sizeof(int32_t) * chosen.size());
  copy_to_host(from.data(), *all_parents_buffer_, sizeof(int32_t) * from.size());
  copy_to_host(scores, *scores_buffer_, sizeof(float) * rows_);
  for (uint32_t row = 0; row < rows_; ++row) {
    int32_t at = static_cast<int32_t>(row);
    for (uint32_t i = steps; i-- > 0;) {
      tokens[size_t{row} * steps + i] = at >= 0 ? chosen[size_t{i} * rows_ + at] : -1;
      at = at >= 0 ? from[size_t{i} * rows_ + at] : -1;
    }
  }
}

} // namespace lrrt::qwen::prefill
