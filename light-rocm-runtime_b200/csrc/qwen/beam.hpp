// Beam search over a paged KV cache: G prompts with K beams each decode as one
// batch of G x K rows. A step runs the prefill module's GEMMs and row kernels
// and the paged-cache operators (include/lrrt_ops.h): the beams' pages are
// forked copy-on-write after their parents, keys are rotated and appended to
// the pages, attention reads them, and the best continuations are selected on
// the device. The step is captured once as a CUDA graph and replayed; only the
// finished search comes back to the host.
//
// light-rocm-runtime decodes greedily, one stream per launch; per row the
// arithmetic is its decode step's, with sums in GEMM order.
#ifndef LRRT_B200_QWEN_BEAM_HPP_
#define LRRT_B200_QWEN_BEAM_HPP_

#include "lrrt_ops.h"
#include "prefill.hpp"

#include <cuda_runtime_api.h>

#include <cstdint>
#include <memory>
#include <optional>
#include <vector>

namespace lrrt::qwen::prefill {

class BeamSearch {
public:
  // groups * beams <= the prefill's chunk size; capacity = positions of a
  // beam; eos_token UINT32_MAX: none.
  BeamSearch(Prefill &prefill, const ModelView &model, const void *ops_image,
             size_t ops_image_size, uint32_t groups, uint32_t beams, uint32_t capacity,
             uint32_t page_size, uint32_t eos_token);
  ~BeamSearch();
  BeamSearch(const BeamSearch &) = delete;
  BeamSearch &operator=(const BeamSearch &) = delete;

  // prompts: the groups' tokens one after another, counts[g] of each. Writes
  // tokens[group][beam][step], best beam first, and scores[group][beam]; a beam
  // that ended goes on with the end token, one that is missing has -1.
  void search(const ModelView &model, const uint32_t *prompts, const uint32_t *counts,
              uint32_t steps, Path path, uint64_t weights_generation, int32_t *tokens,
              float *scores);
  uint32_t groups() const { return groups_; }

private:
  template <typename T> T *allocate(std::optional<DeviceBuffer> &buffer, size_t count);
  float *layer_pages(float *pool, uint32_t layer) const;
  void enqueue_step(const ModelView &model);
  void capture_step(const ModelView &model);

  struct OpsDeleter {
    void operator()(lro_context_t *context) const { lro_context_destroy(context); }
  };

  Prefill &prefill_;
  Module module_; // the bookkeeping kernels
  Kernel begin_, end_;
  std::unique_ptr<lro_context_t, OpsDeleter> ops_;
  uint32_t groups_, beams_, rows_, capacity_, page_size_, columns_, pages_, layers_, eos_token_;
  std::optional<DeviceBuffer> keys_buffer_, values_buffer_, table_buffer_, forked_table_buffer_,
      lengths_buffer_, forked_lengths_buffer_, positions_buffer_, status_buffer_, parents_buffer_,
      tokens_buffer_, next_tokens_buffer_, scores_buffer_, finished_buffer_, logits_buffer_,
      attended_buffer_, history_buffer_, all_tokens_buffer_, all_parents_buffer_;
  float *keys_, *values_, *scores_, *logits_, *attended_;
  int32_t *table_, *forked_table_, *lengths_, *forked_lengths_, *positions_, *status_, *parents_,
      *tokens_, *all_tokens_, *all_parents_;
  uint32_t *next_tokens_, *history_; // history: step, missing pages
  uint8_t *finished_;
  cudaGraphExec_t graph_ = nullptr;
};

} // namespace lrrt::qwen::prefill

#endif // LRRT_B200_QWEN_BEAM_HPP_
