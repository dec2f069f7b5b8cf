// Host checks of the paged-cache operators: division by multiplication, the
// sizes of the argument structs (mirrored by lrrt_b200/native.py), and the
// refusals that need no device.
#include "lrrt_ops.h"

#include "lrrt/interop.h"
#include "lrrt/ops/kernels.hpp"

#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <random>

namespace {

void expect(bool condition, const char *what) {
  if (!condition) {
    std::fprintf(stderr, "failed: %s\n", what);
    std::exit(1);
  }
}

void check_dividers() {
  using lrrt::ops::Divider;
  constexpr uint32_t kTop = 0x7fffffffu;
  std::mt19937_64 random(1);
  for (uint32_t d = 1; d <= 100000u; d += d < 3000u ? 1u : 97u) {
    const Divider divider = Divider::of(d);
    for (const uint32_t n : {0u, 1u, d - 1u, d, d + 1u, kTop, kTop - 1u, kTop / d * d,
                             kTop / d * d - 1u}) {
      expect(n > kTop || divider.quotient(n) == n / d, "quotient at an edge");
    }
    for (int i = 0; i < 50; ++i) {
      const uint32_t n = static_cast<uint32_t>(random() & kTop);
      expect(divider.quotient(n) == n / d, "quotient of a random number");
      const uint32_t m = n / d * d; // a multiple and the number below it
      expect(divider.quotient(m) == m / d, "quotient of a multiple");
      expect(m == 0 || divider.quotient(m - 1u) == (m - 1u) / d, "quotient below a multiple");
    }
  }
  for (int i = 0; i < 200000; ++i) {
    const uint32_t d = static_cast<uint32_t>((random() & kTop) >> (random() % 31u)) | 1u;
    const uint32_t n = static_cast<uint32_t>(random() & kTop);
    expect(Divider::of(d).quotient(n) == n / d, "quotient of a random pair");
  }
}

void check_refusals() {
  expect(lro_context_create(lr_device_t{0}, nullptr, nullptr, 0, nullptr) ==
             LR_ERROR_INVALID_ARGUMENT,
         "a context without a module");
  expect(std::strstr(lro_last_error(), "module image") != nullptr, "its text");
  expect(lro_context_destroy(nullptr) == LR_ERROR_INVALID_ARGUMENT, "no context to destroy");
  expect(lro_context_reserve(nullptr, 1) == LR_ERROR_INVALID_ARGUMENT, "no context to reserve");
  expect(lro_paged_attention(nullptr, nullptr) == LR_ERROR_INVALID_ARGUMENT, "no arguments");
  expect(std::strstr(lro_last_error(), "lro_paged_attention") != nullptr, "names the call");
  expect(lro_rope_append(nullptr, nullptr) == LR_ERROR_INVALID_ARGUMENT, "no arguments");
  expect(lro_pages_fork(nullptr, nullptr) == LR_ERROR_INVALID_ARGUMENT, "no arguments");
  expect(lro_pages_compact(nullptr, nullptr) == LR_ERROR_INVALID_ARGUMENT, "no arguments");
  expect(lro_pages_copy(nullptr, nullptr) == LR_ERROR_INVALID_ARGUMENT, "no arguments");
  expect(lro_beam_select(nullptr, nullptr) == LR_ERROR_INVALID_ARGUMENT, "no arguments");
  lr_queue_t *queue = nullptr;
  expect(lr_queue_wrap_stream(lr_device_t{1000}, nullptr, &queue) != LR_SUCCESS,
         "a stream of no device");
  float x[8];
  expect(lro_rope_tables(1, 3, 1e4, 1, 0, 0, 0, x, x) == LR_ERROR_INVALID_ARGUMENT,
         "an odd rotary_dim");
  expect(lro_rope_tables(1, 2, 0, 1, 0, 0, 0, x, x) == LR_ERROR_INVALID_ARGUMENT, "theta of 0");
  expect(lro_rope_tables(1, 2, 1e4, 0.5, 0, 0, 0, x, x) == LR_ERROR_INVALID_ARGUMENT,
         "a factor below 1");
  expect(lro_rope_tables(1, 2, 1e4, 2, 4, 1, 10, x, x) == LR_ERROR_INVALID_ARGUMENT,
         "turns in the wrong order");
  expect(lro_rope_tables(1, 2, 1e4, 2, 1, 4, 0, x, x) == LR_ERROR_INVALID_ARGUMENT,
         "turns of no positions");
  expect(lro_rope_tables(1, 2, 1e4, 1, 0, 0, 0, nullptr, x) == LR_ERROR_INVALID_ARGUMENT,
         "no table");
}

} // namespace

int main() {
  check_dividers();
  check_refusals();
  std::printf("sizes: rope_append %zu paged_attention %zu fork %zu compact %zu copy %zu beam %zu\n",
              sizeof(lro_rope_append_t), sizeof(lro_paged_attention_t), sizeof(lro_pages_fork_t),
              sizeof(lro_pages_compact_t), sizeof(lro_pages_copy_t), sizeof(lro_beam_select_t));
  std::printf("ops host checks: ok\n");
  return 0;
}
