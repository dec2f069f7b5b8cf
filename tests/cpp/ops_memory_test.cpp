// C entries while memory for their texts and handles runs out: they return an
// error, and no exception leaves them. With the argument "gpu" those that need a
// device too.
#include "lrrt_ops.h"

#include "lrrt/interop.h"

#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <new>

namespace {

long g_left = -1; // allocations that still succeed; -1: all of them

void expect(bool condition, const char *what) {
  if (!condition) {
    std::fprintf(stderr, "failed: %s\n", what);
    std::exit(1);
  }
}

// The call with no, one, two ... allocations left.
template <typename Call> void each_failing(Call call, const char *what) {
  for (long n = 0; n < 12; ++n) {
    g_left = n;
    const lr_status_t status = call();
    g_left = -1;
    expect(status != LR_SUCCESS, what);
  }
}

void wrap_a_stream() {
  expect(lr_init() == LR_SUCCESS, "lr_init");
  lr_device_t device{};
  expect(lr_device_open(0, &device) == LR_SUCCESS, "lr_device_open");
  lr_queue_t *queue = nullptr;
  for (long n = 0;; ++n) {
    g_left = n;
    const lr_status_t status = lr_queue_wrap_stream(device, nullptr, &queue);
    g_left = -1;
    if (status == LR_SUCCESS) {
      expect(n > 0, "a queue takes memory");
      break;
    }
    expect(queue == nullptr && n < 100, "a queue that could not be made");
  }
  expect(lr_queue_destroy(queue) == LR_SUCCESS, "lr_queue_destroy");
}

} // namespace

void *operator new(size_t size) {
  if (g_left == 0) {
    throw std::bad_alloc();
  }
  g_left -= g_left > 0 ? 1 : 0;
  void *memory = std::malloc(size);
  if (memory == nullptr) {
    throw std::bad_alloc();
  }
  return memory;
}
void operator delete(void *memory) noexcept { std::free(memory); }
void operator delete(void *memory, size_t) noexcept { std::free(memory); }

int main(int count, char **arguments) {
  float x[8];
  lro_context_t *context = nullptr;
  each_failing([&] { return lro_rope_tables(1, 3, 1e4, 1, 0, 0, 0, x, x); }, "an odd rotary_dim");
  each_failing([&] { return lro_paged_attention(nullptr, nullptr); }, "no context");
  each_failing([&] { return lro_context_reserve(nullptr, 1); }, "nothing to reserve in");
  each_failing([&] { return lro_context_create(lr_device_t{0}, nullptr, "no module", 9, &context); },
               "no module");
  expect(lro_rope_tables(1, 3, 1e4, 1, 0, 0, 0, x, x) == LR_ERROR_INVALID_ARGUMENT &&
             std::strstr(lro_last_error(), "rotary_dim") != nullptr,
         "texts as before");
  if (count > 1 && std::strcmp(arguments[1], "gpu") == 0) {
    wrap_a_stream();
  }
  std::printf("ops without memory: ok\n");
  return 0;
}
