// What the C++ layer's calls for serving in fewer bits refuse before anything reaches a GPU: members that do not fit together.
#include <cstdio>

#include "irontensor_b200.hpp"

static int failures = 0;

template <typename F>
static void refused(F&& f, const char* text, const char* what) {
  try {
    f();
  } catch (const std::logic_error& e) {
    if (std::string(e.what()).find(text) != std::string::npos) return;
  } catch (const std::exception&) {
  }
  std::printf("FAIL: %s\n", what);
  ++failures;
}

int main() {
  const it::Array<int32_t> none;
  const it::Tensor x;
  it::QuantizedCache c;   // sizes without buffers
  c.batch = 2, c.max_len = 8, c.kv_heads = 2, c.head_dim = 64;
  refused([&] { it::kv_cache_append(c, x, x, none); }, "of the cache's sizes", "append");
  refused([&] { it::kv_cache_read(c, 1); }, "of the cache's sizes", "read");
  refused([&] { it::attention_decode_quantized(x, c, none); }, "of the cache's sizes", "attention");
  c.max_len = size_t{1} << 32;
  refused([&] { it::kv_cache_read(c, 1); }, "below 2^31", "a cache of 2^32 positions");
  c.max_len = 8, c.head_dim = 60;
  refused([&] { it::kv_cache_read(c, 1); }, "multiple of 8", "head_dim");
  it::QuantizedRows a, b;
  a.rows = 3, a.cols = b.cols = 16;
  refused([&] { it::linear_int8_forward(a, b); }, "of the rows' sizes", "rows without codes");
  refused([&] { it::linear_int8_forward(b, a); }, "of the rows' sizes", "weights without codes");
  std::printf(failures == 0 ? "refusals: all checks passed\n" : "refusals: %d check(s) failed\n", failures);
  return failures == 0 ? 0 : 1;
}
