// The C++ layer's calls for serving in fewer bits: a generation step of a ragged batch, from quantised weights to attention over the
// 4-bit cache, against plain loops in double on the values that are held.
#include <cmath>
#include <cstdio>
#include <vector>

#include "irontensor_b200.hpp"

using it::Precision;
using it::Tensor;

static int failures = 0;
#define EXPECT(cond, what)                                        \
  do {                                                            \
    if (!(cond)) {                                                \
      std::printf("FAIL: %s (%s:%d)\n", what, __FILE__, __LINE__); \
      ++failures;                                                 \
    }                                                             \
  } while (0)

template <typename F>
static bool refuses(F&& f, const char* text) {
  try {
    f();
  } catch (const std::exception& e) {
    return std::string(e.what()).find(text) != std::string::npos;
  }
  return false;
}

int main() {
  try {
    const size_t B = 3, H = 4, Hkv = 2, D = 40, in = 64, max_len = 20, out = (H + 2 * Hkv) * D;
    const std::vector<int32_t> at = {0, 7, 18};
    std::vector<float> x(B * in), w(out * in), old(B * max_len * Hkv * D);
    for (size_t i = 0; i < x.size(); ++i) x[i] = std::sin(0.37f * i);
    for (size_t i = 0; i < w.size(); ++i) w[i] = 0.2f * std::cos(0.11f * i);
    for (size_t i = 0; i < old.size(); ++i) old[i] = std::sin(0.05f * i * (1 + i % 7));
    const it::QuantizedRows qx = it::quantize_rows(Tensor::from_f32_slice(x, {B, in})), qw = it::quantize_rows(Tensor::from_f32_slice(w, {out, in}));
    const std::vector<Tensor> qkv = it::linear_int8_forward(qx, qw, {H * D, Hkv * D, Hkv * D}, Precision::FP32);
    const Tensor y = it::linear_int8_forward(qx, qw, Precision::FP32);
    {
      const std::vector<int8_t> cx = qx.codes.to_host(), cw = qw.codes.to_host();
      const std::vector<float> sx = qx.scales.to_host(), sw = qw.scales.to_host(), got = y.to_host_f32(), q = qkv[0].to_host_f32(), v = qkv[2].to_host_f32();
      bool held = true, right = true, split = true;
      for (size_t i = 0; i < x.size(); ++i) held = held && std::fabs(cx[i] * sx[i / in] - x[i]) <= 0.502 * sx[i / in];
      for (size_t b = 0; b < B; ++b)
        for (size_t o = 0; o < out; ++o) {
          int sum = 0;
          for (size_t i = 0; i < in; ++i) sum += cx[b * in + i] * cw[o * in + i];
          const double want = static_cast<double>(sum) * sx[b] * sw[o];   // exact but for three roundings to fp32
          right = right && std::fabs(got[b * out + o] - want) <= 3 * std::ldexp(std::fabs(want), -24);
          if (o < H * D) split = split && q[b * H * D + o] == got[b * out + o];
          if (o >= (H + Hkv) * D) split = split && v[b * Hkv * D + o - (H + Hkv) * D] == got[b * out + o];
        }
      EXPECT(held, "rows are held to half a step (and a scale rounded down by up to 2^-9)");
      EXPECT(right, "8-bit projection");
      EXPECT(split, "column ranges");
    }
    const it::Array<int32_t> lengths = it::Array<int32_t>::from_host(at);
    const auto turned = it::rope_positions(qkv[0].view({B, 1, H, D}), qkv[1].view({B, 1, Hkv, D}), lengths);
    const auto back = it::rope_positions(turned.first, turned.second, lengths, 10000.f, {}, false, true);
    {
      const std::vector<float> a = qkv[1].to_host_f32(), b = back.second.to_host_f32(), c = turned.second.to_host_f32();
      double diff = 0, norm = 0;
      for (size_t i = 0; i < a.size(); ++i) {
        diff = std::max(diff, std::fabs(static_cast<double>(a[i]) - b[i]));
        norm = std::max(norm, std::fabs(static_cast<double>(a[i])));
      }
      EXPECT(diff <= 8 * std::ldexp(norm, -24) * std::sqrt(2.0), "turned and turned back");
      bool first = true;   // position 0 stays
      for (size_t i = 0; i < Hkv * D; ++i) first = first && a[i] == c[i];
      EXPECT(first, "position 0 is the identity");
      EXPECT(it::rope_positions(turned.first, Tensor(), lengths).second.shape().empty(), "q alone");
    }
    const it::QuantizedCache cache = it::QuantizedCache::zeros(B, max_len, Hkv, D);
    const Tensor told = Tensor::from_f32_slice(old, {B, max_len, Hkv, D});
    EXPECT(it::kv_cache_append(cache, told, told, it::Array<int32_t>::from_host({0, 0, 0}), &lengths).to_host() == at, "a padded batch's lengths");
    const it::Array<int32_t> now = it::kv_cache_append(cache, turned.second, qkv[2].view({B, 1, Hkv, D}), lengths);
    EXPECT(now.to_host() == std::vector<int32_t>({1, 8, 19}), "new lengths");
    const Tensor tq = turned.first.view({B, H, D});
    const Tensor o = it::attention_decode_quantized(tq, cache, now);
    {
      const auto held = it::kv_cache_read(cache, max_len, nullptr, &now, Precision::FP32);
      const std::vector<float> k = held.first.to_host_f32(), v = held.second.to_host_f32(), q = tq.to_host_f32(), got = o.to_host_f32(), lse = o.lse->to_host_f32();
      double worst = 0, worst_lse = 0;
      for (size_t b = 0; b < B; ++b)
        for (size_t h = 0; h < H; ++h) {
          const size_t n = at[b] + 1, g = h / (H / Hkv);
          std::vector<double> s(n), sum_o(D, 0.0);
          double sum = 0, most = -1e300;
          for (size_t t = 0; t < n; ++t) {
            double dot = 0;
            for (size_t d = 0; d < D; ++d) dot += static_cast<double>(q[(b * H + h) * D + d]) * k[((b * max_len + t) * Hkv + g) * D + d];
            s[t] = dot / std::sqrt(static_cast<double>(D));
            most = std::max(most, s[t]);
          }
          for (size_t t = 0; t < n; ++t) {
            const double p = std::exp(s[t] - most);
            sum += p;
            for (size_t d = 0; d < D; ++d) sum_o[d] += p * v[((b * max_len + t) * Hkv + g) * D + d];
          }
          for (size_t d = 0; d < D; ++d) worst = std::max(worst, std::fabs(got[(b * H + h) * D + d] - sum_o[d] / sum));
          worst_lse = std::max(worst_lse, std::fabs(lse[b * H + h] - (most + std::log(sum))));
        }
      // scores of at most 40 products and a magnitude below 32 in fp32, twice through exp, values below 2
      EXPECT(worst <= std::ldexp(1.0, -13) && worst_lse <= std::ldexp(1.0, -15), "attention over the cache");
      bool zeros = true;
      for (size_t i = 1 * Hkv * D; i < max_len * Hkv * D; ++i) zeros = zeros && k[i] == 0.f;
      EXPECT(zeros, "positions behind a sequence read as zeros");
    }
    EXPECT(refuses([&] { it::attention_decode_quantized(tq, it::QuantizedCache::zeros(B, max_len, 3, D), now); }, "divisible"), "heads");
    EXPECT(refuses([&] { it::kv_cache_append(cache, told, qkv[2], lengths); }, "same shape"), "shapes of k and v");
    EXPECT(refuses([&] { it::QuantizedCache::zeros(1, 1, 1, 84); }, "multiple of 8"), "head_dim");
    EXPECT(refuses([&] { it::linear_int8_forward(qx, qw, {8, 8}); }, "add up"), "widths");
    EXPECT(refuses([&] { it::rope_positions(tq.view({B, 1, H, D}), Tensor(), lengths, 10000.f, {10, 10}); }, "positions must be"), "axes");
    EXPECT(refuses([&] {
             it::kv_cache_append(cache, turned.second, turned.second, it::Array<int32_t>::from_host({0, 20, 0}));
             it::CommandBatch::poll_device_status();
           }, "length lay outside"), "a full sequence is reported");
    it::CommandBatch::poll_device_status();
  } catch (const std::exception& e) {
    std::printf("FAIL: exception %s\n", e.what());
    return 2;
  }
  std::printf(failures == 0 ? "quantised serving: all checks passed\n" : "quantised serving: %d check(s) failed\n", failures);
  return failures == 0 ? 0 : 1;
}
