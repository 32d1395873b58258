// One attention block of a decoder on the library's entry points: 8-bit projection to q, k and v, append to a paged
// cache with the position rotation, attention of the new tokens over the cache, 8-bit projection back. Two steps: the
// prompts of three sequences, then one more token for each. Every step is checked against the same block in 64 bits on
// the host; the exit code is 0 if both agree.
//
//   decoder_block            (needs one MI355X)
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <random>
#include <vector>

#include "gpu_inference/linear_i8.h"
#include "gpu_inference/paged_kv.h"
#include "gpu_inference/reference.h"
#include "gpu_inference/testing.h"

using namespace gie;

namespace {

constexpr int kHidden = 256, kHeads = 8, kKvHeads = 2, kDim = 64, kPage = 16, kMaxPages = 8, kPages = 24;
constexpr int kQkv = (kHeads + 2 * kKvHeads) * kDim;
const float kBase = 10000.f;

template <typename T>
DeviceBuffer upload(const std::vector<T>& v) {
  DeviceBuffer b(v.size() * sizeof(T));
  GIE_HIP_CHECK(hipMemcpy(b.data(), v.data(), v.size() * sizeof(T), hipMemcpyHostToDevice));
  return b;
}

// 8-bit weights [out][in] with one scale for each row, on the host and on the device
struct Weights {
  int in, out;
  std::vector<int8_t> w;
  std::vector<float> scale;
  DeviceBuffer dw, ds;
  Weights(int in_, int out_, std::mt19937& rng) : in(in_), out(out_), w(size_t(in_) * out_), scale(out_) {
    std::uniform_int_distribution<int> value(-127, 127);
    std::uniform_real_distribution<float> size(0.5f, 1.5f);
    for (auto& v : w) v = int8_t(value(rng));
    for (auto& s : scale) s = size(rng) / (73.f * std::sqrt(float(in)));
    dw = upload(w);
    ds = upload(scale);
  }
  // the layer in 64 bits, tokens quantized as the library does it
  std::vector<double> apply(const std::vector<double>& x, int tokens) const {
    std::vector<double> y(size_t(tokens) * out), q(in);
    for (int t = 0; t < tokens; ++t) {
      double most = 0;
      for (int k = 0; k < in; ++k) most = std::fmax(most, std::fabs(x[size_t(t) * in + k]));
      for (int k = 0; k < in; ++k) q[k] = std::nearbyint(x[size_t(t) * in + k] * 127 / most);
      for (int n = 0; n < out; ++n) {
        double sum = 0;
        for (int k = 0; k < in; ++k) sum += q[k] * w[size_t(n) * in + k];
        y[size_t(t) * out + n] = sum * (most / 127) * scale[n];
      }
    }
    return y;
  }
};

// the cache on the host: keys and values of each sequence in 64 bits, [position][kv head][dim]
struct HostCache {
  std::vector<double> k[3], v[3];
};

std::vector<double> attend(const std::vector<double>& qkv, const std::vector<int>& counts, HostCache& cache) {
  std::vector<double> out;
  const auto turn = [](const double* x, int position) {
    std::vector<double> y(kDim);
    for (int j = 0; j < kDim / 2; ++j) {
      const double a = position * std::pow(double(kBase), -2.0 * j / kDim), c = std::cos(a), s = std::sin(a);
      y[j] = x[j] * c - x[j + kDim / 2] * s;
      y[j + kDim / 2] = x[j] * s + x[j + kDim / 2] * c;
    }
    return y;
  };
  size_t row = 0;
  for (int b = 0; b < 3; ++b) {
    for (int i = 0; i < counts[b]; ++i, ++row) {
      const int position = int(cache.k[b].size() / (kKvHeads * kDim));
      const double* token = &qkv[row * kQkv];
      for (int h = 0; h < kKvHeads; ++h) {
        const auto k = turn(token + (kHeads + h) * kDim, position);
        cache.k[b].insert(cache.k[b].end(), k.begin(), k.end());
        const double* v = token + (kHeads + kKvHeads + h) * kDim;
        cache.v[b].insert(cache.v[b].end(), v, v + kDim);
      }
      for (int h = 0; h < kHeads; ++h) {
        const auto q = turn(token + h * kDim, position);
        const int kv = h / (kHeads / kKvHeads);
        std::vector<double> weight(position + 1);
        double most = -1e300, total = 0;
        for (int j = 0; j <= position; ++j) {
          double s = 0;
          for (int d = 0; d < kDim; ++d) s += q[d] * cache.k[b][(size_t(j) * kKvHeads + kv) * kDim + d];
          weight[j] = s / std::sqrt(double(kDim));
          most = std::fmax(most, weight[j]);
        }
        for (auto& w : weight) total += w = std::exp(w - most);
        for (int d = 0; d < kDim; ++d) {
          double o = 0;
          for (int j = 0; j <= position; ++j) o += weight[j] * cache.v[b][(size_t(j) * kKvHeads + kv) * kDim + d];
          out.push_back(o / total);
        }
      }
    }
  }
  return out;
}

}  // namespace

int main() {
  try {
    std::mt19937 rng(1234);
    std::normal_distribution<float> normal;
    const Weights w_qkv(kHidden, kQkv, rng), w_out(kHeads * kDim, kHidden, rng);
    const DeviceBuffer k_pages(size_t(kPages) * kKvHeads * kPage * kDim * 2), v_pages(k_pages.size());
    std::vector<int> table(3 * kMaxPages);
    for (int i = 0; i < 3 * kMaxPages; ++i) table[i] = (i * 7) % kPages;  // scattered, each page once
    const DeviceBuffer d_table = upload(table);
    std::vector<float> cos(size_t(kMaxPages) * kPage * kDim / 2), sin(cos.size());
    rotary_tables(kMaxPages * kPage, kDim, kBase, 1, 0, 1, cos.data(), sin.data());
    const DeviceBuffer d_cos = upload(cos), d_sin = upload(sin);

    HostCache cache;
    std::vector<int> lens(3, 0);
    bool good = true;
    for (const std::vector<int>& counts : {std::vector<int>{37, 1, 90}, std::vector<int>{1, 1, 1}}) {
      std::vector<int> starts(1, 0);
      int most_new = 0, most_len = 0;
      for (int b = 0; b < 3; ++b) {
        starts.push_back(starts.back() + counts[b]);
        lens[b] += counts[b];
        most_new = std::max(most_new, counts[b]);
        most_len = std::max(most_len, lens[b]);
      }
      const int tokens = starts.back();
      std::vector<float> hidden(size_t(tokens) * kHidden);
      for (auto& v : hidden) v = normal(rng);
      const DeviceBuffer x = upload_as(hidden, DataType::kFloat16);
      hidden = download_as_float(x.data(), DataType::kFloat16, int64_t(hidden.size()));  // as the layer sees them
      const DeviceBuffer qkv(size_t(tokens) * kQkv * 2), q(size_t(tokens) * kHeads * kDim * 2),
                         o(q.size()), y(size_t(tokens) * kHidden * 2), d_starts = upload(starts), d_lens = upload(lens);

      LinearI8Problem in, out;
      in.tokens = out.tokens = tokens;
      in.in_features = out.out_features = kHidden;
      in.out_features = kQkv;
      out.in_features = kHeads * kDim;
      PagedKvProblem kv;
      kv.batch = 3;
      kv.total_tokens = tokens;
      kv.q_heads = kHeads;
      kv.kv_heads = kKvHeads;
      kv.head_dim = kv.rotary_dim = kDim;
      kv.page_size = kPage;
      kv.num_pages = kPages;
      kv.max_pages = kMaxPages;
      kv.max_positions = kMaxPages * kPage;
      kv.max_new = most_new;
      kv.max_len = most_len;
      PagedKvProblem fused = kv;  // q, k and v lie in one row of the projection
      fused.q_stride = fused.k_stride = fused.v_stride = kQkv;
      const size_t bytes =
          std::max({LinearI8::workspace_size(in), LinearI8::workspace_size(out), PagedKv::workspace_size(kv)});
      const DeviceBuffer ws(bytes);

      const auto* d_q = static_cast<const uint16_t*>(qkv.data());
      const auto* i32 = static_cast<const int*>(d_starts.data());
      const auto* l32 = static_cast<const int*>(d_lens.data());
      const auto* t32 = static_cast<const int*>(d_table.data());
      LinearI8::forward(x.data(), nullptr, static_cast<const int8_t*>(w_qkv.dw.data()),
                        static_cast<const float*>(w_qkv.ds.data()), nullptr, in, qkv.data(), ws.data(), bytes, nullptr);
      PagedKv::append(d_q, d_q + kHeads * kDim, d_q + (kHeads + kKvHeads) * kDim,
                      static_cast<const float*>(d_cos.data()), static_cast<const float*>(d_sin.data()), i32, l32, t32,
                      fused, q.data(), k_pages.data(), v_pages.data(), nullptr);
      PagedKv::attention(q.data(), k_pages.data(), v_pages.data(), i32, l32, t32, kv, o.data(), ws.data(), bytes, nullptr);
      LinearI8::forward(o.data(), nullptr, static_cast<const int8_t*>(w_out.dw.data()),
                        static_cast<const float*>(w_out.ds.data()), nullptr, out, y.data(), ws.data(), bytes, nullptr);
      GIE_HIP_CHECK(hipDeviceSynchronize());

      const std::vector<float> got = download_as_float(y.data(), DataType::kFloat16, int64_t(tokens) * kHidden);
      const std::vector<double> first = w_qkv.apply(std::vector<double>(hidden.begin(), hidden.end()), tokens);
      const std::vector<double> want = w_out.apply(attend(first, counts, cache), tokens);
      double off = 0, norm = 0;
      for (size_t i = 0; i < want.size(); ++i) {
        off += (got[i] - want[i]) * (got[i] - want[i]);
        norm += want[i] * want[i];
      }
      // the second projection's 8 bits turn the 16-bit roundings before it into steps of 1/127 of a row's largest value
      // here and there: under half a percent of the result
      const double rel = std::sqrt(off / norm);
      std::printf("%d new tokens, longest sequence %d: rel L2 %.2e -> %s\n", tokens, most_len, rel,
                  rel <= 5e-3 ? "PASS" : "FAIL");
      good = good && rel <= 5e-3;
    }
    return good ? 0 : 1;
  } catch (const Error& e) {
    std::fprintf(stderr, "error: %s\n", e.what());
    return 2;
  }
}
