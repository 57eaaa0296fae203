// A C++ client of HashTable::find_layer_norm: rows of the table normalised on
// their way out, against the formula in 64 bits on the host.  Prints PASS and
// exits 0 when every check holds.
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <memory>
#include <vector>

#include "merlin_hashtable.cuh"

using K = uint64_t;
using S = uint64_t;

#define EXPECT(cond)                                              \
  do {                                                            \
    if (!(cond)) {                                                \
      std::printf("FAIL %s:%d: %s\n", __FILE__, __LINE__, #cond); \
      std::exit(1);                                               \
    }                                                             \
  } while (0)
#define CUDA_OK(call) EXPECT((call) == cudaSuccess)

template <class T>
struct Device {
  T* p = nullptr;
  size_t n;
  explicit Device(const std::vector<T>& v) : n(v.size()) {
    CUDA_OK(cudaMalloc(&p, n * sizeof(T)));
    CUDA_OK(cudaMemcpy(p, v.data(), n * sizeof(T), cudaMemcpyHostToDevice));
  }
  std::vector<T> host() const {
    std::vector<T> v(n);
    CUDA_OK(cudaMemcpy(v.data(), p, n * sizeof(T), cudaMemcpyDeviceToHost));
    return v;
  }
  ~Device() { cudaFree(p); }
};

template <class V, class P>
void check(const size_t dim, const double half_step) {
  constexpr size_t kStored = 1000, kAsked = 1200;   // the last 200 are misses
  nv::merlin::HashTableOptions options;
  options.init_capacity = options.max_capacity = 128 * 64;
  options.max_hbm_for_vectors = 1ull << 30;
  options.dim = dim;
  nv::merlin::HashTable<K, V, S> table;
  table.init(options);
  std::vector<K> keys(kAsked);
  std::vector<V> rows(kStored * dim);
  std::vector<P> weight(dim), bias(dim);
  for (size_t i = 0; i < kAsked; ++i) keys[i] = 7 * i + 1;
  for (size_t i = 0; i < rows.size(); ++i) rows[i] = V(float((i * 2654435761u >> 8) % 1000) / 500.f - 1.f);
  for (size_t i = 0; i < dim; ++i) {
    weight[i] = P(1.f + float(i % 8) / 16.f);
    bias[i] = P(float(i % 4) / 4.f);
  }
  Device<K> d_keys(keys);
  Device<V> d_rows(rows), d_out(std::vector<V>(kAsked * dim, V(5.f)));
  Device<P> d_weight(weight), d_bias(bias);
  Device<char> d_found(std::vector<char>(kAsked, 2));
  Device<float> d_mean(std::vector<float>(kAsked, 5.f)), d_rstd(std::vector<float>(kAsked, 5.f));
  table.insert_or_assign(kStored, d_keys.p, d_rows.p);
  const float eps = 1e-5f;
  table.find_layer_norm(kAsked, d_keys.p, d_weight.p, d_bias.p, eps, d_out.p,
                        reinterpret_cast<bool*>(d_found.p), d_mean.p, d_rstd.p);
  CUDA_OK(cudaDeviceSynchronize());
  const auto out = d_out.host();
  const auto found = d_found.host();
  const auto mean = d_mean.host(), rstd = d_rstd.host();
  // elements lie within [-1, 1]: each of the about 2 * dim + 16 operations of a
  // row's sums is off by at most 2^-24 of a value below 2 times rstd, and the
  // result is rounded once
  const double step = std::ldexp(1.0, -24);
  for (size_t i = 0; i < kAsked; ++i) {
    EXPECT(found[i] == (i < kStored));
    if (i >= kStored) {
      EXPECT(mean[i] == 5.f && rstd[i] == 5.f);
      for (size_t j = 0; j < dim; ++j) EXPECT(float(out[i * dim + j]) == 5.f);
      continue;
    }
    double m = 0, v = 0;
    for (size_t j = 0; j < dim; ++j) m += double(float(rows[i * dim + j])) / double(dim);
    for (size_t j = 0; j < dim; ++j) {
      const double d = double(float(rows[i * dim + j])) - m;
      v += d * d / double(dim);
    }
    const double r = 1 / std::sqrt(v + double(eps));
    const double off = (2 * double(dim) + 16) * step;
    EXPECT(std::fabs(mean[i] - m) <= off);
    EXPECT(std::fabs(rstd[i] - r) <= off * r * (1 + r));
    for (size_t j = 0; j < dim; ++j) {
      const double w = double(float(weight[j])), b = double(float(bias[j]));
      const double want = (double(float(rows[i * dim + j])) - m) * r * w + b;
      EXPECT(std::fabs(double(float(out[i * dim + j])) - want) <=
             half_step * std::fabs(want) + 4 * off * r * (1 + r) * w);
    }
  }
}

int main() {
  check<float, float>(64, std::ldexp(1.0, -24));
  check<float, float>(33, std::ldexp(1.0, -24));
  check<__half, __half>(64, std::ldexp(1.0, -11));
  check<__half, float>(40, std::ldexp(1.0, -11));
  check<__nv_bfloat16, float>(64, std::ldexp(1.0, -8));
  // what the table or the call does not allow is an exception
  nv::merlin::HashTableOptions options;
  options.init_capacity = options.max_capacity = 128 * 8;
  options.max_hbm_for_vectors = 1ull << 30;
  options.dim = 8;
  nv::merlin::HashTable<K, double, S> doubles;
  doubles.init(options);
  Device<K> key(std::vector<K>(1, 1));
  Device<double> row(std::vector<double>(8, 0.0));
  Device<char> found(std::vector<char>(1, 0));
  bool refused = false;
  try {
    doubles.find_layer_norm<float>(1, key.p, nullptr, nullptr, 1e-5f, row.p,
                                   reinterpret_cast<bool*>(found.p));
  } catch (const std::exception&) {
    refused = true;
  }
  EXPECT(refused);
  std::printf("PASS\n");
  return 0;
}
