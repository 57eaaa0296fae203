// HashTable::find_layer_norm with null for the weight, the bias or both, written as
// a caller writes it: the other argument, or else the table's value type, says what
// type the null one has.  Prints PASS and exits 0 when the rows are the right ones.
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "merlin_hashtable.cuh"

using K = uint64_t;

#define EXPECT(cond)                                              \
  do {                                                            \
    if (!(cond)) {                                                \
      std::printf("FAIL %s:%d: %s\n", __FILE__, __LINE__, #cond); \
      std::exit(1);                                               \
    }                                                             \
  } while (0)

template <class T>
T* upload(const std::vector<T>& v) {
  T* p = nullptr;
  EXPECT(cudaMalloc(&p, v.size() * sizeof(T)) == cudaSuccess);
  EXPECT(cudaMemcpy(p, v.data(), v.size() * sizeof(T), cudaMemcpyHostToDevice) == cudaSuccess);
  return p;
}

// P: the type of the parameter that is given
template <class V, class P>
void check(const double half_step) {
  constexpr size_t kDim = 24, kKeys = 100;
  nv::merlin::HashTableOptions options;
  options.init_capacity = options.max_capacity = 128 * 8;
  options.max_hbm_for_vectors = 1ull << 30;
  options.dim = kDim;
  nv::merlin::HashTable<K, V, uint64_t> table;
  table.init(options);
  std::vector<K> keys(kKeys);
  std::vector<V> rows(kKeys * kDim);
  std::vector<P> given(kDim);
  for (size_t i = 0; i < kKeys; ++i) keys[i] = 3 * i + 1;
  for (size_t i = 0; i < rows.size(); ++i) rows[i] = V(float((i * 2654435761u >> 8) % 1000) / 500.f - 1.f);
  for (size_t j = 0; j < kDim; ++j) given[j] = P(1.f + float(j % 8) / 16.f);
  K* d_keys = upload(keys);
  V* d_rows = upload(rows);
  P* d_given = upload(given);
  V* d_out = upload(std::vector<V>(rows.size(), V(0.f)));
  bool* d_found = reinterpret_cast<bool*>(upload(std::vector<char>(kKeys, 0)));
  table.insert_or_assign(kKeys, d_keys, d_rows);
  const float eps = 1e-5f;
  // elements within [-1, 1], as in rows_test.cu: 2 * dim + 16 operations off by a step each
  const double off = (2 * double(kDim) + 16) * std::ldexp(1.0, -24);
  for (int form = 0; form < 3; ++form) {
    if (form == 0) table.find_layer_norm(kKeys, d_keys, nullptr, nullptr, eps, d_out, d_found);
    if (form == 1) table.find_layer_norm(kKeys, d_keys, d_given, nullptr, eps, d_out, d_found);
    if (form == 2) table.find_layer_norm(kKeys, d_keys, nullptr, d_given, eps, d_out, d_found);
    std::vector<V> out(rows.size());
    EXPECT(cudaMemcpy(out.data(), d_out, out.size() * sizeof(V), cudaMemcpyDeviceToHost) == cudaSuccess);
    for (size_t i = 0; i < kKeys; ++i) {
      double m = 0, v = 0;
      for (size_t j = 0; j < kDim; ++j) m += double(float(rows[i * kDim + j])) / double(kDim);
      for (size_t j = 0; j < kDim; ++j) v += std::pow(double(float(rows[i * kDim + j])) - m, 2) / double(kDim);
      const double r = 1 / std::sqrt(v + double(eps));
      for (size_t j = 0; j < kDim; ++j) {
        const double w = form == 1 ? double(float(given[j])) : 1., b = form == 2 ? double(float(given[j])) : 0.;
        const double want = (double(float(rows[i * kDim + j])) - m) * r * w + b;
        EXPECT(std::fabs(double(float(out[i * kDim + j])) - want) <=
               half_step * std::fabs(want) + 4 * off * r * (1 + r) * w);
      }
    }
  }
  cudaFree(d_keys);
  cudaFree(d_rows);
  cudaFree(d_given);
  cudaFree(d_out);
  cudaFree(d_found);
}

int main() {
  check<float, float>(std::ldexp(1.0, -24));
  check<__half, __half>(std::ldexp(1.0, -11));
  check<__half, float>(std::ldexp(1.0, -11));
  check<__nv_bfloat16, float>(std::ldexp(1.0, -8));
  std::printf("PASS\n");
  return 0;
}
