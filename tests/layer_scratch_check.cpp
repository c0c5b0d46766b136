// Host-only check of the learned layers' scratch queries: over many shapes, what a backward pass with
// any part of its gradients takes is at most what the query says.  Linked with the library's objects;
// makes no CUDA call (a pass without a context only counts).
#include <cmath>
#include <cstdio>
#include <random>

#include "af2_internal.h"

using namespace af2;

namespace {

void *const kAnywhere = reinterpret_cast<void *>(uintptr_t(4)), *const kAligned = reinterpret_cast<void *>(uintptr_t(256));
int failures = 0, checked = 0;

void check(const char *what, int64_t a, int64_t b, int64_t c, int dtype, int activation, unsigned need, uint64_t said,
           uint64_t takes) {
  ++checked;
  if (takes <= said) return;
  if (++failures <= 10)
    std::printf("%s %lld x %lld -> %lld, type %d, activation %d, gradients %u: takes %llu, the query says %llu\n", what,
                static_cast<long long>(a), static_cast<long long>(b), static_cast<long long>(c), dtype, activation, need,
                static_cast<unsigned long long>(takes), static_cast<unsigned long long>(said));
}

void dense_shape(int64_t rows, int64_t inner, int64_t columns, int dtype, int activation) {
  const af2_linear_shape shape{rows, inner, columns};
  uint64_t said = 0;
  if (af2_dense_workspace_bytes(&shape, dtype, activation, 1, &said) != AF2_OK) ++failures;
  for (void *at : {kAnywhere, kAligned})
    for (unsigned need = 1; need < 8; ++need) {
      auto want = [&](int bit) { return need >> bit & 1 ? at : nullptr; };
      uint64_t takes = 0;
      dense_backward(nullptr,
                     {rows, inner, columns, dtype, activation, at, at, at, at, columns, inner, inner, want(0), want(1), want(2)},
                     nullptr, &takes, nullptr);
      check("dense", rows, inner, columns, dtype, activation, need, said, takes);
    }
  if (af2_dense_workspace_bytes(&shape, dtype, activation, 0, &said) != AF2_OK) ++failures;
  for (void *at : {kAnywhere, kAligned})
    for (void *saved : {static_cast<void *>(nullptr), at}) {
      uint64_t takes = 0;
      dense_forward(nullptr, {rows, inner, columns, dtype, activation, at, at, at, at, inner, columns, columns, at, saved},
                    nullptr, &takes, nullptr);
      check("dense forward", rows, inner, columns, dtype, activation, saved != nullptr, said, takes);
    }
}

void gated_shape(int64_t rows, int64_t channels, int64_t hidden, int dtype) {
  const af2_transition_shape shape{rows, channels, hidden};
  uint64_t said = 0;
  if (af2_gated_transition_workspace_bytes(&shape, dtype, 1, &said) != AF2_OK) ++failures;
  for (void *at : {kAnywhere, kAligned})
    for (unsigned need = 1; need < 128; ++need) {
      auto want = [&](int bit) { return need >> bit & 1 ? at : nullptr; };
      const af2_gated_weights w{at, at, at, at, at, at};
      uint64_t takes = 0;
      gated_backward(nullptr,
                     {rows, channels, hidden, dtype, 0, at, at, at, w,
                      {want(0), want(1), want(2), want(3), want(4), want(5), want(6)}, channels, channels, channels},
                     nullptr, &takes, nullptr);
      check("gated", rows, channels, hidden, dtype, 0, need, said, takes);
    }
  if (af2_gated_transition_workspace_bytes(&shape, dtype, 0, &said) != AF2_OK) ++failures;
  for (void *at : {kAnywhere, kAligned})
    for (void *saved : {static_cast<void *>(nullptr), at}) {
      const af2_gated_weights w{at, at, at, at, at, at};
      uint64_t takes = 0;
      gated_forward(nullptr, {rows, channels, hidden, dtype, 0, at, at, w, channels, channels, channels, at, saved}, nullptr,
                    &takes, nullptr);
      check("gated forward", rows, channels, hidden, dtype, 0, saved != nullptr, said, takes);
    }
}

}  // namespace

int main() {
  std::mt19937_64 rng(7);
  auto size = [&](double low, double high) {  // spread over the logarithm
    return static_cast<int64_t>(low * std::pow(high / low, std::uniform_real_distribution<>(0, 1)(rng)) + 0.5);
  };
  const int types[] = {AF2_F32, AF2_F16, AF2_BF16};
  dense_shape(2048, 768, 3000, AF2_F32, AF2_ACTIVATION_SILU);
  dense_shape(30224, 293, 1909, AF2_F32, AF2_ACTIVATION_GELU);
  dense_shape(2048, 512, 512, AF2_BF16, AF2_ACTIVATION_NONE);
  gated_shape(2048, 1024, 4096, AF2_BF16);
  for (int i = 0; i < 400; ++i) {
    int64_t rows = size(1, 300000), a = size(1, 4096), b = size(1, 8192);
    if (rng() & 1) a = (a + 7) / 8 * 8, b = (b + 7) / 8 * 8;
    const int dtype = types[rng() % 3];
    dense_shape(rows, a, b, dtype, static_cast<int>(rng() % 5));
    if (i % 4 == 0) gated_shape(rows, a, b, dtype);
  }
  if (failures) {
    std::printf("%d of %d failed\n", failures, checked);
    return 1;
  }
  std::printf("ok\n");
  return 0;
}
