// The options of newton_schulz in the C++ mirror (include/batchlas_b200.hh): bfloat16 with pairs of halves and with single ones, its
// refusal for other types.  `--compile-only-check` exits before touching a GPU.
#include <batchlas_b200.hh>

#include <cmath>
#include <cstdio>
#include <cstring>

using namespace batchlas;
using bf16 = __nv_bfloat16;

int main(int argc, char** argv) {
  if (argc > 1 && std::strcmp(argv[1], "--compile-only-check") == 0) {
    std::puts("compiled: overload set resolves");
    return 0;
  }
  const int r = 40, c = 56;
  Queue ctx(Device::default_device());
  bf16* data = nullptr;
  detail::cuda_check(cudaMallocManaged(&data, 3 * r * c * sizeof(bf16)), "managed");
  bf16 *x = data, *pairs = data + r * c, *halves = pairs + r * c;
  unsigned state = 5;
  for (int i = 0; i < r * c; ++i) {
    state = state * 1664525u + 1013904223u;
    x[i] = bf16((float)(state >> 8) / 8388608.f - 1.f);
  }
  MatrixView<bf16> X(x, r, c);
  newton_schulz<bf16>(ctx, X, MatrixView<bf16>(pairs, r, c));
  newton_schulz<bf16>(ctx, X, MatrixView<bf16>(halves, r, c), {.half_intermediates = true});
  ctx.wait();
  double size = 0, apart = 0;
  for (int i = 0; i < r * c; ++i) {
    const double p = (double)(float)pairs[i], h = (double)(float)halves[i];
    size += p * p;
    apart += (p - h) * (p - h);
  }
  // Both are rounded by at most 2^-8 of each element; fifteen stores of 2^-11, amplified by at most 3.4445 a step, part them further.
  double stores = 0;
  for (int i = 0; i < 5; ++i) stores = 3.4445 * stores + 3 * std::ldexp(1.0, -11);
  int failed = 0;
  if (!(apart > 0) || !(std::sqrt(apart) <= (std::ldexp(2.0, -8) + stores) * std::sqrt(size))) ++failed;
  bool refused = false;
  try {
    float* f = reinterpret_cast<float*>(data);
    newton_schulz<float>(ctx, MatrixView<float>(f, 8, 8), MatrixView<float>(f, 8, 8), {.half_intermediates = true});
  } catch (const std::exception&) {
    refused = true;
  }
  if (!refused) ++failed;
  cudaFree(data);
  std::printf("relative difference %.2e, %d failed\n", std::sqrt(apart / size), failed);
  return failed ? 1 : 0;
}
