// The 8-bit product, its quantiser and the Newton-Schulz orthogonalisation through the C++ mirror
// (include/batchlas_b200.hh), against naive host loops in double.
// Build as gemm_api_tests.cc; `--compile-only-check` exits before touching a GPU.
#include <batchlas_b200.hh>

#include <cmath>
#include <cstdio>
#include <cstring>
#include <functional>

using namespace batchlas;

static int g_failed = 0, g_run = 0;
#define CHECK(cond)                                                         \
  do {                                                                      \
    if (!(cond)) {                                                          \
      std::printf("  CHECK failed %s:%d: %s\n", __FILE__, __LINE__, #cond); \
      ++g_failed;                                                           \
      return;                                                               \
    }                                                                       \
  } while (0)

template <typename T>
struct Managed {
  T* p = nullptr;
  size_t n;
  explicit Managed(size_t count) : n(count) { detail::cuda_check(cudaMallocManaged(&p, count * sizeof(T)), "managed"); }
  ~Managed() { cudaFree(p); }
  Managed(const Managed&) = delete;
  T& operator[](size_t i) { return p[i]; }
};

static float noise(unsigned& state) {
  state = state * 1664525u + 1013904223u;
  return (float)(state >> 8) / 8388608.f - 1.f;
}

template <typename T>
void QuantiseAndMultiply(Queue& ctx) {
  const int m = 48, n = 20, k = 80, batch = 2;
  Managed<float> W((size_t)m * k * batch), sw(m * batch), sx(n * batch);
  Managed<T> X((size_t)n * k * batch), C((size_t)m * n * batch);
  Managed<int8_t> Wq(W.n), Xq(X.n);
  unsigned state = 7;
  for (size_t i = 0; i < W.n; ++i) W[i] = noise(state);
  for (size_t i = 0; i < X.n; ++i) X[i] = T(noise(state));
  quantize_i8<float>(ctx, MatrixView<float>(W.p, k, m, k, (int64_t)m * k, batch), MatrixView<int8_t>(Wq.p, k, m, k, (int64_t)m * k, batch),
                     VectorView<float>(sw.p, m, batch));
  quantize_i8<T>(ctx, MatrixView<T>(X.p, k, n, k, (int64_t)n * k, batch), MatrixView<int8_t>(Xq.p, k, n, k, (int64_t)n * k, batch),
                 VectorView<float>(sx.p, n, batch));
  gemm_i8<T>(ctx, MatrixView<int8_t>(Wq.p, k, m, k, (int64_t)m * k, batch), MatrixView<int8_t>(Xq.p, k, n, k, (int64_t)n * k, batch),
             MatrixView<T>(C.p, m, n, m, (int64_t)m * n, batch), VectorView<float>(sw.p, m, batch), VectorView<float>(sx.p, n, batch),
             {.alpha = 2.0});
  ctx.wait();
  // half a step of the type, and four roundings in float
  const double step = std::is_same_v<T, float> ? std::ldexp(1.0, -24) : std::is_same_v<T, __half> ? std::ldexp(1.0, -11) : std::ldexp(1.0, -8);
  for (int b = 0; b < batch; ++b)
    for (int j = 0; j < m; ++j) {
      float top = 0;
      for (int l = 0; l < k; ++l) top = std::max(top, std::fabs(W[((size_t)b * m + j) * k + l]));
      CHECK(sw[b * m + j] == top * (1.f / 127.f));
      for (int l = 0; l < k; ++l)
        CHECK((float)Wq[((size_t)b * m + j) * k + l] == std::nearbyint(W[((size_t)b * m + j) * k + l] / sw[b * m + j]));
    }
  for (int b = 0; b < batch; ++b)
    for (int i = 0; i < n; ++i)
      for (int j = 0; j < m; ++j) {
        long sum = 0;
        for (int l = 0; l < k; ++l) sum += (long)Wq[((size_t)b * m + j) * k + l] * Xq[((size_t)b * n + i) * k + l];
        const double want = 2.0 * (double)sum * sw[b * m + j] * sx[b * n + i];
        CHECK(std::fabs((double)(float)C[((size_t)b * n + i) * m + j] - want) <= std::fabs(want) * (step + std::ldexp(5.0, -24)) + 1e-7);
      }
}

void OrthogonaliseInPlace(Queue& ctx) {
  const int r = 24, c = 40, batch = 2;
  Managed<float> X((size_t)r * c * batch);
  unsigned state = 3;
  for (size_t i = 0; i < X.n; ++i) X[i] = noise(state);
  std::vector<double> want(X.n);
  for (int b = 0; b < batch; ++b) {
    std::vector<double> x(r * c), s(r * r), t(r * r), y(r * c);
    double norm = 0;
    for (int i = 0; i < r * c; ++i) norm += (double)X[b * r * c + i] * X[b * r * c + i];
    for (int i = 0; i < r * c; ++i) x[i] = X[b * r * c + i] / (std::sqrt(norm) + 1e-7);
    for (int step = 0; step < 8; ++step) {  // the cubic iteration: all singular values go to one
      for (int i = 0; i < r; ++i)
        for (int j = 0; j < r; ++j) {
          s[j * r + i] = 0;
          for (int l = 0; l < c; ++l) s[j * r + i] += x[l * r + i] * x[l * r + j];
        }
      for (int i = 0; i < r; ++i)
        for (int l = 0; l < c; ++l) {
          y[l * r + i] = 1.5 * x[l * r + i];
          for (int j = 0; j < r; ++j) y[l * r + i] -= 0.5 * s[j * r + i] * x[l * r + j];
        }
      x = y;
    }
    std::copy(x.begin(), x.end(), want.begin() + b * r * c);
  }
  MatrixView<float> V(X.p, r, c, r, (int64_t)r * c, batch);
  newton_schulz<float>(ctx, V, V, {.steps = 8, .coefficients = {1.5, -0.5, 0.0}});
  ctx.wait();
  // eight steps whose polynomial amplifies an error by at most 1.5, three stores of 2^-22 each per step and sums of 40 terms
  double off = 0, size = 0;
  for (size_t i = 0; i < X.n; ++i) {
    off += (X[i] - want[i]) * (X[i] - want[i]);
    size += want[i] * want[i];
  }
  double allowed = 0;
  for (int step = 0; step < 8; ++step) allowed = 1.5 * allowed + 3 * (std::ldexp(1.0, -22) + 12 * std::ldexp(1.0, -24));
  CHECK(std::sqrt(off) <= allowed * std::sqrt(size));
}

void Errors(Queue& ctx) {
  Managed<float> X(64), s(8);
  Managed<int8_t> Q(64);
  auto throws = [](auto f) {
    try {
      f();
    } catch (const std::exception&) {
      return true;
    }
    return false;
  };
  MatrixView<float> V(X.p, 8, 8);
  MatrixView<int8_t> W(Q.p, 8, 8);
  CHECK(throws([&] { quantize_i8<float>(ctx, V, MatrixView<int8_t>(Q.p, 8, 4), VectorView<float>(s.p, 8)); }));
  CHECK(throws([&] { quantize_i8<float>(ctx, V, W, VectorView<float>(s.p, 7)); }));
  CHECK(throws([&] { gemm_i8<float>(ctx, W, MatrixView<int8_t>(Q.p, 4, 8), V, {}, {}); }));
  CHECK(throws([&] { newton_schulz<float>(ctx, V, MatrixView<float>(X.p, 4, 8)); }));
  CHECK(throws([&] { newton_schulz<float>(ctx, V, V, {.steps = 0}); }));
  CHECK(throws([&] { newton_schulz<float>(ctx, V, V, {.coefficients = {9.0, 0.0, 0.0}}); }));
}

int main(int argc, char** argv) {
  if (argc > 1 && std::strcmp(argv[1], "--compile-only-check") == 0) {
    std::puts("compiled: overload set resolves");
    return 0;
  }
  Queue ctx(Device::default_device());
  auto run = [&](const char* name, std::function<void()> f) {
    const int before = g_failed;
    ++g_run;
    try {
      f();
    } catch (const std::exception& e) {
      std::printf("  exception: %s\n", e.what());
      ++g_failed;
    }
    std::printf("[%s] %s\n", g_failed == before ? " OK " : "FAIL", name);
  };
  run("QuantiseAndMultiply<float>", [&] { QuantiseAndMultiply<float>(ctx); });
  run("QuantiseAndMultiply<half>", [&] { QuantiseAndMultiply<__half>(ctx); });
  run("QuantiseAndMultiply<bfloat16>", [&] { QuantiseAndMultiply<__nv_bfloat16>(ctx); });
  run("OrthogonaliseInPlace", [&] { OrthogonaliseInPlace(ctx); });
  run("Errors", [&] { Errors(ctx); });
  std::printf("%d test groups, %d failed\n", g_run, g_failed);
  return g_failed ? 1 : 0;
}
