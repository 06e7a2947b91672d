// Orthogonalisation of a batch of matrices by Newton-Schulz products:
//     X <- G / (||G||_F + eps);  steps times:  S = X X^T (shorter side),  B = b S + c S^2,  X <- a X + B X.
// The sum of squares is taken in double, in a fixed order.
#include <math.h>

#include "lowp.cuh"
#include "ptx.cuh"

namespace blb200 {
namespace {

constexpr int kNormParts = 64;
constexpr double kMaxSigma = 64.0, kMaxEntry = 16384.0;

struct Matrices {
  void* p;
  int rows, cols, batch;
  long long ld, stride;
};

__device__ __forceinline__ double block_sum(double v) {
  __shared__ double part[8];
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0;
  for (int i = 0; i < 8; ++i) v += part[i];
  __syncthreads();
  return v;
}

template <typename T>
__global__ void __launch_bounds__(256) norm_parts_kernel(Matrices g, double* parts) {
  const int item = blockIdx.y;
  const T* src = (const T*)g.p + (long long)item * g.stride;
  double sum = 0;
  for (int j = blockIdx.x; j < g.cols; j += gridDim.x)
    for (int i = threadIdx.x; i < g.rows; i += blockDim.x) {
      const double v = (double)to_f32(src[(long long)j * g.ld + i]);
      sum += v * v;
    }
  sum = block_sum(sum);
  if (threadIdx.x == 0) parts[(long long)item * kNormParts + blockIdx.x] = sum;
}

template <typename T>
__global__ void __launch_bounds__(256) normalise_kernel(Matrices g, const double* parts, int n_parts, double eps, float* x) {
  const int item = blockIdx.y;
  double sum = 0;
  for (int i = 0; i < n_parts; ++i) sum += parts[(long long)item * kNormParts + i];
  const double inv = 1.0 / (sqrt(sum) + eps);
  const T* src = (const T*)g.p + (long long)item * g.stride;
  float* dst = x + (long long)item * g.rows * g.cols;
  for (int j = blockIdx.x; j < g.cols; j += gridDim.x)
    for (int i = threadIdx.x; i < g.rows; i += blockDim.x)
      dst[(long long)j * g.rows + i] = (float)((double)to_f32(src[(long long)j * g.ld + i]) * inv);
}

template <typename T>
__global__ void __launch_bounds__(256) store_kernel(const float* x, Matrices y) {
  const int item = blockIdx.y;
  T* dst = (T*)y.p + (long long)item * y.stride;
  const float* src = x + (long long)item * y.rows * y.cols;
  for (int j = blockIdx.x; j < y.cols; j += gridDim.x)
    for (int i = threadIdx.x; i < y.rows; i += blockDim.x)
      dst[(long long)j * y.ld + i] = from_f32<T>(src[(long long)j * y.rows + i]);
}

int validate_ns(const blb200_newton_schulz_desc* d) {
  if (!d) return BLB200_E_NULL;
  if (!valid_ftype(d->ftype)) return BLB200_E_DTYPE;
  if (d->rows < 0 || d->cols < 0 || d->batch < 0) return BLB200_E_SHAPE;
  if (!readable_layout(d->rows, d->ldx, d->stride_x) || !writable_layout(d->rows, d->cols, d->batch, d->ldy, d->stride_y))
    return BLB200_E_SHAPE;
  if (d->batch > 65535) return BLB200_E_TOO_LARGE;
  if (d->steps < 1 || d->steps > 64 || !(d->eps >= 0.0) || !isfinite(d->eps)) return BLB200_E_UNSUPPORTED;
  if (!d->coefficients) return BLB200_E_NULL;
  if (d->coefficient_sets != 1 && d->coefficient_sets != d->steps) return BLB200_E_UNSUPPORTED;
  // |X|_2 <= |X|_F <= 1 at the start; after a step at most the largest |a s + b s^3 + c s^5| over [0, bound]
  double bound = 1.0;
  for (int i = 0; i < d->steps; ++i) {
    const double* q = d->coefficients + 3 * (d->coefficient_sets == 1 ? 0 : i);
    if (!isfinite(q[0]) || !isfinite(q[1]) || !isfinite(q[2])) return BLB200_E_UNSUPPORTED;
    const double s2 = bound * bound;
    if (!(fabs(q[1]) * s2 + fabs(q[2]) * s2 * s2 <= kMaxEntry)) return BLB200_E_TOO_LARGE;
    auto value = [&](double s) { return fabs(s * (q[0] + s * s * (q[1] + s * s * q[2]))); };
    double top = value(bound);
    // critical points: a + 3 b t + 5 c t^2 = 0 with t = s^2
    const double A = 5 * q[2], B = 3 * q[1], C = q[0], disc = B * B - 4 * A * C;
    double roots[2] = {-1, -1};
    if (A == 0) {
      if (B != 0) roots[0] = -C / B;
    } else if (disc >= 0) {
      roots[0] = (-B + sqrt(disc)) / (2 * A);
      roots[1] = (-B - sqrt(disc)) / (2 * A);
    }
    for (double t : roots)
      if (t > 0 && t < s2) top = fmax(top, value(sqrt(t)));
    bound = top * 1.01;  // what the roundings of a step may add
    if (!(bound <= kMaxSigma)) return BLB200_E_TOO_LARGE;
  }
  if (d->rows > 0 && d->cols > 0 && d->batch > 0 && (!d->x || !d->y)) return BLB200_E_NULL;
  return BLB200_OK;
}

size_t round_up(size_t v) { return (v + 255) / 256 * 256; }
struct Layout {
  size_t parts, x, x2, s, b, total;
};
Layout layout_of(const blb200_newton_schulz_desc* d) {
  const size_t p = d->rows < d->cols ? d->rows : d->cols, n = d->batch;
  const size_t full = (size_t)d->rows * d->cols * n * 4, square = p * p * n * 4;
  Layout l;
  l.parts = 0;
  l.x = round_up(n * kNormParts * sizeof(double));
  l.x2 = l.x + round_up(full);
  l.s = l.x2 + round_up(full);
  l.b = l.s + round_up(square);
  l.total = l.b + round_up(square);
  return l;
}

}  // namespace
int newton_schulz_device_status(int* out) { return read_device_status_word(out); }
int newton_schulz_device_status_clear() { return clear_device_status_word(); }
}  // namespace blb200

extern "C" size_t blb200_newton_schulz_workspace_bytes(const blb200_newton_schulz_desc* d) {
  if (!d || d->rows <= 0 || d->cols <= 0 || d->batch <= 0) return 0;
  return blb200::layout_of(d).total;
}

extern "C" int blb200_newton_schulz(const blb200_newton_schulz_desc* d, void* workspace, size_t workspace_bytes, void* cuda_stream) {
  using namespace blb200;
  int rc = validate_ns(d);
  if (rc != BLB200_OK) return rc;
  if (d->rows == 0 || d->cols == 0 || d->batch == 0) return BLB200_OK;
  const Layout l = layout_of(d);
  if (!workspace) return BLB200_E_NULL;
  if (workspace_bytes < l.total || reinterpret_cast<uintptr_t>(workspace) % 256) return BLB200_E_SHAPE;
  cudaStream_t stream = (cudaStream_t)cuda_stream;
  char* ws = (char*)workspace;
  double* parts = (double*)(ws + l.parts);
  float *x = (float*)(ws + l.x), *x2 = (float*)(ws + l.x2), *s = (float*)(ws + l.s), *b = (float*)(ws + l.b);
  const Matrices g{const_cast<void*>(d->x), d->rows, d->cols, d->batch, d->ldx, d->stride_x};
  const Matrices y{d->y, d->rows, d->cols, d->batch, d->ldy, d->stride_y};
  const int n_parts = d->cols < kNormParts ? d->cols : kNormParts;
  const dim3 grid((unsigned)(d->cols < 1024 ? d->cols : 1024), (unsigned)d->batch);
  rc = with_ftype(d->ftype, [&](auto t) {
    using T = decltype(t);
    norm_parts_kernel<T><<<dim3(n_parts, d->batch), 256, 0, stream>>>(g, parts);
    normalise_kernel<T><<<grid, 256, 0, stream>>>(g, parts, n_parts, d->eps, x);
    return (int)cudaGetLastError();
  });
  if (rc != BLB200_OK) return rc;
  const int r = d->rows, c = d->cols, p = r < c ? r : c;
  auto product = [&](const float* A, const float* B, float* C, int m, int n, int k, long long lda, long long ldb, int opa, int opb,
                     double alpha, double beta) {
    blb200_gemm_desc e{};
    e.a = A; e.b = B; e.c = C;
    e.m = m; e.n = n; e.k = k; e.batch = d->batch;
    e.lda = lda; e.ldb = ldb; e.ldc = m;
    auto size = [](const float*, long long ld, int cols) { return ld * cols; };
    e.stride_a = size(A, lda, opa == BLB200_N ? k : m);
    e.stride_b = size(B, ldb, opb == BLB200_N ? n : k);
    e.stride_c = (long long)m * n;
    e.alpha[0] = alpha; e.beta[0] = beta;
    e.dtype = BLB200_S; e.op_a = opa; e.op_b = opb;
    return dispatch(&e, stream);
  };
  const size_t full = (size_t)r * c * d->batch * 4, square = (size_t)p * p * d->batch * 4;
  for (int i = 0; i < d->steps && rc == BLB200_OK; ++i) {
    const double* q = d->coefficients + 3 * (d->coefficient_sets == 1 ? 0 : i);
    rc = r <= c ? product(x, x, s, p, p, c, r, r, BLB200_N, BLB200_T, 1.0, 0.0)
                : product(x, x, s, p, p, r, r, r, BLB200_T, BLB200_N, 1.0, 0.0);
    if (rc == BLB200_OK) rc = (int)cudaMemcpyAsync(b, s, square, cudaMemcpyDeviceToDevice, stream);
    if (rc == BLB200_OK) rc = product(s, s, b, p, p, p, p, p, BLB200_N, BLB200_N, q[2], q[1]);
    if (rc == BLB200_OK) rc = (int)cudaMemcpyAsync(x2, x, full, cudaMemcpyDeviceToDevice, stream);
    if (rc == BLB200_OK)
      rc = r <= c ? product(b, x, x2, r, c, p, p, r, BLB200_N, BLB200_N, 1.0, q[0])
                  : product(x, b, x2, r, c, p, r, p, BLB200_N, BLB200_N, 1.0, q[0]);
    float* swap = x;
    x = x2;
    x2 = swap;
  }
  if (rc != BLB200_OK) return rc;
  return with_ftype(d->ftype, [&](auto t) {
    store_kernel<decltype(t)><<<grid, 256, 0, stream>>>(x, y);
    const int e = (int)cudaGetLastError();
    if (e == 0) note_launch("newton_schulz");
    return e;
  });
}
