// Orthogonalisation of a batch of matrices by Newton-Schulz products:
//     X <- G / (||G||_F + eps);  steps times:  S = X X^T (shorter side),  B = b S + c S^2,  X <- a X + B X.
//
// The products run on the fp16 tensor cores with float accumulation.  X, S and B are stored in half precision, each
// times a power of two of its own that puts the largest value it can reach just below half's range: |X|_2 is known
// from the coefficients (it starts at ||G||/(||G|| + eps) <= 1 and each step maps it through the polynomial), and no
// entry exceeds the norm.  float inputs keep every matrix as a pair hi + lo of halves (22 bits and a sign) and
// multiply three times; half inputs keep one, which is 2^-12 per value at most half a step of 2^-11, eight times
// finer than bfloat16 would be.  What the scales come to is worked out on the device, per item and step, as the
// factors (alpha, beta) of the three products' epilogues  out = alpha * product + beta * old.
//
// Layout: X keeps the caller's orientation (rows fastest), so nothing is transposed.  With rows <= cols the Gram product
// contracts over the slow index (both operands MN-major) and the update over the fast one; with rows > cols the other
// way round.  S and B are symmetric: tiles on and below the diagonal are computed and stored twice.
#include <math.h>

#include "lowp.cuh"
#include "umma_gemm.cuh"

namespace blb200 {
namespace {

enum { kUmmaNsWait = 600 };
constexpr int kNormParts = 256;
constexpr double kMaxSigma = 64.0, kMaxEntry = 16384.0;
constexpr double kGrowth = 1.01;  // what the roundings of a step may add to the bound of X

struct Matrices {
  void* p;
  int rows, cols, batch;
  long long ld, stride;
};

struct Coefficients {
  double v[3 * 64];
};

// Largest |a s + b s^3 + c s^5| over 0 <= s <= top.
__host__ __device__ inline double polynomial_bound(const double* q, double top) {
  auto value = [&](double s) { return fabs(s * (q[0] + s * s * (q[1] + s * s * q[2]))); };
  double best = value(top);
  // critical points: a + 3 b t + 5 c t^2 = 0 with t = s^2
  const double A = 5 * q[2], B = 3 * q[1], C = q[0], disc = B * B - 4 * A * C;
  if (A == 0) {
    if (B != 0 && -C / B > 0 && -C / B < top * top) best = fmax(best, value(sqrt(-C / B)));
  } else if (disc >= 0) {
    const double r = sqrt(disc);
    for (int i = 0; i < 2; ++i) {
      const double t = (-B + (i ? -r : r)) / (2 * A);
      if (t > 0 && t < top * top) best = fmax(best, value(sqrt(t)));
    }
  }
  return best;
}

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

// Sum of squares in double (float's whole range, squared, fits), one part per block, in a fixed order.
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

// Power of two that takes a value of at most `top` below 2^15.
__device__ __forceinline__ double half_scale(double top) {
  if (!(top > 0)) return 1.0;
  const int e = 14 - ilogb(top);
  return scalbn(1.0, e > 400 ? 400 : e);
}
__device__ __forceinline__ float factor(double v) { return (float)v; }

// One block per item: the norm, the scale that G is stored with, and the factors of every product's epilogue.
__global__ void __launch_bounds__(256) plan_kernel(const double* parts, int n_parts, double eps, const __grid_constant__ Coefficients q, int steps,
                                                   int sets, double* scale0, float2* factors, int batch) {
  const int item = blockIdx.x;
  const double sum = block_sum(threadIdx.x < n_parts ? parts[(long long)item * kNormParts + threadIdx.x] : 0.0);
  if (threadIdx.x != 0) return;
  const double norm = sqrt(sum), f = norm + eps;
  // G * t is what is stored first; X = stored / (t f)
  const double t = half_scale(norm);
  double sigma = norm / f, sx = norm > 0 ? t * f : 1.0;  // a zero item stays zero under any finite factors
  scale0[item] = isfinite(sum) && f > 0 ? t : nan("");
  for (int i = 0; i < steps; ++i) {
    const double* v = q.v + 3 * (sets == 1 ? 0 : i);
    const double s2 = sigma * sigma;
    const double ss = half_scale(s2), sb = half_scale(fabs(v[1]) * s2 + fabs(v[2]) * s2 * s2);
    const double next = polynomial_bound(v, sigma) * kGrowth, sn = i + 1 < steps ? half_scale(next) : 1.0;
    float2* out = factors + (long long)i * 3 * batch + item;
    out[0] = make_float2(factor(ss / sx / sx), 0.f);
    out[batch] = make_float2(factor(v[2] * (sb / ss / ss)), factor(v[1] * (sb / ss)));
    out[2 * batch] = make_float2(factor(sn / sb / sx), factor(v[0] * (sn / sx)));
    sigma = next;
    sx = sn;
  }
}

template <int PLANES>
__device__ __forceinline__ void store_half(__half* at, long long plane, float v) {
  const __half hi = __float2half_rn(v);
  at[0] = hi;
  if constexpr (PLANES == 2) at[plane] = __float2half_rn(v - __half2float(hi));
}

// G times its item's power of two, as half planes.
template <typename T, int PLANES>
__global__ void __launch_bounds__(256) ingest_kernel(Matrices g, const double* scale0, __half* x, long long ld, long long plane) {
  const int item = blockIdx.y;
  const double scale = scale0[item];
  const T* src = (const T*)g.p + (long long)item * g.stride;
  __half* dst = x + (long long)item * PLANES * plane;
  for (int j = blockIdx.x; j < g.cols; j += gridDim.x)
    for (int i = threadIdx.x; i < g.rows; i += blockDim.x)
      store_half<PLANES>(dst + (long long)j * ld + i, plane, (float)((double)to_f32(src[(long long)j * g.ld + i]) * scale));
}

// out = alpha * product + beta * old, written as half planes (mirrored across the diagonal when the result is
// symmetric) or, by the last step, in the caller's type and layout.
template <typename T, int PLANES, bool LAST>
struct NsEpilogue {
  struct Params {
    const float2* factors;
    const __half* old;  // null: beta is not used
    void* out;
    long long old_ld, old_plane, out_ld, out_plane, out_item;
  };
  const Params& p;
  const UmmaShape& s;
  const __half* old;
  T* out;
  T* mirror;
  float alpha, beta;
  bool live;
  __device__ NsEpilogue(const Params& p_, const UmmaShape& s_, const UmmaTile& tile, int m) : p(p_), s(s_), live(m < s_.m) {
    const float2 f = p.factors[tile.item];
    alpha = f.x;
    beta = f.y;
    old = p.old ? p.old + (long long)tile.item * PLANES * p.old_plane + m : nullptr;
    T* base = (T*)p.out + (long long)tile.item * p.out_item;
    out = base + m;
    mirror = s.symmetric && tile.tm != tile.tn ? base + (long long)m * p.out_ld : nullptr;
  }
  template <int N>
  __device__ void store(const uint32_t (&v)[N], int n) {
    if (!live) return;
    float r[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      r[i] = alpha * __uint_as_float(v[i]);
      if (old && n + i < s.n) {
        const __half* at = old + (long long)(n + i) * p.old_ld;
        float was = __half2float(at[0]);
        if constexpr (PLANES == 2) was += __half2float(at[p.old_plane]);
        r[i] = fmaf(beta, was, r[i]);
      }
    }
    if constexpr (LAST) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (n + i < s.n) out[(long long)(n + i) * p.out_ld] = from_f32<T>(r[i]);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (n + i < s.n) store_half<PLANES>(out + (long long)(n + i) * p.out_ld, p.out_plane, r[i]);
      if (mirror) {
#pragma unroll
        for (int g = 0; g < N; g += 8) {
          if (n + g + 8 <= s.n) {
            __half h[8], l[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              h[i] = __float2half_rn(r[g + i]);
              l[i] = __float2half_rn(r[g + i] - __half2float(h[i]));
            }
            *reinterpret_cast<uint4*>(mirror + n + g) = *reinterpret_cast<const uint4*>(h);
            if constexpr (PLANES == 2) *reinterpret_cast<uint4*>(mirror + p.out_plane + n + g) = *reinterpret_cast<const uint4*>(l);
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (n + g + i < s.n) store_half<PLANES>(mirror + n + g + i, p.out_plane, r[g + i]);
          }
        }
      }
    }
  }
};

struct HalfMatrix {  // [item][plane][outer][ld], inner fastest
  __half* p;
  int inner, outer;
  long long ld, plane;
};

template <bool A_MN, bool B_MN, int GROUP, int BN, int PLANES, class Epilogue>
int launch_product(const HalfMatrix& a, const HalfMatrix& b, int m, int n, int k, int batch, bool symmetric, const typename Epilogue::Params& ep,
                   cudaStream_t stream) {
  using C = UmmaConfig<false, A_MN, B_MN, GROUP, BN, PLANES>;
  UmmaShape s{};
  s.m = m;
  s.n = n;
  s.k = k;
  s.batch = batch;
  s.a_items = s.b_items = batch > 1 ? batch : 0;  // 0: never shared
  s.symmetric = symmetric;
  CUtensorMap map_a, map_b;
  int rc = encode_operand(&map_a, a.p, false, a.inner, a.outer, (long long)batch * PLANES, a.ld * 2, a.plane * 2, A_MN ? 64 : 128);
  if (rc == BLB200_OK)
    rc = encode_operand(&map_b, b.p, false, b.inner, b.outer, (long long)batch * PLANES, b.ld * 2, b.plane * 2, B_MN ? 64 : C::kBRows);
  if (rc == BLB200_OK) rc = launch_umma<C, Epilogue>(map_a, map_b, s, ep, kUmmaNsWait, stream);
  if (rc == BLB200_OK) note_launch("newton_schulz");
  return rc;
}

// 256 x 256 tiles on CTA pairs or 128 x 128 tiles on single CTAs: whichever needs less time for the number of rounds its
// tiles come to, a single CTA's tile taken as 1.15 quarters of a pair's.
template <bool A_MN, bool B_MN, int PLANES, class Epilogue>
int product(const HalfMatrix& a, const HalfMatrix& b, int m, int n, int k, int batch, bool symmetric, const typename Epilogue::Params& ep,
            cudaStream_t stream) {
  auto tiles = [&](int t) {
    const long long tm = (m + t - 1) / t, tn = (n + t - 1) / t;
    return (symmetric ? tm * (tm + 1) / 2 : tm * tn) * batch;
  };
  const long long sms = device_info().sm_count;
  const double pair = 2.0 * (double)((tiles(256) + sms / 2 - 1) / (sms / 2));
  const double single = 1.15 * (double)((tiles(128) + sms - 1) / sms);
  return pair <= single ? launch_product<A_MN, B_MN, 2, 256, PLANES, Epilogue>(a, b, m, n, k, batch, symmetric, ep, stream)
                        : launch_product<A_MN, B_MN, 1, 128, PLANES, Epilogue>(a, b, m, n, k, batch, symmetric, ep, stream);
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
  double bound = 1.0;  // |X|_2 <= ||X||_F <= 1 at the start
  for (int i = 0; i < d->steps; ++i) {
    const double* q = d->coefficients + 3 * (d->coefficient_sets == 1 ? 0 : i);
    if (!isfinite(q[0]) || !isfinite(q[1]) || !isfinite(q[2])) return BLB200_E_UNSUPPORTED;
    const double s2 = bound * bound;
    if (!(fabs(q[1]) * s2 + fabs(q[2]) * s2 * s2 <= kMaxEntry)) return BLB200_E_TOO_LARGE;
    bound = polynomial_bound(q, bound) * kGrowth;
    if (!(bound <= kMaxSigma)) return BLB200_E_TOO_LARGE;
  }
  if (d->rows > 0 && d->cols > 0 && d->batch > 0 && (!d->x || !d->y)) return BLB200_E_NULL;
  return BLB200_OK;
}

struct Layout {
  int planes, p;
  long long ld_x, plane_x, ld_s, plane_s;  // elements
  size_t parts, scale0, factors, x, x2, s, b, total;
};
Layout layout_of(const blb200_newton_schulz_desc* d) {
  Layout l;
  const size_t n = d->batch;
  l.planes = d->ftype == BLB200_F32 ? 2 : 1;
  l.p = d->rows < d->cols ? d->rows : d->cols;
  l.ld_x = ((long long)d->rows + 7) / 8 * 8;
  l.plane_x = l.ld_x * d->cols;
  l.ld_s = ((long long)l.p + 7) / 8 * 8;
  l.plane_s = l.ld_s * l.p;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  l.parts = take(n * kNormParts * sizeof(double));
  l.scale0 = take(n * sizeof(double));
  l.factors = take(n * 3 * 64 * sizeof(float2));
  l.x = take(n * l.planes * l.plane_x * 2);
  l.x2 = take(n * l.planes * l.plane_x * 2);
  l.s = take(n * l.planes * l.plane_s * 2);
  l.b = take(n * l.planes * l.plane_s * 2);
  l.total = at;
  return l;
}

template <typename T, int PLANES>
int run(const blb200_newton_schulz_desc* d, const Layout& l, char* ws, cudaStream_t stream) {
  const int r = d->rows, c = d->cols, p = l.p, batch = d->batch;
  const Matrices g{const_cast<void*>(d->x), r, c, batch, d->ldx, d->stride_x};
  double* parts = (double*)(ws + l.parts);
  double* scale0 = (double*)(ws + l.scale0);
  float2* factors = (float2*)(ws + l.factors);
  HalfMatrix x{(__half*)(ws + l.x), r, c, l.ld_x, l.plane_x}, x2{(__half*)(ws + l.x2), r, c, l.ld_x, l.plane_x};
  const HalfMatrix s{(__half*)(ws + l.s), p, p, l.ld_s, l.plane_s}, b{(__half*)(ws + l.b), p, p, l.ld_s, l.plane_s};
  Coefficients q;
  for (int i = 0; i < 3 * d->coefficient_sets; ++i) q.v[i] = d->coefficients[i];
  const int n_parts = c < kNormParts ? c : kNormParts;
  norm_parts_kernel<T><<<dim3(n_parts, batch), 256, 0, stream>>>(g, parts);
  plan_kernel<<<batch, 256, 0, stream>>>(parts, n_parts, d->eps, q, d->steps, d->coefficient_sets, scale0, factors, batch);
  ingest_kernel<T, PLANES><<<dim3(c < 1024 ? c : 1024, batch), 256, 0, stream>>>(g, scale0, x.p, l.ld_x, l.plane_x);
  int rc = (int)cudaGetLastError();
  using Inner = NsEpilogue<__half, PLANES, false>;
  using Last = NsEpilogue<T, PLANES, true>;
  for (int i = 0; i < d->steps && rc == BLB200_OK; ++i) {
    const float2* f = factors + (long long)i * 3 * batch;
    const typename Inner::Params gram{f, nullptr, s.p, 0, 0, l.ld_s, l.plane_s, PLANES * l.plane_s};
    rc = r <= c ? product<true, true, PLANES, Inner>(x, x, p, p, c, batch, true, gram, stream)
                : product<false, false, PLANES, Inner>(x, x, p, p, r, batch, true, gram, stream);
    if (rc != BLB200_OK) break;
    const typename Inner::Params square{f + batch, s.p, b.p, l.ld_s, l.plane_s, l.ld_s, l.plane_s, PLANES * l.plane_s};
    rc = product<false, false, PLANES, Inner>(s, s, p, p, p, batch, true, square, stream);
    if (rc != BLB200_OK) break;
    if (i + 1 < d->steps) {
      const typename Inner::Params update{f + 2 * batch, x.p, x2.p, l.ld_x, l.plane_x, l.ld_x, l.plane_x, PLANES * l.plane_x};
      rc = r <= c ? product<false, false, PLANES, Inner>(b, x, r, c, p, batch, false, update, stream)
                  : product<true, false, PLANES, Inner>(x, b, r, c, p, batch, false, update, stream);
      const HalfMatrix swap = x;
      x = x2;
      x2 = swap;
    } else {
      const typename Last::Params last{f + 2 * batch, x.p, d->y, l.ld_x, l.plane_x, d->ldy, 0, d->stride_y};
      rc = r <= c ? product<false, false, PLANES, Last>(b, x, r, c, p, batch, false, last, stream)
                  : product<true, false, PLANES, Last>(x, b, r, c, p, batch, false, last, stream);
    }
  }
  return rc;
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
  const int rc = validate_ns(d);
  if (rc != BLB200_OK) return rc;
  if (d->rows == 0 || d->cols == 0 || d->batch == 0) return BLB200_OK;
  const Layout l = layout_of(d);
  if (!workspace) return BLB200_E_NULL;
  if (workspace_bytes < l.total || reinterpret_cast<uintptr_t>(workspace) % 256) return BLB200_E_SHAPE;
  cudaStream_t stream = (cudaStream_t)cuda_stream;
  if (d->ftype == BLB200_F32) return run<float, 2>(d, l, (char*)workspace, stream);
  if (d->ftype == BLB200_F16) return run<__half, 1>(d, l, (char*)workspace, stream);
  return run<__nv_bfloat16, 1>(d, l, (char*)workspace, stream);
}
