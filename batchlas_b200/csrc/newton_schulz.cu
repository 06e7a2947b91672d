// Orthogonalisation of a batch of matrices by Newton-Schulz products:
//     X <- G / (||G||_F + eps);  steps times:  S = X X^T (shorter side),  B = b S + c S^2,  X <- a X + B X.
//
// The products run on the fp16 tensor cores with float accumulation.  X, S and B are stored in half precision, each
// times a power of two of its own that puts the largest value it can reach just below half's range: |X|_2 is known
// from the coefficients (it starts at ||G||/(||G|| + eps) <= 1 and each step maps it through the polynomial), and no
// entry exceeds the norm.  float inputs keep every matrix as a pair hi + lo of halves (22 bits and a sign) and
// multiply three times, and so do float16 inputs: one half per value would leave 1.2e-3 of the result, four times
// what float16's own rounding does.  bfloat16 inputs keep one half per value, whose half step of 2^-11 is an eighth of
// bfloat16's (2.0e-3 of the result in all, of which bfloat16's rounding is 1.7e-3).  What the scales come to is worked out on the device, per item and step, as the
// factors (alpha, beta) of the three products' epilogues  out = alpha * product + beta * old.
//
// Layout: X keeps the caller's orientation (rows fastest), so nothing is transposed.  With rows <= cols the Gram product
// contracts over the slow index (both operands MN-major) and the update over the fast one; with rows > cols the other
// way round.  S and B are symmetric: tiles on and below the diagonal are computed and stored twice.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "lowp.cuh"
#include "umma_gemm.cuh"

namespace blb200 {
namespace {

enum { kUmmaNsWait = 600 };
constexpr int kNormParts = 1024, kMaxSteps = 64;
constexpr double kMaxSigma = 64.0, kMaxEntry = 16384.0;
constexpr double kGrowth = 1.01;  // what the roundings of a step may add to the bound of X

struct Matrices {
  void* p;
  int rows, cols, batch;
  long long ld, stride;
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

// The passes over G: 256 threads as (256 / tx) columns of tx threads, each thread walking down its column in units of V
// elements (16 bytes where the layout allows it, else single elements).
template <typename T, int V>
struct Unit {
  __align__(16) T v[V];
  __device__ void load(const T* at) {
    if constexpr (V * sizeof(T) == 16) *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(at);
    else v[0] = *at;
  }
};

// Sum of squares in double (float's whole range, squared, fits), one part per block, in a fixed order.
template <typename T, int V>
__global__ void __launch_bounds__(256) norm_parts_kernel(Matrices g, double* parts, int tx) {
  griddep_wait();
  griddep_launch();
  const int item = blockIdx.y, ty = 256 / tx;
  const T* src = (const T*)g.p + (long long)item * g.stride;
  const int units = g.rows / V, x0 = threadIdx.x % tx;  // V divides the rows
  double sum = 0;
  for (int j = blockIdx.x * ty + threadIdx.x / tx; j < g.cols; j += gridDim.x * ty) {
    const T* col = src + (long long)j * g.ld;
#pragma unroll 4
    for (int i = x0; i < units; i += tx) {
      Unit<T, V> u;
      u.load(col + (long long)i * V);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const double v = (double)to_f32(u.v[e]);
        sum = fma(v, v, sum);
      }
    }
  }
  sum = block_sum(sum);
  if (threadIdx.x == 0) parts[(long long)item * kNormParts + blockIdx.x] = sum;
}

// Power of two that takes a value of at most `top` below 2^15.
__host__ __device__ inline double half_scale(double top) {
  if (!(top > 0) || isinf(top)) return 1.0;
  const int e = 14 - ilogb(top);
  return scalbn(1.0, e > 400 ? 400 : e);
}

// The powers of two that S, B and the next X are stored with at one step, from the bound of X before it.
struct StepScales {
  double s, b, next;
};
__host__ __device__ inline StepScales step_scales(const double* q, double& sigma, bool last) {
  const double s2 = sigma * sigma;
  StepScales r;
  r.s = half_scale(s2);
  r.b = half_scale(fabs(q[1]) * s2 + fabs(q[2]) * s2 * s2);
  sigma = polynomial_bound(q, sigma) * kGrowth;
  r.next = last ? 1.0 : half_scale(sigma);
  return r;
}

struct Plan {
  double q[3 * kMaxSteps];        // coefficients, by step
  StepScales scales[kMaxSteps];   // for a matrix that starts with |X| <= 1
  double eps;
  int steps;
};

template <int PLANES>
__device__ __forceinline__ void store_half(__half* at, long long plane, float v) {
  const __half hi = __float2half_rn(v);
  at[0] = hi;
  if constexpr (PLANES == 2) at[plane] = __float2half_rn(v - __half2float(hi));
}

// G times its item's power of two t, as half planes (two factors, so that neither leaves float's range), and, by the
// first block of each item, the factors of every product's epilogue.
template <typename T, int V, int PLANES>
__global__ void __launch_bounds__(256) ingest_kernel(Matrices g, const double* parts, int n_parts, __half* x, long long ld, long long plane, int tx,
                                                     const __grid_constant__ Plan plan, float2* factors) {
  griddep_wait();
  griddep_launch();
  const int item = blockIdx.y, ty = 256 / tx, batch = gridDim.y;
  double sum = 0;
  for (int i = threadIdx.x; i < n_parts; i += 256) sum += parts[(long long)item * kNormParts + i];
  sum = block_sum(sum);
  const double norm = sqrt(sum), f = norm + plan.eps;
  const bool usable = isfinite(sum) && f > 0;
  const int e = sum > 0 && usable ? 14 - ilogb(norm) : 0;
  const float t1 = usable ? scalbnf(1.f, e / 2) : __int_as_float(0x7fffffff), t2 = scalbnf(1.f, e - e / 2);

  if (blockIdx.x == 0) {
    __shared__ StepScales own[kMaxSteps];
    // X = stored / (t f).  The bounds for |X| <= 1 hold for every item; one that eps makes much smaller gets its own, so
    // that its matrices do not sink towards half's smallest numbers.
    const bool small = norm < 0.125 * f;
    if (small) {
      if (threadIdx.x == 0) {
        double sigma = norm / f;
        for (int i = 0; i < plan.steps; ++i) own[i] = step_scales(plan.q + 3 * i, sigma, i + 1 == plan.steps);
      }
      __syncthreads();
    }
    const int i = threadIdx.x;
    if (i < plan.steps) {
      const StepScales* sc = small ? own : plan.scales;
      const double ss = sc[i].s, sb = sc[i].b, sn = sc[i].next;
      // a zero item stays zero under any finite factors
      const double sx = i > 0 ? sc[i - 1].next : (norm > 0 ? scalbn(1.0, e) * f : 1.0);
      const double* q = plan.q + 3 * i;
      float2* out = factors + (long long)i * 3 * batch + item;
      out[0] = make_float2((float)(ss / sx / sx), 0.f);
      out[batch] = make_float2((float)(q[2] * (sb / ss / ss)), (float)(q[1] * (sb / ss)));
      out[2 * batch] = make_float2((float)(sn / sb / sx), (float)(q[0] * (sn / sx)));
    }
  }

  const T* src = (const T*)g.p + (long long)item * g.stride;
  __half* dst = x + (long long)item * PLANES * plane;
  const int units = g.rows / V, x0 = threadIdx.x % tx;
  for (int j = blockIdx.x * ty + threadIdx.x / tx; j < g.cols; j += gridDim.x * ty) {
    const T* col = src + (long long)j * g.ld;
    __half* to = dst + (long long)j * ld;
#pragma unroll 4
    for (int i = x0; i < units; i += tx) {
      Unit<T, V> u;
      u.load(col + (long long)i * V);
      if constexpr (V == 1) {
        store_half<PLANES>(to + i, plane, to_f32(u.v[0]) * t1 * t2);
      } else {
        __align__(16) __half hi[V], lo[V];
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const float v = to_f32(u.v[k]) * t1 * t2;
          hi[k] = __float2half_rn(v);
          lo[k] = __float2half_rn(v - __half2float(hi[k]));
        }
        using Word = typename std::conditional<V == 8, uint4, uint2>::type;
        *reinterpret_cast<Word*>(to + (long long)i * V) = *reinterpret_cast<const Word*>(hi);
        if constexpr (PLANES == 2) *reinterpret_cast<Word*>(to + plane + (long long)i * V) = *reinterpret_cast<const Word*>(lo);
      }
    }
  }
}

__device__ __forceinline__ uint32_t pack_halves(__half a, __half b) {
  return (uint32_t)__half_as_ushort(a) | (uint32_t)__half_as_ushort(b) << 16;
}
__device__ __forceinline__ __half half_of(uint32_t pair, int which) { return __ushort_as_half((unsigned short)(pair >> (16 * which))); }

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
  __device__ NsEpilogue(const Params& p_, const UmmaShape& s_, const UmmaTile& tile, bool twice, int m) : p(p_), s(s_), live(m < s_.m) {
    const float2 f = p.factors[tile.item];
    alpha = f.x;
    beta = f.y;
    old = p.old ? p.old + (long long)tile.item * PLANES * p.old_plane + m : nullptr;
    T* base = (T*)p.out + (long long)tile.item * p.out_item;
    out = base + m;
    mirror = twice ? base + (long long)m * p.out_ld : nullptr;
  }
  // kGroup columns at a time: their old values are requested together (for pairs eight, or the sums spill).
  static constexpr int kGroup = PLANES == 2 ? 8 : 16;
  template <int N>
  __device__ void store(const uint32_t (&v)[N], int n) {
    if (!live) return;
#pragma unroll
    for (int g = 0; g < N; g += kGroup) {
      if (n + g + kGroup <= s.n) store_group<N, true>(v, g, n + g);
      else if (n + g < s.n) store_group<N, false>(v, g, n + g);
    }
  }
  template <int N, bool FULL>
  __device__ __forceinline__ void store_group(const uint32_t (&v)[N], int g, int n) {
    float r[kGroup];
    if (old) {
      const __half* at = old + (long long)n * p.old_ld;
      __half hi[kGroup], lo[kGroup];
#pragma unroll
      for (int i = 0; i < kGroup; ++i) {
        if (FULL || n + i < s.n) {
          hi[i] = at[0];
          if constexpr (PLANES == 2) lo[i] = at[p.old_plane];
        }
        at += p.old_ld;
      }
#pragma unroll
      for (int i = 0; i < kGroup; ++i) {
        float was = __half2float(hi[i]);
        if constexpr (PLANES == 2) was += __half2float(lo[i]);
        r[i] = fmaf(beta, was, alpha * __uint_as_float(v[g + i]));
      }
    } else {
#pragma unroll
      for (int i = 0; i < kGroup; ++i) r[i] = alpha * __uint_as_float(v[g + i]);
    }
    T* at = out + (long long)n * p.out_ld;
    if constexpr (LAST) {
#pragma unroll
      for (int i = 0; i < kGroup; ++i) {
        if (FULL || n + i < s.n) *at = from_f32<T>(r[i]);
        at += p.out_ld;
      }
    } else {
      uint32_t hi[kGroup / 2], lo[kGroup / 2];  // pairs of halves
#pragma unroll
      for (int i = 0; i < kGroup / 2; ++i) {
        const __half h0 = __float2half_rn(r[2 * i]), h1 = __float2half_rn(r[2 * i + 1]);
        hi[i] = pack_halves(h0, h1);
        if constexpr (PLANES == 2)
          lo[i] = pack_halves(__float2half_rn(r[2 * i] - __half2float(h0)), __float2half_rn(r[2 * i + 1] - __half2float(h1)));
      }
#pragma unroll
      for (int i = 0; i < kGroup; ++i) {
        if (FULL || n + i < s.n) {
          at[0] = half_of(hi[i / 2], i & 1);
          if constexpr (PLANES == 2) at[p.out_plane] = half_of(lo[i / 2], i & 1);
        }
        at += p.out_ld;
      }
      if (mirror) {
        if (FULL) {
#pragma unroll
          for (int h = 0; h < kGroup / 2; h += 4) {
            *reinterpret_cast<uint4*>(mirror + n + 2 * h) = make_uint4(hi[h], hi[h + 1], hi[h + 2], hi[h + 3]);
            if constexpr (PLANES == 2)
              *reinterpret_cast<uint4*>(mirror + p.out_plane + n + 2 * h) = make_uint4(lo[h], lo[h + 1], lo[h + 2], lo[h + 3]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < kGroup; ++i)
            if (n + i < s.n) {
              mirror[n + i] = half_of(hi[i / 2], i & 1);
              if constexpr (PLANES == 2) mirror[p.out_plane + n + i] = half_of(lo[i / 2], i & 1);
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

// The tensor maps of one call: every matrix is an operand several times.
struct Maps {
  struct Entry {
    const void* p;
    int box;
    CUtensorMap map;
  };
  Entry e[16];
  int used = 0;
  int get(const CUtensorMap** out, const HalfMatrix& a, int z, int box) {
    for (int i = 0; i < used; ++i)
      if (e[i].p == a.p && e[i].box == box) {
        *out = &e[i].map;
        return BLB200_OK;
      }
    if (used == 16) return BLB200_E_INTERNAL;  // four matrices in three boxes each at most
    const int rc = encode_operand(&e[used].map, a.p, false, a.inner, a.outer, z, a.ld * 2, a.plane * 2, box);
    if (rc != BLB200_OK) return rc;
    e[used].p = a.p;
    e[used].box = box;
    *out = &e[used++].map;
    return BLB200_OK;
  }
};

template <bool A_MN, bool B_MN, int GROUP, int BN, int PLANES, class Epilogue>
int launch_product(Maps& maps, const HalfMatrix& a, const HalfMatrix& b, int m, int n, int k, int batch, bool symmetric,
                   const typename Epilogue::Params& ep, cudaStream_t stream) {
  using C = UmmaConfig<false, A_MN, B_MN, GROUP, BN, PLANES>;
  UmmaShape s{};
  s.m = m;
  s.n = n;
  s.k = k;
  s.batch = batch;
  s.symmetric = symmetric;  // a_items, b_items stay 0: no operand is shared by the items
  const CUtensorMap *map_a, *map_b;
  int rc = maps.get(&map_a, a, batch * PLANES, A_MN ? 64 : 128);
  if (rc == BLB200_OK) rc = maps.get(&map_b, b, batch * PLANES, B_MN ? 64 : C::kBRows);
  if (rc == BLB200_OK) rc = launch_umma<C, Epilogue>(*map_a, *map_b, s, ep, kUmmaNsWait, stream);
  if (rc == BLB200_OK) note_launch("newton_schulz");
  return rc;
}

// Tiles of 256 rows on CTA pairs (256 columns wide, for float 128) or of 128 x 128 on single CTAs: whichever needs less
// time for the number of rounds its tiles come to.
template <bool A_MN, bool B_MN, int PLANES, class Epilogue>
int product(Maps& maps, const HalfMatrix& a, const HalfMatrix& b, int m, int n, int k, int batch, bool symmetric,
            const typename Epilogue::Params& ep, cudaStream_t stream) {
  constexpr int kPairN = PLANES == 2 ? 128 : 256;
  auto tiles = [&](int t_m, int t_n) {
    const int tm = (m + t_m - 1) / t_m, tn = (n + t_n - 1) / t_n;
    const long long each = !symmetric ? (long long)tm * tn : t_m == t_n ? symmetric_tiles<1>(tm, tn) : symmetric_tiles<2>(tm, tn);
    return each * batch;
  };
  const long long sms = device_info().sm_count;
  const double pair = kPairN / 128 * (double)((tiles(256, kPairN) + sms / 2 - 1) / (sms / 2));
  const double single = 1.15 * (double)((tiles(128, 128) + sms - 1) / sms);
  return pair <= single ? launch_product<A_MN, B_MN, 2, kPairN, PLANES, Epilogue>(maps, a, b, m, n, k, batch, symmetric, ep, stream)
                        : launch_product<A_MN, B_MN, 1, 128, PLANES, Epilogue>(maps, a, b, m, n, k, batch, symmetric, ep, stream);
}

int validate_ns(const blb200_newton_schulz_desc* d) {
  if (!d) return BLB200_E_NULL;
  if (!valid_ftype(d->ftype)) return BLB200_E_DTYPE;
  if (d->rows < 0 || d->cols < 0 || d->batch < 0) return BLB200_E_SHAPE;
  if (!readable_layout(d->rows, d->ldx, d->stride_x) || !writable_layout(d->rows, d->cols, d->batch, d->ldy, d->stride_y))
    return BLB200_E_SHAPE;
  if (d->batch > 65535) return BLB200_E_TOO_LARGE;
  if (d->steps < 1 || d->steps > kMaxSteps || !(d->eps >= 0.0) || !isfinite(d->eps)) return BLB200_E_UNSUPPORTED;
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
  size_t parts, factors, x, x2, s, b, total;
};
Layout layout_of(const blb200_newton_schulz_desc* d) {
  Layout l;
  const size_t n = d->batch;
  l.planes = d->ftype == BLB200_BF16 ? 1 : 2;
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
  l.factors = take(n * 3 * d->steps * sizeof(float2));
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
  float2* factors = (float2*)(ws + l.factors);
  HalfMatrix x{(__half*)(ws + l.x), r, c, l.ld_x, l.plane_x}, x2{(__half*)(ws + l.x2), r, c, l.ld_x, l.plane_x};
  const HalfMatrix s{(__half*)(ws + l.s), p, p, l.ld_s, l.plane_s}, b{(__half*)(ws + l.b), p, p, l.ld_s, l.plane_s};
  Plan plan;
  plan.eps = d->eps;
  plan.steps = d->steps;
  double sigma = 1.0;
  for (int i = 0; i < d->steps; ++i) {
    for (int j = 0; j < 3; ++j) plan.q[3 * i + j] = d->coefficients[(d->coefficient_sets == 1 ? 0 : 3 * i) + j];
    plan.scales[i] = step_scales(plan.q + 3 * i, sigma, i + 1 == d->steps);
  }
  constexpr int V = 16 / sizeof(T);
  const bool wide = r % V == 0 && reinterpret_cast<uintptr_t>(d->x) % 16 == 0 && d->ldx % V == 0 && (d->stride_x % V == 0 || batch == 1);
  int tx = 8;
  while (tx < 256 && tx < (wide ? r / V : r)) tx *= 2;
  const int rows_of_blocks = (c + 256 / tx - 1) / (256 / tx), sms = device_info().sm_count;
  const int most = sms * 8 / batch + 1;  // eight blocks per SM fill it
  const int n_parts = std::min(std::min(rows_of_blocks, most), kNormParts);
  auto passes = [&](auto norm, auto ingest) {
    const OverlappedLaunch first(dim3(n_parts, batch), 256, stream);
    const int e = (int)cudaLaunchKernelEx(&first.cfg, norm, g, parts, tx);
    if (e) return e;
    const OverlappedLaunch launch(dim3(std::min(rows_of_blocks, most), batch), 256, stream);
    return (int)cudaLaunchKernelEx(&launch.cfg, ingest, g, (const double*)parts, n_parts, x.p, l.ld_x, l.plane_x, tx, plan, factors);
  };
  int rc = wide ? passes(norm_parts_kernel<T, V>, ingest_kernel<T, V, PLANES>) : passes(norm_parts_kernel<T, 1>, ingest_kernel<T, 1, PLANES>);
  Maps maps;
  using Inner = NsEpilogue<__half, PLANES, false>;
  using Last = NsEpilogue<T, PLANES, true>;
  for (int i = 0; i < d->steps && rc == BLB200_OK; ++i) {
    const float2* f = factors + (long long)i * 3 * batch;
    const typename Inner::Params gram{f, nullptr, s.p, 0, 0, l.ld_s, l.plane_s, PLANES * l.plane_s};
    rc = r <= c ? product<true, true, PLANES, Inner>(maps, x, x, p, p, c, batch, true, gram, stream)
                : product<false, false, PLANES, Inner>(maps, x, x, p, p, r, batch, true, gram, stream);
    if (rc != BLB200_OK) break;
    const typename Inner::Params square{f + batch, s.p, b.p, l.ld_s, l.plane_s, l.ld_s, l.plane_s, PLANES * l.plane_s};
    rc = product<false, false, PLANES, Inner>(maps, s, s, p, p, p, batch, true, square, stream);
    if (rc != BLB200_OK) break;
    if (i + 1 < d->steps) {
      const typename Inner::Params update{f + 2 * batch, x.p, x2.p, l.ld_x, l.plane_x, l.ld_x, l.plane_x, PLANES * l.plane_x};
      rc = r <= c ? product<false, false, PLANES, Inner>(maps, b, x, r, c, p, batch, false, update, stream)
                  : product<true, false, PLANES, Inner>(maps, x, b, r, c, p, batch, false, update, stream);
      const HalfMatrix swap = x;
      x = x2;
      x2 = swap;
    } else {
      const typename Last::Params last{f + 2 * batch, x.p, d->y, l.ld_x, l.plane_x, d->ldy, 0, d->stride_y};
      rc = r <= c ? product<false, false, PLANES, Last>(maps, b, x, r, c, p, batch, false, last, stream)
                  : product<true, false, PLANES, Last>(maps, x, b, r, c, p, batch, false, last, stream);
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
  if (d->ftype == BLB200_F16) return run<__half, 2>(d, l, (char*)workspace, stream);
  return run<__nv_bfloat16, 1>(d, l, (char*)workspace, stream);
}
