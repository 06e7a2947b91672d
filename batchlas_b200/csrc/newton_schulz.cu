// Orthogonalisation of a batch of matrices by Newton-Schulz products:
//     X <- G / (||G||_F + eps);  steps times:  S = X X^T (shorter side),  B = b S + c S^2,  X <- a X + B X.
//
// The products run on the fp16 tensor cores with float accumulation.  X, S and B are stored in half precision, each
// times a power of two of its own that puts the largest value it can reach just below half's range: |X|_2 is known
// from the coefficients (it starts at ||G||/(||G|| + eps) <= 1 and each step maps it through the polynomial), and no
// entry exceeds the norm.  Every matrix is kept as a pair hi + lo of halves (22 bits and a sign) and multiplied three times: one
// half per value leaves 1.0 to 1.4e-3 of the result, five times what float16's own rounding does, and with bfloat16's, which is
// 1.65e-3, 1.9 to 2.2e-3 in all.  Only a caller who asks for it gets that (bfloat16, half_intermediates: 4096 x 16384 4.1 ms, as
// pairs 14.0).  No cheaper way lies between: with any one of the products' operands in single halves 0.3 to 1.0e-3 are
// left.  What the scales come to is worked out on the device, per item and step, as the factors (alpha, beta) of the three
// products' epilogues  out = alpha * product + beta * old.
//
// Layout: X keeps the caller's orientation (rows fastest), so nothing is transposed.  With rows <= cols the Gram product
// contracts over the slow index (both operands MN-major) and the update over the fast one; with rows > cols the other
// way round.  S and B are symmetric: tiles on and below the diagonal are computed and stored twice.
#include <algorithm>
#include <type_traits>
#include <utility>

#include "newton_schulz.cuh"
#include "umma_gemm.cuh"

namespace blb200 {
namespace {

enum { kUmmaNsWait = 600 };
constexpr int kNormParts = 1024;
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
  const ItemScale scale(sum, plan.eps);
  const float t1 = scale.t1, t2 = scale.t2;

  if (blockIdx.x == 0) {
    __shared__ StepScales own[kMaxSteps];
    write_factors(plan, scale.norm, scale.f, scale.e, own, factors + item, batch);
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

// The epilogue's parameters: out = alpha * product + beta * old.
struct NsParams {
  const float2* factors;
  int has_old;  // 0: beta is not used
  void* out;
  long long out_ld, out_plane, out_item;
};

// Into half planes, row by row through the staging buffer: a thread's columns lie side by side in memory.  A symmetric result's
// tiles below the diagonal are also stored across it, where a warp's rows lie side by side.
template <int PLANES>
struct NsInner {
  using Params = NsParams;
  static constexpr bool kStaged = true, kStagedOut = true, kRows = true;
  static constexpr int kWarpBytesPerColumn = 0;
  template <int W, int COLS, int ROWS, int PLANE_BYTES>
  struct Tile {
    static_assert(W == 16, "");
    const Params& p;
    const UmmaShape& s;
    unsigned char* staged;  // this thread's row of the first box
    __half* mirror;
    float alpha, beta;
    int n0, col0, swizzle;
    __device__ __forceinline__ Tile(const Params& p_, const UmmaShape& s_, const UmmaTile& tile, bool twice, int m, int n, unsigned char* staging,
                                    int row, int col)
        : p(p_), s(s_), staged(staging + row * 128), n0(n), col0(col), swizzle(row & 7) {
      const float2 f = p.factors[tile.item];
      alpha = f.x;
      beta = p.has_old ? f.y : 0.f;
      mirror = twice && m < s.m ? (__half*)p.out + (long long)tile.item * p.out_item + m : nullptr;
    }
    // Columns n0 + c ... n0 + c + 15.
    __device__ __forceinline__ void group(const uint32_t (&v)[16], int c) {
      const int n = n0 + c, box = (col0 + c) >> 6, j = ((col0 + c) & 63) >> 3;
      uint32_t hi[8], lo[8];  // pairs of halves
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint4* at = reinterpret_cast<uint4*>(staged + box * (ROWS * 128) + (((j + h) ^ swizzle) << 4));
        uint4* at_lo = reinterpret_cast<uint4*>(reinterpret_cast<unsigned char*>(at) + PLANE_BYTES);
        float r[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) r[i] = alpha * __uint_as_float(v[8 * h + i]);
        if (p.has_old) {
          const uint4 was = *at;
          const uint32_t w[4] = {was.x, was.y, was.z, was.w};
          uint32_t l[4] = {0, 0, 0, 0};
          if constexpr (PLANES == 2) {
            const uint4 low = *at_lo;
            l[0] = low.x; l[1] = low.y; l[2] = low.z; l[3] = low.w;
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            if constexpr (PLANES == 2) {
              const float2 g = __half22float2(*reinterpret_cast<const __half2*>(&l[i]));
              f.x += g.x;
              f.y += g.y;
            }
            r[2 * i] = fmaf(beta, f.x, r[2 * i]);
            r[2 * i + 1] = fmaf(beta, f.y, r[2 * i + 1]);
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const __half2 pair = __floats2half2_rn(r[2 * i], r[2 * i + 1]);
          hi[4 * h + i] = *reinterpret_cast<const uint32_t*>(&pair);
          if constexpr (PLANES == 2) {
            const float2 f = __half22float2(pair);
            const __half2 rest = __floats2half2_rn(r[2 * i] - f.x, r[2 * i + 1] - f.y);
            lo[4 * h + i] = *reinterpret_cast<const uint32_t*>(&rest);
          }
        }
        *at = make_uint4(hi[4 * h], hi[4 * h + 1], hi[4 * h + 2], hi[4 * h + 3]);
        if constexpr (PLANES == 2) *at_lo = make_uint4(lo[4 * h], lo[4 * h + 1], lo[4 * h + 2], lo[4 * h + 3]);
      }
      if (mirror) {
        __half* to = mirror + (long long)n * p.out_ld;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          if (n + i < s.n) {
            to[0] = half_of(hi[i / 2], i & 1);
            if constexpr (PLANES == 2) to[p.out_plane] = half_of(lo[i / 2], i & 1);
          }
          to += p.out_ld;
        }
      }
    }
  };
};

// The last step's, into the caller's type and layout: the rows are the fast index, so that a warp stores 32 consecutive elements
// of a column whatever its alignment; the old values come column by column.
template <typename T, int PLANES>
struct NsLast {
  using Params = NsParams;
  static constexpr bool kStaged = true, kStagedOut = false, kRows = false;
  static constexpr int kWarpBytesPerColumn = 0;
  template <int W, int COLS, int ROWS, int PLANE_BYTES>
  struct Tile {
    const UmmaShape& s;
    const __half* staged;
    T* out;
    long long ld;
    float alpha, beta;
    int n0;
    bool live;
    __device__ __forceinline__ Tile(const Params& p, const UmmaShape& s_, const UmmaTile& tile, bool, int m, int n, unsigned char* staging, int row,
                                    int col)
        : s(s_), staged(reinterpret_cast<const __half*>(staging) + col * 128 + row), ld(p.out_ld), n0(n), live(m < s_.m) {
      const float2 f = p.factors[tile.item];
      alpha = f.x;
      beta = f.y;
      out = (T*)p.out + (long long)tile.item * p.out_item + m;
    }
    __device__ __forceinline__ void group(const uint32_t (&v)[W], int c) {
      if (!live) return;
      T* to = out + (long long)(n0 + c) * ld;
#pragma unroll
      for (int i = 0; i < W; ++i) {
        float was = __half2float(staged[(c + i) * 128]);
        if constexpr (PLANES == 2) was += __half2float(staged[PLANE_BYTES / 2 + (c + i) * 128]);
        if (n0 + c + i < s.n) *to = from_f32<T>(fmaf(beta, was, alpha * __uint_as_float(v[i])));
        to += ld;
      }
    }
  };
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
    int box, staged;
    CUtensorMap map;
  };
  Entry e[32];
  int used = 0;
  int get(const CUtensorMap** out, const HalfMatrix& a, int z, int box, int staged = 0) {
    for (int i = 0; i < used; ++i)
      if (e[i].p == a.p && e[i].box == box && e[i].staged == staged) {
        *out = &e[i].map;
        return BLB200_OK;
      }
    if (used == 32) return BLB200_E_INTERNAL;  // four matrices in six boxes each at most
    const int rc = encode_operand(&e[used].map, a.p, false, a.inner, a.outer, z, a.ld * 2, a.plane * 2, box, staged != 0);
    if (rc != BLB200_OK) return rc;
    e[used].p = a.p;
    e[used].box = box;
    e[used].staged = staged;
    *out = &e[used++].map;
    return BLB200_OK;
  }
};

struct Operands {
  HalfMatrix a, b, old, out;
  int m, n, k, batch;
  bool symmetric;
};

template <bool A_MN, bool B_MN, int GROUP, int BN, int PLANES, int SPLIT, class Epilogue>
int launch_product(Maps& maps, const Operands& o, const typename Epilogue::Params& ep, cudaStream_t stream) {
  using C = UmmaConfig<false, A_MN, B_MN, GROUP, BN, PLANES, SPLIT>;
  UmmaShape s{};
  s.m = o.m;
  s.n = o.n;
  s.k = o.k;
  s.batch = o.batch;
  s.symmetric = o.symmetric;  // a_items, b_items stay 0: no operand is shared by the items
  const CUtensorMap *map_a, *map_b, *map_old, *map_out;
  const int z = o.batch * PLANES;
  int rc = maps.get(&map_a, o.a, z, A_MN ? 64 : 128);
  if (rc == BLB200_OK) rc = maps.get(&map_b, o.b, z, B_MN ? 64 : C::kBRows);
  map_old = map_out = map_a;
  const int box = Epilogue::kRows ? 128 / SPLIT : kStagedColumns;
  if (rc == BLB200_OK && ep.has_old) rc = maps.get(&map_old, o.old, z, box, !Epilogue::kRows);
  if (rc == BLB200_OK && Epilogue::kStagedOut) rc = maps.get(&map_out, o.out, z, box, !Epilogue::kRows);
  if (rc == BLB200_OK) rc = launch_umma<C, Epilogue>(*map_a, *map_b, *map_old, *map_out, s, ep, kUmmaNsWait, stream);
  if (rc == BLB200_OK) note_launch("newton_schulz");
  return rc;
}

// Tiles of 256 rows on CTA pairs (256 columns wide, for pairs of halves 128), of 128 x 128 on single CTAs, or of 128 x 128
// with k split over two or four CTAs: whichever should take the least time, in units of about 0.3 us: per 64 k a tile of 128 x
// 128 takes one (pairs of halves: two and a half), a pair's takes 1.3 (2.5), a tile's start and end 12, an exchange 3.
template <bool A_MN, bool B_MN, int PLANES, class Epilogue>
int product(Maps& maps, const Operands& o, const typename Epilogue::Params& ep, cudaStream_t stream) {
  constexpr int kPairN = PLANES == 2 ? 128 : 256;
  auto tiles = [&](int t_m, int t_n) {
    const int tm = (o.m + t_m - 1) / t_m, tn = (o.n + t_n - 1) / t_n;
    const long long each = !o.symmetric ? (long long)tm * tn : t_m == t_n ? symmetric_tiles<1>(tm, tn) : symmetric_tiles<2>(tm, tn);
    return each * o.batch;
  };
  const long long sms = device_info().sm_count, blocks = (o.k + 63) / 64;
  auto rounds = [](long long n, long long units) { return (double)((n + units - 1) / units); };
  using Pair = UmmaConfig<false, A_MN, B_MN, 2, kPairN, PLANES>;
  const long long pairs = umma_capacity<Pair, Epilogue>();
  const double block = PLANES == 2 ? 2.5 : 1.0, pair_block = PLANES == 2 ? 2.5 : 1.3;
  const double pair = rounds(tiles(256, kPairN), pairs) * (blocks * pair_block + 12);
  const double single = rounds(tiles(128, 128), sms) * (blocks * block + 12);
  const long long most[2] = {umma_capacity<UmmaConfig<false, A_MN, B_MN, 1, 128, PLANES, 2>, Epilogue>(),
                             umma_capacity<UmmaConfig<false, A_MN, B_MN, 1, 128, PLANES, 4>, Epilogue>()};
  auto split = [&](int s) { return tiles(128, 128) > most[s / 4] ? 1e300 : (double)((blocks + s - 1) / s) * block + 15; };
  const double best = std::min(std::min(pair, single), std::min(split(2), split(4)));
  if (best == pair) return launch_product<A_MN, B_MN, 2, kPairN, PLANES, 1, Epilogue>(maps, o, ep, stream);
  if (best == single) return launch_product<A_MN, B_MN, 1, 128, PLANES, 1, Epilogue>(maps, o, ep, stream);
  if (best == split(2)) return launch_product<A_MN, B_MN, 1, 128, PLANES, 2, Epilogue>(maps, o, ep, stream);
  return launch_product<A_MN, B_MN, 1, 128, PLANES, 4, Epilogue>(maps, o, ep, stream);
}

int validate_ns(const blb200_newton_schulz_desc* d) {
  if (!d) return BLB200_E_NULL;
  if (!valid_ftype(d->ftype)) return BLB200_E_DTYPE;
  if (d->rows < 0 || d->cols < 0 || d->batch < 0) return BLB200_E_SHAPE;
  if (!readable_layout(d->rows, d->ldx, d->stride_x) || !writable_layout(d->rows, d->cols, d->batch, d->ldy, d->stride_y))
    return BLB200_E_SHAPE;
  if (d->batch > 65535 || d->rows > kMaxDim || d->cols > kMaxDim) return BLB200_E_TOO_LARGE;
  if (d->half_intermediates != 0 && (d->half_intermediates != 1 || d->ftype != BLB200_BF16)) return BLB200_E_UNSUPPORTED;
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

int planes_of(const blb200_newton_schulz_desc* d) { return d->half_intermediates ? 1 : 2; }

struct Layout {
  int planes, p;
  long long ld_x, plane_x, ld_s, plane_s;  // elements
  size_t parts, factors, x, x2, s, b, total;
};
Layout layout_of(const blb200_newton_schulz_desc* d) {
  Layout l;
  const size_t n = d->batch;
  l.planes = planes_of(d);
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
  l.factors = take(n * 3 * kMaxSteps * sizeof(float2));
  l.x = take(n * l.planes * l.plane_x * 2);
  l.x2 = take(n * l.planes * l.plane_x * 2);
  l.s = take(n * l.planes * l.plane_s * 2);
  l.b = take(n * l.planes * l.plane_s * 2);
  l.total = at;
  return l;
}

// Small matrices need none, but are given some like the others, so that a caller has one rule.
size_t workspace_need(const blb200_newton_schulz_desc* d) {
  return newton_schulz_small_supported(d->rows, d->cols, d->batch, planes_of(d)) ? 256 : layout_of(d).total;
}

Plan plan_of(const blb200_newton_schulz_desc* d) {
  Plan plan;
  plan.eps = d->eps;
  plan.steps = d->steps;
  double sigma = 1.0;
  for (int i = 0; i < d->steps; ++i) {
    for (int j = 0; j < 3; ++j) plan.q[3 * i + j] = d->coefficients[(d->coefficient_sets == 1 ? 0 : 3 * i) + j];
    plan.scales[i] = step_scales(plan.q + 3 * i, sigma, i + 1 == d->steps);
  }
  return plan;
}

template <typename T, int PLANES>
int run(const blb200_newton_schulz_desc* d, const Layout& l, char* ws, cudaStream_t stream) {
  const Plan plan = plan_of(d);
  const int r = d->rows, c = d->cols, p = l.p, batch = d->batch;
  const Matrices g{const_cast<void*>(d->x), r, c, batch, d->ldx, d->stride_x};
  double* parts = (double*)(ws + l.parts);
  float2* factors = (float2*)(ws + l.factors);
  HalfMatrix x{(__half*)(ws + l.x), r, c, l.ld_x, l.plane_x}, x2{(__half*)(ws + l.x2), r, c, l.ld_x, l.plane_x};
  const HalfMatrix s{(__half*)(ws + l.s), p, p, l.ld_s, l.plane_s}, b{(__half*)(ws + l.b), p, p, l.ld_s, l.plane_s};
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
  using Inner = NsInner<PLANES>;
  using Last = NsLast<T, PLANES>;
  for (int i = 0; i < d->steps && rc == BLB200_OK; ++i) {
    const float2* f = factors + (long long)i * 3 * batch;
    const typename Inner::Params gram{f, 0, s.p, l.ld_s, l.plane_s, PLANES * l.plane_s};
    const Operands gram_o{x, x, s, s, p, p, r <= c ? c : r, batch, true};
    rc = r <= c ? product<true, true, PLANES, Inner>(maps, gram_o, gram, stream) : product<false, false, PLANES, Inner>(maps, gram_o, gram, stream);
    if (rc != BLB200_OK) break;
    const typename Inner::Params square{f + batch, 1, b.p, l.ld_s, l.plane_s, PLANES * l.plane_s};
    rc = product<false, false, PLANES, Inner>(maps, Operands{s, s, s, b, p, p, p, batch, true}, square, stream);
    if (rc != BLB200_OK) break;
    if (i + 1 < d->steps) {
      // the columns of X as the tile's rows, so that the epilogue goes along memory
      const typename Inner::Params update{f + 2 * batch, 1, x2.p, l.ld_x, l.plane_x, PLANES * l.plane_x};
      const Operands update_o{r <= c ? x : b, r <= c ? b : x, x, x2, c, r, p, batch, false};
      rc = r <= c ? product<false, false, PLANES, Inner>(maps, update_o, update, stream)
                  : product<false, true, PLANES, Inner>(maps, update_o, update, stream);
      std::swap(x, x2);
    } else {
      const typename Last::Params last{f + 2 * batch, 1, d->y, d->ldy, 0, d->stride_y};
      const Operands last_o{r <= c ? b : x, r <= c ? x : b, x, x2, r, c, p, batch, false};
      rc = r <= c ? product<false, false, PLANES, Last>(maps, last_o, last, stream) : product<true, false, PLANES, Last>(maps, last_o, last, stream);
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
  return blb200::workspace_need(d);
}

extern "C" int blb200_newton_schulz(const blb200_newton_schulz_desc* d, void* workspace, size_t workspace_bytes, void* cuda_stream) {
  using namespace blb200;
  const int rc = validate_ns(d);
  if (rc != BLB200_OK) return rc;
  if (d->rows == 0 || d->cols == 0 || d->batch == 0) return BLB200_OK;
  if (!workspace) return BLB200_E_NULL;
  if (workspace_bytes < workspace_need(d) || reinterpret_cast<uintptr_t>(workspace) % 256) return BLB200_E_SHAPE;
  cudaStream_t stream = (cudaStream_t)cuda_stream;
  if (newton_schulz_small_supported(d->rows, d->cols, d->batch, planes_of(d))) {
    const Matrices g{const_cast<void*>(d->x), d->rows, d->cols, d->batch, d->ldx, d->stride_x};
    return launch_newton_schulz_small(g, Matrices{d->y, d->rows, d->cols, d->batch, d->ldy, d->stride_y}, d->ftype, planes_of(d), plan_of(d), stream);
  }
  const Layout l = layout_of(d);
  if (d->ftype == BLB200_F32) return run<float, 2>(d, l, (char*)workspace, stream);
  if (d->ftype == BLB200_F16) return run<__half, 2>(d, l, (char*)workspace, stream);
  if (l.planes == 2) return run<__nv_bfloat16, 2>(d, l, (char*)workspace, stream);
  return run<__nv_bfloat16, 1>(d, l, (char*)workspace, stream);
}
