// 8-bit integer products with scales:  C <- alpha diag(sa) A^T B diag(sb) + beta C,  A (k x m) and B (k x n)
// int8 with k fastest.  The sums are exact 32-bit integers, so every kernel here gives the same bits.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "lowp.cuh"
#include "umma_gemm.cuh"

namespace blb200 {
namespace {

struct GemmI8Params {
  const int8_t* a;
  const int8_t* b;
  void* c;
  const float* scale_a;
  const float* scale_b;
  int m, n, k, batch;
  long long lda, ldb, ldc, sa, sb, sc, ssa, ssb;
  float alpha, beta;
};

// acc * (alpha sa) * sb + beta * prior, in float, rounded once to T.
template <typename T>
__device__ __forceinline__ void store_c(T* c, int acc, float sa, float sb, float alpha, float beta) {
  float v = (float)acc * (sa * alpha) * sb;
  if (beta != 0.f) v = fmaf(beta, to_f32(*c), v);
  *c = from_f32<T>(v);
}

__device__ __forceinline__ void mma_i8(int (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}

// ---- few columns -----------------------------------------------------------------------------------
// Up to 16 tokens: the weights are read once and that is the time.  A CTA owns MT tiles of 16 rows of C; its eight warps
// split k, and every lane holds its share of a 16 x 64 slab of weights by two 16-byte loads straight into mma.sync
// fragments: the order of k inside a slab does not matter as long as both operands share it, so lane (g, t) takes bytes
// 16 t .. 16 t + 15 of rows g and g + 8 (and of token g), words 0, 1 for one instruction and 2, 3 for the next.  The slabs of
// kFlight row tiles and k steps are in flight per warp before the first is used.  The more rows a CTA owns, the less often
// the tokens are read (from L2); the fewer, the more SMs take part.  Before it waits for the kernel that produced
// its tokens, each lane asks for its first weights to be brought into L2, which has no effect but on time.  The warps' sums
// meet in shared memory.
constexpr int kFlight = 4, kFewColumns = 16;

template <bool WHOLE>
__device__ __forceinline__ uint4 load16(const int8_t* src, int valid, const int8_t* lo, const int8_t* hi) {
  if (WHOLE && valid >= 16) return *reinterpret_cast<const uint4*>(src);
  if (valid <= 0) return make_uint4(0, 0, 0, 0);
  Words16 w;
  w.load(src, valid, lo, hi);
  return w.edge ? load16_bytes(src, valid) : valid < 16 ? first_bytes(w.value(src), valid) : w.value(src);
}

// WHOLE: both operands' columns start on 16-byte boundaries.
template <typename T, int NT, int MT, bool WHOLE>
__global__ void __launch_bounds__(256) gemm_i8_few_kernel(GemmI8Params p, int tiles_m) {
  constexpr int kSlabs = kFlight / MT;  // k steps in flight
  __shared__ int part[8][NT][16][9];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const long long item = blockIdx.x / tiles_m;
  const int m0 = (int)(blockIdx.x - item * tiles_m) * 16 * MT;
  const int8_t* a = p.a + item * p.sa;
  const int8_t* b = p.b + item * p.sb;
  const int8_t* a_end = a + (long long)(p.m - 1) * p.lda + p.k;
  const int8_t* b_end = b + (long long)(p.n - 1) * p.ldb + p.k;
  // this warp's k range, in whole slabs
  const int slabs = (p.k + 63) / 64, each = (slabs + 7) / 8;
  const int k_begin = warp * each * 64 + t * 16, k_end = min(p.k, (warp + 1) * each * 64);
  const int8_t* row[2 * MT];
#pragma unroll
  for (int i = 0; i < 2 * MT; ++i) row[i] = a + (long long)min(m0 + g + 8 * i, p.m - 1) * p.lda;
  const int8_t* col[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) col[j] = b + (long long)min(8 * j + g, p.n - 1) * p.ldb;
#pragma unroll
  for (int s = 0; s < kSlabs; ++s)
    if (k_begin + 64 * s < k_end) {
#pragma unroll
      for (int i = 0; i < 2 * MT; ++i) asm volatile("prefetch.global.L2 [%0];" ::"l"(row[i] + k_begin + 64 * s));
    }
  griddep_wait();
  griddep_launch();

  int acc[MT][NT][4];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][j][e] = 0;
  for (int k0 = k_begin; k0 - t * 16 < k_end; k0 += 64 * kSlabs) {
    uint4 w[kSlabs][2 * MT], x[kSlabs][NT];
#pragma unroll
    for (int s = 0; s < kSlabs; ++s) {
#pragma unroll
      for (int i = 0; i < 2 * MT; ++i) w[s][i] = load16<WHOLE>(row[i] + k0 + 64 * s, k_end - (k0 + 64 * s), a, a_end);
    }
#pragma unroll
    for (int s = 0; s < kSlabs; ++s)
#pragma unroll
      for (int j = 0; j < NT; ++j) x[s][j] = load16<WHOLE>(col[j] + k0 + 64 * s, k_end - (k0 + 64 * s), b, b_end);
#pragma unroll
    for (int s = 0; s < kSlabs; ++s)
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const uint4 lo = w[s][2 * i], hi = w[s][2 * i + 1], y = x[s][j];
          const uint32_t a0[4] = {lo.x, hi.x, lo.y, hi.y}, b0[2] = {y.x, y.y};
          const uint32_t a1[4] = {lo.z, hi.z, lo.w, hi.w}, b1[2] = {y.z, y.w};
          mma_i8(acc[i][j], a0, b0);
          mma_i8(acc[i][j], a1, b1);
        }
  }
  T* c = (T*)p.c + item * p.sc;
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    if (i > 0) __syncthreads();
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) part[warp][j][g + 8 * (e >> 1)][2 * t + (e & 1)] = acc[i][j][e];
    __syncthreads();
    for (int o = threadIdx.x; o < 16 * 8 * NT; o += 256) {
      const int r = o & 15, n = o >> 4, m = m0 + 16 * i + r;
      if (m >= p.m || n >= p.n) continue;
      int sum = 0;
#pragma unroll
      for (int w = 0; w < 8; ++w) sum += part[w][n >> 3][r][n & 7];
      store_c(c + (long long)n * p.ldc + m, sum, p.scale_a ? p.scale_a[item * p.ssa + m] : 1.f,
              p.scale_b ? p.scale_b[item * p.ssb + n] : 1.f, p.alpha, p.beta);
    }
  }
}

bool columns_16(const int8_t* base, long long ld, long long stride, int cols, int batch) {
  return reinterpret_cast<uintptr_t>(base) % 16 == 0 && (ld % 16 == 0 || cols == 1) && (stride % 16 == 0 || batch == 1);
}

int launch_gemm_i8_few(const GemmI8Params& p, int ftype, cudaStream_t stream) {
  const bool whole = columns_16(p.a, p.lda, p.sa, p.m, p.batch) && columns_16(p.b, p.ldb, p.sb, p.n, p.batch);
  // as many rows per CTA as leave a CTA for every SM
  const long long sms = device_info().sm_count;
  auto ctas = [&](int mt) { return (long long)((p.m + 16 * mt - 1) / (16 * mt)) * p.batch; };
  const int mt = ctas(4) >= sms ? 4 : ctas(2) >= sms ? 2 : 1;
  const OverlappedLaunch launch((unsigned)ctas(mt), 256, stream);
  const int tiles_m = (p.m + 16 * mt - 1) / (16 * mt);
  return with_ftype(ftype, [&](auto v) {
    using T = decltype(v);
    auto with_rows = [&](auto nt, auto rows) {
      constexpr int NT = decltype(nt)::value, MT = decltype(rows)::value;
      return whole ? cudaLaunchKernelEx(&launch.cfg, gemm_i8_few_kernel<T, NT, MT, true>, p, tiles_m)
                   : cudaLaunchKernelEx(&launch.cfg, gemm_i8_few_kernel<T, NT, MT, false>, p, tiles_m);
    };
    auto with_columns = [&](auto nt) {
      return mt == 4   ? with_rows(nt, std::integral_constant<int, 4>{})
             : mt == 2 ? with_rows(nt, std::integral_constant<int, 2>{})
                       : with_rows(nt, std::integral_constant<int, 1>{});
    };
    const cudaError_t e = p.n <= 8    ? with_columns(std::integral_constant<int, 1>{})
                                      : with_columns(std::integral_constant<int, 2>{});
    if (e == cudaSuccess) note_launch("gemm_i8_few");
    return (int)e;
  });
}

// ---- tcgen05 tiles ---------------------------------------------------------------------------------
// Rows of C (channels) on the M side, columns (tokens) on the N side: both operands are stored with k fastest, which
// is the K-major form, and a thread of the epilogue owns one row, so that a warp stores 32 consecutive elements of a
// column of C.
enum { kUmmaI8Wait = 500 };

struct I8Params {
  GemmI8Params g;
  int ftype;
};

// The scales of a warp's columns are brought into shared memory while the products run; a whole group of columns with beta = 0
// then costs about seven instructions per column and row of 32 (with the scale read from memory, the bounds and beta
// tested for each element it was 36, and the epilogue, not the MMAs, set the time of an 8192^3 product).
struct I8Epilogue {
  using Params = I8Params;
  static constexpr bool kStaged = false, kRows = false;
  static constexpr int kWarpBytesPerColumn = 4;
  template <int W, int COLS, int ROWS, int PLANE_BYTES>
  struct Tile;
};
template <int W, int COLS, int ROWS, int PLANE_BYTES>
struct I8Epilogue::Tile {
  const I8Params& p;
  float* scales;
  long long item, m;
  int n0;
  float sa;
  bool live;
  __device__ __forceinline__ Tile(const Params& p_, const UmmaShape&, const UmmaTile& tile, bool, int m_, int n, unsigned char* scratch, int, int)
      : p(p_), scales(reinterpret_cast<float*>(scratch)), item(tile.item), m(m_), n0(n), live(m_ < p_.g.m) {
    sa = p.g.scale_a && live ? p.g.scale_a[item * p.g.ssa + m] : 1.f;
    sa *= p.g.alpha;
    const float* sb = p.g.scale_b ? p.g.scale_b + item * p.g.ssb + n : nullptr;
    __syncwarp();
    for (int i = threadIdx.x & 31; i < COLS; i += 32) scales[i] = sb && n + i < p.g.n ? sb[i] : 1.f;
    __syncwarp();
  }
  // Columns n0 + c ... n0 + c + W - 1 of the row.
  __device__ __forceinline__ void group(const uint32_t (&v)[W], int c) {
    if (!live) return;
    if (p.ftype == BLB200_F32) store_as<float>(v, c);
    else if (p.ftype == BLB200_F16) store_as<__half>(v, c);
    else store_as<__nv_bfloat16>(v, c);
  }
  template <typename T>
  __device__ __forceinline__ void store_as(const uint32_t (&v)[W], int c) {
    const int n = n0 + c;
    T* at = (T*)p.g.c + item * p.g.sc + m + (long long)n * p.g.ldc;
    float r[W];
#pragma unroll
    for (int i = 0; i < W; i += 4) {
      const float4 sb = *reinterpret_cast<const float4*>(scales + c + i);
      r[i] = (float)(int)v[i] * sa * sb.x;
      r[i + 1] = (float)(int)v[i + 1] * sa * sb.y;
      r[i + 2] = (float)(int)v[i + 2] * sa * sb.z;
      r[i + 3] = (float)(int)v[i + 3] * sa * sb.w;
    }
    if (p.g.beta == 0.f && n + W <= p.g.n) {
#pragma unroll
      for (int i = 0; i < W; ++i) {
        *at = from_f32<T>(r[i]);
        at += p.g.ldc;
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < W; ++i) {
      if (n + i < p.g.n) *at = from_f32<T>(p.g.beta != 0.f ? fmaf(p.g.beta, to_f32(*at), r[i]) : r[i]);
      at += p.g.ldc;
    }
  }
};

// Estimated time of one way to cut C into tiles, in SM cycles: rounds of tiles, each as long as the slower of its MMAs
// (8192 products per cycle) and of its fetches (about 50 bytes per cycle and SM from L2), and about 2500 cycles for filling the ring
// and the epilogue; splitting k costs an exchange of about 1500.  With plain loads a block of k takes 1.25 us at 64 columns and 1.5
// at 128, a tile's start and end 1.7 and 3, a split 2.7 more (fitted to all choices at twenty sizes, 1.9 GHz): that picks the
// fastest of the seven, or one within 2 % of it, from 17 x 4096 x 129 to 8192 x 1001 x 8191, but for 20 x 100 x 200 (12.9 us, 11.6 split).
struct TileChoice {
  int group, bn, split;
  double time;
};
template <int GROUP, int BN, int SPLIT, bool PLAIN>
double tile_time(const GemmI8Params& p) {
  constexpr int kBM = 128 * GROUP;
  const long long units = umma_capacity<UmmaConfig<true, false, false, GROUP, BN, 1, SPLIT, PLAIN>, I8Epilogue>();
  const long long tiles = (long long)((p.m + kBM - 1) / kBM) * ((p.n + BN - 1) / BN) * p.batch;
  if (SPLIT > 1 && tiles > units) return 1e300;
  const double blocks = (double)((p.k + 127) / 128);
  const double per = PLAIN ? 1900.0 + 7.5 * BN : std::max(2.0 * BN, (16384.0 + 128.0 * BN / GROUP) / 50.0);
  const double tile = PLAIN ? 700.0 + 40.0 * BN : 2500.0, exchange = SPLIT == 1 ? 0.0 : PLAIN ? 5100.0 : 1500.0;
  return (double)((tiles + units - 1) / units) * (ceil(blocks / SPLIT) * per + tile) + exchange;
}
template <bool PLAIN>
TileChoice choose_tiles(const GemmI8Params& p) {
  TileChoice best{1, 128, 1, tile_time<1, 128, 1, PLAIN>(p)};
  auto consider = [&](int group, int bn, int split, double t) {
    if (t < best.time) best = TileChoice{group, bn, split, t};
  };
  consider(1, 128, 2, tile_time<1, 128, 2, PLAIN>(p));
  consider(1, 128, 4, tile_time<1, 128, 4, PLAIN>(p));
  consider(1, 64, 1, tile_time<1, 64, 1, PLAIN>(p));
  consider(1, 64, 2, tile_time<1, 64, 2, PLAIN>(p));
  consider(1, 64, 4, tile_time<1, 64, 4, PLAIN>(p));
  consider(1, 64, 8, tile_time<1, 64, 8, PLAIN>(p));
  if constexpr (!PLAIN) consider(2, 256, 1, tile_time<2, 256, 1, false>(p));
  return best;
}

template <int GROUP, int BN, int SPLIT, bool PLAIN>
int launch_umma_i8(const GemmI8Params& p, int ftype, cudaStream_t stream) {
  using C = UmmaConfig<true, false, false, GROUP, BN, 1, SPLIT, PLAIN>;
  UmmaShape s{};
  s.m = p.m;
  s.n = p.n;
  s.k = p.k;
  s.batch = p.batch;
  s.a_items = p.batch > 1 && p.sa == 0 ? 1 : p.batch;
  s.b_items = p.batch > 1 && p.sb == 0 ? 1 : p.batch;
  CUtensorMap map_a{}, map_b{};
  if (!PLAIN) {
    // a single column's ld is not used for addressing, but the map wants a multiple of 16
    auto ld_of = [](long long ld, int cols) { return cols == 1 ? (ld + 15) / 16 * 16 : ld; };
    int rc = encode_operand(&map_a, p.a, true, p.k, p.m, s.a_items, ld_of(p.lda, p.m), p.sa, 128);
    if (rc == BLB200_OK) rc = encode_operand(&map_b, p.b, true, p.k, p.n, s.b_items, ld_of(p.ldb, p.n), p.sb, C::kBRows);
    if (rc != BLB200_OK) return rc;
  }
  const PlainOperands po{p.a, p.b, p.lda, p.ldb, p.sa, p.sb};
  const int e = launch_umma<C, I8Epilogue>(map_a, map_b, map_a, map_b, s, I8Params{p, ftype}, kUmmaI8Wait, stream, po);
  if (e == 0) note_launch(PLAIN ? "gemm_i8_plain" : "gemm_i8_umma");
  return e;
}

template <bool PLAIN>
int launch_tiles_i8(const GemmI8Params& p, const TileChoice& c, int ftype, cudaStream_t stream) {
  if constexpr (!PLAIN)
    if (c.group == 2) return launch_umma_i8<2, 256, 1, false>(p, ftype, stream);
#define BLB_TILE(BN_, SPLIT_) \
  if (c.bn == BN_ && c.split == SPLIT_) return launch_umma_i8<1, BN_, SPLIT_, PLAIN>(p, ftype, stream);
  BLB_TILE(64, 1) BLB_TILE(64, 2) BLB_TILE(64, 4) BLB_TILE(64, 8)
  BLB_TILE(128, 1) BLB_TILE(128, 2) BLB_TILE(128, 4)
#undef BLB_TILE
  return BLB200_E_INTERNAL;
}

int dispatch_gemm_i8(const GemmI8Params& p, int ftype, cudaStream_t stream) {
  if (p.n <= kFewColumns && ((long long)(p.m + 15) / 16) * p.batch <= 0x7fffffffll) return launch_gemm_i8_few(p, ftype, stream);
  const bool aligned = p.k > 0 && columns_16(p.a, p.lda, p.sa, p.m, p.batch) && columns_16(p.b, p.ldb, p.sb, p.n, p.batch);
  if (aligned) {
    const int rc = launch_tiles_i8<false>(p, choose_tiles<false>(p), ftype, stream);
    if (rc != BLB200_E_INTERNAL) return rc;  // a driver that refuses the tensor maps: plain loads take it
  }
  return launch_tiles_i8<true>(p, choose_tiles<true>(p), ftype, stream);
}

constexpr int kMaxK = 131071;  // 128 * 128 * k stays below 2^31

int validate_gemm_i8(const blb200_gemm_i8_desc* d) {
  if (!d) return BLB200_E_NULL;
  if (!valid_ftype(d->ftype_c)) return BLB200_E_DTYPE;
  if (d->m < 0 || d->n < 0 || d->k < 0 || d->batch < 0) return BLB200_E_SHAPE;
  if (d->k > kMaxK || d->m > kMaxDim || d->n > kMaxDim) return BLB200_E_TOO_LARGE;
  if (!readable_layout(d->k, d->lda, d->stride_a) || !readable_layout(d->k, d->ldb, d->stride_b) ||
      !writable_layout(d->m, d->n, d->batch, d->ldc, d->stride_c) || d->stride_scale_a < 0 || d->stride_scale_b < 0)
    return BLB200_E_SHAPE;
  if (d->m > 0 && d->n > 0 && d->batch > 0 && (!d->c || (d->k > 0 && (!d->a || !d->b)))) return BLB200_E_NULL;
  return BLB200_OK;
}

}  // namespace
int gemm_i8_device_status(int* out) { return read_device_status_word(out); }
int gemm_i8_device_status_clear() { return clear_device_status_word(); }
}  // namespace blb200

extern "C" int blb200_gemm_i8(const blb200_gemm_i8_desc* d, void* cuda_stream) {
  using namespace blb200;
  const int rc = validate_gemm_i8(d);
  if (rc != BLB200_OK) return rc;
  if (d->m == 0 || d->n == 0 || d->batch == 0) return BLB200_OK;
  GemmI8Params p{d->a,   d->b,   d->c,        d->scale_a,  d->scale_b,  d->m,           d->n,
                 d->k,   d->batch, d->lda,    d->ldb,      d->ldc,      d->stride_a,    d->stride_b,
                 d->stride_c, d->stride_scale_a, d->stride_scale_b, (float)d->alpha, (float)d->beta};
  if (p.k == 0) p.scale_a = p.scale_b = nullptr;  // C <- beta * C, whatever the scales hold
  return dispatch_gemm_i8(p, d->ftype_c, (cudaStream_t)cuda_stream);
}
