// 8-bit integer products with scales:  C <- alpha diag(sa) A^T B diag(sb) + beta C,  A (k x m) and B (k x n)
// int8 with k fastest.  The sums are exact 32-bit integers, so every kernel here gives the same bits.
//
// Tile kernel for any alignment: 128 x 128 of C per CTA, eight warps of 32 x 64, mma.sync m16n8k32 on
// 64-byte k chunks staged in shared memory (pitch 80 bytes: the eight rows of a fragment request fall
// into different banks).  Rows that start off a 4-byte boundary are read as aligned words and shifted
// together; a word is read whole only where all of it lies inside the operand.
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

// alpha * (acc * sa) * sb + beta * prior, in float, rounded once to T.
template <typename T>
__device__ __forceinline__ void store_c(T* c, int acc, float sa, float sb, float alpha, float beta) {
  float v = alpha * (((float)acc * sa) * sb);
  if (beta != 0.f) v = fmaf(beta, to_f32(*c), v);
  *c = from_f32<T>(v);
}

constexpr int kTile = 128, kChunk = 64, kPitch = 80;

// 16 bytes at `src` (any alignment) of which the first `valid` exist, the rest zero.  [lo, hi) is the operand.
__device__ __forceinline__ uint4 load16_any(const int8_t* src, int valid, const int8_t* lo, const int8_t* hi) {
  uint32_t w[4] = {0, 0, 0, 0};
  if (valid >= 16) {
    const int off = (int)(reinterpret_cast<uintptr_t>(src) & 3u);
    const int8_t* base = src - off;
    if (off == 0) {
      const uint32_t* s = reinterpret_cast<const uint32_t*>(base);
      return make_uint4(s[0], s[1], s[2], s[3]);
    }
    if (base >= lo && base + 20 <= hi) {
      const uint32_t* s = reinterpret_cast<const uint32_t*>(base);
      const uint32_t x0 = s[0], x1 = s[1], x2 = s[2], x3 = s[3], x4 = s[4];
      const int sh = off * 8;
      return make_uint4(__funnelshift_r(x0, x1, sh), __funnelshift_r(x1, x2, sh), __funnelshift_r(x2, x3, sh),
                        __funnelshift_r(x3, x4, sh));
    }
  }
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (i < valid) w[i >> 2] |= (uint32_t)(uint8_t)src[i] << (8 * (i & 3));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ void mma_i8(int (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}

template <typename T>
__global__ void __launch_bounds__(256) gemm_i8_any_kernel(GemmI8Params p, int tiles_m, long long tiles_per_item, long long tiles) {
  __shared__ __align__(16) unsigned char tile_a[kTile * kPitch];
  __shared__ __align__(16) unsigned char tile_b[kTile * kPitch];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int wm = (warp & 3) * 32, wn = (warp >> 2) * 64;
  for (long long tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const long long item = tile / tiles_per_item;
    const int rem = (int)(tile - item * tiles_per_item);
    const int m0 = rem % tiles_m * kTile, n0 = rem / tiles_m * kTile;
    const int8_t* a = p.a + item * p.sa;
    const int8_t* b = p.b + item * p.sb;
    const int8_t* a_end = a + (long long)(p.m - 1) * p.lda + p.k;
    const int8_t* b_end = b + (long long)(p.n - 1) * p.ldb + p.k;
    int acc[2][8][4];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][j][e] = 0;
    uint4 next[4];
    auto fetch = [&](int k0) {
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int c = tid + (u & 1) * 256, row = c >> 2, kk = k0 + (c & 3) * 16;
        const bool is_a = u < 2;
        const int r = (is_a ? m0 : n0) + row;
        const int valid = r < (is_a ? p.m : p.n) ? p.k - kk : 0;
        next[u] = valid > 0 ? load16_any((is_a ? a + (long long)r * p.lda : b + (long long)r * p.ldb) + kk, valid,
                                         is_a ? a : b, is_a ? a_end : b_end)
                            : make_uint4(0, 0, 0, 0);
      }
    };
    fetch(0);
    for (int k0 = 0; k0 < p.k; k0 += kChunk) {
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int c = tid + (u & 1) * 256;
        *reinterpret_cast<uint4*>((u < 2 ? tile_a : tile_b) + (c >> 2) * kPitch + (c & 3) * 16) = next[u];
      }
      __syncthreads();
      if (k0 + kChunk < p.k) fetch(k0 + kChunk);
#pragma unroll
      for (int ks = 0; ks < kChunk; ks += 32) {
        uint32_t fa[2][4], fb[8][2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const unsigned char* s = tile_a + (wm + i * 16 + g) * kPitch + ks + t * 4;
          fa[i][0] = *reinterpret_cast<const uint32_t*>(s);
          fa[i][1] = *reinterpret_cast<const uint32_t*>(s + 8 * kPitch);
          fa[i][2] = *reinterpret_cast<const uint32_t*>(s + 16);
          fa[i][3] = *reinterpret_cast<const uint32_t*>(s + 8 * kPitch + 16);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const unsigned char* s = tile_b + (wn + j * 8 + g) * kPitch + ks + t * 4;
          fb[j][0] = *reinterpret_cast<const uint32_t*>(s);
          fb[j][1] = *reinterpret_cast<const uint32_t*>(s + 16);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 8; ++j) mma_i8(acc[i][j], fa[i], fb[j]);
      }
      __syncthreads();
    }
    T* c = (T*)p.c + item * p.sc;
    const float* sa = p.scale_a ? p.scale_a + item * p.ssa : nullptr;
    const float* sb = p.scale_b ? p.scale_b + item * p.ssb : nullptr;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int row = m0 + wm + i * 16 + h * 8 + g;
        if (row >= p.m) continue;
        const float fsa = sa ? sa[row] : 1.f;
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int col = n0 + wn + j * 8 + t * 2 + e;
            if (col < p.n)
              store_c(c + (long long)col * p.ldc + row, acc[i][j][h * 2 + e], fsa, sb ? sb[col] : 1.f, p.alpha, p.beta);
          }
      }
  }
}

int launch_gemm_i8_any(const GemmI8Params& p, int ftype, cudaStream_t stream) {
  const int tiles_m = (p.m + kTile - 1) / kTile;
  const long long per_item = (long long)tiles_m * ((p.n + kTile - 1) / kTile), tiles = per_item * p.batch;
  const long long cap = (long long)device_info().sm_count * 2;
  return with_ftype(ftype, [&](auto t) {
    gemm_i8_any_kernel<decltype(t)><<<(unsigned)(tiles < cap ? tiles : cap), 256, 0, stream>>>(p, tiles_m, per_item, tiles);
    const int e = (int)cudaGetLastError();
    if (e == 0) note_launch("gemm_i8_any");
    return e;
  });
}

// ---- few columns -----------------------------------------------------------------------------------
// Up to 32 tokens: the weights are read once and that is the time.  A CTA owns MT tiles of 16 rows of C; its eight warps
// split k, and every lane holds its share of a 16 x 64 slab of weights by two 16-byte loads straight into mma.sync
// fragments: the order of k inside a slab does not matter as long as both operands share it, so lane (g, t) takes bytes
// 16 t .. 16 t + 15 of rows g and g + 8 (and of token g), words 0, 1 for one instruction and 2, 3 for the next.  The slabs of
// kFlight row tiles and k steps are in flight per warp before the first is used.  The more rows a CTA owns, the less often
// the tokens are read (from L2); the fewer, the more SMs take part.  Before it waits for the kernel that produced
// its tokens, each lane asks for its first weights to be brought into L2, which has no effect but on time.  The warps' sums
// meet in shared memory.
constexpr int kFlight = 4;

template <bool WHOLE>
__device__ __forceinline__ uint4 load16(const int8_t* src, int valid, const int8_t* lo, const int8_t* hi) {
  if (WHOLE && valid >= 16) return *reinterpret_cast<const uint4*>(src);
  if (valid <= 0) return make_uint4(0, 0, 0, 0);
  return load16_any(src, valid, lo, hi);
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
                          : p.n <= 16 ? with_columns(std::integral_constant<int, 2>{})
                                      : with_columns(std::integral_constant<int, 4>{});
    if (e == cudaSuccess) note_launch("gemm_i8_few");
    return (int)e;
  });
}

// ---- tcgen05 tiles ---------------------------------------------------------------------------------
// Rows of C (channels) on the M side, columns (tokens) on the N side: both operands are stored with k fastest, which
// is the K-major form, and a thread of the epilogue owns one row, so that a warp stores 32 consecutive elements of a
// column of C.
enum { kUmmaI8Wait = 500 };

template <typename T>
struct I8Epilogue {
  using Params = GemmI8Params;
  T* c;
  const float* sb;
  const Params& p;
  float sa;
  bool live;
  __device__ I8Epilogue(const Params& p_, const UmmaShape&, const UmmaTile& tile, bool, int m) : p(p_), live(m < p_.m) {
    c = (T*)p.c + (long long)tile.item * p.sc + m;
    sa = p.scale_a && live ? p.scale_a[(long long)tile.item * p.ssa + m] : 1.f;
    sb = p.scale_b ? p.scale_b + (long long)tile.item * p.ssb : nullptr;
  }
  template <int N>
  __device__ void store(const uint32_t (&v)[N], int n) {
    if (!live) return;
    T* at = c + (long long)n * p.ldc;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (n + i < p.n) store_c(at + (long long)i * p.ldc, (int)v[i], sa, sb ? sb[n + i] : 1.f, p.alpha, p.beta);
  }
};

bool umma_i8_supported(const GemmI8Params& p) {
  return p.k > 0 && columns_16(p.a, p.lda, p.sa, p.m, p.batch) && columns_16(p.b, p.ldb, p.sb, p.n, p.batch) && encode_tiled_fn() != nullptr;
}

template <int GROUP, int BN>
int launch_umma_i8(const GemmI8Params& p, int ftype, cudaStream_t stream) {
  using C = UmmaConfig<true, false, false, GROUP, BN, 1>;
  UmmaShape s{};
  s.m = p.m;
  s.n = p.n;
  s.k = p.k;
  s.batch = p.batch;
  s.a_items = p.batch > 1 && p.sa == 0 ? 1 : p.batch;
  s.b_items = p.batch > 1 && p.sb == 0 ? 1 : p.batch;
  // a single column's ld is not used for addressing, but the map wants a multiple of 16
  auto ld_of = [](long long ld, int cols) { return cols == 1 ? (ld + 15) / 16 * 16 : ld; };
  CUtensorMap map_a, map_b;
  int rc = encode_operand(&map_a, p.a, true, p.k, p.m, s.a_items, ld_of(p.lda, p.m), p.sa, 128);
  if (rc == BLB200_OK) rc = encode_operand(&map_b, p.b, true, p.k, p.n, s.b_items, ld_of(p.ldb, p.n), p.sb, C::kBRows);
  if (rc != BLB200_OK) return rc;
  return with_ftype(ftype, [&](auto t) {
    const int e = launch_umma<C, I8Epilogue<decltype(t)>>(map_a, map_b, s, p, kUmmaI8Wait, stream);
    if (e == 0) note_launch("gemm_i8_umma");
    return e;
  });
}

int launch_umma_i8_any(const GemmI8Params& p, int ftype, cudaStream_t stream) {
  if (p.n <= 64) return launch_umma_i8<1, 64>(p, ftype, stream);
  const long long pairs = (long long)((p.m + 255) / 256) * ((p.n + 255) / 256) * p.batch, units = device_info().sm_count / 2;
  if (pairs >= units) return launch_umma_i8<2, 256>(p, ftype, stream);
  return launch_umma_i8<1, 128>(p, ftype, stream);
}

constexpr int kMaxK = 131071;  // 128 * 128 * k stays below 2^31

int validate_gemm_i8(const blb200_gemm_i8_desc* d) {
  if (!d) return BLB200_E_NULL;
  if (!valid_ftype(d->ftype_c)) return BLB200_E_DTYPE;
  if (d->m < 0 || d->n < 0 || d->k < 0 || d->batch < 0) return BLB200_E_SHAPE;
  if (d->k > kMaxK) return BLB200_E_TOO_LARGE;
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
  if (p.n <= 32 && p.k > 0 && ((long long)(p.m + 15) / 16) * p.batch <= 0x7fffffffll)
    return launch_gemm_i8_few(p, d->ftype_c, (cudaStream_t)cuda_stream);
  if (umma_i8_supported(p)) {
    const int e = launch_umma_i8_any(p, d->ftype_c, (cudaStream_t)cuda_stream);
    if (e != BLB200_E_INTERNAL) return e;  // a driver that refuses the tensor map: the tile kernel takes it
  }
  return launch_gemm_i8_any(p, d->ftype_c, (cudaStream_t)cuda_stream);
}
