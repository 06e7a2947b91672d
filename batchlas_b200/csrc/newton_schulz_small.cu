// The Newton-Schulz iteration on small matrices: one CTA per matrix, everything but G and the result in its shared memory.
//
// Per step  S = X X^T,  B = b S + c S^2,  X <- a X + B X  are three tcgen05 products of one 128-row tile, issued by one thread,
// each followed by an epilogue of all sixteen warps that scales the accumulator in tensor memory and writes the next operand.
// X (p x q, p the shorter side, padded with zeros to 128 x 64 QB) lies as blocks of 64 columns of 128 rows of 128 bytes in the
// 128-byte swizzle: read as rows of q that is the K-major operand of X X^T, and read as rows of 64 q per p it is the
// MN-major operand of B X, so it is never transposed.  S and B share one place: both S and X are only overwritten, element by
// element by the thread that read them, after the product that uses them.  Scales and pairs of halves as in newton_schulz.cu
// (at most 48 additions per sum here, so no partial sums).
//
// A product takes about half a microsecond of its 128-cycle instructions, waits and the epilogue's pass, against six for a launch
// of its own.
#include "newton_schulz.cuh"
#include "tcgen05.cuh"

namespace blb200 {
namespace {

enum SmallWait { kSmallWait = 651 };
constexpr int kThreads = 512, kParts = kThreads / 128;  // warps per quarter of the rows

template <int PLANES, int QB>
struct SmallMemory {
  static constexpr int kX = QB * 128 * 128, kS = 2 * 128 * 128;  // bytes of one plane
  static constexpr size_t kBytes = 1024 + (size_t)PLANES * (kX + kS);
  static constexpr int kColumns = QB * 64 < 128 ? 128 : QB * 64;
};

// Byte offset of elements (row, 8 j .. 8 j + 7) of an operand.
__device__ __forceinline__ int chunk_at(int row, int j) { return (j >> 3) * 16384 + row * 128 + (((j & 7) ^ (row & 7)) << 4); }

template <typename T, int PLANES, int QB>
__global__ void __launch_bounds__(kThreads) newton_schulz_small_kernel(Matrices g, Matrices y, const __grid_constant__ Plan plan) {
  using M = SmallMemory<PLANES, QB>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* x = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  unsigned char* sb = x + PLANES * M::kX;
  __shared__ uint64_t ready;
  __shared__ uint32_t tmem_slot;
  __shared__ StepScales own[kMaxSteps];
  __shared__ float2 factors[3 * kMaxSteps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(&ready, 1);
    mbar_fence_init();
  }
  if (warp == 0) {
    tmem_alloc<1>(&tmem_slot, M::kColumns);
    tc_fence_before();
  }
  griddep_wait();
  griddep_launch();

  // the norm of G, then G times its power of two into X; columns of the caller's matrix by warps, rows by lanes
  const long long item = blockIdx.x;
  const T* src = (const T*)g.p + item * g.stride;
  double sum = 0;
  for (int j = warp; j < g.cols; j += kThreads / 32)
#pragma unroll 4
    for (int i = lane; i < g.rows; i += 32) {
      const double v = (double)to_f32(src[(long long)j * g.ld + i]);
      sum = fma(v, v, sum);
    }
  const ItemScale scale(block_sum(sum), plan.eps);
  write_factors(plan, scale.norm, scale.f, scale.e, own, factors, 1);
  const bool wide = g.rows <= g.cols;  // rows are the index p
  for (int j = warp; j < (wide ? QB * 64 : 128); j += kThreads / 32)
#pragma unroll 2
    for (int i = lane; i < (wide ? 128 : QB * 64); i += 32) {
      const float v = i < g.rows && j < g.cols ? to_f32(src[(long long)j * g.ld + i]) * scale.t1 * scale.t2 : 0.f;
      const int row = wide ? i : j, col = wide ? j : i;
      __half* at = reinterpret_cast<__half*>(x + chunk_at(row, col >> 3)) + (col & 7);
      const __half hi = __float2half_rn(v);
      at[0] = hi;
      if constexpr (PLANES == 2) at[M::kX / 2] = __float2half_rn(v - __half2float(hi));
    }
  fence_async_smem();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;

  uint32_t phase = 0;
  // One product by thread 0: A from `a` (K-major), B from `b`, K = 16 k_steps; all threads return when it is done.
  auto product = [&](const unsigned char* a, int plane_a, const unsigned char* b, int plane_b, bool b_mn, int k_steps, int n) {
    if (threadIdx.x == 0) {
      const uint32_t idesc = umma_idesc(false, false, b_mn, 128, n);
      const uint32_t lead = b_mn ? 16384 : 16;
#pragma unroll 4
      for (int k = 0; k < k_steps; ++k) {
        const uint32_t step = (k >> 2) * 16384 + (k & 3) * 32, step_b = b_mn ? k * 2048 : step;
        const uint64_t da = umma_desc(smem_u32(a) + step, 16, 1024), db = umma_desc(smem_u32(b) + step_b, lead, 1024);
        umma<1, false>(tmem, da, db, idesc, k > 0);
        if constexpr (PLANES == 2) {
          umma<1, false>(tmem, da, umma_desc(smem_u32(b) + plane_b + step_b, lead, 1024), idesc, true);
          umma<1, false>(tmem, umma_desc(smem_u32(a) + plane_a + step, 16, 1024), db, idesc, true);
        }
      }
      umma_commit<1>(&ready);
    }
    __syncwarp();
    const bool done = mbar_wait(&ready, phase & 1, kSmallWait);
    ++phase;
    tc_fence_after();
    return __syncthreads_and(done) != 0;
  };
  // Each thread takes one row of the tile and a quarter of its columns, sixteen at a time: out = alpha * product + beta * old, old
  // and out at the same place of `at`.
  const int quarter = warp & 3, part = warp >> 2, row = quarter * 32 + lane;
  const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
  auto sixteen = [&](unsigned char* at, int plane, int c, float2 f, bool has_old, float (&r)[16]) {
    uint32_t v[16];
    tmem_ld(v, lanes + c);
    tmem_wait_ld();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint4 was = make_uint4(0, 0, 0, 0), low = make_uint4(0, 0, 0, 0);
      if (has_old) {
        was = *reinterpret_cast<const uint4*>(at + chunk_at(row, (c >> 3) + h));
        if constexpr (PLANES == 2) low = *reinterpret_cast<const uint4*>(at + plane + chunk_at(row, (c >> 3) + h));
      }
      const uint32_t w[4] = {was.x, was.y, was.z, was.w}, l[4] = {low.x, low.y, low.z, low.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        r[8 * h + i] = f.x * __uint_as_float(v[8 * h + i]);
        if (has_old) {
          float old = __half2float(half_of(w[i / 2], i & 1));
          if constexpr (PLANES == 2) old += __half2float(half_of(l[i / 2], i & 1));
          r[8 * h + i] = fmaf(f.y, old, r[8 * h + i]);
        }
      }
    }
  };
  auto epilogue = [&](unsigned char* at, int plane, int columns, float2 f, bool has_old) {
#pragma unroll 1
    for (int c = part * (columns / kParts); c < (part + 1) * (columns / kParts); c += 16) {
      float r[16];
      sixteen(at, plane, c, f, has_old, r);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float r0 = r[8 * h + 2 * i], r1 = r[8 * h + 2 * i + 1];
          const __half h0 = __float2half_rn(r0), h1 = __float2half_rn(r1);
          hi[i] = pack_halves(h0, h1);
          if constexpr (PLANES == 2) lo[i] = pack_halves(__float2half_rn(r0 - __half2float(h0)), __float2half_rn(r1 - __half2float(h1)));
        }
        *reinterpret_cast<uint4*>(at + chunk_at(row, (c >> 3) + h)) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        if constexpr (PLANES == 2) *reinterpret_cast<uint4*>(at + plane + chunk_at(row, (c >> 3) + h)) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      }
    }
    tc_fence_before();
    fence_async_smem();
    __syncthreads();
    tc_fence_after();
  };

  bool ok = true;
#pragma unroll 1
  for (int i = 0; i < plan.steps && ok; ++i) {
    const float2* f = factors + 3 * i;
    ok = product(x, M::kX, x, M::kX, false, QB * 4, 128);
    if (!ok) break;
    epilogue(sb, M::kS, 128, f[0], false);
    ok = product(sb, M::kS, sb, M::kS, false, 8, 128);
    if (!ok) break;
    epilogue(sb, M::kS, 128, f[1], true);
    ok = product(sb, M::kS, x, M::kX, true, 8, QB * 64);
    if (!ok) break;
    if (i + 1 < plan.steps) {
      epilogue(x, M::kX, QB * 64, f[2], true);
    } else {
      T* out = (T*)y.p + item * y.stride;
      const int p = wide ? y.rows : y.cols, q = wide ? y.cols : y.rows;
      const long long to_row = wide ? 1 : y.ld, to_col = wide ? y.ld : 1;
#pragma unroll 1
      for (int c = part * (QB * 64 / kParts); c < (part + 1) * (QB * 64 / kParts) && c < q; c += 16) {
        float r[16];
        sixteen(x, M::kX, c, f[2], true, r);
        if (row < p) {
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (c + e < q) out[row * to_row + (c + e) * to_col] = from_f32<T>(r[e]);
        }
      }
      tc_fence_before();
    }
  }
  if (!ok) {  // a lost completion: leave time for what the tensor cores may still be reading
    for (int i = 0; i < 2000; ++i) __nanosleep(1000);
  }
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_free<1>(tmem, M::kColumns);
  }
}

template <typename T, int PLANES, int QB>
int launch_small(const Matrices& g, const Matrices& y, const Plan& plan, cudaStream_t stream) {
  auto kern = newton_schulz_small_kernel<T, PLANES, QB>;
  using M = SmallMemory<PLANES, QB>;
  static thread_local int configured_for = -1;
  int cur = 0;
  cudaGetDevice(&cur);
  if (configured_for != cur) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)M::kBytes);
    if (e != cudaSuccess) return (int)e;
    configured_for = cur;
  }
  OverlappedLaunch launch(dim3((unsigned)g.batch), dim3(kThreads), stream);
  launch.cfg.dynamicSmemBytes = M::kBytes;
  const int e = (int)cudaLaunchKernelEx(&launch.cfg, kern, g, y, plan);
  if (e == 0) note_launch("newton_schulz_small");
  return e;
}

}  // namespace

bool newton_schulz_small_supported(int rows, int cols) {
  const int p = rows < cols ? rows : cols, q = rows < cols ? cols : rows;
  return p <= 128 && q <= 256;
}

int launch_newton_schulz_small(const Matrices& g, const Matrices& y, int ftype, const Plan& plan, cudaStream_t stream) {
  const bool narrow = g.rows <= 128 && g.cols <= 128;
  if (ftype == BLB200_F32) return narrow ? launch_small<float, 2, 2>(g, y, plan, stream) : launch_small<float, 2, 4>(g, y, plan, stream);
  if (ftype == BLB200_F16) return narrow ? launch_small<__half, 2, 2>(g, y, plan, stream) : launch_small<__half, 2, 4>(g, y, plan, stream);
  return narrow ? launch_small<__nv_bfloat16, 1, 2>(g, y, plan, stream) : launch_small<__nv_bfloat16, 1, 4>(g, y, plan, stream);
}

int newton_schulz_small_device_status(int* out) { return read_device_status_word(out); }
int newton_schulz_small_device_status_clear() { return clear_device_status_word(); }

}  // namespace blb200
