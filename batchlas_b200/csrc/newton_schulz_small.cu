// The Newton-Schulz iteration on matrices with a short side: one CTA per matrix, or a cluster of up to eight CTAs that share the
// long side, everything but G and the result in shared memory.
//
// Per step  S = X X^T,  B = b S + c S^2,  X <- a X + B X  are three tcgen05 products of one 128-row tile, issued by one thread,
// each followed by an epilogue of all sixteen warps that scales the accumulator in tensor memory and writes the next operand.
// X (p x q, p the shorter side, padded with zeros to 128 x 64 QB) lies as blocks of 64 columns of 128 rows of 128 bytes in the
// 128-byte swizzle: read as rows of q that is the K-major operand of X X^T, and read as rows of 64 q per p it is the
// MN-major operand of B X, so it is never transposed.  S and B share one place: both S and X are only overwritten, element by
// element by the thread that read them, after the product that uses them.  Scales and pairs of halves as in newton_schulz.cu
// (at most 16 additions to a sum of full size here, so no partial sums).  Where the caller asks for single halves, B stays a
// pair: with few rows its rounding weighs most (six steps on 128 x 128: 2.1e-3 of the result in all instead of 2.5e-3, for 34 us instead of 30).
//
// In a cluster each CTA holds 64 QB columns of X.  X X^T is then a sum over the CTAs: each sends the rows of its part to the CTA that
// owns them (128 / CL rows each), which adds them up in rank order and writes its rows of S to every CTA; the rest of a step
// is done by each CTA for itself.  The parts arrive where S and B lie, so a cluster barrier stands before and after each
// exchange.  A wait that runs out lets the CTA go through the remaining barriers without products.
//
// Bound by latency: a product, its completion, the epilogue's pass over tensor and shared memory and two barriers of the CTA take
// about 3.3 us as pairs (10 us for a step of 128 x 128, 13 with 256 columns, 20 with a cluster's exchange) and 2.3 in single
// halves: 64 of 128 x 128 take 53 us (35 in single halves, where they took 98 as products over all items), 14 of 128 x 2048
// 117 us (78); fifteen as products 175 (122).
#include "newton_schulz.cuh"
#include "tcgen05.cuh"

namespace blb200 {
namespace {

enum SmallWait { kSmallWait = 651 };
constexpr int kThreads = 512, kParts = kThreads / 128;  // warps per quarter of the rows

template <int PLANES, int QB, int CL>
struct SmallMemory {
  static constexpr int kX = QB * 128 * 128, kS = 2 * 128 * 128;  // bytes of one plane
  static constexpr int kShared = 2 * kS;  // S and then B, which has two planes always, or the parts of 128 x 128 float sums
  static_assert(kShared == 128 * 128 * 4, "");
  static constexpr size_t kBytes = 1024 + (size_t)PLANES * kX + kShared;
  static constexpr int kColumns = QB * 64 < 128 ? 128 : QB * 64;
};

// Byte offset of elements (row, 8 j .. 8 j + 7) of an operand.
__device__ __forceinline__ int chunk_at(int row, int j) { return (j >> 3) * 16384 + row * 128 + (((j & 7) ^ (row & 7)) << 4); }

template <typename T, int PLANES, int QB, int CL>
__global__ void __launch_bounds__(kThreads, PLANES == 1 && QB == 2 ? 2 : 1) newton_schulz_small_kernel(Matrices g, Matrices y, const __grid_constant__ Plan plan) {
  using M = SmallMemory<PLANES, QB, CL>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* x = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  unsigned char* sb = x + PLANES * M::kX;
  __shared__ uint64_t ready;
  __shared__ uint32_t tmem_slot;
  __shared__ StepScales own[kMaxSteps];
  __shared__ float2 factors[3 * kMaxSteps];
  __shared__ double squares[CL];
  const uint32_t cta = CL > 1 ? cluster_rank() : 0;
  const int q0 = (int)cta * QB * 64;  // first of this CTA's columns of X
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
  if constexpr (CL > 1) {  // no CTA's shared memory is written before it has started
    __syncwarp();
    cluster_sync();
  }

  // the norm of G, then G times its power of two into X
  const long long item = blockIdx.x / CL;
  const T* src = (const T*)g.p + item * g.stride;
  const bool wide = g.rows <= g.cols;  // rows are the index p
  const int i0 = wide ? 0 : q0, j0 = wide ? q0 : 0;  // this CTA's part of the caller's matrix
  const int i1 = wide ? g.rows : min(g.rows, q0 + QB * 64), j1 = wide ? min(g.cols, q0 + QB * 64) : g.cols;
  // Its units of V elements (16 bytes where the layout allows it, else one), four per thread in flight.
  constexpr int V = 16 / (int)sizeof(T);
  const bool whole = (i1 - i0) % V == 0 && reinterpret_cast<uintptr_t>(src + i0) % 16 == 0 && g.ld % V == 0;
  auto for_each = [&](auto body) {
    const int size = whole ? V : 1, units = max(0, i1 - i0) / size, total = units * max(0, j1 - j0);
    for (int first = threadIdx.x; first < total; first += 4 * kThreads) {
      __align__(16) T v[4][V];
      int i[4], j[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int at = first + u * kThreads;
        j[u] = at / units;
        i[u] = (at - j[u] * units) * size;
        if (at >= total) j[u] = -1;
        if (at < total) {
          const T* from = src + (long long)(j0 + j[u]) * g.ld + i0 + i[u];
          if (whole) *reinterpret_cast<uint4*>(v[u]) = *reinterpret_cast<const uint4*>(from);
          else v[u][0] = *from;
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (j[u] >= 0) {
#pragma unroll
          for (int e = 0; e < V; ++e)
            if (e == 0 || whole) body(i[u] + e, j[u], to_f32(v[u][e]));
        }
    }
  };
  for (int c = threadIdx.x; c < PLANES * M::kX / 16; c += kThreads) reinterpret_cast<uint4*>(x)[c] = make_uint4(0, 0, 0, 0);
  double sum = 0;
  for_each([&](int, int, float value) {
    const double v = (double)value;
    sum = fma(v, v, sum);
  });
  sum = block_sum(sum);
  if constexpr (CL > 1) {
    if (threadIdx.x < CL) {
      const uint32_t to = cluster_addr(smem_u32(&squares[cta]), threadIdx.x);
      asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(to), "d"(sum) : "memory");
    }
    __syncwarp();
    cluster_sync();
    sum = 0;
    for (int i = 0; i < CL; ++i) sum += squares[i];
  }
  const ItemScale scale(sum, plan.eps);
  write_factors(plan, scale.norm, scale.f, scale.e, own, factors, 1);
  for_each([&](int i, int j, float value) {
    const float v = value * scale.t1 * scale.t2;
    const int row = wide ? i : j, col = wide ? j : i;
    __half* at = reinterpret_cast<__half*>(x + chunk_at(row, col >> 3)) + (col & 7);
    const __half hi = __float2half_rn(v);
    at[0] = hi;
    if constexpr (PLANES == 2) at[M::kX / 2] = __float2half_rn(v - __half2float(hi));
  });
  fence_async_smem();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;

  uint32_t phase = 0;
  bool ok = true;
  // One product by thread 0: A from `a` (K-major), B from `b`, K = 16 k_steps, N = n (a multiple of 256 as several instructions); all
  // threads return when it is done.
  auto product = [&](const unsigned char* a, int plane_a, const unsigned char* b, int plane_b, bool b_mn, int k_steps, int n_all, bool a_low) {
    if (!ok) return;
    const int n = min(n_all, 256);
    for (int n0 = 0; n0 < n_all && threadIdx.x == 0; n0 += n, b += 4 * 16384) {
      const uint32_t d = tmem + n0;
      const uint32_t idesc = umma_idesc(false, false, b_mn, 128, n);
      const uint32_t lead = b_mn ? 16384 : 16;
      auto at = [&](const unsigned char* p, int k, bool mn) {
        return umma_desc(smem_u32(p) + (mn ? k * 2048 : (k >> 2) * 16384 + (k & 3) * 32), mn ? lead : 16, 1024);
      };
      // the small products first: an addition drops what lies below the last place of the sum that it adds to
      if constexpr (PLANES == 2) {
#pragma unroll 4
        for (int k = 0; k < k_steps; ++k) {
          umma<1, false>(d, at(a, k, false), at(b + plane_b, k, b_mn), idesc, k > 0);
          umma<1, false>(d, at(a + plane_a, k, false), at(b, k, b_mn), idesc, true);
        }
      }
      if (PLANES == 1 && a_low) {
#pragma unroll 4
        for (int k = 0; k < k_steps; ++k) umma<1, false>(d, at(a + plane_a, k, false), at(b, k, b_mn), idesc, k > 0);
      }
#pragma unroll 4
      for (int k = 0; k < k_steps; ++k) umma<1, false>(d, at(a, k, false), at(b, k, b_mn), idesc, PLANES == 2 || a_low || k > 0);
    }
    if (threadIdx.x == 0) umma_commit<1>(&ready);
    __syncwarp();
    const bool done = mbar_wait(&ready, phase & 1, kSmallWait);
    ++phase;
    tc_fence_after();
    ok = __syncthreads_and(done) != 0;
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
  auto epilogue = [&](unsigned char* at, int plane, int columns, float2 f, bool has_old, bool low) {
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
          lo[i] = pack_halves(__float2half_rn(r0 - __half2float(h0)), __float2half_rn(r1 - __half2float(h1)));
        }
        *reinterpret_cast<uint4*>(at + chunk_at(row, (c >> 3) + h)) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        if (PLANES == 2 || low) *reinterpret_cast<uint4*>(at + plane + chunk_at(row, (c >> 3) + h)) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      }
    }
    tc_fence_before();
    fence_async_smem();
    __syncthreads();
    tc_fence_after();
  };

  // The cluster's S: parts of the sums to their owners, rows of S back to everyone.
  auto share_gram = [&](float alpha) {
    constexpr int R = 128 / CL, kTasks = R * 16 / kThreads < 1 ? 1 : R * 16 / kThreads;
    cluster_sync();  // every CTA is past the product that read B
#pragma unroll 1
    for (int c = part * 32; c < part * 32 + 32; c += 16) {
      uint32_t v[16];
      tmem_ld(v, lanes + c);
      tmem_wait_ld();
      const uint32_t to = cluster_addr(smem_u32(sb), row / R) + ((cta * 128 + c) * R + row % R) * 4;
#pragma unroll
      for (int i = 0; i < 16; ++i) asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(to + i * R * 4), "r"(v[i]) : "memory");
    }
    tc_fence_before();
    cluster_sync();
    const float* parts = reinterpret_cast<const float*>(sb);
    uint32_t hi[kTasks][4], lo[kTasks][4];
#pragma unroll
    for (int t = 0; t < kTasks; ++t) {
      const int task = threadIdx.x + t * kThreads, r = task % R, chunk = task / R;  // eight columns of one row
      float s[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        s[i] = 0.f;
        if (chunk < 16) {
#pragma unroll
          for (int from = 0; from < CL; ++from) s[i] += parts[(from * 128 + chunk * 8 + i) * R + r];
        }
        s[i] *= alpha;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const __half h0 = __float2half_rn(s[2 * i]), h1 = __float2half_rn(s[2 * i + 1]);
        hi[t][i] = pack_halves(h0, h1);
        lo[t][i] = pack_halves(__float2half_rn(s[2 * i] - __half2float(h0)), __float2half_rn(s[2 * i + 1] - __half2float(h1)));
      }
    }
    cluster_sync();  // the parts are read: S takes their place
#pragma unroll
    for (int t = 0; t < kTasks; ++t) {
      const int task = threadIdx.x + t * kThreads, r = task % R, chunk = task / R;
      if (chunk < 16) {
#pragma unroll
        for (int peer = 0; peer < CL; ++peer) {
          const uint32_t to = cluster_addr(smem_u32(sb), peer) + chunk_at((int)cta * R + r, chunk);
          asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(hi[t][0]), "r"(hi[t][1]), "r"(hi[t][2]), "r"(hi[t][3])
                       : "memory");
          if constexpr (PLANES == 2)
            asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to + M::kS), "r"(lo[t][0]), "r"(lo[t][1]), "r"(lo[t][2]),
                         "r"(lo[t][3])
                         : "memory");
        }
      }
    }
    asm volatile("fence.proxy.async;" ::: "memory");
    __syncwarp();
    cluster_sync();
    asm volatile("fence.proxy.async;" ::: "memory");
    tc_fence_after();
  };

#pragma unroll 1
  for (int i = 0; i < plan.steps; ++i) {
    const float2* f = factors + 3 * i;
    product(x, M::kX, x, M::kX, false, QB * 4, 128, false);
    if constexpr (CL > 1) share_gram(f[0].x);
    else epilogue(sb, M::kS, 128, f[0], false, false);
    product(sb, M::kS, sb, M::kS, false, 8, 128, false);
    epilogue(sb, M::kS, 128, f[1], true, true);
    product(sb, M::kS, x, M::kX, true, 8, QB * 64, true);
    if (i + 1 < plan.steps) {
      epilogue(x, M::kX, QB * 64, f[2], true, false);
    } else {
      T* out = (T*)y.p + item * y.stride;
      const int p = wide ? y.rows : y.cols, q = wide ? y.cols : y.rows;
#pragma unroll 1
      for (int c = part * (QB * 64 / kParts); c < (part + 1) * (QB * 64 / kParts) && q0 + c < q; c += 16) {
        float r[16];
        sixteen(x, M::kX, c, f[2], true, r);
        if (wide) {  // a warp's rows lie side by side in memory
          if (row < p && ok) {
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (q0 + c + e < q) out[row + (long long)(q0 + c + e) * y.ld] = from_f32<T>(r[e]);
          }
        } else {  // the columns do: the values' bits take X's place (a float's two halves its two planes)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const T v0 = from_f32<T>(r[8 * h + 2 * e]), v1 = from_f32<T>(r[8 * h + 2 * e + 1]);
              if constexpr (sizeof(T) == 4) {
                hi[e] = __byte_perm(__float_as_uint(v0), __float_as_uint(v1), 0x7632);
                lo[e] = __byte_perm(__float_as_uint(v0), __float_as_uint(v1), 0x5410);
              } else {
                hi[e] = (uint32_t)*reinterpret_cast<const unsigned short*>(&v0) | (uint32_t)*reinterpret_cast<const unsigned short*>(&v1) << 16;
              }
            }
            *reinterpret_cast<uint4*>(x + chunk_at(row, (c >> 3) + h)) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(x + M::kX + chunk_at(row, (c >> 3) + h)) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
          }
        }
      }
      tc_fence_before();
      __syncthreads();
      if (!wide && ok) {
        const int mine = min(QB * 64, q - q0);
        for (int j = warp; j < p; j += kThreads / 32)
#pragma unroll 4
          for (int i = lane; i < mine; i += 32) {
            const unsigned short* at = reinterpret_cast<const unsigned short*>(x + chunk_at(j, i >> 3)) + (i & 7);
            T v;
            if constexpr (sizeof(T) == 4) v = __uint_as_float((uint32_t)at[0] << 16 | at[M::kX / 2]);
            else v = *reinterpret_cast<const T*>(at);
            out[(long long)j * y.ld + q0 + i] = v;
          }
      }
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

template <typename T, int PLANES, int QB, int CL>
int launch_small(const Matrices& g, const Matrices& y, const Plan& plan, cudaStream_t stream) {
  auto kern = newton_schulz_small_kernel<T, PLANES, QB, CL>;
  using M = SmallMemory<PLANES, QB, CL>;
  static thread_local int configured_for = -1;
  int cur = 0;
  cudaGetDevice(&cur);
  if (configured_for != cur) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)M::kBytes);
    if (e != cudaSuccess) return (int)e;
    configured_for = cur;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(g.batch * CL));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = M::kBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = CL;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CL > 1 ? 2 : 1;
  const int e = (int)cudaLaunchKernelEx(&cfg, kern, g, y, plan);
  if (e == 0) note_launch("newton_schulz_small");
  return e;
}

template <typename T, int PLANES>
int launch_by_size(const Matrices& g, const Matrices& y, const Plan& plan, cudaStream_t stream) {
  const int q = g.rows < g.cols ? g.cols : g.rows;
  if (q <= 128) return launch_small<T, PLANES, 2, 1>(g, y, plan, stream);
  if (q <= 256) return launch_small<T, PLANES, 4, 1>(g, y, plan, stream);
  if (q <= 512) return launch_small<T, PLANES, 4, 2>(g, y, plan, stream);
  if (q <= 1024) return launch_small<T, PLANES, 4, 4>(g, y, plan, stream);
  if (q <= 2048) return launch_small<T, PLANES, 4, 8>(g, y, plan, stream);
  if constexpr (PLANES == 1) return launch_small<T, 1, 8, 8>(g, y, plan, stream);
  return BLB200_E_INTERNAL;
}

}  // namespace

// The shorter side in one tile and the longer one in the shared memory of a cluster.  Batches whose clusters do not all run at
// once (about 14 of eight CTAs do, one CTA per SM) are as fast or faster as products over all items: 14 matrices of 128 x 4096 in
// single halves take 101 us here, and fifteen 165 as products, where two rounds here take 173.  The 112 CTAs are a constant, not
// asked of the device, because the size of the scratch follows from this and must not depend on the device that is current.
bool newton_schulz_small_supported(int rows, int cols, int batch, int planes) {
  const int p = rows < cols ? rows : cols, q = rows < cols ? cols : rows;
  if (p > 128 || q > (planes == 1 ? 4096 : 2048)) return false;
  const int ctas = q <= 256 ? 1 : q <= 512 ? 2 : q <= 1024 ? 4 : 8;
  return ctas == 1 || (long long)batch * ctas <= 112;
}

int launch_newton_schulz_small(const Matrices& g, const Matrices& y, int ftype, int planes, const Plan& plan, cudaStream_t stream) {
  if (ftype == BLB200_F32) return launch_by_size<float, 2>(g, y, plan, stream);
  if (ftype == BLB200_F16) return launch_by_size<__half, 2>(g, y, plan, stream);
  return planes == 1 ? launch_by_size<__nv_bfloat16, 1>(g, y, plan, stream) : launch_by_size<__nv_bfloat16, 2>(g, y, plan, stream);
}

int newton_schulz_small_device_status(int* out) { return read_device_status_word(out); }
int newton_schulz_small_device_status_clear() { return clear_device_status_word(); }

}  // namespace blb200
