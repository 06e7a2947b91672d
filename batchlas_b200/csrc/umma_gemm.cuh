// The product core of the 8-bit gemm and of the Newton-Schulz iteration: D (M x N) = A (M x K) * B (K x N) per batch item on the
// tcgen05 tensor cores, D handed to an epilogue in registers.
//
// One CTA (or a pair sharing one 256-row tile, cta_group::2) is persistent and walks over output tiles.  Three roles
// run side by side: warp 0 fetches operand tiles by tensor-map copies into a ring of stages, one lane of warp 1 issues the
// MMAs, and eight warps carry finished tiles out of tensor memory, which holds two accumulators, so that a tile's
// epilogue overlaps the next tile's products.  In a pair each CTA holds its own 128 rows of A and half of the
// columns of B; the MMAs of both are issued by the first CTA, which also owns the barriers that say "stage full" and
// "accumulator free".
//
// Operands with K fastest are fetched as rows of 128 bytes (128 int8 or 64 half values of one M or N index); those with M or
// N fastest (half only) as blocks of 64 indices x 64 k.  Both lie in the 128-byte swizzle.  Edges are zero-filled by
// the map.  PLANES == 2: each operand is a pair hi + lo of half matrices (consecutive z slices of the map), and
// hi*hi + hi*lo + lo*hi is accumulated: a float product but for the lo*lo term (2^-24 of the product).  The tensor
// cores drop the bits below the accumulator's last one at every addition, which over a long k is a bias (k = 1501,
// three products: 9.5e-6 of the iteration's result against 3e-6 for plain float sums); so for pairs only two k blocks (24
// additions) are summed there, and the partial sums are added up in registers, rounded to nearest.
//
// A wait that runs out records its code, and the role leaves its loop; the other roles' waits then run out as well, the
// copies still in flight are waited for, tensor memory is freed and the kernel returns.
#pragma once

#include "common.cuh"
#include "tcgen05.cuh"

namespace blb200 {

struct UmmaShape {
  int m, n, k, batch;
  int tiles_m, tiles_n;
  long long tiles;       // all tiles of the launch
  long long a_items, b_items;  // 1 when the operand is shared by the batch
  int symmetric;         // D is symmetric (m == n): tiles below the diagonal only
};

enum UmmaWait { kUmmaWaitEmpty = 1, kUmmaWaitFull = 2, kUmmaWaitAccFree = 3, kUmmaWaitAcc = 4, kUmmaWaitDrain = 5 };

template <bool I8_, bool A_MN_, bool B_MN_, int GROUP_, int BN_, int PLANES_>
struct UmmaConfig {
  static constexpr bool I8 = I8_, A_MN = A_MN_, B_MN = B_MN_;
  static constexpr int GROUP = GROUP_, BN = BN_, PLANES = PLANES_;
  static constexpr int kBM = 128 * GROUP;              // rows of a tile
  static constexpr int kBRows = BN / GROUP;            // columns of B held by one CTA
  static_assert(kBM == BN || kBM == 2 * BN || I8, "symmetric results need whole tiles on the diagonal");
  static constexpr int kKStage = I8 ? 128 : 64;        // k per stage: 128 bytes
  static constexpr int kABytes = 128 * 128, kBBytes = kBRows * 128;
  static constexpr int kStageBytes = PLANES * (kABytes + kBBytes);
  static constexpr int kStages = (200 * 1024) / kStageBytes < 8 ? (200 * 1024) / kStageBytes : 8;
  static constexpr int kTmemColumns = 2 * BN < 32 ? 32 : 2 * BN;
  static constexpr int kThreads = 320;
  static constexpr int kChunk = PLANES == 2 ? 2 : 0;   // k blocks summed in tensor memory, 0 = all
  static constexpr int kRatio = kBM / BN;              // tile columns per tile row
  static constexpr size_t kSmem = 1024 + (size_t)kStages * kStageBytes + 256;
  static_assert(!I8 || (!A_MN && !B_MN && PLANES == 1), "8-bit operands are K-major");
  static_assert(kStages >= 2 && kTmemColumns <= 512 && (kTmemColumns & (kTmemColumns - 1)) == 0, "");
};

struct UmmaTile {
  int item, tm, tn;
};
// Tiles of one item in an order that keeps the operands of the tiles in flight together in L2: bands of eight tile
// rows, walked column by column; for a symmetric D the tiles that reach the diagonal or lie below it, row by row
// (tile row i has R (i + 1) of them, R columns of tiles being as wide as one row of tiles is high).
template <int R>
__host__ __device__ inline long long symmetric_tiles(int tiles_m, int tiles_n) {
  const long long full_rows = (long long)R * tiles_m * (tiles_m - 1) / 2, last = (long long)R * tiles_m;
  return full_rows + (last < tiles_n ? last : tiles_n);
}
template <int R>
__device__ __forceinline__ UmmaTile umma_tile(const UmmaShape& s, long long t) {
  UmmaTile r;
  if (s.symmetric) {
    const long long per = symmetric_tiles<R>(s.tiles_m, s.tiles_n);
    r.item = (int)(t / per);
    const int f = (int)(t - (long long)r.item * per);
    int i = (int)((sqrtf((8.f / R) * (float)f + 1.f) - 1.f) * 0.5f);
    while ((long long)R * (i + 1) * (i + 2) / 2 <= f) ++i;
    while ((long long)R * i * (i + 1) / 2 > f) --i;
    r.tm = i;
    r.tn = f - (int)((long long)R * i * (i + 1) / 2);
    return r;
  }
  const long long per = (long long)s.tiles_m * s.tiles_n;
  r.item = (int)(t / per);
  const int f = (int)(t - (long long)r.item * per);
  constexpr int kBand = 8;
  const int band = f / (kBand * s.tiles_n), first = band * kBand;
  const int height = min(kBand, s.tiles_m - first);
  const int rest = f - band * kBand * s.tiles_n;
  r.tn = rest / height;
  r.tm = first + rest - r.tn * height;
  return r;
}

template <class C, class Epilogue>
__global__ void __launch_bounds__(C::kThreads, 1)
    umma_gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const UmmaShape s,
                     const typename Epilogue::Params ep, int wait_code) {
  constexpr int S = C::kStages, G = C::GROUP;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + (size_t)S * C::kStageBytes);
  uint64_t* empty = full + S;
  uint64_t* acc_full = empty + S;
  uint64_t* acc_free = acc_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_free + 2);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = G == 2 ? cluster_rank() : 0;
  const long long first = (long long)blockIdx.x / G, step = gridDim.x / G;
  const int k_blocks = (s.k + C::kKStage - 1) / C::kKStage;

  if (warp == 0 && lane == 0) {
    for (int i = 0; i < S; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_free[i], 8 * G);
    }
    mbar_fence_init();
  }
  if (warp == 1) {
    tmem_alloc<G>(tmem_slot, C::kTmemColumns);
    tc_fence_before();
  }
  __syncthreads();
  if constexpr (G == 2) cluster_sync();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // Everything above may overlap the end of the kernel before this one; its results are read from here on.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  if (warp == 0) {
    if (lane == 0) {
      bool ok = true;
      uint32_t round = 0;
      int slot = 0;
      for (long long t = first; t < s.tiles && ok; t += step) {
        const UmmaTile tile = umma_tile<C::kRatio>(s, t);
        const int za = (s.a_items == 1 ? 0 : tile.item) * C::PLANES, zb = (s.b_items == 1 ? 0 : tile.item) * C::PLANES;
        const int m0 = tile.tm * C::kBM + (int)rank * 128, n0 = tile.tn * C::BN + (int)rank * C::kBRows;
        for (int kb = 0; kb < k_blocks && ok; ++kb) {
          ok = G == 1 ? mbar_wait(&empty[slot], (round & 1) ^ 1, wait_code + kUmmaWaitEmpty)
                      : mbar_wait_cluster(&empty[slot], (round & 1) ^ 1, wait_code + kUmmaWaitEmpty);
          if (!ok) break;
          if (rank == 0) mbar_arrive_expect_tx(&full[slot], G * C::kStageBytes);
          const uint32_t bar = G == 2 ? cluster_addr(smem_u32(&full[slot]), 0) : smem_u32(&full[slot]);
          unsigned char* stage = smem + (size_t)slot * C::kStageBytes;
          auto load = [&](unsigned char* dst, const CUtensorMap* map, int x, int y, int z) {
            if constexpr (G == 2) tma_load_3d_pair(smem_u32(dst), map, x, y, z, bar);
            else tma_load_3d(dst, map, x, y, z, &full[slot]);
          };
          const int k0 = kb * C::kKStage;
#pragma unroll
          for (int pl = 0; pl < C::PLANES; ++pl) {
            unsigned char* a = stage + pl * C::kABytes;
            unsigned char* b = stage + C::PLANES * C::kABytes + pl * C::kBBytes;
            if constexpr (C::A_MN) {
#pragma unroll
              for (int i = 0; i < 2; ++i) load(a + i * 8192, &map_a, m0 + i * 64, k0, za + pl);
            } else {
              load(a, &map_a, k0, m0, za + pl);
            }
            if constexpr (C::B_MN) {
#pragma unroll
              for (int i = 0; i < C::kBRows / 64; ++i) load(b + i * 8192, &map_b, n0 + i * 64, k0, zb + pl);
            } else {
              load(b, &map_b, k0, n0, zb + pl);
            }
          }
          if (++slot == S) {
            slot = 0;
            ++round;
          }
        }
      }
      // No CTA leaves while MMA completions may still be signalled to its barriers.
      for (int i = 0; i < S && ok; ++i) {
        ok = G == 1 ? mbar_wait(&empty[slot], (round & 1) ^ 1, wait_code + kUmmaWaitEmpty)
                    : mbar_wait_cluster(&empty[slot], (round & 1) ^ 1, wait_code + kUmmaWaitEmpty);
        if (ok && ++slot == S) {
          slot = 0;
          ++round;
        }
      }
      if (!ok) {
        // what was sent for and not seen to arrive: the last S stages
        if (rank == 0) {
          for (int i = 0; i < S; ++i) {
            const int at = (slot + i) % S;
            const uint32_t r = at >= slot ? round - 1 : round;  // the stage's last round that was sent for
            if (at >= slot && round == 0) continue;
            mbar_wait_limit(&full[at], r & 1, wait_code + kUmmaWaitDrain, 1u << 12);
          }
        }
        for (int i = 0; i < 2000; ++i) __nanosleep(1000);
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      constexpr uint32_t idesc = umma_idesc(C::I8, C::A_MN, C::B_MN, C::kBM, C::BN);
      bool ok = true;
      uint32_t round = 0;
      int slot = 0;
      long long done = 0;
      for (long long t = first; t < s.tiles && ok; t += step) {
        uint32_t d = 0;
        for (int kb = 0; kb < k_blocks; ++kb) {
          const bool begins = C::kChunk ? kb % (C::kChunk ? C::kChunk : 1) == 0 : kb == 0;
          if (begins) {
            const int acc = (int)(done & 1);
            ok = G == 1 ? mbar_wait(&acc_free[acc], (uint32_t)((done >> 1) & 1) ^ 1, wait_code + kUmmaWaitAccFree)
                        : mbar_wait_cluster(&acc_free[acc], (uint32_t)((done >> 1) & 1) ^ 1, wait_code + kUmmaWaitAccFree);
            if (!ok) break;
            d = tmem + acc * C::BN;
          }
          ok = G == 1 ? mbar_wait(&full[slot], round & 1, wait_code + kUmmaWaitFull)
                      : mbar_wait_cluster(&full[slot], round & 1, wait_code + kUmmaWaitFull);
          if (!ok) break;
          tc_fence_after();
          const uint32_t a = smem_u32(smem + (size_t)slot * C::kStageBytes), b = a + C::PLANES * C::kABytes;
          // 32 bytes of k per instruction: 32 bytes along a K-major row, 16 rows of 128 bytes of an MN-major block
          constexpr uint32_t kAStep = C::A_MN ? 2048 : 32, kBStep = C::B_MN ? 2048 : 32;
          constexpr uint32_t kALead = C::A_MN ? 8192 : 16, kBLead = C::B_MN ? 8192 : 16;
#pragma unroll
          for (int ks = 0; ks < 4; ++ks) {
            const uint64_t da = umma_desc(a + ks * kAStep, kALead, 1024), db = umma_desc(b + ks * kBStep, kBLead, 1024);
            umma<G, C::I8>(d, da, db, idesc, !begins || ks > 0);
            if constexpr (C::PLANES == 2) {
              const uint64_t da2 = umma_desc(a + C::kABytes + ks * kAStep, kALead, 1024);
              const uint64_t db2 = umma_desc(b + C::kBBytes + ks * kBStep, kBLead, 1024);
              umma<G, C::I8>(d, da, db2, idesc, true);
              umma<G, C::I8>(d, da2, db, idesc, true);
            }
          }
          umma_commit<G>(&empty[slot]);
          if (++slot == S) {
            slot = 0;
            ++round;
          }
          if (kb + 1 == k_blocks || (C::kChunk && (kb + 1) % (C::kChunk ? C::kChunk : 1) == 0)) {
            umma_commit<G>(&acc_full[done & 1]);
            ++done;
          }
        }
      }
    }
  } else {
    // Two warps per quarter of the 128 rows: each takes half of the columns (narrow tiles: the first takes all).
    constexpr int kSplit = C::BN >= 64 ? 2 : 1, kCols = C::BN / kSplit, kPiece = kCols < 32 ? 16 : 32;
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    const int row = quarter * 32 + lane;
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16) + half * kCols;
    long long done = 0;
    auto acquire = [&]() {
      const int acc = (int)(done & 1);
      const bool ok = G == 1 ? mbar_wait(&acc_full[acc], (uint32_t)((done >> 1) & 1), wait_code + kUmmaWaitAcc)
                             : mbar_wait_cluster(&acc_full[acc], (uint32_t)((done >> 1) & 1), wait_code + kUmmaWaitAcc);
      if (!__all_sync(0xffffffffu, ok)) return false;
      tc_fence_after();
      return true;
    };
    auto release = [&]() {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (G == 2) mbar_arrive_cluster(cluster_addr(smem_u32(&acc_free[done & 1]), 0));
        else mbar_arrive(&acc_free[done & 1]);
      }
      ++done;
    };
    bool ok = true;
    for (long long t = first; t < s.tiles && ok; t += step) {
      const UmmaTile tile = umma_tile<C::kRatio>(s, t);
      const int n0 = tile.tn * C::BN + half * kCols;
      Epilogue epi(ep, s, tile, s.symmetric && tile.tn < C::kRatio * tile.tm, tile.tm * C::kBM + (int)rank * 128 + row);
      if constexpr (C::kChunk == 0) {
        ok = acquire();
        if (!ok) break;
        if (half < kSplit) {
#pragma unroll 1
          for (int c = 0; c < kCols; c += kPiece) {
            if (n0 + c >= s.n) break;
            uint32_t v[kPiece];
            tmem_ld(v, lanes + (uint32_t)(done & 1) * C::BN + c);
            tmem_wait_ld();
            epi.store(v, n0 + c);
          }
        }
        release();
      } else {
        uint32_t v[kCols / kPiece][kPiece] = {};
        for (int kb = 0; kb < k_blocks; kb += C::kChunk) {
          ok = acquire();
          if (!ok) break;
#pragma unroll
          for (int c = 0; c < kCols / kPiece; ++c) {
            uint32_t w[kPiece];
            tmem_ld(w, lanes + (uint32_t)(done & 1) * C::BN + c * kPiece);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < kPiece; ++i)
              v[c][i] = __float_as_uint(__uint_as_float(v[c][i]) + __uint_as_float(w[i]));
          }
          release();
        }
        if (!ok) break;
#pragma unroll
        for (int c = 0; c < kCols / kPiece; ++c)
          if (n0 + c * kPiece < s.n) epi.store(v[c], n0 + c * kPiece);
      }
    }
  }
  __syncwarp();
  __syncthreads();
  if constexpr (G == 2) cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    tmem_free<G>(tmem, C::kTmemColumns);
  }
}

// ---- host side -----------------------------------------------------------------------------------
// 3-D map (inner, outer, z) over `base`: box of 128 bytes x box_outer rows x 1, 128-byte swizzle.  Strides in bytes.
inline int encode_operand(CUtensorMap* map, const void* base, bool i8, long long inner, long long outer, long long z, long long ld_bytes,
                          long long z_bytes, int box_outer) {
  EncodeTiledFn enc = encode_tiled_fn();
  if (!enc) return BLB200_E_INTERNAL;
  const cuuint64_t dims[3] = {(cuuint64_t)inner, (cuuint64_t)outer, (cuuint64_t)z};
  const cuuint64_t strides[2] = {(cuuint64_t)ld_bytes, (cuuint64_t)(z > 1 ? z_bytes : ld_bytes * outer)};
  const cuuint32_t box[3] = {i8 ? 128u : 64u, (cuuint32_t)box_outer, 1}, estr[3] = {1, 1, 1};
  const CUresult r = enc(map, i8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(base), dims, strides,
                         box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? BLB200_OK : BLB200_E_INTERNAL;
}

template <class C, class Epilogue>
int launch_umma(const CUtensorMap& map_a, const CUtensorMap& map_b, UmmaShape s, const typename Epilogue::Params& ep, int wait_code,
                cudaStream_t stream) {
  s.tiles_m = (s.m + C::kBM - 1) / C::kBM;
  s.tiles_n = (s.n + C::BN - 1) / C::BN;
  s.tiles = (s.symmetric ? symmetric_tiles<C::kRatio>(s.tiles_m, s.tiles_n) : (long long)s.tiles_m * s.tiles_n) * s.batch;
  auto kern = umma_gemm_kernel<C, Epilogue>;
  static thread_local int configured_for = -1;
  int cur = 0;
  cudaGetDevice(&cur);
  if (configured_for != cur) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::kSmem);
    if (e != cudaSuccess) return (int)e;
    configured_for = cur;
  }
  const long long units = device_info().sm_count / C::GROUP;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((s.tiles < units ? s.tiles : units) * C::GROUP));
  cfg.blockDim = dim3(C::kThreads);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = C::GROUP;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = C::GROUP == 2 ? 2 : 1;
  return (int)cudaLaunchKernelEx(&cfg, kern, map_a, map_b, s, ep, wait_code);
}

}  // namespace blb200
