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
// SPLIT > 1: a cluster of SPLIT CTAs shares one output tile, each taking a range of k; their sums are exchanged through
// distributed shared memory (the idle stages), each CTA adding up, in rank order, what it stores.  For calls whose
// tiles would leave most SMs without work.
// PLAIN: the operands are not on 16-byte boundaries, so the eight epilogue warps fetch the stages themselves, as aligned words
// shifted together and written where the swizzle puts them (777 x 4099 x 1003 with its quantisation 32 us; a row at a time, one word
// per lane and the neighbour's by a shuffle, measured 52).
//
// Measured: 8192^3 8-bit 380 us = 2.9 POP/s in a burst (within a full call about 440, at the clock the power limit leaves), where the MMAs alone, without fetches and stores, take 345 and the fetches alone 215;
// half precision, 4096 x 4096 x 16384, 411 us = 1.34 PFLOP/s under the power limit; pairs of halves, 8192 x 4096 x 4096, 726 us,
// 1.14 PFLOP/s of three MMAs per product.  The MMAs are what bounds large
// products; small ones are bounded by the 5 to 7 us between the start of one product and the start of the next that
// needs it (first fetch 1 to 2 us, k blocks 0.3 us each with six in flight, epilogue 1, storing and the next start 2).
//
// Epilogue: a thread owns one row of the tile (32 consecutive rows per warp) and takes its columns in groups of sixteen, in a
// rolled loop: unrolled over the tile the code is 10 KB and more, which a kernel of a few microseconds spends its time
// fetching (128 x 128 tiles: 2.3 us of 5.6).  A staged epilogue reads the old values of the result's tile from, and may leave the new
// ones in, a buffer that tensor-map copies fill while the products run and write out: row-wise, where the columns are the fast
// index in memory (sixteen values are two 16-byte accesses), or column by column.
//
// A wait that runs out records its code, and the role leaves its loop; the other roles' waits then run out as well, the
// copies still in flight are waited for, tensor memory is freed and the kernel returns.
#pragma once

#include <algorithm>

#include "common.cuh"
#include "tcgen05.cuh"

namespace blb200 {

struct UmmaShape {
  int m, n, k, batch;
  int tiles_m, tiles_n;
  int tiles;             // all tiles of the launch
  long long a_items, b_items;  // 1 when the operand is shared by the batch
  int symmetric;         // D is symmetric (m == n): tiles below the diagonal only
};

enum UmmaWait { kUmmaWaitEmpty = 1, kUmmaWaitFull = 2, kUmmaWaitAccFree = 3, kUmmaWaitAcc = 4, kUmmaWaitDrain = 5, kUmmaWaitStaging = 6, kUmmaWaitOld = 7 };
constexpr int kStagedColumns = 32;  // columns per box of a column-wise staging buffer

template <bool I8_, bool A_MN_, bool B_MN_, int GROUP_, int BN_, int PLANES_, int SPLIT_ = 1, bool PLAIN_ = false>
struct UmmaConfig {
  static constexpr int SPLIT = SPLIT_;
  static constexpr bool PLAIN = PLAIN_;
  static constexpr bool I8 = I8_, A_MN = A_MN_, B_MN = B_MN_;
  static constexpr int GROUP = GROUP_, BN = BN_, PLANES = PLANES_;
  static constexpr int kBM = 128 * GROUP;              // rows of a tile
  static constexpr int kBRows = BN / GROUP;            // columns of B held by one CTA
  static_assert(kBM == BN || kBM == 2 * BN || I8, "symmetric results need whole tiles on the diagonal");
  static constexpr int kKStage = I8 ? 128 : 64;        // k per stage: 128 bytes
  static constexpr int kABytes = 128 * 128, kBBytes = kBRows * 128;
  static constexpr int kStageBytes = PLANES * (kABytes + kBBytes);
  static constexpr int kTmemColumns = 2 * BN < 32 ? 32 : 2 * BN;
  static constexpr int kThreads = 320;
  static constexpr int kChunk = PLANES == 2 ? 2 : 0;   // k blocks summed in tensor memory, 0 = all
  static constexpr int kRatio = kBM / BN;              // tile columns per tile row
  static_assert(SPLIT == 1 || (GROUP == 1 && BN % (2 * SPLIT) == 0 && BN >= 32), "");
  static_assert(!PLAIN || (I8 && GROUP == 1 && BN <= 128), "");
  static_assert(!I8 || (!A_MN && !B_MN && PLANES == 1), "8-bit operands are K-major");
  static_assert(kTmemColumns <= 512 && (kTmemColumns & (kTmemColumns - 1)) == 0, "");
};

// Shared memory of one kernel: the ring, the exchange area of the epilogue, the barriers.
template <class C, class Epilogue>
struct UmmaMemory {
  // half columns of the result's tile, or what the epilogue's eight warps keep for themselves
  static constexpr int kStaging = Epilogue::kStaged ? C::PLANES * C::BN * 256 : C::BN / 2 * Epilogue::kWarpBytesPerColumn * 8;
  static constexpr int kFit = (224 * 1024 - kStaging) / C::kStageBytes;
  static constexpr int kStages = kFit < 8 ? kFit : 8;
  static constexpr size_t kBytes = 1024 + kStaging + (size_t)kStages * C::kStageBytes + 256;
  static_assert(kStages >= 2 && kBytes <= 227 * 1024, "");
  static_assert(C::SPLIT == 1 || C::BN * 512 <= kStages * C::kStageBytes, "the exchanged sums have to fit in the stages");
};

struct UmmaTile {
  int item, tm, tn;
};
// Tiles of one item in an order that keeps the operands of the tiles in flight together in L2: bands of eight tile
// rows, walked column by column; for a symmetric D the tiles that reach the diagonal or lie below it, row by row
// (tile row i has R (i + 1) of them, R columns of tiles being as wide as one row of tiles is high).
template <int R>
__host__ __device__ inline int symmetric_tiles(int tiles_m, int tiles_n) {
  const int last = R * tiles_m;
  return R * tiles_m * (tiles_m - 1) / 2 + (last < tiles_n ? last : tiles_n);
}
template <int R>
__device__ __forceinline__ UmmaTile umma_tile(const UmmaShape& s, int t) {
  UmmaTile r;
  if (s.symmetric) {
    const int per = symmetric_tiles<R>(s.tiles_m, s.tiles_n);
    r.item = t / per;
    const int f = t - r.item * per;
    int i = (int)((sqrtf((8.f / R) * (float)f + 1.f) - 1.f) * 0.5f);
    while (R * (i + 1) * (i + 2) / 2 <= f) ++i;
    while (R * i * (i + 1) / 2 > f) --i;
    r.tm = i;
    r.tn = f - R * i * (i + 1) / 2;
    return r;
  }
  const int per = s.tiles_m * s.tiles_n;
  r.item = t / per;
  const int f = t - r.item * per;
  constexpr int kBand = 8;
  const int band = f / (kBand * s.tiles_n), first = band * kBand;
  const int height = min(kBand, s.tiles_m - first);
  const int rest = f - band * kBand * s.tiles_n;
  r.tn = rest / height;
  r.tm = first + rest - r.tn * height;
  return r;
}

// Operands that are fetched with plain loads (8-bit, K-major).
struct PlainOperands {
  const int8_t* a;
  const int8_t* b;
  long long lda, ldb, sa, sb;
};

// 16 bytes at `src` (any alignment) of which the first `valid` exist, the rest zero.  [lo, hi) is the operand.  The five aligned
// words around them are read without branches, so that many such loads can be in flight, and shifted together when they are
// used; where one of them reaches over an end of the operand, `edge` says so and load16_bytes has to do it.
struct Words16 {
  uint32_t x[5];
  bool edge;
  __device__ __forceinline__ void load(const int8_t* src, int valid, const int8_t* lo, const int8_t* hi) {
    const int8_t* base = src - (reinterpret_cast<uintptr_t>(src) & 3u);
    const bool exists = valid > 0, inside = base >= lo && base + 20 <= hi;
#pragma unroll
    for (int j = 0; j < 5; ++j) {
      x[j] = 0;
      if (exists && inside) x[j] = reinterpret_cast<const uint32_t*>(base)[j];
    }
    edge = exists && !inside;
  }
  __device__ __forceinline__ uint4 value(const int8_t* src) const {
    const int sh = (int)(reinterpret_cast<uintptr_t>(src) & 3u) * 8;
    return make_uint4(__funnelshift_r(x[0], x[1], sh), __funnelshift_r(x[1], x[2], sh), __funnelshift_r(x[2], x[3], sh),
                      __funnelshift_r(x[3], x[4], sh));
  }
};
__device__ __forceinline__ uint32_t first_bytes(uint32_t w, int n) { return n >= 4 ? w : n <= 0 ? 0u : w & (0xffffffffu >> (8 * (4 - n))); }
__device__ __forceinline__ uint4 first_bytes(uint4 v, int n) {
  return make_uint4(first_bytes(v.x, n), first_bytes(v.y, n - 4), first_bytes(v.z, n - 8), first_bytes(v.w, n - 12));
}
static __device__ __noinline__ uint4 load16_bytes(const int8_t* src, int valid) {
  uint32_t w[4] = {0, 0, 0, 0};
  for (int i = 0; i < 16 && i < valid; ++i) {
    const uint32_t byte = (uint32_t)(uint8_t)src[i] << (8 * (i & 3));
    if (i < 4) w[0] |= byte;
    else if (i < 8) w[1] |= byte;
    else if (i < 12) w[2] |= byte;
    else w[3] |= byte;
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <class C, class Epilogue>
__global__ void __launch_bounds__(C::kThreads, 1)
    umma_gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                     const __grid_constant__ CUtensorMap map_old, const __grid_constant__ CUtensorMap map_out, const UmmaShape s,
                     const typename Epilogue::Params ep, const PlainOperands po, int wait_code) {
  using M = UmmaMemory<C, Epilogue>;
  constexpr int S = M::kStages, G = C::GROUP;
  constexpr int kCluster = G * C::SPLIT;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  unsigned char* staging = smem + (size_t)S * C::kStageBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(staging + M::kStaging);
  uint64_t* empty = full + S;
  uint64_t* acc_full = empty + S;
  uint64_t* acc_free = acc_full + 2;
  uint64_t* old_full = acc_free + 2;
  uint64_t* staging_free = old_full + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(staging_free + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t cta = kCluster > 1 ? cluster_rank() : 0, rank = G == 2 ? cta : 0;
  const int first = blockIdx.x / kCluster, step = gridDim.x / kCluster;
  // the range of k blocks of this CTA (with an empty sum, one block of zeros)
  const int all_blocks = max(1, (s.k + C::kKStage - 1) / C::kKStage);
  const int kb_begin = C::SPLIT == 1 ? 0 : (int)(all_blocks * cta / C::SPLIT);
  const int k_blocks = C::SPLIT == 1 ? all_blocks : (int)(all_blocks * (cta + 1) / C::SPLIT) - kb_begin;

  if (warp == 0 && lane == 0) {
    if constexpr (!C::PLAIN) {
      asm volatile("prefetch.tensormap [%0];" ::"l"(&map_a) : "memory");
      asm volatile("prefetch.tensormap [%0];" ::"l"(&map_b) : "memory");
    }
    for (int i = 0; i < S; ++i) {
      mbar_init(&full[i], C::PLAIN ? 8 : 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_free[i], 8 * G);
    }
    mbar_init(old_full, 1);
    mbar_init(staging_free, 1);
    mbar_fence_init();
  }
  if (warp == 1) {
    tmem_alloc<G>(tmem_slot, C::kTmemColumns);
    tc_fence_before();
  }
  __syncthreads();
  if constexpr (kCluster > 1) cluster_sync();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // The kernel before this one may still run: its results are read after a wait, which each role puts where it needs them.
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  if (warp == 0) {
    if (lane == 0 && !C::PLAIN) {
      bool ok = true;
      uint32_t round = 0;
      int slot = 0;
      for (int t = first; t < s.tiles && ok; t += step) {
        const UmmaTile tile = umma_tile<C::kRatio>(s, t);
        const int za = (s.a_items == 1 ? 0 : tile.item) * C::PLANES, zb = (s.b_items == 1 ? 0 : tile.item) * C::PLANES;
        const int m0 = tile.tm * C::kBM + (int)rank * 128, n0 = tile.tn * C::BN + (int)rank * C::kBRows;
        for (int kb = 0; kb < k_blocks && ok; ++kb) {
          ok = mbar_wait(&empty[slot], (round & 1) ^ 1, wait_code + kUmmaWaitEmpty);
          if (!ok) break;
          if (rank == 0) mbar_arrive_expect_tx(&full[slot], G * C::kStageBytes);
          const uint32_t bar = G == 2 ? cluster_addr(smem_u32(&full[slot]), 0) : smem_u32(&full[slot]);
          unsigned char* stage = smem + (size_t)slot * C::kStageBytes;
          auto load = [&](unsigned char* dst, const CUtensorMap* map, int x, int y, int z) {
            if constexpr (G == 2) tma_load_3d_pair(smem_u32(dst), map, x, y, z, bar);
            else tma_load_3d(dst, map, x, y, z, &full[slot]);
          };
          const int k0 = (kb_begin + kb) * C::kKStage;
          if (t == first && kb == 0) asm volatile("griddepcontrol.wait;" ::: "memory");
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
        ok = mbar_wait(&empty[slot], (round & 1) ^ 1, wait_code + kUmmaWaitEmpty);
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
      uint32_t done = 0;
      asm volatile("griddepcontrol.wait;" ::: "memory");  // so that the limit of the waits below counts this kernel's time alone
      for (int t = first; t < s.tiles && ok; t += step) {
        uint32_t d = 0;
        for (int kb = 0; kb < k_blocks; ++kb) {
          const bool begins = C::kChunk ? kb % (C::kChunk ? C::kChunk : 1) == 0 : kb == 0;
          if (begins) {
            const int acc = (int)(done & 1);
            ok = mbar_wait(&acc_free[acc], (uint32_t)((done >> 1) & 1) ^ 1, wait_code + kUmmaWaitAccFree);
            if (!ok) break;
            d = tmem + acc * C::BN;
          }
          ok = mbar_wait(&full[slot], round & 1, wait_code + kUmmaWaitFull);
          if (!ok) break;
          tc_fence_after();
          const uint32_t a = smem_u32(smem + (size_t)slot * C::kStageBytes), b = a + C::PLANES * C::kABytes;
          // 32 bytes of k per instruction: 32 bytes along a K-major row, 16 rows of 128 bytes of an MN-major block
          constexpr uint32_t kAStep = C::A_MN ? 2048 : 32, kBStep = C::B_MN ? 2048 : 32;
          constexpr uint32_t kALead = C::A_MN ? 8192 : 16, kBLead = C::B_MN ? 8192 : 16;
          auto desc_a = [&](int plane, int ks) { return umma_desc(a + plane * C::kABytes + ks * kAStep, kALead, 1024); };
          auto desc_b = [&](int plane, int ks) { return umma_desc(b + plane * C::kBBytes + ks * kBStep, kBLead, 1024); };
          if constexpr (C::PLANES == 2) {  // the small products first, while the sum that they are added to is small as well
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {
              umma<G, C::I8>(d, desc_a(0, ks), desc_b(1, ks), idesc, !begins || ks > 0);
              umma<G, C::I8>(d, desc_a(1, ks), desc_b(0, ks), idesc, true);
            }
          }
#pragma unroll
          for (int ks = 0; ks < 4; ++ks) umma<G, C::I8>(d, desc_a(0, ks), desc_b(0, ks), idesc, C::PLANES == 2 || !begins || ks > 0);
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
    asm volatile("griddepcontrol.wait;" ::: "memory");
    // Two warps per quarter of the 128 rows of the accumulator: each takes half of the columns.  Of a split tile a CTA stores
    // some of the rows (row-wise epilogues) or of the columns, cut the same way over the warps.
    constexpr bool kRows = Epilogue::kRows;
    constexpr int kCols = C::BN / 2, kOwnRows = kRows ? 128 / C::SPLIT : 128, kOwnCols = kRows ? C::BN : C::BN / C::SPLIT;
    constexpr int kRowParts = kOwnRows / 32, kMine = kOwnCols * kRowParts / 8, W = kMine < 16 ? kMine : 16;
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    const int row = quarter * 32 + lane;
    const int own_row = C::SPLIT > 1 ? ((warp - 2) % kRowParts) * 32 + lane : row;
    const int own_col = (C::SPLIT > 1 ? (warp - 2) / kRowParts : half) * kMine;
    const int first_row = (int)rank * 128 + (C::SPLIT > 1 && kRows ? (int)cta * kOwnRows : 0);  // of what this CTA stores
    const int first_col = C::SPLIT > 1 && !kRows ? (int)cta * kOwnCols : 0;
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16) + half * kCols;
    uint32_t done = 0, tiles_done = 0;
    auto acquire = [&]() {
      const int acc = (int)(done & 1);
      // the one wait that lasts as long as a tile's whole sum: its limit grows with the number of k blocks
      const bool got = mbar_wait_limit(&acc_full[acc], (uint32_t)((done >> 1) & 1), wait_code + kUmmaWaitAcc,
                                       kSpinLimit * (uint32_t)min(256, 1 + (k_blocks >> 12)));
      tc_fence_after();
      return (bool)__all_sync(0xffffffffu, got);
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
    // The staging buffer: boxes of 64 columns, rows of 128 bytes in the 128-byte swizzle (row-wise), or of kStagedColumns columns of
    // 128 rows.  Its owner sends for a tile's old values as soon as the tile before has left it.
    constexpr int kBoxCols = kRows ? 64 : kStagedColumns, kBoxBytes = kOwnRows * kBoxCols * 2, kPlaneBytes = kOwnRows * kOwnCols * 2;
    auto boxes = [&](const UmmaTile& tile, auto each) {
      for (int pl = 0; pl < C::PLANES; ++pl)
        for (int c = 0; c < kOwnCols; c += kBoxCols) {
          const int n = tile.tn * C::BN + first_col + c, m = tile.tm * C::kBM + first_row;
          each(staging + pl * kPlaneBytes + c / kBoxCols * kBoxBytes, kRows ? n : m, kRows ? m : n, tile.item * C::PLANES + pl, n < s.n && m < s.m);
        }
    };
    auto request_old = [&](int t) {
      mbar_arrive_expect_tx(old_full, C::PLANES * kPlaneBytes);
      boxes(umma_tile<C::kRatio>(s, t), [&](unsigned char* at, int x, int y, int z, bool) { tma_load_3d(at, &map_old, x, y, z, old_full); });
    };
    if constexpr (Epilogue::kStaged) {
      if (threadIdx.x == 64 && ep.has_old && first < s.tiles) request_old(first);
    }
    bool ok = true, fetched = true;
    uint32_t round = 0;
    int slot = 0;
    for (int t = first; t < s.tiles && ok; t += step) {
      const UmmaTile tile = umma_tile<C::kRatio>(s, t);
      if constexpr (C::PLAIN) {
        const int8_t* a = po.a + tile.item * po.sa;
        const int8_t* b = po.b + tile.item * po.sb;
        const int8_t* a_end = a + (long long)(s.m - 1) * po.lda + s.k;
        const int8_t* b_end = b + (long long)(s.n - 1) * po.ldb + s.k;
        // Sixteen bytes of every 32nd row per thread: those of A (i < 4), then those of B; both start on a multiple of eight rows.
        // One half of them is on its way while the other is shifted and stored.  The rows' addresses are formed once per tile: formed
        // again for every block and read as pairs of 16 bytes, 4096^3 took 370 us instead of 300, 401 x 867 x 6043 35 instead of 33.
        constexpr int kEach = (128 + C::kBRows) / 32;
        const int r0 = ((int)threadIdx.x - 64) >> 3, chunk = threadIdx.x & 7, ma = tile.tm * 128 + r0, nb = tile.tn * C::BN + r0;
        const int8_t* at_a = a + (long long)ma * po.lda + chunk * 16;
        const int8_t* at_b = b + (long long)nb * po.ldb + chunk * 16;
        const int8_t* from[kEach];
        bool exists[kEach];
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
          from[i] = (i < 4 ? at_a + (long long)(32 * i) * po.lda : at_b + (long long)(32 * (i - 4)) * po.ldb) + kb_begin * 128;
          exists[i] = i < 4 ? ma + 32 * i < s.m : nb + 32 * (i - 4) < s.n;
        }
        int left = s.k - kb_begin * 128 - chunk * 16;  // bytes of a row from this block on
        constexpr int kHalf = kEach / 2;
        auto load = [&](int part, Words16 (&v)[kHalf], int left, int ahead) {
#pragma unroll
          for (int h = 0; h < kHalf; ++h) {
            const int i = part * kHalf + h;
            v[h].load(from[i] + ahead, exists[i] ? left : 0, i < 4 ? a : b, i < 4 ? a_end : b_end);
          }
        };
        auto store = [&](int part, const Words16 (&v)[kHalf]) {
          unsigned char* to = smem + (size_t)slot * C::kStageBytes + r0 * 128 + ((chunk ^ (r0 & 7)) << 4);
          bool edge = false;
#pragma unroll
          for (int h = 0; h < kHalf; ++h) {
            const int i = part * kHalf + h;
            uint4 w = v[h].value(from[i]);
            if (left < 16) w = first_bytes(w, left);
            *reinterpret_cast<uint4*>(to + i * 32 * 128) = w;
            edge |= v[h].edge;
          }
          if (edge) {
#pragma unroll
            for (int i = part * kHalf; i < (part + 1) * kHalf; ++i)
              *reinterpret_cast<uint4*>(to + i * 32 * 128) = load16_bytes(from[i], exists[i] ? left : 0);
          }
        };
        Words16 v0[kHalf], v1[kHalf];
        load(0, v0, left, 0);
#pragma unroll 1
        for (int kb = 0; kb < k_blocks; ++kb) {
          load(1, v1, left, 0);
          ok = __all_sync(0xffffffffu, mbar_wait(&empty[slot], (round & 1) ^ 1, wait_code + kUmmaWaitEmpty));
          if (!ok) break;
          store(0, v0);
          if (kb + 1 < k_blocks) load(0, v0, left - 128, 128);
          store(1, v1);
#pragma unroll
          for (int i = 0; i < kEach; ++i) from[i] += 128;
          left -= 128;
          fence_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&full[slot]);
          if (++slot == S) {
            slot = 0;
            ++round;
          }
        }
        fetched = ok;
      }
      const int m = tile.tm * C::kBM + first_row + own_row, mine = tile.tn * C::BN + first_col + own_col;
      const bool twice = s.symmetric && tile.tn < C::kRatio * tile.tm;
      unsigned char* scratch = Epilogue::kStaged ? staging : staging + (warp - 2) * (M::kStaging / 8);
      typename Epilogue::template Tile<W, kMine, kOwnRows, kPlaneBytes> epi(ep, s, tile, twice, m, mine, scratch, own_row, own_col);
      if constexpr (C::kChunk == 0) {
        ok = k_blocks == 0 || acquire();
      } else if (k_blocks > 0) {
        // the chunks' sums, rounded to nearest, go back to where the last chunk was
        uint32_t v[kCols / 32][32] = {};
        for (int kb = 0; kb < k_blocks && ok; kb += C::kChunk) {
          ok = acquire();
#pragma unroll
          for (int c = 0; c < kCols / 32; ++c) {
            uint32_t w[32];
            tmem_ld(w, lanes + (uint32_t)(done & 1) * C::BN + c * 32);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) v[c][i] = __float_as_uint(__uint_as_float(v[c][i]) + __uint_as_float(w[i]));
          }
          if (kb + C::kChunk < k_blocks) release();
        }
#pragma unroll
        for (int c = 0; c < kCols / 32; ++c) tmem_st(lanes + (uint32_t)(done & 1) * C::BN + c * 32, v[c]);
        tmem_wait_st();
      }
      if constexpr (Epilogue::kStaged) {
        const uint32_t parity = (uint32_t)(tiles_done & 1);
        if (ep.has_old) ok = mbar_wait(old_full, parity, wait_code + kUmmaWaitOld) && ok;
        else ok = mbar_wait(staging_free, parity ^ 1, wait_code + kUmmaWaitStaging) && ok;
        ++tiles_done;
      }
      ok = named_all(ok && fetched, 256);
      __syncwarp();
      if constexpr (C::SPLIT == 1) {
        if (!ok) break;
#pragma unroll 1
        for (int c = 0; c < kMine; c += W) {
          if (mine + c >= s.n) break;
          uint32_t v[W];
          tmem_ld(v, lanes + (uint32_t)(done & 1) * C::BN + c);
          tmem_wait_ld();
          epi.group(v, c);
        }
        release();
      } else {
        // The cluster has this one tile.  Once every CTA is past its products the stages are free: each element goes to the CTA that
        // stores it, into its slab for this CTA.
        cluster_sync();
#pragma unroll 1
        for (int c = 0; c < kCols; c += 16) {
          uint32_t v[16] = {};
          if (k_blocks > 0) {
            tmem_ld(v, lanes + (uint32_t)(done & 1) * C::BN + c);
            tmem_wait_ld();
          }
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int col = half * kCols + c + i;
            const uint32_t to = cluster_addr(smem_u32(smem), kRows ? row / kOwnRows : col / kOwnCols) +
                                ((cta * kOwnCols + col % kOwnCols) * kOwnRows + row % kOwnRows) * 4;
            asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(to), "r"(v[i]) : "memory");
          }
        }
        cluster_sync();
        if (!ok) break;
        const uint32_t* sums = reinterpret_cast<const uint32_t*>(smem);
#pragma unroll 1
        for (int c = 0; c < kMine; c += W) {
          if (mine + c >= s.n) break;
          uint32_t v[W];
#pragma unroll
          for (int i = 0; i < W; ++i) {
            const int col = own_col + c + i;
            v[i] = sums[col * kOwnRows + own_row];
#pragma unroll
            for (int from = 1; from < C::SPLIT; ++from) {
              const uint32_t w = sums[(from * kOwnCols + col) * kOwnRows + own_row];
              v[i] = C::I8 ? v[i] + w : __float_as_uint(__uint_as_float(v[i]) + __uint_as_float(w));
            }
          }
          epi.group(v, c);
        }
      }
      if constexpr (Epilogue::kStaged) {
        fence_async_smem();
        named_all(true, 256);
        if (threadIdx.x == 64) {
          if constexpr (Epilogue::kStagedOut) {
            boxes(tile, [&](unsigned char* at, int x, int y, int z, bool exists) {
              if (exists) tma_store_3d(&map_out, at, x, y, z);
            });
            bulk_commit();
            bulk_wait_read<0>();
          }
          if (!ep.has_old) mbar_arrive(staging_free);
          else if (t + step < s.tiles) request_old(t + step);
        }
      }
    }
    // as the producer does
    for (int i = 0; i < S && C::PLAIN && ok && fetched; ++i) {
      ok = mbar_wait(&empty[slot], (round & 1) ^ 1, wait_code + kUmmaWaitEmpty);
      if (++slot == S) {
        slot = 0;
        ++round;
      }
    }
  }
  if constexpr (C::SPLIT > 1) {
    if (warp < 2) {  // the two exchanges of the epilogue warps
      __syncwarp();
      cluster_sync();
      cluster_sync();
    }
  }
  __syncwarp();
  __syncthreads();
  if constexpr (kCluster > 1) cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    tmem_free<G>(tmem, C::kTmemColumns);
  }
}

// ---- host side -----------------------------------------------------------------------------------
// 3-D map (inner, outer, z) over `base`: box of 128 bytes x box_outer rows x 1, 128-byte swizzle; `staged` (half only): box of 128
// elements x box_outer rows without a swizzle, for the staging buffer.  Strides in bytes.
inline int encode_operand(CUtensorMap* map, const void* base, bool i8, long long inner, long long outer, long long z, long long ld_bytes,
                          long long z_bytes, int box_outer, bool staged = false) {
  EncodeTiledFn enc = encode_tiled_fn();
  if (!enc) return BLB200_E_INTERNAL;
  const cuuint64_t dims[3] = {(cuuint64_t)inner, (cuuint64_t)outer, (cuuint64_t)z};
  const cuuint64_t strides[2] = {(cuuint64_t)ld_bytes, (cuuint64_t)(z > 1 ? z_bytes : ld_bytes * outer)};
  const cuuint32_t box[3] = {i8 || staged ? 128u : 64u, (cuuint32_t)box_outer, 1}, estr[3] = {1, 1, 1};
  const CUresult r = enc(map, i8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(base), dims, strides,
                         box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, staged ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? BLB200_OK : BLB200_E_INTERNAL;
}

// How many clusters (or CTAs) of this kernel the current device holds at once: clusters do not straddle the device's groups of
// SMs, so it is less than the number of SMs over the cluster's size.  Asked once per device and thread.
template <class C, class Epilogue>
int umma_capacity() {
  constexpr int kCluster = C::GROUP * C::SPLIT;
  if (kCluster == 1) return device_info().sm_count;
  static thread_local int known[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) dev = 0;
  if (known[dev] == 0) {
    auto kern = umma_gemm_kernel<C, Epilogue>;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(kCluster);
    cfg.blockDim = dim3(C::kThreads);
    cfg.dynamicSmemBytes = UmmaMemory<C, Epilogue>::kBytes;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = kCluster;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)UmmaMemory<C, Epilogue>::kBytes) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n < 1) {
      cudaGetLastError();
      n = std::max(1, device_info().sm_count / kCluster - 4);
    }
    known[dev] = n;
  }
  return known[dev];
}

template <class C, class Epilogue>
int launch_umma(const CUtensorMap& map_a, const CUtensorMap& map_b, const CUtensorMap& map_old, const CUtensorMap& map_out, UmmaShape s, const typename Epilogue::Params& ep, int wait_code,
                cudaStream_t stream, const PlainOperands& po = PlainOperands{}) {
  constexpr int kCluster = C::GROUP * C::SPLIT;
  s.tiles_m = (s.m + C::kBM - 1) / C::kBM;
  s.tiles_n = (s.n + C::BN - 1) / C::BN;
  const long long tiles = (s.symmetric ? (long long)symmetric_tiles<C::kRatio>(s.tiles_m, s.tiles_n) : (long long)s.tiles_m * s.tiles_n) * s.batch;
  if (tiles > 0x3fffffffll || (long long)s.tiles_m * s.tiles_n > 0x3fffffffll) return BLB200_E_TOO_LARGE;
  s.tiles = (int)tiles;
  auto kern = umma_gemm_kernel<C, Epilogue>;
  static thread_local int configured_for = -1;
  int cur = 0;
  cudaGetDevice(&cur);
  if (configured_for != cur) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)UmmaMemory<C, Epilogue>::kBytes);
    if (e != cudaSuccess) return (int)e;
    configured_for = cur;
  }
  // a split tile has a cluster of its own, otherwise the CTAs or pairs that the device holds walk over the tiles
  const long long units = C::SPLIT > 1 ? s.tiles : umma_capacity<C, Epilogue>();
  if (units * kCluster > 0x7fffffffll) return BLB200_E_TOO_LARGE;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((s.tiles < units ? s.tiles : units) * kCluster));
  cfg.blockDim = dim3(C::kThreads);
  cfg.dynamicSmemBytes = UmmaMemory<C, Epilogue>::kBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = kCluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = kCluster > 1 ? 2 : 1;
  return (int)cudaLaunchKernelEx(&cfg, kern, map_a, map_b, map_old, map_out, s, ep, po, wait_code);
}

}  // namespace blb200
