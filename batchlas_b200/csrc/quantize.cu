// Quantises every column of a batch of k x cols matrices to 8-bit integers with one scale per column:
// scale = fl32(max |x| * fl32(1 / 127)), q = rne(fl32(x / scale)) clamped to +-127.
// Infinity and NaN travel through the maxima into the scale.
#include <type_traits>

#include "lowp.cuh"
#include "ptx.cuh"

namespace blb200 {
namespace {

struct QuantizeParams {
  const void* x;
  int8_t* q;
  float* scale;
  int k, cols, batch;
  long long ldx, sx, ldq, sq, ss;
};

// Quantises through the reciprocal: r = fma(x, inv, 1.5 * 2^23) holds the integer nearest to x * inv, halves to even, in its
// last bits.  x * inv and fl32(x / scale) differ by a few 2^-24 of their value y, so only where y is as close as that to a
// halfway point can the integers differ.
//   Half types: y = 127 x / max, and 2 y - odd is a multiple of 1 / (the mantissa of max): unless it is zero, y is further
//   than y / (127 * 2047) = 3.8e-6 y from the halfway point, more than the errors together.  It is zero where 254 x = odd max:
//   127 being prime, for y = 63.5 (half the largest value, one element in a thousand), or where max is a multiple of 127, which
//   shows in an exact quotient (one column in a hundred; divided).  So inv is moved by the few last places that make 63.5
//   come out as the division has it, and nothing is left to check.
//   float: |d| = |x * inv - r| within 2^-14 of one half is divided after all (one element in ten thousand).
// Columns whose scale is so small that it or its reciprocal lose bits divide always.
template <bool HALF>
struct Quantiser {
  static constexpr float kShift = 12582912.f;
  float scale, inv;
  bool usable, divide;
  __device__ explicit Quantiser(float top) {
    scale = top * (1.f / 127.f);
    usable = scale > 0.f && top < __int_as_float(0x7f800000);
    divide = scale < 1e-36f || (HALF && fmaf(__fdiv_rn(top, 127.f), 127.f, -top) == 0.f);
    inv = usable && !divide ? __frcp_rn(scale) : 0.f;
    if (HALF && usable && !divide) {
      const int want = exact(0.5f * top);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int got = __float_as_int(fmaf(0.5f * top, inv, kShift)) - __float_as_int(kShift);
        inv = __int_as_float(__float_as_int(inv) + (got < want ? 1 : got > want ? -1 : 0));
      }
    }
  }
  __device__ __forceinline__ int exact(float x) const { return (int)fminf(127.f, fmaxf(-127.f, rintf(__fdiv_rn(x, scale)))); }
  // The last byte of each element of out is the quantised value.  Only called where the column is usable.
  template <int N>
  __device__ __forceinline__ void quantise(const float (&x)[N], uint32_t (&out)[N]) const {
    float off = 0.f;
    if constexpr (N % 2 == 0) {  // two elements per instruction
      const uint64_t inv2 = dup2(inv), shift2 = dup2(kShift), minus2 = dup2(-1.f);
#pragma unroll
      for (int i = 0; i < N; i += 2) {
        const uint64_t x2 = (uint64_t)__float_as_uint(x[i]) | (uint64_t)__float_as_uint(x[i + 1]) << 32;
        uint64_t r2 = shift2;
        ffma2(r2, x2, inv2);
        float r0, r1;
        unpack2(r2, r0, r1);
        out[i] = __float_as_uint(r0);
        out[i + 1] = __float_as_uint(r1);
        if constexpr (!HALF) {
          uint64_t d2 = shift2;
          float d0, d1;
          ffma2(d2, r2, minus2);
          ffma2(d2, x2, inv2);
          unpack2(d2, d0, d1);
          off = fmaxf(off, fmaxf(fabsf(d0), fabsf(d1)));
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float r = fmaf(x[i], inv, kShift);
        out[i] = __float_as_uint(r);
        if constexpr (!HALF) off = fmaxf(off, fabsf(fmaf(x[i], inv, kShift - r)));
      }
    }
    if (divide || (!HALF && off > 0.5f - 0x1p-14f)) {
#pragma unroll
      for (int i = 0; i < N; ++i) out[i] = (uint32_t)exact(x[i]);
    }
  }
};

__device__ __forceinline__ uint32_t pack_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
// max |.| that keeps a NaN
__device__ __forceinline__ float max_abs(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(fabsf(a)), "f"(fabsf(b)));
  return r;
}

// V elements of a column held as 16 bytes.
template <typename T, int V>
struct Unit {
  uint4 w = make_uint4(0, 0, 0, 0);
  __device__ __forceinline__ void load(const T* at) { w = *reinterpret_cast<const uint4*>(at); }
  __device__ __forceinline__ void values(float (&x)[V]) const {
    const uint32_t p[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, float>::value) {
        x[i] = __uint_as_float(p[i]);
      } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        x[2 * i] = __uint_as_float(p[i] << 16);
        x[2 * i + 1] = __uint_as_float(p[i] & 0xffff0000u);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&p[i]));
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
      }
    }
  }
  // max(t, |every element|), keeping NaN
  __device__ __forceinline__ float top(float t) const {
    if constexpr (std::is_same<T, float>::value) {
      return max_abs(max_abs(t, __uint_as_float(w.x)), max_abs(max_abs(__uint_as_float(w.y), __uint_as_float(w.z)), __uint_as_float(w.w)));
    } else {
      using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
      auto pair = [](uint32_t p) { return __habs2(*reinterpret_cast<const T2*>(&p)); };
      const T2 m = __hmax2_nan(__hmax2_nan(pair(w.x), pair(w.y)), __hmax2_nan(pair(w.z), pair(w.w)));
      return max_abs(t, max_abs(to_f32(m.x), to_f32(m.y)));
    }
  }
  template <class Z>
  __device__ __forceinline__ void store(int8_t* to, const Z& z) const {
    float x[V];
    values(x);
    uint32_t q[V];
    z.template quantise<V>(x, q);
    if constexpr (V == 8) *reinterpret_cast<uint2*>(to) = make_uint2(pack_bytes(q[0], q[1], q[2], q[3]), pack_bytes(q[4], q[5], q[6], q[7]));
    else *reinterpret_cast<uint32_t*>(to) = pack_bytes(q[0], q[1], q[2], q[3]);
  }
};

// Largest magnitude over the blockDim.x threads of a column.  Magnitudes order like their bits, NaN above infinity.
__device__ __forceinline__ float column_max(float mine) {
  __shared__ unsigned part[32];
  unsigned top = __reduce_max_sync(0xffffffffu, __float_as_uint(mine) & 0x7fffffffu);
  const int warps = blockDim.x >> 5;
  if (warps == 1) return __uint_as_float(top);
  const int lane = threadIdx.x & 31, first = threadIdx.y * warps;
  if (lane == 0) part[first + (threadIdx.x >> 5)] = top;
  __syncthreads();
  top = __reduce_max_sync(0xffffffffu, lane < warps ? part[first + lane] : 0u);
  return __uint_as_float(top);
}

// A column is held in the registers of blockDim.x threads (a multiple of 32) and read once; a block has blockDim.y columns,
// blockIdx.y and beyond are items (no index is divided: with thirty-odd elements per thread a division costs as much as a
// tenth of the work).  Memory is all that it should cost: 8192 x 8192 bfloat16 moves 201 MB.  WIDE: up to PER units of 16 bytes per thread, for
// columns of x and q that start on their boundaries; else up to PER single elements.
template <typename T, bool WIDE, int PER>
__global__ void __launch_bounds__(1024) quantize_kernel(QuantizeParams p) {
  griddep_wait();
  griddep_launch();
  constexpr int V = WIDE ? 16 / (int)sizeof(T) : 1;
  const long long item = blockIdx.y, col = (long long)blockIdx.x * blockDim.y + threadIdx.y;
  const bool live = col < p.cols;
  const int tx = blockDim.x, x0 = threadIdx.x, units = live ? p.k / V : 0;
  const T* x = (const T*)p.x + item * p.sx + col * p.ldx + (long long)x0 * V;
  int8_t* q = p.q + item * p.sq + col * p.ldq + (long long)x0 * V;
  float top = 0.f;
  if constexpr (WIDE) {
    Unit<T, V> u[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (x0 + i * tx < units) u[i].load(x + i * tx * V);
#pragma unroll
    for (int i = 0; i < PER; ++i) top = u[i].top(top);
    const Quantiser<sizeof(T) == 2> z(column_max(top));
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (x0 + i * tx < units) {
        if (z.usable) u[i].store(q + i * tx * V, z);
        else if constexpr (V == 8) *reinterpret_cast<uint2*>(q + i * tx * V) = make_uint2(0, 0);
        else *reinterpret_cast<uint32_t*>(q + i * tx * V) = 0;
      }
    if (live && x0 == 0) p.scale[item * p.ss + col] = z.scale;
  } else {
    float v[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) v[i] = x0 + i * tx < units ? to_f32(x[i * tx]) : 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) top = max_abs(top, v[i]);
    const Quantiser<sizeof(T) == 2> z(column_max(top));
    uint32_t b[PER];
    if (z.usable) z.template quantise<PER>(v, b);
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (x0 + i * tx < units) q[i * tx] = z.usable ? (int8_t)b[i] : (int8_t)0;
    if (live && x0 == 0) p.scale[item * p.ss + col] = z.scale;
  }
}

// Columns longer than a block's registers: read twice, the second time mostly from L2.
template <typename T, bool WIDE>
__global__ void __launch_bounds__(1024) quantize_long_kernel(QuantizeParams p) {
  griddep_wait();
  griddep_launch();
  constexpr int V = WIDE ? 16 / (int)sizeof(T) : 1;
  const long long item = blockIdx.y, col = blockIdx.x;
  const T* x = (const T*)p.x + item * p.sx + col * p.ldx;
  int8_t* q = p.q + item * p.sq + col * p.ldq;
  const int units = p.k / V;
  float top = 0.f;
#pragma unroll 4
  for (int i = threadIdx.x; i < units; i += blockDim.x) {
    if constexpr (WIDE) {
      Unit<T, V> u;
      u.load(x + (long long)i * V);
      top = u.top(top);
    } else {
      top = max_abs(top, to_f32(x[i]));
    }
  }
  const Quantiser<sizeof(T) == 2> z(column_max(top));
  if (threadIdx.x == 0) p.scale[item * p.ss + col] = z.scale;
#pragma unroll 2
  for (int i = threadIdx.x; i < units; i += blockDim.x) {
    if constexpr (WIDE) {
      Unit<T, V> u;
      if (z.usable) u.load(x + (long long)i * V);
      if (z.usable) u.store(q + (long long)i * V, z);
      else if constexpr (V == 8) *reinterpret_cast<uint2*>(q + (long long)i * V) = make_uint2(0, 0);
      else *reinterpret_cast<uint32_t*>(q + (long long)i * V) = 0;
    } else {
      const float v[1] = {to_f32(x[i])};
      uint32_t b[1] = {0};
      if (z.usable) z.template quantise<1>(v, b);
      q[i] = (int8_t)b[0];
    }
  }
}

template <typename T, bool WIDE>
int launch_quantize(const QuantizeParams& p, cudaStream_t stream) {
  constexpr int V = WIDE ? 16 / (int)sizeof(T) : 1;
  const long long total = (long long)p.cols * p.batch, units = p.k / V;
  // units per thread: one where there are few columns to fill the machine with, else enough to make a thread worth its start
  const bool few = total * ((units + 3) / 4) < device_info().sm_count * 1024ll;
  const int per = few && units <= 1024 ? 1 : WIDE ? (units < 256 ? 4 : 8) : (units < 256 ? 4 : 16);
  const long long threads = (units + per - 1) / per;
  if (threads > 1024) {
    const OverlappedLaunch launch(dim3((unsigned)p.cols, (unsigned)p.batch), 1024, stream);
    return (int)cudaLaunchKernelEx(&launch.cfg, quantize_long_kernel<T, WIDE>, p);
  }
  const unsigned tx = threads <= 32 ? 32 : (unsigned)((threads + 31) / 32 * 32);
  const unsigned columns = tx >= 128 ? 1 : 128 / tx;
  const OverlappedLaunch launch(dim3((p.cols + columns - 1) / columns, (unsigned)p.batch), dim3(tx, columns), stream);
  if (per == 1) return (int)cudaLaunchKernelEx(&launch.cfg, quantize_kernel<T, WIDE, 1>, p);
  if (per == 4) return (int)cudaLaunchKernelEx(&launch.cfg, quantize_kernel<T, WIDE, 4>, p);
  return (int)cudaLaunchKernelEx(&launch.cfg, quantize_kernel<T, WIDE, WIDE ? 8 : 16>, p);
}

int validate_quantize(const blb200_quantize_desc* d) {
  if (!d) return BLB200_E_NULL;
  if (!valid_ftype(d->ftype)) return BLB200_E_DTYPE;
  if (d->k < 0 || d->cols < 0 || d->batch < 0) return BLB200_E_SHAPE;
  if (d->k > kMaxDim || d->cols > kMaxDim) return BLB200_E_TOO_LARGE;
  if (!readable_layout(d->k, d->ldx, d->stride_x) || !writable_layout(d->k, d->cols, d->batch, d->ldq, d->stride_q) ||
      !writable_layout(1, d->cols, d->batch, 1, d->stride_scale))
    return BLB200_E_SHAPE;
  if (d->cols > 0 && d->batch > 0 && (!d->scale || (d->k > 0 && (!d->x || !d->q)))) return BLB200_E_NULL;
  return BLB200_OK;
}

}  // namespace
}  // namespace blb200

extern "C" int blb200_quantize_i8(const blb200_quantize_desc* d, void* cuda_stream) {
  using namespace blb200;
  const int rc = validate_quantize(d);
  if (rc != BLB200_OK) return rc;
  if (d->cols == 0 || d->batch == 0) return BLB200_OK;
  QuantizeParams p{d->x,        d->q,        d->scale,   d->k,        d->cols,        d->batch,
                   d->ldx,      d->stride_x, d->ldq,     d->stride_q, d->stride_scale};
  return with_ftype(d->ftype, [&](auto t) {
    using T = decltype(t);
    constexpr int V = 16 / sizeof(T);
    auto whole = [&](const void* base, long long ld, long long stride, long long bytes) {
      return reinterpret_cast<uintptr_t>(base) % (V * bytes) == 0 && (ld % V == 0 || p.cols == 1) && (stride % V == 0 || p.batch == 1);
    };
    const bool wide = p.k % V == 0 && whole(p.x, p.ldx, p.sx, sizeof(T)) && whole(p.q, p.ldq, p.sq, 1);
    for (int first = 0; first < d->batch; first += 65535) {  // items are the grid's second dimension
      QuantizeParams part = p;
      part.x = (const T*)p.x + first * p.sx;
      part.q = p.q + first * p.sq;
      part.scale = p.scale + first * p.ss;
      part.batch = d->batch - first < 65535 ? d->batch - first : 65535;
      const int e = wide ? launch_quantize<T, true>(part, (cudaStream_t)cuda_stream) : launch_quantize<T, false>(part, (cudaStream_t)cuda_stream);
      if (e != 0) return e;
      note_launch("quantize_i8");
    }
    return (int)BLB200_OK;
  });
}
