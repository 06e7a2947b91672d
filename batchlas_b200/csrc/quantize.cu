// Quantises every column of a batch of k x cols matrices to 8-bit integers with one scale per column:
// scale = fl32(max |x| / 127), q = rne(fl32(x / scale)) clamped to +-127.
// The magnitudes are compared as the bit patterns of |x|: they order as unsigned integers, with infinity
// above every number and NaN above infinity, so one integer maximum also carries non-finite values into
// the scale.
#include "lowp.cuh"

namespace blb200 {
namespace {

struct QuantizeParams {
  const void* x;
  int8_t* q;
  float* scale;
  int k, cols, batch;
  long long ldx, sx, ldq, sq, ss;
};

// Quantises through the reciprocal: y = x * inv differs from fl32(x / scale) by less than 2^-15 (two roundings of a value
// of at most 127), so wherever y is further than 2^-14 from a halfway point both round to the same integer; the
// few others are divided.  Subnormal scales, whose reciprocal is not accurate, divide always.
struct Quantiser {
  float scale, inv;
  bool usable, divide;
  __device__ explicit Quantiser(unsigned top) {
    scale = __fdiv_rn(__uint_as_float(top), 127.f);
    usable = scale > 0.f && top < 0x7f800000u;
    divide = scale < 1e-36f;
    inv = usable && !divide ? __frcp_rn(scale) : 0.f;
  }
  __device__ __forceinline__ int exact(float x) const {
    return (int)fminf(127.f, fmaxf(-127.f, rintf(__fdiv_rn(x, scale))));
  }
  // N values to N bytes.
  template <int N>
  __device__ __forceinline__ void quantise(const float (&x)[N], uint32_t (&out)[(N + 3) / 4]) const {
    constexpr float kShift = 12582912.f;  // 1.5 * 2^23: the sum's last bits are the nearest integer, halves to even
    uint32_t q[N];
    float off = divide ? 1.f : 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float y = usable ? x[i] * inv : 0.f, r = y + kShift;
      q[i] = __float_as_uint(r);
      off = fmaxf(off, fabsf(y - (r - kShift)));
    }
    if (off > 0.5f - 0x1p-14f && usable) {
#pragma unroll
      for (int i = 0; i < N; ++i) q[i] = (uint32_t)exact(x[i]);
    }
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      if constexpr (N >= 4) out[i / 4] = __byte_perm(__byte_perm(q[i], q[i + 1], 0x0040), __byte_perm(q[i + 2], q[i + 3], 0x0040), 0x5410);
      else out[0] = q[0];
    }
  }
};

// V elements of a column: 16 bytes of x, V bytes of q.
template <typename T, int V>
struct Unit {
  __align__(16) T v[V];
  __device__ __forceinline__ void load(const T* at) {
    if constexpr (V > 1) *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(at);
    else v[0] = *at;
  }
  __device__ __forceinline__ unsigned top() const {
    unsigned t = 0;
#pragma unroll
    for (int e = 0; e < V; ++e) t = max(t, __float_as_uint(to_f32(v[e])) & 0x7fffffffu);
    return t;
  }
  __device__ __forceinline__ void store(int8_t* to, const Quantiser& z) const {
    float x[V];
#pragma unroll
    for (int e = 0; e < V; ++e) x[e] = to_f32(v[e]);
    uint32_t out[(V + 3) / 4];
    z.quantise<V>(x, out);
    if constexpr (V == 8) *reinterpret_cast<uint2*>(to) = make_uint2(out[0], out[1]);
    else if constexpr (V == 4) *reinterpret_cast<uint32_t*>(to) = out[0];
    else *to = (int8_t)out[0];
  }
};

// Largest magnitude over the tx threads of a column.
__device__ __forceinline__ unsigned column_max(unsigned top, int tx) {
  __shared__ unsigned part[32];
  top = __reduce_max_sync(0xffffffffu, top);
  if (tx == 32) return top;
  const int warp = threadIdx.x >> 5, first = threadIdx.x / tx * (tx >> 5), n = tx >> 5;
  if ((threadIdx.x & 31) == 0) part[warp] = top;
  __syncthreads();
  top = 0;
  for (int i = 0; i < n; ++i) top = max(top, part[first + i]);
  return top;
}

// A column is held in the registers of its tx threads (a multiple of 32), up to PER units each, and read once; a block has
// blockDim / tx columns.  Memory is all that it costs: 8192 x 8192 bfloat16 moves 201 MB.
template <typename T, int V, int PER>
__global__ void __launch_bounds__(1024) quantize_kernel(QuantizeParams p, int tx) {
  griddep_wait();
  griddep_launch();
  const long long total = (long long)p.cols * p.batch;
  const long long w = (long long)blockIdx.x * (blockDim.x / tx) + threadIdx.x / tx;
  const bool live = w < total;
  const long long item = live ? w / p.cols : 0, col = live ? w - item * p.cols : 0;
  const T* x = (const T*)p.x + item * p.sx + col * p.ldx;
  int8_t* q = p.q + item * p.sq + col * p.ldq;
  const int units = live ? p.k / V : 0, x0 = threadIdx.x % tx;
  Unit<T, V> u[PER];
  unsigned top = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (x0 + i * tx < units) u[i].load(x + (long long)(x0 + i * tx) * V);
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (x0 + i * tx < units) top = max(top, u[i].top());
  const Quantiser z(column_max(top, tx));
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (x0 + i * tx < units) u[i].store(q + (long long)(x0 + i * tx) * V, z);
  if (live && x0 == 0) p.scale[item * p.ss + col] = z.scale;
}

// Columns longer than a block's registers: read twice, the second time mostly from L2.
template <typename T, int V>
__global__ void __launch_bounds__(1024) quantize_long_kernel(QuantizeParams p) {
  griddep_wait();
  griddep_launch();
  const long long item = blockIdx.x / p.cols, col = blockIdx.x - item * p.cols;
  const T* x = (const T*)p.x + item * p.sx + col * p.ldx;
  int8_t* q = p.q + item * p.sq + col * p.ldq;
  const int units = p.k / V;
  unsigned top = 0;
#pragma unroll 4
  for (int i = threadIdx.x; i < units; i += blockDim.x) {
    Unit<T, V> u;
    u.load(x + (long long)i * V);
    top = max(top, u.top());
  }
  const Quantiser z(column_max(top, blockDim.x));
#pragma unroll 4
  for (int i = threadIdx.x; i < units; i += blockDim.x) {
    Unit<T, V> u;
    u.load(x + (long long)i * V);
    u.store(q + (long long)i * V, z);
  }
  if (threadIdx.x == 0) p.scale[item * p.ss + col] = z.scale;
}

template <typename T, int V>
int launch_quantize(const QuantizeParams& p, cudaStream_t stream) {
  const long long total = (long long)p.cols * p.batch, units = p.k / V;
  // units per thread: few where there are few columns to fill the machine with, more where threads would idle
  const bool few = total * ((units + 3) / 4) < 148ll * 1024;
  const int per = few && units <= 1024 ? 1 : V > 1 || units <= 4096 ? 4 : 16;
  const long long threads = (units + per - 1) / per;
  if (threads > 1024) {
    if (total > 0x7fffffffll) return BLB200_E_TOO_LARGE;
    const OverlappedLaunch launch((unsigned)total, 1024, stream);
    return (int)cudaLaunchKernelEx(&launch.cfg, quantize_long_kernel<T, V>, p);
  }
  const int tx = threads <= 32 ? 32 : (int)((threads + 31) / 32 * 32);
  const int columns = tx >= 256 ? 1 : 256 / tx;
  const long long grid = (total + columns - 1) / columns;
  if (grid > 0x7fffffffll) return BLB200_E_TOO_LARGE;
  auto kern = per == 1 ? quantize_kernel<T, V, 1> : per == 4 ? quantize_kernel<T, V, 4> : quantize_kernel<T, V, (V == 1 ? 16 : 4)>;
  const OverlappedLaunch launch((unsigned)grid, columns * tx, stream);
  return (int)cudaLaunchKernelEx(&launch.cfg, kern, p, tx);
}

int validate_quantize(const blb200_quantize_desc* d) {
  if (!d) return BLB200_E_NULL;
  if (!valid_ftype(d->ftype)) return BLB200_E_DTYPE;
  if (d->k < 0 || d->cols < 0 || d->batch < 0) return BLB200_E_SHAPE;
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
    const int e = wide ? launch_quantize<T, V>(p, (cudaStream_t)cuda_stream) : launch_quantize<T, 1>(p, (cudaStream_t)cuda_stream);
    if (e == 0) note_launch("quantize_i8");
    return e;
  });
}
