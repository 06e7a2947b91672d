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

__device__ __forceinline__ int quantize_one(float x, float scale, bool usable) {
  if (!usable) return 0;
  const float r = rintf(__fdiv_rn(x, scale));
  return (int)fminf(127.f, fmaxf(-127.f, r));
}

// One block per column.
template <typename T>
__global__ void __launch_bounds__(256) quantize_column_kernel(QuantizeParams p) {
  __shared__ unsigned warp_max[8];
  const long long total = (long long)p.cols * p.batch;
  for (long long w = blockIdx.x; w < total; w += gridDim.x) {
    const long long item = w / p.cols, col = w - item * p.cols;
    const T* x = (const T*)p.x + item * p.sx + col * p.ldx;
    int8_t* q = p.q + item * p.sq + col * p.ldq;
    unsigned top = 0;
    for (int i = threadIdx.x; i < p.k; i += blockDim.x) top = max(top, __float_as_uint(to_f32(x[i])) & 0x7fffffffu);
    top = __reduce_max_sync(0xffffffffu, top);
    if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = top;
    __syncthreads();
    top = 0;
    for (int i = 0; i < 8; ++i) top = max(top, warp_max[i]);
    __syncthreads();
    const float scale = __fdiv_rn(__uint_as_float(top), 127.f);
    const bool usable = scale > 0.f && top < 0x7f800000u;
    for (int i = threadIdx.x; i < p.k; i += blockDim.x) q[i] = (int8_t)quantize_one(to_f32(x[i]), scale, usable);
    if (threadIdx.x == 0) p.scale[item * p.ss + col] = scale;
  }
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
  const long long total = (long long)p.cols * p.batch;
  const long long cap = (long long)device_info().sm_count * 8;
  const unsigned grid = (unsigned)(total < cap ? total : cap);
  return with_ftype(d->ftype, [&](auto t) {
    quantize_column_kernel<decltype(t)><<<grid, 256, 0, (cudaStream_t)cuda_stream>>>(p);
    const int e = (int)cudaGetLastError();
    if (e == 0) note_launch("quantize_i8");
    return e;
  });
}
