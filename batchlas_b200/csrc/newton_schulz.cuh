// What the two forms of the Newton-Schulz iteration (products over global memory, and one CTA per small matrix) share: the
// bounds and scales of the stored matrices, and the factors of the products' epilogues that follow from them.
#pragma once

#include <math.h>

#include "lowp.cuh"

namespace blb200 {

constexpr int kMaxSteps = 64;
constexpr double kMaxSigma = 64.0, kMaxEntry = 16384.0;
constexpr double kGrowth = 1.01;  // what the roundings of a step may add to the bound of X

struct Matrices {
  void* p;
  int rows, cols, batch;
  long long ld, stride;
};

// Largest |a s + b s^3 + c s^5| over 0 <= s <= top.
__host__ __device__ inline double polynomial_bound(const double* q, double top) {
  auto value = [&](double s) { return fabs(s * (q[0] + s * s * (q[1] + s * s * q[2]))); };
  double best = value(top);
  // Critical points: C + B t + A t^2 = 0 with t = (s / top)^2, its coefficients divided by the largest so that no square
  // leaves double's range.  w adds numbers of one sign, so neither root is lost to cancellation where A or C is next to zero.
  const double s2 = top * top;
  double A = q[2] * s2 * s2 * 5, B = q[1] * s2 * 3, C = q[0];
  const double size = fmax(fabs(A), fmax(fabs(B), fabs(C)));
  if (!(size > 0)) return best;
  A /= size;
  B /= size;
  C /= size;
  const double disc = B * B - 4 * A * C;
  if (disc >= 0) {
    const double w = -0.5 * (B + copysign(sqrt(disc), B));
    const double roots[2] = {w != 0 ? C / w : 0.0, A != 0 ? w / A : 0.0};
    for (double t : roots)
      if (t > 0 && t < 1) best = fmax(best, value(top * sqrt(t)));
  }
  return best;
}

__device__ __forceinline__ double block_sum(double v) {
  __shared__ double part[32];
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0;
  for (int i = 0; i < (int)(blockDim.x >> 5); ++i) v += part[i];
  __syncthreads();
  return v;
}

// Power of two that takes a value of at most `top` below 2^15.
__host__ __device__ inline double half_scale(double top) {
  if (!(top > 0) || isinf(top)) return 1.0;
  const int e = 14 - ilogb(top);
  return scalbn(1.0, e > 400 ? 400 : e);
}

// The powers of two that S, B and the next X are stored with at one step, from the bound of X before it.
struct StepScales {
  double s, b, next;
};
__host__ __device__ inline StepScales step_scales(const double* q, double& sigma, bool last) {
  const double s2 = sigma * sigma;
  StepScales r;
  r.s = half_scale(s2);
  r.b = half_scale(fabs(q[1]) * s2 + fabs(q[2]) * s2 * s2);
  sigma = polynomial_bound(q, sigma) * kGrowth;
  r.next = last ? 1.0 : half_scale(sigma);
  return r;
}

struct Plan {
  double q[3 * kMaxSteps];        // coefficients, by step
  StepScales scales[kMaxSteps];   // for a matrix that starts with |X| <= 1
  double eps;
  int steps;
};

// The factors (alpha, beta) of every product, three per step and `stride` apart, for an item with norm `norm` and f = norm +
// eps, stored as G * 2^e: X = stored / (2^e f).  By all threads of a block of at least kMaxSteps; `own` is shared scratch.  The
// bounds for |X| <= 1 hold for every item; one that eps makes much smaller gets its own, so that its matrices do not sink
// towards half's smallest numbers.
__device__ __forceinline__ void write_factors(const Plan& plan, double norm, double f, int e, StepScales* own, float2* factors, int stride) {
  const bool small = norm < 0.125 * f;
  if (small) {
    if (threadIdx.x == 0) {
      double sigma = norm / f;
      for (int i = 0; i < plan.steps; ++i) own[i] = step_scales(plan.q + 3 * i, sigma, i + 1 == plan.steps);
    }
    __syncthreads();
  }
  const int i = threadIdx.x;
  if (i < plan.steps) {
    const StepScales* sc = small ? own : plan.scales;
    const double ss = sc[i].s, sb = sc[i].b, sn = sc[i].next;
    // a zero item stays zero under any finite factors
    const double sx = i > 0 ? sc[i - 1].next : (norm > 0 ? scalbn(1.0, e) * f : 1.0);
    const double* q = plan.q + 3 * i;
    float2* out = factors + (long long)i * 3 * stride;
    out[0] = make_float2((float)(ss / sx / sx), 0.f);
    out[stride] = make_float2((float)(q[2] * (sb / ss / ss)), (float)(q[1] * (sb / ss)));
    out[2 * stride] = make_float2((float)(sn / sb / sx), (float)(q[0] * (sn / sx)));
  }
}

// An item's norm from its sum of squares: what G is multiplied by when it is stored, 2^e as two factors that stay in
// float's range (NaN for an item that cannot be normalised).
struct ItemScale {
  double norm, f;
  int e;
  float t1, t2;
  __device__ ItemScale(double sum, double eps) {
    norm = sqrt(sum);
    f = norm + eps;
    const bool usable = isfinite(sum) && f > 0;
    e = sum > 0 && usable ? 14 - ilogb(norm) : 0;
    t1 = usable ? scalbnf(1.f, e / 2) : __int_as_float(0x7fffffff);
    t2 = scalbnf(1.f, e - e / 2);
  }
};

__device__ __forceinline__ uint32_t pack_halves(__half a, __half b) {
  return (uint32_t)__half_as_ushort(a) | (uint32_t)__half_as_ushort(b) << 16;
}
__device__ __forceinline__ __half half_of(uint32_t pair, int which) { return __ushort_as_half((unsigned short)(pair >> (16 * which))); }

// One CTA or cluster per matrix, for matrices that fit; planes: halves per stored value.
bool newton_schulz_small_supported(int rows, int cols, int batch, int planes);
int launch_newton_schulz_small(const Matrices& g, const Matrices& y, int ftype, int planes, const Plan& plan, cudaStream_t stream);

}  // namespace blb200
