// Shared by the 8-bit product, its quantiser and the Newton-Schulz orthogonalisation: the floating
// storage types and the layout rules of their operands.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace blb200 {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

inline bool valid_ftype(int t) { return t == BLB200_F32 || t == BLB200_F16 || t == BLB200_BF16; }
inline int ftype_bytes(int t) { return t == BLB200_F32 ? 4 : 2; }

// Calls f with a value of the storage type (its value is unused).
template <typename F>
int with_ftype(int t, F&& f) {
  if (t == BLB200_F32) return f(float{});
  if (t == BLB200_F16) return f(__half{});
  return f(__nv_bfloat16{});
}

// Largest dimension of these calls: coordinates and loop counters past it may reach the end of 32 bits.
constexpr int kMaxDim = 1 << 30;

// ld and stride of a column-major operand that is read: items may overlap or coincide.
inline bool readable_layout(long long rows, long long ld, long long stride) {
  return ld >= (rows > 1 ? rows : 1) && stride >= 0;
}
// ... of one that is written: no element may belong to two columns or two items.  Items lie one after the
// other, or are interleaved inside the leading dimension.
inline bool writable_layout(long long rows, long long cols, long long batch, long long ld, long long stride) {
  if (!readable_layout(rows, ld, stride)) return false;
  if (batch <= 1 || rows == 0 || cols == 0) return true;
  return stride >= (cols - 1) * ld + rows || (stride >= rows && ld >= (batch - 1) * stride + rows);
}

// Launch configuration that lets a kernel's start overlap the end of the kernel before it in the stream.  Such a kernel
// calls griddep_wait() before it touches global memory; griddep_launch() lets its own successor start likewise.
struct OverlappedLaunch {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  OverlappedLaunch(dim3 grid, dim3 block, cudaStream_t stream) {
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
  }
  OverlappedLaunch(const OverlappedLaunch&) = delete;
};
__device__ __forceinline__ void griddep_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void griddep_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

}  // namespace blb200
