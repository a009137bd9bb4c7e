// What the row-wise operators (rms_norm.cu, rotary.cu) share: element types, checks of strides, the join of column sums.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/anode_routines_gpu.h"

namespace anode_b200 {
namespace rows {

__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// A vector of weights (or its gradient) of any of the three types; NULL reads as ones.
struct Weights {
  const void *p;
  int type;
  __device__ __forceinline__ float at(uint32_t i) const
  {
    if (!p) return 1.0f;
    return type == ANODE_TYPE_F32 ? static_cast<const float *>(p)[i]
         : type == ANODE_TYPE_F16 ? to_float(static_cast<const __half *>(p)[i]) : to_float(static_cast<const __nv_bfloat16 *>(p)[i]);
  }
};
__device__ __forceinline__ void put_weight(void *p, int type, uint32_t i, float v)
{
  if (type == ANODE_TYPE_F32) static_cast<float *>(p)[i] = v;
  else if (type == ANODE_TYPE_F16) static_cast<__half *>(p)[i] = from_float<__half>(v);
  else static_cast<__nv_bfloat16 *>(p)[i] = from_float<__nv_bfloat16>(v);
}

__device__ __forceinline__ float warp_sum_all(float v)
{
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sum over a block of up to 32 warps in a fixed order, in every thread.  `buf`: 32 floats that no one reads any more.
__device__ __forceinline__ float block_sum_all(float v, float *buf)
{
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  v = warp_sum_all(v);
  if (lane == 0) buf[warp] = v;
  __syncthreads();
  v = lane < warps ? buf[lane] : 0.0f;
  return warp_sum_all(v);
}

inline bool known_type(int t) { return t == ANODE_TYPE_F32 || t == ANODE_TYPE_F16 || t == ANODE_TYPE_BF16; }
inline size_t type_bytes(int t) { return t == ANODE_TYPE_F32 ? 4 : 2; }
inline bool aligned_to(const void *p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

// f(T()) for the element type of a checked code
template <typename F> inline int by_type(int type, F f)
{
  return type == ANODE_TYPE_F32 ? f(float()) : type == ANODE_TYPE_F16 ? f(__half()) : f(__nv_bfloat16());
}

// A launch that may overlap the tail of the kernel before it on the stream: every kernel here waits for that one's results
// before it touches memory.
template <typename... P, typename... A>
inline int launch(void (*kernel)(P...), dim3 grid, uint32_t threads, size_t shared, cudaStream_t stream, A... args)
{
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid; cfg.blockDim = dim3(threads); cfg.dynamicSmemBytes = shared; cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr; cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kernel, P(args)...) != cudaSuccess) { (void)cudaGetLastError(); return ANODE_E_LAUNCH; }
  return ANODE_OK;
}

}  // namespace rows
}  // namespace anode_b200
