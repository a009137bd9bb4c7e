// What the row-wise operators (rms_norm.cu, rotary.cu) share: element types, checks of strides, the join of column sums.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <type_traits>

#include "../../include/anode_routines_gpu.h"

namespace anode_b200 {
namespace rows {

__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_trigger() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

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
  // N of them from column c on; all at once where they are aligned to 16 bytes
  template <int N> __device__ __forceinline__ void load(uint32_t c, float *f) const
  {
    static_assert(N == 4 || N == 8, "as many as 16 bytes of a type hold");
    if (!p) {
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = 1.0f;
    } else if (type == ANODE_TYPE_F32) {
#pragma unroll
      for (int i = 0; i < N; i += 4) *reinterpret_cast<float4 *>(f + i) = *reinterpret_cast<const float4 *>(static_cast<const float *>(p) + c + i);
    } else {
      uint32_t w[N / 2];
      if constexpr (N == 8) *reinterpret_cast<uint4 *>(w) = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(p) + c);
      else *reinterpret_cast<uint2 *>(w) = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(p) + c);
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        if (type == ANODE_TYPE_F16) {
          const float2 v = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
          f[2 * i] = v.x; f[2 * i + 1] = v.y;
        } else { f[2 * i] = __uint_as_float(w[i] << 16); f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
      }
    }
  }
  // N of them at any columns, those of columns below `end`, the others 0: all asked for before any is used
  template <int N> __device__ __forceinline__ void gather(const uint32_t *c, uint32_t end, float *f) const
  {
    if (!p || type == ANODE_TYPE_F32) {
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = c[i] >= end ? 0.0f : p ? static_cast<const float *>(p)[c[i]] : 1.0f;
    } else {
      uint16_t w[N];
#pragma unroll
      for (int i = 0; i < N; ++i) w[i] = c[i] < end ? static_cast<const uint16_t *>(p)[c[i]] : (uint16_t)0;
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = type == ANODE_TYPE_F16 ? __half2float(__ushort_as_half(w[i])) : __uint_as_float((uint32_t)w[i] << 16);
    }
  }
  // N of them from column c on, one by one
  template <int N> __device__ __forceinline__ void load_each(uint32_t c, float *f) const
  {
    if (!p) {
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = 1.0f;
    } else if (type == ANODE_TYPE_F32) {
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = static_cast<const float *>(p)[c + i];
    } else {
      uint16_t w[N];
#pragma unroll
      for (int i = 0; i < N; ++i) w[i] = static_cast<const uint16_t *>(p)[c + i];
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = type == ANODE_TYPE_F16 ? __half2float(__ushort_as_half(w[i])) : __uint_as_float((uint32_t)w[i] << 16);
    }
  }
  // N of them from any column c on, out of `cols`: those of 16 bytes of the vector, two by two aligned pieces shifted together
  template <int N> __device__ __forceinline__ void load_any(uint32_t c, uint32_t cols, float *f) const
  {
    const uint32_t o = c % N, first = c - o;
    if (!p || o == 0) { load<N>(c, f); return; }
    if (first + 2 * N > cols) { load_each<N>(c, f); return; }
    if (type == ANODE_TYPE_F32) {
      uint32_t w[2 * N];
#pragma unroll
      for (int i = 0; i < 2 * N; i += 4) *reinterpret_cast<uint4 *>(w + i) = *reinterpret_cast<const uint4 *>(static_cast<const float *>(p) + first + i);
#pragma unroll
      for (int b = N / 2; b > 0; b /= 2)
#pragma unroll
        for (int i = 0; i + b < 2 * N; ++i) w[i] = o & b ? w[i + b] : w[i];
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = __uint_as_float(w[i]);
    } else {
      uint32_t w[N];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint16_t *from = static_cast<const uint16_t *>(p) + first + i * N;
        if constexpr (N == 8) *reinterpret_cast<uint4 *>(w + 4 * i) = *reinterpret_cast<const uint4 *>(from);
        else *reinterpret_cast<uint2 *>(w + 2 * i) = *reinterpret_cast<const uint2 *>(from);
      }
#pragma unroll
      for (int b = N / 2; b > 1; b /= 2)
#pragma unroll
        for (int i = 0; i + b / 2 < N; ++i) w[i] = o & b ? w[i + b / 2] : w[i];
      const uint32_t by = o & 1 ? 0x5432u : 0x3210u;
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        const uint32_t v = __byte_perm(w[i], w[i + 1], by);
        if (type == ANODE_TYPE_F16) {
          const float2 x = __half22float2(*reinterpret_cast<const __half2 *>(&v));
          f[2 * i] = x.x; f[2 * i + 1] = x.y;
        } else { f[2 * i] = __uint_as_float(v << 16); f[2 * i + 1] = __uint_as_float(v & 0xffff0000u); }
      }
    }
  }
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

// Copies into shared memory that a thread waits for itself
template <int BYTES> __device__ __forceinline__ void copy_async(void *to, const void *from)
{
  const uint32_t at = (uint32_t)__cvta_generic_to_shared(to);
  if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at), "l"(from) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(at), "l"(from), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }

// Two floats at a time, in one instruction each
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c)
{
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(reinterpret_cast<unsigned long long &>(d))
      : "l"(reinterpret_cast<unsigned long long &>(a)), "l"(reinterpret_cast<unsigned long long &>(b)), "l"(reinterpret_cast<unsigned long long &>(c)));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b)
{
  float2 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<unsigned long long &>(d))
      : "l"(reinterpret_cast<unsigned long long &>(a)), "l"(reinterpret_cast<unsigned long long &>(b)));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b)
{
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<unsigned long long &>(d))
      : "l"(reinterpret_cast<unsigned long long &>(a)), "l"(reinterpret_cast<unsigned long long &>(b)));
  return d;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// 16 bytes of an array: V elements
template <typename T> struct Vec {
  static constexpr int V = 16 / sizeof(T);
  uint4 bits;
  __device__ __forceinline__ static Vec load(const T *p) { return Vec{*reinterpret_cast<const uint4 *>(p)}; }
  __device__ __forceinline__ void store(T *p) const { *reinterpret_cast<uint4 *>(p) = bits; }
  __device__ __forceinline__ uint32_t word(int i) const { return i == 0 ? bits.x : i == 1 ? bits.y : i == 2 ? bits.z : bits.w; }
  __device__ __forceinline__ void floats(float *f) const
  {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w = word(i);
      if constexpr (sizeof(T) == 4) f[i] = __uint_as_float(w);
      else if constexpr (std::is_same<T, __half>::value) {
        const float2 v = __half22float2(*reinterpret_cast<const __half2 *>(&w));
        f[2 * i] = v.x; f[2 * i + 1] = v.y;
      } else { f[2 * i] = __uint_as_float(w << 16); f[2 * i + 1] = __uint_as_float(w & 0xffff0000u); }
    }
  }
  __device__ __forceinline__ static Vec of(const float *f)
  {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(f[i]);
      else if constexpr (std::is_same<T, __half>::value) { const __half2 v = __floats2half2_rn(f[2 * i], f[2 * i + 1]); w[i] = *reinterpret_cast<const uint32_t *>(&v); }
      else { const __nv_bfloat162 v = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]); w[i] = *reinterpret_cast<const uint32_t *>(&v); }
    }
    return Vec{make_uint4(w[0], w[1], w[2], w[3])};
  }
};

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
// The same of a team: a power of two of a warp's lanes, or a block
__device__ __forceinline__ float team_sum_all(float v, uint32_t team, float *buf)
{
  if (team > 32) return block_sum_all(v, buf);
  for (uint32_t o = team / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

inline bool known_type(int t) { return t == ANODE_TYPE_F32 || t == ANODE_TYPE_F16 || t == ANODE_TYPE_BF16; }
inline size_t type_bytes(int t) { return t == ANODE_TYPE_F32 ? 4 : 2; }
inline bool aligned_to(const void *p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

// f(T()) for the element type of a checked code
template <typename F> inline int by_type(int type, F f)
{
  return type == ANODE_TYPE_F32 ? f(float()) : type == ANODE_TYPE_F16 ? f(__half()) : f(__nv_bfloat16());
}

// A kernel's leave to use more shared memory than 48 KB (its own arrays, of a few KB here, among them), asked for once per device and for all that
// a block may have
class SharedMemory {
 public:
  bool up_to(const void *kernel, size_t bytes)
  {
    if (bytes <= 40 * 1024) return true;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
    if (done_.load(std::memory_order_relaxed) >> dev & 1) return true;
    cudaFuncAttributes f;
    if (cudaFuncGetAttributes(&f, kernel) != cudaSuccess ||
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024 - (int)f.sharedSizeBytes) != cudaSuccess) {
      (void)cudaGetLastError();
      return false;
    }
    done_.fetch_or(1ull << dev, std::memory_order_relaxed);
    return true;
  }

 private:
  std::atomic<uint64_t> done_{0};
};

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
