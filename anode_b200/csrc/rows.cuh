// What the row-wise operators (rms_norm.cu, layer_norm.cu, rotary.cu, embed.cu, log_probs.cu) share: element types, checks of strides, the join of column sums.
// Each has a namespace of its own in this one: their plans and helpers are alike and have the same names, but not the same members and values.
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

inline uint32_t row_blocks(uint64_t rows) { return (uint32_t)(rows < (1u << 30) ? rows : (1u << 30)); }

// Columns are counted in 32 bits, up to a block's threads beyond the last one
inline bool served(uint64_t rows, uint32_t cols) { return cols != 0 && !(cols >> 31) && !(rows >> 36); }

// An array of rows: a pointer of the type's alignment; an output's rows do not overlap
inline int check_rows(const void *p, size_t bytes, uint64_t rows, uint32_t cols, uint64_t stride, bool output)
{
  if (!p) return ANODE_E_NULL;
  if (!aligned_to(p, bytes)) return ANODE_E_ALIGN;
  if (output && rows > 1 && stride < cols) return ANODE_E_STRIDE;
  return ANODE_OK;
}
// An output in an input's place has its strides
inline bool apart(const void *out, uint64_t out_stride, const void *in, uint64_t in_stride, uint64_t rows)
{
  return out != in || out_stride == in_stride || rows <= 1;
}

// Whether n bytes from p on and m bytes from q on have one in common; what is not there has none
inline bool overlap(const void *p, uint64_t n, const void *q, uint64_t m) { return p && q && (uintptr_t)p < (uintptr_t)q + m && (uintptr_t)q < (uintptr_t)p + n; }

// Whether two arrays of rows, n of p_len bytes p_step apart and m of q_len bytes q_step apart, have a byte in common
inline bool rows_meet(const void *p, uint64_t p_step, uint64_t n, uint64_t p_len, const void *q, uint64_t q_step, uint64_t m, uint64_t q_len)
{
  if (!n || !m || !overlap(p, (n - 1) * p_step + p_len, q, (m - 1) * q_step + q_len)) return false;
  if (n > m) return rows_meet(q, q_step, m, q_len, p, p_step, n, p_len);
  const uint64_t a = (uintptr_t)p, b = (uintptr_t)q;
  // of q's rows the last that begins before p's row ends reaches farthest
  auto meets = [&](uint64_t i) {
    const uint64_t first = a + i * p_step, end = first + p_len;
    if (end <= b) return false;
    const uint64_t j = q_step ? (end - 1 - b) / q_step : 0;
    return b + (j < m ? j : m - 1) * q_step + q_len > first;
  };
  // at one distance p's rows all lie at the same place among q's, but for those before q's first row or behind its last: the first that ends behind q's first byte
  // tells (overlapping rows, as those of a broadcast, are looked at one by one, and so are those at two distances)
  if (p_step == q_step && p_step >= p_len && p_step >= q_len) return meets(a + p_len > b ? 0 : (b - a - p_len) / p_step + 1);
  for (uint64_t i = 0; i < n; ++i) if (meets(i)) return true;
  return false;
}

// Whether an array's rows all begin at the same place of a slot of `v` elements as those of the first one
inline bool in_step(const void *p, size_t bytes, uint64_t stride, uint32_t v, const void *p0, size_t bytes0, uint64_t stride0, uint64_t rows)
{
  return !p || ((uintptr_t)p / bytes % v == (uintptr_t)p0 / bytes0 % v && (rows <= 1 || stride % v == stride0 % v));
}

#define TRY(call) do { const int rc_ = (call); if (rc_) return rc_; } while (0)

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

// A kernel's leave to be launched in clusters of more than 8 blocks, asked for once per device
class WideClusters {
 public:
  bool of(const void *kernel)
  {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
    if (done_.load(std::memory_order_relaxed) >> dev & 1) return true;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) { (void)cudaGetLastError(); return false; }
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
// The same of a grid of clusters, of up to 8 blocks or as many as the kernel has leave for
template <typename... P, typename... A>
inline int launch_in_clusters(void (*kernel)(P...), dim3 grid, uint32_t cluster, uint32_t threads, size_t shared, cudaStream_t stream, A... args)
{
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid; cfg.blockDim = dim3(threads); cfg.dynamicSmemBytes = shared; cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr; cfg.numAttrs = 2;
  if (cudaLaunchKernelEx(&cfg, kernel, P(args)...) != cudaSuccess) { (void)cudaGetLastError(); return ANODE_E_LAUNCH; }
  return ANODE_OK;
}

// Of a cluster: this block's place in it, a barrier that also orders what was written, and another block's shared memory
__device__ __forceinline__ uint32_t cluster_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void cluster_sync()
{
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t peer_address(const void *p, uint32_t rank)
{
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
  return remote;
}
__device__ __forceinline__ uint32_t peer_load(const uint32_t *p, uint32_t rank)
{
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(peer_address(p, rank)) : "memory");
  return v;
}

// A token as a row of a table or a column of logits, or `vocab` for one outside of them
__device__ __forceinline__ uint32_t token_at(const void *p, int bytes, uint64_t i, uint32_t vocab)
{
  const uint64_t t = bytes == 8 ? static_cast<const uint64_t *>(p)[i] : (uint64_t)(int64_t)static_cast<const int32_t *>(p)[i];
  return t < vocab ? (uint32_t)t : vocab;
}

}  // namespace rows
}  // namespace anode_b200
