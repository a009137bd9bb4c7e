// RMS norm over rows with the residual's addition: forward, adjoint, and the forward pass with an output in 8 bits.
//
//   t = round(x + residual),  r = (mean(t^2) + epsilon)^-1/2,  y = t*r*gamma
//   dx = r*(g - xh*mean(g*xh)) + dt,   g = dy*gamma, xh = t*r,   dgamma = sum over rows of dy*xh
//   a = max |y| of a group, scale = max(a, 2^-96)/448, q = e4m3(y/scale)
//
// A block has a row at a time; statistics and sums are f32.
#include <cuda_fp8.h>

#include "bn_host.h"
#include "rows.cuh"

namespace anode_b200 {
namespace rows {

constexpr uint32_t kThreads = 256;
constexpr float kTiny = 0x1p-96f, kE4M3 = 448.0f;

struct NormArgs {
  uint64_t rows;
  uint32_t cols;
  float epsilon, inv_cols;
  const void *x, *residual;
  uint64_t x_stride, residual_stride;
  Weights gamma;
  void *y, *total;
  uint64_t y_stride, total_stride;
  float *inv_rms;
  // in 8 bits
  uint32_t block;                      // columns of a group (the whole row: cols)
  float *scale;
  uint64_t scale_row, scale_group;
};

// x + residual as it is stored
template <typename T> __device__ __forceinline__ float sum_at(const NormArgs &a, uint64_t row, uint32_t c)
{
  const float x = to_float(static_cast<const T *>(a.x)[row * a.x_stride + c]);
  if (!a.residual) return x;
  return to_float(from_float<T>(x + to_float(static_cast<const T *>(a.residual)[row * a.residual_stride + c])));
}

template <typename T, bool QUANT> __global__ void __launch_bounds__(kThreads) rms_norm_rows_kernel(const NormArgs a)
{
  __shared__ float buf[2][32];
  pdl_wait();
  for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    float sq = 0.0f;
    T *total = a.total ? static_cast<T *>(a.total) + row * a.total_stride : nullptr;
    for (uint32_t c = threadIdx.x; c < a.cols; c += kThreads) {
      const float t = sum_at<T>(a, row, c);
      if (total) total[c] = from_float<T>(t);
      sq = fmaf(t, t, sq);
    }
    const float r = 1.0f / sqrtf(block_sum_all(sq, buf[0]) * a.inv_cols + a.epsilon);
    if (a.inv_rms && threadIdx.x == 0) a.inv_rms[row] = r;
    // (the sum again: from where it was stored, which may be the residual's place)
    auto value = [&](uint32_t c) { return (total ? to_float(total[c]) : sum_at<T>(a, row, c)) * r * a.gamma.at(c); };
    if (!QUANT) {
      for (uint32_t c = threadIdx.x; c < a.cols; c += kThreads) static_cast<T *>(a.y)[row * a.y_stride + c] = from_float<T>(value(c));
    } else {
      // a warp per group; bits of |y| in the order of unsigned numbers, a NaN's above all
      uint8_t *q = static_cast<uint8_t *>(a.y) + row * a.y_stride;
      const bool whole = a.block == a.cols;
      const uint32_t lane = whole ? threadIdx.x : threadIdx.x & 31, lanes = whole ? kThreads : 32, warp = threadIdx.x >> 5;
      __syncthreads();       // (the sum is stored by other threads than read it here)
      for (uint64_t base = whole ? 0 : (uint64_t)warp * a.block, group = whole ? 0 : warp; base < a.cols;
           base += (uint64_t)a.block * (kThreads / 32), group += kThreads / 32) {
        const uint32_t end = (uint32_t)(base + a.block < a.cols ? base + a.block : a.cols);
        uint32_t top = 0;
        for (uint32_t c = (uint32_t)base + lane; c < end; c += lanes) top = max(top, __float_as_uint(value(c)) & 0x7fffffffu);
        top = __reduce_max_sync(0xffffffffu, top);
        if (whole) {
          if ((threadIdx.x & 31) == 0) buf[1][warp] = __uint_as_float(top);
          __syncthreads();
          for (uint32_t w = 0; w < kThreads / 32; ++w) top = max(top, __float_as_uint(buf[1][w]));
        }
        const float scale = __uint_as_float(max(top, __float_as_uint(kTiny))) / kE4M3, inv = 1.0f / scale;
        if (lane == 0) a.scale[row * a.scale_row + group * a.scale_group] = scale;
        for (uint32_t c = (uint32_t)base + lane; c < end; c += lanes) q[c] = __nv_cvt_float_to_fp8(value(c) * inv, __NV_SATFINITE, __NV_E4M3);
        if (whole) break;
      }
    }
    __syncthreads();
  }
}

struct GradArgs {
  uint64_t rows;
  uint32_t cols;
  float inv_cols;
  const void *dy, *total, *dtotal;
  uint64_t dy_stride, total_stride, dtotal_stride;
  const float *inv_rms;
  Weights gamma;
  void *dx;
  uint64_t dx_stride;
  void *dgamma;
  float *partial;
  uint32_t parts;
};

// dgamma's partial sums: a thread has a column and every `parts`-th row; ahead of the kernel below, whose dx may be dy
template <typename T> __global__ void __launch_bounds__(kThreads) rms_norm_dgamma_kernel(const GradArgs a)
{
  pdl_wait();
  const uint64_t c = (uint64_t)blockIdx.x * kThreads + threadIdx.x;
  if (c >= a.cols) return;
  float sum = 0.0f;
  for (uint64_t row = blockIdx.y; row < a.rows; row += a.parts)
    sum += to_float(static_cast<const T *>(a.dy)[row * a.dy_stride + c]) *
           (to_float(static_cast<const T *>(a.total)[row * a.total_stride + c]) * a.inv_rms[row]);
  a.partial[(uint64_t)blockIdx.y * a.cols + c] = sum;
}

__global__ void __launch_bounds__(kThreads) join_columns_kernel(uint32_t cols, uint32_t parts, const float *partial, void *out, int type)
{
  pdl_wait();
  const uint64_t c = (uint64_t)blockIdx.x * kThreads + threadIdx.x;
  if (c >= cols) return;
  float sum = 0.0f;
  for (uint32_t p = 0; p < parts; ++p) sum += partial[(uint64_t)p * cols + c];
  put_weight(out, type, (uint32_t)c, sum);
}

template <typename T> __global__ void __launch_bounds__(kThreads) rms_norm_dx_kernel(const GradArgs a)
{
  __shared__ float buf[32];
  pdl_wait();
  for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T *dy = static_cast<const T *>(a.dy) + row * a.dy_stride, *t = static_cast<const T *>(a.total) + row * a.total_stride;
    const T *dt = a.dtotal ? static_cast<const T *>(a.dtotal) + row * a.dtotal_stride : nullptr;
    T *dx = static_cast<T *>(a.dx) + row * a.dx_stride;
    const float r = a.inv_rms[row];
    float dot = 0.0f;
    for (uint32_t c = threadIdx.x; c < a.cols; c += kThreads) dot = fmaf(to_float(dy[c]) * a.gamma.at(c), to_float(t[c]) * r, dot);
    dot = block_sum_all(dot, buf) * a.inv_cols;
    for (uint32_t c = threadIdx.x; c < a.cols; c += kThreads) {
      const float xh = to_float(t[c]) * r, v = r * (to_float(dy[c]) * a.gamma.at(c) - xh * dot);
      dx[c] = from_float<T>(dt ? v + to_float(dt[c]) : v);
    }
    __syncthreads();
  }
}

inline uint32_t parts_of(uint64_t rows) { return (uint32_t)(rows < 64 ? (rows ? rows : 1) : 64); }
inline uint32_t row_blocks(uint64_t rows) { return (uint32_t)(rows < (1u << 30) ? rows : (1u << 30)); }

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

#define TRY(call) do { const int rc_ = (call); if (rc_) return rc_; } while (0)

int norm_forward(const NormArgs &a, int type, int gamma_type, bool quant, cudaStream_t stream)
{
  if (!known_type(type) || (a.gamma.p && !known_type(gamma_type))) return ANODE_E_TYPE;
  if (a.cols == 0 || a.rows >> 40) return ANODE_E_DIMS;
  if (a.rows == 0) return ANODE_OK;
  const size_t e = type_bytes(type);
  TRY(check_rows(a.x, e, a.rows, a.cols, a.x_stride, false));
  if (a.residual) TRY(check_rows(a.residual, e, a.rows, a.cols, a.residual_stride, false));
  if (a.gamma.p && !aligned_to(a.gamma.p, type_bytes(gamma_type))) return ANODE_E_ALIGN;
  TRY(check_rows(a.y, quant ? 1 : e, a.rows, a.cols, a.y_stride, true));
  if (a.total) {
    if (!a.residual) return ANODE_E_NULL;
    TRY(check_rows(a.total, e, a.rows, a.cols, a.total_stride, true));
    if (a.total == a.y || !apart(a.total, a.total_stride, a.x, a.x_stride, a.rows) ||
        !apart(a.total, a.total_stride, a.residual, a.residual_stride, a.rows)) return ANODE_E_STRIDE;
  }
  if (quant) { if (a.y == a.x || a.y == a.residual) return ANODE_E_STRIDE; }
  else if (!apart(a.y, a.y_stride, a.x, a.x_stride, a.rows) || !apart(a.y, a.y_stride, a.residual, a.residual_stride, a.rows)) return ANODE_E_STRIDE;
  if (a.inv_rms && !aligned_to(a.inv_rms, 4)) return ANODE_E_ALIGN;
  return by_type(type, [&](auto t) {
    using T = decltype(t);
    return quant ? launch(rms_norm_rows_kernel<T, true>, dim3(row_blocks(a.rows)), kThreads, 0, stream, a)
                 : launch(rms_norm_rows_kernel<T, false>, dim3(row_blocks(a.rows)), kThreads, 0, stream, a);
  });
}

}  // namespace rows
}  // namespace anode_b200

using namespace anode_b200::rows;

extern "C" int anode_gpu_rms_norm_add_fwd(
    int type, uint64_t rows, uint32_t cols, float epsilon,
    const void *x, uint64_t x_stride, const void *residual, uint64_t residual_stride,
    const void *gamma, int gamma_type,
    void *y, uint64_t y_stride, void *total, uint64_t total_stride, float *inv_rms,
    const struct KernelConfig *cfg, struct CUstream_st *stream)
{
  (void)cfg;
  NormArgs a = {rows, cols, epsilon, 1.0f / (float)cols, x, residual, x_stride, residual_stride, {gamma, gamma_type}, y, total, y_stride,
                total_stride, inv_rms, 0, nullptr, 0, 0};
  return norm_forward(a, type, gamma_type, false, stream);
}

extern "C" int anode_gpu_rms_norm_add_quant_fwd(
    int type, uint64_t rows, uint32_t cols, float epsilon, uint32_t block,
    const void *x, uint64_t x_stride, const void *residual, uint64_t residual_stride,
    const void *gamma, int gamma_type,
    uint8_t *q, uint64_t q_stride, float *scale, uint64_t scale_row_stride, uint64_t scale_group_stride,
    void *total, uint64_t total_stride,
    const struct KernelConfig *cfg, struct CUstream_st *stream)
{
  (void)cfg;
  if (block != 0 && block != 128) return ANODE_E_DIMS;
  if (rows && !scale) return ANODE_E_NULL;
  if (!aligned_to(scale, 4)) return ANODE_E_ALIGN;
  // no two scales in one place
  const uint64_t groups = block ? ((uint64_t)cols + block - 1) / block : 1;
  const bool many = rows > 1, wide = groups > 1;
  if ((many && !scale_row_stride) || (wide && !scale_group_stride) ||
      (many && wide && scale_row_stride < groups * scale_group_stride && scale_group_stride < rows * scale_row_stride)) return ANODE_E_STRIDE;
  NormArgs a = {rows, cols, epsilon, 1.0f / (float)cols, x, residual, x_stride, residual_stride, {gamma, gamma_type}, q, total, q_stride,
                total_stride, nullptr, block ? block : cols, scale, scale_row_stride, scale_group_stride};
  return norm_forward(a, type, gamma_type, true, stream);
}

extern "C" size_t anode_gpu_rms_norm_add_bwd_workspace_bytes(uint64_t rows, uint32_t cols) { return (size_t)parts_of(rows) * cols * 4; }

extern "C" int anode_gpu_rms_norm_add_bwd(
    int type, uint64_t rows, uint32_t cols,
    const void *dy, uint64_t dy_stride, const void *total, uint64_t total_stride, const float *inv_rms,
    const void *gamma, int gamma_type, const void *dtotal, uint64_t dtotal_stride,
    void *dx, uint64_t dx_stride, void *dgamma, void *workspace, size_t workspace_bytes,
    const struct KernelConfig *cfg, struct CUstream_st *stream)
{
  (void)cfg;
  if (!known_type(type) || ((gamma || dgamma) && !known_type(gamma_type))) return ANODE_E_TYPE;
  if (cols == 0 || rows >> 40) return ANODE_E_DIMS;
  if (gamma && !aligned_to(gamma, type_bytes(gamma_type))) return ANODE_E_ALIGN;
  if (dgamma) {
    if (!aligned_to(dgamma, type_bytes(gamma_type))) return ANODE_E_ALIGN;
    if (rows == 0) return cudaMemsetAsync(dgamma, 0, type_bytes(gamma_type) * cols, stream) == cudaSuccess ? ANODE_OK : ANODE_E_LAUNCH;
    if (!workspace || !aligned_to(workspace, 16) || workspace_bytes < anode_gpu_rms_norm_add_bwd_workspace_bytes(rows, cols)) return ANODE_E_WORKSPACE;
  }
  if (rows == 0) return ANODE_OK;
  const size_t e = type_bytes(type);
  TRY(check_rows(dy, e, rows, cols, dy_stride, false));
  TRY(check_rows(total, e, rows, cols, total_stride, false));
  if (dtotal) TRY(check_rows(dtotal, e, rows, cols, dtotal_stride, false));
  TRY(check_rows(dx, e, rows, cols, dx_stride, true));
  if (!inv_rms) return ANODE_E_NULL;
  if (!aligned_to(inv_rms, 4)) return ANODE_E_ALIGN;
  if (!apart(dx, dx_stride, dy, dy_stride, rows) || !apart(dx, dx_stride, total, total_stride, rows) || !apart(dx, dx_stride, dtotal, dtotal_stride, rows))
    return ANODE_E_STRIDE;
  GradArgs a = {rows, cols, 1.0f / (float)cols, dy, total, dtotal, dy_stride, total_stride, dtotal_stride, inv_rms, {gamma, gamma_type},
                dx, dx_stride, dgamma, static_cast<float *>(workspace), parts_of(rows)};
  const uint32_t wide = (uint32_t)(((uint64_t)cols + kThreads - 1) / kThreads);
  return by_type(type, [&](auto t) {
    using T = decltype(t);
    if (dgamma) {
      TRY(launch(rms_norm_dgamma_kernel<T>, dim3(wide, a.parts), kThreads, 0, stream, a));
      TRY(launch(join_columns_kernel, dim3(wide), kThreads, 0, stream, cols, a.parts, a.partial, dgamma, gamma_type));
    }
    return launch(rms_norm_dx_kernel<T>, dim3(row_blocks(rows)), kThreads, 0, stream, a);
  });
}
