// Layer norm over rows with the residual's addition: forward and adjoint.
//
//   t = round(x + residual),  mu = mean(t),  r = (mean((t - mu)^2) + epsilon)^-1/2,  y = (t - mu)*r*gamma + beta
//   dx = r*(g - mean(g) - xh*mean(g*xh)) + dt,   g = dy*gamma, xh = (t - mu)*r
//   dgamma = sum over rows of dy*xh,  dbeta = sum over rows of dy
//
// Statistics and sums are f32; the squares are those of the values less their mean, so that a row far from zero keeps its spread.
// y, total and dx are rounded once, total before the norm reads it.
#include "bn_host.h"
#include "rows.cuh"

namespace anode_b200 {
namespace rows {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kMostParts = 148;       // of the sums over rows

struct LayerArgs {
  uint64_t rows;
  uint32_t cols;
  float epsilon, inv_cols;
  const void *x, *residual;
  uint64_t x_stride, residual_stride;
  Weights gamma, beta;
  void *y, *total;
  uint64_t y_stride, total_stride;
  float *mean, *inv_std;
};

// x + residual as it is stored
template <typename T> __device__ __forceinline__ float sum_at(const LayerArgs &a, uint64_t row, uint32_t c)
{
  const float x = to_float(static_cast<const T *>(a.x)[row * a.x_stride + c]);
  if (!a.residual) return x;
  return to_float(from_float<T>(x + to_float(static_cast<const T *>(a.residual)[row * a.residual_stride + c])));
}

// Any rows: a block has a row at a time, element by element, and reads it three times
template <typename T> __global__ void __launch_bounds__(kThreads) layer_norm_rows_kernel(const LayerArgs a)
{
  __shared__ float buf[2][32];
  pdl_wait();
  for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    float sum = 0.0f, sq = 0.0f;
    T *total = a.total ? static_cast<T *>(a.total) + row * a.total_stride : nullptr;
    for (uint32_t c = threadIdx.x; c < a.cols; c += kThreads) {
      const float t = sum_at<T>(a, row, c);
      if (total) total[c] = from_float<T>(t);
      sum += t;
    }
    // (the sum again: from where it was stored, which may be the residual's place)
    auto value = [&](uint32_t c) { return total ? to_float(total[c]) : sum_at<T>(a, row, c); };
    const float mean = block_sum_all(sum, buf[0]) * a.inv_cols;
    for (uint32_t c = threadIdx.x; c < a.cols; c += kThreads) {
      const float d = value(c) - mean;
      sq = fmaf(d, d, sq);
    }
    const float r = 1.0f / sqrtf(block_sum_all(sq, buf[1]) * a.inv_cols + a.epsilon);
    if (threadIdx.x == 0) {
      if (a.mean) a.mean[row] = mean;
      if (a.inv_std) a.inv_std[row] = r;
    }
    T *y = static_cast<T *>(a.y) + row * a.y_stride;
    for (uint32_t c = threadIdx.x; c < a.cols; c += kThreads) y[c] = from_float<T>(fmaf((value(c) - mean) * r, a.gamma.at(c), a.beta.p ? a.beta.at(c) : 0.0f));
    __syncthreads();
  }
}

struct LayerGradArgs {
  uint64_t rows;
  uint32_t cols;
  float inv_cols;
  const void *dy, *total, *dtotal;
  uint64_t dy_stride, total_stride, dtotal_stride;
  const float *mean, *inv_std;
  Weights gamma;
  void *dx;
  uint64_t dx_stride;
  void *dgamma, *dbeta;
  int dweight_type;
  float *partial;                      // [parts][2][cols]: dgamma's sums, dbeta's
  uint32_t parts;
};

// Any rows: the weights' partial sums, a thread has a column and every `parts`-th row
template <typename T> __global__ void __launch_bounds__(kThreads) layer_norm_dweights_kernel(const LayerGradArgs a)
{
  pdl_wait();
  const uint64_t c = (uint64_t)blockIdx.x * kThreads + threadIdx.x;
  if (c >= a.cols) return;
  float dg = 0.0f, db = 0.0f;
  for (uint64_t row = blockIdx.y; row < a.rows; row += a.parts) {
    const float dy = to_float(static_cast<const T *>(a.dy)[row * a.dy_stride + c]);
    dg = fmaf(dy, (to_float(static_cast<const T *>(a.total)[row * a.total_stride + c]) - a.mean[row]) * a.inv_std[row], dg);
    db += dy;
  }
  a.partial[(uint64_t)blockIdx.y * 2 * a.cols + c] = dg;
  a.partial[((uint64_t)blockIdx.y * 2 + 1) * a.cols + c] = db;
}

// The parts' sums: a lane has a column of dgamma (blockIdx.y = 0) or dbeta, a warp every eighth part, all of which are asked for at once
__global__ void __launch_bounds__(kThreads) join_weights_kernel(uint32_t cols, uint32_t parts, const float *partial, void *dgamma, void *dbeta, int type)
{
  constexpr uint32_t kWarps = kThreads / 32, kEach = (kMostParts + kWarps - 1) / kWarps;
  __shared__ float sums[kWarps][33];
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint64_t c = (uint64_t)blockIdx.x * 32 + lane;
  void *out = blockIdx.y ? dbeta : dgamma;
  pdl_wait();
  if (!out) return;
  float v[kEach], sum = 0.0f;
#pragma unroll
  for (uint32_t i = 0; i < kEach; ++i)
    v[i] = c < cols && warp + kWarps * i < parts ? partial[((uint64_t)(warp + kWarps * i) * 2 + blockIdx.y) * cols + c] : 0.0f;
#pragma unroll
  for (uint32_t i = 0; i < kEach; ++i) sum += v[i];
  sums[warp][lane] = sum;
  __syncthreads();
  if (warp || c >= cols) return;
#pragma unroll
  for (uint32_t w = 1; w < kWarps; ++w) sum += sums[w][lane];
  put_weight(out, type, (uint32_t)c, sum);
}

template <typename T> __global__ void __launch_bounds__(kThreads) layer_norm_dx_kernel(const LayerGradArgs a)
{
  __shared__ float buf[2][32];
  pdl_wait();
  for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T *dy = static_cast<const T *>(a.dy) + row * a.dy_stride, *t = static_cast<const T *>(a.total) + row * a.total_stride;
    const T *dt = a.dtotal ? static_cast<const T *>(a.dtotal) + row * a.dtotal_stride : nullptr;
    T *dx = static_cast<T *>(a.dx) + row * a.dx_stride;
    const float mu = a.mean[row], r = a.inv_std[row];
    float sum = 0.0f, dot = 0.0f;
    for (uint32_t c = threadIdx.x; c < a.cols; c += kThreads) {
      const float g = to_float(dy[c]) * a.gamma.at(c);
      sum += g;
      dot = fmaf(g, (to_float(t[c]) - mu) * r, dot);
    }
    sum = block_sum_all(sum, buf[0]) * a.inv_cols;
    dot = block_sum_all(dot, buf[1]) * a.inv_cols;
    for (uint32_t c = threadIdx.x; c < a.cols; c += kThreads) {
      const float xh = (to_float(t[c]) - mu) * r, v = r * (to_float(dy[c]) * a.gamma.at(c) - sum - xh * dot);
      dx[c] = from_float<T>(dt ? v + to_float(dt[c]) : v);
    }
    __syncthreads();
  }
}

inline uint32_t parts_of(uint64_t rows) { return (uint32_t)(rows < kMostParts ? (rows ? rows : 1) : kMostParts); }

}  // namespace rows
}  // namespace anode_b200

using namespace anode_b200::rows;

extern "C" int anode_gpu_layer_norm_add_fwd(
    int type, uint64_t rows, uint32_t cols, float epsilon,
    const void *x, uint64_t x_stride, const void *residual, uint64_t residual_stride,
    const void *gamma, const void *beta, int weight_type,
    void *y, uint64_t y_stride, void *total, uint64_t total_stride, float *mean, float *inv_std,
    const struct KernelConfig *cfg, struct CUstream_st *stream)
{
  (void)cfg;
  if (!known_type(type) || ((gamma || beta) && !known_type(weight_type))) return ANODE_E_TYPE;
  if (!served(rows, cols)) return ANODE_E_DIMS;
  if (rows == 0) return ANODE_OK;
  const size_t e = type_bytes(type);
  TRY(check_rows(x, e, rows, cols, x_stride, false));
  if (residual) TRY(check_rows(residual, e, rows, cols, residual_stride, false));
  for (const void *w : {gamma, beta}) if (w && !aligned_to(w, type_bytes(weight_type))) return ANODE_E_ALIGN;
  TRY(check_rows(y, e, rows, cols, y_stride, true));
  if (total) {
    if (!residual) return ANODE_E_NULL;
    TRY(check_rows(total, e, rows, cols, total_stride, true));
    if (total == y || !apart(total, total_stride, x, x_stride, rows) || !apart(total, total_stride, residual, residual_stride, rows)) return ANODE_E_STRIDE;
  }
  if (!apart(y, y_stride, x, x_stride, rows) || !apart(y, y_stride, residual, residual_stride, rows)) return ANODE_E_STRIDE;
  if (!aligned_to(mean, 4) || !aligned_to(inv_std, 4)) return ANODE_E_ALIGN;
  if (mean && mean == inv_std) return ANODE_E_STRIDE;
  const LayerArgs a = {rows, cols, epsilon, 1.0f / (float)cols, x, residual, x_stride, residual_stride, {gamma, weight_type}, {beta, weight_type},
                       y, total, y_stride, total_stride, mean, inv_std};
  return by_type(type, [&](auto t) {
    using T = decltype(t);
    return launch(layer_norm_rows_kernel<T>, dim3(row_blocks(rows)), kThreads, 0, stream, a);
  });
}

extern "C" size_t anode_gpu_layer_norm_add_bwd_workspace_bytes(uint64_t rows, uint32_t cols) { return (size_t)parts_of(rows) * cols * 8; }

extern "C" int anode_gpu_layer_norm_add_bwd(
    int type, uint64_t rows, uint32_t cols,
    const void *dy, uint64_t dy_stride, const void *total, uint64_t total_stride, const float *mean, const float *inv_std,
    const void *gamma, int weight_type, const void *dtotal, uint64_t dtotal_stride,
    void *dx, uint64_t dx_stride, void *dgamma, void *dbeta, void *workspace, size_t workspace_bytes,
    const struct KernelConfig *cfg, struct CUstream_st *stream)
{
  (void)cfg;
  const bool sums = dgamma || dbeta;
  if (!known_type(type) || ((gamma || sums) && !known_type(weight_type))) return ANODE_E_TYPE;
  if (!served(rows, cols)) return ANODE_E_DIMS;
  if (gamma && !aligned_to(gamma, type_bytes(weight_type))) return ANODE_E_ALIGN;
  if (sums) {
    for (void *w : {dgamma, dbeta}) if (w && !aligned_to(w, type_bytes(weight_type))) return ANODE_E_ALIGN;
    if (dgamma == dbeta || (gamma && dbeta == gamma)) return ANODE_E_STRIDE;
    if (rows == 0) {
      for (void *w : {dgamma, dbeta})
        if (w && cudaMemsetAsync(w, 0, type_bytes(weight_type) * cols, stream) != cudaSuccess) { (void)cudaGetLastError(); return ANODE_E_LAUNCH; }
      return ANODE_OK;
    }
    if (!workspace || !aligned_to(workspace, 16) || workspace_bytes < anode_gpu_layer_norm_add_bwd_workspace_bytes(rows, cols)) return ANODE_E_WORKSPACE;
  }
  if (rows == 0) return ANODE_OK;
  const size_t e = type_bytes(type);
  TRY(check_rows(dy, e, rows, cols, dy_stride, false));
  TRY(check_rows(total, e, rows, cols, total_stride, false));
  if (dtotal) TRY(check_rows(dtotal, e, rows, cols, dtotal_stride, false));
  TRY(check_rows(dx, e, rows, cols, dx_stride, true));
  if (!mean || !inv_std) return ANODE_E_NULL;
  if (!aligned_to(mean, 4) || !aligned_to(inv_std, 4)) return ANODE_E_ALIGN;
  if (!apart(dx, dx_stride, dy, dy_stride, rows) || !apart(dx, dx_stride, total, total_stride, rows) || !apart(dx, dx_stride, dtotal, dtotal_stride, rows))
    return ANODE_E_STRIDE;
  const LayerGradArgs a = {rows, cols, 1.0f / (float)cols, dy, total, dtotal, dy_stride, total_stride, dtotal_stride, mean, inv_std, {gamma, weight_type},
                           dx, dx_stride, dgamma, dbeta, weight_type, static_cast<float *>(workspace), parts_of(rows)};
  const uint32_t wide = (uint32_t)(((uint64_t)cols + kThreads - 1) / kThreads);
  return by_type(type, [&](auto t) {
    using T = decltype(t);
    // the weights' parts ahead of dx, which may be dy; dgamma, which may be gamma, behind it
    if (sums) TRY(launch(layer_norm_dweights_kernel<T>, dim3(wide, a.parts), kThreads, 0, stream, a));
    TRY(launch(layer_norm_dx_kernel<T>, dim3(row_blocks(rows)), kThreads, 0, stream, a));
    return sums ? launch(join_weights_kernel, dim3((uint32_t)(((uint64_t)cols + 31) / 32), 2), kThreads, 0, stream, cols, a.parts, (const float *)a.partial, dgamma, dbeta, weight_type)
                : (int)ANODE_OK;
  });
}
