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
constexpr uint32_t kMostParts = 148;       // of dgamma's sums
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

// The launch of the kernels that hold their rows
struct Held {
  uint32_t team, chunks;     // threads of a row, slots of each
  uint32_t slots;            // 16-byte slots of a row
  uint32_t groups;           // of 128 columns, where 8-bit rows have them
};

// Rows held in registers: a team of threads (4 to 32 lanes of a warp, or a block) has a row, a thread CH slots of 16 bytes, so that the
// row is read once.  SHIFT: rows that begin anywhere or are no whole number of slots, as long as all arrays' rows begin at the same place of a slot:
// slots are those of the addresses, the first and the last are moved element by element.
constexpr uint32_t most_threads(int chunks) { return chunks <= 2 ? 1024u : chunks == 4 ? 512u : 640u; }

template <typename T, int CH, bool SHIFT, bool QUANT>
__global__ void __launch_bounds__(most_threads(CH)) rms_norm_held_kernel(const NormArgs a, const Held h)
{
  constexpr int V = Vec<T>::V;
  __shared__ float buf[2][32];
  extern __shared__ uint32_t tops[];            // bits of the largest |y| of each group, where groups are not whole slots
  const uint32_t per_block = blockDim.x / h.team, mine = threadIdx.x / h.team, at = threadIdx.x - mine * h.team;
  const uint64_t row = (uint64_t)blockIdx.x * per_block + mine;
  const bool live = row < a.rows;               // (all threads take part in the teams' sums)
  const T *x = static_cast<const T *>(a.x) + row * a.x_stride;
  const T *res = a.residual ? static_cast<const T *>(a.residual) + row * a.residual_stride : nullptr;
  const int ph = SHIFT ? (int)(((uintptr_t)x & 15) / sizeof(T)) : 0;
  uint32_t *top = tops + mine * h.groups;
  const bool lines = QUANT && a.block != a.cols;
  if (SHIFT && lines) for (uint32_t i = at; i < h.groups; i += h.team) top[i] = 0;
  pdl_wait();
  Vec<T> t[CH], r[CH];
  // slot k of this thread: columns from `col` on, the elements [first, end) of it belong to the row
  auto col = [&](int k) { return (int)((at + k * h.team) * V) - ph; };
  auto first = [&](int k) { return SHIFT ? max(0, -col(k)) : 0; };
  auto end = [&](int k) { return SHIFT ? min(V, (int)a.cols - col(k)) : V; };
  auto has = [&](int k) { return live && at + k * h.team < h.slots && (!SHIFT || end(k) > 0); };
  auto whole = [&](int k) { return !SHIFT || (first(k) == 0 && end(k) == V); };
  auto load = [&](const T *p, int k) { return whole(k) ? Vec<T>::load(p + col(k)) : Vec<T>::load_some(p + col(k), first(k), end(k)); };
#pragma unroll
  for (int k = 0; k < CH; ++k) {
    t[k].bits = make_uint4(0, 0, 0, 0);
    if (has(k)) t[k] = load(x, k);
  }
  if (res) {
#pragma unroll
    for (int k = 0; k < CH; ++k) if (has(k)) r[k] = load(res, k);
  }
  // the weights of few slots are loaded ahead of the sum, those of many when they are needed: they would take the registers
  constexpr bool AHEAD = CH <= 2;
  float g[AHEAD ? CH : 1][V];
  auto weights = [&](int k, float *w) {
    if (!SHIFT) a.gamma.load<V>(col(k), w);
    else {
#pragma unroll
      for (int i = 0; i < V; ++i) w[i] = i >= first(k) && i < end(k) ? a.gamma.at(col(k) + i) : 0.0f;
    }
  };
  if (AHEAD) {
#pragma unroll
    for (int k = 0; k < CH; ++k) if (has(k)) weights(k, g[AHEAD ? k : 0]);
  }
  float sq = 0.0f;
#pragma unroll
  for (int k = 0; k < CH; ++k) {
    if (!has(k)) continue;
    float f[V];
    t[k].floats(f);
    if (res) {
      float e[V];
      r[k].floats(e);
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] += e[i];
      t[k] = Vec<T>::of(f);
      t[k].floats(f);
      if (a.total) {
        T *p = static_cast<T *>(a.total) + row * a.total_stride + col(k);
        if (whole(k)) t[k].store(p); else t[k].store_some(p, first(k), end(k));
      }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) sq = fmaf(f[i], f[i], sq);
  }
  const float inv = 1.0f / sqrtf(team_sum_all(sq, h.team, buf[0]) * a.inv_cols + a.epsilon);
  if (live && a.inv_rms && at == 0) a.inv_rms[row] = inv;
  auto values = [&](int k, float *y) {
    float f[V];
    t[k].floats(f);
    if (AHEAD) {
#pragma unroll
      for (int i = 0; i < V; ++i) y[i] = f[i] * inv * g[AHEAD ? k : 0][i];
    } else {
      weights(k, y);
#pragma unroll
      for (int i = 0; i < V; ++i) y[i] *= f[i] * inv;
    }
  };
  if (!QUANT) {
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      if (!has(k)) continue;
      float f[V];
      values(k, f);
      T *p = static_cast<T *>(a.y) + row * a.y_stride + col(k);
      const Vec<T> y = Vec<T>::of(f);
      if (whole(k)) y.store(p); else y.store_some(p, first(k), end(k));
    }
    return;
  }
  // bits of |y| in the order of unsigned numbers: a NaN's lie above all
  auto largest = [&](const float *y, int from, int to) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) if (!SHIFT || (i >= from && i < to)) m = max(m, __float_as_uint(y[i]) & 0x7fffffffu);
    return m;
  };
  auto scale_of = [&](uint32_t m) { return __uint_as_float(max(m, __float_as_uint(kTiny))) / kE4M3; };
  // V values to 8 bits: those before `edge` times `one`, the others times `two`
  auto put = [&](int k, const float *y, float one, float two, int edge) {
    uint8_t *q = static_cast<uint8_t *>(a.y) + row * a.y_stride + col(k);
    uint32_t w[V / 4];
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
      float f[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) f[j] = y[4 * i + j] * (SHIFT && 4 * i + j >= edge ? two : one);
      w[i] = (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(f[0], f[1]), __NV_SATFINITE, __NV_E4M3) |
             (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(f[2], f[3]), __NV_SATFINITE, __NV_E4M3) << 16;
    }
    if (whole(k)) {
      if constexpr (V == 8) *reinterpret_cast<uint2 *>(q) = make_uint2(w[0], w[V / 4 - 1]);
      else *reinterpret_cast<uint32_t *>(q) = w[0];
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) if (i >= first(k) && i < end(k)) q[i] = (uint8_t)(w[i / 4] >> (8 * (i % 4)));
    }
  };
  if (lines && !SHIFT) {
    // 128 columns: 128/V lanes with a slot each
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      float y[V];
      uint32_t m = 0;
      if (has(k)) { values(k, y); m = largest(y, 0, V); }
#pragma unroll
      for (int o = 64 / V; o > 0; o >>= 1)
        if (o < (int)h.team) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));      // (a smaller team has one group)
      if (!has(k)) continue;
      const float scale = scale_of(m), one = 1.0f / scale;
      if (col(k) % 128 == 0) a.scale[row * a.scale_row + (uint32_t)col(k) / 128 * a.scale_group] = scale;
      put(k, y, one, one, V);
    }
    return;
  }
  if (!lines) {
    uint32_t all = 0;
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      if (!has(k)) continue;
      float y[V];
      values(k, y);
      all = max(all, largest(y, first(k), end(k)));
    }
    for (uint32_t o = min(h.team, 32u) / 2; o > 0; o >>= 1) all = max(all, __shfl_xor_sync(0xffffffffu, all, o));
    if (h.team > 32) {
      if ((threadIdx.x & 31) == 0) buf[1][threadIdx.x >> 5] = __uint_as_float(all);
      __syncthreads();
      all = __reduce_max_sync(0xffffffffu, (threadIdx.x & 31) < blockDim.x / 32 ? __float_as_uint(buf[1][threadIdx.x & 31]) : 0u);
    }
    const float scale = scale_of(all), one = 1.0f / scale;
    if (live && at == 0) a.scale[row * a.scale_row] = scale;
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      if (!has(k)) continue;
      float y[V];
      values(k, y);
      put(k, y, one, one, V);
    }
    return;
  }
  // groups that end inside of slots: elements of a slot before `edge` are of its first group
  auto edge = [&](int k) { return 128 - (col(k) + first(k)) % 128 + first(k); };
  auto sync = [&] { if (h.team > 32) __syncthreads(); else __syncwarp(); };
  sync();
#pragma unroll
  for (int k = 0; k < CH; ++k) {
    if (!has(k)) continue;
    float y[V];
    values(k, y);
    const uint32_t group = (uint32_t)(col(k) + first(k)) / 128;
    atomicMax(top + group, largest(y, first(k), min(end(k), edge(k))));
    if (end(k) > edge(k)) atomicMax(top + group + 1, largest(y, edge(k), end(k)));
  }
  sync();
  if (live) for (uint32_t i = at; i < h.groups; i += h.team) a.scale[row * a.scale_row + i * a.scale_group] = scale_of(top[i]);
#pragma unroll
  for (int k = 0; k < CH; ++k) {
    if (!has(k)) continue;
    float y[V];
    values(k, y);
    const uint32_t group = (uint32_t)(col(k) + first(k)) / 128;
    const float one = 1.0f / scale_of(top[group]);
    put(k, y, one, end(k) > edge(k) ? 1.0f / scale_of(top[group + 1]) : one, edge(k));
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

// How the adjoint's rows are held: `teams` teams of `team` threads to a block, each with a row at a time
struct HeldGrad { uint32_t team, teams, slots; };

constexpr uint32_t kGradThreads = 512;

// W elements of a row: 16 bytes, or one element
template <typename T, int W> struct Piece {
  Vec<T> v;
  __device__ __forceinline__ static Piece load(const T *p) { return Piece{Vec<T>::load(p)}; }
  __device__ __forceinline__ void floats(float *f) const { v.floats(f); }
  __device__ __forceinline__ static void store(T *p, const float *f) { Vec<T>::of(f).store(p); }
};
template <typename T> struct Piece<T, 1> {
  T v;
  __device__ __forceinline__ static Piece load(const T *p) { return Piece{*p}; }
  __device__ __forceinline__ void floats(float *f) const { f[0] = to_float(v); }
  __device__ __forceinline__ static void store(T *p, const float *f) { *p = from_float<T>(f[0]); }
};

// The adjoint with its rows held in registers: a team of threads walks down rows, each thread with the same columns of all of them, so that
// one pass over the arrays gives dx and, in the threads' registers, dgamma's sums.  PRE: the next row is on its way while one is worked on.
// The teams' sums join in shared memory and the blocks' in a second launch, both in a fixed order.
template <typename T, int W, int CH, bool PRE>
__global__ void __launch_bounds__(kGradThreads) rms_norm_grad_kernel(const GradArgs a, const HeldGrad h)
{
  __shared__ float buf[2][kGradThreads / 32];
  extern __shared__ float sums[];               // [teams][cols]
  const uint32_t mine = threadIdx.x / h.team, at = threadIdx.x - mine * h.team, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool works = mine < h.teams;
  auto col = [&](int k) { return (at + k * h.team) * W; };
  auto has = [&](int k) { return works && at + k * h.team < h.slots; };
  pdl_wait();
  float acc[CH][W], g[CH][W];
#pragma unroll
  for (int k = 0; k < CH; ++k) {
#pragma unroll
    for (int i = 0; i < W; ++i) { acc[k][i] = 0.0f; g[k][i] = 0.0f; }
    if (!has(k)) continue;
    if constexpr (W > 1) a.gamma.load<W>(col(k), g[k]); else g[k][0] = a.gamma.at(col(k));
  }
  typedef Piece<T, W> Some;
  struct Row { Some dy[CH], t[CH], dt[CH]; float r; } now, next;
  auto load = [&](Row &w, uint64_t row) {
    const T *dy = static_cast<const T *>(a.dy) + row * a.dy_stride, *t = static_cast<const T *>(a.total) + row * a.total_stride;
    const T *dt = a.dtotal ? static_cast<const T *>(a.dtotal) + row * a.dtotal_stride : nullptr;
    w.r = a.inv_rms[row];
#pragma unroll
    for (int k = 0; k < CH; ++k)
      if (has(k)) { w.dy[k] = Some::load(dy + col(k)); w.t[k] = Some::load(t + col(k)); }
    if (dt) {
#pragma unroll
      for (int k = 0; k < CH; ++k) if (has(k)) w.dt[k] = Some::load(dt + col(k));
    }
  };
  const uint64_t step = (uint64_t)gridDim.x * h.teams;
  uint64_t row = (uint64_t)blockIdx.x * h.teams + mine;
  uint32_t turn = 0;
  if (PRE && works && row < a.rows) load(now, row);
  for (; works && row < a.rows; row += step, turn ^= 1) {
    if (PRE) { if (row + step < a.rows) load(next, row + step); }
    else load(now, row);
    float dot = 0.0f;
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      if (!has(k)) continue;
      float dy[W], t[W];
      now.dy[k].floats(dy); now.t[k].floats(t);
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const float xh = t[i] * now.r;
        acc[k][i] = fmaf(dy[i], xh, acc[k][i]);
        dot = fmaf(dy[i] * g[k][i], xh, dot);
      }
    }
    dot = warp_sum_all(dot);
    if (h.team > 32) {
      if (lane == 0) buf[turn][warp] = dot;
      asm volatile("bar.sync %0, %1;" ::"r"(mine + 1), "r"(h.team) : "memory");
      const uint32_t first = mine * h.team / 32, warps = h.team / 32;
      dot = warp_sum_all(lane < warps ? buf[turn][first + lane] : 0.0f);
    }
    dot *= a.inv_cols;
    T *dx = static_cast<T *>(a.dx) + row * a.dx_stride;
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      if (!has(k)) continue;
      float dy[W], t[W], dt[W];
      now.dy[k].floats(dy); now.t[k].floats(t);
      if (a.dtotal) now.dt[k].floats(dt);
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const float v = now.r * (dy[i] * g[k][i] - t[i] * now.r * dot);
        dy[i] = a.dtotal ? v + dt[i] : v;
      }
      Some::store(dx + col(k), dy);
    }
    if (PRE) now = next;
  }
  if (!a.dgamma) return;
#pragma unroll
  for (int k = 0; k < CH; ++k) {
    if (!has(k)) continue;
#pragma unroll
    for (int i = 0; i < W; ++i) sums[(size_t)mine * a.cols + col(k) + i] = acc[k][i];
  }
  __syncthreads();
  for (uint32_t c = threadIdx.x; c < a.cols; c += kGradThreads) {
    float sum = 0.0f;
    for (uint32_t t = 0; t < h.teams; ++t) sum += sums[(size_t)t * a.cols + c];
    a.partial[(uint64_t)blockIdx.x * a.cols + c] = sum;
  }
}

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

// The blocks' sums: a lane has a column, a warp every eighth part of it
__global__ void __launch_bounds__(kThreads) join_columns_kernel(uint32_t cols, uint32_t parts, const float *partial, void *out, int type)
{
  constexpr uint32_t kWarps = kThreads / 32;
  __shared__ float sums[kWarps][33];
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint64_t c = (uint64_t)blockIdx.x * 32 + lane;
  pdl_wait();
  float sum = 0.0f;
  if (c < cols) {
#pragma unroll 4
    for (uint32_t p = warp; p < parts; p += kWarps) sum += partial[(uint64_t)p * cols + c];
  }
  sums[warp][lane] = sum;
  __syncthreads();
  if (warp || c >= cols) return;
#pragma unroll
  for (uint32_t w = 1; w < kWarps; ++w) sum += sums[w][lane];
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

inline uint32_t parts_of(uint64_t rows) { return (uint32_t)(rows < kMostParts ? (rows ? rows : 1) : kMostParts); }
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

// Whether an array's rows all begin at the same place of a slot of `v` elements as those of the first one
inline bool in_step(const void *p, size_t bytes, uint64_t stride, uint32_t v, const void *p0, size_t bytes0, uint64_t stride0, uint64_t rows)
{
  return !p || ((uintptr_t)p / bytes % v == (uintptr_t)p0 / bytes0 % v && (rows <= 1 || stride % v == stride0 % v));
}

// How the rows of a call are held in registers; false where they are not
bool held_plan(const NormArgs &a, int type, int gamma_type, bool quant, Held &h, bool &shift)
{
  const size_t e = type_bytes(type);
  const uint32_t v = (uint32_t)(16 / e);
  if (!in_step(a.residual, e, a.residual_stride, v, a.x, e, a.x_stride, a.rows) || !in_step(a.total, e, a.total_stride, v, a.x, e, a.x_stride, a.rows) ||
      !in_step(a.y, quant ? 1 : e, a.y_stride, v, a.x, e, a.x_stride, a.rows)) return false;
  shift = !aligned_to(a.x, 16) || a.cols % v || (a.rows > 1 && a.x_stride % v) || !aligned_to(a.gamma.p, 16);
  const uint64_t slots = shift ? ((uint64_t)a.cols + 2 * v - 2) / v : a.cols / v;
  if (slots > 8 * most_threads(8)) return false;
  h.slots = (uint32_t)slots;
  h.groups = quant && a.block != a.cols ? (a.cols + 127) / 128 : 0;
  if (slots <= 128) {
    h.team = 4;
    while (h.team < 32 && h.team < slots) h.team *= 2;
    h.chunks = slots <= 32 ? 1 : slots <= 64 ? 2 : 4;
  } else {
    h.chunks = a.rows <= 2 * 148 && slots <= 2048 ? (slots <= 1024 ? 1 : 2) : slots <= 4 * most_threads(4) ? 4 : 8;
    h.team = (h.slots + h.chunks * 32 - 1) / (h.chunks * 32) * 32;
  }
  return true;
}

template <typename T, int CH> int launch_held(const NormArgs &a, const Held &h, bool shift, bool quant, cudaStream_t stream)
{
  const uint32_t threads = h.team > 32 ? h.team : 128, per_block = threads / h.team;
  const dim3 grid((uint32_t)((a.rows + per_block - 1) / per_block));
  const size_t shared = shift ? (size_t)per_block * h.groups * 4 : 0;
  if (quant) return shift ? launch(rms_norm_held_kernel<T, CH, true, true>, grid, threads, shared, stream, a, h)
                          : launch(rms_norm_held_kernel<T, CH, false, true>, grid, threads, shared, stream, a, h);
  return shift ? launch(rms_norm_held_kernel<T, CH, true, false>, grid, threads, shared, stream, a, h)
               : launch(rms_norm_held_kernel<T, CH, false, false>, grid, threads, shared, stream, a, h);
}

// How the rows of an adjoint are held in registers: pieces of 16 bytes or of one element, `chunks` of them to a thread; false where they are not
bool grad_plan(const GradArgs &a, int type, HeldGrad &h, uint32_t &width, uint32_t &chunks)
{
  const size_t e = type_bytes(type);
  const uint32_t v = (uint32_t)(16 / e);
  auto fits = [&](const void *p, uint64_t stride) { return !p || (aligned_to(p, 16) && (a.rows <= 1 || stride % v == 0)); };
  width = a.cols % v == 0 && fits(a.dy, a.dy_stride) && fits(a.total, a.total_stride) && fits(a.dtotal, a.dtotal_stride) && fits(a.dx, a.dx_stride) &&
          aligned_to(a.gamma.p, 16) ? v : 1;
  h.slots = a.cols / width;
  const uint32_t most = width > 1 ? 4 : 16;
  if (h.slots > most * kGradThreads) return false;
  chunks = width > 1 ? (h.slots <= 32 ? 1 : h.slots <= 2 * kGradThreads ? 2 : 4) : h.slots <= 64 ? 2 : h.slots <= 8 * kGradThreads ? 8 : 16;
  h.team = (h.slots + chunks * 32 - 1) / (chunks * 32) * 32;
  h.teams = kGradThreads / h.team;
  if (a.rows < (uint64_t)h.teams * sm_count()) h.teams = (uint32_t)((a.rows + sm_count() - 1) / sm_count());     // a row per block first
  return true;
}

template <typename T, int W, int CH, bool PRE> int launch_grad(const GradArgs &a, const HeldGrad &h, cudaStream_t stream)
{
  const auto kernel = rms_norm_grad_kernel<T, W, CH, PRE>;
  const size_t shared = a.dgamma ? (size_t)h.teams * a.cols * 4 : 0;
  static SharedMemory allowed;
  if (!allowed.up_to((const void *)kernel, shared)) return ANODE_E_LAUNCH;
  return launch(kernel, dim3(a.parts), kGradThreads, shared, stream, a, h);
}

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
  Held h = {};
  bool shift = false;
  const bool held = a.rows < (1ull << 30) && held_plan(a, type, gamma_type, quant, h, shift);
  return by_type(type, [&](auto t) {
    using T = decltype(t);
    if (held) return h.chunks == 1 ? launch_held<T, 1>(a, h, shift, quant, stream) : h.chunks == 2 ? launch_held<T, 2>(a, h, shift, quant, stream)
                   : h.chunks == 4 ? launch_held<T, 4>(a, h, shift, quant, stream) : launch_held<T, 8>(a, h, shift, quant, stream);
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
  HeldGrad h = {};
  uint32_t width = 0, chunks = 0;
  const bool held = grad_plan(a, type, h, width, chunks);
  const uint32_t wide = (uint32_t)(((uint64_t)cols + kThreads - 1) / kThreads), narrow = (uint32_t)(((uint64_t)cols + 31) / 32);
  return by_type(type, [&](auto t) {
    using T = decltype(t);
    constexpr int V = Vec<T>::V;
    if (held) {
      const uint64_t blocks = (rows + h.teams - 1) / h.teams;
      if (a.parts > blocks) a.parts = (uint32_t)blocks;
      TRY(width > 1 ? (chunks == 1 ? launch_grad<T, V, 1, true>(a, h, stream) : chunks == 2 ? launch_grad<T, V, 2, true>(a, h, stream)
                                   : launch_grad<T, V, 4, false>(a, h, stream))
                    : (chunks == 2 ? launch_grad<T, 1, 2, true>(a, h, stream) : chunks == 8 ? launch_grad<T, 1, 8, true>(a, h, stream)
                                   : launch_grad<T, 1, 16, false>(a, h, stream)));
      return dgamma ? launch(join_columns_kernel, dim3(narrow), kThreads, 0, stream, cols, a.parts, a.partial, dgamma, gamma_type) : (int)ANODE_OK;
    }
    if (dgamma) {
      TRY(launch(rms_norm_dgamma_kernel<T>, dim3(wide, a.parts), kThreads, 0, stream, a));
      TRY(launch(join_columns_kernel, dim3(narrow), kThreads, 0, stream, cols, a.parts, a.partial, dgamma, gamma_type));
    }
    return launch(rms_norm_dx_kernel<T>, dim3(row_blocks(rows)), kThreads, 0, stream, a);
  });
}
