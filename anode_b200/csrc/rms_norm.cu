// RMS norm over rows with the residual's addition: forward, adjoint, and the forward pass with an output in 8 bits.
//
//   t = round(x + residual),  r = (mean(t^2) + epsilon)^-1/2,  y = t*r*gamma
//   dx = r*(g - xh*mean(g*xh)) + dt,   g = dy*gamma, xh = t*r,   dgamma = sum over rows of dy*xh
//   a = max |y| of a group, scale = max(a, 2^-96)/448, q = e4m3(y/scale)
//
// Statistics and sums are f32; y, total and dx are rounded once, total before the norm reads it, and what goes to 8 bits is not rounded before.
//
// All of it is bound by memory where there are many rows (a handful of operations per element), and by the chain launch -> load -> sum -> store
// where there are few.  Measured on one B200 against its copy bandwidth of 6539 GB/s, bf16 with residual, rows of 8192:
//   forward            [16384,8192] 158 us (1.04 of it), without a residual 92 us (0.89); ragged rows of 4095 84 us (0.98); [1,4096] 1.7 us
//   8 bits, per 128    [8192,8192] 77 us (0.93), ragged rows of 8191 107 us (0.67: a slot's two groups are chosen element by element)
//   8 bits, per row    [8192,8192] 72.5 us (0.99)
//   adjoint            [8192,4096] 46.5 us (0.88), [8192,16384] 160 us (1.02), ragged rows of 4095 56 us (0.73); f32 [4096,16384] 181 us (0.91),
//                      [4096,16381] 279 us (0.59: 64 registers to a thread of a row of 4096 slots, and spills)
// Three kernels: rms_norm_held_kernel (forward: a row per team of threads, many small blocks, whose loads and stores overlap one another's;
// persistent teams with the next row on its way took 191 us for the first of these and 87.5 for the fourth), rms_norm_grad_kernel (persistent
// teams, since dgamma's sums stay in registers), and the plain ones below for rows that are too wide or do not begin in step: element by element, two
// or three reads of each.  Those take 221 us forward for [8192,8192] out of step (0.37), 289 in 8 bits (0.25), 220 back for [8192,4096] (0.19).
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
  uint32_t block;                      // columns of a group (0: the whole row)
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

// Any rows: a block has a row at a time, element by element, and reads it again for the second pass
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
      const bool whole = a.block == 0;
      const uint32_t width = whole ? a.cols : a.block;
      const uint32_t lane = whole ? threadIdx.x : threadIdx.x & 31, lanes = whole ? kThreads : 32, warp = threadIdx.x >> 5;
      __syncthreads();       // (the sum is stored by other threads than read it here)
      for (uint64_t base = whole ? 0 : (uint64_t)warp * width, group = whole ? 0 : warp; base < a.cols;
           base += (uint64_t)width * (kThreads / 32), group += kThreads / 32) {
        const uint32_t end = (uint32_t)(base + width < a.cols ? base + width : a.cols);
        uint32_t top = 0;
        for (uint32_t c = (uint32_t)base + lane; c < end; c += lanes) top = max(top, __float_as_uint(value(c)) & 0x7fffffffu);
        top = __reduce_max_sync(0xffffffffu, top);
        if (whole) {
          if ((threadIdx.x & 31) == 0) buf[1][warp] = __uint_as_float(top);
          __syncthreads();
          for (uint32_t w = 0; w < kThreads / 32; ++w) top = max(top, __float_as_uint(buf[1][w]));
        }
        const float peak = __uint_as_float(max(top, __float_as_uint(kTiny))), inv = kE4M3 / peak;
        if (lane == 0) a.scale[row * a.scale_row + group * a.scale_group] = peak / kE4M3;
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
  uint32_t groups;           // of 128 columns, where 8-bit rows have them
};

__host__ __device__ constexpr uint32_t most_threads(int chunks) { return chunks <= 2 ? 1024u : chunks == 4 ? 512u : 640u; }

// A group's scale, and 448 over its largest |y|, which its values are multiplied by, from the bits of that: quotients rounded to nearest, from an approximate
// one and the remainder that it leaves (Markstein 1990).  An infinity leaves none: the scale is infinite, too, and finite values become 0.  Only the lane that
// stores the scale makes it.  [8192,8192] bf16, a scale per 128 columns: 77.1 us; 76.3 with the approximate quotients, whose values were twice as often on
// the other side of the middle of two; both quotients in every lane 78.2; divisions 81.5.
__device__ __forceinline__ float peak_of(uint32_t largest) { return __uint_as_float(max(largest, __float_as_uint(kTiny))); }
__device__ __forceinline__ float scale_of(uint32_t largest)
{
  constexpr float c = 1.0f / kE4M3;
  const float a = peak_of(largest), s = a * c;
  return a == __uint_as_float(0x7f800000u) ? a : fmaf(fmaf(-s, kE4M3, a), c, s);
}
__device__ __forceinline__ float inverse_of(uint32_t largest)
{
  constexpr float c = 1.0f / kE4M3;
  const float r = __fdividef(1.0f, peak_of(largest) * c);      // (of 2^-105 to 2^120: nothing is flushed)
  // (r = 0 of an infinity stays 0 with the largest number in its place; a NaN's stays NaN)
  return fmaf(fmaf(-peak_of(min(largest, 0x7f7fffffu)), r, kE4M3), r * c, r);
}

__device__ __forceinline__ float max_nan(float a, float b)
{
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// Rows held in registers: a team of threads (4 to 32 lanes of a warp, or a block) has a row, a thread CH slots of 16 bytes, so that the
// row is read once.  SHIFT: rows that begin anywhere or are no whole number of slots, as long as all arrays' rows begin at the same place of a
// slot: slots are then those of the addresses, and the elements before the first whole one and after the last have a lane each.
// QUANT: 0 none, else an output in 8 bits with a scale for each row (1) or for each 128 columns (2).
// What bounds it: memory; so a thread's loads are all in flight at once.
template <typename T, int CH, bool SHIFT, int QUANT, bool RES>
__global__ void __launch_bounds__(most_threads(CH)) rms_norm_held_kernel(const NormArgs a, const Held h)
{
  constexpr int V = Vec<T>::V, H = V / 2;
  __shared__ float buf[2][32];
  extern __shared__ uint32_t tops[];            // bits of the largest |y| of each group, where groups are not whole slots
  const uint32_t per_block = blockDim.x / h.team, mine = threadIdx.x / h.team, at = threadIdx.x - mine * h.team;
  const uint64_t row = (uint64_t)blockIdx.x * per_block + mine;
  const bool live = row < a.rows;               // (all threads take part in the teams' sums)
  const T *x = static_cast<const T *>(a.x) + row * a.x_stride;
  const T *res = RES ? static_cast<const T *>(a.residual) + row * a.residual_stride : nullptr;
  T *total = RES && a.total ? static_cast<T *>(a.total) + row * a.total_stride : nullptr;
  // the row's head: columns before its first whole slot; then `slots` of them, and a tail
  const uint32_t head = SHIFT ? min(a.cols, (uint32_t)(-(int)((uintptr_t)x / sizeof(T)) & (V - 1))) : 0, slots = (a.cols - head) / V;
  const uint32_t start = head + at * V, hop = h.team * V;      // this thread's slots: columns start + k*hop
  const uint32_t mine_slots = live && at < slots ? (slots - at + h.team - 1) / h.team : 0;
  // the lane's element of the head or the tail
  const uint32_t tail = a.cols - head - slots * V, edge = at < head ? at : a.cols - tail + (at - head);
  const bool on_edge = SHIFT && live && at < head + tail;
  uint32_t *top = tops + mine * h.groups;
  constexpr bool LINES = QUANT == 2;
  if (SHIFT && LINES) for (uint32_t i = at; i < h.groups; i += h.team) top[i] = 0;
  const bool aligned_gamma = ((uintptr_t)a.gamma.p & 15) == 0;
  pdl_wait();
  pdl_trigger();        // (the next kernel's blocks wait as these did: 0.1 to 0.3 us of a call of few rows)
  Vec<T> t[CH], r[RES ? CH : 1];
#pragma unroll
  for (int k = 0; k < CH; ++k) {
    t[k].bits = make_uint4(0, 0, 0, 0);
    if (k < mine_slots) t[k] = Vec<T>::load(x + start + k * hop);
  }
  if constexpr (RES) {
#pragma unroll
    for (int k = 0; k < CH; ++k) if (k < mine_slots) r[k] = Vec<T>::load(res + start + k * hop);
  }
  float te = 0.0f, ge = 1.0f;
  if (on_edge) {
    te = to_float(x[edge]);
    if (RES) te = to_float(from_float<T>(te + to_float(res[edge])));
    ge = a.gamma.at(edge);
  }
  // the weights of few slots are loaded ahead of the sum, those of many when they are needed: they would take the registers
  constexpr bool AHEAD = CH <= 2;
  float2 g[AHEAD ? CH : 1][H];
  auto weights = [&](int k, float2 *w) {
    float *f = reinterpret_cast<float *>(w);
    const uint32_t c = start + k * hop;
    if (!SHIFT) a.gamma.load<V>(c, f);
    else if (aligned_gamma) a.gamma.load_any<V>(c, a.cols, f);
    else a.gamma.load_each<V>(c, f);
  };
  if (AHEAD) {
#pragma unroll
    for (int k = 0; k < CH; ++k) if (k < mine_slots) weights(k, g[AHEAD ? k : 0]);
  }
  float2 sq2 = make_float2(te * te, 0.0f);
#pragma unroll
  for (int k = 0; k < CH; ++k) {
    float2 f[H];
    if (RES && k < mine_slots) {
      float2 e[H];
      t[k].floats(reinterpret_cast<float *>(f));
      r[RES ? k : 0].floats(reinterpret_cast<float *>(e));
#pragma unroll
      for (int i = 0; i < H; ++i) f[i] = add2(f[i], e[i]);
      t[k] = Vec<T>::of(reinterpret_cast<const float *>(f));
      if (total) t[k].store(total + start + k * hop);
    }
    t[k].floats(reinterpret_cast<float *>(f));
#pragma unroll
    for (int i = 0; i < H; ++i) sq2 = fma2(f[i], f[i], sq2);
  }
  if (on_edge && total) total[edge] = from_float<T>(te);
  const float inv = 1.0f / sqrtf(team_sum_all(sq2.x + sq2.y, h.team, buf[0]) * a.inv_cols + a.epsilon);
  if (live && a.inv_rms && at == 0) a.inv_rms[row] = inv;
  const float2 inv2 = both(inv);
  auto values = [&](int k, float2 *y) {
    float2 f[H];
    t[k].floats(reinterpret_cast<float *>(f));
    if (!AHEAD) weights(k, y);
#pragma unroll
    for (int i = 0; i < H; ++i) y[i] = mul2(mul2(f[i], inv2), AHEAD ? g[AHEAD ? k : 0][i] : y[i]);
  };
  const float ye = te * inv * ge;
  if constexpr (!QUANT) {
    T *y = static_cast<T *>(a.y) + row * a.y_stride;
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      if (k >= mine_slots) continue;
      float2 f[H];
      values(k, f);
      Vec<T>::of(reinterpret_cast<const float *>(f)).store(y + start + k * hop);
    }
    if (on_edge) y[edge] = from_float<T>(ye);
    return;
  }
  // bits of |y| in the order of unsigned numbers: a NaN's lie above all
  auto bits_of = [](float v) { return __float_as_uint(v) & 0x7fffffffu; };
  auto largest = [&](const float2 *y) {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < H; ++i) m = max_nan(max_nan(m, fabsf(y[i].x)), fabsf(y[i].y));
    return bits_of(m);
  };
  uint8_t *q = static_cast<uint8_t *>(a.y) + row * a.y_stride;
  auto eight = [](float u, float v) { return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(u, v), __NV_SATFINITE, __NV_E4M3); };
  // a slot to 8 bits: its elements before `border` times `one`, the others times `two`
  auto put = [&](int k, const float2 *y, float one, float two, int border) {
    uint32_t w[V / 4];
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
      const float2 u = mul2(y[2 * i], SHIFT && LINES ? make_float2(4 * i >= border ? two : one, 4 * i + 1 >= border ? two : one) : both(one));
      const float2 v = mul2(y[2 * i + 1], SHIFT && LINES ? make_float2(4 * i + 2 >= border ? two : one, 4 * i + 3 >= border ? two : one) : both(one));
      w[i] = eight(u.x, u.y) | eight(v.x, v.y) << 16;
    }
    if constexpr (V == 8) *reinterpret_cast<uint2 *>(q + start + k * hop) = make_uint2(w[0], w[V / 4 - 1]);
    else *reinterpret_cast<uint32_t *>(q + start + k * hop) = w[0];
  };
  if constexpr (LINES && !SHIFT) {
    // 128 columns: 128/V lanes with a slot each
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      float2 y[H];
      uint32_t m = 0;
      if (k < mine_slots) { values(k, y); m = largest(y); }
#pragma unroll
      for (int o = 64 / V; o > 0; o >>= 1)
        if (o < (int)h.team) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));      // (a smaller team has one group)
      if (k >= mine_slots) continue;
      const float one = inverse_of(m);
      const uint32_t c = start + k * hop;
      if (c % 128 == 0) a.scale[row * a.scale_row + c / 128 * a.scale_group] = scale_of(m);
      put(k, y, one, one, V);
    }
    return;
  }
  float2 y[CH][H];
#pragma unroll
  for (int k = 0; k < CH; ++k) if (k < mine_slots) values(k, y[k]);
  if constexpr (!LINES) {
    uint32_t all = on_edge ? bits_of(ye) : 0;
#pragma unroll
    for (int k = 0; k < CH; ++k) if (k < mine_slots) all = max(all, largest(y[k]));
    for (uint32_t o = min(h.team, 32u) / 2; o > 0; o >>= 1) all = max(all, __shfl_xor_sync(0xffffffffu, all, o));
    if (h.team > 32) {
      if ((threadIdx.x & 31) == 0) buf[1][threadIdx.x >> 5] = __uint_as_float(all);
      __syncthreads();
      all = __reduce_max_sync(0xffffffffu, (threadIdx.x & 31) < blockDim.x / 32 ? __float_as_uint(buf[1][threadIdx.x & 31]) : 0u);
    }
    const float one = inverse_of(all);
    if (live && at == 0) a.scale[row * a.scale_row] = scale_of(all);
#pragma unroll
    for (int k = 0; k < CH; ++k) if (k < mine_slots) put(k, y[k], one, one, V);
    if (on_edge) q[edge] = (uint8_t)eight(ye * one, 0.0f);
  } else {
    // groups that end inside of slots: elements of a slot before `border` are of its first group
    auto sync = [&] { if (h.team > 32) __syncthreads(); else __syncwarp(); };
    sync();
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      if (k >= mine_slots) continue;
      const uint32_t c = start + k * hop, border = 128 - c % 128;
      if (border >= V) { atomicMax(top + c / 128, largest(y[k])); continue; }
      float m[2] = {0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float v = fabsf(i % 2 ? y[k][i / 2].y : y[k][i / 2].x);
        if (i < border) m[0] = max_nan(m[0], v); else m[1] = max_nan(m[1], v);
      }
      atomicMax(top + c / 128, bits_of(m[0]));
      atomicMax(top + c / 128 + 1, bits_of(m[1]));
    }
    if (on_edge) atomicMax(top + edge / 128, bits_of(ye));
    sync();
    // a group's scale is made once, and its inverse takes the peak's place
    for (uint32_t i = at; i < h.groups; i += h.team) {
      if (live) a.scale[row * a.scale_row + i * a.scale_group] = scale_of(top[i]);
      top[i] = __float_as_uint(inverse_of(top[i]));
    }
    sync();
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      if (k >= mine_slots) continue;
      const uint32_t c = start + k * hop, border = 128 - c % 128;
      const float one = __uint_as_float(top[c / 128]);
      put(k, y[k], one, border < V ? __uint_as_float(top[c / 128 + 1]) : one, border);
    }
    if (on_edge) q[edge] = (uint8_t)eight(ye * __uint_as_float(top[edge / 128]), 0.0f);
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

// How the adjoint's rows are held: `teams` teams of `team` threads to a block, each with a row at a time, `depth` rows on their way or at work;
// a team's rows lie `step` apart
struct HeldGrad {
  uint32_t team, teams, depth, threads;
  uint64_t step;
};

// The adjoint with its rows held on chip: a team of threads (4 to 32 lanes of a warp, or more warps) walks down rows, a thread with CH slots of 16
// bytes of each array, so that one pass gives dx and dgamma's sums.  The next rows are on their way by asynchronous copies, each thread into a
// ring of its own: a thread waits for nothing but its own copies and, once per row, its team's sum.
// A thread's columns are the same in all of its team's rows: weights and dgamma's sums are in its registers.  SHIFT, as in
// rms_norm_held_kernel: rows that begin at different places of a slot do so in turns of at most V, so a team's rows lie a multiple of V
// apart and begin at the same one.
// The sums join in a fixed order, the teams' in shared memory and the blocks' in a second launch.
template <typename T, int CH, int NT, bool SHIFT>
__global__ void __launch_bounds__(NT) rms_norm_grad_kernel(const GradArgs a, const HeldGrad h)
{
  constexpr int V = Vec<T>::V, H = V / 2;
  __shared__ float buf[2][32];
  extern __shared__ float4 shared[];            // the rings [depth][CH][3][thread]; at last the sums [teams][cols]
  const uint32_t mine = threadIdx.x / h.team, at = threadIdx.x - mine * h.team, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint64_t row0 = (uint64_t)blockIdx.x * h.teams + mine;
  const bool works = mine < h.teams && row0 < h.step && row0 < a.rows;
  const uint32_t lanes = h.team < 32 ? ((1u << h.team) - 1) << (lane & ~(h.team - 1)) : 0xffffffffu;      // of this warp in the team
  const uint32_t nt = blockDim.x;
  uint4 *ring = reinterpret_cast<uint4 *>(shared) + threadIdx.x;
  const T *dy = static_cast<const T *>(a.dy) + row0 * a.dy_stride, *t = static_cast<const T *>(a.total) + row0 * a.total_stride;
  const T *dt = static_cast<const T *>(a.dtotal) + row0 * a.dtotal_stride;
  T *dx = static_cast<T *>(a.dx) + row0 * a.dx_stride;
  const float *inv = a.inv_rms + row0;
  // a row's columns before its first whole slot, and what remains behind the last one; this thread's slots, and its element of those
  const uint32_t head = SHIFT ? min(a.cols, (0u - (uint32_t)((uintptr_t)dy / sizeof(T))) & (V - 1)) : 0, slots = (a.cols - head) / V;
  const uint32_t tail = a.cols - head - slots * V, edge = at < head ? at : a.cols - tail + (at - head), start = head + at * V, hop = h.team * V;
  const bool on_edge = SHIFT && works && at < head + tail;
  auto has = [&](int k) { return works && at + k * h.team < slots; };
  pdl_wait();
  float2 acc[CH][H], g[CH][H];
  float acc_edge = 0.0f, g_edge = on_edge ? a.gamma.at(edge) : 0.0f;
  const bool aligned_gamma = ((uintptr_t)a.gamma.p & 15) == 0;
#pragma unroll
  for (int k = 0; k < CH; ++k) {
#pragma unroll
    for (int i = 0; i < H; ++i) acc[k][i] = g[k][i] = both(0.0f);
    if (!has(k)) continue;
    float *w = reinterpret_cast<float *>(g[k]);
    if (!SHIFT) a.gamma.load<V>(start + k * hop, w);
    else if (aligned_gamma) a.gamma.load_any<V>(start + k * hop, a.cols, w);
    else a.gamma.load_each<V>(start + k * hop, w);
  }
  // rows that this team has: at work, and to be copied
  uint32_t left = works ? (uint32_t)((a.rows - row0 + h.step - 1) / h.step) : 0, ahead = left, in = 0, out = 0;
  const uint64_t dy_step = h.step * a.dy_stride, t_step = h.step * a.total_stride, dt_step = h.step * a.dtotal_stride, dx_step = h.step * a.dx_stride;
  // what does not go through the ring, of the row that is worked on next: 1/rms, and an element of the head or the tail
  // (as it lies in memory: nothing waits for it before its row's turn)
  struct Side { float r; T dy, t, dt; } now = {}, next = {};
  const T *dy1 = dy + edge, *t1 = t + edge, *dt1 = dt + edge;
  auto side = [&](Side &o) {
    o.r = *inv;
    inv += h.step;
    if constexpr (SHIFT) {
      if (on_edge) {
        o.dy = *dy1; o.t = *t1;
        if (a.dtotal) o.dt = *dt1;
      }
      dy1 += dy_step; t1 += t_step; dt1 += dt_step;
    }
  };
  dy += start; t += start; dt += start;
  auto copy = [&] {                     // the next row to be copied
    if (ahead) {
      uint4 *to = ring + in * (CH * 3) * nt;
#pragma unroll
      for (int k = 0; k < CH; ++k) {
        if (!has(k)) continue;
        copy_async<16>(to + (3 * k) * nt, dy + k * hop);
        copy_async<16>(to + (3 * k + 1) * nt, t + k * hop);
        if (a.dtotal) copy_async<16>(to + (3 * k + 2) * nt, dt + k * hop);
      }
      --ahead;
      dy += dy_step; t += t_step; dt += dt_step;
    }
    copies_commit();
    in = in + 1 == h.depth ? 0 : in + 1;
  };
  for (uint32_t i = 1; i < h.depth; ++i) copy();
  if (left) side(next);
  uint32_t turn = 0;
  for (; left; --left, turn ^= 1) {
    now = next;
    copy();
    if (left > 1) side(next);
    if (h.depth == 4) copies_wait<3>(); else if (h.depth == 3) copies_wait<2>(); else if (h.depth == 2) copies_wait<1>(); else copies_wait<0>();
    const uint4 *from = ring + out * (CH * 3) * nt;
    out = out + 1 == h.depth ? 0 : out + 1;
    const float dy_edge = to_float(now.dy), t_edge = to_float(now.t);
    float2 dot2 = make_float2(SHIFT ? dy_edge * g_edge * t_edge : 0.0f, 0.0f);
    // a single slot stays in registers between the two passes over the row, more are read again
    constexpr bool ONE = CH == 1;
    float2 u[H], v[H];
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      if (!has(k)) continue;
      Vec<T>{from[(3 * k) * nt]}.floats(reinterpret_cast<float *>(u));
      Vec<T>{from[(3 * k + 1) * nt]}.floats(reinterpret_cast<float *>(v));
#pragma unroll
      for (int i = 0; i < H; ++i) dot2 = fma2(mul2(u[i], g[k][i]), v[i], dot2);
    }
    float dot = dot2.x + dot2.y;
    if (h.team >= 32) {
      dot = warp_sum_all(dot);
      if (h.team > 32) {
        if (lane == 0) buf[turn][warp] = dot;
        asm volatile("bar.sync %0, %1;" ::"r"(mine + 1), "r"(h.team) : "memory");
        const uint32_t first = mine * h.team / 32, warps = h.team / 32;
        dot = warp_sum_all(lane < warps ? buf[turn][first + lane] : 0.0f);
      }
    } else for (uint32_t o = h.team / 2; o > 0; o >>= 1) dot += __shfl_xor_sync(lanes, dot, o);
    // (1/rms meets the sum, a row's element and the bracket one at a time: its powers alone would leave f32's range where rows are large or tiny)
    const float m = dot * now.r * a.inv_cols;
    const float2 r = both(now.r), minus = both(-m);
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      if (!has(k)) continue;
      if (!ONE) {
        Vec<T>{from[(3 * k) * nt]}.floats(reinterpret_cast<float *>(u));
        Vec<T>{from[(3 * k + 1) * nt]}.floats(reinterpret_cast<float *>(v));
      }
      float2 e[H];
#pragma unroll
      for (int i = 0; i < H; ++i) {
        const float2 xh = mul2(v[i], r);
        acc[k][i] = fma2(u[i], xh, acc[k][i]);
        e[i] = fma2(u[i], g[k][i], mul2(xh, minus));
      }
      if (a.dtotal) {
        Vec<T>{from[(3 * k + 2) * nt]}.floats(reinterpret_cast<float *>(v));
#pragma unroll
        for (int i = 0; i < H; ++i) e[i] = fma2(e[i], r, v[i]);
      } else {
#pragma unroll
        for (int i = 0; i < H; ++i) e[i] = mul2(e[i], r);
      }
      Vec<T>::of(reinterpret_cast<const float *>(e)).store(dx + start + k * hop);
    }
    if (on_edge) {
      const float xh = t_edge * now.r;
      acc_edge = fmaf(dy_edge, xh, acc_edge);
      dx[edge] = from_float<T>(fmaf(fmaf(dy_edge, g_edge, -xh * m), now.r, to_float(now.dt)));
    }
    dx += dx_step;
  }
  if (!a.dgamma) return;
  pdl_trigger();
  copies_wait<0>();
  __syncthreads();
  float *sums = reinterpret_cast<float *>(shared);
  uint32_t parts = h.teams;
  const uint32_t apart = SHIFT ? a.cols + a.cols / V + 1 : a.cols;
  if constexpr (SHIFT) {
    // column c at c + c/V, so that threads with V columns each meet in no bank (a team without a row has zeros)
    if (mine < h.teams) {
      float *to = sums + (size_t)mine * apart;
      for (uint32_t c = at; !works && c < apart; c += h.team) to[c] = 0.0f;
#pragma unroll
      for (int k = 0; k < CH; ++k) {
        if (!has(k)) continue;
        float *p = to + start + k * hop + at + k * h.team;
#pragma unroll
        for (int i = 0; i < V; ++i) (head + i < V ? p : p + 1)[i] = reinterpret_cast<const float *>(acc[k])[i];
      }
      if (on_edge) to[edge + edge / V] = acc_edge;
    }
  } else {
    // the teams of a warp join first; a block of one team has its sums in registers
    if (h.team < 32) parts = (h.teams * h.team + 31) / 32;
    const uint32_t part = h.team < 32 ? warp : mine;
    const bool direct = parts == 1 && gridDim.x > 1;
    float *to = direct ? a.partial + (uint64_t)blockIdx.x * a.cols : sums + (size_t)part * a.cols;
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      float *v = reinterpret_cast<float *>(acc[k]);
      for (uint32_t o = h.team; o < 32; o *= 2)
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
      const uint32_t c = start + k * hop;
      if (part >= parts || c >= a.cols || (h.team < 32 && lane >= h.team)) continue;
#pragma unroll
      for (int i = 0; i < V; i += 4) *reinterpret_cast<float4 *>(to + c + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
    }
    if (direct) return;
  }
  __syncthreads();
  for (uint32_t c = threadIdx.x; c < a.cols; c += nt) {
    float sum = 0.0f;
    for (uint32_t t = 0; t < parts; ++t) sum += sums[(size_t)t * apart + (SHIFT ? c + c / V : c)];
    if (gridDim.x == 1) put_weight(a.dgamma, a.gamma.type, c, sum);        // (nothing to join with)
    else a.partial[(uint64_t)blockIdx.x * a.cols + c] = sum;
  }
}

// Any rows: dgamma's partial sums, a thread has a column and every `parts`-th row
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

// The blocks' sums, of few blocks: a thread has a column
constexpr uint32_t kFewParts = 16;
__global__ void __launch_bounds__(kThreads) join_few_kernel(uint32_t cols, uint32_t parts, const float *partial, void *out, int type)
{
  const uint64_t c = (uint64_t)blockIdx.x * kThreads + threadIdx.x;
  pdl_wait();
  if (c >= cols) return;
  float v[kFewParts], sum = 0.0f;
#pragma unroll
  for (uint32_t i = 0; i < kFewParts; ++i) v[i] = i < parts ? partial[(uint64_t)i * cols + c] : 0.0f;
#pragma unroll
  for (uint32_t i = 0; i < kFewParts; ++i) sum += v[i];
  put_weight(out, type, (uint32_t)c, sum);
}

// The blocks' sums: a lane has a column, a warp every eighth block, all of whose sums are asked for at once
__global__ void __launch_bounds__(kThreads) join_columns_kernel(uint32_t cols, uint32_t parts, const float *partial, void *out, int type)
{
  constexpr uint32_t kWarps = kThreads / 32, kEach = (kMostParts + kWarps - 1) / kWarps;
  __shared__ float sums[kWarps][33];
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint64_t c = (uint64_t)blockIdx.x * 32 + lane;
  pdl_wait();
  float v[kEach], sum = 0.0f;
#pragma unroll
  for (uint32_t i = 0; i < kEach; ++i) v[i] = c < cols && warp + kWarps * i < parts ? partial[(uint64_t)(warp + kWarps * i) * cols + c] : 0.0f;
#pragma unroll
  for (uint32_t i = 0; i < kEach; ++i) sum += v[i];
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

#define TRY(call) do { const int rc_ = (call); if (rc_) return rc_; } while (0)

// Whether an array's rows all begin at the same place of a slot of `v` elements as those of the first one
inline bool in_step(const void *p, size_t bytes, uint64_t stride, uint32_t v, const void *p0, size_t bytes0, uint64_t stride0, uint64_t rows)
{
  return !p || ((uintptr_t)p / bytes % v == (uintptr_t)p0 / bytes0 % v && (rows <= 1 || stride % v == stride0 % v));
}

// How the rows of a call are held in registers; false where they are not
bool held_plan(const NormArgs &a, int type, bool quant, Held &h, bool &shift)
{
  const size_t e = type_bytes(type);
  const uint32_t v = (uint32_t)(16 / e);
  if (!in_step(a.residual, e, a.residual_stride, v, a.x, e, a.x_stride, a.rows) || !in_step(a.total, e, a.total_stride, v, a.x, e, a.x_stride, a.rows) ||
      !in_step(a.y, quant ? 1 : e, a.y_stride, v, a.x, e, a.x_stride, a.rows)) return false;
  shift = !aligned_to(a.x, 16) || a.cols % v || (a.rows > 1 && a.x_stride % v) || !aligned_to(a.gamma.p, 16);
  const uint32_t slots = a.cols / v;
  if (slots > 8 * most_threads(8)) return false;
  h.groups = quant && a.block ? (a.cols + 127) / 128 : 0;
  if (slots <= (shift ? 128u : 64u)) {
    h.team = shift ? 16 : 4;              // (a lane for each element before and after whole slots)
    while (h.team < 32 && h.team < slots) h.team *= 2;
    h.chunks = slots <= h.team ? 1 : slots <= 64 ? 2 : 4;
  } else {
    h.chunks = a.rows <= 2 * 148 && slots <= 2048 ? (slots <= 1024 ? 1 : 2) : slots <= 256 ? 2 : slots <= 4 * most_threads(4) ? 4 : 8;
    h.team = (slots + h.chunks * 32 - 1) / (h.chunks * 32) * 32;
  }
  return true;
}

template <typename T, int CH> int launch_held(const NormArgs &a, const Held &h, bool shift, bool quant, cudaStream_t stream)
{
  const uint32_t threads = h.team > 32 ? h.team : 128, per_block = threads / h.team;
  const dim3 grid((uint32_t)((a.rows + per_block - 1) / per_block));
  const size_t shared = shift ? (size_t)per_block * h.groups * 4 : 0;
  auto go = [&](auto form) {
    constexpr int Q = decltype(form)::value;
    return launch(a.residual ? (shift ? rms_norm_held_kernel<T, CH, true, Q, true> : rms_norm_held_kernel<T, CH, false, Q, true>)
                             : (shift ? rms_norm_held_kernel<T, CH, true, Q, false> : rms_norm_held_kernel<T, CH, false, Q, false>), grid, threads, shared, stream, a, h);
  };
  return !quant ? go(std::integral_constant<int, 0>()) : h.groups ? go(std::integral_constant<int, 2>()) : go(std::integral_constant<int, 1>());
}

// How the rows of an adjoint are held on chip: chunks*threads of the kernel; false where they are not
bool grad_plan(const GradArgs &a, int type, HeldGrad &h, uint32_t &chunks, uint32_t &threads, bool &shift)
{
  const size_t e = type_bytes(type);
  const uint32_t v = (uint32_t)(16 / e), slots = a.cols / v;
  if (!in_step(a.total, e, a.total_stride, v, a.dy, e, a.dy_stride, a.rows) || !in_step(a.dtotal, e, a.dtotal_stride, v, a.dy, e, a.dy_stride, a.rows) ||
      !in_step(a.dx, e, a.dx_stride, v, a.dy, e, a.dy_stride, a.rows)) return false;
  shift = !aligned_to(a.dy, 16) || a.cols % v || (a.rows > 1 && a.dy_stride % v) || !aligned_to(a.gamma.p, 16);
  // four slots to a thread, but two where that would be a single team of few warps ([8192,8704] 110 us with four, 97 with two)
  const bool single = !shift && v == 8 && slots > 1024 && slots <= 1536;
  chunks = slots <= 32 ? 1 : slots < 128 || single ? 2 : 4;
  threads = single ? 768 : slots <= 2048 ? 512 : 1024;
  if (slots > (v == 8 ? 2048u : 4096u)) return false;
  h.team = (slots + chunks * 32 - 1) / (chunks * 32) * 32;
  if (slots <= 16) {
    h.team = shift ? 16 : 4;              // (a lane for each element before and after whole slots)
    while (h.team < slots) h.team *= 2;
  }
  if (h.team < 32 && slots > 16) h.team = 32;
  h.teams = threads / h.team;
  if (h.team > 32 && h.teams > 15) h.teams = 15;      // (a named barrier each)
  const uint32_t sms = sm_count();
  // few rows: all in one block, which has nothing to join, or else a row per block first
  if (a.rows <= h.teams) h.teams = (uint32_t)a.rows;
  else if (a.rows < (uint64_t)h.teams * sms) h.teams = (uint32_t)((a.rows + sms - 1) / sms);
  // a single team of many rows leaves out the threads beyond it, whose rings' place gives it more rows ahead; otherwise they help with the sums
  h.threads = h.teams == 1 && a.rows > 4ull * sms ? h.team : threads;
  h.depth = (uint32_t)(226 * 1024 / ((size_t)h.threads * chunks * 48));
  if (h.depth > 4) h.depth = 4;
  return true;
}

int join(const GradArgs &a, int type, cudaStream_t stream)
{
  const uint64_t cols = a.cols;
  return a.parts <= kFewParts ? launch(join_few_kernel, dim3((uint32_t)((cols + kThreads - 1) / kThreads)), kThreads, 0, stream, a.cols, a.parts, a.partial, a.dgamma, type)
                              : launch(join_columns_kernel, dim3((uint32_t)((cols + 31) / 32)), kThreads, 0, stream, a.cols, a.parts, a.partial, a.dgamma, type);
}

template <typename T, int CH, int NT> int launch_grad(const GradArgs &a, const HeldGrad &h, bool shift, cudaStream_t stream)
{
  auto kernel = rms_norm_grad_kernel<T, CH, NT, false>;
  if constexpr (NT != 768) { if (shift) kernel = rms_norm_grad_kernel<T, CH, NT, true>; }       // (ragged rows had no registers for that form)
  const uint32_t threads = h.threads;
  size_t shared = (size_t)h.depth * CH * threads * 48;
  const size_t sums = (size_t)h.teams * (a.cols + (shift ? a.cols / Vec<T>::V + 1 : 0)) * 4;
  if (shared < sums) shared = sums;
  static SharedMemory allowed[2];
  if (!allowed[shift].up_to((const void *)kernel, shared)) return ANODE_E_LAUNCH;
  return launch(kernel, dim3(a.parts), threads, shared, stream, a, h);
}

int norm_forward(const NormArgs &a, int type, int gamma_type, bool quant, cudaStream_t stream)
{
  if (!known_type(type) || (a.gamma.p && !known_type(gamma_type))) return ANODE_E_TYPE;
  if (!served(a.rows, a.cols)) return ANODE_E_DIMS;
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
  const bool held = a.rows < (1ull << 30) && held_plan(a, type, quant, h, shift);
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
                total_stride, nullptr, block, scale, scale_row_stride, scale_group_stride};
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
  if (!served(rows, cols)) return ANODE_E_DIMS;
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
  uint32_t chunks = 0, threads = 0;
  bool shift = false;
  const bool held = grad_plan(a, type, h, chunks, threads, shift);
  const uint32_t wide = (uint32_t)(((uint64_t)cols + kThreads - 1) / kThreads);
  return by_type(type, [&](auto t) {
    using T = decltype(t);
    constexpr uint32_t V = Vec<T>::V;
    if (held) {
      const uint64_t blocks = (rows + h.teams - 1) / h.teams;
      if (a.parts > blocks) a.parts = (uint32_t)blocks;
      h.step = (uint64_t)a.parts * h.teams;
      if (shift && rows > h.step) h.step = h.step / V * V;
      if (chunks == 1) TRY((launch_grad<T, 1, 512>(a, h, shift, stream)));
      else if (chunks == 2 && threads == 512) TRY((launch_grad<T, 2, 512>(a, h, shift, stream)));
      else if (chunks == 2) { if constexpr (sizeof(T) == 2) TRY((launch_grad<T, 2, 768>(a, h, shift, stream))); }
      else if (threads == 512) TRY((launch_grad<T, 4, 512>(a, h, shift, stream)));
      else if constexpr (sizeof(T) == 4) TRY((launch_grad<T, 4, 1024>(a, h, shift, stream)));
      return dgamma && a.parts > 1 ? join(a, gamma_type, stream) : (int)ANODE_OK;
    }
    // dgamma's parts ahead of dx, which may be dy; dgamma, which may be gamma, behind it
    if (dgamma) TRY(launch(rms_norm_dgamma_kernel<T>, dim3(wide, a.parts), kThreads, 0, stream, a));
    TRY(launch(rms_norm_dx_kernel<T>, dim3(row_blocks(rows)), kThreads, 0, stream, a));
    return dgamma ? join(a, gamma_type, stream) : (int)ANODE_OK;
  });
}
