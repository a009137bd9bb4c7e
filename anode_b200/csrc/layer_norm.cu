// Layer norm over rows with the residual's addition: forward and adjoint.
//
//   t = round(x + residual),  mu = mean(t),  r = (mean((t - mu)^2) + epsilon)^-1/2,  y = (t - mu)*r*gamma + beta
//   dx = r*(g - mean(g) - xh*mean(g*xh)) + dt,   g = dy*gamma, xh = (t - mu)*r
//   dgamma = sum over rows of dy*xh,  dbeta = sum over rows of dy
//
// Statistics and sums are f32; the squares are those of the values less their mean, so that a row far from zero keeps its spread.
// y, total and dx are rounded once, total before the norm reads it.
//
// Bound by memory where there are many rows, by the chain launch -> load -> sum -> sum -> store where there are few, and in the adjoint by the latency of its
// instructions (sums of two weights' gradients leave a multiprocessor 16 warps).  Measured on one B200 against its copy bandwidth of 6539 GB/s, with residual, on the device in runs
// of some ms (what is above that bandwidth was still in the second-level cache when the clock stopped; in a loop of calls the first takes 170 us, 0.96):
//   forward   bf16 [16384,8192] 157 to 160 us (1.03 of it), [16384,2048] 43 us (0.95), [1,4096] 2.2 us; f32 [4099,1001] without a residual 11.3 to 13.9 us (a copy of it 11.2 to 12.7)
//   adjoint   bf16 [8192,4096] 51 us (0.80), [8192,16384] 178 us (0.92), [8192,4095] 69 us (0.60); f32 [4096,8192] 86 us (0.96), [4096,16384] 254 us (0.65: gamma is
//             read anew for every row); f16 [2047,1535] 17 us; bf16 rows with f32 weights, whose gamma is read anew, too, [8192,2048] 40 us (30 with bf16 weights),
//             [8192,4096] 70 (0.59), [8192,8192] 137 (93)
// Three kernels, as the RMS norm has: rows held in registers, the adjoint through rings of asynchronous copies, and plain ones, element by element, for rows that
// are too wide or do not begin in step.  Tried and dropped: the next row's sums ahead of this row's gradient (65 us in the place of 55 for [8192,4096]); the
// single row of a ring refilled slot by slot (287 us in the place of 254 for f32 [4096,16384]); joins of a block's warps by loads in the place of shuffles
// ([1,4096] 2.55 us in the place of 2.2).
#include "bn_host.h"
#include "rows.cuh"

namespace anode_b200 {
namespace rows {
namespace layer_norm {

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

// The launch of the kernel that holds its rows
struct Held {
  uint32_t team, chunks;     // threads of a row, slots of each
};

__host__ __device__ constexpr uint32_t most_threads(int chunks) { return chunks == 1 ? 1024u : chunks <= 4 ? 512u : 640u; }

// Rows held in registers: a team of threads (4 to 32 lanes of a warp, or a block) has a row, a thread CH slots of 16 bytes, so that the
// row is read once; the second sum is of what is in registers.  SHIFT: rows that begin anywhere or are no whole number of slots, as long as all
// arrays' rows begin at the same place of a slot: slots are then those of the addresses, and the elements before the first whole one and
// after the last have a lane each.
template <typename T, int CH, bool SHIFT, bool RES>
__global__ void __launch_bounds__(most_threads(CH)) layer_norm_held_kernel(const LayerArgs a, const Held h)
{
  constexpr int V = Vec<T>::V, H = V / 2;
  __shared__ float buf[2][32];
  const uint32_t per_block = blockDim.x / h.team, mine = threadIdx.x / h.team, at = threadIdx.x - mine * h.team;
  const uint64_t row = (uint64_t)blockIdx.x * per_block + mine;
  const bool live = row < a.rows;               // (all threads take part in the teams' sums)
  const T *x = static_cast<const T *>(a.x) + row * a.x_stride;
  const T *res = RES ? static_cast<const T *>(a.residual) + row * a.residual_stride : nullptr;
  T *total = RES && a.total ? static_cast<T *>(a.total) + row * a.total_stride : nullptr;
  // the row's head: columns before its first whole slot; then `slots` of them, and a tail
  const uint32_t head = SHIFT ? min(a.cols, (uint32_t)(-(int)((uintptr_t)x / sizeof(T)) & (V - 1))) : 0, slots = (a.cols - head) / V;
  const uint32_t start = head + at * V, hop = h.team * V;      // this thread's slots: columns start + k*hop
  const int mine_slots = live && at < slots ? (int)((slots - at + h.team - 1) / h.team) : 0;
  // the lane's element of the head or the tail
  const uint32_t tail = a.cols - head - slots * V, edge = at < head ? at : a.cols - tail + (at - head);
  const bool on_edge = SHIFT && live && at < head + tail;
  const bool aligned = (((uintptr_t)a.gamma.p | (uintptr_t)a.beta.p) & 15) == 0;
  pdl_wait();
  pdl_trigger();
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
  float te = 0.0f, ge = 1.0f, be = 0.0f;
  if (on_edge) {
    te = to_float(x[edge]);
    if (RES) te = to_float(from_float<T>(te + to_float(res[edge])));
    ge = a.gamma.at(edge);
    if (a.beta.p) be = a.beta.at(edge);
  }
  auto weights = [&](const Weights &from, int k, float2 *w) {
    float *f = reinterpret_cast<float *>(w);
    const uint32_t c = start + k * hop;
    if (!SHIFT) from.load<V>(c, f);
    else if (aligned) from.load_any<V>(c, a.cols, f);
    else from.load_each<V>(c, f);
  };
  // the weights of few slots are loaded ahead of the sums, those of more when they are needed: they would take the registers
  constexpr bool AHEAD = CH <= 2;
  float2 g[AHEAD ? CH : 1][H], b[AHEAD ? CH : 1][H];
  auto both_weights = [&](int k) {
    float2 *const gk = g[AHEAD ? k : 0], *const bk = b[AHEAD ? k : 0];
    weights(a.gamma, k, gk);
    if (a.beta.p) weights(a.beta, k, bk);
    else {
#pragma unroll
      for (int i = 0; i < H; ++i) bk[i] = both(0.0f);
    }
  };
  if (AHEAD) {
#pragma unroll
    for (int k = 0; k < CH; ++k) if (k < mine_slots) both_weights(k);
  }
  float2 sum = make_float2(te, 0.0f);
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
    for (int i = 0; i < H; ++i) sum = add2(sum, f[i]);
  }
  if (on_edge && total) total[edge] = from_float<T>(te);
  const float mean = team_sum_all(sum.x + sum.y, h.team, buf[0]) * a.inv_cols;
  const float2 minus = both(-mean);
  float2 sq = both(0.0f);
#pragma unroll
  for (int k = 0; k < CH; ++k) {
    if (k >= mine_slots) continue;
    float2 f[H];
    t[k].floats(reinterpret_cast<float *>(f));
#pragma unroll
    for (int i = 0; i < H; ++i) { const float2 d = add2(f[i], minus); sq = fma2(d, d, sq); }
  }
  const float de = on_edge ? te - mean : 0.0f;
  const float inv = 1.0f / sqrtf(team_sum_all(fmaf(de, de, sq.x + sq.y), h.team, buf[1]) * a.inv_cols + a.epsilon);
  if (live && at == 0) {
    if (a.mean) a.mean[row] = mean;
    if (a.inv_std) a.inv_std[row] = inv;
  }
  const float2 inv2 = both(inv);
  T *y = static_cast<T *>(a.y) + row * a.y_stride;
#pragma unroll
  for (int k = 0; k < CH; ++k) {
    if (k >= mine_slots) continue;
    float2 f[H];
    t[k].floats(reinterpret_cast<float *>(f));
    if (!AHEAD) both_weights(k);
#pragma unroll
    for (int i = 0; i < H; ++i) f[i] = fma2(mul2(add2(f[i], minus), inv2), g[AHEAD ? k : 0][i], b[AHEAD ? k : 0][i]);
    Vec<T>::of(reinterpret_cast<const float *>(f)).store(y + start + k * hop);
  }
  if (on_edge) y[edge] = from_float<T>(fmaf(de * inv, ge, be));
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

constexpr uint32_t kGradThreads = 512;
constexpr size_t kMostShared = 226 * 1024;       // of a block, beside a kernel's own arrays

// How the adjoint's rows are held: `teams` teams of `team` threads to a block, each with a row at a time, `depth` rows on their way or at work;
// a team's rows lie `step` apart
struct HeldGrad {
  uint32_t team, teams, depth, threads;
  uint64_t step;
};

// Sums of two numbers over a team, in every thread.  The first half leaves those of a team of up to 32 lanes in each of them, and of more warps in `buf`; the
// second half, behind a barrier of the team, takes them from there.
__device__ __forceinline__ float2 pair_sum_begin(float2 v, uint32_t lanes, uint32_t team, float2 *buf)
{
  for (uint32_t o = min(team, 32u) / 2; o > 0; o >>= 1) { v.x += __shfl_xor_sync(lanes, v.x, o); v.y += __shfl_xor_sync(lanes, v.y, o); }
  if (team > 32 && (threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
  return v;
}
__device__ __forceinline__ float2 pair_sum_end(float2 v, uint32_t team, uint32_t mine, uint32_t wide, const float2 *buf)
{
  if (team <= 32) return v;
  asm volatile("bar.sync %0, %1;" ::"r"(mine + 1), "r"(team) : "memory");
  const uint32_t warps = team / 32, at = threadIdx.x & (wide - 1);       // wide: the power of two from `warps` on
  v = at < warps ? buf[mine * warps + at] : make_float2(0.0f, 0.0f);
  for (uint32_t o = wide / 2; o > 0; o >>= 1) { v.x += __shfl_xor_sync(0xffffffffu, v.x, o); v.y += __shfl_xor_sync(0xffffffffu, v.y, o); }
  return v;
}

// The adjoint with its rows held on chip: a team of threads (4 to 32 lanes of a warp, or more warps) walks down rows, a thread with CH slots of 16
// bytes of each array, so that one pass gives dx and the sums of dgamma and dbeta.  The next rows are on their way by asynchronous copies, each thread into
// a ring of its own: a thread waits for nothing but its own copies and, once per row, its team's sums. 
// A thread's columns are the same in all of its team's rows, whose sums are in its registers; gamma is there, too (G = 0), or else as it lies in memory in the
// shared one (G = 1, if it has the rows' type) or read anew for every row (G = 2).
// SHIFT, as in layer_norm_held_kernel: rows that begin at different places of a slot do so in turns of at most V, so a team's rows lie a multiple
// of V apart and begin at the same one.
// The sums join in a fixed order, the teams' in shared memory and the blocks' in a second launch.
template <typename T, int CH, bool SHIFT, int G>
__global__ void __launch_bounds__(kGradThreads) layer_norm_grad_kernel(const LayerGradArgs a, const HeldGrad h)
{
  constexpr int V = Vec<T>::V, H = V / 2;
  constexpr bool GREGS = G == 0;
  __shared__ float2 buf[2][32];
  extern __shared__ float4 shared[];            // the rings [depth][CH][3][thread], gamma [CH][thread]; at last the sums [teams][2][cols]
  const uint32_t mine = threadIdx.x / h.team, at = threadIdx.x - mine * h.team, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint64_t row0 = (uint64_t)blockIdx.x * h.teams + mine;
  const bool works = mine < h.teams && row0 < h.step && row0 < a.rows;
  const uint32_t lanes = h.team < 32 ? ((1u << h.team) - 1) << (lane & ~(h.team - 1)) : 0xffffffffu;      // of this warp in the team
  constexpr uint32_t NT = kGradThreads;         // (rings lie as far apart whatever the block's threads)
  uint4 *ring = reinterpret_cast<uint4 *>(shared) + threadIdx.x;
  const T *dy = static_cast<const T *>(a.dy) + row0 * a.dy_stride, *t = static_cast<const T *>(a.total) + row0 * a.total_stride;
  const T *dt = static_cast<const T *>(a.dtotal) + row0 * a.dtotal_stride;
  T *dx = static_cast<T *>(a.dx) + row0 * a.dx_stride;
  const float *inv = a.inv_std + row0, *mean = a.mean + row0;
  // a row's columns before its first whole slot, and what remains behind the last one; this thread's slots, and its element of those
  const uint32_t head = SHIFT ? min(a.cols, (0u - (uint32_t)((uintptr_t)dy / sizeof(T))) & (V - 1)) : 0, slots = (a.cols - head) / V;
  const uint32_t tail = a.cols - head - slots * V, edge = at < head ? at : a.cols - tail + (at - head), start = head + at * V, hop = h.team * V;
  const bool on_edge = SHIFT && works && at < head + tail;
  auto has = [&](int k) { return works && at + k * h.team < slots; };
  pdl_wait();
  float2 dg[CH][H], db[CH][H], gs[GREGS ? CH : 1][H];
  float dg_edge = 0.0f, db_edge = 0.0f, g_edge = on_edge ? a.gamma.at(edge) : 0.0f;
  const bool aligned_gamma = ((uintptr_t)a.gamma.p & 15) == 0;
  uint4 *gamma_here = ring + h.depth * (CH * 3) * NT;
  auto gamma = [&](int k, float2 *to) {
    float *w = reinterpret_cast<float *>(to);
    if (G == 1) Vec<T>{gamma_here[k * NT]}.floats(w);
    else if (!SHIFT) a.gamma.load<V>(start + k * hop, w);
    else if (aligned_gamma) a.gamma.load_any<V>(start + k * hop, a.cols, w);
    else a.gamma.load_each<V>(start + k * hop, w);
  };
  if constexpr (G == 1) {               // (each thread reads what it stored itself)
    const T *from = static_cast<const T *>(a.gamma.p) + start;
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      if (!has(k)) continue;
      if (!SHIFT) gamma_here[k * NT] = Vec<T>::load(from + k * hop).bits;
      else {
#pragma unroll
        for (int i = 0; i < V; ++i) reinterpret_cast<T *>(gamma_here + k * NT)[i] = from[k * hop + i];
      }
    }
  }
#pragma unroll
  for (int k = 0; k < CH; ++k) {
#pragma unroll
    for (int i = 0; i < H; ++i) dg[k][i] = db[k][i] = both(0.0f);
    if constexpr (GREGS) {
#pragma unroll
      for (int i = 0; i < H; ++i) gs[k][i] = both(0.0f);
      if (has(k)) gamma(k, gs[k]);
    }
  }
  // rows that this team has: at work, and to be copied
  uint32_t left = works ? (uint32_t)((a.rows - row0 + h.step - 1) / h.step) : 0, ahead = left, in = 0, out = 0;
  const uint64_t dy_step = h.step * a.dy_stride, t_step = h.step * a.total_stride, dt_step = h.step * a.dtotal_stride, dx_step = h.step * a.dx_stride;
  // what does not go through the ring, of the row that is worked on next: mean and 1/std, and an element of the head or the tail
  // (as it lies in memory: nothing waits for it before its row's turn)
  struct Side { float r, mu; T dy, t, dt; } now = {}, next = {};
  const T *dy1 = dy + edge, *t1 = t + edge, *dt1 = dt + edge;
  auto side = [&](Side &o) {
    o.r = *inv; o.mu = *mean;
    inv += h.step; mean += h.step;
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
      uint4 *to = ring + in * (CH * 3) * NT;
#pragma unroll
      for (int k = 0; k < CH; ++k) {
        if (!has(k)) continue;
        copy_async<16>(to + (3 * k) * NT, dy + k * hop);
        copy_async<16>(to + (3 * k + 1) * NT, t + k * hop);
        if (a.dtotal) copy_async<16>(to + (3 * k + 2) * NT, dt + k * hop);
      }
      --ahead;
      dy += dy_step; t += t_step; dt += dt_step;
    }
    copies_commit();
    in = in + 1 == h.depth ? 0 : in + 1;
  };
  auto row_of = [&](uint32_t place) { return ring + place * (CH * 3) * NT; };
  // this thread's part of a row's two sums: of g, and of g*(t - mu)
  auto sums_of = [&](const uint4 *from, const Side &o) {
    const float dy_edge = to_float(o.dy), t_edge = to_float(o.t) - o.mu;
    const float2 away = both(-o.mu);
    float2 sum2 = make_float2(SHIFT ? dy_edge * g_edge : 0.0f, 0.0f), dot2 = make_float2(SHIFT ? dy_edge * g_edge * t_edge : 0.0f, 0.0f);
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      if (!has(k)) continue;
      float2 u[H], v[H], w[H];
      if constexpr (!GREGS) gamma(k, w);
      Vec<T>{from[(3 * k) * NT]}.floats(reinterpret_cast<float *>(u));
      Vec<T>{from[(3 * k + 1) * NT]}.floats(reinterpret_cast<float *>(v));
#pragma unroll
      for (int i = 0; i < H; ++i) {
        const float2 g = mul2(u[i], GREGS ? gs[GREGS ? k : 0][i] : w[i]);
        sum2 = add2(sum2, g);
        dot2 = fma2(g, add2(v[i], away), dot2);
      }
    }
    return make_float2(sum2.x + sum2.y, dot2.x + dot2.y);
  };
  // its part of dx, and what the row adds to dgamma and dbeta
  auto gradient_of = [&](const uint4 *from, const Side &o, float2 all) {
    // (1/std meets the sum, a row's element and the bracket one at a time: its powers alone would leave f32's range where rows are large or tiny)
    const float s = all.x * a.inv_cols, m = all.y * o.r * a.inv_cols;
    const float2 r = both(o.r), minus = both(-m), less = both(-s), away = both(-o.mu);
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      if (!has(k)) continue;
      float2 u[H], v[H], w[H], e[H];
      if constexpr (!GREGS) gamma(k, w);
      Vec<T>{from[(3 * k) * NT]}.floats(reinterpret_cast<float *>(u));
      Vec<T>{from[(3 * k + 1) * NT]}.floats(reinterpret_cast<float *>(v));
#pragma unroll
      for (int i = 0; i < H; ++i) {
        const float2 xh = mul2(add2(v[i], away), r);
        dg[k][i] = fma2(u[i], xh, dg[k][i]);
        db[k][i] = add2(db[k][i], u[i]);
        e[i] = fma2(u[i], GREGS ? gs[GREGS ? k : 0][i] : w[i], fma2(xh, minus, less));
      }
      if (a.dtotal) {
        Vec<T>{from[(3 * k + 2) * NT]}.floats(reinterpret_cast<float *>(v));
#pragma unroll
        for (int i = 0; i < H; ++i) e[i] = fma2(e[i], r, v[i]);
      } else {
#pragma unroll
        for (int i = 0; i < H; ++i) e[i] = mul2(e[i], r);
      }
      Vec<T>::of(reinterpret_cast<const float *>(e)).store(dx + start + k * hop);
    }
    if (on_edge) {
      const float dy_edge = to_float(o.dy), xh = (to_float(o.t) - o.mu) * o.r;
      dg_edge = fmaf(dy_edge, xh, dg_edge);
      db_edge += dy_edge;
      dx[edge] = from_float<T>(fmaf(fmaf(dy_edge, g_edge, fmaf(-xh, m, -s)), o.r, to_float(o.dt)));
    }
    dx += dx_step;
  };
  auto wait_but = [&](uint32_t rows) { if (rows == 3) copies_wait<3>(); else if (rows == 2) copies_wait<2>(); else if (rows == 1) copies_wait<1>(); else copies_wait<0>(); };
  uint32_t wide = 1;
  while (wide < h.team / 32) wide *= 2;
  for (uint32_t i = 1; i < h.depth; ++i) copy();
  uint32_t turn = 0;
  if (left) side(next);
  for (; left; --left, turn ^= 1) {
    now = next;
    copy();
    if (left > 1) side(next);
    wait_but(h.depth - 1);
    const uint4 *from = row_of(out);
    out = out + 1 == h.depth ? 0 : out + 1;
    const float2 part = pair_sum_begin(sums_of(from, now), lanes, h.team, buf[turn]);
    gradient_of(from, now, pair_sum_end(part, h.team, mine, wide, buf[turn]));
  }
  if (!a.dgamma && !a.dbeta) return;
  pdl_trigger();
  copies_wait<0>();
  __syncthreads();
  // dgamma's sums, then dbeta's
  float *sums = reinterpret_cast<float *>(shared);
  uint32_t parts = h.teams;
  const uint32_t apart = SHIFT ? a.cols + a.cols / V + 1 : a.cols;
  if constexpr (SHIFT) {
    // column c at c + c/V, so that threads with V columns each meet in no bank (a team without a row has zeros)
    if (mine < h.teams) {
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        float *to = sums + (size_t)(2 * mine + which) * apart;
        for (uint32_t c = at; !works && c < apart; c += h.team) to[c] = 0.0f;
#pragma unroll
        for (int k = 0; k < CH; ++k) {
          if (!has(k)) continue;
          float *p = to + start + k * hop + at + k * h.team;
#pragma unroll
          for (int i = 0; i < V; ++i) (head + i < V ? p : p + 1)[i] = reinterpret_cast<const float *>(which ? db[k] : dg[k])[i];
        }
        if (on_edge) to[edge + edge / V] = which ? db_edge : dg_edge;
      }
    }
  } else {
    // the teams of a warp join first; a block of one team has its sums in registers
    if (h.team < 32) parts = (h.teams * h.team + 31) / 32;
    const uint32_t part = h.team < 32 ? warp : mine;
    const bool direct = parts == 1 && gridDim.x > 1;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      float *to = direct ? a.partial + ((uint64_t)blockIdx.x * 2 + which) * a.cols : sums + (size_t)(2 * part + which) * a.cols;
#pragma unroll
      for (int k = 0; k < CH; ++k) {
        float *v = reinterpret_cast<float *>(which ? db[k] : dg[k]);
        for (uint32_t o = h.team; o < 32; o *= 2)
#pragma unroll
          for (int i = 0; i < V; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
        const uint32_t c = start + k * hop;
        if (part >= parts || c >= a.cols || (h.team < 32 && lane >= h.team)) continue;
#pragma unroll
        for (int i = 0; i < V; i += 4) *reinterpret_cast<float4 *>(to + c + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
      }
    }
    if (direct) return;
  }
  __syncthreads();
  for (uint32_t c = threadIdx.x; c < a.cols; c += blockDim.x) {
    float sum[2] = {0.0f, 0.0f};
    for (uint32_t t = 0; t < parts; ++t)
#pragma unroll
      for (int which = 0; which < 2; ++which) sum[which] += sums[(size_t)(2 * t + which) * apart + (SHIFT ? c + c / V : c)];
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      void *to = which ? a.dbeta : a.dgamma;
      if (gridDim.x > 1) a.partial[((uint64_t)blockIdx.x * 2 + which) * a.cols + c] = sum[which];
      else if (to) put_weight(to, a.dweight_type, c, sum[which]);        // (nothing to join with)
    }
  }
}

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

// How the rows of a call are held in registers; false where they are not
bool held_plan(const LayerArgs &a, int type, Held &h, bool &shift)
{
  const size_t e = type_bytes(type);
  const uint32_t v = (uint32_t)(16 / e);
  if (!in_step(a.residual, e, a.residual_stride, v, a.x, e, a.x_stride, a.rows) || !in_step(a.total, e, a.total_stride, v, a.x, e, a.x_stride, a.rows) ||
      !in_step(a.y, e, a.y_stride, v, a.x, e, a.x_stride, a.rows)) return false;
  shift = !aligned_to(a.x, 16) || a.cols % v || (a.rows > 1 && a.x_stride % v) || !aligned_to(a.gamma.p, 16) || !aligned_to(a.beta.p, 16);
  const uint32_t slots = a.cols / v;
  if (slots > 8 * most_threads(8)) return false;
  if (slots <= 128) {
    h.team = shift ? 16 : 4;              // (a lane for each element before and after whole slots)
    while (h.team < 32 && h.team < slots) h.team *= 2;
    h.chunks = slots <= h.team ? 1 : slots <= 64 ? 2 : 4;
  } else {
    // few rows: short chains with the weights ahead ([600,2000] bf16 4.4 us with two slots to a thread, 5.4 with four); many: more bytes in flight
    // for a thread's registers ([16384,2048] 49.5 us with two, 43.1 with four)
    h.chunks = a.rows <= 2 * 148 && slots <= 1024 ? 1 : a.rows <= 8 * 148 && slots <= 256 ? 2 : slots <= 4 * most_threads(4) ? 4 : 8;
    h.team = (slots + h.chunks * 32 - 1) / (h.chunks * 32) * 32;
  }
  return true;
}

template <typename T, int CH> int launch_held(const LayerArgs &a, const Held &h, bool shift, cudaStream_t stream)
{
  const uint32_t threads = h.team > 32 ? h.team : 128, per_block = threads / h.team;
  const dim3 grid((uint32_t)((a.rows + per_block - 1) / per_block));
  return launch(a.residual ? (shift ? layer_norm_held_kernel<T, CH, true, true> : layer_norm_held_kernel<T, CH, false, true>)
                           : (shift ? layer_norm_held_kernel<T, CH, true, false> : layer_norm_held_kernel<T, CH, false, false>), grid, threads, 0, stream, a, h);
}

// How the rows of an adjoint are held on chip; false where they are not
bool grad_plan(const LayerGradArgs &a, int type, int weight_type, HeldGrad &h, uint32_t &chunks, bool &shift, int &g)
{
  const size_t e = type_bytes(type);
  const uint32_t v = (uint32_t)(16 / e), slots = a.cols / v, threads = kGradThreads;
  if (!in_step(a.total, e, a.total_stride, v, a.dy, e, a.dy_stride, a.rows) || !in_step(a.dtotal, e, a.dtotal_stride, v, a.dy, e, a.dy_stride, a.rows) ||
      !in_step(a.dx, e, a.dx_stride, v, a.dy, e, a.dy_stride, a.rows)) return false;
  shift = !aligned_to(a.dy, 16) || a.cols % v || (a.rows > 1 && a.dy_stride % v) || !aligned_to(a.gamma.p, 16);
  // four slots to a thread amortize its row's joins ([8192,4096] bf16 51 us, 55 with two), but ragged rows of 16-bit types have no registers for them ([8192,4095] 81
  // us with four, 67 to 69 with two)
  chunks = slots <= 32 ? 1 : slots < 128 || (shift && v == 8 && slots <= 1024) ? 2 : slots <= 2048 ? 4 : 8;
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
  // a single team of many rows leaves out the threads beyond it, whose places in the rings stay empty (f32 [4096,4608] 54.5 us, 56.4 with them; [4096,10240] 183 and 186; bf16
  // [4096,8704] 75 either way); otherwise they help with the sums.  Rings at the block's own distance, which hold more rows of such a team, were slower for what an address then
  // costs: bf16 [4096,8704] 81 us, [4096,11264] 86 (79), f32 [4096,4224] 56 (52), [4096,8704] 199 (164), though f32 [4096,10240] took 169 so (184) and [4096,12288] 187 (203)
  h.threads = h.teams == 1 && a.rows > 4ull * sms ? h.team : threads;
  // gamma in registers, or its slots beside the ring if they are the rows' and leave it two rows
  const size_t slot = (size_t)kGradThreads * chunks * 16;
  g = chunks * v <= 16 ? 0 : a.gamma.p && type == weight_type && 7 * slot <= kMostShared ? 1 : 2;
  h.depth = (uint32_t)((kMostShared - (g == 1 ? slot : 0)) / (3 * slot));
  if (h.depth > 4) h.depth = 4;
  return true;
}

template <typename T, int CH, int G> int launch_grad(const LayerGradArgs &a, const HeldGrad &h, bool shift, size_t shared, cudaStream_t stream)
{
  auto kernel = shift ? layer_norm_grad_kernel<T, CH, true, G> : layer_norm_grad_kernel<T, CH, false, G>;
  static SharedMemory allowed[2];
  if (!allowed[shift].up_to((const void *)kernel, shared)) return ANODE_E_LAUNCH;
  return launch(kernel, dim3(a.parts), h.threads, shared, stream, a, h);
}
template <typename T, int CH> int launch_grad(const LayerGradArgs &a, const HeldGrad &h, bool shift, int g, cudaStream_t stream)
{
  size_t shared = ((size_t)h.depth * 3 + (g == 1)) * CH * kGradThreads * 16;
  const size_t sums = (size_t)h.teams * (a.cols + (shift ? a.cols / Vec<T>::V + 1 : 0)) * 8;
  if (shared < sums) shared = sums;
  if constexpr (CH * Vec<T>::V <= 16) return launch_grad<T, CH, 0>(a, h, shift, shared, stream);
  else return g == 1 ? launch_grad<T, CH, 1>(a, h, shift, shared, stream) : launch_grad<T, CH, 2>(a, h, shift, shared, stream);
}

}  // namespace layer_norm
}  // namespace rows
}  // namespace anode_b200

using namespace anode_b200::rows;
using namespace anode_b200::rows::layer_norm;

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
    if (rows_meet(total, total_stride * e, rows, cols * e, y, y_stride * e, rows, cols * e) || !apart(total, total_stride, x, x_stride, rows) || !apart(total, total_stride, residual, residual_stride, rows)) return ANODE_E_STRIDE;
  }
  if (!apart(y, y_stride, x, x_stride, rows) || !apart(y, y_stride, residual, residual_stride, rows)) return ANODE_E_STRIDE;
  if (!aligned_to(mean, 4) || !aligned_to(inv_std, 4)) return ANODE_E_ALIGN;
  if (overlap(mean, 4 * rows, inv_std, 4 * rows)) return ANODE_E_STRIDE;
  const LayerArgs a = {rows, cols, epsilon, 1.0f / (float)cols, x, residual, x_stride, residual_stride, {gamma, weight_type}, {beta, weight_type},
                       y, total, y_stride, total_stride, mean, inv_std};
  Held h = {};
  bool shift = false;
  const bool held = a.rows < (1ull << 30) && held_plan(a, type, h, shift);
  return by_type(type, [&](auto t) {
    using T = decltype(t);
    if (held) return h.chunks == 1 ? launch_held<T, 1>(a, h, shift, stream) : h.chunks == 2 ? launch_held<T, 2>(a, h, shift, stream)
                   : h.chunks == 4 ? launch_held<T, 4>(a, h, shift, stream) : launch_held<T, 8>(a, h, shift, stream);
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
    // the gradients apart from each other and from gamma, in whose very place dgamma may be
    const uint64_t bytes = (uint64_t)cols * type_bytes(weight_type);
    if (overlap(dgamma, bytes, dbeta, bytes) || overlap(dbeta, bytes, gamma, bytes) || (dgamma != gamma && overlap(dgamma, bytes, gamma, bytes))) return ANODE_E_STRIDE;
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
  LayerGradArgs a = {rows, cols, 1.0f / (float)cols, dy, total, dtotal, dy_stride, total_stride, dtotal_stride, mean, inv_std, {gamma, weight_type},
                     dx, dx_stride, dgamma, dbeta, weight_type, static_cast<float *>(workspace), parts_of(rows)};
  HeldGrad h = {};
  uint32_t chunks = 0;
  bool shift = false;
  int g = 0;
  const bool held = grad_plan(a, type, weight_type, h, chunks, shift, g);
  const uint32_t wide = (uint32_t)(((uint64_t)cols + kThreads - 1) / kThreads);
  auto join = [&] {
    return launch(join_weights_kernel, dim3((uint32_t)(((uint64_t)cols + 31) / 32), 2), kThreads, 0, stream, cols, a.parts, (const float *)a.partial, dgamma, dbeta, weight_type);
  };
  return by_type(type, [&](auto t) {
    using T = decltype(t);
    constexpr uint32_t V = Vec<T>::V;
    if (held) {
      const uint64_t blocks = (rows + h.teams - 1) / h.teams;
      if (a.parts > blocks) a.parts = (uint32_t)blocks;
      h.step = (uint64_t)a.parts * h.teams;
      if (shift && rows > h.step) h.step = h.step / V * V;
      if (chunks == 1) TRY((launch_grad<T, 1>(a, h, shift, g, stream)));
      else if (chunks == 2) TRY((launch_grad<T, 2>(a, h, shift, g, stream)));
      else if (chunks == 4) TRY((launch_grad<T, 4>(a, h, shift, g, stream)));
      else if constexpr (V == 4) TRY((launch_grad<T, 8>(a, h, shift, g, stream)));
      return sums && a.parts > 1 ? join() : (int)ANODE_OK;
    }
    // the weights' parts ahead of dx, which may be dy; dgamma, which may be gamma, behind it
    if (sums) TRY(launch(layer_norm_dweights_kernel<T>, dim3(wide, a.parts), kThreads, 0, stream, a));
    TRY(launch(layer_norm_dx_kernel<T>, dim3(row_blocks(rows)), kThreads, 0, stream, a));
    return sums ? join() : (int)ANODE_OK;
  });
}
