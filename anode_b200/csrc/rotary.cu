// Rotary positions of queries and keys, with the RMS norm of each head before them: forward and adjoint.
//
//   n = x*r*gamma, r = (mean(x^2) + epsilon)^-1/2 over the head;   angle = position*freq[i]
//   (n[u], n[v]) -> A*(n[u] cos - n[v] sin, n[u] sin + n[v] cos);   backward: the same with -sin, then the norm's adjoint
//
// A head is read once and written once.  It belongs to a group of lanes of a warp; a lane has ITEMS of 2V elements each: V pairs,
// or 2V elements that pass.  In the half layout an item is two vectors rot/2 apart, so that both elements of a pair are in one lane and the
// turn needs no exchange; only the norm's sums go across the group.  Lanes keep their items from head to head, and with them the
// weights and the sums of the weights' gradients.
// A block has a few tokens of the queries or of the keys at a time: it makes their cosines and sines once, in shared memory, for all of
// their heads, while the first heads are on their way.
#include "bn_host.h"
#include "rows.cuh"

namespace anode_b200 {
namespace rows {

constexpr uint32_t kThreads = 256, kMostDim = 1024;
constexpr uint32_t kMostParts = 148 * 4;      // blocks that have sums of the weights' gradients
constexpr uint32_t kMostTokens = 64;          // of a block at a time

struct HeadArray {
  void *p;
  uint64_t batch, seq, head;
};
// One of the two arrays' geometry
struct RotarySide {
  HeadArray in, x, out;                // backward: in = dout, x = the norm's input, out = dx
  Weights gamma;
  uint32_t heads;
  uint32_t tokens;                     // of a block at a time
  uint32_t blocks, want;               // blocks of the grid; whether the weights' gradient is asked for
};
struct RotaryArgs {
  uint32_t batch, seq, dim, rot, interleaved;
  float amplitude, epsilon, inv_dim;
  const double *freq;
  const void *positions;
  uint32_t position_bytes;
  uint64_t pos_batch, pos_seq;
  uint64_t total;                      // tokens
  uint32_t norm;
  RotarySide side[2];
  float *partial;                      // [blocks, dim] of the gradients of the weights
  uint32_t lanes, items, turned;       // lanes of a head's group; items of a head, and those of them that turn
  float way;                           // 1 forward, -1 back
};

// V elements, moved at once
template <int BYTES> struct RawOf;
template <> struct RawOf<16> { typedef uint4 type; };
template <> struct RawOf<8> { typedef uint2 type; };
template <> struct RawOf<4> { typedef uint32_t type; };
template <> struct RawOf<2> { typedef uint16_t type; };
template <typename T, int V> struct Few {
  union { typename RawOf<V * sizeof(T)>::type raw; T e[V]; };
  __device__ __forceinline__ Few() {}
  __device__ __forceinline__ void load(const T *p) { raw = *reinterpret_cast<const decltype(raw) *>(p); }
  __device__ __forceinline__ void clear() { raw = decltype(raw){}; }
  __device__ __forceinline__ void store(T *p) const { *reinterpret_cast<decltype(raw) *>(p) = raw; }
  __device__ __forceinline__ void floats(float *f) const
  {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = to_float(e[i]);
  }
  __device__ __forceinline__ void of(const float *f)
  {
#pragma unroll
    for (int i = 0; i < V; ++i) e[i] = from_float<T>(f[i]);
  }
};

__device__ __forceinline__ double position_of(const RotaryArgs &a, uint64_t token)
{
  const uint64_t b = a.batch == 1 ? 0 : token / a.seq, i = b * a.pos_batch + (token - b * a.seq) * a.pos_seq;
  return a.position_bytes == 8 ? (double)static_cast<const long long *>(a.positions)[i] : (double)static_cast<const int *>(a.positions)[i];
}
// cos and sin of position*freq, by whole turns in f64: what is left of them is exact, and small
__device__ __forceinline__ float2 turn_of(double position, double freq, float amplitude)
{
  const double turns = position * (freq * 0.15915494309189533577);      // 1/(2 pi)
  float s, c;
  sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
  return make_float2(c * amplitude, s * amplitude);
}

template <typename T, int V, int IT, bool NORM, bool BWD>
__global__ void __launch_bounds__(kThreads) rotary_heads_kernel(const RotaryArgs a)
{
  // [tokens][rot/2] cosines and sines, pair j = item*V + i of a token at (i/2*turned + item)*2 + i%2, so that lanes read 16 bytes side by
  // side; behind them the sums of the weights' gradients, when the block is done
  extern __shared__ float4 shared[];
  float2 *table = reinterpret_cast<float2 *>(shared);
  const uint32_t which = blockIdx.x >= a.side[0].blocks, block = which ? blockIdx.x - a.side[0].blocks : blockIdx.x;
  const RotarySide &d = a.side[which];
  const uint32_t lane = threadIdx.x & (a.lanes - 1), group = threadIdx.x / a.lanes, groups = kThreads / a.lanes, half = a.rot / 2;
  // this lane's items: two vectors, at e0 and e1
  uint32_t e0[IT], e1[IT];
  bool has[IT], second[IT], turns[IT];
#pragma unroll
  for (int k = 0; k < IT; ++k) {
    const uint32_t p = lane + k * a.lanes;
    turns[k] = p < a.turned;
    has[k] = p < a.items;
    e0[k] = !turns[k] ? a.rot + (p - a.turned) * 2 * V : a.interleaved ? p * 2 * V : p * V;
    e1[k] = turns[k] && !a.interleaved ? half + p * V : e0[k] + V;
    second[k] = has[k] && e1[k] < a.dim;
  }
  pdl_wait();
  float g[IT][2 * V], acc[IT][2 * V];
  if (NORM) {
    const bool aligned_gamma = ((uintptr_t)d.gamma.p & 15) == 0;
#pragma unroll
    for (int k = 0; k < IT; ++k)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const bool any = j ? second[k] : has[k];
        const uint32_t e = j ? e1[k] : e0[k];
#pragma unroll
        for (int i = 0; i < V; ++i) { g[k][j * V + i] = 0.0f; if (BWD) acc[k][j * V + i] = 0.0f; }
        if (!any) continue;
        if (V > 1 && aligned_gamma) { if constexpr (V > 1) d.gamma.load<V>(e, g[k] + j * V); }
        else {
#pragma unroll
          for (int i = 0; i < V; ++i) g[k][j * V + i] = d.gamma.at(e + i);
        }
      }
  }
  struct Head { Few<T, V> in[IT][2], x[BWD && NORM ? IT : 1][2]; } now, next;
  // (what a lane does not have is never loaded, and counts as zeros)
#pragma unroll
  for (int k = 0; k < IT; ++k)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      now.in[k][j].clear(); next.in[k][j].clear();
      if (BWD && NORM) { now.x[k][j].clear(); next.x[k][j].clear(); }
    }
  const uint32_t more = groups / d.heads, rest = groups - more * d.heads;
  for (uint64_t first = (uint64_t)block * d.tokens; first < a.total; first += (uint64_t)d.blocks * d.tokens) {
    const uint32_t count = (uint32_t)min((uint64_t)d.tokens, a.total - first);       // tokens of this round
    uint32_t t = group / d.heads, h = group - t * d.heads;
    auto place = [&](const HeadArray &x, uint32_t t, uint32_t h) {
      const uint64_t token = first + t, b = a.batch == 1 ? 0 : token / a.seq;
      return static_cast<T *>(x.p) + b * x.batch + (token - b * a.seq) * x.seq + h * x.head;
    };
    auto load = [&](Head &w, uint32_t t, uint32_t h) {
      const T *in = place(d.in, t, h);
#pragma unroll
      for (int k = 0; k < IT; ++k) {
        if (has[k]) w.in[k][0].load(in + e0[k]);
        if (second[k]) w.in[k][1].load(in + e1[k]);
      }
      if (BWD && NORM) {
        const T *x = place(d.x, t, h);
#pragma unroll
        for (int k = 0; k < IT; ++k) {
          if (has[k]) w.x[k][0].load(x + e0[k]);
          if (second[k]) w.x[k][1].load(x + e1[k]);
        }
      }
    };
    if (t < count) load(now, t, h);
    __syncthreads();                 // (the table of the round before has been read)
    for (uint32_t i = threadIdx.x; i < count * half; i += kThreads) {
      const uint32_t token = i / half, j = i - token * half, item = j / V, k = j % V;
      table[token * half + (V == 1 ? item : (k / 2 * a.turned + item) * 2 + k % 2)] = turn_of(position_of(a, first + token), a.freq[j], a.amplitude);
    }
    __syncthreads();
    // all groups of a warp go round as often as its first: the sums need every lane
    for (uint32_t t0 = (group & ~(32 / a.lanes - 1)) / d.heads, h0 = (group & ~(32 / a.lanes - 1)) - t0 * d.heads; t0 < count;) {
      const bool live = t < count;
      uint32_t nt = t + more, nh = h + rest;
      if (nh >= d.heads) { nh -= d.heads; ++nt; }
      t0 += more; h0 += rest;
      if (h0 >= d.heads) { h0 -= d.heads; ++t0; }
      if (nt < count) load(next, nt, nh);
      float f[IT][2 * V], x[BWD && NORM ? IT : 1][2 * V], sq = 0.0f, dot = 0.0f, r = 1.0f;
#pragma unroll
      for (int k = 0; k < IT; ++k) {
        now.in[k][0].floats(f[k]);
        now.in[k][1].floats(f[k] + V);
      }
      const float2 *cs = table + t * half;
      auto turn = [&](int k) {
        if (!live || !turns[k]) return;
        const uint32_t p = lane + k * a.lanes;
        float2 w[V];
        if constexpr (V == 1) w[0] = cs[p];
        else {
#pragma unroll
          for (int i = 0; i < V; i += 2) *reinterpret_cast<float4 *>(w + i) = *reinterpret_cast<const float4 *>(cs + (i / 2 * a.turned + p) * 2);
        }
        if (a.interleaved) {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float u = f[k][2 * i], v = f[k][2 * i + 1], s = a.way * w[i].y;
            f[k][2 * i] = u * w[i].x - v * s; f[k][2 * i + 1] = u * s + v * w[i].x;
          }
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float u = f[k][i], v = f[k][V + i], s = a.way * w[i].y;
            f[k][i] = u * w[i].x - v * s; f[k][V + i] = u * s + v * w[i].x;
          }
        }
      };
      if (!BWD) {
        if (NORM) {
#pragma unroll
          for (int k = 0; k < IT; ++k)
#pragma unroll
            for (int i = 0; i < 2 * V; ++i) sq = fmaf(f[k][i], f[k][i], sq);
          for (uint32_t o = a.lanes / 2; o > 0; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
          r = rsqrtf(sq * a.inv_dim + a.epsilon);
#pragma unroll
          for (int k = 0; k < IT; ++k)
#pragma unroll
            for (int i = 0; i < 2 * V; ++i) f[k][i] *= r * g[k][i];
        }
#pragma unroll
        for (int k = 0; k < IT; ++k) turn(k);
      } else {
#pragma unroll
        for (int k = 0; k < IT; ++k) turn(k);
        if (NORM) {
#pragma unroll
          for (int k = 0; k < IT; ++k) {
            now.x[k][0].floats(x[k]);
            now.x[k][1].floats(x[k] + V);
#pragma unroll
            for (int i = 0; i < 2 * V; ++i) { sq = fmaf(x[k][i], x[k][i], sq); dot = fmaf(f[k][i] * g[k][i], x[k][i], dot); }
          }
          for (uint32_t o = a.lanes / 2; o > 0; o >>= 1) {
            sq += __shfl_xor_sync(0xffffffffu, sq, o);
            dot += __shfl_xor_sync(0xffffffffu, dot, o);
          }
          r = rsqrtf(sq * a.inv_dim + a.epsilon);
          const float c = dot * r * r * a.inv_dim;
#pragma unroll
          for (int k = 0; k < IT; ++k)
#pragma unroll
            for (int i = 0; i < 2 * V; ++i) {
              if (live) acc[k][i] = fmaf(f[k][i], x[k][i] * r, acc[k][i]);
              f[k][i] = f[k][i] * (g[k][i] * r) - x[k][i] * (c * r);
            }
        }
      }
      if (live) {
        T *out = place(d.out, t, h);
#pragma unroll
        for (int k = 0; k < IT; ++k) {
          Few<T, V> w;
          if (has[k]) { w.of(f[k]); w.store(out + e0[k]); }
          if (second[k]) { w.of(f[k] + V); w.store(out + e1[k]); }
        }
      }
      now = next; t = nt; h = nh;
    }
  }
  if (!BWD || !NORM || !d.want) return;
  // the groups' sums in turn, in the order of the groups
  float *sums = reinterpret_cast<float *>(shared);
  for (uint32_t i = 0; i < groups; ++i) {
    __syncthreads();
    if (group != i) continue;
#pragma unroll
    for (int k = 0; k < IT; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (has[k]) sums[e0[k] + j] = acc[k][j] + (i ? sums[e0[k] + j] : 0.0f);
        if (second[k]) sums[e1[k] + j] = acc[k][V + j] + (i ? sums[e1[k] + j] : 0.0f);
      }
  }
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < a.dim; i += kThreads) a.partial[(uint64_t)blockIdx.x * a.dim + i] = sums[i];
}

// The blocks' sums: a lane has an element of one of the two gradients, a warp every 32nd block
__global__ void __launch_bounds__(1024) rotary_join_kernel(uint32_t dim, uint32_t q_blocks, uint32_t blocks, const float *partial, void *dq, void *dk, int type)
{
  __shared__ float sums[32][33];
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, wide = (dim + 31) / 32, k = blockIdx.x >= wide, i = (blockIdx.x - k * wide) * 32 + lane;
  void *out = k ? dk : dq;
  pdl_wait();
  if (!out) return;
  float sum = 0.0f;
  if (i < dim) {
#pragma unroll 4
    for (uint32_t b = (k ? q_blocks : 0) + warp; b < (k ? blocks : q_blocks); b += 32) sum += partial[(uint64_t)b * dim + i];
  }
  sums[warp][lane] = sum;
  __syncthreads();
  if (warp || i >= dim) return;
#pragma unroll
  for (uint32_t w = 1; w < 32; ++w) sum += sums[w][lane];
  put_weight(out, type, i, sum);
}

// An array of heads: pointer and alignment; an output's heads do not overlap
inline int check_heads(const AnodeHeads *h, size_t e, uint32_t batch, uint32_t seq, uint32_t dim, bool output)
{
  if (!h->data) return ANODE_E_NULL;
  if (!aligned_to(h->data, e)) return ANODE_E_ALIGN;
  if (!output) return ANODE_OK;
  uint64_t size[3] = {batch, seq, h->heads}, stride[3] = {h->batch_stride, h->seq_stride, h->head_stride}, extent = dim;
  bool done[3] = {size[0] < 2, size[1] < 2, size[2] < 2};
  for (int k = 0; k < 3; ++k) {
    int at = -1;
    for (int i = 0; i < 3; ++i) if (!done[i] && (at < 0 || stride[i] < stride[at])) at = i;
    if (at < 0) break;
    if (stride[at] < extent) return ANODE_E_STRIDE;
    extent += stride[at] * (size[at] - 1);
    done[at] = true;
  }
  return ANODE_OK;
}
inline bool same_place(const AnodeHeads *o, const AnodeHeads *i, uint32_t batch, uint32_t seq)
{
  if (!i || o->data != i->data) return true;
  return (batch < 2 || o->batch_stride == i->batch_stride) && (seq < 2 || o->seq_stride == i->seq_stride) && (o->heads < 2 || o->head_stride == i->head_stride);
}

#define TRY(call) do { const int rc_ = (call); if (rc_) return rc_; } while (0)

struct RotaryCall {
  int type, gamma_type, position_bytes;
  bool bwd;
  const AnodeHeads *in[2], *x[2], *out[2];
  void *dgamma[2];
  void *workspace;
  size_t workspace_bytes;
};

int rotary(RotaryArgs a, const RotaryCall &c, cudaStream_t stream)
{
  if (!known_type(c.type) || (c.position_bytes != 4 && c.position_bytes != 8)) return ANODE_E_TYPE;
  const bool wants = c.dgamma[0] || c.dgamma[1];
  if ((a.side[0].gamma.p || a.side[1].gamma.p || wants) && !known_type(c.gamma_type)) return ANODE_E_TYPE;
  if (a.dim == 0 || a.dim > kMostDim || a.rot < 2 || a.rot > a.dim || a.rot % 2) return ANODE_E_DIMS;
  if (!c.in[0] || !c.out[0] || !c.in[1] != !c.out[1]) return ANODE_E_NULL;
  const bool two = c.in[1] != nullptr;
  if (wants && (!a.norm || (c.dgamma[1] && !two))) return ANODE_E_NULL;
  const size_t e = type_bytes(c.type), ge = type_bytes(c.gamma_type);
  for (int k = 0; k < 1 + two; ++k) {
    if (c.in[k]->heads == 0 || c.in[k]->heads > 65535 || c.in[k]->heads != c.out[k]->heads) return ANODE_E_DIMS;
    if (c.bwd && a.norm) {
      if (!c.x[k]) return ANODE_E_NULL;
      if (c.x[k]->heads != c.in[k]->heads) return ANODE_E_DIMS;
    }
  }
  for (int k = 0; k < 2; ++k)
    if (!aligned_to(a.side[k].gamma.p, ge) || !aligned_to(c.dgamma[k], ge)) return ANODE_E_ALIGN;
  if (a.batch == 0 || a.seq == 0) {
    for (int k = 0; k < 2; ++k)
      if (c.dgamma[k] && cudaMemsetAsync(c.dgamma[k], 0, ge * a.dim, stream) != cudaSuccess) return ANODE_E_LAUNCH;
    return ANODE_OK;
  }
  if (!a.freq || !a.positions) return ANODE_E_NULL;
  if (!aligned_to(a.freq, 8) || !aligned_to(a.positions, (size_t)c.position_bytes)) return ANODE_E_ALIGN;
  for (int k = 0; k < 1 + two; ++k) {
    TRY(check_heads(c.in[k], e, a.batch, a.seq, a.dim, false));
    TRY(check_heads(c.out[k], e, a.batch, a.seq, a.dim, true));
    if (!same_place(c.out[k], c.in[k], a.batch, a.seq)) return ANODE_E_STRIDE;
    auto put = [](HeadArray &to, const AnodeHeads *h) { to = HeadArray{h->data, h->batch_stride, h->seq_stride, h->head_stride}; };
    RotarySide &d = a.side[k];
    put(d.in, c.in[k]);
    put(d.out, c.out[k]);
    d.heads = c.in[k]->heads;
    d.want = c.dgamma[k] != nullptr;
    if (c.bwd && a.norm) {
      TRY(check_heads(c.x[k], e, a.batch, a.seq, a.dim, false));
      if (!same_place(c.out[k], c.x[k], a.batch, a.seq)) return ANODE_E_STRIDE;
      put(d.x, c.x[k]);
    }
  }
  a.total = (uint64_t)a.batch * a.seq;
  a.partial = static_cast<float *>(c.workspace);
  if (wants && (!c.workspace || !aligned_to(c.workspace, 16) ||
                c.workspace_bytes < anode_gpu_rotary_positions_bwd_workspace_bytes(a.batch, a.seq, a.side[0].heads, a.side[1].heads, a.dim)))
    return ANODE_E_WORKSPACE;
  // elements that every array moves at once: all addresses and the pairs' places divide by them
  uint32_t v = (uint32_t)(16 / e);
  auto divides = [&](uint32_t v) {
    if (a.interleaved ? a.rot % (2 * v) : a.rot / 2 % v) return false;
    if ((a.dim - a.rot) % v) return false;
    for (int k = 0; k < 1 + two; ++k)
      for (const AnodeHeads *h : {c.in[k], c.out[k], c.bwd && a.norm ? c.x[k] : nullptr})
        if (h && (!aligned_to(h->data, v * e) || (a.batch > 1 && h->batch_stride % v) || (a.seq > 1 && h->seq_stride % v) || (h->heads > 1 && h->head_stride % v)))
          return false;
    return true;
  };
  while (v > 1 && !divides(v)) v = v == 8 ? 4 : 1;
  a.way = c.bwd ? -1.0f : 1.0f;
  a.turned = a.rot / 2 / v;
  a.items = a.turned + (a.dim - a.rot + 2 * v - 1) / (2 * v);
  a.lanes = 1;
  while (a.lanes < 32 && a.lanes < a.items) a.lanes *= 2;
  const uint32_t each = (a.items + a.lanes - 1) / a.lanes, groups = kThreads / a.lanes;
  uint32_t blocks = 0, most = 0;
  for (int k = 0; k < 1 + two; ++k) {
    RotarySide &d = a.side[k];
    // about four heads to a group, fewer where that leaves SMs without a block
    uint64_t tokens = (4 * groups + d.heads - 1) / d.heads, fit = 32768 / (4 * a.rot);
    if (tokens > fit) tokens = fit;
    if (tokens > kMostTokens) tokens = kMostTokens;
    const uint64_t spread = (a.total + sm_count() - 1) / sm_count();
    if (tokens > spread) tokens = spread;
    if (tokens < 1) tokens = 1;
    d.tokens = (uint32_t)tokens;
    const uint64_t need = (a.total + d.tokens - 1) / d.tokens, limit = wants ? kMostParts / 2 : 1u << 29;
    d.blocks = (uint32_t)(need < limit ? need : limit);
    blocks += d.blocks;
    if (d.tokens > most) most = d.tokens;
  }
  size_t shared = (size_t)most * a.rot / 2 * 8;
  if (wants && shared < a.dim * 4) shared = a.dim * 4;
  TRY(by_type(c.type, [&](auto t) {
    using T = decltype(t);
    auto go = [&](auto kernel) { return launch(kernel, dim3(blocks), kThreads, shared, stream, a); };
    auto with = [&](auto norm, auto bwd) {
      constexpr bool N = decltype(norm)::value, B = decltype(bwd)::value;
      if constexpr (sizeof(T) == 2)
        if (v == 8) return each == 1 ? go(rotary_heads_kernel<T, 8, 1, N, B>) : go(rotary_heads_kernel<T, 8, 2, N, B>);
      if (v == 4) return each == 1 ? go(rotary_heads_kernel<T, 4, 1, N, B>) : each == 2 ? go(rotary_heads_kernel<T, 4, 2, N, B>) : go(rotary_heads_kernel<T, 4, 4, N, B>);
      return each == 1 ? go(rotary_heads_kernel<T, 1, 1, N, B>) : each == 2 ? go(rotary_heads_kernel<T, 1, 2, N, B>)
           : each <= 4 ? go(rotary_heads_kernel<T, 1, 4, N, B>) : go(rotary_heads_kernel<T, 1, 16, N, B>);
    };
    const std::true_type yes;
    const std::false_type no;
    return !a.norm ? with(no, no) : c.bwd ? with(yes, yes) : with(yes, no);       // (without a norm the two differ by the turn's sign)
  }));
  if (!wants) return ANODE_OK;
  return launch(rotary_join_kernel, dim3((1 + two) * ((a.dim + 31) / 32)), 1024, 0, stream, a.dim, a.side[0].blocks, blocks, a.partial, c.dgamma[0], c.dgamma[1],
                c.gamma_type);
}

}  // namespace rows
}  // namespace anode_b200

using namespace anode_b200::rows;

extern "C" int anode_gpu_rotary_positions_fwd(
    int type, uint32_t batch, uint32_t seq, uint32_t dim, uint32_t rot, int interleaved, float amplitude,
    const double *freq, const void *positions, int position_bytes, uint64_t pos_batch_stride, uint64_t pos_seq_stride,
    int norm, float epsilon, const void *gamma_q, const void *gamma_k, int gamma_type,
    const struct AnodeHeads *q, const struct AnodeHeads *k, const struct AnodeHeads *q_out, const struct AnodeHeads *k_out,
    const struct KernelConfig *cfg, struct CUstream_st *stream)
{
  (void)cfg;
  RotaryArgs a = {batch, seq, dim, rot, interleaved != 0, amplitude, epsilon, 1.0f / (float)dim, freq, positions, (uint32_t)position_bytes,
                  pos_batch_stride, pos_seq_stride};
  a.norm = norm != 0;
  a.side[0].gamma = Weights{gamma_q, gamma_type};
  a.side[1].gamma = Weights{gamma_k, gamma_type};
  return rotary(a, RotaryCall{type, gamma_type, position_bytes, false, {q, k}, {}, {q_out, k_out}, {}, nullptr, 0}, stream);
}

extern "C" size_t anode_gpu_rotary_positions_bwd_workspace_bytes(uint32_t batch, uint32_t seq, uint32_t q_heads, uint32_t k_heads, uint32_t dim)
{
  (void)batch; (void)seq; (void)q_heads; (void)k_heads;
  return (size_t)kMostParts * dim * 4;
}

extern "C" int anode_gpu_rotary_positions_bwd(
    int type, uint32_t batch, uint32_t seq, uint32_t dim, uint32_t rot, int interleaved, float amplitude,
    const double *freq, const void *positions, int position_bytes, uint64_t pos_batch_stride, uint64_t pos_seq_stride,
    int norm, float epsilon, const void *gamma_q, const void *gamma_k, int gamma_type,
    const struct AnodeHeads *dq_out, const struct AnodeHeads *dk_out, const struct AnodeHeads *q, const struct AnodeHeads *k,
    const struct AnodeHeads *dq, const struct AnodeHeads *dk, void *dgamma_q, void *dgamma_k,
    void *workspace, size_t workspace_bytes,
    const struct KernelConfig *cfg, struct CUstream_st *stream)
{
  (void)cfg;
  RotaryArgs a = {batch, seq, dim, rot, interleaved != 0, amplitude, epsilon, 1.0f / (float)dim, freq, positions, (uint32_t)position_bytes,
                  pos_batch_stride, pos_seq_stride};
  a.norm = norm != 0;
  a.side[0].gamma = Weights{gamma_q, gamma_type};
  a.side[1].gamma = Weights{gamma_k, gamma_type};
  return rotary(a, RotaryCall{type, gamma_type, position_bytes, true, {dq_out, dk_out}, {q, k}, {dq, dk}, {dgamma_q, dgamma_k}, workspace, workspace_bytes},
                stream);
}
