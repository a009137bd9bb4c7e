// Rotary positions of queries and keys, with the RMS norm of each head before them: forward and adjoint.
//
//   n = x*r*gamma, r = (mean(x^2) + epsilon)^-1/2 over the head;   angle = position*freq[i]
//   (n[u], n[v]) -> A*(n[u] cos - n[v] sin, n[u] sin + n[v] cos);   backward: the same with -sin, then the norm's adjoint
//
// A head is read once and written once.  It belongs to a group of lanes of a warp; a lane has ITEMS of 2V elements each: V pairs,
// or 2V elements that pass.  In the half layout an item is two vectors rot/2 apart, so that both elements of a pair are in one lane and the
// turn needs no exchange; only the norm's sums go across the group.  Lanes keep their items from head to head, and with them the
// weights and the sums of the weights' gradients.
// A warp takes a token of the queries or of the keys (or as many tokens as fill it, or part of a token's heads where there are few tokens),
// makes its cosines and sines once, in shared memory of its own, and goes through the heads with the next ones' data on their way by
// asynchronous copies, each lane into a ring of its own: no warp waits for another, and no lane for what another lane copies.
#include "bn_host.h"
#include "rows.cuh"

namespace anode_b200 {
namespace rows {

constexpr uint32_t kThreads = 256, kMostDim = 1024;
constexpr uint32_t kMostParts = 148 * 4;      // blocks that have sums of the weights' gradients
constexpr uint32_t kWarps = kThreads / 32;

struct HeadArray {
  void *p;
  uint64_t batch, seq, head;
};
// One of the two arrays' geometry
struct RotarySide {
  HeadArray in, x, out;                // backward: in = dout, x = the norm's input, out = dx
  Weights gamma;
  uint32_t heads;
  uint32_t tokens, parts, span;        // a unit of a warp: `tokens` tokens, or one of the `parts` spans of a token's heads
  uint32_t units;
  uint32_t blocks, want;               // blocks of the grid; whether the weights' gradient is asked for
};
struct RotaryArgs {
  uint32_t batch, seq, dim, rot, interleaved;
  float amplitude, epsilon, inv_dim;
  const double *freq;
  const void *positions;
  uint32_t position_bytes;
  uint64_t pos_batch, pos_seq;
  uint32_t total;                      // tokens
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
  union { typename RawOf<V * sizeof(T)>::type raw; T e[V]; uint32_t w[(V * sizeof(T) + 3) / 4]; };
  __device__ __forceinline__ Few() {}
  __device__ __forceinline__ void load(const T *p) { raw = *reinterpret_cast<const decltype(raw) *>(p); }
  __device__ __forceinline__ void clear() { raw = decltype(raw){}; }
  __device__ __forceinline__ void store(T *p) const { *reinterpret_cast<decltype(raw) *>(p) = raw; }
  __device__ __forceinline__ void floats(float *f) const
  {
    if constexpr (std::is_same<T, __nv_bfloat16>::value && V > 1) {
#pragma unroll
      for (int i = 0; i < V / 2; ++i) { f[2 * i] = __uint_as_float(w[i] << 16); f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] = to_float(e[i]);
    }
  }
  __device__ __forceinline__ void of(const float *f)
  {
    if constexpr (sizeof(T) == 2 && V > 1) {
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        if constexpr (std::is_same<T, __half>::value) { const __half2 v = __floats2half2_rn(f[2 * i], f[2 * i + 1]); w[i] = *reinterpret_cast<const uint32_t *>(&v); }
        else { const __nv_bfloat162 v = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]); w[i] = *reinterpret_cast<const uint32_t *>(&v); }
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) e[i] = from_float<T>(f[i]);
    }
  }
};

template <int BYTES> __device__ __forceinline__ void copy_async(void *to, const void *from)
{
  const uint32_t at = (uint32_t)__cvta_generic_to_shared(to);
  if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at), "l"(from) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(at), "l"(from), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }

__device__ __forceinline__ double position_of(const RotaryArgs &a, uint32_t token)
{
  const uint32_t b = a.batch == 1 ? 0 : token / a.seq;
  const uint64_t i = b * a.pos_batch + (token - b * a.seq) * a.pos_seq;
  return a.position_bytes == 8 ? (double)static_cast<const long long *>(a.positions)[i] : (double)static_cast<const int *>(a.positions)[i];
}
// cos and sin of position*freq, by whole turns in f64: what is left of them is exact, and small
__device__ __forceinline__ float2 turn_of(double position, double freq, float amplitude, float way)
{
  const double turns = position * (freq * 0.15915494309189533577);      // 1/(2 pi)
  float s, c;
  sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
  return make_float2(c * amplitude, s * amplitude * way);
}

// Registers: two or three blocks of a multiprocessor
constexpr int resident(int floats, bool both) { return floats > 16 ? 1 : both ? 2 : 3; }
// Heads of a lane's ring, and its bytes: pieces of less than four bytes cannot be copied asynchronously and go through registers
__host__ __device__ constexpr int ring_depth(int v, int it) { return v == 1 ? 1 : it == 1 ? 4 : 2; }
__host__ __device__ constexpr size_t ring_bytes(int v, int it, bool both, size_t e) { return v == 1 ? 0 : (size_t)ring_depth(v, it) * kThreads * it * 2 * v * e * (both ? 2 : 1); }

template <typename T, int V, int IT, bool NORM, bool BWD>
__global__ void __launch_bounds__(kThreads, resident(2 * V * IT, NORM && BWD)) rotary_heads_kernel(const RotaryArgs a)
{
  constexpr bool BOTH = NORM && BWD;        // two arrays are read
  constexpr bool KEEP = V * IT <= 8;        // a lane's cosines and sines stay in its registers from head to head
  constexpr int DEPTH = ring_depth(V, IT), PIECES = IT * 2 * (BOTH ? 2 : 1);
  typedef typename RawOf<V * sizeof(T)>::type Raw;
  // the rings, [depth][piece][thread]; of each warp, [tokens][rot/2] cosines and sines, pair j = item*V + i of a token at
  // (i/2*turned + item)*2 + i%2, so that lanes read 16 bytes side by side; in their place the warps' sums of the weights' gradients, when the block is done
  extern __shared__ float4 shared[];
  const uint32_t which = blockIdx.x >= a.side[0].blocks, block = which ? blockIdx.x - a.side[0].blocks : blockIdx.x;
  const RotarySide &d = a.side[which];
  const uint32_t wlane = threadIdx.x & 31, warp = threadIdx.x >> 5, lane = wlane & (a.lanes - 1), group = wlane / a.lanes, groups = 32 / a.lanes;
  const uint32_t half = a.rot / 2, heads = d.heads;
  Raw *ring = reinterpret_cast<Raw *>(shared) + threadIdx.x;
  float2 *table = reinterpret_cast<float2 *>(reinterpret_cast<char *>(shared) + ring_bytes(V, IT, BOTH, sizeof(T))) + (size_t)warp * d.tokens * half;
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
  float g[NORM ? IT : 1][2 * V], acc[NORM && BWD ? IT : 1][2 * V];
  if constexpr (NORM) {
    const bool aligned_gamma = ((uintptr_t)d.gamma.p & 15) == 0;
#pragma unroll
    for (int k = 0; k < IT; ++k)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const bool any = j ? second[k] : has[k];
        const uint32_t e = j ? e1[k] : e0[k];
#pragma unroll
        for (int i = 0; i < V; ++i) { g[k][j * V + i] = 0.0f; if constexpr (BWD) acc[k][j * V + i] = 0.0f; }
        if (!any) continue;
        if (V > 1 && aligned_gamma) { if constexpr (V > 1) d.gamma.load<V>(e, g[k] + j * V); }
        else {
#pragma unroll
          for (int i = 0; i < V; ++i) g[k][j * V + i] = d.gamma.at(e + i);
        }
      }
  }
  struct Head { Few<T, V> in[IT][2], x[BOTH ? IT : 1][2]; } now, next;
  // (what a lane does not have is never loaded, and counts as zeros)
#pragma unroll
  for (int k = 0; k < IT; ++k)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if constexpr (V == 1) {
        now.in[k][j].clear(); next.in[k][j].clear();
        if constexpr (BOTH) { now.x[k][j].clear(); next.x[k][j].clear(); }
      } else if (!(j ? second[k] : has[k])) {
        for (int i = 0; i < DEPTH; ++i) {
          ring[(i * PIECES + 2 * k + j) * kThreads] = Raw{};
          if constexpr (BOTH) ring[(i * PIECES + 2 * IT + 2 * k + j) * kThreads] = Raw{};
        }
      }
    }
  // Where this group is: the unit, its head (none: from `end` on), the passes that the unit has left, and addresses
  struct Place { uint32_t unit, head, end, left; const T *p, *x; };
  const uint32_t step = d.blocks * kWarps, mine = d.tokens > 1 ? group / heads : 0;      // mine: of the unit's tokens
  const uint64_t hop = d.in.head * groups, hop_x = BOTH ? d.x.head * groups : 0, hop_out = d.out.head * groups;
  auto enter = [&](Place &w, const HeadArray &p, const HeadArray *x) {       // the first head of its unit
    if (w.unit >= d.units) { w.head = w.end = 0; w.left = 1; return; }
    const uint32_t first = d.parts > 1 ? w.unit / d.parts : w.unit * d.tokens, low = d.parts > 1 ? (w.unit - first * d.parts) * d.span : 0;
    const uint32_t token = first + mine;
    w.end = min(heads, low + d.span);
    w.left = d.tokens > 1 ? 1 : (w.end - low + groups - 1) / groups;
    w.head = low + group - mine * heads;
    if (mine >= d.tokens || token >= a.total) w.head = w.end;
    const uint32_t b = a.batch == 1 ? 0 : token / a.seq, s = token - b * a.seq;
    w.p = static_cast<const T *>(p.p) + b * p.batch + s * p.seq + w.head * p.head;
    if (x) w.x = static_cast<const T *>(x->p) + b * x->batch + s * x->seq + w.head * x->head;
  };
  uint32_t turn_in = 0;                  // the ring's place that is filled next
  auto load = [&](const Place &w) {
    if (w.head < w.end) {
#pragma unroll
      for (int k = 0; k < IT; ++k)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if (!(j ? second[k] : has[k])) continue;
          const uint32_t e = j ? e1[k] : e0[k];
          if constexpr (V == 1) {
            next.in[k][j].load(w.p + e);
            if constexpr (BOTH) next.x[k][j].load(w.x + e);
          } else {
            copy_async<V * sizeof(T)>(ring + (turn_in * PIECES + 2 * k + j) * kThreads, w.p + e);
            if constexpr (BOTH) copy_async<V * sizeof(T)>(ring + (turn_in * PIECES + 2 * IT + 2 * k + j) * kThreads, w.x + e);
          }
        }
    }
    if constexpr (V > 1) {
      copies_commit();
      turn_in = turn_in + 1 == DEPTH ? 0 : turn_in + 1;
    }
  };
  auto advance = [&](Place &w, uint64_t hop, uint64_t hop_x, const HeadArray &p, const HeadArray *x) {
    if (--w.left) { w.head += groups; w.p += hop; if (x) w.x += hop_x; }
    else { w.unit += step; enter(w, p, x); }
  };
  float2 w[KEEP ? IT : 1][V];
  auto fetch = [&](int k, uint32_t t, float2 *w) {
    const uint32_t p = lane + k * a.lanes;
    const float2 *cs = table + t * half;
    if constexpr (V == 1) w[0] = cs[p];
    else {
#pragma unroll
      for (int i = 0; i < V; i += 2) *reinterpret_cast<float4 *>(w + i) = *reinterpret_cast<const float4 *>(cs + (i / 2 * a.turned + p) * 2);
    }
  };
  Place at, ahead;
  at.unit = ahead.unit = block * kWarps + warp;
  enter(at, d.out, nullptr);
  enter(ahead, d.in, BOTH ? &d.x : nullptr);
  uint32_t turn_out = 0;
#pragma unroll
  for (int i = 0; i < (V == 1 ? 1 : DEPTH - 1); ++i) {
    load(ahead);
    advance(ahead, hop, hop_x, d.in, BOTH ? &d.x : nullptr);
  }
  for (; at.unit < d.units;) {
    // the unit's cosines and sines
    const uint32_t first = d.parts > 1 ? at.unit / d.parts : at.unit * d.tokens, count = min(d.tokens, a.total - first) * half;
    __syncwarp();
    for (uint32_t i = wlane; i < count; i += 32) {
      const uint32_t t = d.tokens > 1 ? i / half : 0, j = i - t * half, item = j / V, k = j % V;
      table[t * half + (V == 1 ? item : (k / 2 * a.turned + item) * 2 + k % 2)] = turn_of(position_of(a, first + t), a.freq[j], a.amplitude, a.way);
    }
    __syncwarp();
    if (KEEP && at.head < at.end) {
#pragma unroll
      for (int k = 0; k < IT; ++k) if (turns[k]) fetch(k, mine, w[KEEP ? k : 0]);
    }
    // heads of this unit, as many at a time as the warp has groups
    for (const uint32_t unit = at.unit; at.unit == unit;) {
      const bool live = at.head < at.end;
      if constexpr (V == 1) now = next;
      load(ahead);
      advance(ahead, hop, hop_x, d.in, BOTH ? &d.x : nullptr);
      if constexpr (V > 1) {
        copies_wait<DEPTH - 1>();
#pragma unroll
        for (int k = 0; k < IT; ++k)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            now.in[k][j].raw = ring[(turn_out * PIECES + 2 * k + j) * kThreads];
            if constexpr (BOTH) now.x[k][j].raw = ring[(turn_out * PIECES + 2 * IT + 2 * k + j) * kThreads];
          }
        turn_out = turn_out + 1 == DEPTH ? 0 : turn_out + 1;
      }
      float f[IT][2 * V], sq = 0.0f;
#pragma unroll
      for (int k = 0; k < IT; ++k) { now.in[k][0].floats(f[k]); now.in[k][1].floats(f[k] + V); }
      auto turn = [&](int k) {
        if (!live || !turns[k]) return;
        float2 own[V];
        if constexpr (!KEEP) fetch(k, mine, own);
        const float2 *cs = KEEP ? w[KEEP ? k : 0] : own;
        if (a.interleaved) {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float u = f[k][2 * i], v = f[k][2 * i + 1];
            f[k][2 * i] = u * cs[i].x - v * cs[i].y; f[k][2 * i + 1] = u * cs[i].y + v * cs[i].x;
          }
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float u = f[k][i], v = f[k][V + i];
            f[k][i] = u * cs[i].x - v * cs[i].y; f[k][V + i] = u * cs[i].y + v * cs[i].x;
          }
        }
      };
      if constexpr (!BWD) {
        if constexpr (NORM) {
#pragma unroll
          for (int k = 0; k < IT; ++k)
#pragma unroll
            for (int i = 0; i < 2 * V; ++i) sq = fmaf(f[k][i], f[k][i], sq);
          for (uint32_t o = a.lanes / 2; o > 0; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
          const float r = rsqrtf(sq * a.inv_dim + a.epsilon);
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
        float x[IT][2 * V], dot = 0.0f;
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
        const float r = rsqrtf(sq * a.inv_dim + a.epsilon), c = dot * r * r * r * a.inv_dim;
        if (live) {
#pragma unroll
          for (int k = 0; k < IT; ++k)
#pragma unroll
            for (int i = 0; i < 2 * V; ++i) {
              acc[k][i] = fmaf(f[k][i], x[k][i] * r, acc[k][i]);
              f[k][i] = f[k][i] * (g[k][i] * r) - x[k][i] * c;
            }
        }
      }
      if (live) {
        T *out = const_cast<T *>(at.p);
#pragma unroll
        for (int k = 0; k < IT; ++k) {
          Few<T, V> o;
          if (has[k]) { o.of(f[k]); o.store(out + e0[k]); }
          if (second[k]) { o.of(f[k] + V); o.store(out + e1[k]); }
        }
      }
      advance(at, hop_out, 0, d.out, nullptr);
    }
  }
  if constexpr (BWD && NORM) {
    if (!d.want) return;
    // the groups' sums join within the warp, the warps' in shared memory
    float *sums = reinterpret_cast<float *>(shared);
    if constexpr (V > 1) copies_wait<0>();
    __syncthreads();
#pragma unroll
    for (int k = 0; k < IT; ++k)
#pragma unroll
      for (int j = 0; j < 2 * V; ++j) {
        for (uint32_t o = a.lanes; o < 32; o *= 2) acc[k][j] += __shfl_xor_sync(0xffffffffu, acc[k][j], o);
        const bool any = j < V ? has[k] : second[k];
        if (group == 0 && any) sums[(size_t)warp * a.dim + (j < V ? e0[k] + j : e1[k] + j - V)] = acc[k][j];
      }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < a.dim; i += kThreads) {
      float sum = 0.0f;
#pragma unroll
      for (uint32_t n = 0; n < kWarps; ++n) sum += sums[(size_t)n * a.dim + i];
      a.partial[(uint64_t)blockIdx.x * a.dim + i] = sum;
    }
  }
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

template <typename T, int V, int IT, bool NORM, bool BWD>
int launch_rotary(const RotaryArgs &a, uint32_t blocks, size_t tables, size_t sums, cudaStream_t stream)
{
  const auto kernel = rotary_heads_kernel<T, V, IT, NORM, BWD>;
  size_t shared = ring_bytes(V, IT, NORM && BWD, sizeof(T)) + tables;
  if (shared < sums) shared = sums;
  static SharedMemory allowed;
  if (!allowed.up_to((const void *)kernel, shared)) return ANODE_E_LAUNCH;
  return launch(kernel, dim3(blocks), kThreads, shared, stream, a);
}

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
  if ((uint64_t)a.batch * a.seq >> 31) return ANODE_E_DIMS;
  a.total = a.batch * a.seq;
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
  const uint32_t each = (a.items + a.lanes - 1) / a.lanes, groups = 32 / a.lanes;
  // blocks that the device holds; both arrays' warps work side by side, as many on either as its share of the heads asks for
  const uint32_t room = sm_count() * (c.bwd && a.norm ? 2 : 3);
  uint32_t blocks = 0, most = 1, units[2] = {0, 0}, passes[2];
  double cost[2] = {0.0, 0.0};
  for (int k = 0; k < 1 + two; ++k) {
    RotarySide &d = a.side[k];
    // a warp has tokens that fill it, or a token's heads
    d.tokens = d.heads < groups ? groups / d.heads : 1;
    while (d.tokens > 1 && d.tokens * a.rot / 2 > 512) --d.tokens;
    units[k] = (a.total - 1) / d.tokens + 1;
    passes[k] = (d.heads + groups - 1) / groups;
    if (d.tokens > most) most = d.tokens;
  }
  for (int k = 0; k < 1 + two; ++k) {
    RotarySide &d = a.side[k];
    // or, where that leaves warps of the device idle, a span of them
    d.parts = room * kWarps / ((uint64_t)units[0] + units[1]);
    if (d.parts > passes[k]) d.parts = passes[k];
    if (d.parts < 1 || d.tokens > 1) d.parts = 1;
    d.span = (passes[k] + d.parts - 1) / d.parts * groups;
    d.parts = (d.heads + d.span - 1) / d.span;
    d.units = units[k] * d.parts;
    cost[k] = (double)units[k] * (passes[k] + 1.5 * d.parts);        // (the cosines and sines cost a unit about one and a half passes)
  }
  for (int k = 0; k < 1 + two; ++k) {
    RotarySide &d = a.side[k];
    const uint32_t need = (d.units - 1) / kWarps + 1, share = (uint32_t)(room * cost[k] / (cost[0] + cost[1]));
    d.blocks = need < share ? need : share ? share : 1;
    blocks += d.blocks;
  }
  const size_t tables = (size_t)kWarps * most * a.rot / 2 * 8, sums = wants ? (size_t)kWarps * a.dim * 4 : 0;
  TRY(by_type(c.type, [&](auto t) {
    using T = decltype(t);
    auto with = [&](auto norm, auto bwd) {
      constexpr bool N = decltype(norm)::value, B = decltype(bwd)::value;
      if constexpr (sizeof(T) == 2)
        if (v == 8) return each == 1 ? launch_rotary<T, 8, 1, N, B>(a, blocks, tables, sums, stream) : launch_rotary<T, 8, 2, N, B>(a, blocks, tables, sums, stream);
      if (v == 4) return each == 1 ? launch_rotary<T, 4, 1, N, B>(a, blocks, tables, sums, stream)
                       : each == 2 ? launch_rotary<T, 4, 2, N, B>(a, blocks, tables, sums, stream) : launch_rotary<T, 4, 4, N, B>(a, blocks, tables, sums, stream);
      return each == 1 ? launch_rotary<T, 1, 1, N, B>(a, blocks, tables, sums, stream) : each == 2 ? launch_rotary<T, 1, 2, N, B>(a, blocks, tables, sums, stream)
           : each <= 4 ? launch_rotary<T, 1, 4, N, B>(a, blocks, tables, sums, stream) : launch_rotary<T, 1, 16, N, B>(a, blocks, tables, sums, stream);
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
