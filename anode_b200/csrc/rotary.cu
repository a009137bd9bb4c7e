// Rotary positions of queries and keys, with the RMS norm of each head before them: forward and adjoint.
//
//   n = x*r*gamma, r = (mean(x^2) + epsilon)^-1/2 over the head;   angle = position*freq[i]
//   (n[u], n[v]) -> A*(n[u] cos - n[v] sin, n[u] sin + n[v] cos);   backward: the same with -sin, then the norm's adjoint
//
// A head is read once and written once.  It belongs to a group of lanes of a warp, and a warp takes a token of the queries or of the keys (or
// as many tokens as fill it, or part of a token's heads where there are few tokens), makes its cosines and sines once, in shared memory of its
// own, and goes through the heads with the next ones' data on their way by asynchronous copies: no warp waits for another.
//
// rotary_heads_kernel: the pairs' places divide by 16 (or 8) bytes.  A lane has ITEMS of 2V elements each: V pairs, or 2V elements that pass.
// An item is two vectors rot/2 apart, so that both elements of a pair are in one lane in either layout and the turn needs no exchange;
// only the norm's sums go across the group.  What a lane computes with is what it copied itself.  Lanes keep their items from head to head,
// and with them the weights and the sums of the weights' gradients.
// rotary_pairs_kernel: pairs anywhere.  Heads are copied as they lie, a lane has single pairs of them and puts the results in their place.
//
// What bounds it: memory, and the instructions of a pass over a warp's heads (161 of a warp with a norm, 121 without, some 330 backward, for
// 32 lanes' 16 elements each) and of a token's cosines and sines (some 550, which is why a warp has all of a token's heads).  On one B200, of
// 6539 GB/s, bf16, 40 heads of 128: 16384 tokens forward 56.7 us with a norm (0.91) and 60 without (0.85); 8192 tokens backward 51.7 us with a
// norm (0.74) and 29 without (0.88); 62 of 128 elements turned (pairs anywhere) 116 us either way; 32 tokens 2.7 us.
#include "bn_host.h"
#include "rows.cuh"

namespace anode_b200 {
namespace rows {

constexpr uint32_t kThreads = 128, kMostDim = 1024;
constexpr uint32_t kWarps = kThreads / 32;
constexpr uint32_t kMostParts = 148 * 8;      // blocks that have sums of the weights' gradients

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
  uint32_t passes, last;               // heads of a group in a span, and in a token's last one
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
  uint32_t copy, slot;                 // of rotary_pairs_kernel: bytes of a copy, bytes of a head's place in shared memory
};

// V elements, moved at once
template <int BYTES> struct RawOf;
template <> struct RawOf<16> { typedef uint4 type; };
template <> struct RawOf<8> { typedef uint2 type; };
template <typename T, int V> struct Few {
  typedef typename RawOf<V * sizeof(T)>::type Raw;
  union { Raw raw; uint32_t w[V * sizeof(T) / 4]; };
  __device__ __forceinline__ Few() {}
  // elements 2m and 2m + 1
  __device__ __forceinline__ float2 two(int m) const
  {
    if constexpr (sizeof(T) == 4) return make_float2(__uint_as_float(w[2 * m]), __uint_as_float(w[2 * m + 1]));
    else if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2 *>(&w[m]));
    else return make_float2(__uint_as_float(w[m] << 16), __uint_as_float(w[m] & 0xffff0000u));
  }
  __device__ __forceinline__ void put(int m, float x, float y)
  {
    if constexpr (sizeof(T) == 4) { w[2 * m] = __float_as_uint(x); w[2 * m + 1] = __float_as_uint(y); }
    else if constexpr (std::is_same<T, __half>::value) { const __half2 v = __floats2half2_rn(x, y); w[m] = *reinterpret_cast<const uint32_t *>(&v); }
    else { const __nv_bfloat162 v = __floats2bfloat162_rn(x, y); w[m] = *reinterpret_cast<const uint32_t *>(&v); }
  }
};
// An item's 2V elements as pairs of floats: f[0..V/2) the first elements of the pairs that turn together, f[V/2..V) the second ones
template <bool interleaved, typename T, int V> __device__ __forceinline__ void spread(const Few<T, V> (&in)[2], float2 *f)
{
  if constexpr (interleaved) {
#pragma unroll
    for (int j = 0; j < V / 2; ++j) {
      const float2 a = in[2 * j / (V / 2)].two(2 * j % (V / 2)), b = in[(2 * j + 1) / (V / 2)].two((2 * j + 1) % (V / 2));
      f[j] = make_float2(a.x, b.x); f[V / 2 + j] = make_float2(a.y, b.y);
    }
  } else {
#pragma unroll
    for (int j = 0; j < V / 2; ++j) { f[j] = in[0].two(j); f[V / 2 + j] = in[1].two(j); }
  }
}
template <bool interleaved, typename T, int V> __device__ __forceinline__ void gather(Few<T, V> (&out)[2], const float2 *f)
{
  if constexpr (interleaved) {
#pragma unroll
    for (int j = 0; j < V / 2; ++j) {
      out[2 * j / (V / 2)].put(2 * j % (V / 2), f[j].x, f[V / 2 + j].x);
      out[(2 * j + 1) / (V / 2)].put((2 * j + 1) % (V / 2), f[j].y, f[V / 2 + j].y);
    }
  } else {
#pragma unroll
    for (int j = 0; j < V / 2; ++j) { out[0].put(j, f[j].x, f[j].y); out[1].put(j, f[V / 2 + j].x, f[V / 2 + j].y); }
  }
}

// The position of a unit's token `lane` (lanes beyond its tokens: 0), as it is asked for a unit ahead
__device__ __forceinline__ long long position_of(const RotaryArgs &a, uint32_t first, uint32_t tokens, uint32_t lane)
{
  if (lane >= tokens || first >= a.total || lane >= a.total - first) return 0;
  const uint32_t token = first + lane, b = a.batch == 1 ? 0 : token / a.seq;
  const uint64_t i = b * a.pos_batch + (token - b * a.seq) * a.pos_seq;
  return a.position_bytes == 8 ? static_cast<const long long *>(a.positions)[i] : static_cast<const int *>(a.positions)[i];
}
// Whole turns per position of each pair, for the block
__device__ __forceinline__ void make_rates(const RotaryArgs &a, double *rates)
{
  for (uint32_t i = threadIdx.x; i < a.rot / 2; i += kThreads) rates[i] = a.freq[i] * 0.15915494309189533577;      // 1/(2 pi)
}
// The cosines and sines of a unit's tokens: put(t, j, (cos, sin)) for each pair j of token t.  Angles are reduced to what is left of
// whole turns in f64: that is exact, and small.
template <typename Put> __device__ __forceinline__ void make_table(const RotaryArgs &a, const double *rates, uint32_t tokens, long long position, Put put)
{
  const uint32_t half = a.rot / 2, lane = threadIdx.x & 31, count = tokens * half, rounds = (count + 31) / 32;
  const uint32_t inverse = 0xffffffffu / half + 1;          // i/half = the upper half of i*inverse, for the few hundred i there are (half = 1: 0)
  const double own = (double)position;
#pragma unroll 2
  for (uint32_t n = 0; n < rounds; ++n) {
    const uint32_t i = n * 32 + lane, t = tokens == 1 ? 0 : half == 1 ? i : __umulhi(i, inverse), j = min(i - t * half, half - 1);
    const double turns = __shfl_sync(0xffffffffu, own, min(t, 31u)) * rates[j];
    float s, c;
    sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
    if (i < count) put(t, j, make_float2(c * a.amplitude, s * a.amplitude * a.way));
  }
}

// Where a group of lanes is: the unit, its head (none: from `end` on), the passes that the unit has left, and addresses
template <typename T> struct Place { uint32_t unit, head, end, left; const T *p, *x; };
// A group's way through its warp's units: as many heads at a time as the warp has groups
template <typename T> struct Walk {
  const RotaryArgs &a;
  const RotarySide &d;
  uint32_t group, groups, mine, step;       // mine: of the unit's tokens
  __device__ __forceinline__ Walk(const RotaryArgs &a, const RotarySide &d, uint32_t group, uint32_t groups)
      : a(a), d(d), group(group), groups(groups), mine(d.tokens > 1 ? group / d.heads : 0), step(d.blocks * kWarps) {}
  // the first token of a unit; none, beyond the last one
  __device__ __forceinline__ uint32_t token(uint32_t unit) const { return unit >= d.units ? a.total : d.parts > 1 ? unit / d.parts : unit * d.tokens; }
  // the first head of the unit
  __device__ __forceinline__ void enter(Place<T> &w, const HeadArray &p, const HeadArray *x) const
  {
    w.left = 1;
    w.head = w.end = 0;
    if (w.unit >= d.units) return;
    uint32_t token = w.unit * d.tokens + mine, low = 0;
    if (d.parts > 1) {
      token = w.unit / d.parts;
      const uint32_t part = w.unit - token * d.parts;
      low = part * d.span;
      w.left = part + 1 < d.parts ? d.passes : d.last;
    } else if (d.tokens == 1) w.left = d.last;
    const uint32_t head = low + group - mine * d.heads;
    uint32_t b = 0, s = token;
    if (a.batch > 1) { b = token / a.seq; s = token - b * a.seq; }
    w.p = static_cast<const T *>(p.p) + s * p.seq + head * p.head;
    if (x) w.x = static_cast<const T *>(x->p) + s * x->seq + head * x->head;
    if (a.batch > 1) {
      w.p += b * p.batch;
      if (x) w.x += b * x->batch;
    }
    if (mine < d.tokens && token < a.total && group < groups) { w.head = head; w.end = min(d.heads, low + d.span); }
  }
  // to the group's next head, `hop` further
  __device__ __forceinline__ void advance(Place<T> &w, const HeadArray &p, uint64_t hop, const HeadArray *x, uint64_t hop_x) const
  {
    if (--w.left) {
      w.head += groups; w.p += hop;         // (a group without a head stays without: its end is 0)
      if (x) w.x += hop_x;
    } else { w.unit += step; enter(w, p, x); }
  }
};
// The sum over a group of lanes, the same bits in all of them
__device__ __forceinline__ float group_sum(float v, uint32_t lanes, uint32_t first)
{
  if ((lanes & (lanes - 1)) == 0) {
#pragma unroll
    for (uint32_t o = 1; o < 32; o *= 2) if (o < lanes) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  }
  float sum = 0.0f;
  for (uint32_t i = 0; i < lanes; ++i) sum += __shfl_sync(0xffffffffu, v, first + i);
  return sum;
}

// Blocks of a multiprocessor: with more, which the forms without a norm would have registers for, [16384,40,128] took 62.3 us in the place of 58.7,
// with a norm 62.7 in the place of 56.5
__host__ __device__ constexpr int resident(int floats) { return floats > 16 ? 2 : 4; }
// Heads of a lane's ring, and its bytes
__host__ __device__ constexpr int ring_depth(int it) { return it == 1 ? 4 : 2; }
__host__ __device__ constexpr size_t ring_bytes(int v, int it, bool both, size_t e) { return (size_t)ring_depth(it) * kThreads * it * 2 * v * e * (both ? 2 : 1); }

template <typename T, int V, int IT, bool NORM, bool BWD, bool interleaved>
__global__ void __launch_bounds__(kThreads, resident(2 * V * IT)) rotary_heads_kernel(const RotaryArgs a)
{
  constexpr bool BOTH = NORM && BWD;        // two arrays are read
  constexpr bool KEEP = V * IT <= (BOTH ? 4 : 8);       // a lane's cosines and sines stay in its registers from head to head
  constexpr int DEPTH = ring_depth(IT), PIECES = IT * 2 * (BOTH ? 2 : 1), H = V / 2;
  typedef typename Few<T, V>::Raw Raw;
  // each pair's turns per position; the rings, [depth][piece][thread]; of each warp, [tokens] cosines and sines: pairs n and n + 1 of an item of a token at n/2*turned + item,
  // both cosines and then both sines, so that lanes read 16 bytes side by side; in their place the warps' sums of the weights' gradients, when
  // the block is done
  extern __shared__ float4 shared[];
  const uint32_t which = blockIdx.x >= a.side[0].blocks, block = which ? blockIdx.x - a.side[0].blocks : blockIdx.x;
  const RotarySide &d = a.side[which];
  const uint32_t wlane = threadIdx.x & 31, warp = threadIdx.x >> 5, groups = 32 / a.lanes, group = wlane / a.lanes, lane = wlane - group * a.lanes;
  const uint32_t half = a.rot / 2;
  double *rates = reinterpret_cast<double *>(shared);
  Raw *ring = reinterpret_cast<Raw *>(shared + half / 2) + threadIdx.x;
  float4 *table = shared + half / 2 + ring_bytes(V, IT, BOTH, sizeof(T)) / 16 + (size_t)warp * d.tokens * half / 2;
  // this lane's items: two vectors, at e0 and e1
  uint32_t e0[IT], e1[IT];
  bool has[IT], second[IT], turns[IT];
#pragma unroll
  for (int k = 0; k < IT; ++k) {
    const uint32_t p = lane + k * a.lanes;
    turns[k] = p < a.turned;
    has[k] = p < a.items;
    // (interleaved pairs are whole in either vector: these two lie apart, too, so that lanes side by side move 16 bytes side by side)
    e0[k] = turns[k] ? p * V : a.rot + (p - a.turned) * V;
    e1[k] = turns[k] ? half + p * V : e0[k] + (a.items - a.turned) * V;
    second[k] = has[k] && e1[k] < a.dim;
  }
  pdl_wait();
  make_rates(a, rates);
  const bool aligned_gamma = ((uintptr_t)d.gamma.p & 15) == 0;
  auto weights = [&](int k, float2 *g) {
    float v[2 * V];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t e = j ? e1[k] : e0[k];
#pragma unroll
      for (int i = 0; i < V; ++i) v[j * V + i] = 0.0f;
      if (!(j ? second[k] : has[k])) continue;
      if (aligned_gamma) d.gamma.load<V>(e, v + j * V);
      else d.gamma.load_each<V>(e, v + j * V);
    }
#pragma unroll
    for (int j = 0; j < V / 2; ++j) {
      g[j] = interleaved ? make_float2(v[4 * j], v[4 * j + 2]) : make_float2(v[2 * j], v[2 * j + 1]);
      g[V / 2 + j] = interleaved ? make_float2(v[4 * j + 1], v[4 * j + 3]) : make_float2(v[V + 2 * j], v[V + 2 * j + 1]);
    }
  };
  float2 g[NORM ? IT : 1][V], acc[BOTH ? IT : 1][V];
  if constexpr (NORM) {
#pragma unroll
    for (int k = 0; k < IT; ++k) {
      weights(k, g[k]);
#pragma unroll
      for (int i = 0; i < V; ++i) if constexpr (BOTH) acc[k][i] = both(0.0f);
    }
  }
  // (what a lane does not have is never copied, and counts as zeros)
#pragma unroll
  for (int k = 0; k < IT; ++k)
#pragma unroll
    for (int j = 0; j < 2; ++j)
      if (!(j ? second[k] : has[k]))
        for (int i = 0; i < DEPTH; ++i) {
          ring[(i * PIECES + 2 * k + j) * kThreads] = Raw{};
          if constexpr (BOTH) ring[(i * PIECES + 2 * IT + 2 * k + j) * kThreads] = Raw{};
        }
  const Walk<T> walk(a, d, group, groups);
  const uint64_t hop = d.in.head * groups, hop_x = BOTH ? d.x.head * groups : 0, hop_out = d.out.head * groups;
  uint32_t turn_in = 0, turn_out = 0;        // the ring's places that are filled and emptied next
  auto load = [&](const Place<T> &w) {
    if (w.head < w.end) {
#pragma unroll
      for (int k = 0; k < IT; ++k)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if (!(j ? second[k] : has[k])) continue;
          const uint32_t e = j ? e1[k] : e0[k];
          copy_async<V * sizeof(T)>(ring + (turn_in * PIECES + 2 * k + j) * kThreads, w.p + e);
          if constexpr (BOTH) copy_async<V * sizeof(T)>(ring + (turn_in * PIECES + 2 * IT + 2 * k + j) * kThreads, w.x + e);
        }
    }
    copies_commit();
    turn_in = (turn_in + 1) & (DEPTH - 1);
  };
  // f -> f*straight + (its partner)*across, with the forward pass's weights in it (without them the two halves share their cosines, and
  // across holds the sines)
  constexpr bool WEIGHED = NORM && !BWD;
  struct Turn { float2 straight[WEIGHED ? V : H], across[WEIGHED ? V : H]; };
  const uint32_t row = min(walk.mine, d.tokens - 1);       // (a group without a token reads another's: it stays within the table)
  auto coefficients = [&](int k, Turn &o) {
    const float2 *by = g[NORM ? k : 0];
    const uint32_t from = row * half / 2 + (turns[k] ? lane + k * a.lanes : 0);
#pragma unroll
    for (int i = 0; i < H; ++i) {
      float4 t = table[from + i * a.turned];
      if constexpr (WEIGHED) {
        if (!turns[k]) t = make_float4(1.0f, 1.0f, 0.0f, 0.0f);
        const float2 c = make_float2(t.x, t.y), s = make_float2(t.z, t.w), minus = make_float2(-t.z, -t.w);
        o.straight[i] = mul2(by[i], c); o.across[i] = mul2(by[H + i], minus);
        o.straight[H + i] = mul2(by[H + i], c); o.across[H + i] = mul2(by[i], s);
      } else {
        o.straight[i] = make_float2(t.x, t.y);
        o.across[i] = make_float2(t.z, t.w);
      }
    }
  };
  auto turn = [&](int k, float2 *f, const Turn &o) {
    if (turns[k]) {
#pragma unroll
      for (int j = 0; j < H; ++j) {
        const float2 u = f[j], v = f[H + j];
        if constexpr (WEIGHED) f[j] = fma2(v, o.across[j], mul2(u, o.straight[j]));
        else f[j] = fma2(mul2(v, o.across[j]), both(-1.0f), mul2(u, o.straight[j]));
        f[H + j] = fma2(u, o.across[WEIGHED ? H + j : j], mul2(v, o.straight[WEIGHED ? H + j : j]));
      }
    } else if (WEIGHED) {      // (elements that pass have no partner: its infinity would be a NaN here)
#pragma unroll
      for (int j = 0; j < V; ++j) f[j] = mul2(f[j], o.straight[j]);
    }
  };
  Turn kept[KEEP ? IT : 1];
  const HeadArray *from = BOTH ? &d.x : nullptr;
  Place<T> at, ahead;
  at.unit = ahead.unit = block * kWarps + warp;
  walk.enter(at, d.out, nullptr);
  walk.enter(ahead, d.in, from);
  long long position = position_of(a, walk.token(at.unit), d.tokens, wlane);
#pragma unroll
  for (int i = 0; i < DEPTH - 1; ++i) {
    load(ahead);
    walk.advance(ahead, d.in, hop, from, hop_x);
  }
  __syncthreads();
  while (at.unit < d.units) {
    // the unit's cosines and sines
    __syncwarp();
    make_table(a, rates, d.tokens, position, [&](uint32_t t, uint32_t j, float2 cs) {
      // pair n of item `item`
      const uint32_t late = interleaved && j >= half / 2, of = interleaved ? j - late * (half / 2) : j;
      const uint32_t item = of / (interleaved ? H : V), n = interleaved ? late * H + of % H : of % V;
      float *to = reinterpret_cast<float *>(table + t * half / 2 + n / 2 * a.turned + item) + n % 2;
      to[0] = cs.x; to[2] = cs.y;
    });
    position = position_of(a, walk.token(at.unit + walk.step), d.tokens, wlane);
    __syncwarp();
    if constexpr (KEEP) {
#pragma unroll
      for (int k = 0; k < IT; ++k) coefficients(k, kept[k]);
    }
    for (const uint32_t unit = at.unit; at.unit == unit;) {
      const bool live = at.head < at.end;
      load(ahead);
      walk.advance(ahead, d.in, hop, from, hop_x);
      copies_wait<DEPTH - 1>();
      float2 f[IT][V], sq2 = both(0.0f);
#pragma unroll
      for (int k = 0; k < IT; ++k) {
        Few<T, V> in[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) in[j].raw = ring[(turn_out * PIECES + 2 * k + j) * kThreads];
        spread<interleaved>(in, f[k]);
      }
      if constexpr (NORM && !BWD) {
#pragma unroll
        for (int k = 0; k < IT; ++k)
#pragma unroll
          for (int i = 0; i < V; ++i) sq2 = fma2(f[k][i], f[k][i], sq2);
        const float2 r = both(rsqrtf(group_sum(sq2.x + sq2.y, a.lanes, wlane - lane) * a.inv_dim + a.epsilon));
#pragma unroll
        for (int k = 0; k < IT; ++k)
#pragma unroll
          for (int i = 0; i < V; ++i) f[k][i] = mul2(f[k][i], r);
      }
#pragma unroll
      for (int k = 0; k < IT; ++k) {
        if constexpr (KEEP) turn(k, f[k], kept[KEEP ? k : 0]);
        else {
          Turn own;
          coefficients(k, own);
          turn(k, f[k], own);
        }
      }
      if constexpr (BOTH) {
        float2 x[IT][V], dot2 = both(0.0f);
#pragma unroll
        for (int k = 0; k < IT; ++k) {
          Few<T, V> in[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) in[j].raw = ring[(turn_out * PIECES + 2 * IT + 2 * k + j) * kThreads];
          spread<interleaved>(in, x[k]);
#pragma unroll
          for (int i = 0; i < V; ++i) { sq2 = fma2(x[k][i], x[k][i], sq2); dot2 = fma2(mul2(f[k][i], g[k][i]), x[k][i], dot2); }
        }
        const float r = rsqrtf(group_sum(sq2.x + sq2.y, a.lanes, wlane - lane) * a.inv_dim + a.epsilon);
        // (1/rms meets the sum, the head's elements and the bracket one at a time: its powers alone may leave f32's range)
        const float2 r2 = both(r), minus = both(-group_sum(dot2.x + dot2.y, a.lanes, wlane - lane) * r * a.inv_dim);
        if (live) {
#pragma unroll
          for (int k = 0; k < IT; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) {
              const float2 xh = mul2(x[k][i], r2);
              acc[k][i] = fma2(f[k][i], xh, acc[k][i]);
              f[k][i] = mul2(fma2(f[k][i], g[k][i], mul2(xh, minus)), r2);
            }
        }
      }
      turn_out = (turn_out + 1) & (DEPTH - 1);
      if (live) {
        T *out = const_cast<T *>(at.p);
#pragma unroll
        for (int k = 0; k < IT; ++k) {
          Few<T, V> o[2];
          gather<interleaved>(o, f[k]);
          if (has[k]) *reinterpret_cast<Raw *>(out + e0[k]) = o[0].raw;
          if (second[k]) *reinterpret_cast<Raw *>(out + e1[k]) = o[1].raw;
        }
      }
      walk.advance(at, d.out, hop_out, nullptr, 0);
    }
  }
  if constexpr (BOTH) {
    if (!d.want) return;
    // the groups' sums join within the warp (those of other than a power of two lanes add theirs in turn), then the warps'
    float *sums = reinterpret_cast<float *>(shared);
    copies_wait<0>();
    pdl_trigger();
    const bool even = (a.lanes & (a.lanes - 1)) == 0;
    if (even) {
#pragma unroll
      for (int k = 0; k < IT; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i)
          for (uint32_t o = a.lanes; o < 32; o *= 2) {
            acc[k][i].x += __shfl_xor_sync(0xffffffffu, acc[k][i].x, o);
            acc[k][i].y += __shfl_xor_sync(0xffffffffu, acc[k][i].y, o);
          }
    }
    __syncthreads();
    for (uint32_t n = 0; n < (even ? 1 : groups); ++n) {
      if (group == n) {
#pragma unroll
        for (int k = 0; k < IT; ++k)
#pragma unroll
          for (int j = 0; j < 2 * V; ++j) {
            // element j of the item, of the pairs as spread() has them
            const float2 v2 = interleaved ? acc[k][(j % 2) * (V / 2) + j / 4] : acc[k][(j / V) * (V / 2) + j % V / 2];
            const float v = (interleaved ? j / 2 % 2 : j % 2) ? v2.y : v2.x;
            if (!(j < V ? has[k] : second[k])) continue;
            float *to = sums + (size_t)warp * a.dim + (j < V ? e0[k] + j : e1[k] + j - V);
            *to = n ? *to + v : v;
          }
      }
      __syncwarp();
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

constexpr int kPairsDepth = 4;

// Heads whose pairs lie anywhere.  They are copied as they lie, `copy` bytes at a time, into places of `slot` bytes; a lane has IT pairs, lanes
// side by side, or as many elements that pass.  DEPTH places to a group: the next heads are on their way while one is worked on.
template <typename T, int IT, bool NORM, bool BWD>
__global__ void __launch_bounds__(kThreads, IT > 8 ? 2 : 4) rotary_pairs_kernel(const RotaryArgs a)
{
  constexpr bool BOTH = NORM && BWD;
  constexpr int DEPTH = kPairsDepth, ARRAYS = BOTH ? 2 : 1;
  // each pair's turns per position; of each warp, the heads' places [depth][array][group] and the cosines and sines [tokens][rot/2]; then the
  // sums of the weights' gradients
  extern __shared__ float4 shared[];
  const uint32_t which = blockIdx.x >= a.side[0].blocks, block = which ? blockIdx.x - a.side[0].blocks : blockIdx.x;
  const RotarySide &d = a.side[which];
  const uint32_t wlane = threadIdx.x & 31, warp = threadIdx.x >> 5, groups = 32 / a.lanes, group = wlane / a.lanes, lane = wlane - group * a.lanes;
  const uint32_t half = a.rot / 2, bytes = a.dim * (uint32_t)sizeof(T);
  double *rates = reinterpret_cast<double *>(shared);
  char *base = reinterpret_cast<char *>(shared + (half + 1) / 2), *places = base + (size_t)warp * DEPTH * ARRAYS * groups * a.slot;
  float2 *table = reinterpret_cast<float2 *>(base + (size_t)kWarps * DEPTH * ARRAYS * groups * a.slot) + (size_t)warp * d.tokens * half;
  // (lanes beyond the last group read, and drop, what it has)
  auto place = [&](uint32_t turn, int array) { return places + ((turn * ARRAYS + array) * groups + min(group, groups - 1)) * a.slot; };
  uint32_t e0[IT], e1[IT];
  bool has[IT], second[IT], turns[IT];
#pragma unroll
  for (int k = 0; k < IT; ++k) {
    const uint32_t p = lane + k * a.lanes;
    turns[k] = p < half;
    has[k] = p < a.items;
    e0[k] = !turns[k] ? a.rot + (p - half) * 2 : a.interleaved ? p * 2 : p;
    e1[k] = turns[k] && !a.interleaved ? half + p : e0[k] + 1;
    second[k] = has[k] && e1[k] < a.dim;
  }
  pdl_wait();
  make_rates(a, rates);
  float2 g[NORM ? IT : 1], acc[BOTH ? IT : 1];
  if constexpr (NORM) {
    uint32_t column[2 * IT];
#pragma unroll
    for (int k = 0; k < IT; ++k) {
      column[2 * k] = has[k] ? e0[k] : a.dim;
      column[2 * k + 1] = second[k] ? e1[k] : a.dim;
      if constexpr (BOTH) acc[k] = both(0.0f);
    }
    d.gamma.gather<2 * IT>(column, a.dim, reinterpret_cast<float *>(g));
  }
  const Walk<T> walk(a, d, group, groups);
  const uint64_t hop = d.in.head * groups, hop_x = BOTH ? d.x.head * groups : 0, hop_out = d.out.head * groups;
  const HeadArray *from = BOTH ? &d.x : nullptr;
  uint32_t turn_in = 0, turn_out = 0;
  auto load = [&](const Place<T> &w) {
    if (w.head < w.end) {
#pragma unroll
      for (int n = 0; n < ARRAYS; ++n) {
        char *to = place(turn_in, n);
        const char *p = reinterpret_cast<const char *>(n ? w.x : w.p);
        for (uint32_t i = lane * a.copy; i < bytes; i += a.lanes * a.copy) {
          if (a.copy == 16) copy_async<16>(to + i, p + i);
          else if (a.copy == 8) copy_async<8>(to + i, p + i);
          else if (a.copy == 4) copy_async<4>(to + i, p + i);
          else *reinterpret_cast<uint16_t *>(to + i) = *reinterpret_cast<const uint16_t *>(p + i);
        }
      }
    }
    copies_commit();
    turn_in = (turn_in + 1) & (DEPTH - 1);
  };
  Place<T> at, ahead;
  at.unit = ahead.unit = block * kWarps + warp;
  walk.enter(at, d.out, nullptr);
  walk.enter(ahead, d.in, from);
  long long position = position_of(a, walk.token(at.unit), d.tokens, wlane);
#pragma unroll
  for (int i = 0; i < DEPTH - 1; ++i) {
    load(ahead);
    walk.advance(ahead, d.in, hop, from, hop_x);
  }
  __syncthreads();
  while (at.unit < d.units) {
    __syncwarp();
    make_table(a, rates, d.tokens, position, [&](uint32_t t, uint32_t j, float2 cs) { table[t * half + j] = cs; });
    position = position_of(a, walk.token(at.unit + walk.step), d.tokens, wlane);
    __syncwarp();
    const float2 *cs = table + min(walk.mine, d.tokens - 1) * half;
    for (const uint32_t unit = at.unit; at.unit == unit;) {
      const bool live = at.head < at.end;
      load(ahead);
      walk.advance(ahead, d.in, hop, from, hop_x);
      copies_wait<DEPTH - 1>();
      __syncwarp();                       // (lanes read what others copied)
      T *in = reinterpret_cast<T *>(place(turn_out, 0));
      const T *xin = BOTH ? reinterpret_cast<const T *>(place(turn_out, 1)) : nullptr;
      float2 f[IT];
      float sq = 0.0f, dot = 0.0f;
#pragma unroll
      for (int k = 0; k < IT; ++k) f[k] = make_float2(has[k] ? to_float(in[e0[k]]) : 0.0f, second[k] ? to_float(in[e1[k]]) : 0.0f);
      auto turned = [&](int k) {
        if (!turns[k]) return;
        const float2 w = cs[lane + k * a.lanes], v = f[k];
        f[k] = make_float2(v.x * w.x - v.y * w.y, v.x * w.y + v.y * w.x);
      };
      if constexpr (NORM && !BWD) {
#pragma unroll
        for (int k = 0; k < IT; ++k) sq = fmaf(f[k].x, f[k].x, fmaf(f[k].y, f[k].y, sq));
        const float r = rsqrtf(group_sum(sq, a.lanes, wlane - lane) * a.inv_dim + a.epsilon);
#pragma unroll
        for (int k = 0; k < IT; ++k) f[k] = mul2(f[k], mul2(g[k], both(r)));
      }
#pragma unroll
      for (int k = 0; k < IT; ++k) turned(k);
      if constexpr (BOTH) {
        float2 x[IT];
#pragma unroll
        for (int k = 0; k < IT; ++k) {
          x[k] = make_float2(has[k] ? to_float(xin[e0[k]]) : 0.0f, second[k] ? to_float(xin[e1[k]]) : 0.0f);
          sq = fmaf(x[k].x, x[k].x, fmaf(x[k].y, x[k].y, sq));
          dot = fmaf(f[k].x * g[k].x, x[k].x, fmaf(f[k].y * g[k].y, x[k].y, dot));
        }
        const float r = rsqrtf(group_sum(sq, a.lanes, wlane - lane) * a.inv_dim + a.epsilon);
        const float2 r2 = both(r), minus = both(-group_sum(dot, a.lanes, wlane - lane) * r * a.inv_dim);
        if (live) {
#pragma unroll
          for (int k = 0; k < IT; ++k) {
            const float2 xh = mul2(x[k], r2);
            acc[k] = fma2(f[k], xh, acc[k]);
            f[k] = mul2(fma2(f[k], g[k], mul2(xh, minus)), r2);
          }
        }
      }
      // back into the place, each element by the lane that read it, and out as it was copied in
      if (live) {
#pragma unroll
        for (int k = 0; k < IT; ++k) {
          if (has[k]) in[e0[k]] = from_float<T>(f[k].x);
          if (second[k]) in[e1[k]] = from_float<T>(f[k].y);
        }
      }
      __syncwarp();
      if (live) {
        char *out = reinterpret_cast<char *>(const_cast<T *>(at.p));
        const char *p = reinterpret_cast<const char *>(in);
        for (uint32_t i = lane * a.copy; i < bytes; i += a.lanes * a.copy) {
          if (a.copy == 16) *reinterpret_cast<uint4 *>(out + i) = *reinterpret_cast<const uint4 *>(p + i);
          else if (a.copy == 8) *reinterpret_cast<uint2 *>(out + i) = *reinterpret_cast<const uint2 *>(p + i);
          else if (a.copy == 4) *reinterpret_cast<uint32_t *>(out + i) = *reinterpret_cast<const uint32_t *>(p + i);
          else *reinterpret_cast<uint16_t *>(out + i) = *reinterpret_cast<const uint16_t *>(p + i);
        }
      }
      turn_out = (turn_out + 1) & (DEPTH - 1);
      walk.advance(at, d.out, hop_out, nullptr, 0);
      // (the place is filled anew by copies of the lanes that emptied it, and the array beside it after every lane has passed the barrier above)
    }
  }
  if constexpr (BOTH) {
    if (!d.want) return;
    float *sums = reinterpret_cast<float *>(shared);
    copies_wait<0>();
    __syncthreads();
    for (uint32_t n = 0; n < groups; ++n) {
      if (group == n) {
#pragma unroll
        for (int k = 0; k < IT; ++k) {
          float *to = sums + (size_t)warp * a.dim;
          if (has[k]) to[e0[k]] = n ? to[e0[k]] + acc[k].x : acc[k].x;
          if (second[k]) to[e1[k]] = n ? to[e1[k]] + acc[k].y : acc[k].y;
        }
      }
      __syncwarp();
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
  // (half of the blocks that there may be are asked for at once)
  constexpr uint32_t kEach = kMostParts / 64;
  const uint32_t end = k ? blocks : q_blocks;
  float sum = 0.0f;
  for (uint32_t first = (k ? q_blocks : 0) + warp; first < end; first += 32 * kEach) {
    float v[kEach];
#pragma unroll
    for (uint32_t n = 0; n < kEach; ++n) v[n] = i < dim && first + 32 * n < end ? partial[(uint64_t)(first + 32 * n) * dim + i] : 0.0f;
#pragma unroll
    for (uint32_t n = 0; n < kEach; ++n) sum += v[n];
  }
  sums[warp][lane] = sum;
  __syncthreads();
  // a warp per element: a lane's term of each
  sum = warp_sum_all(sums[lane][warp]);
  const uint32_t mine = (blockIdx.x - k * wide) * 32 + warp;
  if (lane == 0 && mine < dim) put_weight(out, type, mine, sum);
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

// V = 1: pairs anywhere
template <typename T, int V, int IT, bool NORM, bool BWD>
int launch_rotary(const RotaryArgs &a, uint32_t blocks, size_t tables, size_t sums, cudaStream_t stream)
{
  void (*kernel)(RotaryArgs);
  size_t shared;
  if constexpr (V == 1) {
    kernel = rotary_pairs_kernel<T, IT, NORM, BWD>;
    shared = (size_t)kWarps * kPairsDepth * (NORM && BWD ? 2 : 1) * (32 / a.lanes) * a.slot + tables;
  } else {
    kernel = a.interleaved ? rotary_heads_kernel<T, V, IT, NORM, BWD, true> : rotary_heads_kernel<T, V, IT, NORM, BWD, false>;
    shared = ring_bytes(V, IT, NORM && BWD, sizeof(T)) + tables;
  }
  if (shared < sums) shared = sums;
  static SharedMemory allowed[2];
  if (!allowed[a.interleaved].up_to((const void *)kernel, shared)) return ANODE_E_LAUNCH;
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
  // queries and keys are worked on side by side: no output of one is in the place of an array of the other
  if (two) {
    if (c.dgamma[0] && c.dgamma[0] == c.dgamma[1]) return ANODE_E_STRIDE;
    for (int k = 0; k < 2; ++k) {
      const void *out = c.out[k]->data;
      if (out && (out == c.out[!k]->data || out == c.in[!k]->data || (c.bwd && a.norm && out == c.x[!k]->data))) return ANODE_E_STRIDE;
    }
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
  // lanes of a head's group: as many as it has items, in a power of two where others would not make more groups of a warp
  // (pairs anywhere: eight to a lane where the heads fill the device, else two, which a warp is done with sooner: backward, 64 tokens
  // of 40 heads, 62 of 128 turned, 12.5 us and 7.5)
  const bool few = (uint64_t)a.batch * a.seq * (a.side[0].heads + a.side[1].heads) < 64ull * sm_count();
  const uint32_t per_lane = v > 1 ? 1 : few && a.items <= 64 ? 2 : a.items > 32 ? 8 : (a.items + 3) / 4, wide = (a.items + per_lane - 1) / per_lane;
  a.lanes = 1;
  while (a.lanes < 32 && a.lanes < wide) a.lanes *= 2;
  if (wide < 32 && 32 / wide > 32 / a.lanes) a.lanes = wide;
  const uint32_t each = (a.items + a.lanes - 1) / a.lanes, groups = 32 / a.lanes;
  if (v == 1) {
    a.copy = 16;
    auto copies = [&](uint32_t n) {
      if (a.dim * e % n) return false;
      for (int k = 0; k < 1 + two; ++k)
        for (const AnodeHeads *h : {c.in[k], c.out[k], c.bwd && a.norm ? c.x[k] : nullptr})
          if (h && (!aligned_to(h->data, n) || (a.batch > 1 && h->batch_stride * e % n) || (a.seq > 1 && h->seq_stride * e % n) || (h->heads > 1 && h->head_stride * e % n)))
            return false;
      return true;
    };
    while (a.copy > e && !copies(a.copy)) a.copy /= 2;
    a.slot = (uint32_t)((a.dim * e + 15) / 16 * 16 + 16);      // (16 more, so that groups side by side read other banks)
  }
  // blocks that the device holds; both arrays' warps work side by side, as many on either as its share of the heads asks for
  const uint32_t room = sm_count() * (uint32_t)(v == 1 ? each > 8 ? 2 : 4 : resident((int)(2 * v * each)));
  uint64_t all_passes = 0;
  uint32_t blocks = 0, most = 1, units[2], passes[2];
  double cost[2] = {0.0, 0.0};
  for (int k = 0; k < 1 + two; ++k) {
    RotarySide &d = a.side[k];
    // a warp has tokens that fill it, or a token's heads
    d.tokens = d.heads < groups ? groups / d.heads : 1;
    while (d.tokens > 1 && d.tokens * (a.rot / 2) > 512) --d.tokens;
    units[k] = (a.total - 1) / d.tokens + 1;
    passes[k] = (d.heads + groups - 1) / groups;
    if (d.tokens > most) most = d.tokens;
    all_passes += (uint64_t)units[k] * passes[k];
  }
  const uint64_t each_passes = (all_passes - 1) / (room * kWarps) + 1;
  for (int k = 0; k < 1 + two; ++k) {
    RotarySide &d = a.side[k];
    // or, where that leaves warps of the device idle, a span of them
    d.span = (d.tokens > 1 || each_passes > passes[k] ? passes[k] : (uint32_t)each_passes) * groups;
    d.parts = (d.heads + d.span - 1) / d.span;
    d.passes = d.span / groups;
    d.last = (d.heads - (d.parts - 1) * d.span + groups - 1) / groups;
    d.units = units[k] * d.parts;
    cost[k] = (double)units[k] * (passes[k] + 2.5 * d.parts);        // (the cosines and sines cost a unit about two and a half passes)
  }
  for (int k = 0; k < 1 + two; ++k) {
    RotarySide &d = a.side[k];
    const uint32_t need = (d.units - 1) / kWarps + 1, share = (uint32_t)(room * cost[k] / (cost[0] + cost[1]));
    d.blocks = need < share ? need : share ? share : 1;
    blocks += d.blocks;
  }
  const size_t tables = (size_t)kWarps * most * (a.rot / 2) * 8 + (a.rot / 2 + 1) / 2 * 16,      // and the pairs' rates
                sums = wants ? (size_t)kWarps * a.dim * 4 : 0;
  TRY(by_type(c.type, [&](auto t) {
    using T = decltype(t);
    auto with = [&](auto norm, auto bwd) {
      constexpr bool N = decltype(norm)::value, B = decltype(bwd)::value;
      if constexpr (sizeof(T) == 2)
        if (v == 8) return each == 1 ? launch_rotary<T, 8, 1, N, B>(a, blocks, tables, sums, stream) : launch_rotary<T, 8, 2, N, B>(a, blocks, tables, sums, stream);
      if (v == 4) return each == 1 ? launch_rotary<T, 4, 1, N, B>(a, blocks, tables, sums, stream)
                       : each == 2 ? launch_rotary<T, 4, 2, N, B>(a, blocks, tables, sums, stream) : launch_rotary<T, 4, 4, N, B>(a, blocks, tables, sums, stream);
      return each <= 2 ? launch_rotary<T, 1, 2, N, B>(a, blocks, tables, sums, stream) : each <= 8 ? launch_rotary<T, 1, 8, N, B>(a, blocks, tables, sums, stream) : launch_rotary<T, 1, 16, N, B>(a, blocks, tables, sums, stream);
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
