// Log probabilities of given tokens, the entropies of their rows and the likeliest tokens, and the gradient of the logits.
//
//   m = max x, z = scale*(x - m), L = log(sum(exp(z))):   logprob = z[token] - L,   H = L - sum(z*exp(z))/sum(exp(z))
//   p = exp(z - L):   dx = scale*(dlogprob*([token] - p) - dentropy*p*(z - L + H))
//
// A row keeps m and L apart, since their sum would lose L's digits beside a large m.
//
// Measured on one B200 against its copy bandwidth of 6539 GB/s: bf16 [4096,131072] with entropies 163 us (1.00; 188 in a loop of seconds, near the power cap), [4096,50021]
// 72 to 74 us (0.85 to 0.87), [256,131072] 15 to 16 us; f32 [16,131072] with the likeliest twenty 11.4 to 12.5 us, without 5.7.  Gradient bf16 [4096,50021] with entropies 128 us (0.98), without 123 (1.02: its last writes
// are still in the second-level cache when the clock stops); where dlogits does not begin its rows at the logits' places of 16 bytes, element by element, 439 us.
// Many long rows are bound by memory (an exponential for each logit keeps its unit busy for 60 % of the time), few by the chain load -> sums -> cluster -> store.
#include "bn_host.h"
#include "rows.cuh"

namespace anode_b200 {
namespace rows {
namespace log_probs {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kMostThreads = 512, kMostTop = 128;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kFloor = -1e4f;            // below what exp leaves above zero: 0 takes the place of 0 * -infinity

struct ProbsArgs {
  uint64_t rows;
  uint32_t vocab;
  float scale;
  const void *logits;
  uint64_t stride;
  const void *token;
  int token_bytes;
  float *logprob, *entropy;
  float2 *stats;
  uint32_t top;
  float *top_logprob;
  void *top_token;
  int top_token_bytes;
};

struct ProbsGradArgs {
  uint64_t rows;
  uint32_t vocab;
  float scale;
  const void *logits;
  uint64_t stride;
  const void *token;
  int token_bytes;
  const float2 *stats;
  const float *entropy, *dlogprob, *dentropy;
  void *dlogits;
  uint64_t dstride;
};

__device__ __forceinline__ float max_nan(float a, float b)
{
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
// Bits in the order of the values, of either zero the same; a NaN above all
__device__ __forceinline__ uint32_t order_of(float v)
{
  const uint32_t b = __float_as_uint(v + 0.0f);
  return v != v ? 0xffffffffu : b >> 31 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t order)
{
  return __uint_as_float(order == 0xffffffffu ? 0x7fffffffu : order >> 31 ? order & 0x7fffffffu : ~order);
}
// the larger value, of equal ones the lower index, is the larger key
__device__ __forceinline__ uint64_t key_of(float v, uint32_t index) { return (uint64_t)order_of(v) << 32 | (uint32_t)~index; }

__device__ __forceinline__ void put_top(const ProbsArgs &a, uint64_t row, uint32_t k, uint64_t key, float m, float log_sum)
{
  const float v = value_of((uint32_t)(key >> 32));
  const uint64_t at = row * a.top + k;
  if (a.top_logprob) a.top_logprob[at] = m == -INFINITY ? m : a.scale * (v - m) - log_sum;
  if (a.top_token) {
    if (a.top_token_bytes == 8) static_cast<int64_t *>(a.top_token)[at] = (uint32_t)~key;
    else static_cast<int32_t *>(a.top_token)[at] = (int32_t)~(uint32_t)key;
  }
}

// 2^v; v below -126 gives 0
__device__ __forceinline__ float exp2_of(float v)
{
  float d;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(d) : "f"(v));
  return d;
}

// Slots of 16 bytes of logits: the largest and the smallest (a NaN is the largest), two at a time where they have 16 bits; and a slot of what is none
template <typename T> struct Extremes {
  typedef typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type Pair;
  typedef typename std::conditional<sizeof(T) == 4, float, Pair>::type Value;
  Value high, low;
  __device__ __forceinline__ static Value at(const uint4 &v, int i)
  {
    const uint32_t w = i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
    return *reinterpret_cast<const Value *>(&w);
  }
  __device__ __forceinline__ void start(const uint4 &v) { high = low = at(v, 0); }
  template <bool LOW> __device__ __forceinline__ void take(const uint4 &v, int from)
  {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i < from) continue;
      if constexpr (sizeof(T) == 4) { high = max_nan(high, at(v, i)); if (LOW) low = fminf(low, at(v, i)); }
      else { high = __hmax2_nan(high, at(v, i)); if (LOW) low = __hmin2(low, at(v, i)); }
    }
  }
  __device__ __forceinline__ float largest() const { if constexpr (sizeof(T) == 4) return high; else return max_nan(to_float(high.x), to_float(high.y)); }
  __device__ __forceinline__ float smallest() const { if constexpr (sizeof(T) == 4) return low; else return fminf(to_float(low.x), to_float(low.y)); }
};
template <typename T> __device__ __forceinline__ uint4 nothing()
{
  constexpr uint32_t w = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;      // -infinity
  return make_uint4(w, w, w, w);
}

// Of some logits: the largest, the sum of 2^d over them and that of d*2^d, d = (x - largest)*rate in powers of two (log2(e)*scale is `rate`)
struct Sums {
  float m, sum, dot;
  // as if the largest were `to`
  __device__ __forceinline__ void move(float to, float rate)
  {
    const float d = max_nan((m - (to == -INFINITY ? 0.0f : to)) * rate, kFloor), by = exp2_of(d);
    dot = by * fmaf(d, sum, dot);
    sum *= by;
    m = to;
  }
};

constexpr uint32_t kBuffer = 512;          // keys that may be among the likeliest

// A row's logits are shared out to a cluster's blocks, and theirs to the threads by slots of 16 bytes in turn: one pass with a running maximum and sums that
// follow it.  The likeliest: the k-th largest of the threads' maxima is a bound that k logits reach at least, so that few threads have more of them, whose
// slots are read again.
template <typename T, bool ENTROPY, bool TOP>
__global__ void __launch_bounds__(kMostThreads, 2) token_log_probs_kernel(const ProbsArgs a, const uint32_t cluster)
{
  constexpr int V = Vec<T>::V, U = 4;
  __shared__ Sums sums[kMostThreads / 32], block_sums;
  __shared__ uint64_t buffer[TOP ? kBuffer : 1], best[TOP ? kMostTop : 1];
  extern __shared__ uint64_t lists[];        // of a cluster: its blocks' likeliest
  __shared__ uint32_t listed[TOP ? kMostThreads : 1], count, bound_count;
  const uint32_t threads = blockDim.x, warps = threads / 32, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t rank = cluster > 1 ? cluster_rank() : 0;
  const float rate = fminf(a.scale * kLog2e, 3.402823466e38f);
  auto sync = [&] { if (cluster > 1) cluster_sync(); else __syncthreads(); };
  pdl_wait();
  pdl_trigger();
  for (uint64_t row = blockIdx.x / cluster; row < a.rows; row += gridDim.x / cluster) {
    const T *x = static_cast<const T *>(a.logits) + row * a.stride;
    // logits before the first whole slot, slots, and logits behind the last; this block's slots [begin, end)
    const uint32_t head = min(a.vocab, (uint32_t)(-(int)((uintptr_t)x / sizeof(T)) & (V - 1))), slots = (a.vocab - head) / V, tail = a.vocab - head - slots * V;
    const uint32_t part = (slots + cluster - 1) / cluster, begin = min(slots, rank * part), end = min(slots, begin + part);
    const uint4 *from = reinterpret_cast<const uint4 *>(x + head);
    const bool on_edge = rank == 0 && threadIdx.x < head + tail, first = rank == 0 && threadIdx.x == 0;
    const uint32_t edge = threadIdx.x < head ? threadIdx.x : a.vocab - tail + (threadIdx.x - head);
    uint32_t token = a.vocab;
    float picked = 0.0f;
    if (first && a.logprob) {
      token = token_at(a.token, a.token_bytes, row, a.vocab);
      if (token < a.vocab) picked = to_float(x[token]);
    }
    // (sums of every second logit)
    float m = -INFINITY;
    float2 sum = both(0.0f), dot = both(0.0f);
    const float2 times = both(rate);
    auto absorb = [&](const uint4 *v, auto slots_here) {
      constexpr int N = decltype(slots_here)::value;
      Extremes<T> x;
      x.start(v[0]);
#pragma unroll
      for (int u = 0; u < N; ++u) x.template take<ENTROPY>(v[u], u == 0);
      const float to = max_nan(m, x.largest()), base = to == -INFINITY ? 0.0f : to;
      const float moved = max_nan((m - base) * rate, kFloor);
      const float2 by = both(exp2_of(moved));
      if (ENTROPY) dot = mul2(by, fma2(both(moved), sum, dot));
      sum = mul2(by, sum);
      m = to;
      const float2 minus = both(-base);
      auto add = [&](auto clamped) {
#pragma unroll
        for (int u = 0; u < N; ++u) {
          float2 f[V / 2];
          Vec<T>{v[u]}.floats(reinterpret_cast<float *>(f));
#pragma unroll
          for (int i = 0; i < V / 2; ++i) {
            float2 d = mul2(add2(f[i], minus), times);
            if (decltype(clamped)::value) d = make_float2(max_nan(d.x, kFloor), max_nan(d.y, kFloor));
            const float2 e = make_float2(exp2_of(d.x), exp2_of(d.y));
            sum = add2(sum, e);
            if (ENTROPY) dot = fma2(d, e, dot);
          }
        }
      };
      // (0 times -infinity is to be 0: where some logit is that far below)
      if (!ENTROPY || (x.smallest() - base) * rate >= kFloor) add(std::false_type());
      else add(std::true_type());
    };
    const uint32_t at = begin + threadIdx.x, mine = at < end ? (end - at + threads - 1) / threads : 0;       // this thread's slots
    const uint4 *p = from + at;
    auto fetch = [&](uint4 *to) {
#pragma unroll
      for (int u = 0; u < U; ++u) to[u] = p[u * threads];
      p += U * threads;
    };
    typedef std::integral_constant<int, U> Step;
    // two steps in turn, one on its way while the other is used
    uint4 one[U], two[U];
    uint32_t steps = mine / U;
    if (steps) fetch(one);
    for (; steps >= 2; steps -= 2) {
      fetch(two);
      absorb(one, Step());
      if (steps > 2) fetch(one);
      absorb(two, Step());
    }
    // what is left of a step, slot by slot, and a logit beside whole slots
    uint32_t rest = mine % U;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      two[u] = nothing<T>();
      if (u < rest) two[u] = p[u * threads];
    }
    if (on_edge) {
      uint4 beside = nothing<T>();
      *reinterpret_cast<T *>(&beside) = x[edge];
#pragma unroll
      for (int u = 0; u < U; ++u) if (u == rest) two[u] = beside;      // (U - 1 slots at most are left)
      ++rest;
    }
    if (steps) absorb(one, Step());
#pragma unroll 1
    for (; rest; --rest) {
      absorb(two, std::integral_constant<int, 1>());
#pragma unroll
      for (int u = 0; u + 1 < U; ++u) two[u] = two[u + 1];
    }
    Sums own = {m, 0.0f, 0.0f};
    own.sum = sum.x + sum.y; own.dot = dot.x + dot.y;
    const uint32_t order = order_of(own.m);
    // the block's sums
    auto warp_join = [&](Sums &v) {
      float m = v.m;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
      v.move(m, rate);
      v.sum = warp_sum_all(v.sum);
      if (ENTROPY) v.dot = warp_sum_all(v.dot);
    };
    warp_join(own);
    if (lane == 0) sums[warp] = own;
    __syncthreads();
    if (warp == 0) {
      own = lane < warps ? sums[lane] : Sums{-INFINITY, 0.0f, 0.0f};
      if (warps > 1) warp_join(own);
      if (lane == 0) block_sums = own;
    }
    if constexpr (TOP) {
      // the a.top-th of the maxima of groups of lanes, as many as leave half as many again: as many logits reach it at least
      uint32_t group = 32, least_order = 0;
      while (group > 1 && threads / group < a.top + a.top / 2 + 8) group /= 2;
      const uint32_t groups = threads / group;
      uint32_t of_group = order;
      for (uint32_t o = group / 2; o > 0; o >>= 1) of_group = max(of_group, __shfl_xor_sync(0xffffffffu, of_group, o));
      if ((threadIdx.x & (group - 1)) == 0) listed[threadIdx.x / group] = of_group;
      if (threadIdx.x == 0) bound_count = 0;
      __syncthreads();
      if (threadIdx.x < groups) {
        const uint32_t mine = listed[threadIdx.x];
        uint32_t before = 0;
#pragma unroll 8
        for (uint32_t j = 0; j < groups; ++j) before += listed[j] > mine || (listed[j] == mine && j < threadIdx.x);
        if (before == a.top - 1) bound_count = mine;
      }
      __syncthreads();
      least_order = bound_count;
      uint64_t least = least_order ? (uint64_t)least_order << 32 : 1;      // (no logit has the key 0)
      // lanes that read a thread's slots side by side
      const uint32_t each = (end - begin + threads - 1) / threads;
      uint32_t lanes = 1;
      while (lanes < 32 && lanes < each) lanes *= 2;
      // a key from `least` on, the at-th: beyond the buffer's size, one in `at`/size takes another's place, so that the buffer holds some of all alike
      auto put = [&](uint64_t key, uint32_t at) {
        const uint32_t place = at < kBuffer ? at : __umulhi(at * 2654435769u, at);
        if (place < kBuffer) buffer[place] = key;
      };
      // those of a slot (a warp's lanes have one each, or none)
      auto push_slot = [&](uint32_t slot, bool there) {
        const uint4 raw = there ? from[slot] : nothing<T>();
        Extremes<T> of;
        of.start(raw);
        of.template take<false>(raw, 1);
        const bool some = there && order_of(of.largest()) >= (uint32_t)(least >> 32);
        const uint32_t lanes_with = __ballot_sync(0xffffffffu, some);
        if (!lanes_with) return;
        float f[V];
        Vec<T>{raw}.floats(f);
        const uint32_t c = head + slot * V;
        if (__popc(lanes_with) <= 4) {   // few: each for itself
          if (some) {
#pragma unroll
            for (int i = 0; i < V; ++i) { const uint64_t key = key_of(f[i], c + i); if (key >= least) put(key, atomicAdd(&count, 1u)); }
          }
          return;
        }
        uint32_t mine = 0;
#pragma unroll
        for (int i = 0; i < V; ++i) mine += some && key_of(f[i], c + i) >= least;
        uint32_t at = mine;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) { const uint32_t w = __shfl_up_sync(0xffffffffu, at, o); if (lane >= o) at += w; }
        uint32_t start = 0;
        if (lane == 31) start = atomicAdd(&count, at);
        at += __shfl_sync(0xffffffffu, start, 31) - mine;
        if (!mine) return;
#pragma unroll
        for (int i = 0; i < V; ++i) { const uint64_t key = key_of(f[i], c + i); if (key >= least) put(key, at++); }
      };
      auto restart = [&] {
        __syncthreads();
        if (threadIdx.x == 0) count = bound_count = 0;
        __syncthreads();
      };
      // a better bound: a.top keys of the buffer's n reach it, or a few more (bit by bit; where all have the value of the bound that there is, by their indices alone)
      auto tighten = [&](uint32_t n) {
        bool other = false;
        for (uint32_t i = threadIdx.x; i < n; i += threads) other |= buffer[i] >> 32 != least >> 32;
        const bool values = __syncthreads_or(other);
        uint64_t to = values ? 0 : least >> 32 << 32;
        uint32_t reach = n;
        for (uint64_t bit = values ? 1ull << 63 : 1ull << 31; bit && reach > a.top + 32; bit >>= 1) {
          uint32_t now = 0;
          for (uint32_t i = 0; i < n; i += threads) now += __syncthreads_count(i + threadIdx.x < n && buffer[i + threadIdx.x] >= (to | bit));
          if (now >= a.top) { to |= bit; reach = now; }
        }
        if (to > least) least = to;
      };
      for (bool tried = false; ; ) {
        // the threads whose maxima reach the bound, and whether by more than its value
        restart();
        const uint32_t value = (uint32_t)(least >> 32), last = ~(uint32_t)least;
        if (order >= value) listed[atomicAdd(&bound_count, 1u)] = threadIdx.x | (order > value ? 1u << 31 : 0u);
        __syncthreads();
        const uint32_t found = bound_count;
        if (found > 2 * a.top + 64 && !tried) {
          // many threads with one value: since of equal ones the first count, a bound from the first slots
          tried = true;
          restart();
          push_slot(begin + threadIdx.x, begin + threadIdx.x < end);
          __syncthreads();
          const uint32_t had = count;
          if (had >= a.top) tighten(min(had, kBuffer));
          continue;
        }
        for (uint32_t q = warp * (32 / lanes); q < found; q += warps * (32 / lanes)) {
          const uint32_t which = q + lane / lanes, who = which < found ? listed[which] : 0, slot0 = begin + (who & ~(1u << 31));
          // (of a thread that has the value only, what lies up to the bound's index)
          auto there = [&](uint32_t j) { const uint32_t slot = slot0 + j * threads; return which < found && j < each && slot < end && (who >> 31 || head + slot * V <= last); };
          for (uint32_t j = lane & (lanes - 1); __any_sync(0xffffffffu, there(j)); j += lanes) push_slot(slot0 + j * threads, there(j));
        }
        if (on_edge) {
          const uint64_t key = key_of(to_float(x[edge]), edge);
          if (key >= least) put(key, atomicAdd(&count, 1u));
        }
        __syncthreads();
        if (count <= kBuffer) break;
        tighten(kBuffer);               // (too many)
      }
      const uint32_t n = count;
      for (uint32_t i = threadIdx.x; i < a.top; i += threads) best[i] = 0;
      __syncthreads();
      for (uint32_t i = threadIdx.x; i < n; i += threads) {
        const uint64_t key = buffer[i];
        uint32_t before = 0;
#pragma unroll 8
        for (uint32_t j = 0; j < n; ++j) before += buffer[j] > key;
        if (before < a.top) best[before] = key;
      }
    }
    sync();
    if (rank == 0) {
      // the cluster's
      if (warp == 0) {
        own = block_sums;
        if (cluster > 1) {
          own = Sums{-INFINITY, 0.0f, 0.0f};
          if (lane < cluster) {
            uint32_t w[3];
#pragma unroll
            for (int i = 0; i < 3; ++i) w[i] = peer_load(reinterpret_cast<const uint32_t *>(&block_sums) + i, lane);
            own = Sums{__uint_as_float(w[0]), __uint_as_float(w[1]), __uint_as_float(w[2])};
          }
          warp_join(own);
        }
      }
      const bool empty = own.m == -INFINITY;
      const float log_sum = empty ? 0.0f : logf(own.sum);
      if (first) {
        if (a.logprob) a.logprob[row] = token == a.vocab ? 0.0f : empty ? own.m : a.scale * (picked - own.m) - log_sum;
        if (ENTROPY && a.entropy) a.entropy[row] = empty ? 0.0f : log_sum - own.dot / own.sum * kLn2;
        if (a.stats) a.stats[row] = make_float2(own.m, log_sum);
      }
      if constexpr (TOP) {
        if (first) sums[0] = Sums{own.m, log_sum, 0.0f};
        const uint32_t all = cluster * a.top;
        for (uint32_t i = threadIdx.x; cluster > 1 && i < all; i += threads) {
          const uint32_t r = i / a.top;
          const uint32_t *p = reinterpret_cast<const uint32_t *>(best + (i - r * a.top));
          lists[i] = (uint64_t)peer_load(p + 1, r) << 32 | peer_load(p, r);
        }
        __syncthreads();
        const float m = sums[0].m, l = sums[0].sum;
        if (cluster == 1) { for (uint32_t i = threadIdx.x; i < a.top; i += threads) put_top(a, row, i, best[i], m, l); }      // (a row has that many)
        else for (uint32_t i = threadIdx.x; i < all; i += threads) {
          // the keys that are larger: all of a few are looked at side by side; of more, a list's come in falling order
          const uint64_t key = lists[i];
          uint32_t place = 0;
          if (all <= 256) {
#pragma unroll 8
            for (uint32_t j = 0; j < all; ++j) place += lists[j] > key;
          } else
            for (uint32_t r = 0; r < cluster; ++r) {
              uint32_t low = 0, high = a.top;
              while (low < high) { const uint32_t mid = (low + high) / 2; if (lists[r * a.top + mid] > key) low = mid + 1; else high = mid; }
              place += low;
            }
          if (key && place < a.top) put_top(a, row, place, key, m, l);
        }
      }
    }
    sync();
  }
}

// Any rows: a block has a row at a time, element by element
template <typename T> __global__ void __launch_bounds__(kThreads) token_log_probs_grad_rows_kernel(const ProbsGradArgs a)
{
  pdl_wait();
  for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T *x = static_cast<const T *>(a.logits) + row * a.stride;
    T *dx = static_cast<T *>(a.dlogits) + row * a.dstride;
    const float2 s = a.stats[row];
    const bool empty = s.x == -INFINITY;
    const uint32_t t = a.dlogprob ? token_at(a.token, a.token_bytes, row, a.vocab) : a.vocab;
    const float dl = t < a.vocab ? a.dlogprob[row] : 0.0f, dh = a.dentropy ? a.dentropy[row] : 0.0f, h = a.dentropy ? a.entropy[row] : 0.0f;
    for (uint32_t c = threadIdx.x; c < a.vocab; c += kThreads) {
      const float l = max_nan(a.scale * (to_float(x[c]) - s.x), kFloor) - s.y, p = expf(l);
      const float d = (c == t ? dl : 0.0f) - p * (dl + dh * (l + h));
      dx[c] = from_float<T>(empty ? 0.0f : a.scale * d);
    }
  }
}

// The gradient where logits and dlogits begin their rows at the same places of 16 bytes: a block has a stretch of a row and walks it in steps of four slots to a thread,
// the first of which is asked for before the row's numbers are; logits before the first slot and behind the last have a thread each.
// Stretches of up to four steps: the row's numbers, once for each, are many instructions ([1024,131072] bf16: 55 M warp instructions with one step, 45 M with four).
constexpr uint32_t kGradSlots = 4, kGradSteps = 4;
template <typename T, bool ENTROPY> __global__ void __launch_bounds__(kThreads, 6) token_log_probs_grad_kernel(const ProbsGradArgs a, const uint32_t cuts, const uint32_t stretch)
{
  constexpr int V = Vec<T>::V, U = kGradSlots;
  const uint32_t threads = blockDim.x;
  const float rate = fminf(a.scale * kLog2e, 3.402823466e38f);
  pdl_wait();
  pdl_trigger();
  for (uint64_t at = blockIdx.x; at < a.rows * cuts; at += gridDim.x) {
    const uint64_t row = at >> 32 ? at / cuts : (uint32_t)at / cuts;
    const uint32_t cut = (uint32_t)(at - row * cuts);
    const T *x = static_cast<const T *>(a.logits) + row * a.stride;
    T *dx = static_cast<T *>(a.dlogits) + row * a.dstride;
    const uint32_t head = min(a.vocab, (uint32_t)(-(int)((uintptr_t)x / sizeof(T)) & (V - 1))), slots = (a.vocab - head) / V, tail = a.vocab - head - slots * V;
    const uint32_t end = min(slots, (cut + 1) * stretch);
    const bool on_edge = cut == 0 && threadIdx.x < head + tail;
    const uint32_t edge = threadIdx.x < head ? threadIdx.x : a.vocab - tail + (threadIdx.x - head);
    uint32_t first = cut * stretch + threadIdx.x;
    Vec<T> v[U];
    auto fetch = [&] {
      const T *from = x + head + (uint64_t)first * V;
#pragma unroll
      for (int u = 0; u < U; ++u) if (first + u * threads < end) v[u] = Vec<T>::load(from + u * threads * V);
    };
    fetch();
    T one = {};
    if (on_edge) one = x[edge];
    const float2 stats = a.stats[row];
    const uint32_t token = a.dlogprob ? token_at(a.token, a.token_bytes, row, a.vocab) : a.vocab;
    const float dl = token < a.vocab ? a.dlogprob[row] : 0.0f, dh = ENTROPY ? a.dentropy[row] : 0.0f, h = ENTROPY ? a.entropy[row] : 0.0f;
    // with l = z - L in powers of two, dx = 2^l*(flat + slope*l), and scale*dlogprob more for the token
    const bool empty = stats.x == -INFINITY;
    const float log_sum = stats.y * kLog2e, flat = empty ? 0.0f : -a.scale * fmaf(dh, h, dl), slope = empty ? 0.0f : -a.scale * dh * kLn2, more = empty ? 0.0f : a.scale * dl;
    const float2 minus = both(empty ? 0.0f : -stats.x), times = both(rate), less = both(-log_sum), flat2 = both(flat), slope2 = both(slope);
    // (0 times -infinity is to be 0: CLAMP where some logit is that far below)
    auto gradient = [&](float2 f, auto clamp) {
      float2 l = fma2(add2(f, minus), times, less);
      if (decltype(clamp)::value) l = make_float2(max_nan(l.x, kFloor), max_nan(l.y, kFloor));
      const float2 p = make_float2(exp2_of(l.x), exp2_of(l.y));
      return mul2(p, ENTROPY ? fma2(slope2, l, flat2) : flat2);
    };
    auto slot = [&](int u, auto clamp) {
      const uint32_t c = head + (first + u * threads) * V;
      float2 f[V / 2];
      v[u].floats(reinterpret_cast<float *>(f));
#pragma unroll
      for (int i = 0; i < V / 2; ++i) f[i] = gradient(f[i], clamp);
      if (token - c < V) {
#pragma unroll
        for (int i = 0; i < V; ++i) if (token - c == i) reinterpret_cast<float *>(f)[i] += more;
      }
      Vec<T>::of(reinterpret_cast<const float *>(f)).store(dx + c);
    };
    while (first < end) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (first + u * threads >= end) continue;
        bool far = false;
        if (ENTROPY) {
          Extremes<T> low;
          low.start(v[u].bits);
          low.template take<true>(v[u].bits, 1);
          far = !(fmaf(low.smallest() + minus.x, rate, less.x) >= kFloor);
        }
        if (far) slot(u, std::true_type()); else slot(u, std::false_type());
      }
      first += U * threads;
      fetch();
    }
    if (on_edge) {
      const float d = gradient(both(to_float(one)), std::true_type()).x;
      dx[edge] = from_float<T>(edge == token ? d + more : d);
    }
  }
}

// Blocks to a row and threads of a block: by what a multiprocessor takes for its blocks, of its share of the bandwidth (44 KB/us) or in steps of four slots to a
// thread (0.8 us, of 1024 threads at a time), and what a row takes beside that: 3 us, in a cluster twice that, and the joins of its threads, 1 ns of each
void split(uint64_t rows, uint32_t slots, uint32_t top, uint32_t &cluster, uint32_t &threads)
{
  const uint64_t sms = sm_count();
  double least = 0.0;
  for (uint32_t c = 1; c <= 8 && (c == 1 || slots / c >= 256); c *= 2)
    for (uint32_t t = 128; t <= kMostThreads; t *= 2) {
      const uint64_t blocks = (rows * c + sms - 1) / sms, steps = ((uint64_t)slots + c * t * 4ull - 1) / (c * t * 4ull), room = 1024 / t;
      // (few threads are slower over long rows: [4096,131072] bf16 170 us with 128, 164 with 256; [4096,50021] 73 and 83)
      const double moved = (double)blocks * slots * 16 / c / 44e3 * (t == 128 && steps > 16 ? 1.04 : 1.0), waited = 0.8 * (double)(steps * ((blocks + room - 1) / room));
      const double cost = (moved > waited ? moved : waited) + (c > 1 ? 6.0 : 3.0) + 1e-3 * (double)(blocks * t);
      if (least == 0.0 || cost < least) { least = cost; cluster = c; threads = t; }
    }
  // short rows: four slots to a thread, one where there are few rows, and enough threads that their maxima bound the likeliest well
  const uint32_t part = slots / cluster + 1, most = (part + 31) / 32 * 32, enough = (2 * top + 31) / 32 * 32;
  uint32_t each = rows * cluster <= 2 * sms ? most : (part + 127) / 128 * 32;
  if (each < enough) each = enough < most ? enough : most;
  if (each < threads) threads = each < 32 ? 32 : each;
}

}  // namespace log_probs
}  // namespace rows
}  // namespace anode_b200

using namespace anode_b200::rows;
using namespace anode_b200::rows::log_probs;

static int check_logits(int type, uint64_t rows, uint32_t vocab, float scale)
{
  if (!known_type(type)) return ANODE_E_TYPE;
  if (!served(rows, vocab)) return ANODE_E_DIMS;
  return scale > 0.0f && scale <= 3.402823466e38f ? ANODE_OK : ANODE_E_VALUE;
}

extern "C" int anode_gpu_token_log_probs_fwd(
    int type, uint64_t rows, uint32_t vocab, float scale,
    const void *logits, uint64_t logits_stride, const void *token, int token_bytes,
    float *logprob, float *entropy, float *stats, uint32_t top, float *top_logprob, void *top_token, int top_token_bytes,
    const struct KernelConfig *cfg, struct CUstream_st *stream)
{
  (void)cfg;
  TRY(check_logits(type, rows, vocab, scale));
  if (top > kMostTop || top > vocab) return ANODE_E_DIMS;
  if (logprob && token_bytes != 4 && token_bytes != 8) return ANODE_E_TYPE;
  if (top && top_token && top_token_bytes != 4 && top_token_bytes != 8) return ANODE_E_TYPE;
  if (rows == 0) return ANODE_OK;
  TRY(check_rows(logits, type_bytes(type), rows, vocab, logits_stride, false));
  if ((logprob && !token) || (top && !top_logprob && !top_token) || !(logprob || entropy || stats || top)) return ANODE_E_NULL;
  if ((logprob && !aligned_to(token, (size_t)token_bytes)) || !aligned_to(logprob, 4) || !aligned_to(entropy, 4) || !aligned_to(stats, 8) ||
      (top && (!aligned_to(top_logprob, 4) || (top_token && !aligned_to(top_token, (size_t)top_token_bytes))))) return ANODE_E_ALIGN;
  // outputs apart from one another
  const struct { const void *p; uint64_t bytes; } outs[] = {{logprob, 4 * rows}, {entropy, 4 * rows}, {stats, 8 * rows}, {top ? top_logprob : nullptr, 4 * top * rows},
                                                            {top ? top_token : nullptr, (uint64_t)top_token_bytes * top * rows}};
  for (int i = 0; i < 5; ++i) for (int j = 0; j < i; ++j) if (overlap(outs[i].p, outs[i].bytes, outs[j].p, outs[j].bytes)) return ANODE_E_STRIDE;
  const ProbsArgs a = {rows, vocab, scale, logits, logits_stride, token, token_bytes, logprob, entropy, reinterpret_cast<float2 *>(stats), top,
                       top ? top_logprob : nullptr, top ? top_token : nullptr, top_token_bytes};
  const uint32_t v = (uint32_t)(16 / type_bytes(type)), slots = vocab / v;
  uint32_t cluster = 1, threads;
  split(rows, slots, top, cluster, threads);
  const uint64_t most = (1u << 30) / cluster;
  const dim3 grid((uint32_t)(rows < most ? rows : most) * cluster);
  return by_type(type, [&](auto t) {
    using T = decltype(t);
    auto kernel = top ? (entropy ? token_log_probs_kernel<T, true, true> : token_log_probs_kernel<T, false, true>)
                      : (entropy ? token_log_probs_kernel<T, true, false> : token_log_probs_kernel<T, false, false>);
    return cluster > 1 ? launch_in_clusters(kernel, grid, cluster, threads, (size_t)cluster * top * 8, stream, a, cluster) : launch(kernel, grid, threads, 0, stream, a, cluster);
  });
}

extern "C" int anode_gpu_token_log_probs_bwd(
    int type, uint64_t rows, uint32_t vocab, float scale,
    const void *logits, uint64_t logits_stride, const void *token, int token_bytes, const float *stats, const float *entropy,
    const float *dlogprob, const float *dentropy, void *dlogits, uint64_t dlogits_stride,
    const struct KernelConfig *cfg, struct CUstream_st *stream)
{
  (void)cfg;
  TRY(check_logits(type, rows, vocab, scale));
  if (dlogprob && token_bytes != 4 && token_bytes != 8) return ANODE_E_TYPE;
  if (rows == 0) return ANODE_OK;
  const size_t e = type_bytes(type);
  TRY(check_rows(logits, e, rows, vocab, logits_stride, false));
  TRY(check_rows(dlogits, e, rows, vocab, dlogits_stride, true));
  if (!stats || (dlogprob && !token) || (dentropy && !entropy) || !(dlogprob || dentropy)) return ANODE_E_NULL;
  if (!aligned_to(stats, 8) || !aligned_to(dlogprob, 4) || (dlogprob && !aligned_to(token, (size_t)token_bytes)) || !aligned_to(dentropy, 4) ||
      (dentropy && !aligned_to(entropy, 4))) return ANODE_E_ALIGN;
  if (!apart(dlogits, dlogits_stride, logits, logits_stride, rows)) return ANODE_E_STRIDE;
  const ProbsGradArgs a = {rows, vocab, scale, logits, logits_stride, token, token_bytes, reinterpret_cast<const float2 *>(stats), entropy, dlogprob, dentropy,
                           dlogits, dlogits_stride};
  const uint32_t v = (uint32_t)(16 / e), slots = vocab / v, each = (slots + 32 * kGradSlots - 1) / (32 * kGradSlots) * 32;
  const uint32_t threads = each < 32 ? 32 : each < kThreads ? each : kThreads, step_slots = threads * kGradSlots;
  // more steps to a block where the blocks of one step each would fill the device's places (six of a multiprocessor) four times, and the entropy's gradient is asked for,
  // whose numbers cost more ([4096,50021] bf16 128 us, 133 with one step).  Without it one step is better: 122.6 us, 126 with four, f32 [2048,65536] 156 and 163; only in
  // a loop of seconds, near the power cap, is it worse (130 and 127)
  const uint64_t blocks = rows * (slots / step_slots + 1), steps = !dentropy ? 1 : blocks / (24ull * anode_b200::sm_count());
  const uint32_t stretch = step_slots * (uint32_t)(steps < 1 ? 1 : steps < kGradSteps ? steps : kGradSteps), cuts = slots ? (slots + stretch - 1) / stretch : 1;
  const bool step = in_step(dlogits, e, dlogits_stride, v, logits, e, logits_stride, rows);
  return by_type(type, [&](auto t) {
    using T = decltype(t);
    return step ? launch(dentropy ? token_log_probs_grad_kernel<T, true> : token_log_probs_grad_kernel<T, false>, dim3(row_blocks(rows * cuts)), threads, 0, stream, a, cuts, stretch)
                : launch(token_log_probs_grad_rows_kernel<T>, dim3(row_blocks(rows)), kThreads, 0, stream, a);
  });
}
