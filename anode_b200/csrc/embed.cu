// Rows of a table by tokens, and the table's gradient.
//
//   y[i] = scale*table[token[i]],   dtable[v] = scale * sum of dy[i] over token[i] = v
//
// A token outside of the table has a row of zeros and no gradient.  Sums are f32, in an order that follows from the tokens alone.
//
// The gradient in three launches:
//   1. one cluster sorts (token, place) by tokens, a stable radix sort, while the others write zeros to the rows that no token names;
//   2. the sorted places are cut into pieces, and a thread per 16 bytes of columns walks down a piece's rows of dy: it writes the sum where a token's run
//      of places ends.  A run of up to kLong places belongs to the piece where it begins; of a longer one each piece leaves its part in the workspace;
//   3. the parts of each long run are joined, in order.
// All but the sort is bound by memory.
#include "bn_host.h"
#include "rows.cuh"

namespace anode_b200 {
namespace rows {

constexpr uint32_t kThreads = 256;

// N elements side by side
template <typename T, int N> struct Unit {
  static constexpr int BYTES = N * (int)sizeof(T);
  typedef typename std::conditional<BYTES == 16, uint4, typename std::conditional<BYTES == 8, uint2, typename std::conditional<BYTES == 4, uint32_t, uint16_t>::type>::type>::type Word;
  Word w;
  __device__ __forceinline__ static Unit load(const T *p) { return Unit{*reinterpret_cast<const Word *>(p)}; }
  __device__ __forceinline__ void store(T *p) const { *reinterpret_cast<Word *>(p) = w; }
  __device__ __forceinline__ void floats(float *f) const
  {
    if constexpr (BYTES == 16) Vec<T>{w}.floats(f);
    else {
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = to_float(reinterpret_cast<const T *>(&w)[i]);
    }
  }
  __device__ __forceinline__ static Unit of(const float *f)
  {
    Unit u;
    if constexpr (BYTES == 16) u.w = Vec<T>::of(f).bits;
    else {
#pragma unroll
      for (int i = 0; i < N; ++i) reinterpret_cast<T *>(&u.w)[i] = from_float<T>(f[i]);
    }
    return u;
  }
};
// N floats of an array of T: in one piece, or two where they are more than 16 bytes
template <typename T, int N> __device__ __forceinline__ void put_floats(T *p, const float *f)
{
  constexpr int M = N * (int)sizeof(T) > 16 ? 16 / (int)sizeof(T) : N;
#pragma unroll
  for (int i = 0; i < N; i += M) Unit<T, M>::of(f + i).store(p + i);
}
template <typename T, int N> __device__ __forceinline__ void get_floats(const T *p, float *f)
{
  constexpr int M = N * (int)sizeof(T) > 16 ? 16 / (int)sizeof(T) : N;
#pragma unroll
  for (int i = 0; i < N; i += M) Unit<T, M>::load(p + i).floats(f + i);
}

struct EmbedArgs {
  uint64_t tokens;
  uint32_t vocab, cols;
  float scale;
  const void *token;
  int token_bytes;
  const void *table;
  uint64_t table_stride;
  void *y;
  uint64_t y_stride;
};

// A team of lanes (a power of two, up to a warp) has a token and M units of E columns per lane; the grid's second dimension has the rest of wide rows
template <typename T, int E, int M> __global__ void __launch_bounds__(128) embed_kernel(const EmbedArgs a, const uint32_t team)
{
  const uint64_t i = ((uint64_t)blockIdx.x * 128 + threadIdx.x) / team;
  const uint32_t lane = threadIdx.x & (team - 1), units = a.cols / E;
  pdl_wait();
  pdl_trigger();
  if (i >= a.tokens) return;
  const uint32_t t = token_at(a.token, a.token_bytes, i, a.vocab);
  const T *in = static_cast<const T *>(a.table) + t * a.table_stride;
  T *y = static_cast<T *>(a.y) + i * a.y_stride;
  for (uint32_t first = blockIdx.y * team * M + lane; first < units; first += gridDim.y * team * M) {
    Unit<T, E> v[M];
#pragma unroll
    for (int k = 0; k < M; ++k)
      if (t < a.vocab && first + k * team < units) v[k] = Unit<T, E>::load(in + (uint64_t)(first + k * team) * E);
#pragma unroll
    for (int k = 0; k < M; ++k) {
      if (first + k * team >= units) continue;
      float f[E];
      v[k].floats(f);
#pragma unroll
      for (int j = 0; j < E; ++j) f[j] = t < a.vocab ? f[j] * a.scale : 0.0f;
      Unit<T, E>::of(f).store(y + (uint64_t)(first + k * team) * E);
    }
  }
}

// ---- the gradient ---------------------------------------------------------------------------------------------------------------

constexpr uint32_t kCluster = 8, kSortThreads = 512, kSortWarps = kSortThreads / 32;
constexpr uint32_t kMostBits = 9;                    // of a token to a pass of the sort
constexpr uint32_t kRowsAtOnce = 65536;              // of the table, whose bits a block has
constexpr uint32_t kLong = 32;                       // places of a run that one piece adds up
constexpr uint32_t kMostPiece = 32;                  // places of a piece
constexpr uint32_t kLeastLanes = 4;                  // threads of a piece

struct SortArgs {
  uint32_t n, vocab;
  const void *token;
  int token_bytes;
  uint32_t bits, passes;
  uint32_t *key[2], *place[2];          // the last pass writes the first of each
  // rows of zeros
  void *dtable;
  uint64_t stride;                      // in units
  uint32_t units, rows;                 // units of a row, rows of a block at a time
};

// The first cluster: passes of a radix sort, each over `bits` of the tokens.  A warp has a stretch of the places.  It counts its digits (lanes with the same
// one find each other, and the first adds for all, so that the order stays); the counts of all warps and blocks before it and of smaller digits
// are where its own begin.
__device__ __forceinline__ void sort_tokens(const SortArgs &a, uint32_t (*count)[1u << kMostBits], uint32_t *totals, uint32_t *base)
{
  constexpr uint32_t STEPS = 4;
  const uint32_t rank = cluster_rank(), warp = threadIdx.x >> 5, lane = threadIdx.x & 31, bins = 1u << a.bits;
  const uint32_t stretch = (a.n + kCluster * kSortWarps * 32 - 1) / (kCluster * kSortWarps * 32) * 32;
  const uint64_t lo = (uint64_t)(rank * kSortWarps + warp) * stretch, hi = min((uint64_t)a.n, lo + stretch);
  uint32_t *mine = count[warp];
  for (uint32_t pass = 0; pass < a.passes; ++pass) {
    const bool last = (a.passes - 1 - pass) % 2 == 0;      // (or another that writes the first pair of arrays)
    const uint32_t shift = pass * a.bits;
    uint32_t *const key_to = last ? a.key[0] : a.key[1], *const place_to = last ? a.place[0] : a.place[1];
    const uint32_t *const key_from = last ? a.key[1] : a.key[0], *const place_from = last ? a.place[1] : a.place[0];
    uint32_t key[STEPS], place[STEPS];
    auto fetch = [&](uint64_t from) {
#pragma unroll
      for (uint32_t s = 0; s < STEPS; ++s) {
        const uint64_t i = from + 32 * s + lane;
        if (i >= hi) continue;
        key[s] = pass == 0 ? token_at(a.token, a.token_bytes, i, a.vocab) : __ldcg(key_from + i);
        place[s] = pass == 0 ? (uint32_t)i : __ldcg(place_from + i);
      }
    };
    // the lanes that have this one's digit; lanes beyond the stretch have each other
    auto peers = [&](uint64_t from, uint32_t s, uint32_t &digit) {
      digit = from + 32 * s + lane < hi ? key[s] >> shift & (bins - 1) : bins;
      return __match_any_sync(0xffffffffu, digit);
    };
    for (uint32_t i = lane; i < bins; i += 32) mine[i] = 0;
    __syncwarp();
    for (uint64_t from = lo; from < hi; from += 32 * STEPS) {
      fetch(from);
#pragma unroll
      for (uint32_t s = 0; s < STEPS; ++s) {
        uint32_t digit;
        const uint32_t same = peers(from, s, digit);
        if (digit < bins && lane == (uint32_t)__ffs((int)same) - 1) mine[digit] += __popc(same);
        __syncwarp();
      }
    }
    __syncthreads();
    const uint32_t t = threadIdx.x;
    if (t < bins) {
      uint32_t sum = 0, c[kSortWarps];
#pragma unroll
      for (uint32_t w = 0; w < kSortWarps; ++w) c[w] = count[w][t];
#pragma unroll
      for (uint32_t w = 0; w < kSortWarps; ++w) { count[w][t] = sum; sum += c[w]; }
      totals[t] = sum;
    }
    cluster_sync();
    uint32_t before = 0, all = 0;
    if (t < bins) {
      uint32_t c[kCluster];
#pragma unroll
      for (uint32_t r = 0; r < kCluster; ++r) c[r] = peer_load(totals + t, r);
#pragma unroll
      for (uint32_t r = 0; r < kCluster; ++r) { before += r < rank ? c[r] : 0; all += c[r]; }
    }
    uint32_t sum = all;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) { const uint32_t v = __shfl_up_sync(0xffffffffu, sum, o); if (lane >= o) sum += v; }
    if (lane == 31) base[kSortThreads + warp] = sum;
    __syncthreads();
    uint32_t less = 0;
    for (uint32_t w = 0; w < warp; ++w) less += base[kSortThreads + w];
    if (t < bins) base[t] = less + sum - all + before;
    __syncthreads();
    for (uint32_t i = lane; i < bins; i += 32) mine[i] += base[i];
    __syncwarp();
    for (uint64_t from = lo; from < hi; from += 32 * STEPS) {
      if (stretch > 32 * STEPS) fetch(from);
#pragma unroll
      for (uint32_t s = 0; s < STEPS; ++s) {
        uint32_t digit;
        const uint32_t same = peers(from, s, digit), first = (uint32_t)__ffs((int)same) - 1;
        uint32_t at = 0;
        if (digit < bins && lane == first) { at = mine[digit]; mine[digit] = at + __popc(same); }
        at = __shfl_sync(0xffffffffu, at, first) + __popc(same & ((1u << lane) - 1));
        if (digit < bins) { key_to[at] = key[s]; place_to[at] = place[s]; }
        __syncwarp();
      }
    }
    cluster_sync();
  }
}

// The other clusters: each block has rows of the table, and its cluster's blocks look through the tokens together for those that are named
template <typename W> __device__ __forceinline__ void zero_rows(const SortArgs &a, uint32_t *named)
{
  const uint32_t rank = cluster_rank(), clusters = gridDim.x / kCluster - 1, first = blockIdx.x / kCluster - 1, each = kCluster * a.rows;
  uint32_t team = 1;
  while (team < 32 && team < a.units) team *= 2;
  const uint32_t lane = threadIdx.x & (team - 1);
  for (uint64_t begin = (uint64_t)first * each; begin < a.vocab; begin += (uint64_t)clusters * each) {
    for (uint32_t i = threadIdx.x; i < (a.rows + 31) / 32; i += kSortThreads) named[i] = 0;
    cluster_sync();
    for (uint64_t i = rank * kSortThreads + threadIdx.x; i < a.n; i += kCluster * kSortThreads) {
      const uint64_t t = token_at(a.token, a.token_bytes, i, a.vocab);
      if (t < begin || t >= begin + each || t >= a.vocab) continue;
      const uint32_t of = (uint32_t)(t - begin) / a.rows, row = (uint32_t)(t - begin) - of * a.rows;
      asm volatile("red.relaxed.cluster.shared::cluster.or.b32 [%0], %1;" ::"r"(peer_address(named + row / 32, of)), "r"(1u << (row & 31)) : "memory");
    }
    cluster_sync();
    const uint64_t mine = begin + (uint64_t)rank * a.rows;
    for (uint32_t row = threadIdx.x / team; row < a.rows && mine + row < a.vocab; row += kSortThreads / team) {
      if (named[row / 32] >> (row & 31) & 1) continue;
      W *to = static_cast<W *>(a.dtable) + (mine + row) * a.stride;
      for (uint32_t u = lane; u < a.units; u += team) to[u] = W{};
    }
    __syncthreads();
  }
}

template <typename W> __global__ void __launch_bounds__(kSortThreads) embed_sort_kernel(const SortArgs a)
{
  __shared__ uint32_t count[kSortWarps][1u << kMostBits], totals[1u << kMostBits], base[kSortThreads + kSortWarps];
  static_assert(sizeof(count) >= kRowsAtOnce / 8 && kSortThreads >= 1u << kMostBits, "a bit per row, a thread per digit");
  pdl_wait();
  pdl_trigger();
  if (blockIdx.x < kCluster) { if (a.n) sort_tokens(a, count, totals, base); }
  else zero_rows<W>(a, count[0]);
}

struct SumArgs {
  uint32_t n, vocab, cols;
  float scale;
  const uint32_t *key, *place;          // sorted
  const void *dy;
  uint64_t dy_stride;
  void *dtable;
  uint64_t stride;
  uint32_t piece, pieces;
  uint32_t *begins;                     // of each piece: whether a long run begins in it
  float *part;                          // [pieces][2][part_cols]: of a long run that begins before the piece, and of one that begins in it
  uint32_t part_cols;
  uint32_t lanes;                       // threads of a piece
};

// What a piece adds up: places [from, to), of which the runs of `head` and `tail` are long (else they are ~0)
struct Piece { uint32_t from, to, head, tail; bool head_before; };

// M units of E columns per thread; a block has kThreads/lanes pieces side by side.  All rows of a step are asked for before one is used, whatever runs they
// belong to, and with them what the table holds where a run ends (ACC).
template <typename T, typename O, int E, int M, int STEP, bool ACC>
__global__ void __launch_bounds__(kThreads) embed_sums_kernel(const SumArgs a)
{
  constexpr uint32_t PIECES = kThreads / kLeastLanes;
  __shared__ uint32_t key[PIECES * kMostPiece + 2 * kLong], place[PIECES * kMostPiece + 2 * kLong];
  __shared__ Piece piece[PIECES];
  pdl_wait();
  pdl_trigger();
  const uint32_t per_block = kThreads / a.lanes, first = blockIdx.x * per_block, lane = threadIdx.x & 31;
  // the places of the block's pieces and kLong on either side; what is no token ends the sorted ones
  const int64_t begin = (int64_t)first * a.piece - kLong;
  for (uint32_t i = threadIdx.x; i < per_block * a.piece + 2 * kLong; i += kThreads) {
    const int64_t at = begin + i;
    const bool inside = at >= 0 && at < a.n;
    key[i] = inside ? a.key[at] : ~0u;
    place[i] = inside ? a.place[at] : 0;
  }
  __syncthreads();
  // a warp looks at a piece: how far the runs of its first and last token go, up to kLong places
  for (uint32_t p = threadIdx.x >> 5; p < per_block; p += kThreads / 32) {
    const uint32_t at = kLong + p * a.piece, size = min(a.piece, a.n - min(a.n, (first + p) * a.piece)), last = at + size - 1;
    auto run = [&](uint32_t k, uint32_t from, int step) {        // places from `from` on, in steps, that have token k
      const uint32_t other = ~__ballot_sync(0xffffffffu, key[(int)from + step * (int)lane] == k);
      return other ? (uint32_t)__ffs((int)other) - 1 : 32u;
    };
    Piece q = {at, at, ~0u, ~0u, false};
    if (size && key[at] < a.vocab) {
      const uint32_t k0 = key[at], before = run(k0, at - 1, -1), after = run(k0, at + 1, 1);
      const bool long0 = before + 1 + after > kLong;
      const uint32_t k1 = key[last], ahead = run(k1, last - 1, -1), behind = run(k1, last + 1, 1);
      const bool long1 = k1 < a.vocab && ahead + 1 + behind > kLong, whole = k0 == k1;
      q.head_before = before > 0;
      if (before && !long0) q.from = at + 1 + after;             // (that run is an earlier piece's)
      if (long0) q.head = k0;
      if (long1) q.tail = k1;
      q.to = long1 || k1 >= a.vocab ? last + 1 : last + 1 + behind;
      if (q.from > q.to || (whole && before && !long0)) q.to = q.from;
    }
    if (lane == 0) {
      piece[p] = q;
      if (first + p < a.pieces && blockIdx.y == 0) a.begins[first + p] = q.tail != ~0u && !(q.tail == q.head && q.head_before);
    }
  }
  __syncthreads();
  const uint32_t mine = threadIdx.x / a.lanes;
  const Piece q = piece[mine];
  const uint64_t unit = (uint64_t)blockIdx.y * a.lanes * M + (threadIdx.x & (a.lanes - 1));
  const T *dy = static_cast<const T *>(a.dy) + unit * E;
  O *out = static_cast<O *>(a.dtable) + unit * E;
  float *part = a.part + ((uint64_t)(first + mine) * 2 * a.part_cols) + unit * E;
  bool has[M];
#pragma unroll
  for (int m = 0; m < M; ++m) has[m] = (unit + (uint64_t)m * a.lanes) * E < a.cols;
  float sum[M][E];
#pragma unroll
  for (int m = 0; m < M; ++m)
#pragma unroll
    for (int j = 0; j < E; ++j) sum[m][j] = 0.0f;
  for (uint32_t i = q.from; i < q.to; i += STEP) {
    Unit<T, E> v[STEP][M];
    float old[ACC ? STEP : 1][M][E];
    uint32_t k[STEP + 1];
#pragma unroll
    for (int s = 0; s <= STEP; ++s) { k[s] = i + s < q.to ? key[i + s] : ~0u; if (k[s] >= a.vocab) k[s] = ~0u; }
#pragma unroll
    for (int s = 0; s < STEP; ++s) {
      if (k[s] == ~0u) continue;
      const T *row = dy + place[i + s] * a.dy_stride;
#pragma unroll
      for (int m = 0; m < M; ++m) if (has[m]) v[s][m] = Unit<T, E>::load(row + (uint64_t)m * a.lanes * E);
    }
    if constexpr (ACC) {
#pragma unroll
      for (int s = 0; s < STEP; ++s) {
        if (k[s] == k[s + 1] || k[s] == ~0u) continue;
#pragma unroll
        for (int m = 0; m < M; ++m) if (has[m]) get_floats<O, E>(out + k[s] * a.stride + (uint64_t)m * a.lanes * E, old[s][m]);
      }
    }
#pragma unroll
    for (int s = 0; s < STEP; ++s) {
      if (k[s] == ~0u) continue;
#pragma unroll
      for (int m = 0; m < M; ++m) {
        float f[E];
        v[s][m].floats(f);
#pragma unroll
        for (int j = 0; j < E; ++j) sum[m][j] += f[j];
      }
      if (k[s] == k[s + 1]) continue;
      // the run's end, or that of the piece's part of a long one
      const bool is_long = k[s] == q.head || k[s] == q.tail;
      float *to = part + (k[s] == q.head && q.head_before ? 0 : a.part_cols);
#pragma unroll
      for (int m = 0; m < M; ++m) {
        if (has[m] && is_long) {
#pragma unroll
          for (int j = 0; j < E; ++j) to[(uint64_t)m * a.lanes * E + j] = sum[m][j];
        } else if (has[m]) {
#pragma unroll
          for (int j = 0; j < E; ++j) sum[m][j] = ACC ? fmaf(sum[m][j], a.scale, old[ACC ? s : 0][m][j]) : sum[m][j] * a.scale;
          put_floats<O, E>(out + k[s] * a.stride + (uint64_t)m * a.lanes * E, sum[m]);
        }
#pragma unroll
        for (int j = 0; j < E; ++j) sum[m][j] = 0.0f;
      }
    }
  }
}

// The parts of long runs: a block has 128 columns and every gridDim.y-th piece that such a run begins in; a warp adds an eighth of the run's parts, in order
template <typename O> __global__ void __launch_bounds__(kThreads) embed_join_kernel(const SumArgs a, const int accumulate)
{
  __shared__ float sums[kThreads / 32][4][32];
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint64_t c = ((uint64_t)blockIdx.x * 32 + lane) * 4;
  pdl_wait();
  for (uint32_t group = blockIdx.y * kThreads; group < a.pieces; group += gridDim.y * kThreads)
    for (uint32_t p = group; p < min(a.pieces, group + kThreads); ++p) {
      // the next piece with such a run
      const uint32_t look = p + threadIdx.x;
      const bool here = look < min(a.pieces, group + kThreads) && a.begins[look];
      __shared__ uint32_t next, end;
      __syncthreads();
      if (threadIdx.x == 0) { next = ~0u; end = ~0u; }
      __syncthreads();
      if (here) atomicMin(&next, look);
      __syncthreads();
      p = next;
      if (p == ~0u) break;
      // the pieces behind it that the run fills, and one that it ends in
      const uint32_t k = a.key[(uint64_t)p * a.piece + a.piece - 1];
      for (uint32_t from = p + 1; end == ~0u; from += kThreads) {
        const uint32_t r = from + threadIdx.x;
        const uint64_t last = (uint64_t)r * a.piece + a.piece - 1;
        __syncthreads();
        if (last >= a.n || a.key[last] != k) atomicMin(&end, r);
        __syncthreads();
      }
      const uint32_t filled = end;
      const uint32_t stop = filled < a.pieces && a.key[(uint64_t)filled * a.piece] == k ? filled + 1 : filled;
      const uint32_t parts = stop - p, each = (parts + kThreads / 32 - 1) / (kThreads / 32), lo = min(parts, warp * each), hi = min(parts, lo + each);
      float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (c < a.cols) {
#pragma unroll 8
        for (uint32_t i = lo; i < hi; ++i) {
          const float4 v = *reinterpret_cast<const float4 *>(a.part + ((uint64_t)(p + i) * 2 + (i == 0)) * a.part_cols + c);
          sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
        }
      }
      sums[warp][0][lane] = sum.x; sums[warp][1][lane] = sum.y; sums[warp][2][lane] = sum.z; sums[warp][3][lane] = sum.w;
      __syncthreads();
      if (warp < 4 && c + warp < a.cols) {
        float all = 0.0f;
#pragma unroll
        for (uint32_t w = 0; w < kThreads / 32; ++w) all += sums[w][warp][lane];
        O *to = static_cast<O *>(a.dtable) + k * a.stride + c + warp;
        *to = from_float<O>(accumulate ? fmaf(all, a.scale, to_float(*to)) : all * a.scale);
      }
    }
}

inline int check_tokens(const void *token, int bytes)
{
  if (bytes != 4 && bytes != 8) return ANODE_E_TYPE;
  if (!token) return ANODE_E_NULL;
  return aligned_to(token, (size_t)bytes) ? ANODE_OK : ANODE_E_ALIGN;
}

// Columns to a unit that both arrays' rows allow: as many as 16 bytes of the narrower type hold, two, or one
inline uint32_t unit_of(const void *p, size_t bytes, uint64_t stride, uint64_t rows, const void *q, size_t q_bytes, uint64_t q_stride, uint64_t q_rows, uint32_t cols)
{
  auto fits = [&](const void *x, size_t e, uint64_t s, uint64_t n, uint32_t width) {
    const size_t most = width * e < 16 ? width * e : 16;
    return aligned_to(x, most) && (n <= 1 || s * e % most == 0);
  };
  const size_t least = bytes < q_bytes ? bytes : q_bytes;
  for (uint32_t width : {(uint32_t)(16 / least), 2u})
    if (cols % width == 0 && fits(p, bytes, stride, rows, width) && fits(q, q_bytes, q_stride, q_rows, width)) return width;
  return 1;
}
inline uint32_t power_up_to(uint64_t n, uint32_t most)
{
  uint32_t v = 1;
  while (v < most && v < n) v *= 2;
  return v;
}

// Places of a piece: few where there are few, so that more threads have some
inline uint32_t piece_of(uint64_t tokens) { return tokens >= 8192 ? 32 : tokens >= 4096 ? 16 : tokens >= 1024 ? 8 : 4; }

// Where the workspace's arrays begin
struct Layout {
  uint64_t n, piece, pieces, part_cols, begins, part, bytes;
  Layout(uint64_t tokens, uint32_t cols) : n((tokens + 3) / 4 * 4), piece(piece_of(tokens)), pieces((tokens + piece - 1) / piece), part_cols(((uint64_t)cols + 3) / 4 * 4)
  {
    begins = 16 * n;
    part = begins + (pieces + 3) / 4 * 16;
    bytes = part + pieces * 2 * part_cols * 4;
  }
};

template <typename T, typename O, int E> int launch_sums(SumArgs a, int accumulate, cudaStream_t stream)
{
  constexpr int M = E * sizeof(T) == 16 ? 1 : 4;
  const uint32_t units = a.cols / E;
  a.lanes = power_up_to((units + M - 1) / M, kThreads);
  if (a.lanes < kLeastLanes) a.lanes = kLeastLanes;
  const uint32_t per_block = kThreads / a.lanes, wide = (units + a.lanes * M - 1) / (a.lanes * M);
  const dim3 grid((a.pieces + per_block - 1) / per_block, wide);
  return accumulate ? launch(embed_sums_kernel<T, O, E, M, M == 1 ? 4 : 2, true>, grid, kThreads, 0, stream, a)
                    : launch(embed_sums_kernel<T, O, E, M, M == 1 ? 8 : 4, false>, grid, kThreads, 0, stream, a);
}
template <typename T, typename O> int launch_sums(const SumArgs &a, uint32_t unit, int accumulate, cudaStream_t stream)
{
  constexpr int V = 16 / sizeof(T);
  TRY((unit == (uint32_t)V ? launch_sums<T, O, V>(a, accumulate, stream) : unit == 2 ? launch_sums<T, O, 2>(a, accumulate, stream)
                                                                                      : launch_sums<T, O, 1>(a, accumulate, stream)));
  // a run is long beyond kLong places
  if (a.n <= kLong) return ANODE_OK;
  const uint32_t groups = (a.pieces + kThreads - 1) / kThreads;
  return launch(embed_join_kernel<O>, dim3((uint32_t)(((uint64_t)a.cols + 127) / 128), groups < 16 ? groups : 16), kThreads, 0, stream, a, accumulate);
}

}  // namespace rows
}  // namespace anode_b200

using namespace anode_b200::rows;

extern "C" int anode_gpu_embed_tokens_fwd(
    int type, uint64_t tokens, uint32_t vocab, uint32_t cols, float scale,
    const void *token, int token_bytes, const void *table, uint64_t table_stride, void *y, uint64_t y_stride,
    const struct KernelConfig *cfg, struct CUstream_st *stream)
{
  (void)cfg;
  if (!known_type(type)) return ANODE_E_TYPE;
  if (!served(0, cols) || !served(0, vocab) || tokens >> 31) return ANODE_E_DIMS;
  if (tokens == 0) return ANODE_OK;
  const size_t e = type_bytes(type);
  TRY(check_tokens(token, token_bytes));
  TRY(check_rows(table, e, vocab, cols, table_stride, false));
  TRY(check_rows(y, e, tokens, cols, y_stride, true));
  if (y == table) return ANODE_E_STRIDE;
  const EmbedArgs a = {tokens, vocab, cols, scale, token, token_bytes, table, table_stride, y, y_stride};
  const uint32_t unit = unit_of(table, e, table_stride, vocab, y, e, y_stride, tokens, cols);
  return by_type(type, [&](auto t) {
    using T = decltype(t);
    constexpr uint32_t V = 16 / sizeof(T);
    const uint32_t units = cols / unit, each = unit == V ? 4 : 8, team = power_up_to((units + each - 1) / each, 32);
    const uint64_t wide = ((uint64_t)units + team * each - 1) / (team * each);
    const dim3 grid((uint32_t)((tokens * team + 127) / 128), (uint32_t)(wide < 65535 ? wide : 65535));
    return unit == V ? launch(embed_kernel<T, (int)V, 4>, grid, 128, 0, stream, a, team)
         : unit == 2 ? launch(embed_kernel<T, 2, 8>, grid, 128, 0, stream, a, team) : launch(embed_kernel<T, 1, 8>, grid, 128, 0, stream, a, team);
  });
}

extern "C" size_t anode_gpu_embed_tokens_bwd_workspace_bytes(uint64_t tokens, uint32_t vocab, uint32_t cols)
{
  (void)vocab;
  return (size_t)Layout(tokens, cols).bytes;
}

extern "C" int anode_gpu_embed_tokens_bwd(
    int type, uint64_t tokens, uint32_t vocab, uint32_t cols, float scale,
    const void *token, int token_bytes, const void *dy, uint64_t dy_stride, void *dtable, uint64_t dtable_stride, int dtable_type, int accumulate,
    void *workspace, size_t workspace_bytes,
    const struct KernelConfig *cfg, struct CUstream_st *stream)
{
  (void)cfg;
  if (!known_type(type) || (dtable_type != type && dtable_type != ANODE_TYPE_F32)) return ANODE_E_TYPE;
  if (!served(0, cols) || !served(0, vocab) || tokens >> 31) return ANODE_E_DIMS;
  if (tokens == 0 && accumulate) return ANODE_OK;
  const size_t e = type_bytes(type), oe = type_bytes(dtable_type);
  TRY(check_rows(dtable, oe, vocab, cols, dtable_stride, true));
  if (tokens) {
    TRY(check_tokens(token, token_bytes));
    TRY(check_rows(dy, e, tokens, cols, dy_stride, false));
    if (dy == dtable) return ANODE_E_STRIDE;
    if (!workspace || !aligned_to(workspace, 16) || workspace_bytes < anode_gpu_embed_tokens_bwd_workspace_bytes(tokens, vocab, cols)) return ANODE_E_WORKSPACE;
  }
  const Layout l(tokens, cols);
  uint32_t *words = static_cast<uint32_t *>(workspace);
  SortArgs s = {(uint32_t)tokens, vocab, token, token_bytes, 0, 0, {words, words + l.n}, {words + 2 * l.n, words + 3 * l.n}, dtable, 0, 0, 0};
  // tokens up to `vocab`, which stands for none
  uint32_t bits = 0;
  while (vocab >> bits) ++bits;
  s.passes = (bits + kMostBits - 1) / kMostBits;
  s.bits = (bits + s.passes - 1) / s.passes;
  // rows of zeros in units of 16 bytes, or as many as their columns and places allow
  uint32_t bytes = 16;
  while ((uint64_t)cols * oe % bytes || (uint64_t)dtable_stride * oe % bytes || !aligned_to(dtable, bytes)) bytes /= 2;
  s.units = (uint32_t)((uint64_t)cols * oe / bytes);
  s.stride = dtable_stride * oe / bytes;
  uint32_t clusters = 0;
  if (!accumulate) {
    const uint64_t work = ((uint64_t)vocab * cols * oe + (kCluster << 15) - 1) / (kCluster << 15);      // 32 KB for a block
    clusters = (uint32_t)(work < 24 ? work : 24);
    const uint64_t rows = ((uint64_t)vocab + clusters * kCluster - 1) / (clusters * kCluster);
    s.rows = (uint32_t)(rows < kRowsAtOnce ? rows : kRowsAtOnce);
  }
  const dim3 grid((clusters + 1) * kCluster);
  TRY(bytes == 16 ? launch_in_clusters(embed_sort_kernel<uint4>, grid, kCluster, kSortThreads, 0, stream, s)
    : bytes == 8 ? launch_in_clusters(embed_sort_kernel<uint2>, grid, kCluster, kSortThreads, 0, stream, s)
    : bytes == 4 ? launch_in_clusters(embed_sort_kernel<uint32_t>, grid, kCluster, kSortThreads, 0, stream, s)
                 : launch_in_clusters(embed_sort_kernel<uint16_t>, grid, kCluster, kSortThreads, 0, stream, s));
  if (!tokens) return ANODE_OK;
  const SumArgs a = {(uint32_t)tokens, vocab, cols, scale, s.key[0], s.place[0], dy, dy_stride, dtable, dtable_stride, (uint32_t)l.piece, (uint32_t)l.pieces,
                     words + l.begins / 4, reinterpret_cast<float *>(static_cast<char *>(workspace) + l.part), (uint32_t)l.part_cols, 0};
  const uint32_t unit = unit_of(dy, e, dy_stride, tokens, dtable, oe, dtable_stride, vocab, cols);
  return by_type(type, [&](auto t) {
    using T = decltype(t);
    if constexpr (sizeof(T) == 2) { if (dtable_type != ANODE_TYPE_F32) return launch_sums<T, T>(a, unit, accumulate, stream); }
    return launch_sums<T, float>(a, unit, accumulate, stream);
  });
}
