// Rows of a table by tokens, and the table's gradient.
//
//   y[i] = scale*table[token[i]],   dtable[v] = scale * sum of dy[i] over token[i] = v
//
// A token outside of the table has a row of zeros and no gradient.  Sums are f32, in an order that follows from the tokens alone.
//
// The gradient in three launches:
//   1. (token, place) are sorted by tokens, and equal ones by places, while other blocks write zeros to the whole table: few by counting for each how many come
//      before it, more by a radix sort in one cluster;
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
// N elements as they lie in memory, in one piece or two
template <typename T, int N> struct Held {
  static constexpr int M = N * (int)sizeof(T) > 16 ? 16 / (int)sizeof(T) : N;
  Unit<T, M> part[N / M];
  __device__ __forceinline__ void load(const T *p)
  {
#pragma unroll
    for (int i = 0; i < N / M; ++i) part[i] = Unit<T, M>::load(p + i * M);
  }
  __device__ __forceinline__ void floats(float *f) const
  {
#pragma unroll
    for (int i = 0; i < N / M; ++i) part[i].floats(f + i * M);
  }
};

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
constexpr uint32_t kZeros = 65536;                   // bytes of the table that a block sets to zero
constexpr uint32_t kCounted = 8192;                  // tokens that are sorted by counting
constexpr uint32_t kLong = 32;                       // places of a run that one piece adds up, at most
constexpr uint32_t kMostPiece = 32;                  // places of a piece
constexpr uint32_t kLeastLanes = 4;                  // threads of a piece

struct SortArgs {
  uint32_t n, vocab;
  const void *token;
  int token_bytes;
  uint32_t bits, passes;
  uint32_t *key[2], *place[2];          // the last pass writes the first of each
  uint32_t sorting;                     // blocks that sort
  uint32_t *runs;                       // the count of long runs, set to 0
  // rows of zeros
  void *dtable;
  uint64_t zero_rows, stride, row_bytes;        // in bytes
  uint32_t rows, cuts;                          // of a block; a row's blocks
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

// Zeros in kZeros bytes of the table: whole rows, or part of a long one.  Rows that tokens name get theirs, too: to leave them out, blocks had to know them, and
// as many as could look through the tokens had shares that the slower ones ended late with ([32768,4096] bf16 52 us, 37 as it is: 7.2 TB/s).
template <typename W> __device__ __forceinline__ void zero_part(const SortArgs &a)
{
  // (from the end on, so that the common tokens' rows, which come first, are the last to leave the second-level cache before their sums are written)
  const uint64_t block = gridDim.x - 1 - blockIdx.x, first = block / a.cuts * a.rows, cut = (block % a.cuts) * kZeros;
  const uint64_t bytes = a.cuts > 1 ? min((uint64_t)kZeros, a.row_bytes - cut) : a.row_bytes;
  uint32_t team = 1;
  while (team < kSortThreads && team * 16 < bytes) team *= 2;
  const uint32_t lane = threadIdx.x & (team - 1);
  for (uint64_t row = first + threadIdx.x / team; row < first + a.rows && row < a.zero_rows; row += kSortThreads / team) {
    char *to = static_cast<char *>(a.dtable) + row * a.stride + cut;
    // whole 16 bytes of it, and what lies before and behind them
    const uint32_t head = (uint32_t)min((uint64_t)(-(uintptr_t)to & 15), bytes), units = (uint32_t)((bytes - head) / 16);
    uint4 *body = reinterpret_cast<uint4 *>(to + head);
#pragma unroll 4
    for (uint32_t u = lane; u < units; u += team) body[u] = make_uint4(0, 0, 0, 0);
    W *behind = reinterpret_cast<W *>(body + units);
    for (uint32_t i = lane; i < head / sizeof(W); i += team) reinterpret_cast<W *>(to)[i] = W{};
    for (uint32_t i = lane; i < (bytes - head - (uint64_t)units * 16) / sizeof(W); i += team) behind[i] = W{};
  }
}

template <typename W> __global__ void __launch_bounds__(kSortThreads) embed_sort_kernel(const SortArgs a)
{
  __shared__ uint32_t count[kSortWarps][1u << kMostBits], totals[1u << kMostBits], base[kSortThreads + kSortWarps];
  static_assert(kSortThreads >= 1u << kMostBits, "a thread per digit");
  pdl_wait();
  pdl_trigger();
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.runs = 0;
  if (blockIdx.x < a.sorting) sort_tokens(a, count, totals, base);
  else zero_part<W>(a);
}

// Up to kCounted tokens: a block finds the places of 32 of them, a lane each, its warps each among a part of all tokens, of which those before it come before it if
// they are no larger, and those behind it if they are smaller
template <typename W> __global__ void __launch_bounds__(kSortThreads) embed_count_kernel(const SortArgs a)
{
  __shared__ __align__(16) uint32_t key[kCounted];
  __shared__ uint32_t counts[kSortWarps][32];
  pdl_wait();
  pdl_trigger();
  if (blockIdx.x >= a.sorting) { zero_part<W>(a); return; }
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.runs = 0;
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, begin = blockIdx.x * 32, i = begin + lane;
  const uint32_t part = (a.n + kSortWarps * 32 - 1) / (kSortWarps * 32) * 32;       // whole blocks' tokens of 32, so that none has tokens on both sides
  constexpr uint32_t AT_ONCE = 8;
  for (uint32_t j = threadIdx.x; j < part * kSortWarps; j += AT_ONCE * kSortThreads) {
    uint32_t k[AT_ONCE];
#pragma unroll
    for (uint32_t u = 0; u < AT_ONCE; ++u) k[u] = j + u * kSortThreads < a.n ? token_at(a.token, a.token_bytes, j + u * kSortThreads, a.vocab) : ~0u;
#pragma unroll
    for (uint32_t u = 0; u < AT_ONCE; ++u) if (j + u * kSortThreads < part * kSortWarps) key[j + u * kSortThreads] = k[u];
  }
  __syncthreads();
  const uint32_t mine = key[i], lo = warp * part, hi = lo + part;
  uint32_t before = 0;
  auto count_up = [&](uint32_t from, uint32_t to, uint32_t limit) {        // keys below `limit`
#pragma unroll 4
    for (uint32_t j = from; j < to; j += 4) {
      const uint4 k = *reinterpret_cast<const uint4 *>(key + j);
      before += (k.x < limit) + (k.y < limit) + (k.z < limit) + (k.w < limit);
    }
  };
  count_up(lo, min(hi, max(lo, begin)), mine + 1);
  if (begin >= lo && begin < hi) {
    for (uint32_t j = 0; j < 32; ++j) before += key[begin + j] < (j < lane ? mine + 1 : mine);
    count_up(begin + 32, hi, mine);
  } else if (begin < lo) count_up(lo, hi, mine);
  counts[warp][lane] = before;
  __syncthreads();
  if (warp || i >= a.n) return;
#pragma unroll
  for (uint32_t w = 1; w < kSortWarps; ++w) before += counts[w][lane];
  a.key[0][before] = mine;
  a.place[0][before] = i;
}

struct SumArgs {
  uint32_t n, vocab, cols;
  float scale;
  const uint32_t *key, *place;          // sorted
  const void *dy;
  uint64_t dy_stride;
  void *dtable;
  uint64_t stride;
  uint32_t piece, pieces, longest;      // places of a piece; a run of more than `longest` (from `piece` to kLong) is long
  uint32_t *runs;                       // how many runs are long, in whatever order: each one's first piece, token and count of parts
  uint4 *run;
  float *part;                          // [pieces][2][part_cols]: of a long run that begins before the piece, and of one that begins in it
  uint32_t part_cols;
  uint32_t lanes;                       // threads of a piece
};

// What a piece adds up: places [from, to), of which the runs of `head` and `tail` are long (else they are ~0)
struct Piece { uint32_t from, to, head, tail; bool head_before; };

// M units of E columns per thread; a block has kThreads/lanes pieces side by side.  The rows of one step are asked for before those of the step before it are
// used, whatever runs they belong to, and with them what the table holds where a run ends (ACC).
template <typename T, typename O, int E, int M, int STEP, bool ACC>
__global__ void __launch_bounds__(kThreads, ACC && M == 1 ? 2 : 3) embed_sums_kernel(const SumArgs a)
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
      const bool long0 = before + 1 + after > a.longest;
      const uint32_t k1 = key[last], ahead = run(k1, last - 1, -1), behind = run(k1, last + 1, 1);
      const bool long1 = k1 < a.vocab && ahead + 1 + behind > a.longest, whole = k0 == k1;
      q.head_before = before > 0;
      if (before && !long0) q.from = at + 1 + after;             // (that run is an earlier piece's)
      if (long0) q.head = k0;
      if (long1) q.tail = k1;
      q.to = long1 || k1 >= a.vocab ? last + 1 : last + 1 + behind;
      if (q.from > q.to || (whole && before && !long0)) q.to = q.from;
    }
    if (lane == 0) piece[p] = q;
    if (first + p >= a.pieces || blockIdx.y) continue;
    // the parts of a long run that begins here: this one, the pieces behind it that it fills, and one that it ends in
    if (q.tail != ~0u && !(q.tail == q.head && q.head_before)) {
      uint32_t filled = 32, r = first + p + 1;
      for (; filled == 32; r += filled) {
        const uint64_t end = (uint64_t)(r + lane + 1) * a.piece;
        const uint32_t others = ~__ballot_sync(0xffffffffu, end <= a.n && a.key[end - 1] == q.tail);
        filled = others ? (uint32_t)__ffs((int)others) - 1 : 32u;
      }
      const uint32_t parts = r - (first + p) + (r < a.pieces && a.key[(uint64_t)r * a.piece] == q.tail);
      if (lane == 0) a.run[atomicAdd(a.runs, 1u)] = make_uint4(first + p, q.tail, parts, 0);
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
  struct Stage {
    uint32_t k[STEP + 1];               // the places' tokens, and the one behind them; ~0: none
    Unit<T, E> v[STEP][M];
    Held<O, E> old[ACC ? STEP : 1][M];
  };
  auto fetch = [&](Stage &g, uint32_t i) {
#pragma unroll
    for (int s = 0; s <= STEP; ++s) { g.k[s] = i + s < q.to ? key[i + s] : ~0u; if (g.k[s] >= a.vocab) g.k[s] = ~0u; }
#pragma unroll
    for (int s = 0; s < STEP; ++s) {
      if (g.k[s] == ~0u) continue;
      const T *row = dy + place[i + s] * a.dy_stride;
#pragma unroll
      for (int m = 0; m < M; ++m) if (has[m]) g.v[s][m] = Unit<T, E>::load(row + (uint64_t)m * a.lanes * E);
    }
    if constexpr (ACC) {
#pragma unroll
      for (int s = 0; s < STEP; ++s) {
        if (g.k[s] == g.k[s + 1]) continue;
#pragma unroll
        for (int m = 0; m < M; ++m) if (has[m]) g.old[s][m].load(out + g.k[s] * a.stride + (uint64_t)m * a.lanes * E);
      }
    }
  };
  auto use = [&](const Stage &g) {
#pragma unroll
    for (int s = 0; s < STEP; ++s) {
      if (g.k[s] == ~0u) continue;
#pragma unroll
      for (int m = 0; m < M; ++m) {
        float f[E];
        g.v[s][m].floats(f);
#pragma unroll
        for (int j = 0; j < E; ++j) sum[m][j] += f[j];
      }
      if (g.k[s] == g.k[s + 1]) continue;
      // the run's end, or that of the piece's part of a long one
      const bool is_long = g.k[s] == q.head || g.k[s] == q.tail;
      float *to = part + (g.k[s] == q.head && q.head_before ? 0 : a.part_cols);
#pragma unroll
      for (int m = 0; m < M; ++m) {
        if (has[m] && is_long) {
#pragma unroll
          for (int j = 0; j < E; ++j) to[(uint64_t)m * a.lanes * E + j] = sum[m][j];
        } else if (has[m]) {
          float f[E];
          if constexpr (ACC) g.old[s][m].floats(f);
#pragma unroll
          for (int j = 0; j < E; ++j) sum[m][j] = ACC ? fmaf(sum[m][j], a.scale, f[j]) : sum[m][j] * a.scale;
          put_floats<O, E>(out + g.k[s] * a.stride + (uint64_t)m * a.lanes * E, sum[m]);
        }
#pragma unroll
        for (int j = 0; j < E; ++j) sum[m][j] = 0.0f;
      }
    }
  };
  Stage one, two;
  fetch(one, q.from);
  for (uint32_t i = q.from; i < q.to; i += 2 * STEP) {
    fetch(two, i + STEP);
    use(one);
    fetch(one, i + 2 * STEP);
    use(two);
  }
}

// The parts of long runs: a block has 128 columns and every gridDim.y-th such run; a warp adds a quarter of the run's parts, in order
constexpr uint32_t kJoinThreads = 128;
template <typename O> __global__ void __launch_bounds__(kJoinThreads) embed_join_kernel(const SumArgs a, const int accumulate)
{
  constexpr uint32_t WARPS = kJoinThreads / 32;
  __shared__ float sums[WARPS][4][32];
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint64_t c = ((uint64_t)blockIdx.x * 32 + lane) * 4;
  pdl_wait();
  const uint32_t runs = *a.runs;
  for (uint32_t i = blockIdx.y; i < runs; i += gridDim.y) {
    const uint4 run = a.run[i];
    const uint32_t parts = run.z, each = (parts + WARPS - 1) / WARPS, lo = min(parts, warp * each), hi = min(parts, lo + each);
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (c < a.cols) {
#pragma unroll 8
      for (uint32_t j = lo; j < hi; ++j) {
        const float4 v = *reinterpret_cast<const float4 *>(a.part + ((uint64_t)(run.x + j) * 2 + (j == 0)) * a.part_cols + c);
        sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
      }
    }
    sums[warp][0][lane] = sum.x; sums[warp][1][lane] = sum.y; sums[warp][2][lane] = sum.z; sums[warp][3][lane] = sum.w;
    // a warp writes 32 columns side by side
    const uint32_t mine = warp * 32 + lane;
    const uint64_t column = (uint64_t)blockIdx.x * 128 + mine;
    O *to = static_cast<O *>(a.dtable) + run.y * a.stride + column;
    const float old = accumulate && column < a.cols ? to_float(*to) : 0.0f;
    __syncthreads();
    if (column < a.cols) {
      float total = 0.0f;
#pragma unroll
      for (uint32_t w = 0; w < WARPS; ++w) total += sums[w][mine & 3][mine >> 2];
      *to = from_float<O>(accumulate ? fmaf(total, a.scale, old) : total * a.scale);
    }
    __syncthreads();
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

// Places of a piece: as many as give each multiprocessor three blocks of a row's width; a run of more is long, or of more than 8
inline uint32_t piece_of(uint64_t tokens)
{
  const uint64_t each = (tokens + 3 * 148 - 1) / (3 * 148);
  return (uint32_t)(each < 4 ? 4 : each < kMostPiece ? each : kMostPiece);
}

// Where the workspace's arrays begin, in bytes
struct Layout {
  uint64_t n, piece, longest, pieces, part_cols, runs, run, part, bytes;
  Layout(uint64_t tokens, uint32_t cols) : n((tokens + 3) / 4 * 4), piece(piece_of(tokens)), longest(piece < 8 ? 8 : piece), pieces((tokens + piece - 1) / piece), part_cols(((uint64_t)cols + 3) / 4 * 4)
  {
    runs = 16 * n;
    run = runs + 16;
    part = run + tokens / (longest + 1) * 16;
    bytes = part + pieces * 2 * part_cols * 4;
  }
};

template <typename T, typename O, int E> int launch_sums(SumArgs a, int accumulate, cudaStream_t stream)
{
  constexpr int M = E * sizeof(T) == 16 ? 1 : 2;
  const uint32_t units = a.cols / E;
  a.lanes = power_up_to((units + M - 1) / M, kThreads);
  if (a.lanes < kLeastLanes) a.lanes = kLeastLanes;
  const uint32_t per_block = kThreads / a.lanes, wide = (units + a.lanes * M - 1) / (a.lanes * M);
  const dim3 grid((a.pieces + per_block - 1) / per_block, wide);
  return accumulate ? launch(embed_sums_kernel<T, O, E, M, 4, true>, grid, kThreads, 0, stream, a)
                    : launch(embed_sums_kernel<T, O, E, M, 4, false>, grid, kThreads, 0, stream, a);
}
template <typename T, typename O> int launch_sums(const SumArgs &a, uint32_t unit, int accumulate, cudaStream_t stream)
{
  constexpr int V = 16 / sizeof(T);
  TRY((unit == (uint32_t)V ? launch_sums<T, O, V>(a, accumulate, stream) : unit == 2 ? launch_sums<T, O, 2>(a, accumulate, stream)
                                                                                      : launch_sums<T, O, 1>(a, accumulate, stream)));
  if (a.n <= a.longest) return ANODE_OK;
  // a run to a block, of the tokens of a training batch: some 50 of 16384 come more than 32 times
  const uint32_t wide = (uint32_t)(((uint64_t)a.cols + 127) / 128), most = a.n / (a.longest + 1), blocks = (16 * sm_count() + wide - 1) / wide;
  return launch(embed_join_kernel<O>, dim3(wide, blocks < most ? blocks : most), kJoinThreads, 0, stream, a, accumulate);
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
  SortArgs s = {(uint32_t)tokens, vocab, token, token_bytes, 0, 0, {words, words + l.n}, {words + 2 * l.n, words + 3 * l.n}, 0, words + l.runs / 4, dtable, 0, 0, 0, 1, 1};
  // tokens up to `vocab`, which stands for none
  uint32_t bits = 0;
  while (vocab >> bits) ++bits;
  s.passes = (bits + kMostBits - 1) / kMostBits;
  s.bits = (bits + s.passes - 1) / s.passes;
  const bool counted = tokens <= kCounted;
  s.sorting = !tokens ? 0 : counted ? (uint32_t)((tokens + 31) / 32) : kCluster;
  uint64_t blocks = 0;
  if (!accumulate) {
    s.zero_rows = vocab; s.stride = dtable_stride * oe; s.row_bytes = (uint64_t)cols * oe;
    if (dtable_stride == cols) { s.row_bytes *= vocab; s.zero_rows = 1; }      // (one long row)
    s.cuts = (uint32_t)((s.row_bytes + kZeros - 1) / kZeros);
    s.rows = s.cuts > 1 ? 1 : (uint32_t)(kZeros / s.row_bytes);
    blocks = (s.zero_rows + s.rows - 1) / s.rows * s.cuts;
    if (!counted) blocks = (blocks + kCluster - 1) / kCluster * kCluster;
    if (blocks >> 30) return ANODE_E_DIMS;
  }
  const dim3 grid(s.sorting + (uint32_t)blocks);
  TRY((counted ? (oe == 4 ? launch(embed_count_kernel<uint32_t>, grid, kSortThreads, 0, stream, s) : launch(embed_count_kernel<uint16_t>, grid, kSortThreads, 0, stream, s))
               : (oe == 4 ? launch_in_clusters(embed_sort_kernel<uint32_t>, grid, kCluster, kSortThreads, 0, stream, s)
                          : launch_in_clusters(embed_sort_kernel<uint16_t>, grid, kCluster, kSortThreads, 0, stream, s))));
  if (!tokens) return ANODE_OK;
  const SumArgs a = {(uint32_t)tokens, vocab, cols, scale, s.key[0], s.place[0], dy, dy_stride, dtable, dtable_stride, (uint32_t)l.piece, (uint32_t)l.pieces, (uint32_t)l.longest,
                     words + l.runs / 4, reinterpret_cast<uint4 *>(static_cast<char *>(workspace) + l.run), reinterpret_cast<float *>(static_cast<char *>(workspace) + l.part), (uint32_t)l.part_cols, 0};
  const uint32_t unit = unit_of(dy, e, dy_stride, tokens, dtable, oe, dtable_stride, vocab, cols);
  return by_type(type, [&](auto t) {
    using T = decltype(t);
    if constexpr (sizeof(T) == 2) { if (dtable_type != ANODE_TYPE_F32) return launch_sums<T, T>(a, unit, accumulate, stream); }
    return launch_sums<T, float>(a, unit, accumulate, stream);
  });
}
