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
//      of places ends.  A run of no more places than a piece has belongs to the piece where it begins; of a longer one each piece leaves its part in the workspace;
//   3. the parts of each long run are joined, in order.
//
// Measured on one B200 against its copy bandwidth of 6539 GB/s: rows of 16384 tokens of [32768,8192] bf16 59 us (0.93), of [.,4096] f16 30, of [.,4095] 51 (two loads
// to a slot, and a row's first and last elements one by one), 32 tokens 1.6 us.  The gradient
// of 16384 tokens of [32768,4096] bf16, whose tokens are common ones mostly, 81 us (0.76): zeros 37 (7.2 TB/s, the sort beside them), sums 35, join 8; rows named twice are
// written twice.  Added to what is there 66 us, where the sort (16 us with caches flushed, a chain of eight waits of a cluster) is seen; to f32 82; 131072 to [32768,1024] 143.  4099 tokens of [50021,1001] f16 into f32 47 us,
// added 23.5.  The zeros and the sums are bound by memory, small calls by the chain token -> place -> row -> sum.
#include "bn_host.h"
#include "rows.cuh"

namespace anode_b200 {
namespace rows {
namespace embed {

constexpr uint32_t kThreads = 256;

// 16 bytes' elements of a row from column c on, wherever they begin: two aligned pieces that are shifted together when they are used, or, where those would reach
// beyond the row, elements apart, put together when they are used, too, so that nothing waits for a load before then (columns that the row does not have are 0)
template <typename T> struct Shifted {
  static constexpr int V = Vec<T>::V;
  typedef typename std::conditional<sizeof(T) == 4, uint32_t, uint16_t>::type Bits;
  static constexpr uint32_t APART = 8;
  uint32_t w[8], o;
  __device__ __forceinline__ void load(const T *row, int64_t c, uint32_t cols)
  {
    const T *p = row + c;
    o = (uint32_t)((uintptr_t)p & 15) / sizeof(T);
    if (c >= (int64_t)o && c - o + (o ? 2 * V : V) <= (int64_t)cols) {
      *reinterpret_cast<uint4 *>(w) = *reinterpret_cast<const uint4 *>(p - o);
      if (o) *reinterpret_cast<uint4 *>(w + 4) = *reinterpret_cast<const uint4 *>(p - o + V);
      return;
    }
    o = APART;
#pragma unroll
    for (int i = 0; i < V; ++i) w[i] = c + i >= 0 && c + i < cols ? reinterpret_cast<const Bits *>(p)[i] : Bits(0);
  }
  __device__ __forceinline__ void floats(float *f) const
  {
    if (o == APART) {
#pragma unroll
      for (int i = 0; i < V; ++i) { const Bits bits = (Bits)w[i]; f[i] = to_float(*reinterpret_cast<const T *>(&bits)); }
    } else shifted(f);
  }
  __device__ __forceinline__ void shifted(float *f) const
  {
    // (words, and half a word)
    const uint32_t by = sizeof(T) == 4 ? o : o / 2;
    uint32_t v[6], u[5];
#pragma unroll
    for (int i = 0; i < 6; ++i) v[i] = by & 2 ? w[i + 2] : w[i];
#pragma unroll
    for (int i = 0; i < 5; ++i) u[i] = by & 1 ? v[i + 1] : v[i];
    uint4 all = make_uint4(u[0], u[1], u[2], u[3]);
    if constexpr (sizeof(T) == 2) {
      const uint32_t pick = o & 1 ? 0x5432u : 0x3210u;
      all = make_uint4(__byte_perm(u[0], u[1], pick), __byte_perm(u[1], u[2], pick), __byte_perm(u[2], u[3], pick), __byte_perm(u[3], u[4], pick));
    }
    Vec<T>{all}.floats(f);
  }
};
// The same where no piece reaches beyond the row; or, of a thread with a single column, that element (the other words stay 0)
template <typename T> struct Inside {
  static constexpr int V = Vec<T>::V;
  Shifted<T> s;
  __device__ __forceinline__ void clear()
  {
    s.o = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) s.w[i] = 0;
  }
  __device__ __forceinline__ void load(const T *p, bool single)
  {
    if (single) { s.w[0] = *reinterpret_cast<const typename Shifted<T>::Bits *>(p); return; }
    s.o = (uint32_t)((uintptr_t)p & 15) / sizeof(T);
    *reinterpret_cast<uint4 *>(s.w) = *reinterpret_cast<const uint4 *>(p - s.o);
    if (s.o) *reinterpret_cast<uint4 *>(s.w + 4) = *reinterpret_cast<const uint4 *>(p - s.o + V);
  }
  __device__ __forceinline__ void floats(float *f) const { s.shifted(f); }
};
// The same of rows that all begin at 16 bytes
template <typename T> struct Whole {
  __device__ __forceinline__ void clear() {}
  __device__ __forceinline__ void load(const T *p, bool) { v = Vec<T>::load(p); }
  Vec<T> v;
  __device__ __forceinline__ void load(const T *row, int64_t c, uint32_t) { v = Vec<T>::load(row + c); }
  __device__ __forceinline__ void floats(float *f) const { v.floats(f); }
};

// N elements of a row that is written, as they lie in memory
template <typename T, int N> struct Held {
  static constexpr int V = Vec<T>::V, K = N / V ? N / V : 1;
  Vec<T> part[K];
  static_assert(N % V == 0, "a table's gradient is of dy's type or a wider one");
  __device__ __forceinline__ void load(const T *p)
  {
#pragma unroll
    for (int i = 0; i < K; ++i) part[i] = Vec<T>::load(p + i * V);
  }
  __device__ __forceinline__ void load_each(const T *p, uint32_t n)
  {
#pragma unroll
    for (int i = 0; i < N; ++i) if ((uint32_t)i < n) reinterpret_cast<T *>(part)[i] = p[i];
  }
  __device__ __forceinline__ void floats(float *f) const
  {
#pragma unroll
    for (int i = 0; i < K; ++i) part[i].floats(f + i * V);
  }
  __device__ __forceinline__ static void store(T *p, const float *f)
  {
#pragma unroll
    for (int i = 0; i < K; ++i) Vec<T>::of(f + i * V).store(p + i * V);
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

// A team of lanes (a power of two, up to a warp) has a token and four slots of 16 bytes of its row per lane; the grid's second dimension has the rest of wide
// rows.  SHIFT: rows that begin anywhere; slots are those of y's addresses, and a row's first and last may be parts of one.
template <typename T, bool SHIFT> __global__ void __launch_bounds__(128) embed_kernel(const EmbedArgs a, const uint32_t team)
{
  constexpr int V = Vec<T>::V, M = 4;
  const uint64_t i = ((uint64_t)blockIdx.x * 128 + threadIdx.x) / team;
  const uint32_t lane = threadIdx.x & (team - 1);
  pdl_wait();
  pdl_trigger();
  if (i >= a.tokens) return;
  const uint32_t t = token_at(a.token, a.token_bytes, i, a.vocab);
  const T *in = static_cast<const T *>(a.table) + t * a.table_stride;
  T *y = static_cast<T *>(a.y) + i * a.y_stride;
  const uint32_t ahead = SHIFT ? (uint32_t)((uintptr_t)y & 15) / sizeof(T) : 0, slots = (a.cols + ahead + V - 1) / V;
  for (uint32_t first = blockIdx.y * team * M + lane; first < slots; first += gridDim.y * team * M) {
    typename std::conditional<SHIFT, Shifted<T>, Whole<T>>::type v[M];
    auto column = [&](int k) { return (int64_t)(first + k * team) * V - ahead; };
#pragma unroll
    for (int k = 0; k < M; ++k) if (t < a.vocab && first + k * team < slots) v[k].load(in, column(k), a.cols);
#pragma unroll
    for (int k = 0; k < M; ++k) {
      if (first + k * team >= slots) continue;
      const int64_t c = column(k);
      float f[V];
      v[k].floats(f);
#pragma unroll
      for (int j = 0; j < V; ++j) f[j] = t < a.vocab ? f[j] * a.scale : 0.0f;
      if (!SHIFT || (c >= 0 && c + V <= a.cols)) Vec<T>::of(f).store(y + c);
      else {
#pragma unroll
        for (int j = 0; j < V; ++j) if (c + j >= 0 && c + j < a.cols) y[c + j] = from_float<T>(f[j]);
      }
    }
  }
}

// ---- the gradient ---------------------------------------------------------------------------------------------------------------

constexpr uint32_t kCluster = 16, kFewer = 8;         // blocks that sort
constexpr uint32_t kSortThreads = 512, kSortWarps = kSortThreads / 32;
constexpr uint32_t kMostBits = 9;                    // of a token to a pass of the sort
constexpr uint32_t kZeros = 65536;                   // bytes of the table that a block sets to zero
constexpr uint32_t kCounted = 8192;                  // tokens that are sorted by counting
constexpr uint32_t kMostPiece = 32;                  // places of a piece
constexpr uint32_t kLong = kMostPiece;               // places on either side that a piece looks at
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
template <uint32_t CLUSTER> __device__ __forceinline__ void sort_tokens(const SortArgs &a, uint32_t (*count)[1u << kMostBits], uint32_t *totals, uint32_t *base)
{
  constexpr uint32_t STEPS = 4;
  const uint32_t rank = cluster_rank(), warp = threadIdx.x >> 5, lane = threadIdx.x & 31, bins = 1u << a.bits;
  const uint32_t stretch = (a.n + CLUSTER * kSortWarps * 32 - 1) / (CLUSTER * kSortWarps * 32) * 32;
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
      uint32_t c[CLUSTER];
#pragma unroll
      for (uint32_t r = 0; r < CLUSTER; ++r) c[r] = peer_load(totals + t, r);
#pragma unroll
      for (uint32_t r = 0; r < CLUSTER; ++r) { before += r < rank ? c[r] : 0; all += c[r]; }
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

template <typename W, uint32_t CLUSTER> __global__ void __launch_bounds__(kSortThreads) embed_sort_kernel(const SortArgs a)
{
  __shared__ uint32_t count[kSortWarps][1u << kMostBits], totals[1u << kMostBits], base[kSortThreads + kSortWarps];
  static_assert(kSortThreads >= 1u << kMostBits, "a thread per digit");
  pdl_wait();
  pdl_trigger();
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.runs = 0;
  if (blockIdx.x < a.sorting) sort_tokens<CLUSTER>(a, count, totals, base);
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
  uint32_t piece, pieces;               // places of a piece; a run of more is long
  uint32_t *runs;                       // how many runs are long, in whatever order: each one's first piece, token and count of parts
  uint4 *run;
  float *part;                          // [pieces][2][part_cols]: of a long run that begins before the piece, and of one that begins in it
  uint32_t part_cols;
  uint32_t lanes;                       // threads of a piece
  uint32_t slots, singles;              // of them, those with 16 bytes of columns, and those with a column each
};

// What a piece adds up: places [from, to), of which the runs of `head` and `tail` are long (else they are ~0)
struct Piece { uint32_t from, to, head, tail; bool head_before; };

// A thread has 16 bytes of columns; a block has pieces side by side, each with `lanes` threads.  The rows of one step are asked for before those of the step before it are
// used, whatever runs they belong to, and with them what the table holds where a run ends (ACC).  SHIFT: rows that begin anywhere, whose first and last columns have
// a thread each.
template <typename T, typename O, bool SHIFT, bool ACC>
__global__ void __launch_bounds__(kThreads, ACC ? 2 : 3) embed_sums_kernel(const SumArgs a)
{
  constexpr int E = Vec<T>::V, STEP = SHIFT || (ACC && sizeof(O) > sizeof(T)) ? 2 : 4;      // (as there are registers for)
  constexpr uint32_t PIECES = kThreads / kLeastLanes;
  __shared__ uint32_t key[PIECES * kMostPiece + 2 * kLong], place[PIECES * kMostPiece + 2 * kLong];
  __shared__ Piece piece[PIECES];
  pdl_wait();
  pdl_trigger();
  const uint32_t per_block = blockDim.x / a.lanes, first = blockIdx.x * per_block, lane = threadIdx.x & 31;
  // the places of the block's pieces and kLong on either side; what is no token ends the sorted ones
  const int64_t begin = (int64_t)first * a.piece - kLong;
  for (uint32_t i = threadIdx.x; i < per_block * a.piece + 2 * kLong; i += blockDim.x) {
    const int64_t at = begin + i;
    const bool inside = at >= 0 && at < a.n;
    const uint32_t k = inside ? a.key[at] : ~0u;
    key[i] = k < a.vocab ? k : ~0u;
    place[i] = inside ? a.place[at] : 0;
  }
  __syncthreads();
  // a warp looks at a piece: how far the runs of its first and last token go, up to kLong places
  for (uint32_t p = threadIdx.x >> 5; p < per_block; p += blockDim.x / 32) {
    const uint32_t at = kLong + p * a.piece, size = min(a.piece, a.n - min(a.n, (first + p) * a.piece)), last = at + size - 1;
    auto run = [&](uint32_t k, uint32_t from, int step) {        // places from `from` on, in steps, that have token k
      const uint32_t other = ~__ballot_sync(0xffffffffu, key[(int)from + step * (int)lane] == k);
      return other ? (uint32_t)__ffs((int)other) - 1 : 32u;
    };
    Piece q = {at, at, ~0u, ~0u, false};
    if (size && key[at] != ~0u) {
      const uint32_t k0 = key[at], before = run(k0, at - 1, -1), after = run(k0, at + 1, 1);
      const bool long0 = before + 1 + after > a.piece;
      const uint32_t k1 = key[last], ahead = run(k1, last - 1, -1), behind = run(k1, last + 1, 1);
      const bool long1 = k1 != ~0u && ahead + 1 + behind > a.piece, whole = k0 == k1;
      q.head_before = before > 0;
      if (before && !long0) q.from = at + 1 + after;             // (that run is an earlier piece's)
      if (long0) q.head = k0;
      if (long1) q.tail = k1;
      q.to = long1 || k1 == ~0u ? last + 1 : last + 1 + behind;
      if (q.from > q.to || (whole && before && !long0)) q.to = q.from;
    }
    if (lane == 0) piece[p] = q;
  }
  __syncthreads();
  const uint32_t mine = threadIdx.x / a.lanes;
  const Piece q = piece[mine];
  // slots from the row's start on, or with a slot left out there; then single columns: those before the slots, and those behind them
  const uint32_t at = blockIdx.y * a.lanes + (threadIdx.x - mine * a.lanes);
  const bool single = SHIFT && at >= a.slots, has = at < a.slots + a.singles;
  const uint32_t ahead = SHIFT && a.slots ? E : 0, width = !has ? 0 : single ? 1 : E;
  const uint64_t column = !single ? (uint64_t)at * E + ahead : at - a.slots < ahead ? at - a.slots : (uint64_t)a.slots * E + (at - a.slots);
  const T *dy = static_cast<const T *>(a.dy) + column;
  O *out = static_cast<O *>(a.dtable) + column;
  float *part = a.part + ((uint64_t)(first + mine) * 2 * a.part_cols) + column;
  float sum[E];
#pragma unroll
  for (int j = 0; j < E; ++j) sum[j] = 0.0f;
  struct Stage {
    uint32_t k[STEP + 1];               // the places' tokens, and the one behind them; ~0: none
    typename std::conditional<SHIFT, Inside<T>, Whole<T>>::type v[STEP];
    Held<O, E> old[ACC ? STEP : 1];
  };
  auto fetch = [&](Stage &g, uint32_t i) {
#pragma unroll
    for (int s = 0; s <= STEP; ++s) g.k[s] = has && i + s < q.to ? key[i + s] : ~0u;
#pragma unroll
    for (int s = 0; s < STEP; ++s) if (g.k[s] != ~0u) g.v[s].load(dy + place[i + s] * a.dy_stride, single);
    if constexpr (ACC) {
#pragma unroll
      for (int s = 0; s < STEP; ++s) {
        if (g.k[s] == g.k[s + 1]) continue;
        const O *from = out + g.k[s] * a.stride;
        if constexpr (SHIFT) g.old[s].load_each(from, width); else g.old[s].load(from);
      }
    }
  };
  auto use = [&](const Stage &g) {
#pragma unroll
    for (int s = 0; s < STEP; ++s) {
      if (g.k[s] == ~0u) continue;
      float f[E];
      g.v[s].floats(f);
#pragma unroll
      for (int j = 0; j < E; ++j) sum[j] += f[j];
      if (g.k[s] == g.k[s + 1]) continue;
      // the run's end, or that of the piece's part of a long one
      if (g.k[s] == q.head || g.k[s] == q.tail) {
        float *to = part + (g.k[s] == q.head && q.head_before ? 0 : a.part_cols);
#pragma unroll
        for (int j = 0; j < E; ++j) if ((uint32_t)j < width) to[j] = sum[j];
      } else {
        O *to = out + g.k[s] * a.stride;
        if constexpr (ACC) g.old[s].floats(f);
#pragma unroll
        for (int j = 0; j < E; ++j) sum[j] = ACC ? fmaf(sum[j], a.scale, f[j]) : sum[j] * a.scale;
        if constexpr (!SHIFT) Held<O, E>::store(to, sum);
        else {
#pragma unroll
          for (int j = 0; j < E; ++j) if ((uint32_t)j < width) to[j] = from_float<O>(sum[j]);
        }
      }
#pragma unroll
      for (int j = 0; j < E; ++j) sum[j] = 0.0f;
    }
  };
  Stage one, two;
#pragma unroll
  for (int s = 0; s < STEP; ++s) { one.v[s].clear(); two.v[s].clear(); }
  fetch(one, q.from);
  for (uint32_t i = q.from; i < q.to; i += 2 * STEP) {
    fetch(two, i + STEP);
    use(one);
    fetch(one, i + 2 * STEP);
    use(two);
  }
  // the long runs that begin here: this piece, those behind it that the run fills, and one that it ends in
  for (uint32_t p = threadIdx.x >> 5; p < per_block && blockIdx.y == 0; p += blockDim.x / 32) {
    const uint32_t k = piece[p].tail;
    if (k == ~0u || (k == piece[p].head && piece[p].head_before)) continue;
    uint32_t filled = 32, r = first + p + 1;
    for (; filled == 32; r += filled) {
      const uint64_t end = (uint64_t)(r + lane + 1) * a.piece;
      const uint32_t others = ~__ballot_sync(0xffffffffu, end <= a.n && a.key[end - 1] == k);
      filled = others ? (uint32_t)__ffs((int)others) - 1 : 32u;
    }
    const uint32_t parts = r - (first + p) + (r < a.pieces && a.key[(uint64_t)r * a.piece] == k);
    if (lane == 0) a.run[atomicAdd(a.runs, 1u)] = make_uint4(first + p, k, parts, 0);
  }
}

// The parts of long runs: a block has 64 columns, four to a lane, and every gridDim.y-th such run, whose parts its 16 groups of lanes add in order, each a stretch
template <typename O> __global__ void __launch_bounds__(kThreads) embed_join_kernel(const SumArgs a, const int accumulate)
{
  constexpr uint32_t LANES = 16, GROUPS = kThreads / LANES;
  __shared__ float sums[GROUPS][4 * LANES + 1];
  const uint32_t group = threadIdx.x / LANES, lane = threadIdx.x % LANES;
  const uint64_t c = ((uint64_t)blockIdx.x * LANES + lane) * 4, column = (uint64_t)blockIdx.x * 4 * LANES + threadIdx.x;
  pdl_wait();
  const uint32_t runs = *a.runs;
  uint4 next = a.run[blockIdx.y];        // (what the list does not hold is not used)
  for (uint32_t i = blockIdx.y; i < runs; i += gridDim.y) {
    const uint4 run = next;
    if (i + gridDim.y < runs) next = a.run[i + gridDim.y];
    const uint32_t parts = run.z, each = (parts + GROUPS - 1) / GROUPS, lo = min(parts, group * each), hi = min(parts, lo + each);
    O *out = static_cast<O *>(a.dtable) + run.y * a.stride + column;
    const bool writes = threadIdx.x < 4 * LANES && column < a.cols;
    const float old = accumulate && writes ? to_float(*out) : 0.0f;
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (c < a.cols) {
#pragma unroll 8
      for (uint32_t j = lo; j < hi; ++j) {
        const float4 v = *reinterpret_cast<const float4 *>(a.part + ((uint64_t)(run.x + j) * 2 + (j == 0)) * a.part_cols + c);
        sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
      }
    }
    float *const to = sums[group] + lane * 4;
    to[0] = sum.x; to[1] = sum.y; to[2] = sum.z; to[3] = sum.w;
    __syncthreads();
    if (writes) {
      float all = 0.0f;
#pragma unroll
      for (uint32_t g = 0; g < GROUPS; ++g) all += sums[g][threadIdx.x];
      *out = from_float<O>(accumulate ? fmaf(all, a.scale, old) : all * a.scale);
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

// Whether rows all begin at 16 bytes and are whole numbers of them
inline bool whole(const void *p, size_t bytes, uint64_t stride, uint64_t rows, uint32_t cols)
{
  return aligned_to(p, 16) && cols * bytes % 16 == 0 && (rows <= 1 || stride * bytes % 16 == 0);
}
inline uint32_t power_up_to(uint64_t n, uint32_t most)
{
  uint32_t v = 1;
  while (v < most && v < n) v *= 2;
  return v;
}

// How the columns of a piece are shared out: slots of 16 bytes, single columns (SHIFT), threads of a piece, pieces of a block, and blocks side by side
struct Shares {
  uint32_t slots, singles, lanes, per_block, wide;
  Shares(uint32_t cols, uint32_t v, bool shift) : slots(cols / v)
  {
    // (rows that begin anywhere: two aligned pieces around each slot are to be inside of the row)
    if (shift) slots = slots > 2 ? slots - 2 : 0;
    singles = cols - slots * v;
    const uint32_t all = slots + singles;
    lanes = all > kThreads ? kThreads : all > 32 ? (all + 31) / 32 * 32 : power_up_to(all, 32);
    if (lanes < kLeastLanes) lanes = kLeastLanes;
    per_block = kThreads / lanes;
    wide = (all + lanes - 1) / lanes;
  }
};

// Places of a piece; a run of more is long.  Short pieces are short chains of rows, long ones have fewer parts to join and fewer borders to look at.  As many as leave
// the device 2^18 threads of rows of 16-bit columns, and of those where that is few: as many as let all blocks run at once (with 512 threads to a multiprocessor, for which the
// adding form has registers), if 16 are enough for that, and 8 at least.  Added to what is there, us, tokens of a frequency-ordered vocabulary (8 / 10 / 16 places):
// [2048,2048] bf16 12.3 / 12.9 / 13.6, [512,1024] 8.2 / 8.9 / 9.2, [1000,768] f32 9.1 / 9.9 / 10.8, [3001,333] f16 18.2 / 20.7 / 26.2, whose blocks all run at once with 8; [4099,1001] f16
// into f32 26.2 / 23.3 / 27.7 (at once from 10 on), [8192,1024] bf16 28.5 / 28.9 / 25.9 (from 14 on); [16384,4096] 102 with 8, 86 with 16, 81 with 32.
// The limit of 16: at once from 32 and 28 on, [5000,3001] into f32 65.8 (54.3 with 8) and [32768,300] bf16, assigned, 52.6 (49.6).
// (from sizes alone, since the workspace's size goes by it)
inline uint32_t piece_of(uint64_t tokens, uint32_t cols)
{
  const Shares s(cols, 8, cols % 8 != 0);
  const uint64_t threads = tokens * ((uint64_t)cols / 8 + 16), each = (threads + (1u << 18) - 1) >> 18;
  const uint64_t blocks = 148 * (2 * kThreads / (s.per_block * s.lanes)) / s.wide, at_once = (blocks ? blocks : 1) * s.per_block, fits = (tokens + at_once - 1) / at_once;
  const uint64_t least = fits <= 16 && fits > 8 ? fits : 8, piece = each < least ? least : each;
  return (uint32_t)(piece < kMostPiece ? piece : kMostPiece);
}

// Where the workspace's arrays begin, in bytes
struct Layout {
  uint64_t n, piece, pieces, part_cols, runs, run, part, bytes;
  Layout(uint64_t tokens, uint32_t cols) : n((tokens + 3) / 4 * 4), piece(piece_of(tokens, cols)), pieces((tokens + piece - 1) / piece), part_cols(((uint64_t)cols + 3) / 4 * 4)
  {
    runs = 16 * n;
    run = runs + 16;
    part = run + tokens / (piece + 1) * 16;
    bytes = part + pieces * 2 * part_cols * 4;
  }
};

template <typename W> int launch_sort(dim3 grid, cudaStream_t stream, const SortArgs &s)
{
  static WideClusters allowed;
  if (s.sorting == kFewer) return launch_in_clusters(embed_sort_kernel<W, kFewer>, grid, kFewer, kSortThreads, 0, stream, s);
  if (!allowed.of((const void *)embed_sort_kernel<W, kCluster>)) return ANODE_E_LAUNCH;
  return launch_in_clusters(embed_sort_kernel<W, kCluster>, grid, kCluster, kSortThreads, 0, stream, s);
}

template <typename T, typename O> int launch_sums(SumArgs a, bool shift, int accumulate, cudaStream_t stream)
{
  constexpr uint32_t V = Vec<T>::V;
  const Shares part(a.cols, V, shift);
  a.slots = part.slots; a.singles = part.singles; a.lanes = part.lanes;
  const dim3 grid((a.pieces + part.per_block - 1) / part.per_block, part.wide);
  TRY(launch(accumulate ? (shift ? embed_sums_kernel<T, O, true, true> : embed_sums_kernel<T, O, false, true>)
                        : (shift ? embed_sums_kernel<T, O, true, false> : embed_sums_kernel<T, O, false, false>), grid, part.per_block * a.lanes, 0, stream, a));
  if (a.n <= a.piece) return ANODE_OK;
  // a run to a block, of the tokens of a training batch: some 50 of 16384 come more than 32 times
  const uint32_t wide = (uint32_t)(((uint64_t)a.cols + 63) / 64), most = a.n / (a.piece + 1), blocks = (8 * sm_count() + wide - 1) / wide;
  return launch(embed_join_kernel<O>, dim3(wide, blocks < most ? blocks : most), kThreads, 0, stream, a, accumulate);
}

}  // namespace embed
}  // namespace rows
}  // namespace anode_b200

using namespace anode_b200::rows;
using namespace anode_b200::rows::embed;

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
  if (rows_meet(y, y_stride * e, tokens, cols * e, table, table_stride * e, vocab, cols * e)) return ANODE_E_STRIDE;
  const EmbedArgs a = {tokens, vocab, cols, scale, token, token_bytes, table, table_stride, y, y_stride};
  const bool shift = !whole(table, e, table_stride, vocab, cols) || !whole(y, e, y_stride, tokens, cols);
  return by_type(type, [&](auto t) {
    using T = decltype(t);
    constexpr uint32_t V = Vec<T>::V;
    const uint32_t slots = (cols + (shift ? 2 * V - 2 : V - 1)) / V, team = power_up_to((slots + 3) / 4, 32);
    const uint64_t wide = ((uint64_t)slots + team * 4 - 1) / (team * 4);
    const dim3 grid((uint32_t)((tokens * team + 127) / 128), (uint32_t)(wide < 65535 ? wide : 65535));
    return launch(shift ? embed_kernel<T, true> : embed_kernel<T, false>, grid, 128, 0, stream, a, team);
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
  if (!served(0, cols) || !served(0, vocab) || tokens >> 31 || cols >> 25) return ANODE_E_DIMS;      // (a grid's second dimension)
  if (tokens == 0 && accumulate) return ANODE_OK;
  const size_t e = type_bytes(type), oe = type_bytes(dtable_type);
  TRY(check_rows(dtable, oe, vocab, cols, dtable_stride, true));
  if (tokens) {
    TRY(check_tokens(token, token_bytes));
    TRY(check_rows(dy, e, tokens, cols, dy_stride, false));
    if (rows_meet(dtable, dtable_stride * oe, vocab, cols * oe, dy, dy_stride * e, tokens, cols * e)) return ANODE_E_STRIDE;
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
  // sixteen blocks to the sort, which sums wait for (16384 tokens added to [32768,4096] bf16 66 us, 69 with eight; 131072 to [32768,1024] 143 and 179), but eight where the zeros take
  // longer, which clusters of sixteen would write more slowly (16384 tokens of [32768,4096] 81 us, 84 with sixteen; of [32768,1024], 4 KB to a token, 40 and 38).  Of 55 sizes, 8200 to
  // 131072 tokens of bf16 tables of 4096 to 262144 rows of 256 to 8192 columns, the line of 8 KB to a token was wrong by more than 1 % at one (40000 of [262144,1000], 13 KB: 118, 110 with sixteen)
  const bool hidden = !accumulate && (uint64_t)vocab * cols * oe > 8192 * tokens;
  s.sorting = !tokens ? 0 : counted ? (uint32_t)((tokens + 31) / 32) : hidden ? kFewer : kCluster;
  uint64_t blocks = 0;
  if (!accumulate) {
    s.zero_rows = vocab; s.stride = dtable_stride * oe; s.row_bytes = (uint64_t)cols * oe;
    if (dtable_stride == cols) { s.row_bytes *= vocab; s.zero_rows = 1; }      // (one long row)
    const uint64_t cuts = (s.row_bytes + kZeros - 1) / kZeros;
    s.rows = cuts > 1 ? 1 : (uint32_t)(kZeros / s.row_bytes);
    blocks = (s.zero_rows + s.rows - 1) / s.rows * cuts;
    if (!counted) blocks = (blocks + s.sorting - 1) / s.sorting * s.sorting;
    if (cuts >> 30 || blocks >> 30) return ANODE_E_DIMS;
    s.cuts = (uint32_t)cuts;
  }
  const dim3 grid(s.sorting + (uint32_t)blocks);
  TRY((counted ? (oe == 4 ? launch(embed_count_kernel<uint32_t>, grid, kSortThreads, 0, stream, s) : launch(embed_count_kernel<uint16_t>, grid, kSortThreads, 0, stream, s))
               : (oe == 4 ? launch_sort<uint32_t>(grid, stream, s) : launch_sort<uint16_t>(grid, stream, s))));
  if (!tokens) return ANODE_OK;
  const SumArgs a = {(uint32_t)tokens, vocab, cols, scale, s.key[0], s.place[0], dy, dy_stride, dtable, dtable_stride, (uint32_t)l.piece, (uint32_t)l.pieces,
                     words + l.runs / 4, reinterpret_cast<uint4 *>(static_cast<char *>(workspace) + l.run), reinterpret_cast<float *>(static_cast<char *>(workspace) + l.part), (uint32_t)l.part_cols, 0};
  const bool shift = !whole(dy, e, dy_stride, tokens, cols) || !whole(dtable, oe, dtable_stride, vocab, cols);
  return by_type(type, [&](auto t) {
    using T = decltype(t);
    if constexpr (sizeof(T) == 2) { if (dtable_type != ANODE_TYPE_F32) return launch_sums<T, T>(a, shift, accumulate, stream); }
    return launch_sums<T, float>(a, shift, accumulate, stream);
  });
}
