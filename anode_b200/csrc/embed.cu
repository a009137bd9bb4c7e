// Rows of a table by tokens, and the table's gradient.
//
//   y[i] = scale*table[token[i]],   dtable[v] = scale * sum of dy[i] over token[i] = v
//
// A token outside of the table has a row of zeros and no gradient.  Sums are f32 and in the order of the tokens.
#include "bn_host.h"
#include "rows.cuh"

namespace anode_b200 {
namespace rows {

constexpr uint32_t kThreads = 256;

struct EmbedArgs {
  uint64_t tokens;
  uint32_t vocab, cols;
  float scale;
  const void *token;
  int token_bytes;
  const void *in;                       // the table, or dy
  uint64_t in_stride;
  void *out;                            // y, or the table's gradient
  uint64_t out_stride;
  int out_type, accumulate;
};

// a token as a row of the table, or `vocab` for one outside of it
__device__ __forceinline__ uint32_t token_at(const void *p, int bytes, uint64_t i, uint32_t vocab)
{
  const uint64_t t = bytes == 8 ? static_cast<const uint64_t *>(p)[i] : (uint64_t)(int64_t)static_cast<const int32_t *>(p)[i];
  return t < vocab ? (uint32_t)t : vocab;
}

template <typename T> __global__ void __launch_bounds__(kThreads) embed_rows_kernel(const EmbedArgs a)
{
  pdl_wait();
  for (uint64_t i = blockIdx.x; i < a.tokens; i += gridDim.x) {
    const uint32_t t = token_at(a.token, a.token_bytes, i, a.vocab);
    const T *in = static_cast<const T *>(a.in) + t * a.in_stride;
    T *y = static_cast<T *>(a.out) + i * a.out_stride;
    for (uint32_t c = threadIdx.x; c < a.cols; c += kThreads) y[c] = from_float<T>(t < a.vocab ? to_float(in[c]) * a.scale : 0.0f);
  }
}

// A block has a row of the table at a time, a thread a column, which walks down all tokens
template <typename T> __global__ void __launch_bounds__(kThreads) embed_grad_rows_kernel(const EmbedArgs a)
{
  pdl_wait();
  for (uint64_t v = blockIdx.x; v < a.vocab; v += gridDim.x)
    for (uint64_t c = (uint64_t)blockIdx.y * kThreads + threadIdx.x; c < a.cols; c += (uint64_t)gridDim.y * kThreads) {
      float sum = 0.0f;
      bool any = false;
      for (uint64_t i = 0; i < a.tokens; ++i)
        if (token_at(a.token, a.token_bytes, i, a.vocab) == v) { sum += to_float(static_cast<const T *>(a.in)[i * a.in_stride + c]); any = true; }
      if (a.accumulate && !any) continue;
      sum *= a.scale;
      const uint64_t at = v * a.out_stride + c;
      if (a.out_type == ANODE_TYPE_F32) { float *o = static_cast<float *>(a.out) + at; *o = a.accumulate ? *o + sum : sum; }
      else { T *o = static_cast<T *>(a.out) + at; *o = from_float<T>(a.accumulate ? to_float(*o) + sum : sum); }
    }
}

inline int check_tokens(const void *token, int bytes)
{
  if (bytes != 4 && bytes != 8) return ANODE_E_TYPE;
  if (!token) return ANODE_E_NULL;
  return aligned_to(token, (size_t)bytes) ? ANODE_OK : ANODE_E_ALIGN;
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
  const EmbedArgs a = {tokens, vocab, cols, scale, token, token_bytes, table, table_stride, y, y_stride, type, 0};
  return by_type(type, [&](auto t) { return launch(embed_rows_kernel<decltype(t)>, dim3(row_blocks(tokens)), kThreads, 0, stream, a); });
}

extern "C" size_t anode_gpu_embed_tokens_bwd_workspace_bytes(uint64_t tokens, uint32_t vocab, uint32_t cols)
{
  (void)tokens; (void)vocab; (void)cols;
  return 16;
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
  TRY(check_rows(dtable, type_bytes(dtable_type), vocab, cols, dtable_stride, true));
  if (tokens) {
    TRY(check_tokens(token, token_bytes));
    TRY(check_rows(dy, type_bytes(type), tokens, cols, dy_stride, false));
    if (dy == dtable) return ANODE_E_STRIDE;
    if (!workspace || !aligned_to(workspace, 16) || workspace_bytes < anode_gpu_embed_tokens_bwd_workspace_bytes(tokens, vocab, cols)) return ANODE_E_WORKSPACE;
  }
  const EmbedArgs a = {tokens, vocab, cols, scale, token, token_bytes, dy, dy_stride, dtable, dtable_stride, dtable_type, accumulate};
  const uint32_t wide = cols < 64 * kThreads ? (cols + kThreads - 1) / kThreads : 64;
  return by_type(type, [&](auto t) { return launch(embed_grad_rows_kernel<decltype(t)>, dim3(row_blocks(vocab), wide), kThreads, 0, stream, a); });
}
