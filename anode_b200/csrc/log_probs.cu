// Log probabilities of given tokens, the entropies of their rows and the likeliest tokens, and the gradient of the logits.
//
//   m = max x, z = scale*(x - m), L = log(sum(exp(z))):   logprob = z[token] - L,   H = L - sum(z*exp(z))/sum(exp(z))
//   p = exp(z - L):   dx = scale*(dlogprob*([token] - p) - dentropy*p*(z - L + H))
//
// A row keeps m and L apart, since their sum would lose L's digits beside a large m.
#include "bn_host.h"
#include "rows.cuh"

namespace anode_b200 {
namespace rows {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kMostTop = 128;
constexpr float kLog2e = 1.4426950408889634f;
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

__device__ __forceinline__ uint64_t block_max_all(uint64_t v, uint64_t *buf)
{
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) { const uint64_t w = __shfl_xor_sync(0xffffffffu, v, o); v = w > v ? w : v; }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
  __syncthreads();
  for (uint32_t i = 0; i < blockDim.x / 32; ++i) v = buf[i] > v ? buf[i] : v;
  return v;
}

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

// Any rows: a block has a row at a time, element by element: once for the largest, once for the sums, once for each of the likeliest
template <typename T> __global__ void __launch_bounds__(kThreads) token_log_probs_rows_kernel(const ProbsArgs a)
{
  __shared__ float buf[2][32];
  __shared__ uint64_t keys[kThreads / 32];
  pdl_wait();
  for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T *x = static_cast<const T *>(a.logits) + row * a.stride;
    uint64_t best = 0;
    for (uint32_t c = threadIdx.x; c < a.vocab; c += kThreads) { const uint64_t k = key_of(to_float(x[c]), c); best = k > best ? k : best; }
    best = block_max_all(best, keys);
    const float m = value_of((uint32_t)(best >> 32)), from = m == -INFINITY ? 0.0f : m;
    float sum = 0.0f, dot = 0.0f;
    for (uint32_t c = threadIdx.x; c < a.vocab; c += kThreads) {
      const float z = max_nan(a.scale * (to_float(x[c]) - from), kFloor), e = expf(z);
      sum += e;
      dot = fmaf(z, e, dot);
    }
    sum = block_sum_all(sum, buf[0]);
    dot = block_sum_all(dot, buf[1]);
    const bool empty = m == -INFINITY;
    const float log_sum = empty ? 0.0f : logf(sum);
    if (threadIdx.x == 0) {
      if (a.logprob) {
        const uint32_t t = token_at(a.token, a.token_bytes, row, a.vocab);
        a.logprob[row] = t == a.vocab ? 0.0f : empty ? m : a.scale * (to_float(x[t]) - m) - log_sum;
      }
      if (a.entropy) a.entropy[row] = empty ? 0.0f : log_sum - dot / sum;
      if (a.stats) a.stats[row] = make_float2(m, log_sum);
      if (a.top) put_top(a, row, 0, best, m, log_sum);
    }
    for (uint32_t k = 1; k < a.top; ++k) {
      uint64_t next = 0;
      for (uint32_t c = threadIdx.x; c < a.vocab; c += kThreads) { const uint64_t q = key_of(to_float(x[c]), c); if (q < best && q > next) next = q; }
      best = block_max_all(next, keys);
      if (threadIdx.x == 0) put_top(a, row, k, best, m, log_sum);
    }
    __syncthreads();
  }
}

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

}  // namespace rows
}  // namespace anode_b200

using namespace anode_b200::rows;

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
  const ProbsArgs a = {rows, vocab, scale, logits, logits_stride, token, token_bytes, logprob, entropy, reinterpret_cast<float2 *>(stats), top,
                       top ? top_logprob : nullptr, top ? top_token : nullptr, top_token_bytes};
  return by_type(type, [&](auto t) { return launch(token_log_probs_rows_kernel<decltype(t)>, dim3(row_blocks(rows)), kThreads, 0, stream, a); });
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
  return by_type(type, [&](auto t) { return launch(token_log_probs_grad_rows_kernel<decltype(t)>, dim3(row_blocks(rows)), kThreads, 0, stream, a); });
}
