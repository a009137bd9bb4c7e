// Rotary positions of queries and keys, with the RMS norm of each head before them: forward and adjoint.
//
//   n = x*r*gamma, r = (mean(x^2) + epsilon)^-1/2 over the head;   angle = position*freq[i]
//   (n[u], n[v]) -> A*(n[u] cos - n[v] sin, n[u] sin + n[v] cos);   backward: the same with -sin, then the norm's adjoint
//
// A warp has a head of a token at a time; statistics are f32, angles f64.
#include "bn_host.h"
#include "rows.cuh"

namespace anode_b200 {
namespace rows {

constexpr uint32_t kThreads = 256, kWarps = kThreads / 32, kMostDim = 1024;

struct HeadArray {
  void *p;
  uint64_t batch, seq, head;
};
struct RotaryArgs {
  uint32_t batch, seq, dim, rot, interleaved;
  float amplitude, epsilon, inv_dim;
  const double *freq;
  const void *positions;
  uint32_t position_bytes;
  uint64_t pos_batch, pos_seq;
  uint32_t norm, q_heads, heads;       // heads: of q and k
  Weights gamma[2];
  HeadArray in[2], x[2], out[2];       // backward: in = dout, x = the norm's input, out = dx
  float *partial;                      // [blocks, 2, dim] of the gradients of the weights
  uint32_t blocks, want[2];
};

__device__ __forceinline__ double position_of(const RotaryArgs &a, uint32_t b, uint32_t s)
{
  const uint64_t i = b * a.pos_batch + s * a.pos_seq;
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

template <typename T, bool BWD> __global__ void __launch_bounds__(kThreads) rotary_heads_kernel(const RotaryArgs a)
{
  extern __shared__ float sums[];            // [warps][2][dim] where gradients of weights are wanted
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, half = a.rot / 2;
  float *mine = sums + (size_t)warp * 2 * a.dim;
  const bool wants = BWD && (a.want[0] || a.want[1]);
  if (wants) for (uint32_t i = lane; i < 2 * a.dim; i += 32) mine[i] = 0.0f;
  __syncwarp();
  pdl_wait();
  const uint64_t units = (uint64_t)a.batch * a.seq * a.heads;
  for (uint64_t u = (uint64_t)blockIdx.x * kWarps + warp; u < units; u += (uint64_t)gridDim.x * kWarps) {
    const uint64_t token = u / a.heads;
    const uint32_t h = (uint32_t)(u - token * a.heads), b = (uint32_t)(token / a.seq), s = (uint32_t)(token - (uint64_t)b * a.seq);
    const uint32_t which = h >= a.q_heads, head = which ? h - a.q_heads : h;
    auto at = [&](const HeadArray &x) { return static_cast<T *>(x.p) + b * x.batch + s * x.seq + head * x.head; };
    const T *in = at(a.in[which]), *x = a.norm ? at(BWD ? a.x[which] : a.in[which]) : nullptr;
    T *out = at(a.out[which]);
    const Weights gamma = a.gamma[which];
    const double position = position_of(a, b, s);
    float r = 1.0f, dot = 0.0f;
    if (a.norm) {
      float sq = 0.0f;
      for (uint32_t d = lane; d < a.dim; d += 32) { const float v = to_float(x[d]); sq = fmaf(v, v, sq); }
      r = 1.0f / sqrtf(warp_sum_all(sq) * a.inv_dim + a.epsilon);
    }
    // pairs first, then what passes
    auto each = [&](auto f) {
      for (uint32_t i = lane; i < half; i += 32) {
        const uint32_t d = a.interleaved ? 2 * i : i, e = a.interleaved ? d + 1 : i + half;
        const float2 cs = turn_of(position, a.freq[i], a.amplitude);
        const float p = to_float(in[d]), q = to_float(in[e]);
        if (BWD) {
          f(d, p * cs.x + q * cs.y); f(e, q * cs.x - p * cs.y);
        } else {
          const float m = a.norm ? p * r * gamma.at(d) : p, n = a.norm ? q * r * gamma.at(e) : q;
          f(d, m * cs.x - n * cs.y); f(e, m * cs.y + n * cs.x);
        }
      }
      for (uint32_t d = a.rot + lane; d < a.dim; d += 32) {
        const float p = to_float(in[d]);
        f(d, BWD || !a.norm ? p : p * r * gamma.at(d));
      }
    };
    if (BWD && a.norm) {
      each([&](uint32_t d, float dn) { dot = fmaf(dn * gamma.at(d), to_float(x[d]) * r, dot); });
      dot = warp_sum_all(dot) * a.inv_dim;
      each([&](uint32_t d, float dn) {
        const float xh = to_float(x[d]) * r;
        out[d] = from_float<T>(r * (dn * gamma.at(d) - xh * dot));
        if (wants) mine[which * a.dim + d] += dn * xh;
      });
    } else {
      each([&](uint32_t d, float v) { out[d] = from_float<T>(v); });
    }
    __syncwarp();
  }
  if (wants) {
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < 2 * a.dim; i += kThreads) {
      float sum = 0.0f;
      for (uint32_t w = 0; w < kWarps; ++w) sum += sums[(size_t)w * 2 * a.dim + i];
      a.partial[(uint64_t)blockIdx.x * 2 * a.dim + i] = sum;
    }
  }
}

__global__ void __launch_bounds__(kThreads) rotary_join_kernel(uint32_t dim, uint32_t blocks, const float *partial, void *dq, void *dk, int type)
{
  pdl_wait();
  const uint32_t i = blockIdx.x * kThreads + threadIdx.x;
  if (i >= 2 * dim) return;
  void *out = i < dim ? dq : dk;
  if (!out) return;
  float sum = 0.0f;
  for (uint32_t b = 0; b < blocks; ++b) sum += partial[(uint64_t)b * 2 * dim + i];
  put_weight(out, type, i < dim ? i : i - dim, sum);
}

inline uint32_t head_blocks(uint64_t units)
{
  const uint64_t most = 148 * 8, need = (units + kWarps - 1) / kWarps;
  return (uint32_t)(need < most ? need : most);
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
  if ((a.gamma[0].p || a.gamma[1].p || wants) && !known_type(c.gamma_type)) return ANODE_E_TYPE;
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
    if (!aligned_to(a.gamma[k].p, ge) || !aligned_to(c.dgamma[k], ge)) return ANODE_E_ALIGN;
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
    put(a.in[k], c.in[k]);
    put(a.out[k], c.out[k]);
    if (c.bwd && a.norm) {
      TRY(check_heads(c.x[k], e, a.batch, a.seq, a.dim, false));
      if (!same_place(c.out[k], c.x[k], a.batch, a.seq)) return ANODE_E_STRIDE;
      put(a.x[k], c.x[k]);
    }
  }
  a.q_heads = c.in[0]->heads;
  a.heads = a.q_heads + (two ? c.in[1]->heads : 0);
  a.blocks = head_blocks((uint64_t)a.batch * a.seq * a.heads);
  a.partial = static_cast<float *>(c.workspace);
  a.want[0] = c.dgamma[0] != nullptr; a.want[1] = c.dgamma[1] != nullptr;
  if (wants && (!c.workspace || !aligned_to(c.workspace, 16) ||
                c.workspace_bytes < anode_gpu_rotary_positions_bwd_workspace_bytes(a.batch, a.seq, a.q_heads, a.heads - a.q_heads, a.dim)))
    return ANODE_E_WORKSPACE;
  const size_t shared = wants ? (size_t)kWarps * 2 * a.dim * 4 : 0;
  TRY(by_type(c.type, [&](auto t) {
    using T = decltype(t);
    if (!c.bwd) return launch(rotary_heads_kernel<T, false>, dim3(a.blocks), kThreads, 0, stream, a);
    if (shared > 48 * 1024 && cudaFuncSetAttribute(rotary_heads_kernel<T, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)shared) != cudaSuccess)
      return (int)ANODE_E_LAUNCH;
    return launch(rotary_heads_kernel<T, true>, dim3(a.blocks), kThreads, shared, stream, a);
  }));
  if (!wants) return ANODE_OK;
  return launch(rotary_join_kernel, dim3((2 * a.dim + kThreads - 1) / kThreads), kThreads, 0, stream, a.dim, a.blocks, a.partial, c.dgamma[0], c.dgamma[1],
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
                  pos_batch_stride, pos_seq_stride, norm != 0, 0, 0, {{gamma_q, gamma_type}, {gamma_k, gamma_type}}, {}, {}, {}, nullptr, 0, {}};
  return rotary(a, RotaryCall{type, gamma_type, position_bytes, false, {q, k}, {}, {q_out, k_out}, {}, nullptr, 0}, stream);
}

extern "C" size_t anode_gpu_rotary_positions_bwd_workspace_bytes(uint32_t batch, uint32_t seq, uint32_t q_heads, uint32_t k_heads, uint32_t dim)
{
  return (size_t)head_blocks((uint64_t)batch * seq * (q_heads + (uint64_t)k_heads)) * 2 * dim * 4;
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
                  pos_batch_stride, pos_seq_stride, norm != 0, 0, 0, {{gamma_q, gamma_type}, {gamma_k, gamma_type}}, {}, {}, {}, nullptr, 0, {}};
  return rotary(a, RotaryCall{type, gamma_type, position_bytes, true, {dq_out, dk_out}, {q, k}, {dq, dk}, {dgamma_q, dgamma_k}, workspace, workspace_bytes},
                stream);
}
