// Normalization over rows, rotary positions, rows of a table by tokens and log probabilities of tokens on top of anode_ops.hpp (included from there): f32 arrays, sizes fastest-varying first, so
// rows are [cols, rows...] and heads [dim, heads, tokens].  No counterpart in the reference.
#pragma once

namespace anode {

// Device memory of a type other than f32 (positions, frequencies, values in 8 bits, scratch)
template <typename T> class DeviceVector {
 public:
  DeviceVector() = default;
  explicit DeviceVector(size_t n) : len_(n) { cuda_check(cudaMalloc(&ptr_, n ? n * sizeof(T) : 1), "cudaMalloc"); }
  static DeviceVector from_host(const std::vector<T> &h, cudaStream_t s = 0)
  {
    DeviceVector v(h.size());
    cuda_check(cudaMemcpyAsync(v.ptr_, h.data(), h.size() * sizeof(T), cudaMemcpyHostToDevice, s), "cudaMemcpyAsync");
    cuda_check(cudaStreamSynchronize(s), "cudaStreamSynchronize");
    return v;
  }
  std::vector<T> to_host(cudaStream_t s = 0) const
  {
    std::vector<T> h(len_);
    cuda_check(cudaMemcpyAsync(h.data(), ptr_, len_ * sizeof(T), cudaMemcpyDeviceToHost, s), "cudaMemcpyAsync");
    cuda_check(cudaStreamSynchronize(s), "cudaStreamSynchronize");
    return h;
  }
  DeviceVector(DeviceVector &&o) noexcept { *this = std::move(o); }
  DeviceVector &operator=(DeviceVector &&o) noexcept
  {
    if (this != &o) { if (ptr_) (void)cudaFree(ptr_); ptr_ = o.ptr_; len_ = o.len_; o.ptr_ = nullptr; o.len_ = 0; }
    return *this;
  }
  DeviceVector(const DeviceVector &) = delete;
  DeviceVector &operator=(const DeviceVector &) = delete;
  ~DeviceVector() { if (ptr_) (void)cudaFree(ptr_); }
  T *ptr() { return ptr_; }
  const T *ptr() const { return ptr_; }
  size_t len() const { return len_; }
  size_t bytes() const { return len_ * sizeof(T); }

 private:
  T *ptr_ = nullptr;
  size_t len_ = 0;
};
using RowScratch = DeviceVector<unsigned char>;

// [cols, rows...]
struct RowDims { uint32_t cols; uint64_t rows; };
inline RowDims row_dims(const DeviceArray &x)
{
  if (x.size().empty() || x.size()[0] == 0) throw Error(ANODE_E_DIMS, "array of rows needs [cols, rows...]");
  return RowDims{x.size()[0], x.len() / x.size()[0]};
}
inline void want_opt(const DeviceArray *a, size_t n, const char *what) { if (a && !a->empty()) want_len(*a, n, what); }

// y = total*r*gamma with total = x + residual, r = (mean(total^2) + epsilon)^-1/2 per row; gamma, residual, total, inv_rms may be null
struct RmsNormalizeAddOp {
  static void apply(float epsilon, const DeviceArray &x, DeviceArray &y, const DeviceArray *gamma, const DeviceArray *residual, DeviceArray *total,
                    DeviceArray *inv_rms, cudaStream_t s = 0)
  {
    const RowDims d = row_dims(x);
    want_len(y, x.len(), "y"); want_opt(gamma, d.cols, "gamma"); want_opt(residual, x.len(), "residual"); want_opt(total, x.len(), "total");
    want_opt(inv_rms, d.rows, "inv_rms");
    check(anode_gpu_rms_norm_add_fwd(ANODE_TYPE_F32, d.rows, d.cols, epsilon, x.ptr(), d.cols, opt(residual), d.cols, opt(gamma), ANODE_TYPE_F32, y.ptr(),
                                     d.cols, opt(total), d.cols, opt(inv_rms), kernel_config(), raw(s)), "anode_gpu_rms_norm_add_fwd");
  }
  static size_t scratch_bytes(const DeviceArray &dy) { const RowDims d = row_dims(dy); return anode_gpu_rms_norm_add_bwd_workspace_bytes(d.rows, d.cols); }
  // the gradient of x and of the residual; with Accumulate it is added to dx, which then takes the place of dtotal
  static void adjoint(const DeviceArray &dy, const DeviceArray &total, const DeviceArray &inv_rms, DeviceArray &dx, const DeviceArray *gamma,
                      const DeviceArray *dtotal, DeviceArray *dgamma, WriteCap cap, RowScratch *scratch, cudaStream_t s = 0)
  {
    const RowDims d = row_dims(dy);
    const bool adds = cap == WriteCap::Accumulate;
    if (adds && dtotal && !dtotal->empty()) throw Error(ANODE_E_DIMS, "Accumulate adds into dx, which takes the place of dtotal");
    want_len(total, dy.len(), "total"); want_len(dx, dy.len(), "dx"); want_len(inv_rms, d.rows, "inv_rms");
    want_opt(gamma, d.cols, "gamma"); want_opt(dtotal, dy.len(), "dtotal"); want_opt(dgamma, d.cols, "dgamma");
    check(anode_gpu_rms_norm_add_bwd(ANODE_TYPE_F32, d.rows, d.cols, dy.ptr(), d.cols, total.ptr(), d.cols, inv_rms.ptr(), opt(gamma), ANODE_TYPE_F32,
                                     adds ? dx.ptr() : opt(dtotal), d.cols, dx.ptr(), d.cols, opt(dgamma), scratch ? scratch->ptr() : nullptr,
                                     scratch ? scratch->bytes() : 0, kernel_config(), raw(s)), "anode_gpu_rms_norm_add_bwd");
  }
};

// The same with its output in e4m3 and a scale per row (block 0: [rows]) or per 128 columns (block 128: [groups, rows])
struct RmsNormalizeAddQuantOp {
  static void apply(float epsilon, uint32_t block, const DeviceArray &x, DeviceVector<uint8_t> &q, DeviceArray &scale, const DeviceArray *gamma,
                    const DeviceArray *residual, DeviceArray *total, cudaStream_t s = 0)
  {
    const RowDims d = row_dims(x);
    const uint64_t groups = block ? (d.cols + 127ull) / 128 : 1;
    if (q.len() != x.len()) throw Error(ANODE_E_DIMS, "q: wrong length");
    want_len(scale, d.rows * groups, "scale"); want_opt(gamma, d.cols, "gamma"); want_opt(residual, x.len(), "residual"); want_opt(total, x.len(), "total");
    check(anode_gpu_rms_norm_add_quant_fwd(ANODE_TYPE_F32, d.rows, d.cols, epsilon, block, x.ptr(), d.cols, opt(residual), d.cols, opt(gamma), ANODE_TYPE_F32,
                                           q.ptr(), d.cols, scale.ptr(), groups, 1, opt(total), d.cols, kernel_config(), raw(s)),
          "anode_gpu_rms_norm_add_quant_fwd");
  }
};

// Rotary positions of [dim, heads, tokens] arrays, after the norm of each head where `norm`; keys may be null
struct RotaryPositionsOp {
  struct Form { bool interleaved = false, norm = false; float amplitude = 1.0f, epsilon = 1e-5f; };

  static void apply(const Form &f, const DeviceVector<int64_t> &positions, const DeviceVector<double> &freq, const DeviceArray &q, const DeviceArray *k,
                    DeviceArray &q_out, DeviceArray *k_out, const DeviceArray *gamma_q, const DeviceArray *gamma_k, cudaStream_t s = 0)
  {
    const Shape d = shape(q, k, positions);
    if (!k != !k_out) throw Error(ANODE_E_NULL, "k and k_out are given together");
    want_heads(q_out, q, "q_out"); if (k) want_heads(*k_out, *k, "k_out");
    want_opt(gamma_q, d.dim, "gamma_q"); want_opt(gamma_k, d.dim, "gamma_k");
    const AnodeHeads a = heads(q), b = k ? heads(*k) : AnodeHeads{}, ao = heads(q_out), bo = k ? heads(*k_out) : AnodeHeads{};
    check(anode_gpu_rotary_positions_fwd(ANODE_TYPE_F32, 1, d.tokens, d.dim, 2 * (uint32_t)freq.len(), f.interleaved, f.amplitude, freq.ptr(), positions.ptr(), 8,
                                         0, 1, f.norm, f.epsilon, opt(gamma_q), opt(gamma_k), ANODE_TYPE_F32, &a, k ? &b : nullptr, &ao, k ? &bo : nullptr,
                                         kernel_config(), raw(s)), "anode_gpu_rotary_positions_fwd");
  }
  static size_t scratch_bytes(const DeviceArray &q, const DeviceArray *k)
  {
    if (q.size().size() != 3 || (k && k->size().size() != 3)) throw Error(ANODE_E_DIMS, "heads need [dim, heads, tokens]");
    return anode_gpu_rotary_positions_bwd_workspace_bytes(1, q.size()[2], q.size()[1], k ? k->size()[1] : 0, q.size()[0]);
  }
  // q and k (the forward pass's inputs) are read where there is a norm
  static void adjoint(const Form &f, const DeviceVector<int64_t> &positions, const DeviceVector<double> &freq, const DeviceArray &dq_out,
                      const DeviceArray *dk_out, DeviceArray &dq, DeviceArray *dk, const DeviceArray *q, const DeviceArray *k, const DeviceArray *gamma_q,
                      const DeviceArray *gamma_k, DeviceArray *dgamma_q, DeviceArray *dgamma_k, RowScratch *scratch, cudaStream_t s = 0)
  {
    const Shape d = shape(dq_out, dk_out, positions);
    if (!dk_out != !dk) throw Error(ANODE_E_NULL, "dk_out and dk are given together");
    want_heads(dq, dq_out, "dq"); if (dk_out) want_heads(*dk, *dk_out, "dk");
    if (f.norm) { if (!q || (dk_out && !k)) throw Error(ANODE_E_NULL, "q, k"); want_heads(*q, dq_out, "q"); if (dk_out) want_heads(*k, *dk_out, "k"); }
    want_opt(gamma_q, d.dim, "gamma_q"); want_opt(gamma_k, d.dim, "gamma_k"); want_opt(dgamma_q, d.dim, "dgamma_q"); want_opt(dgamma_k, d.dim, "dgamma_k");
    const AnodeHeads a = heads(dq_out), b = dk_out ? heads(*dk_out) : AnodeHeads{}, ao = heads(dq), bo = dk_out ? heads(*dk) : AnodeHeads{};
    const AnodeHeads x = f.norm ? heads(*q) : AnodeHeads{}, z = f.norm && dk_out ? heads(*k) : AnodeHeads{};
    check(anode_gpu_rotary_positions_bwd(ANODE_TYPE_F32, 1, d.tokens, d.dim, 2 * (uint32_t)freq.len(), f.interleaved, f.amplitude, freq.ptr(), positions.ptr(), 8,
                                         0, 1, f.norm, f.epsilon, opt(gamma_q), opt(gamma_k), ANODE_TYPE_F32, &a, dk_out ? &b : nullptr, f.norm ? &x : nullptr,
                                         f.norm && dk_out ? &z : nullptr, &ao, dk_out ? &bo : nullptr, opt(dgamma_q), opt(dgamma_k),
                                         scratch ? scratch->ptr() : nullptr, scratch ? scratch->bytes() : 0, kernel_config(), raw(s)),
          "anode_gpu_rotary_positions_bwd");
  }

 private:
  struct Shape { uint32_t dim, tokens; };
  static Shape shape(const DeviceArray &q, const DeviceArray *k, const DeviceVector<int64_t> &positions)
  {
    if (q.size().size() != 3 || (k && (k->size().size() != 3 || k->size()[0] != q.size()[0] || k->size()[2] != q.size()[2])))
      throw Error(ANODE_E_DIMS, "heads need [dim, heads, tokens] of one dim and one number of tokens");
    if (positions.len() != q.size()[2]) throw Error(ANODE_E_DIMS, "positions: one per token");
    return Shape{q.size()[0], q.size()[2]};
  }
  // heads of `like`'s sizes, the tokens behind them in as many dimensions as they please
  static void want_heads(const DeviceArray &a, const DeviceArray &like, const char *what)
  {
    want_len(a, like.len(), what);
    if (a.size().size() < 2 || a.size()[0] != like.size()[0] || a.size()[1] != like.size()[1]) throw Error(ANODE_E_DIMS, std::string(what) + ": expected [dim, heads, tokens]");
  }
  static AnodeHeads heads(const DeviceArray &x)
  {
    const uint64_t dim = x.size()[0], n = x.size()[1];
    return AnodeHeads{const_cast<float *>(x.ptr()), 0, dim * n, dim, (uint32_t)n};
  }
};

// y = (total - mu)*r*gamma + beta with total = x + residual, mu its mean and r = (mean((total - mu)^2) + epsilon)^-1/2 per row; gamma, beta, residual, total,
// mean, inv_std may be null
struct LayerNormalizeAddOp {
  static void apply(float epsilon, const DeviceArray &x, DeviceArray &y, const DeviceArray *gamma, const DeviceArray *beta, const DeviceArray *residual,
                    DeviceArray *total, DeviceArray *mean, DeviceArray *inv_std, cudaStream_t s = 0)
  {
    const RowDims d = row_dims(x);
    want_len(y, x.len(), "y"); want_opt(gamma, d.cols, "gamma"); want_opt(beta, d.cols, "beta"); want_opt(residual, x.len(), "residual");
    want_opt(total, x.len(), "total"); want_opt(mean, d.rows, "mean"); want_opt(inv_std, d.rows, "inv_std");
    check(anode_gpu_layer_norm_add_fwd(ANODE_TYPE_F32, d.rows, d.cols, epsilon, x.ptr(), d.cols, opt(residual), d.cols, opt(gamma), opt(beta), ANODE_TYPE_F32,
                                       y.ptr(), d.cols, opt(total), d.cols, opt(mean), opt(inv_std), kernel_config(), raw(s)), "anode_gpu_layer_norm_add_fwd");
  }
  static size_t scratch_bytes(const DeviceArray &dy) { const RowDims d = row_dims(dy); return anode_gpu_layer_norm_add_bwd_workspace_bytes(d.rows, d.cols); }
  // the gradient of x and of the residual; with Accumulate it is added to dx, which then takes the place of dtotal
  static void adjoint(const DeviceArray &dy, const DeviceArray &total, const DeviceArray &mean, const DeviceArray &inv_std, DeviceArray &dx, const DeviceArray *gamma,
                      const DeviceArray *dtotal, DeviceArray *dgamma, DeviceArray *dbeta, WriteCap cap, RowScratch *scratch, cudaStream_t s = 0)
  {
    const RowDims d = row_dims(dy);
    const bool adds = cap == WriteCap::Accumulate;
    if (adds && dtotal && !dtotal->empty()) throw Error(ANODE_E_DIMS, "Accumulate adds into dx, which takes the place of dtotal");
    want_len(total, dy.len(), "total"); want_len(dx, dy.len(), "dx"); want_len(mean, d.rows, "mean"); want_len(inv_std, d.rows, "inv_std");
    want_opt(gamma, d.cols, "gamma"); want_opt(dtotal, dy.len(), "dtotal"); want_opt(dgamma, d.cols, "dgamma"); want_opt(dbeta, d.cols, "dbeta");
    check(anode_gpu_layer_norm_add_bwd(ANODE_TYPE_F32, d.rows, d.cols, dy.ptr(), d.cols, total.ptr(), d.cols, mean.ptr(), inv_std.ptr(), opt(gamma), ANODE_TYPE_F32,
                                       adds ? dx.ptr() : opt(dtotal), d.cols, dx.ptr(), d.cols, opt(dgamma), opt(dbeta), scratch ? scratch->ptr() : nullptr,
                                       scratch ? scratch->bytes() : 0, kernel_config(), raw(s)), "anode_gpu_layer_norm_add_bwd");
  }
};

// y[i] = scale*table[token[i]]: a table of [cols, vocab], y of [cols, tokens...]; a token outside of the table has a row of zeros and no gradient
struct EmbedTokensOp {
  static void apply(const DeviceVector<int64_t> &token, const DeviceArray &table, DeviceArray &y, float scale, cudaStream_t s = 0)
  {
    const uint32_t vocab = rows_of(table);
    want_rows(y, table, token.len(), "y");
    check(anode_gpu_embed_tokens_fwd(ANODE_TYPE_F32, token.len(), vocab, table.size()[0], scale, token.ptr(), 8, table.ptr(), table.size()[0], y.ptr(),
                                     table.size()[0], kernel_config(), raw(s)), "anode_gpu_embed_tokens_fwd");
  }
  static size_t scratch_bytes(const DeviceVector<int64_t> &token, const DeviceArray &table)
  {
    return anode_gpu_embed_tokens_bwd_workspace_bytes(token.len(), rows_of(table), table.size()[0]);
  }
  // the whole table's gradient; with Accumulate what the tokens add to it
  static void adjoint(const DeviceVector<int64_t> &token, const DeviceArray &dy, DeviceArray &dtable, float scale, WriteCap cap, RowScratch *scratch, cudaStream_t s = 0)
  {
    const uint32_t vocab = rows_of(dtable);
    want_rows(dy, dtable, token.len(), "dy");
    check(anode_gpu_embed_tokens_bwd(ANODE_TYPE_F32, token.len(), vocab, dtable.size()[0], scale, token.ptr(), 8, dy.ptr(), dtable.size()[0], dtable.ptr(),
                                     dtable.size()[0], ANODE_TYPE_F32, cap == WriteCap::Accumulate, scratch ? scratch->ptr() : nullptr,
                                     scratch ? scratch->bytes() : 0, kernel_config(), raw(s)), "anode_gpu_embed_tokens_bwd");
  }

 private:
  static uint32_t rows_of(const DeviceArray &table)
  {
    if (table.size().size() != 2) throw Error(ANODE_E_DIMS, "a table needs [cols, vocab]");
    return table.size()[1];
  }
  static void want_rows(const DeviceArray &rows, const DeviceArray &table, size_t n, const char *what)
  {
    want_len(rows, n * table.size()[0], what);
    if (rows.size().empty() || rows.size()[0] != table.size()[0]) throw Error(ANODE_E_DIMS, std::string(what) + ": expected [cols, tokens...] of the table's columns");
  }
};

// Log probabilities of tokens at a temperature of 1/scale: logits of [vocab, rows...], a token, a log probability and an entropy per row, stats of [2, rows...] for
// the adjoint, the likeliest `top` tokens and their log probabilities of [top, rows...]; what is null is not computed
struct TokenLogProbsOp {
  static void apply(const DeviceArray &logits, const DeviceVector<int64_t> *token, DeviceArray *logprob, DeviceArray *entropy, DeviceArray *stats, uint32_t top,
                    DeviceArray *top_logprob, DeviceVector<int64_t> *top_token, float scale, cudaStream_t s = 0)
  {
    const RowDims d = row_dims(logits);
    want_tokens(token, d.rows);
    want_opt(logprob, d.rows, "logprob"); want_opt(entropy, d.rows, "entropy"); want_opt(stats, 2 * d.rows, "stats"); want_opt(top_logprob, top * d.rows, "top_logprob");
    if (top_token && top_token->len() != top * d.rows) throw Error(ANODE_E_DIMS, "top_token: wrong length");
    check(anode_gpu_token_log_probs_fwd(ANODE_TYPE_F32, d.rows, d.cols, scale, logits.ptr(), d.cols, token ? token->ptr() : nullptr, 8, opt(logprob), opt(entropy),
                                        opt(stats), top, opt(top_logprob), top_token ? top_token->ptr() : nullptr, 8, kernel_config(), raw(s)),
          "anode_gpu_token_log_probs_fwd");
  }
  // dlogits may be logits
  static void adjoint(const DeviceArray &logits, const DeviceVector<int64_t> *token, const DeviceArray &stats, const DeviceArray *entropy, const DeviceArray *dlogprob,
                      const DeviceArray *dentropy, DeviceArray &dlogits, float scale, cudaStream_t s = 0)
  {
    const RowDims d = row_dims(logits);
    want_tokens(token, d.rows);
    want_len(stats, 2 * d.rows, "stats"); want_len(dlogits, logits.len(), "dlogits");
    want_opt(entropy, d.rows, "entropy"); want_opt(dlogprob, d.rows, "dlogprob"); want_opt(dentropy, d.rows, "dentropy");
    check(anode_gpu_token_log_probs_bwd(ANODE_TYPE_F32, d.rows, d.cols, scale, logits.ptr(), d.cols, token ? token->ptr() : nullptr, 8, stats.ptr(), opt(entropy),
                                        opt(dlogprob), opt(dentropy), dlogits.ptr(), d.cols, kernel_config(), raw(s)), "anode_gpu_token_log_probs_bwd");
  }

 private:
  static void want_tokens(const DeviceVector<int64_t> *token, uint64_t rows)
  {
    if (token && token->len() != rows) throw Error(ANODE_E_DIMS, "token: one per row");
  }
};

}  // namespace anode
