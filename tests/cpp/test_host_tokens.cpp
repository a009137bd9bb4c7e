// Layer norm, rows of a table by tokens and log probabilities of tokens through the C++ host layer (anode_b200/host/anode_rows.hpp) on a GPU, against the
// formulas in double: f32 sums of up to a few hundred terms and a handful of further steps stay within 1e-5 of the largest magnitude that they are made of.
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <functional>
#include <string>
#include <vector>

#include "../../anode_b200/host/anode_ops.hpp"

using namespace anode;

static int g_checks = 0;
struct Failure { std::string what; };
#define EXPECT(cond, msg) do { ++g_checks; if (!(cond)) throw Failure{std::string(msg) + " [" #cond "]"}; } while (0)

static std::vector<float> values(size_t n, uint64_t seed, double loc = 0.0)
{
  std::vector<float> v(n);
  uint64_t s = seed * 6364136223846793005ull + 1442695040888963407ull;
  for (auto &e : v) {
    s = s * 6364136223846793005ull + 1442695040888963407ull;
    e = (float)(loc + 4.0 * ((double)(s >> 11) / 9007199254740992.0 - 0.5));
  }
  return v;
}
static void near(const std::vector<float> &got, const std::vector<double> &want, double size, const char *what)
{
  EXPECT(got.size() == want.size(), what);
  for (size_t i = 0; i < got.size(); ++i) EXPECT(std::fabs(got[i] - want[i]) <= 1e-5 * (size + std::fabs(want[i])), what);
}

constexpr uint32_t kCols = 100, kRows = 37;
constexpr double kEps = 1e-5;

static void test_layer_norm_both_ways()
{
  const size_t n = kCols * kRows;
  const auto hx = values(n, 1), hr = values(n, 2, 1.0), hg = values(kCols, 3, 1.0), hb = values(kCols, 6), hdy = values(n, 4), hdt = values(n, 5);
  DeviceArray x = DeviceArray::from_host({kCols, kRows}, hx.data()), res = DeviceArray::from_host({kCols, kRows}, hr.data());
  DeviceArray gamma = DeviceArray::from_host({kCols}, hg.data()), beta = DeviceArray::from_host({kCols}, hb.data());
  DeviceArray dy = DeviceArray::from_host({kCols, kRows}, hdy.data()), dt = DeviceArray::from_host({kCols, kRows}, hdt.data());
  DeviceArray y({kCols, kRows}), total({kCols, kRows}), mean({kRows}), inv({kRows}), dx({kCols, kRows}), dgamma({kCols}), dbeta({kCols});
  LayerNormalizeAddOp::apply((float)kEps, x, y, &gamma, &beta, &res, &total, &mean, &inv);
  RowScratch scratch(LayerNormalizeAddOp::scratch_bytes(dy));
  LayerNormalizeAddOp::adjoint(dy, total, mean, inv, dx, &gamma, &dt, &dgamma, &dbeta, WriteCap::Assign, &scratch);
  std::vector<double> wy(n), wm(kRows), wi(kRows), wdx(n), wdg(kCols, 0.0), wdb(kCols, 0.0);
  for (uint32_t r = 0; r < kRows; ++r) {
    double sum = 0.0, sq = 0.0, s = 0.0, dot = 0.0, t[kCols];
    for (uint32_t c = 0; c < kCols; ++c) { t[c] = hx[r * kCols + c] + hr[r * kCols + c]; sum += t[c]; }
    const double mu = wm[r] = sum / kCols;
    for (uint32_t c = 0; c < kCols; ++c) sq += (t[c] - mu) * (t[c] - mu);
    const double k = wi[r] = 1.0 / std::sqrt(sq / kCols + kEps);
    for (uint32_t c = 0; c < kCols; ++c) {
      const size_t i = r * kCols + c;
      const double xh = (t[c] - mu) * k, g = hdy[i] * hg[c];
      wy[i] = xh * hg[c] + hb[c]; s += g; dot += g * xh; wdg[c] += hdy[i] * xh; wdb[c] += hdy[i];
    }
    for (uint32_t c = 0; c < kCols; ++c) { const size_t i = r * kCols + c; wdx[i] = k * (hdy[i] * hg[c] - s / kCols - (t[c] - mu) * k * dot / kCols) + hdt[i]; }
  }
  near(mean.to_host(), wm, 4.0, "mean"); near(inv.to_host(), wi, 1.0, "inv_std"); near(y.to_host(), wy, 10.0, "y"); near(dx.to_host(), wdx, 20.0, "dx");
  near(dgamma.to_host(), wdg, 4.0 * kRows, "dgamma"); near(dbeta.to_host(), wdb, 4.0 * kRows, "dbeta");
  // accumulated into dx in the place of dtotal, without the weights' gradients
  DeviceArray sum = DeviceArray::from_host({kCols, kRows}, hdt.data());
  LayerNormalizeAddOp::adjoint(dy, total, mean, inv, sum, &gamma, nullptr, nullptr, nullptr, WriteCap::Accumulate, nullptr);
  near(sum.to_host(), wdx, 20.0, "accumulated dx");
}

static void test_table_both_ways()
{
  constexpr uint32_t vocab = 53, tokens = 211;
  const auto ht = values((size_t)kCols * vocab, 7), hdy = values((size_t)kCols * tokens, 8);
  std::vector<int64_t> hk(tokens);
  for (uint32_t i = 0; i < tokens; ++i) hk[i] = i % 11 == 3 ? -1 : i % 7 == 5 ? 2 : (int64_t)(i * i % (vocab + 2));      // (some outside of the table)
  const auto token = DeviceVector<int64_t>::from_host(hk);
  DeviceArray table = DeviceArray::from_host({kCols, vocab}, ht.data()), dy = DeviceArray::from_host({kCols, tokens}, hdy.data()), y({kCols, tokens}), dtable({kCols, vocab});
  EmbedTokensOp::apply(token, table, y, 2.5f);
  RowScratch scratch(EmbedTokensOp::scratch_bytes(token, dtable));
  std::vector<double> wy((size_t)kCols * tokens, 0.0), wd((size_t)kCols * vocab, 0.0);
  for (uint32_t i = 0; i < tokens; ++i) {
    if (hk[i] < 0 || hk[i] >= vocab) continue;
    for (uint32_t c = 0; c < kCols; ++c) { wy[i * kCols + c] = 2.5 * ht[hk[i] * kCols + c]; wd[hk[i] * kCols + c] += 2.5 * hdy[i * kCols + c]; }
  }
  near(y.to_host(), wy, 1.0, "rows by tokens");
  EmbedTokensOp::adjoint(token, dy, dtable, 2.5f, WriteCap::Assign, &scratch);
  near(dtable.to_host(), wd, 200.0, "the table's gradient");
  EmbedTokensOp::adjoint(token, dy, dtable, 2.5f, WriteCap::Accumulate, &scratch);
  for (auto &v : wd) v *= 2.0;
  near(dtable.to_host(), wd, 400.0, "added to itself");
}

static void test_log_probs_both_ways()
{
  constexpr uint32_t vocab = 301, top = 4;
  constexpr float scale = 1.5f;
  const auto hx = values((size_t)vocab * kRows, 9), hw = values(kRows, 10), hv = values(kRows, 11);
  std::vector<int64_t> hk(kRows);
  for (uint32_t r = 0; r < kRows; ++r) hk[r] = r % 5 == 4 ? -100 : (int64_t)(r * 17 % vocab);
  const auto token = DeviceVector<int64_t>::from_host(hk);
  DeviceArray x = DeviceArray::from_host({vocab, kRows}, hx.data()), w = DeviceArray::from_host({kRows}, hw.data()), v = DeviceArray::from_host({kRows}, hv.data());
  DeviceArray logprob({kRows}), entropy({kRows}), stats({2, kRows}), top_logprob({top, kRows}), dx({vocab, kRows});
  DeviceVector<int64_t> top_token(top * kRows);
  TokenLogProbsOp::apply(x, &token, &logprob, &entropy, &stats, top, &top_logprob, &top_token, scale);
  TokenLogProbsOp::adjoint(x, &token, stats, &entropy, &w, &v, dx, scale);
  std::vector<double> wl(kRows, 0.0), we(kRows), wt(top * kRows), wd((size_t)vocab * kRows);
  std::vector<int64_t> wk(top * kRows);
  for (uint32_t r = 0; r < kRows; ++r) {
    const float *row = hx.data() + (size_t)r * vocab;
    std::vector<int64_t> order(vocab);
    for (uint32_t c = 0; c < vocab; ++c) order[c] = c;
    std::stable_sort(order.begin(), order.end(), [&](int64_t a, int64_t b) { return row[a] > row[b]; });
    double sum = 0.0, h = 0.0;
    for (uint32_t c = 0; c < vocab; ++c) sum += std::exp(scale * (double)row[c]);
    const double whole = std::log(sum);
    auto lp = [&](int64_t c) { return scale * (double)row[c] - whole; };
    for (uint32_t c = 0; c < vocab; ++c) h -= std::exp(lp(c)) * lp(c);
    we[r] = h;
    const bool has = hk[r] >= 0;
    if (has) wl[r] = lp(hk[r]);
    for (uint32_t k = 0; k < top; ++k) { wk[r * top + k] = order[k]; wt[r * top + k] = lp(order[k]); }
    for (uint32_t c = 0; c < vocab; ++c) {
      const double p = std::exp(lp(c));
      wd[(size_t)r * vocab + c] = scale * ((has ? hw[r] * ((int64_t)c == hk[r] ? 1.0 - p : -p) : 0.0) - hv[r] * p * (lp(c) + h));
    }
  }
  near(logprob.to_host(), wl, 10.0, "log probabilities"); near(entropy.to_host(), we, 10.0, "entropies"); near(top_logprob.to_host(), wt, 10.0, "of the likeliest");
  EXPECT(top_token.to_host() == wk, "the likeliest tokens");
  near(dx.to_host(), wd, 10.0, "the logits' gradient");
}

static void test_refusals()
{
  DeviceArray x({8, 4}), y({8, 3}), ok({8, 4}), stat({4}), table({8, 5}), flat({40});
  DeviceVector<int64_t> token(4), few(3);
  auto refused = [&](const std::function<void()> &f) { try { f(); } catch (const Error &) { return true; } return false; };
  EXPECT(refused([&] { LayerNormalizeAddOp::apply(1e-5f, x, y, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr); }), "another length");
  EXPECT(refused([&] { LayerNormalizeAddOp::apply(1e-5f, x, ok, nullptr, nullptr, nullptr, &x, nullptr, nullptr); }), "a total without a residual");
  DeviceArray dgamma({8});
  EXPECT(refused([&] { LayerNormalizeAddOp::adjoint(x, x, stat, stat, ok, nullptr, nullptr, &dgamma, nullptr, WriteCap::Assign, nullptr); }), "no scratch");
  EXPECT(refused([&] { EmbedTokensOp::apply(few, table, ok, 1.0f); }), "fewer tokens than rows");
  EXPECT(refused([&] { EmbedTokensOp::apply(token, flat, ok, 1.0f); }), "a flat table");
  EXPECT(refused([&] { EmbedTokensOp::adjoint(token, x, table, 1.0f, WriteCap::Assign, nullptr); }), "no scratch for the table's gradient");
  EXPECT(refused([&] { TokenLogProbsOp::apply(x, &few, &stat, nullptr, nullptr, 0, nullptr, nullptr, 1.0f); }), "fewer tokens than rows of logits");
  EXPECT(refused([&] { TokenLogProbsOp::apply(x, &token, &stat, nullptr, nullptr, 0, nullptr, nullptr, 0.0f); }), "a scale of 0");
  EXPECT(refused([&] { TokenLogProbsOp::adjoint(x, &token, table, nullptr, &stat, nullptr, ok, 1.0f); }), "stats of another length");
}

int main()
{
  int devs = 0;
  if (cudaGetDeviceCount(&devs) != cudaSuccess || devs == 0) { fprintf(stderr, "no CUDA device\n"); return 2; }
  const std::pair<const char *, std::function<void()>> tests[] = {{"layer_norm_both_ways", test_layer_norm_both_ways}, {"table_both_ways", test_table_both_ways},
                                                                  {"log_probs_both_ways", test_log_probs_both_ways}, {"refusals", test_refusals}};
  int failed = 0;
  for (const auto &t : tests) {
    try { t.second(); printf("ok   %s\n", t.first); }
    catch (const Failure &f) { printf("FAIL %s: %s\n", t.first, f.what.c_str()); ++failed; }
    catch (const std::exception &e) { printf("FAIL %s: exception %s\n", t.first, e.what()); ++failed; }
  }
  printf("%d checks, %d tests failed\n", g_checks, failed);
  return failed ? 1 : 0;
}
