// Normalization over rows and rotary positions through the C++ host layer (anode_b200/host/anode_rows.hpp) on a GPU, against the formulas in
// double: f32 sums of a hundred terms and a handful of further steps stay within 1e-5 of the largest magnitude that they are made of.
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

static void test_norm_both_ways()
{
  const auto hx = values(kCols * kRows, 1), hr = values(kCols * kRows, 2), hg = values(kCols, 3, 1.0), hdy = values(kCols * kRows, 4), hdt = values(kCols * kRows, 5);
  DeviceArray x = DeviceArray::from_host({kCols, kRows}, hx.data()), res = DeviceArray::from_host({kCols, kRows}, hr.data());
  DeviceArray gamma = DeviceArray::from_host({kCols}, hg.data()), dy = DeviceArray::from_host({kCols, kRows}, hdy.data()), dt = DeviceArray::from_host({kCols, kRows}, hdt.data());
  DeviceArray y({kCols, kRows}), total({kCols, kRows}), inv({kRows}), dx({kCols, kRows}), dgamma({kCols});
  RmsNormalizeAddOp::apply((float)kEps, x, y, &gamma, &res, &total, &inv);
  RowScratch scratch(RmsNormalizeAddOp::scratch_bytes(dy));
  RmsNormalizeAddOp::adjoint(dy, total, inv, dx, &gamma, &dt, &dgamma, WriteCap::Assign, &scratch);
  std::vector<double> wy(kCols * kRows), wt(kCols * kRows), wi(kRows), wdx(kCols * kRows), wdg(kCols, 0.0);
  for (uint32_t r = 0; r < kRows; ++r) {
    double sq = 0.0, dot = 0.0;
    for (uint32_t c = 0; c < kCols; ++c) { const size_t i = r * kCols + c; wt[i] = hx[i] + hr[i]; sq += wt[i] * wt[i]; }
    const double k = wi[r] = 1.0 / std::sqrt(sq / kCols + kEps);
    for (uint32_t c = 0; c < kCols; ++c) { const size_t i = r * kCols + c; wy[i] = wt[i] * k * hg[c]; dot += hdy[i] * hg[c] * wt[i] * k; }
    for (uint32_t c = 0; c < kCols; ++c) {
      const size_t i = r * kCols + c;
      wdx[i] = k * (hdy[i] * hg[c] - wt[i] * k * dot / kCols) + hdt[i];
      wdg[c] += hdy[i] * wt[i] * k;
    }
  }
  near(total.to_host(), wt, 4.0, "total"); near(inv.to_host(), wi, 1.0, "inv_rms"); near(y.to_host(), wy, 4.0, "y");
  near(dx.to_host(), wdx, 20.0, "dx"); near(dgamma.to_host(), wdg, 4.0 * kRows, "dgamma");
  // accumulated into dx in the place of dtotal
  DeviceArray sum = DeviceArray::from_host({kCols, kRows}, hdt.data());
  RmsNormalizeAddOp::adjoint(dy, total, inv, sum, &gamma, nullptr, nullptr, WriteCap::Accumulate, nullptr);
  near(sum.to_host(), wdx, 20.0, "accumulated dx");
}

static void test_eight_bits()
{
  const auto hx = values(300 * 5, 7);
  DeviceArray x = DeviceArray::from_host({300, 5}, hx.data()), scale({3, 5});
  DeviceVector<uint8_t> q(300 * 5);
  RmsNormalizeAddQuantOp::apply((float)kEps, 128, x, q, scale, nullptr, nullptr, nullptr);
  const auto hq = q.to_host();
  const auto hs = scale.to_host();
  for (int r = 0; r < 5; ++r) {
    double sq = 0.0;
    for (int c = 0; c < 300; ++c) sq += (double)hx[r * 300 + c] * hx[r * 300 + c];
    const double k = 1.0 / std::sqrt(sq / 300 + kEps);
    for (int g = 0; g < 3; ++g) {
      double top = 0.0;
      for (int c = g * 128; c < 300 && c < g * 128 + 128; ++c) top = std::fmax(top, std::fabs(hx[r * 300 + c] * k));
      EXPECT(std::fabs(hs[r * 3 + g] * 448.0 - top) <= 1e-5 * top, "scale");
    }
    for (int c = 0; c < 300; ++c) {
      const uint8_t b = hq[r * 300 + c];
      const int e = b >> 3 & 15, m = b & 7;
      const double v = (b & 128 ? -1.0 : 1.0) * (e ? std::ldexp(8 + m, e - 10) : std::ldexp(m, -9)), want = hx[r * 300 + c] * k / hs[r * 3 + c / 128];
      EXPECT(std::fabs(v - want) <= std::fmax(std::ldexp(std::fabs(want), -4), std::ldexp(1.0, -10)) * 1.0001, "value in 8 bits");
    }
  }
}

static void test_rotary_both_ways()
{
  constexpr uint32_t dim = 24, rot = 16, heads = 3, keys = 2, tokens = 11;
  RotaryPositionsOp::Form form;
  form.interleaved = true; form.norm = true; form.amplitude = 1.25f;
  std::vector<int64_t> hp(tokens);
  std::vector<double> hf(rot / 2);
  for (uint32_t t = 0; t < tokens; ++t) hp[t] = 100000 + 7 * t;
  for (uint32_t i = 0; i < rot / 2; ++i) hf[i] = std::pow(10000.0, -2.0 * i / rot);
  const auto positions = DeviceVector<int64_t>::from_host(hp);
  const auto freq = DeviceVector<double>::from_host(hf);
  const auto hg = values(dim, 5, 1.0);
  DeviceArray gamma = DeviceArray::from_host({dim}, hg.data());
  const uint32_t n[2] = {heads, keys};
  std::vector<float> hx[2], hd[2];
  DeviceArray x[2], y[2], d[2], dx[2], dg[2];
  for (int k = 0; k < 2; ++k) {
    hx[k] = values(dim * n[k] * tokens, 10 + k); hd[k] = values(dim * n[k] * tokens, 20 + k);
    x[k] = DeviceArray::from_host({dim, n[k], tokens}, hx[k].data()); d[k] = DeviceArray::from_host({dim, n[k], tokens}, hd[k].data());
    y[k] = DeviceArray({dim, n[k], tokens}); dx[k] = DeviceArray({dim, n[k], tokens}); dg[k] = DeviceArray({dim});
  }
  RotaryPositionsOp::apply(form, positions, freq, x[0], &x[1], y[0], &y[1], &gamma, &gamma);
  RowScratch scratch(RotaryPositionsOp::scratch_bytes(d[0], &d[1]));
  RotaryPositionsOp::adjoint(form, positions, freq, d[0], &d[1], dx[0], &dx[1], &x[0], &x[1], &gamma, &gamma, &dg[0], &dg[1], &scratch);
  for (int k = 0; k < 2; ++k) {
    std::vector<double> wy(hx[k].size()), wdx(hx[k].size()), wdg(dim, 0.0);
    for (uint32_t t = 0; t < tokens; ++t)
      for (uint32_t h = 0; h < n[k]; ++h) {
        const size_t o = ((size_t)t * n[k] + h) * dim;
        double sq = 0.0, dot = 0.0, v[dim], w[dim];
        for (uint32_t i = 0; i < dim; ++i) sq += (double)hx[k][o + i] * hx[k][o + i];
        const double r = 1.0 / std::sqrt(sq / dim + form.epsilon);
        for (uint32_t i = 0; i < dim; ++i) { v[i] = hx[k][o + i] * r * hg[i]; w[i] = hd[k][o + i]; }
        for (uint32_t i = 0; i < rot / 2; ++i) {
          const double c = form.amplitude * std::cos(hp[t] * hf[i]), s = form.amplitude * std::sin(hp[t] * hf[i]);
          const double a = v[2 * i], b = v[2 * i + 1], p = w[2 * i], q = w[2 * i + 1];
          v[2 * i] = a * c - b * s; v[2 * i + 1] = a * s + b * c;
          w[2 * i] = p * c + q * s; w[2 * i + 1] = q * c - p * s;
        }
        for (uint32_t i = 0; i < dim; ++i) { wy[o + i] = v[i]; dot += w[i] * hg[i] * hx[k][o + i] * r; wdg[i] += w[i] * hx[k][o + i] * r; }
        for (uint32_t i = 0; i < dim; ++i) wdx[o + i] = r * (w[i] * hg[i] - hx[k][o + i] * r * dot / dim);
      }
    near(y[k].to_host(), wy, 8.0, "turned heads"); near(dx[k].to_host(), wdx, 30.0, "their gradient"); near(dg[k].to_host(), wdg, 8.0 * tokens * n[k], "the weight's gradient");
  }
}

static void test_refusals()
{
  DeviceArray x({8, 4}), y({8, 3}), ok({8, 4}), inv({4});
  auto refused = [&](const std::function<void()> &f) { try { f(); } catch (const Error &) { return true; } return false; };
  EXPECT(refused([&] { RmsNormalizeAddOp::apply(1e-5f, x, y, nullptr, nullptr, nullptr, nullptr); }), "another length");
  EXPECT(refused([&] { RmsNormalizeAddOp::apply(1e-5f, x, ok, nullptr, nullptr, &x, nullptr); }), "a total without a residual");
  DeviceArray dgamma({8});
  EXPECT(refused([&] { RmsNormalizeAddOp::adjoint(x, x, inv, ok, nullptr, nullptr, &dgamma, WriteCap::Assign, nullptr); }), "no scratch");
}

int main()
{
  int devs = 0;
  if (cudaGetDeviceCount(&devs) != cudaSuccess || devs == 0) { fprintf(stderr, "no CUDA device\n"); return 2; }
  const std::pair<const char *, std::function<void()>> tests[] = {
      {"norm_both_ways", test_norm_both_ways}, {"eight_bits", test_eight_bits}, {"rotary_both_ways", test_rotary_both_ways}, {"refusals", test_refusals}};
  int failed = 0;
  for (const auto &t : tests) {
    try { t.second(); printf("ok   %s\n", t.first); }
    catch (const Failure &f) { printf("FAIL %s: %s\n", t.first, f.what.c_str()); ++failed; }
    catch (const std::exception &e) { printf("FAIL %s: exception %s\n", t.first, e.what()); ++failed; }
  }
  printf("%d checks, %d tests failed\n", g_checks, failed);
  return failed ? 1 : 0;
}
