// What the C++ host layer of rows and heads (anode_b200/host/anode_rows.hpp) refuses before it asks anything of a device.  Device memory is host memory here:
// the program has its own cudaMalloc and cudaFree, so that it runs on any machine, and every call below has to end in an anode::Error.
#include <cstdio>
#include <cstdlib>
#include <functional>
#include <string>
#include <vector>

#include "../../anode_b200/host/anode_ops.hpp"

extern "C" cudaError_t cudaMalloc(void **p, size_t n) { return (*p = malloc(n)) ? cudaSuccess : cudaErrorMemoryAllocation; }
extern "C" cudaError_t cudaFree(void *p) { free(p); return cudaSuccess; }

using namespace anode;

static int g_failed = 0;
static void refused(const char *what, int code, const std::function<void()> &call)
{
  try { call(); }
  catch (const Error &e) {
    if (e.code == code) { printf("ok   %s\n", what); return; }
    printf("FAIL %s: %s\n", what, e.what()); ++g_failed; return;
  }
  printf("FAIL %s: not refused\n", what); ++g_failed;
}

int main(int argc, char **argv)
{
  const std::string which = argc > 1 ? argv[1] : "";
  constexpr uint32_t dim = 8, heads = 3, keys = 2, tokens = 5;
  RotaryPositionsOp::Form plain, norm;
  norm.norm = true;
  const DeviceVector<int64_t> positions(tokens);
  const DeviceVector<double> freq(dim / 2);
  DeviceArray q({dim, heads, tokens}), k({dim, keys, tokens}), qo({dim, heads, tokens}), ko({dim, keys, tokens});
  const auto forward = [&](const DeviceArray *k, DeviceArray &qo, DeviceArray *ko) { RotaryPositionsOp::apply(plain, positions, freq, q, k, qo, ko, nullptr, nullptr); };
  const auto back = [&](const RotaryPositionsOp::Form &f, const DeviceArray *dko, DeviceArray &dq, DeviceArray *dk, const DeviceArray *x, const DeviceArray *z) {
    RotaryPositionsOp::adjoint(f, positions, freq, q, dko, dq, dk, x, z, nullptr, nullptr, nullptr, nullptr, nullptr);
  };
  if (which == "missing") {
    refused("keys without k_out", ANODE_E_NULL, [&] { forward(&k, qo, nullptr); });
    refused("k_out without keys", ANODE_E_NULL, [&] { forward(nullptr, qo, &ko); });
    refused("dk_out without dk", ANODE_E_NULL, [&] { back(plain, &k, qo, nullptr, nullptr, nullptr); });
    refused("dk without dk_out", ANODE_E_NULL, [&] { back(plain, nullptr, qo, &ko, nullptr, nullptr); });
    refused("a norm without q", ANODE_E_NULL, [&] { back(norm, &k, qo, &ko, nullptr, &k); });
    refused("a norm without k", ANODE_E_NULL, [&] { back(norm, &k, qo, &ko, &q, nullptr); });
  } else if (which == "shapes") {
    // of the right length, but not [dim, heads, tokens]
    DeviceArray flat({dim * heads * tokens}), flat_keys({dim * keys * tokens}), turned({heads, dim, tokens}), other({dim, tokens, heads});
    refused("a flat q_out", ANODE_E_DIMS, [&] { forward(&k, flat, &ko); });
    refused("a flat k_out", ANODE_E_DIMS, [&] { forward(&k, qo, &flat_keys); });
    refused("q_out as [heads, dim, tokens]", ANODE_E_DIMS, [&] { forward(&k, turned, &ko); });
    refused("q_out as [dim, tokens, heads]", ANODE_E_DIMS, [&] { forward(&k, other, &ko); });
    refused("a flat dq", ANODE_E_DIMS, [&] { back(plain, &k, flat, &ko, nullptr, nullptr); });
    refused("a flat dk", ANODE_E_DIMS, [&] { back(plain, &k, qo, &flat_keys, nullptr, nullptr); });
    refused("a flat q of the norm", ANODE_E_DIMS, [&] { back(norm, &k, qo, &ko, &flat, &k); });
    refused("a flat k of the norm", ANODE_E_DIMS, [&] { back(norm, &k, qo, &ko, &q, &flat_keys); });
    refused("scratch for flat queries", ANODE_E_DIMS, [&] { (void)RotaryPositionsOp::scratch_bytes(flat, nullptr); });
    refused("scratch for flat keys", ANODE_E_DIMS, [&] { (void)RotaryPositionsOp::scratch_bytes(q, &flat_keys); });
  } else { fprintf(stderr, "missing | shapes\n"); return 2; }
  printf("%d failed\n", g_failed);
  return g_failed ? 1 : 0;
}
