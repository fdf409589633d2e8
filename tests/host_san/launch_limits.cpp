// Launches of very many workgroups over the stub HIP runtime: HIP refuses a launch of 2^32 or more threads along one axis, so a
// call whose sizes the card's memory holds must not ask for one.  Every size is taken just below and above the place
// where one workgroup per item would reach it.  Kernels do not run, and no operand exists behind the pointers.
#include <cstdint>
#include <cstdio>
#include <functional>

#include "sbamd_ffn.h"

extern "C" long hip_stub_launches();
extern "C" uint64_t hip_stub_widest_launch();

static int g_failed = 0;

// `call` is accepted and none of its launches is too wide
static void fits(const char* what, int64_t size, const std::function<int()>& call) {
  const long before = hip_stub_launches();
  const int status = call();
  const uint64_t widest = hip_stub_widest_launch();
  if (status != SBAMD_OK || widest >= (uint64_t(1) << 32) || hip_stub_launches() == before) {
    std::fprintf(stderr, "%s at %lld: status %d, %ld launches, the widest of %llu threads\n", what, (long long)size, status, hip_stub_launches() - before,
                 (unsigned long long)widest);
    ++g_failed;
  }
}

int main() {
  sbamd_handle_t h = nullptr;
  if (sbamd_create(&h, 0, nullptr) != SBAMD_OK) return 1;
  void* room = nullptr;
  if (sbamd_malloc(h, &room, 4096) != SBAMD_OK) return 1;
  auto* f = static_cast<float*>(room);
  auto* d = static_cast<double*>(room);
  auto* u = static_cast<uint16_t*>(room);
  auto* q = static_cast<int8_t*>(room);
  const int64_t around[] = {-1, 0, 1, 12345};

  // quantisation: 4 columns a workgroup of 256 up to 512 rows, a workgroup of 256 up to 4096, one of 1024 beyond
  struct {
    int64_t m, n;
  } columns[] = {{1, int64_t(1) << 26}, {512, int64_t(1) << 26}, {513, int64_t(1) << 24}, {4096, int64_t(1) << 24}, {4097, int64_t(1) << 22}};
  for (auto c : columns)
    for (int64_t e : around) {
      const int64_t n = c.n + e;
      fits("quantise bfloat16", n, [&] { return sbamd_bquantize_i8(h, c.m, n, u, c.m, q, c.m, f); });
      fits("quantise half", n, [&] { return sbamd_hquantize_i8(h, c.m, n, u, c.m, q, c.m, f); });
      fits("quantise float", n, [&] { return sbamd_squantize_i8(h, c.m, n, f, c.m, q, c.m, f); });
    }
  // C <- beta C, an element per thread
  for (int64_t e : around) {
    const int64_t n = (int64_t(1) << 30) + e, m = 4;
    fits("scaled float, alpha 0", n, [&] { return sbamd_i8sgemm(h, 't', 'n', m, n, 8, 0, q, 8, f, q, 8, f, 2, f, m); });
    fits("scaled half, alpha 0", n, [&] { return sbamd_i8hgemm(h, 't', 'n', m, n, 8, 0, q, 8, f, q, 8, f, 2, u, m); });
    fits("scaled bfloat16, alpha 0", n, [&] { return sbamd_i8bgemm(h, 't', 'n', m, n, 8, 0, q, 8, f, q, 8, f, 2, u, m); });
    fits("sgemm, alpha 0", n, [&] { return sbamd_sgemm(h, 't', 'n', m, n, 8, 0, f, 8, f, 8, 2, f, m); });
    fits("dgemm, alpha 0", n, [&] { return sbamd_dgemm(h, 't', 'n', m, n, 8, 0, d, 8, d, 8, 2, d, m); });
    fits("hgemm, alpha 0", n, [&] { return sbamd_hgemm(h, 't', 'n', m, n, 8, 0, u, 8, u, 8, 2, u, m); });
  }
  // the narrow kernel: 64 tokens by 32 channels, or 16 of the gated block, a workgroup of 256
  sbamd_set_kernel(h, SBAMD_KERNEL_SMALL, 0);
  for (int64_t e : around) {
    const int64_t n = (int64_t(1) << 30) + e, m = (int64_t(1) << 28) + e;
    fits("scaled product, many tokens", n, [&] { return sbamd_i8hgemm(h, 't', 'n', 1, n, 1, 1, q, 1, f, q, 1, f, 0, u, 1); });
    fits("gated block, many tokens", n, [&] { return sbamd_bgated_gemm(h, SBAMD_ACT_SILU, 't', 'n', 1, n, 1, u, 1, u, 1, u, 1, u, 2); });
    fits("gated block, many channels", m, [&] { return sbamd_bgated_gemm(h, SBAMD_ACT_SILU, 't', 'n', m, 1, 1, u, 1, u, 1, u, m, u, 2 * m); });
    fits("sum over nothing, many tokens", n, [&] { return sbamd_i8sgemm(h, 't', 'n', 1, n, 0, 1, q, 0, f, q, 0, f, 1, f, 1); });
  }
  sbamd_set_kernel(h, SBAMD_KERNEL_AUTO, 0);
  // the elementwise half of the gradient: eight channels of a token per thread
  for (int64_t e : around) {
    const int64_t n = (int64_t(1) << 32) + e;
    fits("gradient of P", n, [&] { return sbamd_bgated_gemm_grad(h, SBAMD_ACT_SILU, 't', 'n', 1, n, 1, nullptr, 0, nullptr, 0, u, 2, u, 1, u, 2, 0, nullptr, 0, 0, nullptr, 0); });
    fits("gradient and its products", n / 4, [&] { return sbamd_bgated_gemm_grad(h, SBAMD_ACT_SILU, 't', 'n', 8, n / 4, 8, u, 8, u, 8, u, 16, u, 8, u, 16, 0, u, 8, 0, u, 8); });
  }
  if (sbamd_free(h, room) != SBAMD_OK || sbamd_destroy(h) != SBAMD_OK) return 1;
  std::printf("%ld launches, %d calls failed\n", hip_stub_launches(), g_failed);
  return g_failed ? 1 : 0;
}
