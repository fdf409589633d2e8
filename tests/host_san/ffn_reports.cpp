// What sbamd_last_kernel and sbamd_last_splitk report after the feed-forward entry points, over the stub HIP runtime: both
// have to describe the same product, also where one of a gradient's two products was cut along k and the other was not.
#include <cstdint>
#include <cstdio>

#include "sbamd_ffn.h"

static int g_failed = 0;

static void reports(sbamd_handle_t h, const char* what, bool cut, int64_t k, bool ring = true) {
  int64_t depth = 0, chunk = 0;
  const int kernel = sbamd_last_kernel(h);
  sbamd_last_splitk(h, &depth, &chunk);
  const bool right = cut ? depth > 1 && chunk < k && depth * chunk >= k && (depth - 1) * chunk < k : depth == 1 && chunk == k;
  if (!right || kernel < 0 || (ring && kernel != SBAMD_KERNEL_LARGE)) {
    std::fprintf(stderr, "%s: kernel %d, %lld slabs of %lld, sum of %lld\n", what, kernel, (long long)depth, (long long)chunk, (long long)k);
    ++g_failed;
  }
}

int main() {
  sbamd_handle_t h = nullptr;
  if (sbamd_create(&h, 0, nullptr) != SBAMD_OK) return 1;
  void* room = nullptr;
  if (sbamd_malloc(h, &room, 4096) != SBAMD_OK) return 1;
  auto* u = static_cast<uint16_t*>(room);
  sbamd_set_kernel(h, SBAMD_KERNEL_LARGE, 0);
  auto gradient = [&](int64_t m, int64_t n, int64_t k, bool a, bool b, int64_t pad_w = 0) {
    uint16_t* da = a ? u : nullptr;
    uint16_t* db = b ? u : nullptr;
    if (sbamd_bgated_gemm_grad(h, SBAMD_ACT_SILU, 't', 'n', m, n, k, u, k + pad_w, u, k, u, 2 * m, u, m, u, 2 * m, 0, da, k, 0, db, k) != SBAMD_OK) ++g_failed;
  };
  // dA sums over the tokens, dB over the 2m rows of P
  gradient(128, 4096, 128, true, false);
  reports(h, "dA cut, alone", true, 4096);
  gradient(128, 4096, 128, false, true);
  reports(h, "dB whole, alone", false, 256);
  gradient(128, 4096, 128, true, true);
  reports(h, "dA cut, dB whole", false, 256);
  gradient(2048, 256, 128, true, true);
  reports(h, "dA whole, dB cut", true, 4096);
  gradient(128, 4096, 128, true, true);
  gradient(128, 256, 128, false, true);
  reports(h, "dB whole after another call", false, 256);
  gradient(128, 4096, 128, true, true, 1);  // rows of A at odd addresses: dB runs on the 16-bit GEMM
  reports(h, "dA cut, dB elsewhere", false, 256, false);
  if (sbamd_free(h, room) != SBAMD_OK || sbamd_destroy(h) != SBAMD_OK) return 1;
  std::printf("%d reports wrong\n", g_failed);
  return g_failed ? 1 : 0;
}
