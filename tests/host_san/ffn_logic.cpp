// Host side of the feed-forward entry points over the stub HIP runtime under AddressSanitizer and
// UndefinedBehaviorSanitizer: every refusal with its status and no launch, then a walk of accepted shapes, layouts and
// types (launch arithmetic, growth of the repack area).  Kernels do not run.
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <vector>

#include "sbamd_ffn.h"

extern "C" long hip_stub_launches();
extern "C" long hip_stub_live_allocations();

static int g_failed = 0;
#define EXPECT(cond)                                                                      \
  do {                                                                                    \
    if (!(cond)) {                                                                        \
      std::fprintf(stderr, "%s:%d: expectation failed: %s\n", __FILE__, __LINE__, #cond); \
      ++g_failed;                                                                         \
    }                                                                                     \
  } while (0)

// `call` is refused with `status` and launches nothing
#define REFUSED(status, call)                 \
  do {                                        \
    const long before = hip_stub_launches();  \
    EXPECT((call) == (status));               \
    EXPECT(hip_stub_launches() == before);    \
  } while (0)

int main() {
  sbamd_handle_t h = nullptr;
  EXPECT(sbamd_create(&h, 0, nullptr) == SBAMD_OK);
  void* room = nullptr;
  EXPECT(sbamd_malloc(h, &room, size_t(64) << 20) == SBAMD_OK);
  auto* f = static_cast<float*>(room);
  auto* u = static_cast<uint16_t*>(room);
  auto* q = static_cast<int8_t*>(room);
  const int64_t far = int64_t(1) << 41;

  // ---- leading dimensions whose matrices no address space holds
  const int64_t huge = int64_t(1) << 62;
  REFUSED(SBAMD_INVALID_VALUE, sbamd_squantize_i8(h, 4, 4, f, huge, q, 4, f));
  REFUSED(SBAMD_INVALID_VALUE, sbamd_squantize_i8(h, 4, 4, f, 4, q, huge, f));
  REFUSED(SBAMD_INVALID_VALUE, sbamd_i8sgemm(h, 't', 'n', 4, 4, 4, 1, q, huge, f, q, 4, f, 0, f, 4));
  REFUSED(SBAMD_INVALID_VALUE, sbamd_i8sgemm(h, 't', 'n', 4, 4, 4, 1, q, 4, f, q, huge, f, 0, f, 4));
  REFUSED(SBAMD_INVALID_VALUE, sbamd_i8sgemm(h, 't', 'n', 4, 4, 4, 1, q, 4, f, q, 4, f, 0, f, huge));
  REFUSED(SBAMD_INVALID_VALUE, sbamd_i8sgemm(h, 't', 'n', 4, 4, 4, 0, q, 4, f, q, 4, f, 0, f, huge));
  REFUSED(SBAMD_INVALID_VALUE, sbamd_bgated_gemm(h, SBAMD_ACT_SILU, 't', 'n', 4, 4, 4, u, 4, u, 4, u, 4, u, huge));
  REFUSED(SBAMD_INVALID_VALUE, sbamd_bgated_gemm_grad(h, SBAMD_ACT_SILU, 't', 'n', 4, 4, 4, u, 4, u, 4, u, 8, u, huge, u, 8, 0, u, 4, 0, u, 4));
  REFUSED(SBAMD_INVALID_VALUE, sbamd_bgated_gemm_grad(h, SBAMD_ACT_SILU, 't', 'n', 4, 4, 4, u, huge, u, 4, u, 8, u, 4, u, 8, 0, u, 4, 0, u, 4));

  // ---- quantisation
  REFUSED(SBAMD_INVALID_HANDLE, sbamd_squantize_i8(nullptr, 4, 4, f, 4, q, 4, f));
  REFUSED(SBAMD_INVALID_VALUE, sbamd_squantize_i8(h, -1, 4, f, 4, q, 4, f));
  REFUSED(SBAMD_INVALID_VALUE, sbamd_hquantize_i8(h, 4, -1, u, 4, q, 4, f));
  REFUSED(SBAMD_INVALID_VALUE, sbamd_bquantize_i8(h, 4, 4, u, 3, q, 4, f));
  REFUSED(SBAMD_INVALID_VALUE, sbamd_bquantize_i8(h, 4, 4, u, 4, q, 3, f));
  REFUSED(SBAMD_INVALID_VALUE, sbamd_bquantize_i8(h, 4, 4, u, 4, q, 4, nullptr));
  REFUSED(SBAMD_INVALID_VALUE, sbamd_bquantize_i8(h, 4, 4, nullptr, 4, q, 4, f));
  REFUSED(SBAMD_INVALID_VALUE, sbamd_bquantize_i8(h, 4, 4, u, 4, nullptr, 4, f));
  REFUSED(SBAMD_OK, sbamd_bquantize_i8(h, 4, 0, nullptr, 4, nullptr, 4, nullptr));
  for (int64_t m : {0, 1, 512, 513, 4096, 4097, 20000}) {
    EXPECT(sbamd_squantize_i8(h, m, 3, f, m, q, m, f) == SBAMD_OK);
    EXPECT(sbamd_hquantize_i8(h, m, 3, u, m + 1, q, m + 3, f) == SBAMD_OK);
    EXPECT(sbamd_bquantize_i8(h, m, 70000, u, m, q, m, f) == SBAMD_OK);
  }

  // ---- scaled product
  REFUSED(SBAMD_INVALID_HANDLE, sbamd_i8sgemm(nullptr, 't', 'n', 4, 4, 4, 1, q, 4, f, q, 4, f, 0, f, 4));
  REFUSED(SBAMD_INVALID_TRANSA, sbamd_i8sgemm(h, 'x', 'n', 4, 4, 4, 1, q, 4, f, q, 4, f, 0, f, 4));
  REFUSED(SBAMD_INVALID_TRANSB, sbamd_i8hgemm(h, 't', 'x', 4, 4, 4, 1, q, 4, f, q, 4, f, 0, u, 4));
  REFUSED(SBAMD_INVALID_VALUE, sbamd_i8bgemm(h, 't', 'n', -4, 4, 4, 1, q, 4, f, q, 4, f, 0, u, 4));
  REFUSED(SBAMD_INVALID_VALUE, sbamd_i8bgemm(h, 't', 'n', far, 4, 4, 1, q, 4, f, q, 4, f, 0, u, far));
  REFUSED(SBAMD_INVALID_VALUE, sbamd_i8bgemm(h, 't', 'n', 4, 4, 4, 1, q, 3, f, q, 4, f, 0, u, 4));
  REFUSED(SBAMD_INVALID_VALUE, sbamd_i8bgemm(h, 'n', 'n', 5, 4, 4, 1, q, 4, f, q, 4, f, 0, u, 5));
  REFUSED(SBAMD_INVALID_VALUE, sbamd_i8bgemm(h, 't', 'n', 4, 4, 4, 1, q, 4, f, q, 3, f, 0, u, 4));
  REFUSED(SBAMD_INVALID_VALUE, sbamd_i8bgemm(h, 't', 't', 4, 5, 4, 1, q, 4, f, q, 4, f, 0, u, 4));
  REFUSED(SBAMD_INVALID_VALUE, sbamd_i8bgemm(h, 't', 'n', 4, 4, 4, 1, q, 4, f, q, 4, f, 0, u, 3));
  REFUSED(SBAMD_INVALID_VALUE, sbamd_i8sgemm(h, 't', 'n', 4, 4, 4, 1, nullptr, 4, f, q, 4, f, 0, f, 4));
  REFUSED(SBAMD_INVALID_VALUE, sbamd_i8sgemm(h, 't', 'n', 4, 4, 4, 1, q, 4, f, nullptr, 4, f, 0, f, 4));
  REFUSED(SBAMD_INVALID_VALUE, sbamd_i8sgemm(h, 't', 'n', 4, 4, 4, 1, q, 4, f, q, 4, f, 0, nullptr, 4));
  REFUSED(SBAMD_NOT_SUPPORTED, sbamd_i8sgemm(h, 't', 'n', 4, 4, SBAMD_I8_MAX_K + 1, 1, q, SBAMD_I8_MAX_K + 1, f, q, SBAMD_I8_MAX_K + 1, f, 0, f, 4));
  REFUSED(SBAMD_OK, sbamd_i8sgemm(h, 't', 'n', 0, 4, 4, 1, q, 4, f, q, 4, f, 0, f, 0));
  REFUSED(SBAMD_OK, sbamd_i8sgemm(h, 't', 'n', 4, 0, 4, 1, q, 4, f, q, 4, f, 0, f, 4));
  // alpha == 0 comes before everything that reads A or B, as in GEMM
  EXPECT(sbamd_i8sgemm(h, 'x', 'x', 4, 4, 4, 0, nullptr, 4, nullptr, nullptr, 4, nullptr, 2, f, 4) == SBAMD_OK);
  EXPECT(sbamd_i8bgemm(h, 'x', 'x', 4, 4, 4, 0, nullptr, 4, nullptr, nullptr, 4, nullptr, 0, u, 4) == SBAMD_OK);
  REFUSED(SBAMD_OK, sbamd_i8hgemm(h, 'x', 'x', 4, 4, 4, 0, nullptr, 4, nullptr, nullptr, 4, nullptr, 1, u, 4));
  REFUSED(SBAMD_INVALID_VALUE, sbamd_i8hgemm(h, 'x', 'x', 4, 4, 4, 0, nullptr, 4, nullptr, nullptr, 4, nullptr, 2, nullptr, 4));

  // ---- gated block
  REFUSED(SBAMD_INVALID_HANDLE, sbamd_bgated_gemm(nullptr, SBAMD_ACT_SILU, 't', 'n', 4, 4, 4, u, 4, u, 4, u, 4, nullptr, 0));
  REFUSED(SBAMD_INVALID_VALUE, sbamd_bgated_gemm(h, -1, 't', 'n', 4, 4, 4, u, 4, u, 4, u, 4, nullptr, 0));
  REFUSED(SBAMD_INVALID_VALUE, sbamd_bgated_gemm(h, 4, 't', 'n', 4, 4, 4, u, 4, u, 4, u, 4, nullptr, 0));
  REFUSED(SBAMD_INVALID_TRANSA, sbamd_hgated_gemm(h, SBAMD_ACT_SILU, 'q', 'n', 4, 4, 4, u, 4, u, 4, u, 4, nullptr, 0));
  REFUSED(SBAMD_INVALID_TRANSB, sbamd_hgated_gemm(h, SBAMD_ACT_SILU, 'n', 'q', 4, 4, 4, u, 8, u, 4, u, 4, nullptr, 0));
  REFUSED(SBAMD_INVALID_VALUE, sbamd_hgated_gemm(h, SBAMD_ACT_SILU, 'n', 'n', 4, 4, 4, u, 7, u, 4, u, 4, nullptr, 0));  // op(A) has 2m rows
  REFUSED(SBAMD_INVALID_VALUE, sbamd_hgated_gemm(h, SBAMD_ACT_SILU, 't', 'n', 4, 4, 4, u, 4, u, 4, u, 4, u, 7));        // P has 2m rows
  REFUSED(SBAMD_INVALID_VALUE, sbamd_hgated_gemm(h, SBAMD_ACT_SILU, 't', 'n', 4, 4, 4, u, 4, u, 4, nullptr, 4, nullptr, 0));
  REFUSED(SBAMD_INVALID_VALUE, sbamd_i8hgated_gemm(h, 9, 't', 'n', 4, 4, 4, q, 4, f, q, 4, f, u, 4));
  REFUSED(SBAMD_NOT_SUPPORTED, sbamd_i8hgated_gemm(h, SBAMD_ACT_GELU, 't', 'n', 4, 4, SBAMD_I8_MAX_K + 1, q, SBAMD_I8_MAX_K + 1, f, q, SBAMD_I8_MAX_K + 1, f, u, 4));
  REFUSED(SBAMD_OK, sbamd_bgated_gemm(h, SBAMD_ACT_RELU, 't', 'n', 0, 4, 4, u, 4, u, 4, u, 0, nullptr, 0));

  // ---- gradient
#define GRAD(...) sbamd_bgated_gemm_grad(h, __VA_ARGS__)
  REFUSED(SBAMD_INVALID_HANDLE, sbamd_bgated_gemm_grad(nullptr, SBAMD_ACT_SILU, 't', 'n', 4, 4, 4, u, 4, u, 4, u, 8, u, 4, u, 8, 0, u, 4, 0, u, 4));
  REFUSED(SBAMD_INVALID_VALUE, GRAD(7, 't', 'n', 4, 4, 4, u, 4, u, 4, u, 8, u, 4, u, 8, 0, u, 4, 0, u, 4));
  REFUSED(SBAMD_INVALID_TRANSA, GRAD(SBAMD_ACT_SILU, 'q', 'n', 4, 4, 4, u, 4, u, 4, u, 8, u, 4, u, 8, 0, u, 4, 0, u, 4));
  REFUSED(SBAMD_INVALID_TRANSB, GRAD(SBAMD_ACT_SILU, 't', 'q', 4, 4, 4, u, 4, u, 4, u, 8, u, 4, u, 8, 0, u, 4, 0, u, 4));
  REFUSED(SBAMD_INVALID_VALUE, GRAD(SBAMD_ACT_SILU, 't', 'n', 4, 4, 4, u, 4, u, 4, u, 7, u, 4, u, 8, 0, u, 4, 0, u, 4));   // ldp
  REFUSED(SBAMD_INVALID_VALUE, GRAD(SBAMD_ACT_SILU, 't', 'n', 4, 4, 4, u, 4, u, 4, u, 8, u, 3, u, 8, 0, u, 4, 0, u, 4));   // lddc
  REFUSED(SBAMD_INVALID_VALUE, GRAD(SBAMD_ACT_SILU, 't', 'n', 4, 4, 4, u, 4, u, 4, u, 8, u, 4, u + 9, 7, 0, u, 4, 0, u, 4));  // lddp
  REFUSED(SBAMD_INVALID_VALUE, GRAD(SBAMD_ACT_SILU, 't', 'n', 4, 4, 4, u, 4, u, 4, u, 8, u, 4, u, 9, 0, u, 4, 0, u, 4));   // in place, other ld
  REFUSED(SBAMD_INVALID_VALUE, GRAD(SBAMD_ACT_SILU, 't', 'n', 4, 4, 4, u, 4, u, 4, u, 8, u, 4, u, 8, 0, u, 3, 0, u, 4));   // ldda
  REFUSED(SBAMD_INVALID_VALUE, GRAD(SBAMD_ACT_SILU, 't', 'n', 4, 4, 4, u, 4, u, 4, u, 8, u, 4, u, 8, 0, u, 4, 0, u, 3));   // lddb
  REFUSED(SBAMD_INVALID_VALUE, GRAD(SBAMD_ACT_SILU, 't', 'n', 4, 4, 4, u, 4, u, 3, u, 8, u, 4, u, 8, 0, u, 4, 0, u, 4));   // ldb, needed for dA
  REFUSED(SBAMD_INVALID_VALUE, GRAD(SBAMD_ACT_SILU, 't', 'n', 4, 4, 4, u, 3, u, 4, u, 8, u, 4, u, 8, 0, u, 4, 0, u, 4));   // lda, needed for dB
  REFUSED(SBAMD_INVALID_VALUE, GRAD(SBAMD_ACT_SILU, 't', 'n', 4, 4, 4, u, 4, u, 4, nullptr, 8, u, 4, u, 8, 0, u, 4, 0, u, 4));
  REFUSED(SBAMD_INVALID_VALUE, GRAD(SBAMD_ACT_SILU, 't', 'n', 4, 4, 4, u, 4, u, 4, u, 8, nullptr, 4, u, 8, 0, u, 4, 0, u, 4));
  REFUSED(SBAMD_INVALID_VALUE, GRAD(SBAMD_ACT_SILU, 't', 'n', 4, 4, 4, u, 4, u, 4, u, 8, u, 4, nullptr, 8, 0, u, 4, 0, u, 4));
  REFUSED(SBAMD_INVALID_VALUE, GRAD(SBAMD_ACT_SILU, 't', 'n', 4, 4, 4, u, 4, nullptr, 4, u, 8, u, 4, u, 8, 0, u, 4, 0, nullptr, 4));
  REFUSED(SBAMD_INVALID_VALUE, GRAD(SBAMD_ACT_SILU, 't', 'n', 4, 4, 4, nullptr, 4, u, 4, u, 8, u, 4, u, 8, 0, nullptr, 4, 0, u, 4));
  // one gradient alone needs the other operand only
  EXPECT(GRAD(SBAMD_ACT_SILU, 't', 'n', 4, 4, 4, nullptr, 0, u, 4, u, 8, u, 4, u, 8, 0, u, 4, 0, nullptr, 0) == SBAMD_OK);
  EXPECT(GRAD(SBAMD_ACT_SILU, 't', 'n', 4, 4, 4, u, 4, nullptr, 0, u, 8, u, 4, u, 8, 0, nullptr, 0, 0, u, 4) == SBAMD_OK);
  EXPECT(GRAD(SBAMD_ACT_SILU, 't', 'n', 4, 4, 4, nullptr, 0, nullptr, 0, u, 8, u, 4, u, 8, 0, nullptr, 0, 0, nullptr, 0) == SBAMD_OK);
  // no tokens, no channels, no k
  EXPECT(GRAD(SBAMD_ACT_SILU, 't', 'n', 4, 0, 4, u, 4, u, 4, nullptr, 8, nullptr, 4, nullptr, 8, 1, u, 4, 0, u, 4) == SBAMD_OK);
  EXPECT(GRAD(SBAMD_ACT_SILU, 't', 'n', 0, 4, 4, u, 4, u, 4, nullptr, 0, nullptr, 0, nullptr, 0, 0, u, 4, 1, u, 4) == SBAMD_OK);
  EXPECT(GRAD(SBAMD_ACT_SILU, 't', 'n', 4, 4, 0, nullptr, 0, nullptr, 0, u, 8, u, 4, u, 8, 0, u, 0, 0, u, 0) == SBAMD_OK);

  // ---- a walk of accepted calls
  long walked = 0;
  for (int64_t m : {1, 16, 17, 130, 1000})
    for (int64_t n : {1, 16, 33, 70, 300})
      for (int64_t k : {0, 1, 31, 128, 1001})
        for (char ta : {'n', 't'})
          for (char tb : {'n', 'c'}) {
            const int64_t la = ta == 'n' ? m : k, la2 = ta == 'n' ? 2 * m : k, lb = tb == 'n' ? k : n;
            EXPECT(sbamd_i8sgemm(h, ta, tb, m, n, k, 1, q, la, f, q, lb, nullptr, 1, f, m) == SBAMD_OK);
            EXPECT(sbamd_i8bgated_gemm(h, SBAMD_ACT_GELU, ta, tb, m, n, k, q, la2, nullptr, q, lb, f, u, m) == SBAMD_OK);
            EXPECT(sbamd_hgated_gemm(h, SBAMD_ACT_GELU_TANH, ta, tb, m, n, k, u, la2 + 3, u, lb, u, m, u, 2 * m) == SBAMD_OK);
            EXPECT(sbamd_hgated_gemm_grad(h, SBAMD_ACT_RELU, ta, tb, m, n, k, u, la2, u, lb, u, 2 * m, u, m, u, 2 * m, 0, u, la2, 1, u, lb) == SBAMD_OK);
            EXPECT(sbamd_bgated_gemm_grad(h, SBAMD_ACT_SILU, ta, tb, m, n, k, u, la2, u, lb, u, 2 * m, u, m, u, 2 * m, 1, u, la2, 0, u, lb) == SBAMD_OK);
            ++walked;
          }
  EXPECT(sbamd_free(h, room) == SBAMD_OK);
  EXPECT(sbamd_destroy(h) == SBAMD_OK);
  EXPECT(hip_stub_live_allocations() == 0);
  std::printf("%ld accepted walks, %ld launches, %d expectations failed\n", walked, hip_stub_launches(), g_failed);
  return g_failed ? 1 : 0;
}
