/*
 * sbamd_ffn.h -- the feed-forward layers of language models on the GEMM engine:
 * products of 8-bit integers with a scale per token and per channel, the
 * quantisation that makes such operands, and the gated block (two projections
 * of one input, an activation, a product) in one kernel, with its gradient.
 *
 * Conventions are those of sbamd_gemm.h: column-major matrices, device pointers,
 * 64-bit sizes, calls asynchronous on the handle's stream, an int status, nothing
 * throws.  "Token" and "channel" are the columns of op(B) and the rows of op(A): a
 * row-major activation tensor [tokens, k] is the k x tokens matrix B ('n', ldb = k),
 * a row-major weight [channels, k] is op(A) with transa 't' and lda = k.  That pair of
 * layouts (both operands contiguous along k) is the one the kernels read in place;
 * the other transposes work too, some of them through a repacked copy of the
 * operand in the handle's own scratch area.
 *
 * Scratch and graphs: repacked operands and products cut along k use scratch areas of the handle, which grow
 * at the first call that needs them; such a call has to have run once before it is captured.  Graphs captured
 * from one handle and the handle's ordinary calls share the areas: on the handle's own stream they run one after the
 * other, but a replay on another stream must not run beside another such replay or beside calls of the handle.
 *
 * sbamd_set_kernel pins SBAMD_KERNEL_SMALL (few tokens), _LARGE (128 x 128 tiles) or _HUGE (256 x 256);
 * sbamd_last_kernel and sbamd_last_splitk report what ran; after a gradient, its last product (-1 if it had none).
 *
 * Every leading dimension must be at least the number of rows of its matrix.
 * Outputs must not overlap inputs unless an entry point says so.
 *
 * The reference has no counterpart of these entry points; they stand beside the products
 * of include/interface/blas3_interface.h:86-123.
 */
#ifndef SBAMD_FFN_H
#define SBAMD_FFN_H

#include "sbamd_gemm.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Activation of the gated block, act(g):
 *   SILU       g / (1 + exp(-g))
 *   GELU       g * Phi(g), Phi the normal distribution function
 *   GELU_TANH  g / 2 * (1 + tanh(sqrt(2/pi) * (g + 0.044715 g^3)))
 *   RELU       max(g, 0), its slope at 0 is 0 */
enum { SBAMD_ACT_SILU = 0, SBAMD_ACT_GELU = 1, SBAMD_ACT_GELU_TANH = 2, SBAMD_ACT_RELU = 3 };

/* Largest k of the products of 8-bit integers: their sums are held in 32 bits, and
 * 131071 * 128 * 128 is the last one that always fits.  Beyond: SBAMD_NOT_SUPPORTED. */
#define SBAMD_I8_MAX_K 131071

/* ------------------------------------------------------------ quantisation */

/* Columns of the m x n matrix x to 8-bit integers: scale[j] = max_i |x(i,j)| / 127 and
 * q(i,j) = the integer nearest to 127 * x(i,j) / max_i |x(i,j)|, ties to even, exactly
 * (as of the real quotient, not of a rounded one).  A column of zeros gets q = 0 and
 * scale 0.  A column that holds a NaN or an infinity gets q = 0 and scale NaN or
 * infinity, so that every product with it is NaN.  s / h / b: x is float / half /
 * bfloat16 (16-bit storage as bit patterns).  m == 0: scale 0 per column. */
int sbamd_squantize_i8(sbamd_handle_t h, int64_t m, int64_t n, const float* x, int64_t ldx, int8_t* q,
                       int64_t ldq, float* scale);
int sbamd_hquantize_i8(sbamd_handle_t h, int64_t m, int64_t n, const uint16_t* x, int64_t ldx, int8_t* q,
                       int64_t ldq, float* scale);
int sbamd_bquantize_i8(sbamd_handle_t h, int64_t m, int64_t n, const uint16_t* x, int64_t ldx, int8_t* q,
                       int64_t ldq, float* scale);

/* ---------------------------------------------------------- scaled product */

/* C <- alpha * diag(scale_a) * op(A) * op(B) * diag(scale_b) + beta * C with A and B of
 * 8-bit integers: the sum over k is an exact integer, then the scales, alpha and
 * beta * C follow in float and the result is rounded once to C's type (s / h / b:
 * float, half, bfloat16).  scale_a has m entries, scale_b has n; NULL stands for ones.
 * alpha == 0 and beta == 0 as in GEMM: alpha == 0 reads neither A, B nor the scales,
 * beta == 0 does not read C.  k <= SBAMD_I8_MAX_K. */
int sbamd_i8sgemm(sbamd_handle_t h, char transa, char transb, int64_t m, int64_t n, int64_t k, float alpha,
                  const int8_t* a, int64_t lda, const float* scale_a, const int8_t* b, int64_t ldb,
                  const float* scale_b, float beta, float* c, int64_t ldc);
int sbamd_i8hgemm(sbamd_handle_t h, char transa, char transb, int64_t m, int64_t n, int64_t k, float alpha,
                  const int8_t* a, int64_t lda, const float* scale_a, const int8_t* b, int64_t ldb,
                  const float* scale_b, float beta, uint16_t* c, int64_t ldc);
int sbamd_i8bgemm(sbamd_handle_t h, char transa, char transb, int64_t m, int64_t n, int64_t k, float alpha,
                  const int8_t* a, int64_t lda, const float* scale_a, const int8_t* b, int64_t ldb,
                  const float* scale_b, float beta, uint16_t* c, int64_t ldc);

/* ------------------------------------------------------------- gated block */

/* P = op(A) * op(B), where op(A) is 2m x k: rows 0 .. m-1 make the gate G, rows m .. 2m-1
 * the other projection U (one weight matrix that holds both, gate first).
 * C(i,j) = act(G(i,j)) * U(i,j), m x n.  Sums and activation are float, C is rounded once.
 * p: NULL, or a 2m x n matrix (ldp >= 2m) that receives P, rounded, for the backward pass.
 * h / b: half / bfloat16 storage throughout. */
int sbamd_hgated_gemm(sbamd_handle_t h, int act, char transa, char transb, int64_t m, int64_t n, int64_t k,
                      const uint16_t* a, int64_t lda, const uint16_t* b, int64_t ldb, uint16_t* c, int64_t ldc,
                      uint16_t* p, int64_t ldp);
int sbamd_bgated_gemm(sbamd_handle_t h, int act, char transa, char transb, int64_t m, int64_t n, int64_t k,
                      const uint16_t* a, int64_t lda, const uint16_t* b, int64_t ldb, uint16_t* c, int64_t ldc,
                      uint16_t* p, int64_t ldp);

/* The same block on 8-bit integers: P = diag(scale_a) op(A) op(B) diag(scale_b), scale_a
 * with 2m entries, scale_b with n (NULL: ones).  C in float, half or bfloat16. */
int sbamd_i8sgated_gemm(sbamd_handle_t h, int act, char transa, char transb, int64_t m, int64_t n, int64_t k,
                        const int8_t* a, int64_t lda, const float* scale_a, const int8_t* b, int64_t ldb,
                        const float* scale_b, float* c, int64_t ldc);
int sbamd_i8hgated_gemm(sbamd_handle_t h, int act, char transa, char transb, int64_t m, int64_t n, int64_t k,
                        const int8_t* a, int64_t lda, const float* scale_a, const int8_t* b, int64_t ldb,
                        const float* scale_b, uint16_t* c, int64_t ldc);
int sbamd_i8bgated_gemm(sbamd_handle_t h, int act, char transa, char transb, int64_t m, int64_t n, int64_t k,
                        const int8_t* a, int64_t lda, const float* scale_a, const int8_t* b, int64_t ldb,
                        const float* scale_b, uint16_t* c, int64_t ldc);

/* Gradient of the gated block.  Given P (as the forward call kept it, 2m x n) and dC, the
 * gradient of C (m x n):
 *   dP: rows 0 .. m-1   dC * U * act'(G),  rows m .. 2m-1   dC * act(G)   (2m x n, lddp >= 2m)
 *   dA <- the gradient of A + beta_a * dA,  dop(A) = dP * op(B)^T, stored as A is
 *   dB <- the gradient of B + beta_b * dB,  dop(B) = op(A)^T * dP, stored as B is
 * A beta accumulates (0: the old contents are not read).  da and db may be NULL: that
 * gradient is not computed, and the operand that only it reads (B for dA, A for dB) may
 * be NULL too.  dP is always computed; it is rounded to the storage type (the products
 * take 16-bit operands) and may be the same matrix as p (dp == p with lddp == ldp).
 * h / b: half / bfloat16 storage throughout; dA and dB are summed in float and rounded once. */
int sbamd_hgated_gemm_grad(sbamd_handle_t h, int act, char transa, char transb, int64_t m, int64_t n,
                           int64_t k, const uint16_t* a, int64_t lda, const uint16_t* b, int64_t ldb,
                           const uint16_t* p, int64_t ldp, const uint16_t* dc, int64_t lddc, uint16_t* dp,
                           int64_t lddp, float beta_a, uint16_t* da, int64_t ldda, float beta_b, uint16_t* db,
                           int64_t lddb);
int sbamd_bgated_gemm_grad(sbamd_handle_t h, int act, char transa, char transb, int64_t m, int64_t n,
                           int64_t k, const uint16_t* a, int64_t lda, const uint16_t* b, int64_t ldb,
                           const uint16_t* p, int64_t ldp, const uint16_t* dc, int64_t lddc, uint16_t* dp,
                           int64_t lddp, float beta_a, uint16_t* da, int64_t ldda, float beta_b, uint16_t* db,
                           int64_t lddb);

#ifdef __cplusplus
} /* extern "C" */
#endif

#endif /* SBAMD_FFN_H */
