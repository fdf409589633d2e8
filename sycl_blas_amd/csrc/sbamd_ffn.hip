// C ABI of the feed-forward entry points (include/sbamd_ffn.h): argument rules, repacking, launches.
#include <algorithm>
#include <cctype>
#include <cmath>
#include <string>

#include "gemm_dispatch.hpp"
#include "gemm_ffn.hpp"

namespace sbamd {
namespace {

int ffn_fail(Handle* h, hipError_t e, const char* what) {
  if (e == hipErrorNotSupported) return SBAMD_NOT_SUPPORTED;
  h->last_error = std::string(what) + ": " + hipGetErrorString(e);
  return e == hipErrorOutOfMemory ? SBAMD_ALLOC_FAILED : SBAMD_HIP_ERROR;
}

void forget_last(Handle* h, int64_t k) {
  h->last_kernel = -1;
  h->last_depth = 1;
  h->last_k_chunk = k;
  h->last_tile_m = h->last_tile_n = 0;
  h->last_fused = false;
}

// 'n' -> 0, 't' / 'c' -> 1, anything else -> -1
int trans_of(char t) {
  const char c = char(std::tolower(static_cast<unsigned char>(t)));
  return c == 'n' ? 0 : c == 't' || c == 'c' ? 1 : -1;
}

template <typename Tag, typename TOut, bool GATED, int NB, int DEPTH, int OCC>
hipError_t launch_narrow(FfnArgs<TOut> g, hipStream_t stream) {
  auto kernel = ffn_narrow_kernel<Tag, TOut, GATED, NB, DEPTH, OCC>;
  constexpr int lds = narrow_lds_bytes<NB>();
  static_assert(lds <= 64 * 1024, "within the default limit of dynamic LDS");
  const int64_t tm = ceil_div(g.m, GATED ? NARROW_ROWS / 2 : NARROW_ROWS), tn = ceil_div(g.n, 16 * NB);
  if (tm > 0x7fffffffLL / tn) return hipErrorInvalidValue;
  g.tiles_m = int32_t(tm);
  g.tiles_n = int32_t(tn);
  hipLaunchKernelGGL(kernel, folded_grid(tm * tn, NARROW_WAVES * 64), dim3(NARROW_WAVES * 64), lds, stream, g);
  return hipGetLastError();
}

// An operand as the caller has it, and what the kernels read.
struct Rows {
  const void* x;
  int64_t ld;     // elements
  int64_t rows, k;
  bool across;    // element (row, k) at row + k * ld instead of k + row * ld
};

template <int BYTES>
hipError_t pack(Handle* h, const Rows& o, unsigned char* dst, int64_t row_bytes) {
  const unsigned char* src = static_cast<const unsigned char*>(o.x);
  const int64_t grid = o.across ? ceil_div(o.rows, PACK_R_BYTES / BYTES) * ceil_div(row_bytes, PACK_K_BYTES) : ceil_div(row_bytes / 16 * o.rows, 256);
  if (grid > MAX_GRID) return hipErrorInvalidValue;
  if (o.across)
    hipLaunchKernelGGL((ffn_pack_across_kernel<BYTES>), folded_grid(grid, 256), dim3(256), 0, h->stream, src, o.ld, dst, row_bytes, o.rows, o.k);
  else
    hipLaunchKernelGGL((ffn_pack_rows_kernel<BYTES>), folded_grid(grid, 256), dim3(256), 0, h->stream, src, o.ld, dst, row_bytes, o.rows, o.k);
  return hipGetLastError();
}

template <typename Tag, typename TOut, bool GATED, bool TA, bool TB, int BM, int BN, int WM, int WN>
hipError_t launch_ring(FfnArgs<TOut> g, int cus, hipStream_t stream) {
  auto kernel = ffn_ring_kernel<Tag, TOut, GATED, TA, TB, BM, BN, WM, WN>;
  constexpr int lds = ring_lds_bytes(BM, BN);
  static PerDeviceOnce lds_limit;
  const hipError_t e = lds_limit.run([&] {
    return hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  });
  if (e != hipSuccess) return e;
  const int64_t tm = ceil_div(g.m, GATED ? BM / 2 : BM), tn = ceil_div(g.n, BN);
  // (the kernel's tile counter runs past the last tile by up to a grid)
  if (tm > 0x7fff0000LL / tn) return hipErrorInvalidValue;
  g.tiles_m = int32_t(tm);
  g.tiles_n = int32_t(tn);
  const int64_t resident = int64_t(cus) * (160 * 1024 / lds), units = GATED ? tm * tn : g.whole + (tm * tn - g.whole) * g.slabs;
  if (units > 0x7fff0000LL) return hipErrorInvalidValue;
  hipLaunchKernelGGL(kernel, dim3((unsigned)std::min(units, resident)), dim3(WM * WN * 64), lds, stream, g);
  return hipGetLastError();
}

template <typename Tag, typename TOut, bool GATED, int BM, int BN, int WM, int WN>
hipError_t launch_ring_trans(const FfnArgs<TOut>& g, bool ta, bool tb, int cus, hipStream_t stream) {
  // 8-bit operands always lie along k here: the transposing LDS reads the other layouts need move 16-bit elements
  if constexpr (std::is_same<Tag, I8Tag>::value) {
    return launch_ring<Tag, TOut, GATED, true, false, BM, BN, WM, WN>(g, cus, stream);
  } else {
    if (ta) return tb ? launch_ring<Tag, TOut, GATED, true, true, BM, BN, WM, WN>(g, cus, stream) : launch_ring<Tag, TOut, GATED, true, false, BM, BN, WM, WN>(g, cus, stream);
    return tb ? launch_ring<Tag, TOut, GATED, false, true, BM, BN, WM, WN>(g, cus, stream) : launch_ring<Tag, TOut, GATED, false, false, BM, BN, WM, WN>(g, cus, stream);
  }
}

inline bool aligned16(const void* p, int64_t ld_bytes) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld_bytes % 16 == 0; }

// How the ring works through the tiles of EDGE x EDGE: the first `whole` in one go, the rest in `slabs` pieces along k.
struct RingPlan {
  double time;  // estimated microseconds
  int32_t whole, slabs;
  int64_t chunk;
};
// Lengths along k in bytes make one model of 8-bit and 16-bit operands: a fragment, a stage and a cache line hold the same
// bytes, and a matrix instruction takes the same time for either.  Measured on MI355X over n = 16 ... 21504, (k, m) = (1024, 4096),
// (4096, 1024), (4096, 4096), (4096, 16384), (16384, 4096), plain and gated:
//   128 x 128: 3.3e-3 us per byte of k with few tiles, 5.9e-3 with one per unit (8192 bytes: 33 / 51; 2048: 10 / 13.6), 6e-3 per
//     tile and unit beyond (two share a unit, so no whole rounds: 448 tiles, 16384 bytes: 160); operands at 4.2 TB/s;
//   256 x 256: 6 us and 13e-3 per byte and round of one tile per unit (2048 bytes, 10.5 rounds: 354; 8192: 1196), 8.2e-3
//     with few units busy.
// A tile count that leaves units idle in the last round (128 or 336 tiles of 256 x 256 on 256 units) has that round's tiles cut
// along k into as many pieces as fill it, at the price of the pieces' sums going out and coming back (4.5 TB/s) and a second
// launch.  (rows, n): the product's; len: bytes along k; cut: whether tiles may be cut.
template <int EDGE>
RingPlan plan_ring(int64_t rows, int64_t n, int64_t len, int cus, bool cut) {
  const int64_t tiles = ceil_div(rows, EDGE) * ceil_div(n, EDGE), k = len / 2;
  const double bytes = double(len), q = double(tiles) / cus;
  auto one_round = [&](double share, double b) {  // with `share` of the units busy
    return EDGE == 256 ? 6.0 + b * (8.2e-3 + 4.5e-3 * share) : b * (3.3e-3 + 2.6e-3 * share);
  };
  RingPlan best = {0.0, int32_t(std::min<int64_t>(tiles, 0x7fff0000LL)), 1, k};
  const int64_t rounds = EDGE == 256 ? tiles / cus : 0, rest = tiles - rounds * cus;
  const double t_whole = 3.0 + double(rounds) * (6.0 + bytes * 13e-3);
  best.time = EDGE == 128 && q > 1.0 ? 3.0 + q * (bytes * 6.0e-3 + 0.7) : t_whole + (rest ? one_round(double(rest) / cus, bytes) : 0.0);
  best.time = std::max(best.time, 3.0 + double(rows + n) * bytes / 4.2e6);
  constexpr int64_t SHORTEST = 8 * RING_BK;  // a slab, in 16-bit units: below that its prologue costs more than its work
  if (!cut || rest == 0 || k < 2 * SHORTEST || tiles > 0x7fff0000LL) return best;
  for (int64_t s = 2; s <= 32 && s * rest <= cus; ++s) {
    const int64_t chunk = RING_BK * ceil_div(k, RING_BK * s), slabs = ceil_div(k, chunk);
    if (slabs < 2 || chunk < SHORTEST) continue;
    const double cube = double(rest) * double(slabs) * EDGE * EDGE * 4.0;
    const double t = t_whole + one_round(double(rest * slabs) / cus, 2.0 * double(chunk)) + 4.0 + 2.0 * cube / 4.5e6;
    if (t < best.time) best = {t, int32_t(rounds * cus), int32_t(slabs), chunk};
  }
  return best;
}

// The narrow kernel: operands at 6.2 TB/s; what the workgroups (32 rows x up to 64 tokens) read again through L2 at 28 TB/s, 12
// where the tokens outgrow an XCD's 4 MB of it, both at 0.6 of that where rows are not 16-byte aligned; 2 us for each further
// round of 512 workgroups; 1.2e-3 us per byte of k for a workgroup alone (rows 32768,
// 8192 bytes: n = 16 45 us, 48 58, 128 102; rows 8192: n = 224 43, 512 91).
inline double narrow_time(int64_t rows, int64_t n, int64_t len, bool aligned) {
  const double b = double(len);
  const int64_t tok = n <= 16 ? 16 : n <= 32 ? 32 : n <= 48 ? 48 : 64;
  const double blocks = double(ceil_div(n, tok)), wgs = double(ceil_div(rows, NARROW_ROWS)) * blocks;
  const double again = (wgs * double(tok) + (blocks - 1.0) * double(rows)) * b;
  const double moved = double(rows + n) * b / 6.2e6 + again / (double(n) * b <= 4.5e6 ? 28e6 : 12e6);
  return 4.0 + std::max(b * 1.2e-3, aligned ? moved : moved / 0.6) + 2.0 * std::max(0.0, wgs / 512.0 - 1.0);
}

// One ring launch by its plan, and the join of what it cut.  g has operands, sizes and outputs set.
template <typename Tag, typename TOut, bool GATED, int EDGE, int WM, int WN>
hipError_t run_ring(Handle* h, FfnArgs<TOut> g, bool ta, bool tb, int64_t rows, const RingPlan& plan, int cus) {
  g.whole = plan.whole, g.slabs = plan.slabs, g.chunk = plan.chunk;
  const int64_t tm = ceil_div(rows, EDGE), tn = ceil_div(g.n, EDGE), cut = GATED ? 0 : tm * tn - plan.whole;
  hipError_t e = hipSuccess;
  if (cut > 0) {
    if ((e = ensure_scratch(h, size_t(cut) * size_t(plan.slabs) * EDGE * EDGE * sizeof(float))) != hipSuccess) return e;
    g.cube = h->scratch;
    h->last_depth = plan.slabs;
    h->last_k_chunk = plan.chunk * 2 / FfnMma<Tag>::BYTES;
  }
  e = launch_ring_trans<Tag, TOut, GATED, EDGE, EDGE, WM, WN>(g, ta, tb, cus, h->stream);
  if constexpr (!GATED) {
    if (e != hipSuccess || cut <= 0) return e;
    g.tiles_m = int32_t(tm), g.tiles_n = int32_t(tn);
    hipLaunchKernelGGL((ffn_join_kernel<Tag, TOut, EDGE, EDGE>), dim3((unsigned)(cut * (EDGE * EDGE / 8 / 256))), dim3(256), 0, h->stream, g);
    e = hipGetLastError();
  }
  return e;
}

// The product behind all forward entry points.
template <typename Tag, typename TOut, bool GATED>
hipError_t run_ffn(Handle* h, const Rows& a, const Rows& b, FfnArgs<TOut> g) {
  constexpr int BYTES = FfnMma<Tag>::BYTES;
  constexpr int STEP = RING_BK * 2;  // bytes of k per step of the ring
  const int64_t kb = a.k * BYTES, row_bytes = ceil_div(kb, STEP) * STEP;
  const int cus = h->compute_units > 0 ? h->compute_units : 256;
  // What the kernel can read in place.  The narrow kernel: rows along k at any alignment.  The ring: 16-byte aligned rows
  // of at least one step along k (8-bit: an even number), or 16-bit operands across k whose rows come in whole
  // 16-byte pieces.  Everything else is repacked along k, zero-padded to whole steps, in the handle's second scratch area.
  auto ring_reads = [&](const Rows& o, int64_t whole_rows) {
    return aligned16(o.x, o.ld * BYTES) && (!o.across || (BYTES == 2 && whole_rows % 8 == 0)) && kb >= STEP && kb % 2 == 0;
  };
  // (the gated block's two halves of op(A) are clamped apart: m itself has to be whole pieces.  One length along k serves
  // both operands, so a short or odd one is padded on both sides: the conditions on kb are the same for both.)
  const bool ring_pack_a = !ring_reads(a, GATED ? a.rows / 2 : a.rows), ring_pack_b = !ring_reads(b, b.rows);
  auto pack_time = [&](bool packed, const Rows& o) { return packed ? 3.0 + 2.0 * double(o.rows) * double(row_bytes) / 3.0e6 : 0.0; };
  const RingPlan big = plan_ring<256>(a.rows, b.rows, row_bytes, cus, !GATED), small = plan_ring<128>(a.rows, b.rows, row_bytes, cus, !GATED);
  int family = h->kernel_override;
  if (family != SBAMD_KERNEL_SMALL && family != SBAMD_KERNEL_LARGE && family != SBAMD_KERNEL_HUGE) {
    const double extra = pack_time(ring_pack_a, a) + pack_time(ring_pack_b, b) - pack_time(a.across, a) - pack_time(b.across, b);
    const double t_ring = std::min(big.time, small.time);
    const bool rows_aligned = (a.across || aligned16(a.x, a.ld * BYTES)) && (b.across || aligned16(b.x, b.ld * BYTES));
    family = narrow_time(a.rows, b.rows, kb, rows_aligned) <= t_ring + extra ? SBAMD_KERNEL_SMALL : small.time <= big.time ? SBAMD_KERNEL_LARGE : SBAMD_KERNEL_HUGE;
  }
  if (kb == 0) family = SBAMD_KERNEL_SMALL;  // nothing to pipeline: the narrow kernel writes the sums over nothing
  const bool ring = family != SBAMD_KERNEL_SMALL;
  const bool pack_a = kb > 0 && (ring ? ring_pack_a : a.across), pack_b = kb > 0 && (ring ? ring_pack_b : b.across);
  if (pack_a || pack_b) {
    const size_t bytes_a = pack_a ? size_t(a.rows) * size_t(row_bytes) : 0, bytes_b = pack_b ? size_t(b.rows) * size_t(row_bytes) : 0;
    const hipError_t e = ensure_aux(h, bytes_a + bytes_b);  // (rows of whole steps: b stays aligned behind a)
    if (e != hipSuccess) return e;
    unsigned char* at = static_cast<unsigned char*>(h->aux);
    hipError_t st = hipSuccess;
    if (pack_a) st = pack<BYTES>(h, a, at, row_bytes);
    if (st == hipSuccess && pack_b) st = pack<BYTES>(h, b, at + bytes_a, row_bytes);
    if (st != hipSuccess) return st;
    g.a = at, g.b = at + bytes_a;
  }
  g.lda = pack_a ? row_bytes : a.ld * BYTES;
  g.ldb = pack_b ? row_bytes : b.ld * BYTES;
  if (!pack_a) g.a = static_cast<const unsigned char*>(a.x);
  if (!pack_b) g.b = static_cast<const unsigned char*>(b.x);
  g.kb = pack_a && pack_b ? row_bytes : kb;  // (zeros add nothing)
  const bool ta = pack_a || !a.across, tb = !pack_b && b.across;

  h->last_kernel = family;
  if (family == SBAMD_KERNEL_HUGE) return run_ring<Tag, TOut, GATED, 256, 2, 4>(h, g, ta, tb, a.rows, big, cus);
  if (family == SBAMD_KERNEL_LARGE) return run_ring<Tag, TOut, GATED, 128, 2, 2>(h, g, ta, tb, a.rows, small, cus);
  if (g.n <= 16) return launch_narrow<Tag, TOut, GATED, 1, 4, 2>(g, h->stream);
  if (g.n <= 32) return launch_narrow<Tag, TOut, GATED, 2, 2, 3>(g, h->stream);
  if (g.n <= 48) return launch_narrow<Tag, TOut, GATED, 3, 2, 2>(g, h->stream);
  return launch_narrow<Tag, TOut, GATED, 4, 2, 2>(g, h->stream);
}

// ------------------------------------------------------------------ front ends
template <typename TOut>
hipError_t scale_c(Handle* h, TOut* c, int64_t m, int64_t n, int64_t ldc, float beta);
template <>
hipError_t scale_c<float>(Handle* h, float* c, int64_t m, int64_t n, int64_t ldc, float beta) {
  return run_scale_f32(h, c, m, n, ldc, 0, 1, beta, beta == 0.0f);
}
template <>
hipError_t scale_c<uint16_t>(Handle* h, uint16_t* c, int64_t m, int64_t n, int64_t ldc, float beta) {
  return run_scale_f16(h, c, m, n, ldc, 0, 1, beta, beta == 0.0f);
}
__global__ void __launch_bounds__(256) ffn_scale_bf16_kernel(bf16_bits* c, int64_t m, int64_t n, int64_t ldc, float beta, int beta_zero) {
  const int64_t idx = folded_block() * 256 + threadIdx.x;
  if (idx >= m * n) return;
  bf16_bits* p = c + idx % m + idx / m * ldc;
  store_out(p, beta_zero ? 0.0f : beta * load_out(p));
}
template <>
hipError_t scale_c<bf16_bits>(Handle* h, bf16_bits* c, int64_t m, int64_t n, int64_t ldc, float beta) {
  const int64_t grid = ceil_div(m * n, 256);
  if (grid > MAX_GRID) return hipErrorInvalidValue;
  hipLaunchKernelGGL(ffn_scale_bf16_kernel, folded_grid(grid, 256), dim3(256), 0, h->stream, c, m, n, ldc, beta, beta == 0.0f ? 1 : 0);
  return hipGetLastError();
}

// Is `ld` a leading dimension for `rows` rows, and does a matrix of `cols` such columns of `bytes`-byte elements have a size that
// address arithmetic can hold at all?
bool holds(int64_t ld, int64_t rows, int64_t cols, int64_t bytes) {
  int64_t size = 0;
  return ld >= rows && !__builtin_mul_overflow(ld, cols, &size) && !__builtin_mul_overflow(size, bytes, &size) && size < (int64_t(1) << 60);
}

template <typename Tag, typename TOut, bool GATED>
int forward(sbamd_handle_t hh, int act, char transa, char transb, int64_t m, int64_t n, int64_t k, float alpha, const void* a,
            int64_t lda, const float* scale_a, const void* b, int64_t ldb, const float* scale_b, float beta, TOut* c, int64_t ldc,
            TOut* p, int64_t ldp) {
  if (!hh) return SBAMD_INVALID_HANDLE;
  Handle* h = &hh->impl;
  // (so that 2m and sums of sizes stay far from 63 bits; the matrices' own sizes are checked below)
  constexpr int64_t LIMIT = int64_t(1) << 40;
  if (m < 0 || n < 0 || k < 0 || m > LIMIT || n > LIMIT || k > LIMIT) return SBAMD_INVALID_VALUE;
  if (GATED && (act < SBAMD_ACT_SILU || act > SBAMD_ACT_RELU)) return SBAMD_INVALID_VALUE;
  DeviceGuard guard(h->device);
  if (!guard.ok) return SBAMD_HIP_ERROR;
  forget_last(h, k);
  if (!GATED && alpha == 0.0f) {  // as in GEMM: before the trans flags, A and B are not read
    if (m == 0 || n == 0) return SBAMD_OK;
    if (!c || !holds(ldc, m, n, sizeof(TOut))) return SBAMD_INVALID_VALUE;
    if (beta == 1.0f) return SBAMD_OK;
    const hipError_t e = scale_c<TOut>(h, c, m, n, ldc, beta);
    return e == hipSuccess ? SBAMD_OK : ffn_fail(h, e, "scale launch");
  }
  const int ta = trans_of(transa), tb = trans_of(transb);
  if (ta < 0) return SBAMD_INVALID_TRANSA;
  if (tb < 0) return SBAMD_INVALID_TRANSB;
  if (std::is_same<Tag, I8Tag>::value && k > SBAMD_I8_MAX_K) return SBAMD_NOT_SUPPORTED;
  const int64_t rows_a = GATED ? 2 * m : m;
  constexpr int64_t BYTES = FfnMma<Tag>::BYTES, BYTES_C = sizeof(TOut);
  if (!holds(lda, ta ? k : rows_a, ta ? rows_a : k, BYTES) || !holds(ldb, tb ? n : k, tb ? k : n, BYTES) || !holds(ldc, m, n, BYTES_C))
    return SBAMD_INVALID_VALUE;
  if (GATED && p && !holds(ldp, 2 * m, n, BYTES_C)) return SBAMD_INVALID_VALUE;
  if (m == 0 || n == 0) return SBAMD_OK;
  if (!c || (k > 0 && (!a || !b))) return SBAMD_INVALID_VALUE;
  FfnArgs<TOut> g{};
  g.m = m, g.n = n;
  g.scale_a = scale_a, g.scale_b = scale_b;
  g.c = c, g.ldc = ldc;
  g.p = p, g.ldp = ldp;
  g.alpha = alpha, g.beta = beta, g.beta_zero = beta == 0.0f ? 1 : 0;
  g.act = act;
  const Rows ra = {a, lda, rows_a, k, ta == 0}, rb = {b, ldb, n, k, tb != 0};
  const hipError_t e = run_ffn<Tag, TOut, GATED>(h, ra, rb, g);
  return e == hipSuccess ? SBAMD_OK : ffn_fail(h, e, "feed-forward launch");
}

template <typename Tag, int TPC, int HOLD>
hipError_t launch_quantize(Handle* h, int64_t m, int64_t n, const typename QuantIn<Tag>::type* x, int64_t ldx, int8_t* q, int64_t ldq,
                           float* scale) {
  constexpr int COLS = TPC < 256 ? 256 / TPC : 1, THREADS = TPC < 256 ? 256 : TPC;
  const int64_t grid = ceil_div(n, COLS);
  if (grid > MAX_GRID) return hipErrorInvalidValue;
  hipLaunchKernelGGL((ffn_quantize_kernel<Tag, TPC, HOLD>), folded_grid(grid, THREADS), dim3(THREADS), 0, h->stream, m, n, x, ldx, q,
                     ldq, scale);
  return hipGetLastError();
}

template <typename Tag>
int quantize(sbamd_handle_t hh, int64_t m, int64_t n, const typename QuantIn<Tag>::type* x, int64_t ldx, int8_t* q, int64_t ldq,
             float* scale) {
  if (!hh) return SBAMD_INVALID_HANDLE;
  Handle* h = &hh->impl;
  if (m < 0 || n < 0 || !holds(ldx, m, n, sizeof(typename QuantIn<Tag>::type)) || !holds(ldq, m, n, 1)) return SBAMD_INVALID_VALUE;
  DeviceGuard guard(h->device);
  if (!guard.ok) return SBAMD_HIP_ERROR;
  forget_last(h, 0);
  if (n == 0) return SBAMD_OK;
  if (!scale || (m > 0 && (!x || !q))) return SBAMD_INVALID_VALUE;
  hipError_t e;
  if (m <= 64 * 8) e = launch_quantize<Tag, 64, 1>(h, m, n, x, ldx, q, ldq, scale);
  else if (m <= 256 * 8 * 2) e = launch_quantize<Tag, 256, 2>(h, m, n, x, ldx, q, ldq, scale);
  else e = launch_quantize<Tag, 1024, 2>(h, m, n, x, ldx, q, ldq, scale);
  return e == hipSuccess ? SBAMD_OK : ffn_fail(h, e, "quantise launch");
}

// C = op(A) op(B) + beta C in 16 bits, C rounded once: the gradients' products.
template <typename TOut>
struct Product {
  bool ta, tb;
  int64_t m, n, k;
  const uint16_t* a;
  int64_t lda;
  const uint16_t* b;
  int64_t ldb;
  float beta;
  TOut* c;
  int64_t ldc;
  int64_t lim_b;  // see FfnArgs
};

hipError_t run_product16(Handle* h, const Problem<uint16_t, uint16_t>& p, float beta) { return run_gemm_h(h, p, 1.0f, beta); }
hipError_t run_product16(Handle* h, const Problem<uint16_t, bf16_bits>& p, float beta) { return run_gemm_b(h, p, 1.0f, beta); }

template <typename TOut>
bool ring_reads_product(const Product<TOut>& q) {
  const int64_t lim_b = q.lim_b > 0 ? q.lim_b : q.n;
  return aligned16(q.a, q.lda * 2) && aligned16(q.b, q.ldb * 2) && q.k >= RING_BK && (q.ta || q.m % 8 == 0) && (!q.tb || lim_b % 8 == 0);
}

template <typename Tag, typename TOut>
hipError_t run_product(Handle* h, const Product<TOut>& q) {
  const int cus = h->compute_units > 0 ? h->compute_units : 256;
  h->last_depth = 1, h->last_k_chunk = q.k;  // (the gradient's other product may have been cut)
  if (ring_reads_product(q) && h->kernel_override != SBAMD_KERNEL_SMALL) {
    const RingPlan big = plan_ring<256>(q.m, q.n, 2 * q.k, cus, true), small = plan_ring<128>(q.m, q.n, 2 * q.k, cus, true);
    const bool take_big = h->kernel_override == SBAMD_KERNEL_HUGE || (h->kernel_override != SBAMD_KERNEL_LARGE && big.time < small.time);
    h->last_kernel = take_big ? SBAMD_KERNEL_HUGE : SBAMD_KERNEL_LARGE;
    FfnArgs<TOut> g{};
    g.a = reinterpret_cast<const unsigned char*>(q.a), g.lda = q.lda * 2;
    g.b = reinterpret_cast<const unsigned char*>(q.b), g.ldb = q.ldb * 2;
    g.m = q.m, g.n = q.n, g.kb = q.k * 2;
    g.c = q.c, g.ldc = q.ldc;
    g.alpha = 1.0f, g.beta = q.beta, g.beta_zero = q.beta == 0.0f ? 1 : 0;
    g.lim_b = q.lim_b;
    return take_big ? run_ring<Tag, TOut, false, 256, 2, 4>(h, g, q.ta, q.tb, q.m, big, cus)
                    : run_ring<Tag, TOut, false, 128, 2, 2>(h, g, q.ta, q.tb, q.m, small, cus);
  }
  // operands the ring cannot read as they lie: the 16-bit GEMM back end
  Problem<uint16_t, TOut> p{};
  p.ta = q.ta, p.tb = q.tb, p.m = q.m, p.n = q.n, p.k = q.k;
  p.a = q.a, p.lda = q.lda, p.b = q.b, p.ldb = q.ldb, p.c = q.c, p.ldc = q.ldc;
  p.batch = 1;
  p.beta_zero = q.beta == 0.0f;
  return run_product16(h, p, q.beta);
}

template <typename Tag, typename TOut>
int gradient(sbamd_handle_t hh, int act, char transa, char transb, int64_t m, int64_t n, int64_t k, const uint16_t* a, int64_t lda,
             const uint16_t* b, int64_t ldb, const uint16_t* p, int64_t ldp, const uint16_t* dc, int64_t lddc, uint16_t* dp,
             int64_t lddp, float beta_a, uint16_t* da, int64_t ldda, float beta_b, uint16_t* db, int64_t lddb) {
  if (!hh) return SBAMD_INVALID_HANDLE;
  Handle* h = &hh->impl;
  constexpr int64_t LIMIT = int64_t(1) << 40;
  if (m < 0 || n < 0 || k < 0 || m > LIMIT || n > LIMIT || k > LIMIT) return SBAMD_INVALID_VALUE;
  if (act < SBAMD_ACT_SILU || act > SBAMD_ACT_RELU) return SBAMD_INVALID_VALUE;
  DeviceGuard guard(h->device);
  if (!guard.ok) return SBAMD_HIP_ERROR;
  forget_last(h, k);
  const int ta = trans_of(transa), tb = trans_of(transb);
  if (ta < 0) return SBAMD_INVALID_TRANSA;
  if (tb < 0) return SBAMD_INVALID_TRANSB;
  const int64_t rows_a = ta ? k : 2 * m, rows_b = tb ? n : k;
  const int64_t cols_a = ta ? 2 * m : k, cols_b = tb ? k : n;
  if (!holds(ldp, 2 * m, n, 2) || !holds(lddc, m, n, 2) || !holds(lddp, 2 * m, n, 2)) return SBAMD_INVALID_VALUE;
  if (da && (!holds(ldda, rows_a, cols_a, 2) || !holds(ldb, rows_b, cols_b, 2))) return SBAMD_INVALID_VALUE;
  if (db && (!holds(lddb, rows_b, cols_b, 2) || !holds(lda, rows_a, cols_a, 2))) return SBAMD_INVALID_VALUE;
  const bool tokens = m > 0 && n > 0;  // is there a dP at all?
  if (tokens && (!p || !dc || !dp)) return SBAMD_INVALID_VALUE;
  if (dp == p && lddp != ldp) return SBAMD_INVALID_VALUE;  // in place means element for element
  if (tokens && k > 0 && ((da && !b) || (db && !a))) return SBAMD_INVALID_VALUE;
  TOut* out_a = reinterpret_cast<TOut*>(da);
  TOut* out_b = reinterpret_cast<TOut*>(db);
  // the two products on a given dP (`lim`: how many elements of its rows may be read)
  auto product_a = [&](const uint16_t* x, int64_t ldx, int64_t lim) -> Product<TOut> {
    if (ta) return {bool(tb), true, k, 2 * m, n, b, ldb, x, ldx, beta_a, out_a, ldda, lim};
    return {false, !tb, 2 * m, k, n, x, ldx, b, ldb, beta_a, out_a, ldda, 0};
  };
  auto product_b = [&](const uint16_t* x, int64_t ldx) -> Product<TOut> {
    if (tb) return {true, bool(ta), n, k, 2 * m, x, ldx, a, lda, beta_b, out_b, lddb, 0};
    return {!ta, false, k, n, 2 * m, a, lda, x, ldx, beta_b, out_b, lddb, 0};
  };
  const bool want_a = da && m > 0 && k > 0, want_b = db && n > 0 && k > 0;
  // A dP whose rows do not come in whole 16-byte pieces keeps the ring from reading it (2 * 2730 rows, 1119 tokens, k = 1000:
  // 47 us for dA where the padded copy takes 29; later steps brought that to 25): the elementwise pass then writes a second, padded one into the handle's scratch area.
  const int64_t grid = ceil_div(ceil_div(m, 8) * n, 256);
  if (grid > MAX_GRID) return SBAMD_INVALID_VALUE;
  uint16_t* copy = nullptr;
  const int64_t ld_copy = ceil_div(2 * m, 8) * 8;
  if (tokens && h->kernel_override != SBAMD_KERNEL_SMALL) {
    uint16_t* aligned = reinterpret_cast<uint16_t*>(uintptr_t(256));  // stands for the copy's place in the questions below
    if ((want_a && !ring_reads_product(product_a(dp, lddp, 0)) && ring_reads_product(product_a(aligned, ld_copy, ld_copy))) ||
        (want_b && !ring_reads_product(product_b(dp, lddp)) && ring_reads_product(product_b(aligned, ld_copy)))) {
      const hipError_t e = ensure_aux(h, size_t(ld_copy) * size_t(n) * sizeof(uint16_t));
      if (e != hipSuccess) return ffn_fail(h, e, "gradient scratch");
      copy = static_cast<uint16_t*>(h->aux);
    }
  }
  if (tokens) {
    hipLaunchKernelGGL((ffn_gate_grad_kernel<Tag, TOut>), folded_grid(grid, 256), dim3(256), 0, h->stream, act, m, n, p, ldp, dc, lddc, dp, lddp, copy,
                       ld_copy);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return ffn_fail(h, e, "gradient launch");
  }
  // The products run with n (m) == 0 too: a sum over nothing is beta times what was there.
  Product<TOut> qa = product_a(dp, lddp, 0), qb = product_b(dp, lddp);
  const bool copy_a = copy && want_a && !ring_reads_product(qa) && ring_reads_product(product_a(copy, ld_copy, ld_copy));
  const bool copy_b = copy && want_b && !ring_reads_product(qb) && ring_reads_product(product_b(copy, ld_copy));
  if (copy_a) qa = product_a(copy, ld_copy, ld_copy);
  if (copy_b) qb = product_b(copy, ld_copy);
  // A product the ring does not take may repack its operands into the scratch area that the copy is in, or have
  // it replaced by a larger one: whichever reads the copy goes first.
  hipError_t e = hipSuccess;
  if (copy_b && !copy_a) e = run_product<Tag, TOut>(h, qb);
  if (e == hipSuccess && want_a) e = run_product<Tag, TOut>(h, qa);
  if (e == hipSuccess && want_b && !(copy_b && !copy_a)) e = run_product<Tag, TOut>(h, qb);
  if (e != hipSuccess) return ffn_fail(h, e, "gradient product");
  return SBAMD_OK;
}

}  // namespace
}  // namespace sbamd

using namespace sbamd;

extern "C" {

int sbamd_squantize_i8(sbamd_handle_t h, int64_t m, int64_t n, const float* x, int64_t ldx, int8_t* q, int64_t ldq, float* scale) {
  return quantize<F32Tag>(h, m, n, x, ldx, q, ldq, scale);
}
int sbamd_hquantize_i8(sbamd_handle_t h, int64_t m, int64_t n, const uint16_t* x, int64_t ldx, int8_t* q, int64_t ldq, float* scale) {
  return quantize<HalfTag>(h, m, n, x, ldx, q, ldq, scale);
}
int sbamd_bquantize_i8(sbamd_handle_t h, int64_t m, int64_t n, const uint16_t* x, int64_t ldx, int8_t* q, int64_t ldq, float* scale) {
  return quantize<Bf16Tag>(h, m, n, x, ldx, q, ldq, scale);
}

#define SBAMD_SCALED(NAME, COUT, TOUT)                                                                                          \
  int NAME(sbamd_handle_t h, char transa, char transb, int64_t m, int64_t n, int64_t k, float alpha, const int8_t* a,           \
           int64_t lda, const float* scale_a, const int8_t* b, int64_t ldb, const float* scale_b, float beta, COUT* c,          \
           int64_t ldc) {                                                                                                       \
    return forward<I8Tag, TOUT, false>(h, SBAMD_ACT_SILU, transa, transb, m, n, k, alpha, a, lda, scale_a, b, ldb, scale_b,     \
                                       beta, reinterpret_cast<TOUT*>(c), ldc, nullptr, 0);                                      \
  }
SBAMD_SCALED(sbamd_i8sgemm, float, float)
SBAMD_SCALED(sbamd_i8hgemm, uint16_t, uint16_t)
SBAMD_SCALED(sbamd_i8bgemm, uint16_t, bf16_bits)
#undef SBAMD_SCALED

#define SBAMD_GATED(NAME, TAG, TOUT)                                                                                            \
  int NAME(sbamd_handle_t h, int act, char transa, char transb, int64_t m, int64_t n, int64_t k, const uint16_t* a,             \
           int64_t lda, const uint16_t* b, int64_t ldb, uint16_t* c, int64_t ldc, uint16_t* p, int64_t ldp) {                   \
    return forward<TAG, TOUT, true>(h, act, transa, transb, m, n, k, 1.0f, a, lda, nullptr, b, ldb, nullptr, 0.0f,              \
                                    reinterpret_cast<TOUT*>(c), ldc, reinterpret_cast<TOUT*>(p), ldp);                          \
  }
SBAMD_GATED(sbamd_hgated_gemm, HalfTag, uint16_t)
SBAMD_GATED(sbamd_bgated_gemm, Bf16Tag, bf16_bits)
#undef SBAMD_GATED

#define SBAMD_GATED_I8(NAME, COUT, TOUT)                                                                                        \
  int NAME(sbamd_handle_t h, int act, char transa, char transb, int64_t m, int64_t n, int64_t k, const int8_t* a,               \
           int64_t lda, const float* scale_a, const int8_t* b, int64_t ldb, const float* scale_b, COUT* c, int64_t ldc) {       \
    return forward<I8Tag, TOUT, true>(h, act, transa, transb, m, n, k, 1.0f, a, lda, scale_a, b, ldb, scale_b, 0.0f,            \
                                      reinterpret_cast<TOUT*>(c), ldc, nullptr, 0);                                             \
  }
SBAMD_GATED_I8(sbamd_i8sgated_gemm, float, float)
SBAMD_GATED_I8(sbamd_i8hgated_gemm, uint16_t, uint16_t)
SBAMD_GATED_I8(sbamd_i8bgated_gemm, uint16_t, bf16_bits)
#undef SBAMD_GATED_I8

#define SBAMD_GRAD(NAME, TAG, TOUT)                                                                                             \
  int NAME(sbamd_handle_t h, int act, char transa, char transb, int64_t m, int64_t n, int64_t k, const uint16_t* a,             \
           int64_t lda, const uint16_t* b, int64_t ldb, const uint16_t* p, int64_t ldp, const uint16_t* dc, int64_t lddc,       \
           uint16_t* dp, int64_t lddp, float beta_a, uint16_t* da, int64_t ldda, float beta_b, uint16_t* db, int64_t lddb) {    \
    return gradient<TAG, TOUT>(h, act, transa, transb, m, n, k, a, lda, b, ldb, p, ldp, dc, lddc, dp, lddp, beta_a, da, ldda,   \
                               beta_b, db, lddb);                                                                               \
  }
SBAMD_GRAD(sbamd_hgated_gemm_grad, HalfTag, uint16_t)
SBAMD_GRAD(sbamd_bgated_gemm_grad, Bf16Tag, bf16_bits)
#undef SBAMD_GRAD

}  // extern "C"
