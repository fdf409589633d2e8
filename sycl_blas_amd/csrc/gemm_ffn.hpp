// Kernels of the feed-forward entry points (include/sbamd_ffn.h): products of 8-bit
// integers with scales, the gated block in 16 and 8 bits, token quantisation and the
// elementwise half of the gated block's gradient.
//
// Layout: the column-major C is m (channels, contiguous) x n (tokens).  Both operands are
// read along k ([channel][k] and [token][k]); the host repacks what lies otherwise.
// Lengths along k are in BYTES throughout, so one kernel serves 16-bit and 8-bit
// operands: a matrix-instruction fragment is 16 bytes per lane for either (8 k of a
// 16-bit type, 16 k of an 8-bit one), and the order in which k is walked does not matter
// as long as both operands share it.
#pragma once

#include "gemm_half_dma.hpp"
#include "../../include/sbamd_ffn.h"

namespace sbamd {

struct I8Tag {};  // 8-bit integers, 32-bit integer sums

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
// 16 bytes at any address (global memory takes a misaligned vector; the type says so to the compiler)
typedef u16x8 u16x8_at1 __attribute__((aligned(1)));

// 16 x 16 matrix instruction: op0 carries the token index, op1 the channel; lane l ends up with channel l % 16 and
// tokens 4 * (l / 16) .. + 3.  K: 32 of a 16-bit type, 64 of 8-bit integers.
template <typename Tag>
struct FfnMma;
template <>
struct FfnMma<HalfTag> {
  static constexpr int BYTES = 2;
  using acc_t = f32x4_t;
  using sum_t = float;
  __device__ static inline acc_t mma(u16x8 x, u16x8 y, acc_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, x), __builtin_bit_cast(f16x8, y), c, 0, 0, 0);
  }
};
template <>
struct FfnMma<Bf16Tag> {
  static constexpr int BYTES = 2;
  using acc_t = f32x4_t;
  using sum_t = float;
  __device__ static inline acc_t mma(u16x8 x, u16x8 y, acc_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, y), c, 0, 0, 0);
  }
};
template <>
struct FfnMma<I8Tag> {
  static constexpr int BYTES = 1;
  using acc_t = i32x4;
  using sum_t = int;
  __device__ static inline acc_t mma(u16x8 x, u16x8 y, acc_t c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, x), __builtin_bit_cast(i32x4, y), c, 0, 0, 0);
  }
};

// 32 x 32 instruction of the ring: 64 bytes of k per two steps, like the 16-bit ones.
template <>
struct Mfma16<I8Tag> {
  __device__ static inline i32x16 mma(u16x8 op0, u16x8 op1, i32x16 c) {
    return __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(i32x4, op0), __builtin_bit_cast(i32x4, op1), c, 0, 0, 0);
  }
};

template <typename TOut>
struct FfnArgs {
  const unsigned char* a;  // [rows][k bytes], rows = m or 2m
  const unsigned char* b;  // [n][k bytes]
  int64_t lda, ldb;        // bytes from one row to the next
  int64_t m, n, kb;        // channels of C, tokens, bytes along k
  const float* scale_a;    // per row of a, NULL = ones
  const float* scale_b;    // per token, NULL = ones
  TOut* c;
  int64_t ldc;
  TOut* p;                 // pre-activations (2m x n) or NULL; gated only
  int64_t ldp;
  float alpha, beta;
  int32_t beta_zero;
  int32_t act;
  int32_t tiles_m, tiles_n;
  // Cut products (not the gated block): the first `whole` tiles are worked through in one go, the others in `slabs` pieces of
  // `chunk` 16-bit units of k whose sums (float, or integer) go to the cube, piece after piece, tile [BN tokens][BM channels].
  int32_t whole = 0, slabs = 1;
  int64_t chunk = 0;
  void* cube = nullptr;
  int64_t lim_b = 0;  // tokens of b that may be read where b lies across k and is padded behind the last one (0: n)
};

// ---------------------------------------------------------------- activations
// e^x through the hardware's 2^x (1 ulp): the roundings of the argument and of log2(e) make it good to about |x| * 2^-23.6, far
// below the 16-bit roundings behind it and within 7e-6 for a float result.  Overflow gives infinity and a quotient of 0.
__device__ inline float ffn_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896341f); }
__device__ inline float ffn_sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + ffn_exp(-x)); }

// tanh(y) = 2 sigmoid(2y) - 1, so 0.5 g (1 + tanh(y)) = g sigmoid(2y), without the cancellation for negative g.
__device__ inline float gelu_tanh_arg2(float g) { return 1.5957691216057308f * (g + 0.044715f * g * g * g); }

// Phi(g) and e^(-g^2/2), one exponential for both: with x = |g| / sqrt(2), erfc(x) = e^(-x^2) R(x), and R is a polynomial in
// t = 1 / (1 + 0.4 x), fitted for the least largest relative error over 0 <= x <= 9.5 (1.6e-7 with the coefficients as stored,
// below 5e-7 as evaluated in float), so the small values of Phi far on the negative side keep their relative
// precision, which 1 + erf would cancel away.
// (With the device library's erfc the elementwise gradient took 11.8 us at 1119 x 2730, so 8.5.)
__device__ inline void normal_parts(float g, float& phi, float& bell) {
  const float x = __builtin_fabsf(g) * 0.70710678118654752f;
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.4f, x, 1.0f));
  float r = 0.07275442034006119f;
  r = __builtin_fmaf(r, t, -0.39065292477607727f);
  r = __builtin_fmaf(r, t, 0.685164749622345f);
  r = __builtin_fmaf(r, t, -0.38698726892471313f);
  r = __builtin_fmaf(r, t, 0.4279186427593231f);
  r = __builtin_fmaf(r, t, 0.12624987959861755f);
  r = __builtin_fmaf(r, t, 0.24152310192584991f);
  r = __builtin_fmaf(r, t, 0.22394883632659912f);
  r = __builtin_fmaf(r, t, 8.045712456805632e-05f);
  bell = __builtin_amdgcn_exp2f(-0.72134752044448170f * g * g);
  const float tail = 0.5f * bell * r;
  phi = g < 0.0f ? tail : 1.0f - tail;
}

template <int ACT>
__device__ inline float act_value(float g) {
  if constexpr (ACT == SBAMD_ACT_SILU) return g * ffn_sigmoid(g);
  else if constexpr (ACT == SBAMD_ACT_GELU) {
    float phi, bell;
    normal_parts(g, phi, bell);
    return g * phi;
  } else if constexpr (ACT == SBAMD_ACT_GELU_TANH) return g * ffn_sigmoid(gelu_tanh_arg2(g));
  else return g <= 0.0f ? 0.0f : g;  // NaN stays NaN
}

// act(g) and act'(g)
template <int ACT>
__device__ inline void act_value_slope(float g, float& value, float& slope) {
  if constexpr (ACT == SBAMD_ACT_SILU) {
    const float s = ffn_sigmoid(g);
    value = g * s;
    slope = s + value * (1.0f - s);
  } else if constexpr (ACT == SBAMD_ACT_GELU) {
    float phi, bell;
    normal_parts(g, phi, bell);
    value = g * phi;
    slope = phi + g * 0.3989422804014327f * bell;
  } else if constexpr (ACT == SBAMD_ACT_GELU_TANH) {
    // value = g s(z), z = 2 sqrt(2/pi) (g + 0.044715 g^3); slope = s + g s (1 - s) z'.  Far out s (1 - s) is 0
    // and z' is not: the product is taken only where s (1 - s) is not 0 (0 * inf would be NaN).
    const float s = ffn_sigmoid(gelu_tanh_arg2(g));
    value = g * s;
    const float bell = s * (1.0f - s);
    slope = bell > 0.0f ? s + g * bell * (1.5957691216057308f * (1.0f + 0.134145f * g * g)) : s;
  } else {
    value = g <= 0.0f ? 0.0f : g;
    slope = g > 0.0f ? 1.0f : (g == g ? 0.0f : g);
  }
}

// f(integral_constant<int, act>): one uniform branch for a whole epilogue instead of one per element
template <typename F>
__device__ inline void with_act(int act, F&& f) {
  switch (act) {
    case SBAMD_ACT_SILU: f(std::integral_constant<int, SBAMD_ACT_SILU>{}); break;
    case SBAMD_ACT_GELU: f(std::integral_constant<int, SBAMD_ACT_GELU>{}); break;
    case SBAMD_ACT_GELU_TANH: f(std::integral_constant<int, SBAMD_ACT_GELU_TANH>{}); break;
    default: f(std::integral_constant<int, SBAMD_ACT_RELU>{});
  }
}

// One integer or float sum -> the scaled float: ((sum * sa) * sb), in this order so that two tiny scales do not
// underflow against each other.
template <typename Sum>
__device__ inline float ffn_scaled(Sum s, float sa, float sb) {
  return (float(s) * sa) * sb;
}

// ------------------------------------------------------------- narrow kernel
// C for a block of 32 operand rows (32 channels, or 16 gates with their 16 partners) and 16 * NB tokens.  The W
// wavefronts of the workgroup share out k in chunks of 128 bytes (a cache line of each row) and join their sums through
// LDS in wavefront order, so few rows still put many loads in flight and neither a second launch nor a workspace is
// needed.  A wavefront's chunk goes global -> registers
// (lane = one 16-byte piece, 8 lanes = one row's cache line; DEPTH chunks ahead) -> its own corner of LDS -> fragments:
// the detour through LDS turns the coalesced pieces into the matrix instruction's layout.  No barrier inside the loop:
// LDS operations of one wavefront execute in order.  Bound by the weights' way out of memory for few tokens.
constexpr int NARROW_CHUNK = 128, NARROW_WAVES = 4, NARROW_ROWS = 32;

// Image: 128-byte rows of eight 16-byte pieces; piece c of row r sits at c ^ ((r >> 1) & 7).  A fragment read has 16 lanes
// on 16 rows at the same c: two rows share a turn of the 64 banks, the eight pairs are told apart by the XOR.
__device__ inline int narrow_slot(int row, int piece) { return row * NARROW_CHUNK + ((piece ^ ((row >> 1) & 7)) << 4); }

template <int NB>
constexpr int narrow_lds_bytes() {
  constexpr int stage = NARROW_WAVES * (NARROW_ROWS + 16 * NB) * NARROW_CHUNK;
  constexpr int join = NARROW_WAVES * 16 * NB * (NARROW_ROWS + 1) * 4;
  return stage > join ? stage : join;
}

// The first `have` of 16 bytes at p, zeros behind them, without reading past them: the 16 bytes that END there, shifted down
// (all of them lie inside the row when the row has 16 bytes at all), byte by byte in a shorter row.  One load and a
// shift for each piece instead of up to 16 dependent loads.
__device__ inline u16x8 partial_piece(const unsigned char* p, int have, bool long_row) {
  typedef uint64_t u64x2 __attribute__((ext_vector_type(2)));
  typedef u64x2 u64x2_at1 __attribute__((aligned(1)));
  u64x2 v = {0, 0};
  if (have > 0) {
    const int drop = have < 16 ? 16 - have : 0;  // bytes of the load in front of p
    if (long_row) {
      v = *reinterpret_cast<const u64x2_at1*>(p - drop);
      const int bits = drop * 8;
      if (bits >= 64) {
        v[0] = v[1] >> (bits - 64);
        v[1] = 0;
      } else if (bits > 0) {
        v[0] = (v[0] >> bits) | (v[1] << (64 - bits));
        v[1] = v[1] >> bits;
      }
    } else {
      for (int e = 0; e < have; ++e) v[e >> 3] |= uint64_t(p[e]) << (8 * (e & 7));
    }
  }
  return __builtin_bit_cast(u16x8, v);
}

template <typename Tag, typename TOut, bool GATED, int NB, int DEPTH, int OCC>
__global__ void __launch_bounds__(NARROW_WAVES * 64, OCC) ffn_narrow_kernel(const FfnArgs<TOut> g) {
  using M = FfnMma<Tag>;
  using Sum = typename M::sum_t;
  constexpr int W = NARROW_WAVES, ROWS = NARROW_ROWS, TOK = 16 * NB;
  constexpr int CH = GATED ? ROWS / 2 : ROWS;  // channels of C per workgroup
  constexpr int LA = ROWS / 8, LB = TOK / 8, NL = LA + LB;  // load instructions per chunk
  extern __shared__ __attribute__((aligned(16))) unsigned char smem_raw[];
  SBAMD_LDS unsigned char* smem = (SBAMD_LDS unsigned char*)smem_raw;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t block = folded_block();
  const int blocks = g.tiles_m * g.tiles_n;
  if (block >= blocks) return;
  const int logical = xcd_remap(int(block), blocks);
  const int tm = logical / g.tiles_n, tn = logical - tm * g.tiles_n;  // the token blocks of one row block are neighbours
  const int64_t m0 = int64_t(tm) * CH, n0 = int64_t(tn) * TOK;

  // Rows past the edge read the last valid one: they only feed elements that are never stored.
  const int piece = lane & 7, row8 = lane >> 3;
  const unsigned char* src[NL];
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    if (i < LA) {
      const int row = i * 8 + row8;
      int64_t ch = m0 + (GATED ? row & 15 : row);
      ch = ch < g.m ? ch : g.m - 1;
      if (GATED && row >= 16) ch += g.m;
      src[i] = g.a + ch * g.lda + piece * 16;
    } else {
      int64_t t = n0 + (i - LA) * 8 + row8;
      t = t < g.n ? t : g.n - 1;
      src[i] = g.b + t * g.ldb + piece * 16;
    }
  }

  typename M::acc_t acc[2][NB];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[i][j][r] = 0;

  SBAMD_LDS unsigned char* mine = smem + wave * (ROWS + TOK) * NARROW_CHUNK;
  u16x8 reg[DEPTH][NL];
  auto issue = [&](u16x8 (&v)[NL], int64_t chunk) {
#pragma unroll
    for (int i = 0; i < NL; ++i) v[i] = *reinterpret_cast<const u16x8_at1*>(src[i] + chunk * NARROW_CHUNK);
  };
  auto consume = [&](const u16x8 (&v)[NL]) {
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int row = i < LA ? i * 8 + row8 : (i - LA) * 8 + row8;
      *reinterpret_cast<SBAMD_LDS u16x8*>(mine + (i < LA ? 0 : ROWS * NARROW_CHUNK) + narrow_slot(row, piece)) = v[i];
    }
    // other lanes of this wavefront read what this lane wrote: keep the compiler from moving the reads up (the
    // hardware keeps a wavefront's LDS operations in order)
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      u16x8 fa[2], fb[NB];
      const int at = 4 * s + (lane >> 4);
#pragma unroll
      for (int i = 0; i < 2; ++i)
        fa[i] = *reinterpret_cast<const SBAMD_LDS u16x8*>(mine + narrow_slot(i * 16 + (lane & 15), at));
#pragma unroll
      for (int j = 0; j < NB; ++j)
        fb[j] = *reinterpret_cast<const SBAMD_LDS u16x8*>(mine + ROWS * NARROW_CHUNK + narrow_slot(j * 16 + (lane & 15), at));
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[i][j] = M::mma(fb[j], fa[i], acc[i][j]);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  };

  // Each wavefront takes a run of its own of the whole chunks and starts inside it at a place that goes by wavefront and
  // row block: rows are often a power of two apart, and without this the rows of all workgroups walk the same few memory
  // channels together (reading 268 MB as rows of 8192 bytes: chunks dealt out in turn 4.5 TB/s, runs 6.1, runs with turned
  // starts 6.1; rows of 16384: 5.7 / 4.9 / 6.1; 32768: 5.4 / 5.0 / 6.0).  The order of a row's sum is fixed by its place.
  const int64_t whole = g.kb / NARROW_CHUNK;
  const int64_t first = whole * wave / W, count = whole * (wave + 1) / W - first;
  const uint32_t turns = uint32_t(count < 0x7fffffff ? count : 0x7fffffff);
  const int64_t turn = count > 0 ? (uint32_t(tm) * 8u + uint32_t(wave) * 2u) % turns : 0;
  auto chunk = [&](int64_t i) {
    i += turn;
    return first + (i < count ? i : i - count);
  };
  const int64_t piped = count / DEPTH * DEPTH;
  // the pipelined part: no branch between a load and its use, so the compiler's waits stay counted
  if (piped > 0) {
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) issue(reg[d], chunk(d));
    for (int64_t it = DEPTH; it < piped; it += DEPTH) {
#pragma unroll
      for (int d = 0; d < DEPTH; ++d) {
        consume(reg[d]);
        issue(reg[d], chunk(it + d));
      }
    }
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) consume(reg[d]);
  }
  if (piped < count) {
#pragma unroll
    for (int d = 0; d < DEPTH - 1; ++d)
      if (piped + d < count) issue(reg[d], chunk(piped + d));
#pragma unroll
    for (int d = 0; d < DEPTH - 1; ++d)
      if (piped + d < count) consume(reg[d]);
  }
  // the last, partial chunk: zeros behind the end of k (the rows' ends are not read past)
  const int rest = int(g.kb - whole * NARROW_CHUNK);
  if (rest > 0 && wave == 0) {  // (no wavefront has fewer whole ones)
    const int have = rest - piece * 16;  // bytes of this lane's piece that exist
    const bool long_row = g.kb >= 16;
#pragma unroll
    for (int i = 0; i < NL; ++i) reg[0][i] = partial_piece(src[i] + whole * NARROW_CHUNK, have, long_row);
    consume(reg[0]);
  }

  // Join: [wavefront][token][row], rows padded to 33 words.
  __syncthreads();
  SBAMD_LDS Sum* part = (SBAMD_LDS Sum*)smem;
  constexpr int LDJ = ROWS + 1;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        part[(wave * TOK + j * 16 + 4 * (lane >> 4) + r) * LDJ + i * 16 + (lane & 15)] = acc[i][j][r];
  __syncthreads();
  auto joined = [&](int tok, int row) {
    Sum s = part[tok * LDJ + row];
#pragma unroll
    for (int w = 1; w < W; ++w) s = s + part[(w * TOK + tok) * LDJ + row];
    return s;
  };
  auto each = [&](auto&& store) {
    for (int e = tid; e < CH * TOK; e += W * 64) {
      const int ch = e % CH, tok = e / CH;
      const int64_t mm = m0 + ch, nn = n0 + tok;
      if (mm < g.m && nn < g.n) store(ch, tok, mm, nn, g.scale_b ? g.scale_b[nn] : 1.0f);
    }
  };
  if constexpr (GATED) {
    with_act(g.act, [&](auto act) {
      each([&](int ch, int tok, int64_t mm, int64_t nn, float sb) {
        const float gate = ffn_scaled(joined(tok, ch), g.scale_a ? g.scale_a[mm] : 1.0f, sb);
        const float up = ffn_scaled(joined(tok, 16 + ch), g.scale_a ? g.scale_a[g.m + mm] : 1.0f, sb);
        if (g.p) {
          store_out(g.p + mm + nn * g.ldp, gate);
          store_out(g.p + g.m + mm + nn * g.ldp, up);
        }
        store_out(g.c + mm + nn * g.ldc, act_value<decltype(act)::value>(gate) * up);
      });
    });
  } else {
    each([&](int ch, int tok, int64_t mm, int64_t nn, float sb) {
      TOut* at = g.c + mm + nn * g.ldc;
      float out = g.alpha * ffn_scaled(joined(tok, ch), g.scale_a ? g.scale_a[mm] : 1.0f, sb);
      if (!g.beta_zero) out = out + g.beta * load_out(at);
      store_out(at, out);
    });
  }
}

// --------------------------------------------------------------- ring kernel
// The 16-bit GEMM's ring (gemm_half_dma.hpp: operand tiles straight into LDS through five stages, 256 x 256 tiles on eight
// wavefronts or 128 x 128 on four) with the feed-forward epilogue.  8-bit operands run through it as pairs: 64 bytes of
// k per stage and row, the same pieces and fragments, half the steps for the same k.  GATED: the rows of A alternate 32 gates
// and their 32 partners, so both halves of a channel meet in one lane and P never leaves the kernel unless asked for.
//
// The grid is as many workgroups as the chip holds and each walks its tiles.  The first loads of the next tile (stages
// 0 .. 3) are issued before the epilogue of the current one, which works in the last stage alone: with a tile per workgroup
// the unit stood still for about 10 us per 256 x 256 tile (launch, first loads, epilogue), of 35 for k = 1024.
//
// Epilogue: a lane holds one token and runs of four channels; they go through the wavefront's corner of LDS ([32 tokens][128
// bytes], 16-byte piece c of row r at c ^ ((r >> 1) & 7)) and leave as whole rows of up to 128 bytes (element by element where
// C's rows are not 16-byte aligned or the tile hangs over the edge).  16-bit results are rounded on the way into the
// corner; with beta * C to add they stay float there and are rounded once behind the addition.
// Bands of four tile rows instead of the GEMM's eight: 8-bit gated 1712 x 4096 -> 16384 229 -> 224 us, the rest within 1 %.
constexpr int RING_BAND = 4;
constexpr int CORNER_ROW = 128, CORNER_BYTES = 32 * CORNER_ROW;
__device__ inline int corner_at(int row, int byte) { return row * CORNER_ROW + (((byte >> 4) ^ ((row >> 1) & 7)) << 4) + (byte & 15); }

// 32 tokens x SLAB channels of SB-byte elements (2: already of type TOut; 4: floats) from the corner to rows of `out`.
// (One store instruction per 64 pieces, always, where `vec` and every row and channel exists: the ring counts on it.)
template <int SB, int SLAB, typename TOut>
__device__ inline void corner_to_rows(const SBAMD_LDS unsigned char* corner, TOut* out, int64_t ld, int64_t ch0, int64_t ch_lim, int64_t t0,
                                      int64_t t_lim, bool vec, int lane, bool read_c, float beta) {
  constexpr int V = 16 / SB, PER = SLAB / V, ROWS = 64 / PER;  // channels per piece, pieces per row, rows per instruction
  typedef unsigned int piece_t __attribute__((ext_vector_type(V * sizeof(TOut) / 4)));
  if (vec && ch0 + SLAB <= ch_lim) {
    const int piece = lane % PER;
#pragma unroll
    for (int r = 0; r < 32; r += ROWS) {
      const int row = r + lane / PER;
      if (t0 + row >= t_lim) continue;
      TOut* at = out + ch0 + piece * V + (t0 + row) * ld;
      const i32x4 raw = *reinterpret_cast<const SBAMD_LDS i32x4*>(corner + corner_at(row, piece * 16));
      if constexpr (SB == 2) {
        *reinterpret_cast<i32x4*>(at) = raw;
      } else {
        union {
          TOut e[V];
          piece_t q;
        } x;
        f32x4_t v = __builtin_bit_cast(f32x4_t, raw);
        if (read_c) {
          x.q = *reinterpret_cast<const piece_t*>(at);
#pragma unroll
          for (int e = 0; e < V; ++e) v[e] = v[e] + beta * load_out(&x.e[e]);
        }
#pragma unroll
        for (int e = 0; e < V; ++e) store_out(&x.e[e], v[e]);
        *reinterpret_cast<piece_t*>(at) = x.q;
      }
    }
  } else {
    // one element per lane, a whole slab of a row (or two) per instruction; eight reads ahead of their stores
    constexpr int AT_ONCE = 64 / SLAB, STEPS = 32 / AT_ONCE, BATCH = 8;
    const int ch = lane % SLAB, row0 = lane / SLAB;
    const bool live = ch0 + ch < ch_lim;
    typedef typename std::conditional<SB == 2, uint16_t, float>::type staged_t;
#pragma unroll 1
    for (int r = 0; r < STEPS; r += BATCH) {
      staged_t v[BATCH];
#pragma unroll
      for (int i = 0; i < BATCH; ++i) v[i] = *reinterpret_cast<const SBAMD_LDS staged_t*>(corner + corner_at((r + i) * AT_ONCE + row0, ch * SB));
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        const int row = (r + i) * AT_ONCE + row0;
        if (!live || t0 + row >= t_lim) continue;
        TOut* at = out + ch0 + ch + (t0 + row) * ld;
        if constexpr (SB == 2) {
          *reinterpret_cast<uint16_t*>(at) = v[i];
        } else {
          float f = v[i];
          if (read_c) f = f + beta * load_out(at);
          store_out(at, f);
        }
      }
    }
  }
}

template <typename Tag, typename TOut, bool GATED, bool TA, bool TB, int BM, int BN, int WM, int WN>
__global__ void __launch_bounds__(WM* WN * 64, 2) ffn_ring_kernel(const FfnArgs<TOut> g) {
  constexpr int NT = WM * WN * 64;
  constexpr int WTM = BM / WM, WTN = BN / WN;
  constexpr int MI = WTM / 32, NI = WTN / 32;
  constexpr int CHW = GATED ? WTM / 2 : WTM;  // channels of C per wavefront tile
  constexpr int CHB = GATED ? BM / 2 : BM;    // and per workgroup
  constexpr bool SCALED = std::is_same<Tag, I8Tag>::value;
  constexpr bool CUT = !GATED;  // tiles may be cut along k
  using OpA = RingOperand<TA, BM, NT>;
  using OpB = RingOperand<!TB, BN, NT>;
  using Acc = typename std::conditional<SCALED, i32x16, f32x16>::type;
  constexpr int STAGE_BYTES = OpA::BYTES + OpB::BYTES;
  static_assert(!GATED || MI % 2 == 0, "gates and partners in pairs");
  static_assert(WM * WN * CORNER_BYTES <= STAGE_BYTES, "the corners fit one stage");
  static_assert(WTM % 64 == 0, "a wavefront tile's row scales lie in whole registers");

  extern __shared__ __attribute__((aligned(1024))) unsigned char smem_raw[];
  SBAMD_LDS unsigned char* smem = (SBAMD_LDS unsigned char*)smem_raw;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave % WM, wn = wave / WM;

  const int64_t lda = g.lda / 2, ldb = g.ldb / 2;  // in 16-bit units
  const int tiles = g.tiles_m * g.tiles_n;
  const int units = CUT ? g.whole + (tiles - g.whole) * g.slabs : tiles;  // a unit of work: a tile, or a slab of one
  OpA oa;
  OpB ob;
  int64_t m0, n0, k_len;
  float sa[WTM / 64], sb[NI];  // scales: lane's rows lane, lane + 64 of the wavefront tile; lane's token of each 32-token block
  int piece = 0;  // CUT: which slab of the cube, counted from 0; whole tiles have none
  auto begin = [&](int unit) {
    const uint16_t* a = reinterpret_cast<const uint16_t*>(g.a);
    const uint16_t* b = reinterpret_cast<const uint16_t*>(g.b);
    int tm, tn, tile;
    k_len = g.kb / 2;
    if (!CUT || unit < g.whole) {
      tile = xcd_remap(unit, CUT ? g.whole : tiles);
    } else {
      piece = xcd_remap(unit - g.whole, units - g.whole);
      tile = g.whole + piece / g.slabs;
      const int64_t k0 = int64_t(piece % g.slabs) * g.chunk;
      k_len = k_len - k0 < g.chunk ? k_len - k0 : g.chunk;
      a += TA ? k0 : k0 * lda;
      b += TB ? k0 * ldb : k0;
    }
    tile_coords(tile, g.tiles_m, g.tiles_n, tm, tn, BM == 256 ? RING_BAND : 0);
    m0 = int64_t(tm) * CHB, n0 = int64_t(tn) * BN;
    if constexpr (GATED) oa.init_gated(a, lda, m0, g.m, tid);
    else oa.init(a, lda, m0, g.m, tid);
    ob.init(b, ldb, n0, CUT && g.lim_b > 0 ? g.lim_b : g.n, tid);
    if constexpr (SCALED) {  // (rows and tokens past the edge read the last one: they only feed what is not stored)
#pragma unroll
      for (int i = 0; i < WTM / 64; ++i) {
        const int row = wm * WTM + i * 64 + lane;
        int64_t ch = m0 + (GATED ? (row >> 6) * 32 + (row & 31) : row);
        ch = ch < g.m ? ch : g.m - 1;
        if (GATED && (row & 32)) ch += g.m;
        sa[i] = g.scale_a ? g.scale_a[ch] : 1.0f;
      }
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        const int64_t t = n0 + wn * WTN + j * 32 + (lane & 31);
        sb[j] = g.scale_b ? g.scale_b[t < g.n ? t : g.n - 1] : 1.0f;
      }
    }
    ring_start(oa, ob, lda, ldb, int(k_len / RING_BK), smem, wave);
  };

  // vector stores of a whole tile's epilogue, per wavefront
  constexpr int STORES = NI * 32 * CHW * int(sizeof(TOut)) / 1024;
  bool stored = false;  // the last epilogue issued at least that many behind the loads of the tile to come
  begin(blockIdx.x);
  for (int unit = blockIdx.x;;) {
    Acc acc[MI][NI];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;
    // (its first barrier lies behind every wavefront's epilogue of the tile before, so the last stage may be refilled)
    ring_multiply<Tag, OpA, OpB, MI, NI, WTM, WTN, 0, false, STORES>(acc, oa, ob, lda, ldb, k_len, smem, tid, lane, wave, wm,
                                                                                       wn, stored);

    __syncthreads();  // every wavefront is through with the ring's stages
    const int64_t ch0 = m0 + wm * CHW, tok0 = n0 + wn * WTN;
    const bool partial = CUT && unit >= g.whole;
    const int piece_now = piece;
    float sa_now[WTM / 64], sb_now[NI];
    if constexpr (SCALED) {
#pragma unroll
      for (int i = 0; i < WTM / 64; ++i) sa_now[i] = sa[i];
#pragma unroll
      for (int j = 0; j < NI; ++j) sb_now[j] = sb[j];
    }
    const int next = unit + int(gridDim.x);
    if (next < units) begin(next);

    // The epilogue's addresses are made from a lane index the compiler cannot see through: it would otherwise compute them
    // all in front of the tile loop and spill them.
    int lane_e = lane;
    asm volatile("" : "+v"(lane_e));
    SBAMD_LDS unsigned char* corner = smem + (RING_STAGES - 1) * STAGE_BYTES + wave * CORNER_BYTES;
    const int tok = lane_e & 31, half = lane_e >> 5;
    auto settle = []() __attribute__((always_inline)) {  // between the lanes' writes and other lanes' reads (one wavefront: LDS keeps its order)
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    };
    // (always_inline below: a lambda that is called twice and left as a function would put the accumulators into memory)
    // the four floats of rows 8 Q + 4 half .. + 3 of the wavefront tile's 32-row block I, tokens of block J
    auto four = [&](auto i_tag, auto j_tag, auto q_tag) __attribute__((always_inline)) {
      constexpr int I = decltype(i_tag)::value, J = decltype(j_tag)::value, Q = decltype(q_tag)::value;
      f32x4_t v;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (SCALED) v[e] = ffn_scaled(acc[I][J][Q * 4 + e], __shfl(sa_now[I / 2], (I % 2) * 32 + Q * 8 + half * 4 + e, 64), sb_now[J]);
        else v[e] = acc[I][J][Q * 4 + e];
      }
      return v;
    };
    // value(i, q) of 32-channel blocks i = B0 .. B0 + BLOCKS - 1 of the wavefront's channels, through the corner to `out`
    auto emit_at = [&](auto sb_tag, auto j_tag, auto&& value, auto* out, int64_t ld, int64_t ch_at, int64_t ch_lim, int64_t tok_at,
                       int64_t tok_lim, bool vec, bool read_c) __attribute__((always_inline)) {
      constexpr int SB = decltype(sb_tag)::value, J = decltype(j_tag)::value;
      using TTo = std::remove_pointer_t<decltype(out)>;
      constexpr int SLAB = CHW * SB < CORNER_ROW ? CHW : CORNER_ROW / SB, BLOCKS = SLAB / 32;
      static_for<CHW / SLAB>([&](auto slab) __attribute__((always_inline)) {
        constexpr int B0 = decltype(slab)::value * BLOCKS;
        static_for<BLOCKS>([&](auto block) __attribute__((always_inline)) {
          static_for<4>([&](auto q) __attribute__((always_inline)) {
            const f32x4_t v = value(std::integral_constant<int, B0 + decltype(block)::value>{}, j_tag, q);
            const int at = corner_at(tok, (decltype(block)::value * 32 + decltype(q)::value * 8 + half * 4) * SB);
            if constexpr (SB == 4) {
              *reinterpret_cast<SBAMD_LDS f32x4_t*>(corner + at) = v;
            } else {
              union {
                TOut e[4];
                uint64_t w;
              } x;
#pragma unroll
              for (int e = 0; e < 4; ++e) store_out(&x.e[e], v[e]);
              *reinterpret_cast<SBAMD_LDS uint64_t*>(corner + at) = x.w;
            }
          });
        });
        settle();
        corner_to_rows<SB, SLAB, TTo>(corner, out, ld, ch_at + decltype(slab)::value * SLAB, ch_lim, tok_at + J * 32, tok_lim, vec, lane_e,
                                      read_c, g.beta);
        settle();
      });
    };
    auto emit = [&](auto sb_tag, auto j_tag, auto&& value, TOut* out, int64_t ld, bool vec, bool read_c) __attribute__((always_inline)) {
      emit_at(sb_tag, j_tag, value, out, ld, ch0, g.m, tok0, g.n, vec, read_c);
    };
    auto rows_aligned = [](const void* p, int64_t ld) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (ld * int64_t(sizeof(TOut))) % 16 == 0; };
    using own_size = std::integral_constant<int, int(sizeof(TOut))>;
    using as_float = std::integral_constant<int, 4>;
    const bool vec_c = rows_aligned(g.c, g.ldc);
    if constexpr (GATED) {
      auto gate = [&](auto i, auto j, auto q) __attribute__((always_inline)) { return four(std::integral_constant<int, 2 * decltype(i)::value>{}, j, q); };
      auto up = [&](auto i, auto j, auto q) __attribute__((always_inline)) { return four(std::integral_constant<int, 2 * decltype(i)::value + 1>{}, j, q); };
      if (g.p) {
        const bool vec_p = rows_aligned(g.p, g.ldp);
        static_for<NI>([&](auto j) __attribute__((always_inline)) {
          emit(own_size{}, j, gate, g.p, g.ldp, vec_p, false);
          emit(own_size{}, j, up, g.p + g.m, g.ldp, vec_p && rows_aligned(g.p + g.m, g.ldp), false);
        });
      }
      with_act(g.act, [&](auto act) __attribute__((always_inline)) {
        static_for<NI>([&](auto j_tag) __attribute__((always_inline)) {
          emit(own_size{}, j_tag, [&](auto i, auto j, auto q) __attribute__((always_inline)) {
            const f32x4_t x = gate(i, j, q), y = up(i, j, q);
            f32x4_t v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = act_value<decltype(act)::value>(x[e]) * y[e];
            return v;
          }, g.c, g.ldc, vec_c, false);
        });
      });
    } else {
      auto scaled = [&](auto i, auto j, auto q) __attribute__((always_inline)) {
        f32x4_t v = four(i, j, q);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = g.alpha * v[e];
        return v;
      };
      if (partial) {
        float* tile_sums = static_cast<float*>(g.cube) + int64_t(piece_now) * (BM * BN);
        auto sums = [&](auto i, auto j, auto q) __attribute__((always_inline)) {  // as they are (an integer's bits merely travel as a float's)
          f32x4_t v;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const typename FfnMma<Tag>::sum_t sum = acc[decltype(i)::value][decltype(j)::value][decltype(q)::value * 4 + e];
            v[e] = __builtin_bit_cast(float, sum);  // (of a vector's element directly it takes element 0)
          }
          return v;
        };
        static_for<NI>([&](auto j) __attribute__((always_inline)) { emit_at(as_float{}, j, sums, tile_sums, BM, wm * CHW, BM, wn * WTN, BN, true, false); });
      } else if (g.beta_zero) {
        static_for<NI>([&](auto j) __attribute__((always_inline)) { emit(own_size{}, j, scaled, g.c, g.ldc, vec_c, false); });
      } else {
        static_for<NI>([&](auto j) __attribute__((always_inline)) { emit(as_float{}, j, scaled, g.c, g.ldc, vec_c, true); });
      }
    }
    // (with P kept there are more stores than that: the wait is then merely earlier than it need be)
    stored = vec_c && !partial && (GATED || g.beta_zero) && ch0 + CHW <= g.m && tok0 + WTN <= g.n;
    if (next >= units) return;
    unit = next;
  }
}

// The cut tiles: slabs added in order, then scales, alpha and beta * C as in the ring's epilogue, rounded once.  Eight channels
// of one token per thread.
template <typename Tag, typename TOut, int BM, int BN>
__global__ void __launch_bounds__(256) ffn_join_kernel(const FfnArgs<TOut> g) {
  using Sum = typename FfnMma<Tag>::sum_t;
  typedef Sum sum4 __attribute__((ext_vector_type(4)));
  const int64_t v = int64_t(blockIdx.x) * 256 + threadIdx.x;
  constexpr int PER_TILE = BM * BN / 8;
  const int t = int(v / PER_TILE), at = int(v % PER_TILE) * 8;  // (the grid is whole tiles)
  int tm, tn;
  tile_coords(g.whole + t, g.tiles_m, g.tiles_n, tm, tn, BM == 256 ? RING_BAND : 0);
  const int64_t ch = int64_t(tm) * BM + at % BM, tok = int64_t(tn) * BN + at / BM;
  if (ch >= g.m || tok >= g.n) return;
  const Sum* src = static_cast<const Sum*>(g.cube) + int64_t(t) * g.slabs * (BM * BN) + at;
  sum4 lo = *reinterpret_cast<const sum4*>(src), hi = *reinterpret_cast<const sum4*>(src + 4);
  for (int s = 1; s < g.slabs; ++s) {
    src += BM * BN;
    lo += *reinterpret_cast<const sum4*>(src);
    hi += *reinterpret_cast<const sum4*>(src + 4);
  }
  TOut* out = g.c + ch + tok * g.ldc;
  const bool vec = ch + 8 <= g.m && reinterpret_cast<uintptr_t>(out) % 16 == 0;
  constexpr int QUADS = int(sizeof(TOut)) / 2;  // 16-byte pieces of the eight results
  union {
    TOut e[8];
    i32x4 q[QUADS];
  } x;
  if (vec && !g.beta_zero) {
#pragma unroll
    for (int i = 0; i < QUADS; ++i) x.q[i] = reinterpret_cast<const i32x4*>(out)[i];
  }
  const float sb = g.scale_b ? g.scale_b[tok] : 1.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const bool live = ch + e < g.m;
    const float sa = g.scale_a && live ? g.scale_a[ch + e] : 1.0f;
    float f = g.alpha * ffn_scaled(e < 4 ? lo[e & 3] : hi[e & 3], sa, sb);
    if (vec) {
      if (!g.beta_zero) f = f + g.beta * load_out(&x.e[e]);
      store_out(&x.e[e], f);
    } else if (live) {
      if (!g.beta_zero) f = f + g.beta * load_out(out + e);
      store_out(out + e, f);
    }
  }
  if (vec) {
#pragma unroll
    for (int i = 0; i < QUADS; ++i) reinterpret_cast<i32x4*>(out)[i] = x.q[i];
  }
}

// -------------------------------------------------------------------- repack
// dst[r][0 .. row_bytes) = row r of the operand along k, zeros from k on (elements of BYTES bytes; row_bytes a multiple of 64).
// Bound by memory: the operand in and out once.
//
// Rows that lie along k already, at any alignment: one 16-byte piece per thread.
template <int BYTES>
__global__ void __launch_bounds__(256)
    ffn_pack_rows_kernel(const unsigned char* __restrict__ src, int64_t ld, unsigned char* __restrict__ dst, int64_t row_bytes, int64_t rows,
                         int64_t k) {
  const int64_t per = row_bytes / 16, v = folded_block() * 256 + threadIdx.x;
  if (v >= per * rows) return;
  const int64_t r = v / per, at = (v - r * per) * 16, kb = k * BYTES;
  const unsigned char* s = src + r * ld * BYTES + at;
  const int64_t left = kb - at;
  *reinterpret_cast<u16x8*>(dst + r * row_bytes + at) = partial_piece(s, int(left < 16 ? (left < 0 ? 0 : left) : 16), kb >= 16);
}

// Element (r, k) at r + k * ld: a tile of 256 bytes of rows by 128 bytes of k per workgroup.  A thread takes blocks of U x U elements
// (U = 4 bytes' worth): U words of U rows each, one per k, turned in registers into U words of U k each, through LDS into
// 16-byte pieces along k.  Whole cache lines both ways (8-bit 50400 x 4096: element by element 0.9 ms).
constexpr int PACK_K_BYTES = 128, PACK_R_BYTES = 256;
template <int BYTES>
__global__ void __launch_bounds__(256)
    ffn_pack_across_kernel(const unsigned char* __restrict__ src, int64_t ld, unsigned char* __restrict__ dst, int64_t row_bytes, int64_t rows,
                           int64_t k) {
  constexpr int U = 4 / BYTES, ROWS = PACK_R_BYTES / BYTES, KS = PACK_K_BYTES / BYTES;
  constexpr int PITCH = PACK_K_BYTES + 4;  // bytes of a tile row in LDS
  typedef uint32_t u32_at1 __attribute__((aligned(1)));
  __shared__ uint32_t tile[ROWS * PITCH / 4];
  const int64_t k_tiles = (row_bytes + PACK_K_BYTES - 1) / PACK_K_BYTES;
  const int64_t r0 = folded_block() / k_tiles * ROWS, k0 = folded_block() % k_tiles * KS;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t r = r0 + lane * U;
  uint32_t in[KS / U / 4][U];
#pragma unroll
  for (int b = 0; b < KS / U / 4; ++b)  // this wavefront's blocks along k: b * 4 + wave
#pragma unroll
    for (int e = 0; e < U; ++e) {
      const int64_t kk = k0 + (b * 4 + wave) * U + e;
      const unsigned char* s = src + (r + kk * ld) * BYTES;
      uint32_t w = 0;
      if (kk < k) {
        if (r + U <= rows) {
          w = *reinterpret_cast<const u32_at1*>(s);
        } else {
          for (int i = 0; r + i < rows; ++i)
            for (int j = 0; j < BYTES; ++j) w |= uint32_t(s[i * BYTES + j]) << (8 * (i * BYTES + j));
        }
      }
      in[b][e] = w;
    }
#pragma unroll
  for (int b = 0; b < KS / U / 4; ++b) {
    uint32_t out[U];
    if constexpr (BYTES == 2) {
      out[0] = (in[b][0] & 0xffffu) | (in[b][1] << 16);
      out[1] = (in[b][0] >> 16) | (in[b][1] & 0xffff0000u);
    } else {
      // bytes of (a, b): v_perm's selector counts the second operand's bytes 0-3, the first's 4-7
      const uint32_t lo01 = __builtin_amdgcn_perm(in[b][1], in[b][0], 0x05010400u), lo23 = __builtin_amdgcn_perm(in[b][3], in[b][2], 0x05010400u);
      const uint32_t hi01 = __builtin_amdgcn_perm(in[b][1], in[b][0], 0x07030602u), hi23 = __builtin_amdgcn_perm(in[b][3], in[b][2], 0x07030602u);
      out[0] = (lo01 & 0xffffu) | (lo23 << 16);
      out[1] = (lo01 >> 16) | (lo23 & 0xffff0000u);
      out[2] = (hi01 & 0xffffu) | (hi23 << 16);
      out[3] = (hi01 >> 16) | (hi23 & 0xffff0000u);
    }
#pragma unroll
    for (int i = 0; i < U; ++i) tile[(lane * U + i) * (PITCH / 4) + b * 4 + wave] = out[i];
  }
  __syncthreads();
  constexpr int PIECES = PACK_K_BYTES / 16;
#pragma unroll
  for (int i = 0; i < ROWS * PIECES / 256; ++i) {
    const int p = i * 256 + threadIdx.x, row = p / PIECES, piece = p % PIECES;
    const int64_t at = k0 * BYTES + piece * 16;
    if (r0 + row < rows && at < row_bytes) {
      const uint32_t* t = tile + row * (PITCH / 4) + piece * 4;
      const i32x4 v = {int(t[0]), int(t[1]), int(t[2]), int(t[3])};
      *reinterpret_cast<i32x4*>(dst + (r0 + row) * row_bytes + at) = v;
    }
  }
}

// -------------------------------------------------------------- quantisation
// Storage -> float, eight elements at any address.
struct F32Tag {};
template <typename Tag>
struct QuantIn {
  using type = uint16_t;
  __device__ static inline void load8(const uint16_t* p, float (&v)[8]) {
    const u16x8 x = *reinterpret_cast<const u16x8_at1*>(p);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = widen(Tag{}, x[e]);
  }
  __device__ static inline float load(const uint16_t* p) { return widen(Tag{}, *p); }
};
template <>
struct QuantIn<F32Tag> {
  using type = float;
  typedef f32x4_t f32x4_at4 __attribute__((aligned(4)));
  __device__ static inline void load8(const float* p, float (&v)[8]) {
    const f32x4_t x = *reinterpret_cast<const f32x4_at4*>(p), y = *reinterpret_cast<const f32x4_at4*>(p + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = x[e], v[4 + e] = y[e];
  }
  __device__ static inline float load(const float* p) { return *p; }
};

// The integer nearest to 127 x / largest, ties to even, as of the real quotient.  x * (127 / largest) in float is off by
// less than 127 * 2^-23 < 2^-16, so only a result within 2^-14 of a half can round to the wrong side; those few (and
// everything where 127 / largest does not fit a float) are divided in double: 127 x is exact there, and a quotient that is
// no tie differs from one by more than 2^-33, so the double's rounding cannot make or break a tie.
__device__ inline int quant_round(float x, float inv, float largest, bool tiny) {
  const float r = x * inv;
  const float q = __builtin_rintf(r);
  if (tiny || __builtin_fabsf(r - q) > 0.5f - 0x1p-14f) return int(__builtin_rint(127.0 * double(x) / double(largest)));
  return int(q);
}

// A column on TPC consecutive threads (64 or 256 / 1024: a whole workgroup).  Each thread keeps HOLD vectors of eight elements in
// registers between finding the maximum and rounding, so a column is read once; what a longer column has beyond is
// read again.  Bound by memory: 2 (4) bytes in and 1 out per element.
template <typename Tag, int TPC, int HOLD>
__global__ void __launch_bounds__(TPC < 256 ? 256 : TPC)
    ffn_quantize_kernel(int64_t m, int64_t n, const typename QuantIn<Tag>::type* __restrict__ x, int64_t ldx, int8_t* __restrict__ q,
                        int64_t ldq, float* __restrict__ scale) {
  using In = QuantIn<Tag>;
  constexpr int COLS = TPC < 256 ? 256 / TPC : 1;
  typedef uint32_t u32x2_at1 __attribute__((ext_vector_type(2), aligned(1)));
  const int t = threadIdx.x % TPC;
  const int64_t col = folded_block() * COLS + threadIdx.x / TPC;
  const bool live = col < n;  // (whole wavefronts are live or not)
  const typename In::type* src = x + (live ? col : n - 1) * ldx;
  const int64_t vecs = m / 8;
  float held[HOLD][8];
  uint32_t top = 0;  // the maximum of |x| as bits: a NaN is above infinity, infinity above all else
  auto look = [&](float v) {
    const uint32_t b = __float_as_uint(v) & 0x7fffffffu;
    top = b > top ? b : top;
  };
#pragma unroll
  for (int i = 0; i < HOLD; ++i) {
    const int64_t v = t + int64_t(i) * TPC;
    if (v < vecs) {
      In::load8(src + v * 8, held[i]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) held[i][e] = 0.0f;
    }
  }
#pragma unroll
  for (int i = 0; i < HOLD; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) look(held[i][e]);
  for (int64_t v = t + int64_t(HOLD) * TPC; v < vecs; v += TPC) {
    float y[8];
    In::load8(src + v * 8, y);
#pragma unroll
    for (int e = 0; e < 8; ++e) look(y[e]);
  }
  const int64_t last = vecs * 8 + t;  // the odd elements behind the last vector: one per thread
  const float odd = last < m ? In::load(src + last) : 0.0f;
  look(odd);
#pragma unroll
  for (int s = 32; s; s >>= 1) {
    const uint32_t o = __shfl_xor(top, s, 64);
    top = o > top ? o : top;
  }
  if constexpr (TPC > 64) {
    __shared__ uint32_t tops[TPC / 64];
    if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < TPC / 64; ++w) top = tops[w] > top ? tops[w] : top;
  }
  if (!live) return;
  const float largest = __uint_as_float(top);
  if (t == 0) scale[col] = largest / 127.0f;
  const bool blank = top == 0 || top >= 0x7f800000u;  // nothing but zeros, or something not finite: all zeros
  const bool tiny = largest < 1e-30f;                  // 127 / largest could overflow
  const float inv = blank || tiny ? 0.0f : 127.0f / largest;
  int8_t* dst = q + col * ldq;
  auto store8 = [&](int64_t v, const float (&y)[8]) {
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int r = blank ? 0 : quant_round(y[e], inv, largest, tiny);
      w[e / 4] |= uint32_t(uint8_t(int8_t(r))) << (8 * (e % 4));
    }
    u32x2_at1 out = {w[0], w[1]};
    *reinterpret_cast<u32x2_at1*>(dst + v * 8) = out;
  };
#pragma unroll
  for (int i = 0; i < HOLD; ++i) {
    const int64_t v = t + int64_t(i) * TPC;
    if (v < vecs) store8(v, held[i]);
  }
  for (int64_t v = t + int64_t(HOLD) * TPC; v < vecs; v += TPC) {
    float y[8];
    In::load8(src + v * 8, y);
    store8(v, y);
  }
  if (last < m) dst[last] = int8_t(blank ? 0 : quant_round(odd, inv, largest, tiny));
}

// -------------------------------------------------- gradient, elementwise half
// dG = dC U act'(G), dU = dC act(G): eight channels of one token per thread.  p and dp may be the same matrix: a thread
// reads what it overwrites, and nothing else, before it writes.  (Hence no __restrict__ on them.)
// dP is rounded to the storage type because the products' matrix instructions take 16-bit operands (a second, low half of it
// would double their time): dA and dB carry sqrt(2) of one rounding's error (relative to 64 bits, half 2.9e-4 where one
// rounding makes 2.1e-4, bfloat16 2.4e-3 and 1.7e-3).  copy: NULL, or a second
// dP with aligned rows of ld_copy (a multiple of 8) elements, zeros behind 2m, for products that need whole 16-byte pieces.
template <typename Tag, typename TOut>
__global__ void __launch_bounds__(256)
    ffn_gate_grad_kernel(int act, int64_t m, int64_t n, const uint16_t* p, int64_t ldp, const uint16_t* dc, int64_t lddc, uint16_t* dp,
                         int64_t lddp, uint16_t* copy, int64_t ld_copy) {
  const int64_t per = (m + 7) / 8;
  const int64_t v = folded_block() * 256 + threadIdx.x;
  if (v >= per * n) return;
  const int64_t col = v / per, i = (v - col * per) * 8;
  const uint16_t* pg = p + col * ldp + i;
  const uint16_t* pd = dc + col * lddc + i;
  uint16_t* out = dp + col * lddp + i;
  uint16_t* also = copy + col * ld_copy + i;
  with_act(act, [&](auto act_tag) {
  auto one = [&](uint16_t gb, uint16_t ub, uint16_t db, uint16_t& dg, uint16_t& du) {
    float value, slope;
    act_value_slope<decltype(act_tag)::value>(widen(Tag{}, gb), value, slope);
    const float d = widen(Tag{}, db), u = widen(Tag{}, ub);
    // d u may pass the float range where a small slope brings the product back (0 times the infinity would be NaN); the
    // slope goes first there: with |d u| >= 2^128 both are above 1, so nothing underflows that the slope itself kept
    float du_slope = d * u * slope;
    if constexpr (std::is_same<Tag, Bf16Tag>::value) {  // (two halves stay below 2^32)
      if (__builtin_fabsf(d * u) > 3.4028234663852886e38f) du_slope = d * slope * u;
    }
    TOut og, ou;
    store_out(&og, du_slope);
    store_out(&ou, d * value);
    dg = __builtin_bit_cast(uint16_t, og);
    du = __builtin_bit_cast(uint16_t, ou);
  };
  if (i + 8 <= m) {
    const u16x8 gv = *reinterpret_cast<const u16x8_at1*>(pg), uv = *reinterpret_cast<const u16x8_at1*>(pg + m);
    const u16x8 dv = *reinterpret_cast<const u16x8_at1*>(pd);
    u16x8 og, ou;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      uint16_t x, y;
      one(gv[e], uv[e], dv[e], x, y);
      og[e] = x;
      ou[e] = y;
    }
    *reinterpret_cast<u16x8_at1*>(out) = og;
    *reinterpret_cast<u16x8_at1*>(out + m) = ou;
    if (copy) {
      *reinterpret_cast<u16x8_at1*>(also) = og;
      *reinterpret_cast<u16x8_at1*>(also + m) = ou;
    }
  } else {
    for (int e = 0; i + e < m; ++e) {
      uint16_t x, y;
      one(pg[e], pg[m + e], pd[e], x, y);
      out[e] = x;
      out[m + e] = y;
      if (copy) {
        also[e] = x;
        also[m + e] = y;
      }
    }
  }
  });
  if (copy && i + 8 >= m)  // the thread of a token's last channels
    for (int64_t e = 2 * m; e < ld_copy; ++e) copy[col * ld_copy + e] = 0;
}

}  // namespace sbamd
