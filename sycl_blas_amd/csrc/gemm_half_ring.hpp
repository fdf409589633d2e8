// The ring's K loop: acc += (the tile of op(A)) * (the tile of op(B)) over k_len, after ring_start has set off the first tiles.
// A piece of a function's body, included where it runs (so no include guard).  In scope: Tag, OpA, OpB, MI, NI, WTM, WTN,
// acc, oa, ob, lda, ldb, k_len, smem, tid, lane, wave, wm, wn, and
//   ABLATE   a timing-only diagnostic, see gemm_mfma16_ring_kernel;
//   M_FIRST  a lane ends up with one index of A (lane & 31) and sixteen of B, else the other way round;
//   STORES, stores  `stores` says that at least STORES vector stores were issued behind the first tiles' loads: memory
//            operations complete in order, so these tiles are waited for without waiting for those stores.
// Included, not called, by the GEMM: as a function's parameters these were turned into addresses before the kernel's
// constants were known, and the prologue and the last steps came out longer (bf16 1024^3 9.87 -> 10.04 us, half 2048^3
// 23.7 -> 23.9).
  constexpr int NM = MI * NI;   // matrix instructions per half step
  constexpr int NPA = OpA::NP, NPB = OpB::NP;    // load instructions per thread and tile of each operand
  constexpr int LPA = NPA / 2, LPH = LPA + NPB / 2;  // of them per half step: A's, both operands'
  constexpr int RING_OPERAND_BYTES = OpA::BYTES;  // offset of the B image inside a stage
  constexpr int RING_STAGE_BYTES = OpA::BYTES + OpB::BYTES;
  const int nk = int(k_len / RING_BK);

  auto stage_ptr = [&](int t) { return smem + (t % RING_STAGES) * RING_STAGE_BYTES; };

  // tile 0 must have landed for every wave before anyone reads it (the tiles behind it may be in flight)
  static_assert((RING_AHEAD - 1) * (NPA + NPB) + STORES < 64, "the counter's range");
  if (STORES > 0 && stores && nk > RING_AHEAD - 1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((RING_AHEAD - 1) * (NPA + NPB) + STORES) : "memory");
  else if (nk > RING_AHEAD - 1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((RING_AHEAD - 1) * (NPA + NPB)) : "memory");
  else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();

  u16x8 fa[2][MI], fb[2][NI];
  // Read unit U of a half step: the B fragments first, then the A fragments.
  auto read_unit = [&](auto unit_tag, auto s_tag, const SBAMD_LDS unsigned char* st, u16x8 (&xa)[MI], u16x8 (&xb)[NI]) {
    constexpr int U = decltype(unit_tag)::value, S = decltype(s_tag)::value;
    if constexpr (U < NI) xb[U] = OpB::template fragment<S>(st + RING_OPERAND_BYTES, wn * WTN + U * 32, lane);
    else xa[U - NI] = OpA::template fragment<S>(st, wm * WTM + (U - NI) * 32, lane);
  };
  using yes = std::integral_constant<bool, true>;
  using no = std::integral_constant<bool, false>;

  // One half step with its issue order written out: matrix instruction n, then read
  // unit n of the NEXT half step (six units for eight matrix instructions), a load
  // piece behind the third and the sixth.  sched_barrier(0) keeps the compiler from
  // regrouping; the operands of the matrix instructions were waited for before the
  // last barrier, so nothing in here stalls on memory.
  auto half_step = [&](auto s_next_tag, auto loads_tag, auto reads_tag, auto piece_tag, const SBAMD_LDS unsigned char* st_next,
                       SBAMD_LDS unsigned char* fill, u16x8 (&ca)[MI], u16x8 (&cb)[NI], u16x8 (&na)[MI], u16x8 (&nb)[NI]) {
    constexpr bool LOADS = decltype(loads_tag)::value, READS = decltype(reads_tag)::value;
    constexpr int PIECE = decltype(piece_tag)::value;
    auto slot = [&](auto n_tag) {
      constexpr int N = decltype(n_tag)::value;
      constexpr int I = N / NI, J = N % NI;
      if constexpr (!(ABLATE & 2)) acc[I][J] = M_FIRST ? Mfma16<Tag>::mma(cb[J], ca[I], acc[I][J]) : Mfma16<Tag>::mma(ca[I], cb[J], acc[I][J]);
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (READS && N < MI + NI && !(ABLATE & 4)) read_unit(std::integral_constant<int, N>{}, s_next_tag, st_next, na, nb);
      if constexpr (LOADS && !(ABLATE & 1)) {
        // this half step's load instructions (A's pieces, then B's) behind matrix instructions 2 and 5 of
        // eight, 1 and 3 of four, 2 / 6 / 10 / 14 of sixteen
        static_for<LPH>([&](auto l_tag) {
          constexpr int L = decltype(l_tag)::value;
          constexpr int AT = LPH == 2 ? (L == 0 ? NM / 4 : NM / 2 + NM / 4 - (NM > 4 ? 1 : 0)) : (2 * L + 1) * NM / (2 * LPH);
          if constexpr (N == AT) {
            if constexpr (L < LPA) oa.template issue_piece<PIECE * LPA + L>(fill, wave);
            else ob.template issue_piece<PIECE * (LPH - LPA) + L - LPA>(fill + RING_OPERAND_BYTES, wave);
          }
        });
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    static_for<NM>(slot);
  };
  static_assert((NM == 16 || NM == 8 || NM == 4) && MI + NI <= NM, "wave tiles of 128 x 128, 128 x 64 and 64 x 64");

  // first fragments of tile 0
  {
    static_for<MI + NI>([&](auto u) { read_unit(u, std::integral_constant<int, 0>{}, smem, fa[0], fb[0]); });
  }

  // One K step.  LOADS: tile t + RING_AHEAD exists and is issued here; NEXT: tile
  // t + 1 exists.
  auto step = [&](const SBAMD_LDS unsigned char* cur, const SBAMD_LDS unsigned char* next, SBAMD_LDS unsigned char* fill,
                  auto loads_tag, auto next_tag, auto extra_tag) {
    constexpr bool LOADS = decltype(loads_tag)::value;
    constexpr int EXTRA = decltype(extra_tag)::value;  // stores that may still be out as well

    // the fragments fetched during the previous half step must have arrived (the
    // transposing reads are inline assembly: the compiler does not wait for them)
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);

    // first half step: matrix work on k 0..15, fragments of k 16..31, piece 0 of A and B
    half_step(std::integral_constant<int, 1>{}, loads_tag, yes{}, std::integral_constant<int, 0>{}, cur, fill, fa[0], fb[0],
              fa[1], fb[1]);

    // every fragment read of tile t has returned; own pieces of tile t + 1 have landed
    // (in flight and allowed to stay so: tiles t + 2 .. t + RING_AHEAD - 1 and the first half of tile t + RING_AHEAD)
    if (LOADS && !(ABLATE & 1)) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((RING_AHEAD - 2) * (NPA + NPB) + LPH + EXTRA) : "memory");
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);

    // second half step: matrix work on k 16..31, first fragments of tile t + 1, piece 1
    half_step(std::integral_constant<int, 0>{}, loads_tag, next_tag, std::integral_constant<int, 1>{}, next, fill, fa[1],
              fb[1], fa[0], fb[0]);
    if (LOADS) {
      oa.advance(lda);
      ob.advance(ldb);
    }
  };
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the first fragments
  __builtin_amdgcn_sched_barrier(0);

  // Steady state: five steps per trip, one per ring stage, so that every LDS address is the lane's offset plus a
  // compile-time constant.
  int t = 0;
  using none = std::integral_constant<int, 0>;
  if constexpr (STORES > 0) {
    // the tiles that were in flight before the stores: RING_AHEAD - 1 of them are waited for in steps 0 .. RING_AHEAD - 2
    if (stores && t + RING_STAGES - 1 + RING_AHEAD < nk) {
      static_for<RING_STAGES>([&](auto i_tag) {
        constexpr int I = decltype(i_tag)::value;
        step(smem + I * RING_STAGE_BYTES, smem + (I + 1) % RING_STAGES * RING_STAGE_BYTES, smem + (I + RING_STAGES - 1) % RING_STAGES * RING_STAGE_BYTES,
             yes{}, yes{}, std::integral_constant<int, (I < RING_AHEAD - 1 ? STORES : 0)>{});
      });
      t = RING_STAGES;
    }
  }
  for (; t + RING_STAGES - 1 + RING_AHEAD < nk; t += RING_STAGES) {
    static_for<RING_STAGES>([&](auto i_tag) {
      constexpr int I = decltype(i_tag)::value;
      step(smem + I * RING_STAGE_BYTES, smem + (I + 1) % RING_STAGES * RING_STAGE_BYTES, smem + (I + RING_STAGES - 1) % RING_STAGES * RING_STAGE_BYTES, yes{},
           yes{}, none{});
    });
  }
  // the remaining steps (t is a multiple of RING_STAGES here) with the stage computed at run time
  for (; t + RING_AHEAD < nk; ++t) step(stage_ptr(t), stage_ptr(t + 1), stage_ptr(t + RING_AHEAD), yes{}, yes{}, none{});
  for (; t + 1 < nk; ++t) step(stage_ptr(t), stage_ptr(t + 1), stage_ptr(t + RING_AHEAD), no{}, yes{}, none{});
  if (t < nk) step(stage_ptr(t), stage_ptr(t + 1), stage_ptr(t + RING_AHEAD), no{}, no{}, none{});

  // K tail (k % 32 valid k): one more tile, zero-padded, staged through registers into stage 0 once every
  // wavefront has finished the last ring step; the zeros add nothing to the sums.
  const int k_rem = int(k_len - int64_t(nk) * RING_BK);
  if (k_rem > 0) {
    __syncthreads();
    u16x8 ta[NPA], tb[NPB];
    static_for<NPA>([&](auto i) { ta[decltype(i)::value] = oa.template load_tail<decltype(i)::value>(k_rem, tid); });
    static_for<NPB>([&](auto i) { tb[decltype(i)::value] = ob.template load_tail<decltype(i)::value>(k_rem, tid); });
    static_for<NPA>([&](auto i) { OpA::template store_tail<decltype(i)::value>(smem, tid, ta[decltype(i)::value]); });
    static_for<NPB>([&](auto i) { OpB::template store_tail<decltype(i)::value>(smem + RING_OPERAND_BYTES, tid, tb[decltype(i)::value]); });
    __syncthreads();
    auto tail_half = [&](auto s_tag) {
      static_for<MI + NI>([&](auto u) { read_unit(u, s_tag, smem, fa[0], fb[0]); });
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the transposing reads are not tracked by the compiler
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) acc[i][j] = M_FIRST ? Mfma16<Tag>::mma(fb[0][j], fa[0][i], acc[i][j]) : Mfma16<Tag>::mma(fa[0][i], fb[0][j], acc[i][j]);
      __builtin_amdgcn_sched_barrier(0);
    };
    tail_half(std::integral_constant<int, 0>{});
    if (k_rem > 16) tail_half(std::integral_constant<int, 1>{});
  }
