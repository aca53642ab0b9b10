// The tile loop of the flash attention kernels as text for their bodies (one wave's view; see prefill.hip for the design): its
// V reads, products and softmax, one key tile, the prologue and the loop over the tiles. The kernel has defined
//   D, RG, IPW, CPR, DT, NQ, Sm, ks_, vs_        its shapes and LDS stages
//   lane, fr, fk, kh, qf, scale_log2             the lane's place and its Q fragments
//   nt, n_full                                   key tiles, and how many at the front hold no masked key for this wave
//   issue_k(i, st), issue_v(i, st)               DMA instruction i of the next K (V) tile into stage st
//   advance(st)                                  called once before the DMA of each K tile (into stage st) but the first: ahead
//                                                of the others by first_advance()
//   kFeed                                        kFeedDma, or kFeedWiden: the prologue has filled the stages already; issue_k(i, st) and
//                                                issue_v(i, st) are vector work and a write to LDS, codes_v() comes before the latter,
//                                                and refill() follows the last of a tile
//   before_barrier(), after_barrier()            called around the prologue's barrier, before n_full is read
//   kGuard, odd_tile                             whether infinities and NaN in V are taken out of masked tiles, and the first
//                                                tile where any were (INT_MAX)
//   enter_masked(t), hidden(t, kt, e)            whether the lane's query does not see element e of key block kt of tile t
//   xor32(v)                                     lane l ^ 32's v
//   m_i, l_i, o                                  the row's reference max (-inf), the lane's share of its sum (0), O^T (0)
//   live(t)                                      whether the wave's keys of tile t are visible to any of its rows; never again once false
// and is left with m_i (the same in lanes l and l ^ 32), l_i (over the lane's own keys) and o (O^T).
  // transpose reads of V: lane j of each 16-lane group g reads 4 d of key 4 (g / 2) + j / 4 (+ the
  // step's key base), d = 16 (g % 2) + 4 (j % 4) (+ the output tile's d base); the group's lane i
  // then holds d = 16 (g % 2) + i of those 4 keys. Keys of one read are 4-aligned, so the swizzle
  // term is the lane's own.
  const int vr = 4 * fk + ((lane & 15) >> 2);                  // key within a 16-key step
  const int vc0 = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);   // logical chunk within a 32-d tile
  const f16* vb[DT];                                           // the lane's first read of each output tile
#pragma unroll
  for (int dt = 0; dt < DT; dt++)
    vb[dt] = reinterpret_cast<const f16*>(vs_) + (kFpKPW * kh + vr) * D + 8 * ((4 * dt + vc0) ^ v_swz<D>(vr)) + 4 * (lane & 1);
  const int kr = kFpKPW * kh + fr;                             // K row of this lane's first fragments
  const int ksw = k_swz<D>(kr);                                // the same for every block (kr % 16)
  // S^T = K Q^T over 32-key block kt of the wave's keys in K stage st; lane (row fr, half fk) gets
  // keys 32 kt + 8 g + 4 fk + e
  auto logits = [&](int st, int kt, f32x16& s) {
    f32x16 a;
#pragma unroll
    for (int e = 0; e < 16; e++) a[e] = 0.f;
#pragma unroll
    for (int ks = 0; ks < NQ; ks++) {
      const f16x8 kf = __builtin_bit_cast(f16x8, ks_[st * Sm::kTile + (kr + 32 * kt) * CPR + ((2 * ks + fk) ^ ksw)]);
      a = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, qf[ks], a, 0, 0, 0);
    }
    s = a;
  };
  // the V^T fragments of block kt (V stage st): of step ss, lane half fk holds keys 32 kt + 16 ss +
  // 4 fk + 0..3 and 32 kt + 16 ss + 8 + 4 fk + 0..3 of the wave's keys, as P's registers do
  auto load_v = [&](int st, int kt, f16x8 (&vf)[2][DT]) {
#pragma unroll
    for (int ss = 0; ss < 2; ss++)
#pragma unroll
      for (int dt = 0; dt < DT; dt++) {
        const f16* pa = vb[dt] + st * (Sm::kTile * 8) + (32 * kt + 16 * ss) * D;
        const f16x4 fa = lds_read_tr16(pa), fb = lds_read_tr16(pa + 8 * D);  // key + 8: same swizzle term
        vf[ss][dt] = f16x8{fa[0], fa[1], fa[2], fa[3], fb[0], fb[1], fb[2], fb[3]};
      }
  };
  // O^T += V^T P^T of one 32-key block
  auto pv = [&](const f16x8 (&vf)[2][DT], const f16x8 (&pf)[2]) {
#pragma unroll
    for (int ss = 0; ss < 2; ss++)
#pragma unroll
      for (int dt = 0; dt < DT; dt++) o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[ss][dt], pf[ss], o[dt], 0, 0, 0);
  };
  // p = exp2(c s - m) of one block, its sum into l_i, fp16 p in P.V operand order
  auto softmax = [&](const f32x16& s, float m_use, f16x8 (&pf)[2]) {
    float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
    for (int e = 0; e < 16; e += 2) {
      const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], scale_log2, -m_use));
      const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e + 1], scale_log2, -m_use));
      sum0 += p;
      sum1 += p1;
      pf[e >> 3][e & 7] = (f16)p;
      pf[e >> 3][(e & 7) + 1] = (f16)p1;
    }
    l_i += sum0 + sum1;
  };

  // Infinities and NaN in the V rows of a masked tile t: a row that does not see them has weight 0 there, and 0 times either is
  // NaN. They leave the fragments, and the kernel gives them to the rows that do see them.
  auto guard = [&](int t, f16x8 (&vf)[2][DT]) __attribute__((always_inline)) {
    uint32_t odd = 0;
#pragma unroll
    for (int ss = 0; ss < 2; ss++)
#pragma unroll
      for (int dt = 0; dt < DT; dt++) {
        const u32x4 w = __builtin_bit_cast(u32x4, vf[ss][dt]);
#pragma unroll
        for (int i = 0; i < 4; i++) odd |= (w[i] & 0x7fff7fffu) + 0x04000400u;  // an exponent of ones carries into the sign
      }
    if (!__any((odd & 0x80008000u) != 0)) return;
    odd_tile = min(odd_tile, t);
#pragma unroll
    for (int ss = 0; ss < 2; ss++)
#pragma unroll
      for (int dt = 0; dt < DT; dt++) {
        u32x4 w = __builtin_bit_cast(u32x4, vf[ss][dt]);
#pragma unroll
        for (int i = 0; i < 4; i++) {
          if ((w[i] & 0x7c00u) == 0x7c00u) w[i] &= 0xffff0000u;
          if ((w[i] & 0x7c000000u) == 0x7c000000u) w[i] &= 0x0000ffffu;
        }
        vf[ss][dt] = __builtin_bit_cast(f16x8, w);
      }
  };

  // One key tile t (stage t & 1, given as a constant in the main loop): the softmax and P.V of its
  // logits sc, with the logits of tile t + 1 into sn in between. A wave issues in order, so the
  // MFMAs of one product are interleaved with the vector work of the other tile's softmax by
  // scheduling groups; otherwise each product's MFMAs run back to back, then the softmax with the
  // matrix cores idle (both waves of a SIMD leave the tile's barrier together). The P.V of the
  // tile's second block (pl, its V fragments vl read before the next barrier) runs after that
  // barrier: matrix work that needs no LDS while the first K fragments are on their way.
  f16x8 pl[2], vl[2][DT];
#pragma unroll
  for (int ss = 0; ss < 2; ss++) {
    pl[ss] = f16x8{};
#pragma unroll
    for (int dt = 0; dt < DT; dt++) vl[ss][dt] = f16x8{};
  }
  auto tile = [&](auto stc, auto maskc, auto nextc, int t, f32x16 (&sc)[2], f32x16 (&sn)[2]) {
    constexpr bool MASK = decltype(maskc)::value;  // the tile holds keys past some row's diagonal
    constexpr bool NEXT = decltype(nextc)::value;  // there is a tile t + 1
    const int st = stc;
    wait_lgkm0();
    wait_vmcnt<0>();     // this wave's shares of K tile t + 1 and V tile t are in LDS
    barrier_no_fence();  // every share is, and every wave is done with K tile t and V tile t - 1
    advance(st);
    if constexpr (MASK) {
      enter_masked(t);
#pragma unroll
      for (int kt = 0; kt < 2; kt++)
#pragma unroll
        for (int e = 0; e < 16; e++)
          if (hidden(t, kt, e)) sc[kt][e] = -__builtin_huge_valf();
    }
    // the row's reference max m_i moves only when the tile's scaled max exceeds it by more than 2^8,
    // so p = exp2(c s - m_i) stays at most 256 (exact range for fp16 P and fp32 sums) and O is
    // rescaled only then; lanes l and l ^ 32 then agree on the new one. The max of the raw logits is
    // scaled once (c > 0 keeps the order) and c s - m_i is one fma
    // The MFMAs of this tile up to its first P.V, in slots: the last block's P.V, then (NEXT) the
    // logits of tile t + 1. The 2 IPW DMA instructions of K tile t + 2 and V tile t + 1 go out over the
    // slots of the first logits block; with 4 waves, each issuing twice as many and without a second
    // wave on its SIMD to fill its stalls, over all of them (64 rows after 2000 positions 26.1 ->
    // 22.6 us, 512 after 2048 36.0 -> 32.7; 8 waves: no gain, 2 % slower at T = 2048 after 4096).
    // (With kFeedWiden they go between the MFMAs of the last block's P.V, in the order written.)
    constexpr bool WIDEN = kFeed == kFeedWiden;
    constexpr int ND = WIDEN ? 0 : 2 * IPW, LA = 3;  // DMA instructions, LDS reads ahead of their MFMA
    constexpr int S0 = RG == 2 ? 0 : 2 * DT, NS = RG == 2 ? 2 * DT + 2 * NQ : NQ;
    auto dma_here = [](int m) constexpr {  // DMA instructions that go before slot m
      int n = 0;
      for (int j = 0; j < ND; j++) n += S0 + j * NS / (ND ? ND : 1) == m;
      return n;
    };
    constexpr int kDma = (ND + NS - 1) / NS;  // at most this many before one slot
    auto dma = [&](int m) {
#pragma unroll
      for (int j = 0; j < ND; j++)
        if (S0 + j * NS / (ND ? ND : 1) == m) j < IPW ? issue_k(j, st) : issue_v(j - IPW, st ^ 1);
    };
    auto load_k = [&](int kt, int ks) {
      return __builtin_bit_cast(f16x8, ks_[(st ^ 1) * Sm::kTile + (kr + 32 * kt) * CPR + ((2 * ks + fk) ^ ksw)]);
    };
    float mx = -__builtin_huge_valf();
    f16x8 kf[NQ];
    f32x16 a0;
#pragma unroll
    for (int e = 0; e < 16; e++) a0[e] = 0.f;
#pragma unroll
    for (int m = 0; m < 2 * DT; m++) {
      if constexpr (NEXT) {
        dma(m);
        if (m >= 2 * DT - LA) kf[m - (2 * DT - LA)] = load_k(0, m - (2 * DT - LA));
      }
      o[m % DT] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vl[m / DT][m % DT], pl[m / DT], o[m % DT], 0, 0, 0);
      if constexpr (NEXT && WIDEN) {
        constexpr int PER = IPW / DT;  // chunks a slot: K's in the first half of the slots, V's in the second
        static_assert(PER * DT == IPW, "chunks per slot");
        if (m == DT / 2 - 1) codes_v();
#pragma unroll
        for (int j = m * PER; j < (m + 1) * PER; j++) j < IPW ? issue_k(j, st) : issue_v(j - IPW, st ^ 1);
        if (m == 2 * DT - 1) refill();
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if constexpr (NEXT) {
#pragma unroll
      for (int ks = 0; ks < NQ; ks++) {
        dma(2 * DT + ks);
        if (ks + LA < NQ) kf[ks + LA] = load_k(0, ks + LA);
        a0 = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[ks], qf[ks], a0, 0, 0, 0);
      }
      sn[0] = a0;
    }
#pragma unroll
    for (int kt = 0; kt < 2; kt++)
#pragma unroll
      for (int e = 0; e < 16; e++) mx = fmaxf(mx, sc[kt][e]);
    constexpr int kMaskOps = MASK ? 8 : 0;  // more vector work per MFMA
#pragma unroll
    for (int m = 0; m < (NEXT && WIDEN ? 0 : 2 * DT); m++) {
      if (NEXT && dma_here(m)) __builtin_amdgcn_sched_group_barrier(0x020, kDma, 0);  // DMA
      if (NEXT && m >= 2 * DT - LA) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);  // LDS read
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);             // MFMA (the last block's P.V)
      __builtin_amdgcn_sched_group_barrier(0x002, 2 + kMaskOps, 0);  // VALU (the max)
    }
    if constexpr (NEXT) {
#pragma unroll
      for (int ks = 0; ks < NQ; ks++) {
        if (dma_here(2 * DT + ks)) __builtin_amdgcn_sched_group_barrier(0x020, kDma, 0);
        if (ks + LA < NQ) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);           // MFMA (logits)
        __builtin_amdgcn_sched_group_barrier(0x002, 2, 0);
      }
    }
    if (__any(mx * scale_log2 > m_i + kFpMaxLag)) {  // m_i = -inf: moves to the first finite max
      mx = fmaxf(mx, xor32(mx)) * scale_log2;
      const bool move = mx > m_i + kFpMaxLag;
      const float alpha = move ? __builtin_amdgcn_exp2f(m_i - mx) : 1.f;
      if (move) m_i = mx;
      l_i *= alpha;
#pragma unroll
      for (int dt = 0; dt < DT; dt++)
#pragma unroll
        for (int e = 0; e < 16; e++) o[dt][e] *= alpha;
    }
    // m_i is -inf only for a row that has seen no key yet (one whose first key lies in the other
    // half): every logit is then -inf and every p 0
    const float m_use = m_i == -__builtin_huge_valf() ? 0.f : m_i;
    f16x8 pf[2], vf[2][DT];
    if constexpr (NEXT) {
      f32x16 a1;
#pragma unroll
      for (int e = 0; e < 16; e++) a1[e] = 0.f;
#pragma unroll
      for (int ks = 0; ks < LA; ks++) kf[ks] = load_k(1, ks);
#pragma unroll
      for (int ks = 0; ks < NQ; ks++) {
        dma(2 * DT + NQ + ks);
        if (ks + LA < NQ) kf[ks + LA] = load_k(1, ks + LA);
        a1 = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[ks], qf[ks], a1, 0, 0, 0);
      }
      sn[1] = a1;
    }
    softmax(sc[0], m_use, pf);
    load_v(st, 0, vf);
    if constexpr (MASK && kGuard) guard(t, vf);
    pv(vf, pf);
    softmax(sc[1], m_use, pl);
    load_v(st, 1, vl);
    if constexpr (MASK && kGuard) guard(t, vl);
    if constexpr (NEXT) {
      __builtin_amdgcn_sched_group_barrier(0x100, LA, 0);
#pragma unroll
      for (int ks = 0; ks < NQ; ks++) {
        if (dma_here(2 * DT + NQ + ks)) __builtin_amdgcn_sched_group_barrier(0x020, kDma, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        if (ks + LA >= NQ) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);             // MFMA (logits)
        __builtin_amdgcn_sched_group_barrier(0x002, 56 / NQ, 0);       // VALU (softmax of block 0)
      }
#pragma unroll
      for (int i = 0; i < 2 * DT; i++) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);             // MFMA (P.V of block 0)
        __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, 56 / (2 * DT), 0); // VALU (softmax of block 1)
      }
    }
  };

  // ---- prologue: K tiles 0 and 1 and V tile 0 in flight, the logits of tile 0
  if constexpr (kFeed == kFeedDma) {
#pragma unroll
    for (int i = 0; i < IPW; i++) issue_k(i, 0);
    first_advance();
#pragma unroll
    for (int i = 0; i < IPW; i++) {
      issue_v(i, 0);
      issue_k(i, 1);
    }
  }
  before_barrier();
  wait_vmcnt<2 * IPW>();
  barrier_no_fence();
  after_barrier();
  f32x16 sa[2], sb[2];
  logits(0, 0, sa[0]);
  logits(0, 1, sa[1]);
  constexpr std::integral_constant<int, 0> kEven{};
  constexpr std::integral_constant<int, 1> kOdd{};
  int t = 0;
  const std::true_type yes{};
  const std::false_type no{};
  for (; t + 2 <= n_full && t + 2 < nt; t += 2) {
    tile(kEven, no, yes, t, sa, sb);
    tile(kOdd, no, yes, t + 1, sb, sa);
  }
  // The other tiles may hold masked keys. A wave leaves out a tile whose keys (its half) lie wholly past
  // its rows' diagonal or the block's last key, as it does every later one, but for its share of the
  // DMA and the barrier: their weights are 0, but 0 times an infinity or NaN in a later row's V is not.
  for (; t + 1 < nt; t++) {  // an odd full tile, the first of two tiles on the diagonal
    if (live(t)) {
      tile(t & 1, yes, yes, t, sa, sb);
      sa[0] = sb[0];
      sa[1] = sb[1];
    } else {
      wait_lgkm0();
      wait_vmcnt<0>();
      barrier_no_fence();
      advance(t & 1);
      if constexpr (kFeed == kFeedWiden) codes_v();
#pragma unroll
      for (int i = 0; i < IPW; i++) {
        issue_k(i, t & 1);
        issue_v(i, (t & 1) ^ 1);
      }
      if constexpr (kFeed == kFeedWiden) refill();
    }
  }
  if (live(t)) {
    tile(t & 1, yes, no, t, sa, sb);
  } else {
    wait_lgkm0();
    wait_vmcnt<0>();
    barrier_no_fence();
  }

  pv(vl, pl);

