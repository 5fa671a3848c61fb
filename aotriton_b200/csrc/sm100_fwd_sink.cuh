// Forward of sink attention (a sliding window and a few first keys) for head dims up to 128.  Included by sm100_fwd.cu inside its
// namespaces; the arithmetic is the tile kernel's.
//
// A window is a few blocks of keys, so what the tile kernel does once for a long row of blocks -- set up, fill the pipeline, write out -- is most of
// a CTA's time here, and a step's chain (S ready, softmax, P V, the next Q K^T into the same columns) is what the rest waits for: with a CTA of
// two tiles to an SM, 10 us beside 2.2 us for each block of both tiles; with one tile a CTA and two CTAs an SM, 1500 of a step's 4000 clocks went by
// between a softmax and the next scores.  So here
//   * a CTA owns one tile of 128 query rows, two CTAs share an SM: one works while the other starts or ends;
//   * blocks are of 64 keys, and S has two buffers of 64 columns: Q K^T runs a block and a half ahead of the softmax, which finds the next scores
//     ready; a window's edges, masked along a diagonal, cost half as many keys that nobody sees; first keys are one such block;
//   * warps as in the tile kernel: 0 TMA, 1 MMA issuer, 4-7 softmax (thread = query row), half the registers of an SM to a CTA.
// Tensor memory (256 columns): S0 [0,64)  S1 [64,128)  O [128,128+HD); P (32 packed columns) over its S.  Shared memory: Q, two stages each of K and V.
// order on the tensor pipe:  S_0 S_1 | O += P_0 V_0, S_2 | O += P_1 V_1, S_3 | ...
// Measured on the device, bf16, 1 x 32:8 heads x 8192 of 128, 4 first keys, us, two tiles to a CTA / one with blocks of 128 keys / this: window 2048
// 310 / 282 / 249, 1024 229 / 192 / 167 (0.98 PFLOP/s of products that are issued), 512 151 / 140 / 122, 128 101 / 95 / 85.  At window 1024 the tensor pipe and the
// exponential unit are each busy 45% of the time (56% in the tile kernel on a long row), L2 27%: what is left is a step's chain in a softmax warp, loads
// from tensor memory, maximum, exponentials, store, of which two warps a scheduler overlap.  CTAs that stay and walk over the tiles (the
// next Q loaded under the last blocks, O staged beside it) came out 1 to 5% slower: the second CTA of the SM covers a start as well, and the hardware hands tiles out in the order they end.
// Every wait is bounded.

constexpr int kSinkBN = 64, kSinkThreads = 256;

template <int HD>
struct SinkSmem {
  static constexpr int kHalves = HD / 64;
  static constexpr int kQBox = 16384, kBox = 8192;           // 128 / 64 rows x 64 columns x 2 bytes
  static constexpr int kQBytes = kHalves * kQBox, kTile = kHalves * kBox;
  static constexpr int kQ = 0, kK = kQBytes, kV = kK + 2 * kTile, kBars = kV + 2 * kTile;
  static constexpr int bQFull = 0, bKFull = 1, bKEmpty = 3, bVFull = 5, bVEmpty = 7, bSFull = 9, bPFull = 11, bPvDone = 13, bCount = 15;
  static constexpr int kTmemSlot = kBars + bCount * 8;
  static constexpr int kAbort = kTmemSlot + 8;               // abort word, then the launch's wait limit
  static constexpr int kDynamic = kAbort + 8 + 1024;         // slack for manual 1024-byte alignment
  static constexpr uint32_t kTmemCols = 256, kColO = 128;
};
static_assert(2 * (SinkSmem<128>::kDynamic + 1024) <= 228 * 1024, "two CTAs an SM");

// EXACT as in the tile kernel (lengths multiples of 128)
template <typename T, int HD, bool EXACT>
__global__ void __launch_bounds__(kSinkThreads, 2)
sm100_fwd_sink_kernel(const __grid_constant__ Params p, const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                      const __grid_constant__ CUtensorMap tm_v, unsigned int* status) {
  wait_for_earlier_grids();
  using L = SinkSmem<HD>;
  constexpr int kBlk = kSinkBN;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBars);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kTmemSlot);
  volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(smem + L::kAbort);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // Order of the CTAs as in the tile kernel: groups of 32 (batch, head) pairs, the row tiles of a group slowest.
  int z = blockIdx.z, h = blockIdx.y, m0 = (int)(gridDim.x - 1 - blockIdx.x) * kBM;
  if (!p.hw_order) {
    constexpr int kHeadGroup = 32;
    const int nx = (int)gridDim.x, nh = (int)gridDim.y, nhz = nh * (int)gridDim.z;
    const int lin = (int)blockIdx.x + nx * ((int)blockIdx.y + nh * (int)blockIdx.z);
    const int grp = quick_div(lin, kHeadGroup * nx), r = lin - grp * (kHeadGroup * nx);
    const int gsize = min(kHeadGroup, nhz - grp * kHeadGroup);
    const int xi = quick_div(r, gsize), hz = grp * kHeadGroup + (r - xi * gsize);
    z = quick_div(hz, nh);
    h = hz - z * nh;
    m0 = (nx - 1 - xi) * kBM;
  }
  const unsigned int failed_before = *reinterpret_cast<volatile unsigned int*>(status);      // (decided on behind the set-up)
  if (warp == 2 && lane == 0) { prefetch_tmap(&tm_q); prefetch_tmap(&tm_k); prefetch_tmap(&tm_v); }
  int4 ends;
  if (!EXACT && p.packed_tiles > 0) {      // one-dimensional grid: the heads of a tile next to each other
    const int tile = quick_div((int)blockIdx.x, p.hq);
    h = (int)blockIdx.x - tile * p.hq;
    if (!packed_tile<kBM>(p, tile, lane, z, m0, ends)) return;
  } else if (p.varlen_mode != 0) {
    ends = make_int4(p.cu_q[z], p.cu_q[z + 1], p.cu_k[z], p.cu_k[z + 1]);
  }
  const Seq sq = seq_for<kSinks>(p, z, ends);
  if (p.varlen_mode == 2 && m0 + kBM > sq.sq) write_rows_behind<T>(p, sq, h, m0, kBM);
  if (m0 >= sq.sq) return;
  const int hk = quick_div(h, p.group);
  int n_lo, n_hi;
  key_range(p, sq, m0, min(m0 + kBM, sq.sq) - 1, n_lo, n_hi);
  if (n_hi < n_lo) {      // CTA-uniform: nothing to attend to
    write_dead_rows<T>(p, sq, h, m0, kBM);
    return;
  }
  const int jb_lo = n_lo / kBlk, before = blocks_before<kSinks>(p, n_hi, jb_lo, kBlk);
  const int nblk = before + n_hi / kBlk - jb_lo + 1;
  auto block = [&](int j) { return block_at<kSinks>(j, before, jb_lo); };
  auto load = [&](const CUtensorMap* map, int base, int full, int j) {      // K or V of block j
    const int s = j & 1, row = (int)(sq.k0 + (int64_t)block(j) * kBlk);
    mbar_expect_tx(&bars[full + s], L::kTile);
    for (int hf = 0; hf < L::kHalves; ++hf)
      tma_load_4d(smem + base + s * L::kTile + hf * L::kBox, map, &bars[full + s], hf * 64, row, hk, sq.bidx);
  };

  // ---- set-up -----------------------------------------------------------------------
  if (threadIdx.x == 0) {
    init_abort_and_limit(abort_flag, p.wait_limit_kcycles);
    mbar_init(&bars[L::bQFull], 1);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&bars[L::bKFull + s], 1);
      mbar_init(&bars[L::bKEmpty + s], 1);
      mbar_init(&bars[L::bVFull + s], 1);
      mbar_init(&bars[L::bVEmpty + s], 1);
      mbar_init(&bars[L::bSFull + s], 1);
      mbar_init(&bars[L::bPFull + s], 4);      // one arrival per softmax warp
      mbar_init(&bars[L::bPvDone + s], 1);     // (S_j there means P V of block j-2 done, not of j-1: one for even, one for odd blocks)
    }
    fence_barrier_init();
    // Q and the first block of K are requested right away, before the CTA-wide synchronisation and the tensor-memory allocation.
    mbar_expect_tx(&bars[L::bQFull], L::kQBytes);
    for (int hf = 0; hf < L::kHalves; ++hf)
      tma_load_4d(smem + L::kQ + hf * L::kQBox, &tm_q, &bars[L::bQFull], hf * 64, (int)(sq.q0 + m0), h, sq.bidx);
    load(&tm_k, L::kK, L::bKFull, 0);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, L::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  const bool leave = __syncthreads_or(failed_before != 0u) != 0;      // (one CTA-wide decision)
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  if (leave) {
    if (threadIdx.x == 0) {      // the copies requested above land before the CTA gives its shared memory back
      mbar_wait_quiet(&bars[L::bQFull], 0, abort_flag);
      mbar_wait_quiet(&bars[L::bKFull], 0, abort_flag);
    }
    __syncthreads();
    if (warp == 1) tmem_dealloc(tmem_base, L::kTmemCols);
    return;
  }

  if (warp < 4) {
    reg_dealloc<56>();
    if (warp == 0) {
      // =============================== TMA producer ===================================
      if (lane == 0) {
        int k_done = 1, v_done = 0;      // blocks requested
        for (int j = 0; j < nblk; ++j) {
          const uint32_t free_parity = ((uint32_t)(j >> 1) & 1u) ^ 1u;
          if (j > 0) {
            if (!mbar_wait(&bars[L::bKEmpty + (j & 1)], free_parity, abort_flag, status, 0x100 + j)) break;
            load(&tm_k, L::kK, L::bKFull, j);
            k_done = j + 1;
          }
          if (!mbar_wait(&bars[L::bVEmpty + (j & 1)], free_parity, abort_flag, status, 0x200 + j)) break;
          if (!(p.drop_copy == 1 && j == 0)) load(&tm_v, L::kV, L::bVFull, j);      // (test hook: this block's V never arrives)
          v_done = j + 1;
        }
        if (*abort_flag) {      // copies that are still in flight land before the CTA gives its shared memory back
          mbar_wait_quiet(&bars[L::bQFull], 0, abort_flag);
          for (int j = max(0, k_done - 2); j < k_done; ++j) mbar_wait_quiet(&bars[L::bKFull + (j & 1)], (uint32_t)(j >> 1) & 1u, abort_flag);
          for (int j = max(p.drop_copy == 1 ? 1 : 0, v_done - 2); j < v_done; ++j)
            mbar_wait_quiet(&bars[L::bVFull + (j & 1)], (uint32_t)(j >> 1) & 1u, abort_flag);
        }
      }
      __syncwarp();
    } else if (warp == 1) {
      // ================================ MMA issuer ====================================
      constexpr uint32_t kIdescQK = instr_desc_f16(Fmt<T>::code, 128, kBlk, 0, 0);
      const uint32_t kIdescPV = instr_desc_f16(Fmt<T>::code, 128, EXACT ? (uint32_t)HD : (uint32_t)((p.dvo + 15) & ~15), 0, 1);
      const int ksteps = EXACT ? HD / 16 : (p.dqk + 15) >> 4;
      const uint64_t q_desc = smem_desc_sw128(smem_u32(smem + L::kQ), 16, 1024);
      const uint64_t k_desc = smem_desc_sw128(smem_u32(smem + L::kK), 16, 1024);
      const uint64_t v_desc = smem_desc_sw128(smem_u32(smem + L::kV), L::kBox, 1024);
      constexpr uint32_t kStageStep = L::kTile >> 4;
      auto wait = [&](int bar, uint32_t parity, uint32_t where) {
        return __all_sync(0xffffffffu, mbar_wait(&bars[bar], parity, abort_flag, status, where)) != 0;
      };
      auto issue_qk = [&](int j) {      // S_j = Q K_j^T into buffer j & 1, whose P has been read (the pipe runs in issue order)
        if (!wait(L::bKFull + (j & 1), (uint32_t)(j >> 1) & 1u, 0x400 + j)) return false;
        tc_fence_after();
        const uint64_t kd = k_desc + (uint64_t)((uint32_t)(j & 1) * kStageStep);
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk) {
            const uint32_t in = (uint32_t)(kk & 3) * (32u >> 4), box = (uint32_t)(kk >> 2);
            if (kk < ksteps)
              mma_ss(tmem_base + (uint32_t)(j & 1) * kBlk, q_desc + box * (L::kQBox >> 4) + in, kd + box * (L::kBox >> 4) + in, kIdescQK, kk > 0 ? 1u : 0u);
          }
          mma_commit(&bars[L::bSFull + (j & 1)]);
          mma_commit(&bars[L::bKEmpty + (j & 1)]);
        }
        __syncwarp();
        return true;
      };
      bool ok = wait(L::bQFull, 0, 0x300) && issue_qk(0);
      if (ok && nblk > 1) ok = issue_qk(1);
      int hidden_from, hidden_to;
      hidden_keys(p, sq, hidden_from, hidden_to);
      for (int j = 0; ok && j < nblk; ++j) {
        const int s = j & 1, n0 = block(j) * kBlk;
        const uint32_t par = (uint32_t)(j >> 1) & 1u;
        if (!wait(L::bVFull + s, par, 0x600 + j)) break;
        // Rows of V that no query may take anything from: beyond the sequence's end, and between the first keys and the window.
        if constexpr (!EXACT) {
          if (sq.sk - n0 < kBlk) zero_rows_between(smem + L::kV + s * L::kTile, sq.sk - n0, kBlk, L::kHalves, L::kBox, lane);
        }
        const int from = max(hidden_from - n0, 0), to = min(hidden_to - n0, kBlk);
        if (from < to) zero_rows_between(smem + L::kV + s * L::kTile, from, to, L::kHalves, L::kBox, lane);
        if (!wait(L::bPFull + s, par, 0x500 + j)) break;
        tc_fence_after();
        const uint64_t vd = v_desc + (uint64_t)((uint32_t)s * kStageStep);
        const uint32_t first = (j > 0) ? 1u : 0u;
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < kBlk / 16; ++kk)
            mma_ts(tmem_base + L::kColO, tmem_base + (uint32_t)s * kBlk + (uint32_t)kk * 8u, vd + (uint32_t)kk * (2048u >> 4), kIdescPV, kk > 0 ? 1u : first);
          mma_commit(&bars[L::bPvDone + s]);
          mma_commit(&bars[L::bVEmpty + s]);
        }
        __syncwarp();
        if (j + 2 < nblk) ok = issue_qk(j + 2);
      }
    }
  } else {
    // ================================== softmax =====================================
    reg_alloc<200>();      // (56 and 200 for four warps each are the launch's 128 a thread)
    const int quarter = warp & 3, r = quarter * 32 + lane, m = m0 + r;
    const uint32_t lane_addr = tmem_base + ((uint32_t)(quarter * 32) << 16);
    const uint32_t o_addr = lane_addr + L::kColO;
    const int mb = min(m, sq.sq - 1);      // (rows beyond the sequence's end take the last row's bounds: nothing of theirs is stored)
    int row_lo = 0, row_hi = sq.sk - 1;
    {
      const int64_t lo = (int64_t)mb - sq.wl, hi = (int64_t)mb + sq.wr;
      if (lo > row_lo) row_lo = (int)(lo > 0x7fffffffLL ? 0x7fffffffLL : lo);
      if (hi < row_hi) row_hi = (int)(hi < -1 ? -1 : hi);
    }
    // the tightest bounds over the warp's rows: a block needs masking iff it is not inside them
    const int warp_lo = __reduce_max_sync(0xffffffffu, row_lo), warp_hi = __reduce_min_sync(0xffffffffu, row_hi);
    float m_used = -INFINITY, l = 0.f;
    bool ok = true;
    for (int j = 0; j < nblk; ++j) {
      const int n0 = block(j) * kBlk;
      const uint32_t s_addr = lane_addr + (uint32_t)(j & 1) * kBlk;
      // (a vote: the warp leaves as a whole)
      ok = __all_sync(0xffffffffu, mbar_wait(&bars[L::bSFull + (j & 1)], (uint32_t)(j >> 1) & 1u, abort_flag, status, 0x700 + j)) != 0;
      if (!ok) break;
      tc_fence_after();
      float sc[kBlk];
      tmem_ld32f(s_addr, sc);
      tmem_ld32f(s_addr + 32, sc + 32);
      tmem_wait_ld();
      const bool any_mask = !(n0 >= warp_lo && n0 + kBlk - 1 <= warp_hi);
      auto mask = [&] {
        if (!any_mask) return;
        if (n0 < p.sinks) mask_sink_columns<kBlk>(sc, n0, row_lo, row_hi, p.sinks, -INFINITY);
        else mask_columns<kBlk, true>(sc, n0, row_lo, row_hi, n0 >= warp_lo, -INFINITY);
      };
      auto largest = [&] {
        float m8[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) m8[c] = fmaxf(sc[2 * c], sc[2 * c + 1]);
#pragma unroll
        for (int c = 16; c < kBlk; c += 2) m8[(c >> 1) & 7] = fmax3(m8[(c >> 1) & 7], sc[c], sc[c + 1]);
        return fmaxf(fmax3(m8[0], m8[1], m8[2]), fmaxf(fmax3(m8[3], m8[4], m8[5]), fmaxf(m8[6], m8[7])));
      };
      // Scores -> exponent arguments, as in the tile kernel: raw scores with scale and maximum in one multiply-add each, or, where that
      // could round equal scores apart, scaled first.
      bool simple = p.qk_scale > 0.f;
      float mx = 0.f;
      if (simple) {
        mask();
        mx = largest() * p.qk_scale;
        const bool huge = fabsf(mx) > 1.0e6f && mx != -INFINITY && m < sq.sq;      // (rows that are not stored decide nothing)
        if (__any_sync(0xffffffffu, huge)) simple = false;
      }
      if (!simple) {
#pragma unroll
        for (int c = 0; c < kBlk; ++c) sc[c] *= p.qk_scale;
        mask();
        mx = largest();
      }
      // The reference maximum advances only when it moved by more than the threshold.
      const bool grow = mx > m_used + kRescaleThreshold;     // false when mx == -inf
      float alpha = 1.f;
      if (grow) {
        alpha = ex2(m_used - mx);                            // m_used == -inf -> 0
        m_used = mx;
      }
      if (j > 0 && __any_sync(0xffffffffu, grow)) {      // O must be complete up to block j-1 before it is rescaled
        ok = __all_sync(0xffffffffu, mbar_wait(&bars[L::bPvDone + ((j - 1) & 1)], (uint32_t)((j - 1) >> 1) & 1u, abort_flag, status, 0x800 + j)) != 0;
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < HD / 32; ++c) {
          if (c * 32 >= p.dvo) break;          // columns the P V product never writes
          uint32_t o[32];
          tmem_ld32(o_addr + c * 32, o);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
          tmem_st32(o_addr + c * 32, o);
        }
        tmem_wait_st();
      }
      const float m_safe = (m_used == -INFINITY) ? 0.f : m_used;
      const float2 scale2 = simple ? make_float2(p.qk_scale, p.qk_scale) : make_float2(1.f, 1.f), nm2 = make_float2(-m_safe, -m_safe);
      float2 s4[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) s4[c] = make_float2(0.f, 0.f);
      uint32_t pk[kBlk / 2];
#pragma unroll
      for (int c = 0; c < kBlk; c += 2) {
        const float2 a = fma2(make_float2(sc[c], sc[c + 1]), scale2, nm2);      // (times 1 is exact)
        const float2 e = make_float2(ex2(a.x), ex2(a.y));
        s4[(c >> 1) & 3] = add2(s4[(c >> 1) & 3], e);
        pk[c >> 1] = pack2<T>(e.x, e.y);      // (the type the tensor pipe takes: half a step off, 2^-8 of P in bf16; the sum keeps 32 bits)
      }
      tmem_st32(s_addr, pk);
      l = l * alpha + (((s4[0].x + s4[0].y) + (s4[1].x + s4[1].y)) + ((s4[2].x + s4[2].y) + (s4[3].x + s4[3].y)));
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars[L::bPFull + (j & 1)]);
    }
    // ---- epilogue: as in the tile kernel, through the (now idle) Q tile ----------------
    if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&bars[L::bPvDone + ((nblk - 1) & 1)], (uint32_t)((nblk - 1) >> 1) & 1u, abort_flag, status, 0x900)) != 0;
    if (ok) {
      tc_fence_after();
      const float inv = (l > 0.f) ? 1.f / l : 0.f;
      const uint32_t stage = smem_u32(smem + L::kQ);
#pragma unroll
      for (int c = 0; c < HD / 32; c += 2) {
        if (c * 32 >= p.dvo) break;
        float o[2][32];
        tmem_ld32f(o_addr + c * 32, o[0]);
        tmem_ld32f(o_addr + c * 32 + 32, o[1]);
        tmem_wait_ld();
        stage_put32<T>(stage, r, c * 32, o[0], inv, HD * 2);
        if (c * 32 + 32 < p.dvo) stage_put32<T>(stage, r, c * 32 + 32, o[1], inv, HD * 2);
      }
      __syncwarp();
      warp_copy_out<T, HD / 8>(stage, reinterpret_cast<T*>(p.out.ptr) + (int64_t)sq.bidx * p.out.s[0] + (int64_t)h * p.out.s[1] + (sq.q0 + m0) * p.out.s[2],
                               p.out.s[2], min(kBM, sq.sq - m0), p.dvo, quarter * 32, 0, lane, HD * 2);
      if (p.lse != nullptr && m < sq.sq)
        p.lse[lse_offset(p, sq, h) + m] = (l > 0.f) ? (m_used + log2f(l)) * kLn2 : INFINITY;
    }
  }

  // ---- tear-down ------------------------------------------------------------------------
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, L::kTmemCols);
  }
}
