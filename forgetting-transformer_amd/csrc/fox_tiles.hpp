// Tiles of the attention kernels: what one wave does with a key tile (forward, dQ) or a step of query rows (dK/dV).  The kernels
// around them (fox_fwd.hip, fox_bwd.hip, fox_packed.hip) find the tiles, bring them into LDS and store the results.
#pragma once
#include "fox_common.hpp"
#include "fox_kernels.hpp"

namespace fox {

// ---------------------------------------------------------------------------
// Forward
// ---------------------------------------------------------------------------
constexpr float kLazyMaxLog2 = 8.0f;
constexpr int kMinPipelinedTiles = 4;   // interior tiles below which the software-pipelined path is not entered

template <typename Tr, int D>
__device__ __forceinline__ void fwd_tile(const char* k_tile, const char* v_tile, const float* cn_s, const u32x4 (&qreg)[D / 16],
                                f32x16 (&oacc)[(D + 31) / 32], float& m_i, float& l_i, int n0, int a_m, float qk_scale,
                                int lane, bool diag) {
  constexpr int BN = kFwdBN, KK = D / 16, DB = (D + 31) / 32, NB = BN / 32;
  const int g = lane >> 5, i = lane & 31;

  // S^T = K Q^T + key term
  f32x16 s[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    u32x4 ka[KK];
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) ka[kk] = lds_row_operand<D>(k_tile, 32 * nb + i, 2 * kk + g);
    s[nb] = acc_init(cn_s, 32 * nb, g);
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) s[nb] = Tr::mfma32(ka[kk], qreg[kk], s[nb]);
  }

  // scores in the log2 domain and their maximum
  float mloc = -INFINITY;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int r = 0; r < 16; ++r) s[nb][r] *= qk_scale;
  if (diag) {  // causal compare, only on tiles that cross the diagonal
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int n = n0 + 32 * nb + c_row(r, g);
        s[nb][r] = (n > a_m) ? -INFINITY : s[nb][r];
      }
  }
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int r = 0; r < 16; ++r) mloc = fmaxf(mloc, s[nb][r]);
  mloc = half_max(mloc);
  const bool raise = mloc > m_i + kLazyMaxLog2;
  if (__any(raise)) {  // rare: rescale what has been accumulated so far
    const float m_new = raise ? mloc : m_i;
    const float alpha = __builtin_amdgcn_exp2f(m_i - m_new);
    m_i = m_new;
    l_i *= alpha;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) oacc[db][r] *= alpha;
  }
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int r = 0; r < 16; ++r) s[nb][r] = __builtin_amdgcn_exp2f(s[nb][r] - m_i);

  // O^T += V^T P^T.  The row sum is taken over the probabilities as rounded for the MFMA (the weights that
  // multiply V then add up to exactly l), two at a time: per-lane partial sum, the two halves are added in the epilogue.
  float rsum = 0.f;
#pragma unroll
  for (int sl = 0; sl < BN / 16; ++sl) {
    const u32x4 pb = pack8<Tr>(s[sl >> 1], 8 * (sl & 1));
#pragma unroll
    for (int e = 0; e < 4; ++e) rsum = Tr::add_pair(pb[e], rsum);
    u32x4 va[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db) va[db] = lds_col_operand<D>(v_tile, 16 * sl, db, lane);
#pragma unroll
    for (int db = 0; db < DB; ++db) oacc[db] = Tr::mfma32(va[db], pb, oacc[db]);
  }
  l_i += rsum;
}

// Interior tile (no key of the tile is right of any query row of the workgroup): branch-free and
// software-pipelined across tiles.  While the vector ALU turns the scores of the current tile into
// probabilities, the matrix pipe already computes the scores of the next tile (from k_next) and then
// accumulates the current tile's P V (from v_cur).  s_cur holds the raw scores of the current tile
// on entry; s_next holds those of the next tile on exit.  Work is issued in small chunks separated
// by scheduling fences so that MFMA and vector instructions alternate in the instruction stream.
// dma(u) issues chunk u's share of the global loads of the tiles after next: spread over the tile they
// do not hold the wave's issue slot back to back right after the barrier.
// ROW_TERM: m_i counts the term of the row, and the row sum is taken over the probabilities in 32 bits, for a backward whose probabilities are to add up to one
// better than their 16-bit rounding does (fox_packed.hip).
template <typename Tr, int D, bool ROW_TERM = false, typename Dma>
__device__ __forceinline__ void fwd_tile_pipelined(const char* k_next, const char* v_cur, const float* cn_next,
                                                  const u32x4 (&qreg)[D / 16], f32x16 (&oacc)[(D + 31) / 32], float& m_i,
                                                  float& l_i, float qk_scale, int lane, f32x16 (&s_cur)[kFwdBN / 32],
                                                  f32x16 (&s_next)[kFwdBN / 32], Dma dma, float row_term = 0.f) {
  constexpr int BN = kFwdBN, KK = D / 16, DB = (D + 31) / 32, NB = BN / 32, NSL = BN / 16;
  constexpr int SPC = 16 * NB / KK;  // scores handled per chunk of phase A
  static_assert(16 * NB % KK == 0 && SPC % 4 == 0, "whole float4 groups of scores per chunk");
  const int g = lane >> 5, i = lane & 31;

  // Phase A: scores of the next tile  ||  maximum of the current tile's raw scores (sm_scale > 0 here)
  float mloc = -INFINITY;
  u32x4 ka[NB][KK + 1];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    ka[nb][0] = lds_row_operand<D>(k_next, 32 * nb + i, g);
    s_next[nb] = acc_init(cn_next, 32 * nb, g);
  }
  static_for<0, KK>([&](auto uc) {
    constexpr int u = decltype(uc)::value;
    dma(u);  // this chunk's share of the global loads of the tiles after next
    if constexpr (u + 1 < KK) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) ka[nb][u + 1] = lds_row_operand<D>(k_next, 32 * nb + i, 2 * (u + 1) + g);
    }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) s_next[nb] = Tr::mfma32(ka[nb][u], qreg[u], s_next[nb]);
#pragma unroll
    for (int e = 0; e < SPC; ++e) {
      const int idx = u * SPC + e;
      mloc = fmaxf(mloc, s_cur[idx >> 4][idx & 15]);
    }
#pragma unroll
    for (int k = 0; k < NB; ++k) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x002, (SPC / 2 + NB - 1) / NB, 0);  // the chunk's v_max3 dealt out over its MFMAs
    }
    __builtin_amdgcn_sched_barrier(0);
  });
  mloc = half_max(mloc) * qk_scale;
  if constexpr (ROW_TERM) mloc += row_term;
  const bool raise = mloc > m_i + kLazyMaxLog2;
  if (__any(raise)) {  // rare: rescale what has been accumulated so far
    const float m_new = raise ? mloc : m_i;
    const float alpha = __builtin_amdgcn_exp2f(m_i - m_new);
    m_i = m_new;
    l_i *= alpha;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) oacc[db][r] *= alpha;
  }

  // Phase B: p = exp2(s*scale - m), row sums, pack  ||  O^T += V^T P^T, one 16-key slice behind
  const float neg_m = ROW_TERM ? row_term - m_i : -m_i;
  float rsum = 0.f;
  u32x4 pb[NSL];
  u32x4 va[NSL][DB];
#pragma unroll
  for (int c = 0; c <= NSL; ++c) {
    if (c < NSL) {
#pragma unroll
      for (int db = 0; db < DB; ++db) va[c][db] = lds_col_operand<D>(v_cur, 16 * c, db, lane);
    }
    if (c >= 1) {
#pragma unroll
      for (int db = 0; db < DB; ++db) oacc[db] = Tr::mfma32(va[c - 1][db], pb[c - 1], oacc[db]);
    }
    if (c < NSL) {
      const int nb = c >> 1, r0 = 8 * (c & 1);
#pragma unroll
      for (int e = 0; e < 8; ++e) s_cur[nb][r0 + e] = __builtin_amdgcn_exp2f(fmaf(s_cur[nb][r0 + e], qk_scale, neg_m));
      pb[c] = pack8<Tr>(s_cur[nb], r0);
      if constexpr (ROW_TERM) {
#pragma unroll
        for (int e = 0; e < 8; ++e) rsum += s_cur[nb][r0 + e];
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) rsum = Tr::add_pair(pb[c][e], rsum);  // row sum of the rounded probabilities
      }
    }
    if (c >= 1 && c < NSL) {
#pragma unroll
      for (int k = 0; k < DB; ++k) {  // a slice has 16 vector (20 with ROW_TERM) and 8 exp instructions: dealt out over its DB MFMAs
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, (ROW_TERM ? 20 : 16) / DB, 0);
        __builtin_amdgcn_sched_group_barrier(0x400, 8 / DB, 0);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  l_i += rsum;
}

// The global loads of a K tile and a V tile, dealt out over the D/16 chunks of a pipelined tile:
// dma(u) issues chunk u's share.
template <int D, int AUX>
struct TileDma {
  static constexpr int KK = D / 16, PER = DirectTileLoader<D, kFwdBN, 4, AUX>::PER, PER_CHUNK = (2 * PER + KK - 1) / KK;
  const DirectTileLoader<D, kFwdBN, 4, AUX>& kld;
  const DirectTileLoader<D, kFwdBN, 4, AUX>& vld;
  const uint16_t* k_src;
  const uint16_t* v_src;
  int k_bytes, v_bytes;
  char* k_fill;
  char* v_fill;
  __device__ __forceinline__ void all() const {
#pragma unroll
    for (int j = 0; j < PER; ++j) kld.issue_one(j, k_src, k_bytes, k_fill);
#pragma unroll
    for (int j = 0; j < PER; ++j) vld.issue_one(j, v_src, v_bytes, v_fill);
  }
  __device__ __forceinline__ void operator()(int u) const {  // u is a constant at every call site
#pragma unroll
    for (int r = 0; r < PER_CHUNK; ++r) {
      const int idx = u * PER_CHUNK + r;
      if (idx < PER) kld.issue_one(idx, k_src, k_bytes, k_fill);
      else if (idx < 2 * PER) vld.issue_one(idx - PER, v_src, v_bytes, v_fill);
    }
  }
};

// ---------------------------------------------------------------------------
// One step (BMQ query rows) of the dK/dV kernel for one wave (32 key rows).
// rc_s holds rowc_i / (sm_scale*log2e) and dl_s holds -delta_i.  The wave accumulates the NDB 32-column
// blocks of dK and dV that start at block db0 (all of them, or one half of the head dim when two waves
// share a block of keys).
template <typename Tr, int D, int BMQ = kKvBM, int NDB = (D + 31) / 32>
__device__ __forceinline__ void dkdv_step(const char* q_tile, const char* do_tile, const float* rc_s, const float* dl_s,
                                 const u32x4 (&kreg)[D / 16], const u32x4 (&vreg)[D / 16], f32x16 (&dkacc)[NDB],
                                 f32x16 (&dvacc)[NDB], float& csum, int a_s0, int n, int n_w0, float qk_scale,
                                 float colc, int lane, int db0 = 0) {
  constexpr int KK = D / 16, MB = BMQ / 32;
  const int g = lane >> 5, i = lane & 31;
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) {
    const int a_b0 = a_s0 + 32 * mb;   // key position of the block's first query row
    if (a_b0 + 31 < n_w0) continue;    // block entirely above the diagonal for this wave
    f32x16 s = acc_init(rc_s, 32 * mb, g), dp = acc_init(dl_s, 32 * mb, g);
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) s = Tr::mfma32(lds_row_operand<D>(q_tile, 32 * mb + i, 2 * kk + g), kreg[kk], s);
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) dp = Tr::mfma32(lds_row_operand<D>(do_tile, 32 * mb + i, 2 * kk + g), vreg[kk], dp);
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], qk_scale, -colc));
    if (a_b0 < n_w0 + 31) {  // causal compare, only on blocks that cross the diagonal
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = (n > a_b0 + c_row(r, g)) ? 0.f : s[r];
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const float ds = s[r] * dp[r];
      dp[r] = ds;
      csum += ds;
    }
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
      const u32x4 pb = pack8<Tr>(s, 8 * hh);
      const u32x4 dsb = pack8<Tr>(dp, 8 * hh);
#pragma unroll
      for (int db = 0; db < NDB; ++db) {
        dvacc[db] = Tr::mfma32(lds_col_operand<D>(do_tile, 32 * mb + 16 * hh, db0 + db, lane), pb, dvacc[db]);
        dkacc[db] = Tr::mfma32(lds_col_operand<D>(q_tile, 32 * mb + 16 * hh, db0 + db, lane), dsb, dkacc[db]);
      }
    }
  }
}

// Interior step (every query row of the step sits at or below every key of the
// tile: no causal compare, nothing to skip): branch-free and software-pipelined by
// hand, because the kernel holds one wave per SIMD and nobody else can fill the
// matrix pipe while this wave does its exp/scale arithmetic.  The step is cut
// into slots; slot b issues, interleaved in chunks of 4 MFMAs + 2 scores,
//   * the score MFMAs        S, dP   of block b+1,
//   * the vector arithmetic  P, dS   of block b,
//   * the accumulation MFMAs dV, dK  of block b-1,
// which are mutually independent (one MFMA, then a few vector instructions, four times per chunk, in source order
// between scheduling fences).  The global loads of the next tile are spread over
// the step as well (dma(k) issues the k-th of NDMA instructions): issued back to back
// after the barrier by all four waves they would hold every wave's issue slot, and
// with one wave per SIMD the matrix pipe, for over a thousand cycles per step.
// The LDS operands of a chunk are requested three
// chunks (about twelve MFMAs) ahead, across slot boundaries, so their latency hides
// behind the chunks in between.
template <typename Tr, int D, int NDMA, typename Dma>
__device__ __forceinline__ void dkdv_step_interior(const char* q_tile, const char* do_tile, const float* rc_s, const float* dl_s,
                                          const u32x4 (&kreg)[D / 16], const u32x4 (&vreg)[D / 16],
                                          f32x16 (&dkacc)[(D + 31) / 32], f32x16 (&dvacc)[(D + 31) / 32], float& csum,
                                          float qk_scale, float colc, int lane, Dma dma) {
  constexpr int BMQ = kKvBM, KK = D / 16, DB = (D + 31) / 32, MB = BMQ / 32;
  // chunks per slot: as many as the larger of the two MFMA groups needs (one k-step of S and dP, one accumulation
  // pair of dV and dK per chunk), so that every chunk carries matrix work; the 16 scores per lane of a block are
  // dealt out evenly over them
  constexpr int NCH = KK > 2 * DB ? KK : 2 * DB, SPC = 16 / NCH;
  static_assert(16 % NCH == 0 && (SPC == 2 || SPC == 4 || SPC == 8), "whole scores per chunk, whole operands per 8 scores");
  constexpr int NC = (MB + 2) * NCH;  // chunks of the step: slots -1 .. MB
  constexpr int PF = 3;               // LDS operands are requested this many chunks before their MFMAs
  constexpr int kDmaEvery = (NC - NCH) / (NDMA > 0 ? NDMA : 1) > 0 ? (NC - NCH) / (NDMA > 0 ? NDMA : 1) : 1;
  static_assert(NDMA * kDmaEvery <= NC - NCH, "every load instruction of the next tile finds a chunk");
  static_assert(KK <= NCH && 2 * DB <= NCH, "one k-step and one accumulation pair per chunk");
  const int g = lane >> 5, i = lane & 31;
  f32x16 s[MB], dp[MB];
  u32x4 pb[MB][2], dsb[MB][2];
  u32x4 aq[NC + PF], ado[NC + PF], cq[NC + PF], cdo[NC + PF];  // indexed by chunk; only a few are live at a time
  auto fetch = [&](auto ic) {
    constexpr int c = decltype(ic)::value;
    constexpr int slot = c / NCH - 1, u = c % NCH, bs = slot + 1, bc = slot - 1;
    if constexpr (c < NC && bs < MB && u < KK) {
      aq[c] = lds_row_operand<D>(q_tile, 32 * bs + i, 2 * u + g);
      ado[c] = lds_row_operand<D>(do_tile, 32 * bs + i, 2 * u + g);
    }
    if constexpr (c < NC && slot >= 1 && u < 2 * DB) {
      cdo[c] = lds_col_operand<D>(do_tile, 32 * bc + 16 * (u / DB), u % DB, lane);
      cq[c] = lds_col_operand<D>(q_tile, 32 * bc + 16 * (u / DB), u % DB, lane);
    }
  };
  // the accumulators of block b start from the row terms instead of zero; requested PF chunks early too
  auto init_block = [&](int b) {  // b is a constant at every call site
    if (b < MB) {
      s[b] = acc_init(rc_s, 32 * b, g);
      dp[b] = acc_init(dl_s, 32 * b, g);
    }
  };
  init_block(0);
  static_for<0, PF>([&](auto ic) { fetch(ic); });
  static_for<0, NC>([&](auto ic) {
    constexpr int c = decltype(ic)::value;
    constexpr int slot = c / NCH - 1, u = c % NCH;
    constexpr bool do_s = slot + 1 < MB, do_v = slot >= 0 && slot < MB, do_c = slot >= 1;
    constexpr int bs = slot + 1, bv = slot, bc = slot - 1;
    fetch(std::integral_constant<int, c + PF>{});
    if constexpr (u == (NCH > PF ? NCH - PF : 0)) init_block(bs + 1);
    // the next tile's load instructions, one every kDmaEvery chunks from the second slot on
    if constexpr (c >= NCH && (c - NCH) % kDmaEvery == 0 && (c - NCH) / kDmaEvery < NDMA)
      dma(std::integral_constant<int, (c - NCH) / kDmaEvery>{});
    // The chunk in issue order, every group fenced so that matrix and vector instructions alternate: S MFMA, exp2 of
    // SPC scores, dP MFMA, dS and the column sum of those scores, dV MFMA, pack P (when eight scores are complete),
    // dK MFMA, pack dS.  S and dP accumulate in VGPRs (mfma32_vgpr_acc), so this code keeps the distance between an
    // MFMA that writes s[b] / dp[b] and the first vector instruction that reads them (12 issued instructions).  Block
    // b's last S MFMA opens chunk NCH-1 of slot b-1 and its first score is read in chunk 0 of slot b, after that
    // chunk's S MFMA.  For b >= 1 the instructions in between are the 2*SPC exp2 / fma, the dP MFMA, the 2*SPC multiply
    // / add and the 8 packs of chunk NCH-1 (it completes eight scores), then the next chunk's operand requests and
    // S MFMA: >= 20.  dP's last MFMA is followed by 2*SPC + 8 of those, the requests, the S MFMA and 2*SPC exp2 / fma
    // before dS reads it: >= 18.  Block 0 is computed in a slot without vector work, so its first chunk of vector
    // work starts with explicit wait states.
    constexpr bool mf_s = do_s && u < KK, mf_c = do_c && u < 2 * DB;
    constexpr bool pack_due = do_v && (SPC * (u + 1)) % 8 == 0;   // eight scores complete: one MFMA operand each of P and dS
    constexpr int hh = pack_due ? SPC * (u + 1) / 8 - 1 : 0;
    static_assert(SPC >= 2 && NCH * SPC == 16, "the distances above count on at least two scores per chunk, eight per pack");
    if constexpr (mf_s) Tr::mfma32_vgpr_acc(s[bs], aq[c], kreg[u]);
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (do_v && bv == 0 && u == 0) {
      asm volatile("s_nop 11");
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (do_v) {
#pragma unroll
      for (int e = 0; e < SPC; ++e) s[bv][SPC * u + e] = __builtin_amdgcn_exp2f(fmaf(s[bv][SPC * u + e], qk_scale, -colc));
    }
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (mf_s) Tr::mfma32_vgpr_acc(dp[bs], ado[c], vreg[u]);
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (do_v) {
#pragma unroll
      for (int e = 0; e < SPC; ++e) {
        const float ds = s[bv][SPC * u + e] * dp[bv][SPC * u + e];
        dp[bv][SPC * u + e] = ds;
        csum += ds;
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (mf_c) dvacc[u % DB] = Tr::mfma32(cdo[c], pb[bc][u / DB], dvacc[u % DB]);
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (pack_due) pb[bv][hh] = pack8<Tr>(s[bv], 8 * hh);
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (mf_c) dkacc[u % DB] = Tr::mfma32(cq[c], dsb[bc][u / DB], dkacc[u % DB]);
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (pack_due) dsb[bv][hh] = pack8<Tr>(dp[bv], 8 * hh);
    __builtin_amdgcn_sched_barrier(0);
  });
}

// Two elements' part of delta.  (One expression for both walks, with the rounding spelled out.)
template <typename Tr>
__device__ __forceinline__ float delta_term(uint32_t o, uint32_t d_o) {
  return __builtin_fmaf(Tr::lo(o), Tr::lo(d_o), Tr::hi(o) * Tr::hi(d_o));
}

// ---------------------------------------------------------------------------
// One 64-key tile of the dQ kernel for one wave (32 query rows).
// cn_s holds -colc_j / (sm_scale*log2e), the start value of the score accumulators.
template <typename Tr, int D>
__device__ __forceinline__ void dq_tile(const char* k_tile, const char* v_tile, const float* cn_s, const u32x4 (&qreg)[D / 16],
                               const u32x4 (&doreg)[D / 16], f32x16 (&dqacc)[(D + 31) / 32], float& rsum, int n0, int a_m,
                               int a_w0, float qk_scale, float rowc, float delta, int lane) {
  constexpr int BN = kFwdBN, KK = D / 16, DB = (D + 31) / 32, NB = BN / 32;
  const int g = lane >> 5, i = lane & 31;
  // dP starts from -delta (constant along a query row, i.e. per lane) instead of zero: the matrix pipe does the
  // subtraction.  The sixteen equal registers are loop-invariant for the caller.
  f32x16 neg_delta;
#pragma unroll
  for (int r = 0; r < 16; ++r) neg_delta[r] = -delta;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const int nb0 = n0 + 32 * nb;
    if (nb0 > a_w0 + 31) continue;  // block entirely above this wave's rows
    f32x16 s = acc_init(cn_s, 32 * nb, g);
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) s = Tr::mfma32(lds_row_operand<D>(k_tile, 32 * nb + i, 2 * kk + g), qreg[kk], s);
    f32x16 dp = Tr::mfma32(lds_row_operand<D>(v_tile, 32 * nb + i, g), doreg[0], neg_delta);
#pragma unroll
    for (int kk = 1; kk < KK; ++kk) dp = Tr::mfma32(lds_row_operand<D>(v_tile, 32 * nb + i, 2 * kk + g), doreg[kk], dp);
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], qk_scale, rowc));
    if (nb0 + 31 > a_w0) {  // causal compare, only on blocks that cross the diagonal
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = (nb0 + c_row(r, g) > a_m) ? 0.f : s[r];
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const float ds = s[r] * dp[r];
      dp[r] = ds;
      rsum += ds;
    }
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
      const u32x4 dsb = pack8<Tr>(dp, 8 * hh);
#pragma unroll
      for (int db = 0; db < DB; ++db)
        dqacc[db] = Tr::mfma32(lds_col_operand<D>(k_tile, 32 * nb + 16 * hh, db, lane), dsb, dqacc[db]);
    }
  }
}

}  // namespace fox
