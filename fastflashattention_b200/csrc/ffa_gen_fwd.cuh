// ffa_gen_fwd.cuh — forward of general attention (ffa_gen_common.cuh) for sm_100a.
//
//   O_i = sum_j softmax_j(S_ij) v_j,   LSE_i = base-2 log-sum-exp of S_i (-inf: no key)
//
// The plan of the plain forward (ffa_fwd.cuh): a CTA owns 256 queries of one head as two
// 128-row tiles; two softmax warpgroups (thread = row), a TMA warp and an MMA warp; S and O
// in tensor memory, P handed back through it in two 64-key halves; the running max is
// rescaled lazily.  What differs:
//   * operands are 4-D tensor maps, so any strides of batch, head and row do, and the key
//     head of a query head is found by division;
//   * the number of key tiles follows the sequence's own length and offset;
//   * a tile whose relative positions all lie in the last bucket of a side has one bias: it
//     joins the row max and the exponent's constant for free.  Only tiles near the diagonal
//     look the bias up, one shared-memory word for each score;
//   * with few CTAs the keys are split: each split writes its normalised O in fp32 and its
//     LSE, and ffa_gen_join_kernel weighs them (2^(LSE - max LSE)).
#pragma once
#include "ffa_fwd.cuh"
#include "ffa_gen_common.cuh"

namespace ffa {
namespace gen {

template <int D, bool BIAS>
struct FwdLayout {
  static constexpr int TILE = 128 * D * 2;
  static constexpr int STAGES = 3;
  static constexpr int Q_OFF = 0;
  static constexpr int KV_OFF = 2 * TILE;
  static constexpr int TAB_OFF = KV_OFF + STAGES * TILE;
  static constexpr int BAR_OFF = TAB_OFF + (BIAS ? (kTableMax * 4 + 15) / 16 * 16 : 0);
  // q_full, kv_full[3], kv_empty[3], s_full[2], p_ready[2], o_final[2], drain, p_half[2], exp_done[2]
  static constexpr int NBARS = 1 + 2 * STAGES + 2 + 2 + 2 + 1 + 2 + 2;
  static constexpr int MISC_OFF = BAR_OFF + NBARS * 8;
  static constexpr int SMEM_BYTES = MISC_OFF + 16 + 1024;
};

template <int D, bool CAUSAL, bool BIAS, int EMU = fwd::emu_pairs<D>(), bool SEQ = fwd::seq_turns<D>()>
__global__ void __launch_bounds__(fwd::NTHREADS, 1)
    ffa_gen_fwd_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                       const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_o,
                       const __grid_constant__ Problem pr, const __grid_constant__ Bias bias, float* __restrict__ LSE,
                       float* __restrict__ part, float* __restrict__ part_lse, int n_split, int group) {
  using L = FwdLayout<D, BIAS>;
  constexpr int SLABS = D / 64, STAGES = L::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  const uint32_t bar0 = sbase + L::BAR_OFF;
  const uint32_t q_full = bar0;
  auto kv_full = [&](int s) { return bar0 + 8 * (1 + s); };
  auto kv_empty = [&](int s) { return bar0 + 8 * (1 + STAGES + s); };
  auto s_full = [&](int i) { return bar0 + 8 * (1 + 2 * STAGES + i); };
  auto p_ready = [&](int i) { return bar0 + 8 * (3 + 2 * STAGES + i); };
  auto o_final = [&](int i) { return bar0 + 8 * (5 + 2 * STAGES + i); };
  const uint32_t drain_bar = bar0 + 8 * (7 + 2 * STAGES);
  auto p_half = [&](int i) { return bar0 + 8 * (8 + 2 * STAGES + i); };
  auto exp_done = [&](int i) { return bar0 + 8 * (10 + 2 * STAGES + i); };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::MISC_OFF);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::MISC_OFF + 4);
  float* tab = reinterpret_cast<float*>(smem + L::TAB_OFF);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  // work: (block of 256 queries, split of the keys) of one (sequence, query head); under a
  // causal mask the last blocks have the most keys and come first
  const int n_mblk = (pr.Sq + 255) / 256;
  const CtaWork cw = cta_work(n_mblk * n_split, pr.B * pr.Hq, group);
  const int mblk = CAUSAL ? n_mblk - 1 - cw.rank / n_split : cw.rank / n_split;
  const int split = cw.rank % n_split;
  const int b = cw.bh / pr.Hq, h = cw.bh % pr.Hq, hk = h / pr.G;
  const int m0 = mblk * 256;
  const int off = (CAUSAL || BIAS) ? pr.offset(b) : 0;
  const int n_keys = pr.keys(b, off, CAUSAL);
  // key tiles [t0, t0 + nt_i) of query tile i in this split
  auto tiles_of = [&](int mi) {
    if (mi >= pr.Sq) return 0;
    const int end = CAUSAL ? min(n_keys, max(off + mi + 128, 0)) : n_keys;
    return (end + 127) / 128;
  };
  const int all0 = tiles_of(m0), all1 = tiles_of(m0 + 128);
  const int per_split = (max(all0, all1) + n_split - 1) / n_split;
  const int t0 = split * per_split;
  const int nt0 = max(0, min(all0 - t0, per_split)), nt1 = max(0, min(all1 - t0, per_split));
  const int n_kv = max(nt0, nt1);

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(kv_full(s), 1);
      mbar_init(kv_empty(s), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(s_full(i), 1);
      mbar_init(p_ready(i), 128);
      mbar_init(o_final(i), 1);
      mbar_init(p_half(i), 128);
      mbar_init(exp_done(i), 128);
    }
    mbar_init(drain_bar, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == fwd::MMA_WARP) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  if (warp == fwd::PRODUCER_WARP && lane == 0) {
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  if (BIAS && warp < 8) build_table(bias, h, pr.Hq, tab, threadIdx.x, 256);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp >= 8) {
    setmaxnreg_dec<fwd::REGS_CONTROL>();
    if (warp == fwd::PRODUCER_WARP) {
      // ---------------------------------------------------------------- producer
      if (lane == 0 && n_kv > 0) {
        const uint64_t keep = policy_evict_last();
        mbar_arrive_expect_tx(q_full, 2 * L::TILE);
        for (int i = 0; i < 2; ++i)
          for (int sl = 0; sl < SLABS; ++sl)
            tma_load_4d(sbase + L::Q_OFF + i * L::TILE + sl * 16384, &tm_q, q_full, sl * 64, m0 + i * 128, h, b, keep);
        int issued = 0;
        for (; issued < 2 * n_kv; ++issued) {
          const int s = issued % STAGES;
          if (!mbar_wait(kv_empty(s), ((issued / STAGES) & 1) ^ 1, abort_flag, kErrGenFwdProducer)) break;
          mbar_arrive_expect_tx(kv_full(s), L::TILE);
          const CUtensorMap* tm = (issued & 1) ? &tm_v : &tm_k;
          for (int sl = 0; sl < SLABS; ++sl)
            tma_load_4d(sbase + L::KV_OFF + s * L::TILE + sl * 16384, tm, kv_full(s), sl * 64,
                        (t0 + (issued >> 1)) * 128, hk, b, keep);
        }
        if (*abort_flag) {
          // let in-flight copies land before the CTA's shared memory goes away
          for (int it = max(0, issued - STAGES); it < issued; ++it)
            mbar_wait_drain(kv_full(it % STAGES), (it / STAGES) & 1);
          mbar_wait_drain(q_full, 0);
        }
      }
    } else if (warp == fwd::MMA_WARP) {
      // ---------------------------------------------------------------- MMA issuer
      constexpr uint32_t IDESC_QK = idesc_bf16(128, 128, false, false);
      constexpr uint32_t IDESC_PV = idesc_bf16(128, D, false, true);
      bool ok = n_kv > 0 && mbar_wait(q_full, 0, abort_flag, kErrGenFwdMma);
      int it = 0;
      auto commit = [&](uint32_t bar) {
        if (elect_one()) mma_commit(bar);
        __syncwarp();
      };
      auto kv_addr = [&](int n) { return sbase + L::KV_OFF + (n % STAGES) * L::TILE; };
      auto kv_wait = [&](int n) {
        const bool r = mbar_wait(kv_full(n % STAGES), (n / STAGES) & 1, abort_flag, kErrGenFwdMma);
        tc_fence_after();
        return r;
      };
      const uint64_t qdesc0 = kmajor_desc(sbase + L::Q_OFF, 128, 0);
      const uint64_t qdesc1 = kmajor_desc(sbase + L::Q_OFF + L::TILE, 128, 0);
      auto issue_qk = [&](int i, uint32_t k_addr) {
        const uint64_t qd = i ? qdesc1 : qdesc0;
        const uint64_t kd = kmajor_desc(k_addr, 128, 0);
        const uint32_t d = tmem + i * 128;
        if (elect_one()) {
          mma_ss(d, qd, kd, IDESC_QK, 0u);
#pragma unroll
          for (int ks = 1; ks < D / 16; ++ks)
            mma_ss_acc(d, qd + kmajor_step(128, ks), kd + kmajor_step(128, ks), IDESC_QK);
          mma_commit(s_full(i));
        }
        __syncwarp();
      };
      // K-steps [k0, k1) of O_i += P_i V_j (16 keys = 8 TMEM columns of packed P each)
      auto issue_pv = [&](int i, uint32_t v_addr, int j, int k0, int k1) {
        const uint64_t vd = mnmajor_desc(v_addr, 128, 0);
        const uint32_t d = tmem + 256 + i * 128, a = tmem + i * 128;
        if (elect_one()) {
          for (int ks = k0; ks < k1; ++ks) {
            if (ks == 0)
              mma_ts(d, a, vd, IDESC_PV, j > 0 ? 1u : 0u);
            else
              mma_ts_acc(d, a + ks * 8, vd + mnmajor_step(ks), IDESC_PV);
          }
        }
        __syncwarp();
      };
      auto issue_pv_tile = [&](int i, uint32_t v_addr, int j) -> bool {
        if (!mbar_wait(p_half(i), j & 1, abort_flag, kErrGenFwdMma)) return false;
        tc_fence_after();
        issue_pv(i, v_addr, j, 0, 4);
        if (!mbar_wait(p_ready(i), j & 1, abort_flag, kErrGenFwdMma)) return false;
        tc_fence_after();
        issue_pv(i, v_addr, j, 4, 8);
        return true;
      };
      if (ok && (ok = kv_wait(it))) {
        const uint32_t k_addr = kv_addr(it);
        if (nt0 > 0) issue_qk(0, k_addr);
        if (nt1 > 0) issue_qk(1, k_addr);
        commit(kv_empty(it % STAGES));
        ++it;
      }
      for (int j = 0; j < n_kv && ok; ++j) {
        const int sv = it % STAGES;
        if (!(ok = kv_wait(it))) break;
        const uint32_t v_addr = kv_addr(it);
        ++it;
        const int tail = n_keys - (t0 + j) * 128;
        if (tail < 128 && n_keys < pr.Sk) zero_tail(v_addr, SLABS, tail, lane);
        const bool next = (j + 1 < n_kv);
        uint32_t k_addr = 0;
        // tile 0: O0 += P0 V_j, then S0 = Q0 K_{j+1}^T
        if (j < nt0 && !(ok = issue_pv_tile(0, v_addr, j))) break;
        if (next) {
          if (!(ok = kv_wait(it))) break;
          k_addr = kv_addr(it);
          if (j + 1 < nt0) issue_qk(0, k_addr);
        }
        // tile 1: O1 += P1 V_j, then S1 = Q1 K_{j+1}^T
        if (j < nt1 && !(ok = issue_pv_tile(1, v_addr, j))) break;
        commit(kv_empty(sv));
        if (next) {
          if (j + 1 < nt1) issue_qk(1, k_addr);
          commit(kv_empty(it % STAGES));
          ++it;
        }
      }
      if (ok && nt0 > 0) commit(o_final(0));
      if (ok && nt1 > 0) commit(o_final(1));
      // every issued MMA has finished before TMEM is released
      commit(drain_bar);
      mbar_wait_drain(drain_bar, 0);
    }
  } else {
    setmaxnreg_inc<fwd::REGS_SOFTMAX>();
    // ------------------------------------------------------------------ softmax
    const int i = warp >> 2;  // tile
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + lane_off + i * 128;
    const uint32_t t_o = tmem + lane_off + 256 + i * 128;
    const int mi = m0 + i * 128;
    const int grow = mi + row;
    const int wrow = mi + (warp & 3) * 32;  // the warp's first row
    const int nt = i ? nt1 : nt0;
    const int nt_other = i ? nt0 : nt1;
    // last key that this row sees
    const int lim = CAUSAL ? min(n_keys - 1, grow + off) : n_keys - 1;
    const float scale_log2 = pr.scale_log2;
    float bias_l = 0.f, bias_r = 0.f;
    if (BIAS) {
      bias_l = tab[0];
      bias_r = tab[table_size(bias) - 1];
    }
    bool ok = true;
    float m_used = -INFINITY;
    float l = 0.f;
    for (int j = 0; j < nt; ++j) {
      if (!(ok = mbar_wait(s_full(i), j & 1, abort_flag, kErrGenFwdSoftmax))) break;
      tc_fence_after();
      float s[128];
      {
        uint32_t r[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(t_s + c * 32, r[c]);
        tmem_ld_wait();
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int e = 0; e < 32; ++e) s[c * 32 + e] = __uint_as_float(r[c][e]);
      }
      const int n0 = (t0 + j) * 128;
      bool masked = (n0 + 128 > n_keys) || (CAUSAL && n0 + 127 > wrow + off);
      // relative positions of the warp's part of the tile: all in a last bucket, or looked up
      bool near = false;
      float fb = 0.f;
      if (BIAS) {
        const int r_min = n0 - (off + wrow + 31), r_max = n0 + 127 - (off + wrow);
        near = r_min < bias.right && r_max > -bias.left;
        fb = r_min >= bias.right ? bias_r : bias_l;
        masked |= !near && fb == -INFINITY;  // an infinite constant must not meet the polynomial exp2
      }
      const bool adjusted = masked || near;
      float tmax;
      if (adjusted) {
        if (BIAS && near) {
          const float* tp = tab + (n0 - off - grow + bias.left + kPad);
#pragma unroll
          for (int c = 0; c < 128; ++c) s[c] = fmaf(s[c], scale_log2, tp[c]);
        } else {
#pragma unroll
          for (int c = 0; c < 128; ++c) s[c] = BIAS ? fmaf(s[c], scale_log2, fb) : s[c] * scale_log2;
        }
        if (masked) {
#pragma unroll
          for (int c = 0; c < 128; ++c) s[c] = (n0 + c > lim) ? -INFINITY : s[c];
        }
        tmax = row_max128(s);
      } else if (scale_log2 >= 0.f) {
        tmax = BIAS ? fmaf(row_max128(s), scale_log2, fb) : row_max128(s) * scale_log2;
      } else {
        float a = s[0];
#pragma unroll
        for (int c = 1; c < 128; ++c) a = fminf(a, s[c]);
        tmax = fmaf(a, scale_log2, fb);
      }
      const float m_new = fmaxf(m_used, tmax);
      const bool need = m_new > m_used + fwd::RESCALE_THRESHOLD;
      if (__any_sync(0xffffffffu, need)) {
        const float m_safe = (m_new == -INFINITY) ? 0.f : m_new;
        const float alpha = fast_exp2(m_used - m_safe);
        if (j > 0) {
          // O_i(j-1) is complete: S_i(j) was committed after P_i(j-1) V_{j-1}.
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t r[32];
            tmem_ld32(t_o + c * 32, r);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; ++e) r[e] = __float_as_uint(__uint_as_float(r[e]) * alpha);
            tmem_st32(t_o + c * 32, r);
          }
        }
        l *= alpha;
        m_used = m_new;
      }
      const float m_safe = (m_used == -INFINITY) ? 0.f : m_used;
      uint32_t p[2][32];
      float2 sum2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
      const float shift = BIAS ? fb - m_safe : -m_safe;
      const float2 c2 = make_float2(scale_log2, scale_log2), nm2 = make_float2(shift, shift);
      // Column pairs [hf*32, hf*32+32) -> p[hf] -> TMEM columns [hf*32, hf*32+32) of S_i.
      auto half = [&](const int hf) {
        if (adjusted) {
#pragma unroll
          for (int u = 0; u < 32; ++u) {
            const int c = hf * 32 + u;
            const float p0 = fast_exp2(s[2 * c] - m_safe);
            const float p1 = fast_exp2(s[2 * c + 1] - m_safe);
            sum2[u & 1] = add2(sum2[u & 1], make_float2(p0, p1));
            p[hf][u] = pack_bf16x2(p0, p1);
          }
        } else {
          // EMU of every 8 column pairs take the FMA-pipe exp2, the rest MUFU.EX2
#pragma unroll
          for (int u = 0; u < 32; ++u) {
            const int c = hf * 32 + u;
            const float2 x = fma2(make_float2(s[2 * c], s[2 * c + 1]), c2, nm2);
            float p0, p1;
            if ((c & 7) < EMU) {
              const float2 e2 = exp2_fma2(x);
              p0 = e2.x;
              p1 = e2.y;
            } else {
              p0 = fast_exp2(x.x);
              p1 = fast_exp2(x.y);
            }
            sum2[u & 1] = add2(sum2[u & 1], make_float2(p0, p1));
            p[hf][u] = pack_bf16x2(p0, p1);
          }
        }
        if (SEQ && hf == 1) mbar_arrive(exp_done(i));
        tmem_st32(t_s + 32 * hf, p[hf]);
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(hf == 0 ? p_half(i) : p_ready(i));
      };
      if (SEQ) {
        // take turns with the other warpgroup: wait for its exponentials of step j (tile 1)
        // or j-1 (tile 0), when it has such a step
        const int oj = i ? j : j - 1;
        if (oj >= 0 && oj < nt_other && !(ok = mbar_wait(exp_done(i ^ 1), oj & 1, abort_flag, kErrGenFwdSoftmax)))
          break;
      }
      half(0);
      half(1);
      const float2 sv = add2(sum2[0], sum2[1]);
      l += sv.x + sv.y;
    }
    // Epilogue.  Every thread of the warpgroup reaches the barrier, finished or not.  A tile
    // that saw no key writes zeros.
    // (its Q tile, where the zeros are staged, may still be on its way when the other tile has keys)
    const bool done = ok && (n_kv == 0 || mbar_wait(nt > 0 ? o_final(i) : q_full, 0, abort_flag, kErrGenFwdSoftmax));
    const bool valid = done && grow < pr.Sq;
    const float inv_l = (l == 0.f) ? 0.f : 1.f / l;
    const float lse = (l == 0.f) ? -INFINITY : m_used + __log2f(l);
    const long long ridx = static_cast<long long>(b * pr.Hq + h) * pr.Sq + grow;
    const uint32_t o_tile = sbase + L::Q_OFF + i * L::TILE;
    if (n_split > 1) {
      const long long idx = static_cast<long long>(split) * pr.B * pr.Hq * pr.Sq + ridx;
      if (valid) part_lse[idx] = lse;
      if (done && nt > 0) {
        tc_fence_after();
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t r[32];
          tmem_ld32(t_o + c * 32, r);
          tmem_ld_wait();
          if (valid && l != 0.f) write_row32(part + idx * pr.D, 32 * c, pr.D, r, inv_l);
        }
      }
    } else {
      if (done) {
        tc_fence_after();
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t r[32];
          if (nt > 0) {
            tmem_ld32(t_o + c * 32, r);
            tmem_ld_wait();
          }
          if (l == 0.f) {  // no key: tensor memory may hold anything
#pragma unroll
            for (int e = 0; e < 32; ++e) r[e] = 0u;
          }
          stage_row32_sw128(o_tile, row, 32 * c, r, inv_l);
        }
        if (LSE != nullptr && valid) LSE[ridx] = lse;
      }
      // the Q tile is free once every MMA has finished; the store leaves out rows from Sq on
      fence_proxy_async_smem();
      const bool store = named_barrier_and(1 + i, 128, done);
      if (row == 0 && store && mi < pr.Sq) {
#pragma unroll
        for (int sl = 0; sl < SLABS; ++sl) tma_store_4d(&tm_o, o_tile + sl * 16384, sl * 64, mi, h, b);
        bulk_commit_group();
        bulk_wait_read();
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == fwd::MMA_WARP) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace gen
}  // namespace ffa
