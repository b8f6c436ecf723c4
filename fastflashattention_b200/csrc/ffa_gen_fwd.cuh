// ffa_gen_fwd.cuh — forward of general attention (ffa_gen_common.cuh) for sm_100a.
//
//   O_i = sum_j softmax_j(S_ij) v_j,   LSE_i = base-2 log-sum-exp of S_i (-inf: no key)
//
// The plan of the plain forward (ffa_fwd.cuh): a softmax warpgroup for each 128-row query
// tile (thread = row), and warps that load and issue MMAs; S and O in tensor memory, P handed back
// through it over S; the running max is rescaled lazily.  What differs:
//   * operands are 4-D tensor maps, so any strides of batch, head and row do, and the key
//     head of a query head is found by division;
//   * head dims up to 64: the softmax bounds the kernel, and one warp of a scheduler waits
//     for its own loads and MMAs most of the time.  So a CTA has one tile and walks 64 keys
//     a step, 128 columns of tensor memory, four CTAs to an SM.  One warp loads and issues
//     MMAs, whose commits free the slots that it loads: with five warps a thread has 96
//     registers, with six 80 and spills (B8 H16 S4096: 749 us with six, 684 so; with a bias 857
//     and 732);
//   * head dims up to 128: two tiles and 128 keys a step, one CTA to an SM;
//   * the loop bodies are 64 scores long and the same for every kind of tile; a mask, a bias
//     for each score or a negative scale is applied where the scores come into registers for
//     their maximum.  A short launch spends much of its time
//     fetching instructions that it runs for the first time (B8 H12 S1024 D64 without a bias:
//     91 us with bodies of 128 scores for each kind, 59 with these);
//   * a tile whose relative positions all lie in the last bucket of a side has one bias: it
//     joins the row max and the exponent's constant for free;
//   * EXACT, for a training step that wants the bias's gradient: P goes to the product as two
//     bf16 values (rounded and remainder, twice the MMAs), and O is written with its own
//     remainder (o_lo), which gives the backward delta = O . dO to 16 bits.  The bias's
//     gradient adds dS over whole rows, whose sum is 0: an error of delta, common to a row,
//     adds up where dS cancels (with O in 8 bits: up to 0.7 % of the gradient's norm at 16
//     buckets, S = 1485; with the remainder 0.2 %, its rounding to bf16);
//   * with few CTAs the keys are split in units of `per_split` steps (the same for all
//     sequences, so that units of sequences of different lengths take the same time); each
//     split writes its normalised O in fp32 and its LSE, and ffa_gen_join_kernel weighs them.
#pragma once
#include "ffa_fwd.cuh"
#include "ffa_gen_common.cuh"

namespace ffa {
namespace gen {

template <int D>
struct FwdLayout {
  static constexpr int NT = D == 64 ? 1 : 2;        // 128-row tiles (softmax warpgroups) of a CTA
  // CTAs of an SM.  EXACT holds 32 registers more: three CTAs without spills beat four (B8 H16
  // S4096 D64: 963 us against 995; B8 H12 S1000: 76 against 82)
  static constexpr int ctas(bool exact) { return D == 64 ? (exact ? 3 : 4) : 1; }
  static constexpr int KEYS = D == 64 ? 64 : 128;   // keys of a step
  static constexpr int HALVES = KEYS / 64;          // P is handed over 64 keys at a time
  static constexpr int ROWS = 128 * NT;
  // D = 128 moves registers between warpgroups (setmaxnreg), so the control warps fill one up
  static constexpr int THREADS = D == 64 ? 160 : 384;
  static constexpr int TMEM = D == 64 ? 128 : 512;  // S [0, KEYS) of each tile, then O
  static constexpr uint32_t O_COL = KEYS * NT;
  static constexpr int Q_TILE = 128 * D * 2, TILE = KEYS * D * 2;
  static constexpr int STAGES = 4;
  static constexpr int Q_OFF = 0;
  static constexpr int KV_OFF = NT * Q_TILE;
  // q_full, kv_full[], kv_empty[], tab_full; for each tile s_full, o_final, p_ready[2]; drain
  static constexpr int BAR_OFF = KV_OFF + STAGES * TILE;
  static constexpr int NBARS = 1 + 2 * STAGES + 1 + 4 * NT + 1;
  static constexpr int MISC_OFF = BAR_OFF + NBARS * 8;
  static constexpr int TAB_OFF = (MISC_OFF + 16 + 15) / 16 * 16;
  static int smem_bytes(const Bias& bias) { return TAB_OFF + (bias.table ? table_size(bias) * 4 : 0) + 1024; }
};

// max(a, b, c), NaN if one of them is.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Row max of 64 scores (16 chains of three-input maxima, then a short tree).
__device__ __forceinline__ float row_max64(const uint32_t (&a)[32], const uint32_t (&b)[32]) {
  float x[16];
#pragma unroll
  for (int u = 0; u < 16; ++u)
    x[u] = max3_nan(__uint_as_float(a[u]), __uint_as_float(a[16 + u]), __uint_as_float(b[u]));
#pragma unroll
  for (int u = 0; u < 16; u += 2) x[u] = max3_nan(x[u], __uint_as_float(b[16 + u]), __uint_as_float(b[17 + u]));
  const float y0 = max3_nan(x[0], x[1], x[2]), y1 = max3_nan(x[3], x[4], x[5]), y2 = max3_nan(x[6], x[7], x[8]);
  const float y3 = max3_nan(x[9], x[10], x[11]), y4 = max3_nan(x[12], x[13], x[14]);
  return max3_nan(max3_nan(y0, y1, y2), max3_nan(y3, y4, x[15]), y0);
}

// EMU of every 8 column pairs take their exponentials on the FMA pipe.  At D = 64 one is best
// (B8 H16 S4096 with a bias: 729 us, 743 with two, 766 with none; without 672, 676 and 698);
// at D = 128 it changes nothing.
template <int D, bool CAUSAL, bool BIAS, bool EXACT, int EMU = D == 64 ? 1 : 0>
__global__ void __launch_bounds__(FwdLayout<D>::THREADS, FwdLayout<D>::ctas(EXACT))
    ffa_gen_fwd_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                       const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_o,
                       const __grid_constant__ CUtensorMap tm_lo, const __grid_constant__ Problem pr, const __grid_constant__ Bias bias,
                       const float* tables, float* __restrict__ LSE, float* __restrict__ part,
                       float* __restrict__ part_lse, int n_split, int per_split, int group) {
  using L = FwdLayout<D>;
  constexpr int SLABS = D / 64, STAGES = L::STAGES, NT = L::NT, KEYS = L::KEYS;
  constexpr int HALVES = L::HALVES;
  constexpr bool ONE = NT == 1;  // one warp loads and issues MMAs
  constexpr int PRODUCER = 4 * NT, MMA = ONE ? PRODUCER : PRODUCER + 1;  // warps
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  const uint32_t bar0 = sbase + L::BAR_OFF;
  const uint32_t q_full = bar0;
  auto kv_full = [&](int n) { return bar0 + 8 * (1 + n % STAGES); };
  auto kv_empty = [&](int n) { return bar0 + 8 * (1 + STAGES + n % STAGES); };
  const uint32_t tab_full = bar0 + 8 * (1 + 2 * STAGES);
  auto s_full = [&](int i) { return tab_full + 8 * (1 + 4 * i); };
  auto o_final = [&](int i) { return tab_full + 8 * (2 + 4 * i); };
  auto p_ready = [&](int i, int half) { return tab_full + 8 * (3 + 4 * i + half); };
  const uint32_t drain_bar = tab_full + 8 * (1 + 4 * NT);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::MISC_OFF);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::MISC_OFF + 4);
  const float* tab = reinterpret_cast<const float*>(smem + L::TAB_OFF);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  // work: (block of ROWS queries, split of the keys) of one (sequence, query head); under a
  // causal mask the last blocks have the most keys and come first
  const int n_mblk = (pr.Sq + L::ROWS - 1) / L::ROWS;
  const CtaWork cw = cta_work(n_mblk * n_split, pr.B * pr.Hq, group);
  const int mblk = CAUSAL ? n_mblk - 1 - cw.rank / n_split : cw.rank / n_split;
  const int split = cw.rank % n_split;
  const int b = pr.seq_at(cw.bh / pr.Hq), h = cw.bh % pr.Hq, hk = h / pr.G;
  const int m0 = mblk * L::ROWS;
  const int off = (CAUSAL || BIAS) ? pr.offset(b) : 0;
  const int n_keys = pr.keys(b, off, CAUSAL);
  asm volatile("griddepcontrol.launch_dependents;");
  const int t0 = split * per_split;
  // a split behind the sequence's last key leaves at once; the join counts the splits in the same way
  if (split > 0 && t0 * KEYS >= n_keys) return;
  // steps [t0, t0 + cnt_i) of query tile i in this split
  auto steps_of = [&](int mi) {
    if (mi >= pr.Sq) return 0;
    const int end = CAUSAL ? min(n_keys, max(off + mi + 128, 0)) : n_keys;
    return max(0, min((end + KEYS - 1) / KEYS - t0, per_split));
  };
  const int cnt0 = steps_of(m0), cnt1 = NT == 1 ? 0 : steps_of(m0 + 128);
  const int n_kv = max(cnt0, cnt1);

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(kv_full(s), 1);
      mbar_init(kv_empty(s), 1);
    }
    mbar_init(tab_full, 1);
    for (int i = 0; i < NT; ++i) {
      mbar_init(s_full(i), 1);
      mbar_init(o_final(i), 1);
      mbar_init(p_ready(i, 0), 128);
      mbar_init(p_ready(i, 1), 128);
    }
    mbar_init(drain_bar, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == MMA) {
    tmem_alloc(smem_u32(tmem_slot), L::TMEM);
    tmem_relinquish();
  }
  if (warp == PRODUCER && lane == 0) {
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp >= 4 * NT) {
    if constexpr (D == 128) setmaxnreg_dec<fwd::REGS_CONTROL>();
    const uint64_t keep = policy_evict_last();
    auto load_q = [&]() {
      mbar_arrive_expect_tx(q_full, NT * L::Q_TILE);
      for (int i = 0; i < NT; ++i)
        for (int sl = 0; sl < SLABS; ++sl)
          tma_load_4d(sbase + L::Q_OFF + i * L::Q_TILE + sl * 16384, &tm_q, q_full, sl * 64, m0 + i * 128, h, b, keep);
    };
    auto load_kv = [&](int n) {  // K_0, V_0, K_1, V_1, ..
      mbar_arrive_expect_tx(kv_full(n), L::TILE);
      for (int sl = 0; sl < SLABS; ++sl)
        tma_load_4d(sbase + L::KV_OFF + (n % STAGES) * L::TILE + sl * (KEYS * 128), (n & 1) ? &tm_v : &tm_k, kv_full(n),
                    sl * 64, (t0 + (n >> 1)) * KEYS, hk, b, keep);
    };
    auto slot_free = [&](int n) {
      return mbar_wait(kv_empty(n), ((n / STAGES) & 1) ^ 1, abort_flag, kErrGenFwdProducer);
    };
    // the table, once its kernel has written it (this one may start before that ends)
    auto load_table = [&]() {
      asm volatile("griddepcontrol.wait;" ::: "memory");
      const int bytes = table_size(bias) * 4;
      mbar_arrive_expect_tx(tab_full, bytes);
      bulk_load(smem_u32(tab), tables + static_cast<long long>(h) * table_size(bias), bytes, tab_full);
    };
    // let the copies in flight, of the first n tiles, land before the CTA's shared memory goes away
    auto drain_loads = [&](int n) {
      if (!*abort_flag) return;
      for (int x = max(0, n - STAGES); x < n; ++x) mbar_wait_drain(kv_full(x), (x / STAGES) & 1);
      mbar_wait_drain(q_full, 0);
      if (BIAS && n > 0) mbar_wait_drain(tab_full, 0);
    };
    // without tiles nobody waits for the tables: the launch ends after theirs all the same
    if (BIAS && warp == PRODUCER && n_kv == 0) asm volatile("griddepcontrol.wait;" ::: "memory");
    if (!ONE && warp == PRODUCER) {
      // ---------------------------------------------------------------- producer
      if (lane == 0 && n_kv > 0) {
        load_q();
        int n = 0;
        for (; n < 2 * n_kv && slot_free(n); ++n) {
          load_kv(n);
          if (BIAS && n == 0) load_table();
        }
        drain_loads(n);
      }
    } else if (warp == MMA) {
      // ---------------------------------------------------------------- MMA issuer
      int loaded = 0;  // tiles (ONE)
      if (ONE && n_kv > 0) {
        loaded = min(STAGES, 2 * n_kv);
        if (lane == 0) {
          load_q();
          for (int n = 0; n < loaded; ++n) load_kv(n);
          if (BIAS) load_table();
        }
        __syncwarp();
      }
      constexpr uint32_t IDESC_QK = idesc_bf16(128, KEYS, false, false);
      constexpr uint32_t IDESC_PV = idesc_bf16(128, D, false, true);
      bool ok = n_kv > 0 && mbar_wait(q_full, 0, abort_flag, kErrGenFwdMma);
      auto commit = [&](uint32_t bar) {
        if (elect_one()) mma_commit(bar);
        __syncwarp();
      };
      auto kv_addr = [&](int n) { return sbase + L::KV_OFF + (n % STAGES) * L::TILE; };
      auto kv_wait = [&](int n) {
        const bool r = mbar_wait(kv_full(n), (n / STAGES) & 1, abort_flag, kErrGenFwdMma);
        tc_fence_after();
        return r;
      };
      auto issue_qk = [&](int i, int n) {  // S_i = Q_i K^T
        const uint64_t qd = kmajor_desc(sbase + L::Q_OFF + i * L::Q_TILE, 128, 0);
        const uint64_t kd = kmajor_desc(kv_addr(n), KEYS, 0);
        const uint32_t d = tmem + i * KEYS;
        if (elect_one()) {
          mma_ss(d, qd, kd, IDESC_QK, 0u);
#pragma unroll
          for (int ks = 1; ks < D / 16; ++ks)
            mma_ss_acc(d, qd + kmajor_step(128, ks), kd + kmajor_step(KEYS, ks), IDESC_QK);
          mma_commit(s_full(i));
        }
        __syncwarp();
      };
      auto issue_pv = [&](int i, int j, int n) -> bool {  // O_i (+)= P_i V_j, as P comes
        const uint64_t vd = mnmajor_desc(kv_addr(n), KEYS, 0);
        const uint32_t d = tmem + L::O_COL + i * 128, a = tmem + i * KEYS;
#pragma unroll 1
        for (int half = 0; half < HALVES; ++half) {
          if (!mbar_wait(p_ready(i, half), j & 1, abort_flag, kErrGenFwdMma)) return false;
          tc_fence_after();
          if (elect_one()) {
            const uint64_t vh = vd + mnmajor_step(4 * half);
            mma_ts(d, a + 64 * half, vh, IDESC_PV, (j > 0 || half > 0) ? 1u : 0u);
#pragma unroll
            for (int ks = 1; ks < (EXACT ? 8 : 4); ++ks)  // 4 to 7: the remainders of P, behind it
              mma_ts_acc(d, a + 64 * half + ks * 8, vh + mnmajor_step(ks & 3), IDESC_PV);
          }
          __syncwarp();
        }
        return true;
      };
      if (ok && (ok = kv_wait(0))) {
        if (cnt0 > 0) issue_qk(0, 0);
        if (NT > 1 && cnt1 > 0) issue_qk(1, 0);
        commit(kv_empty(0));
      }
      for (int j = 0; j < n_kv && ok; ++j) {
        const int nv = 2 * j + 1, nk = 2 * j + 2;  // V_j and K_{j+1}
        if (ONE) {
          // S_j is there: the slots of V_{j-1} and K_j are free, or will be at once
          for (; loaded <= nk + 2 && loaded < 2 * n_kv; ++loaded) {
            if (!(ok = slot_free(loaded))) break;
            if (lane == 0) load_kv(loaded);
          }
          __syncwarp();
          if (!ok) break;
        }
        if (!(ok = kv_wait(nv))) break;
        const int tail = n_keys - (t0 + j) * KEYS;
        if (tail < KEYS && n_keys < pr.Sk) zero_tail<KEYS>(kv_addr(nv), SLABS, tail, lane);
        const bool next = j + 1 < n_kv;
        // tile by tile: O_i += P_i V_j, then S_i = Q_i K_{j+1}^T over P_i
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          const int cnt = i ? cnt1 : cnt0;
          if (j < cnt && !(ok = issue_pv(i, j, nv))) break;
          if (next) {
            if (i == 0 && !(ok = kv_wait(nk))) break;
            if (j + 1 < cnt) issue_qk(i, nk);
          }
        }
        if (!ok) break;
        commit(kv_empty(nv));
        if (next) commit(kv_empty(nk));
      }
      if (ok && cnt0 > 0) commit(o_final(0));
      if (NT > 1 && ok && cnt1 > 0) commit(o_final(1));
      // every issued MMA has finished before TMEM is released
      commit(drain_bar);
      mbar_wait_drain(drain_bar, 0);
      if (ONE && n_kv > 0) drain_loads(loaded);
    }
  } else {
    if constexpr (D == 128) setmaxnreg_inc<fwd::REGS_SOFTMAX>();
    // ------------------------------------------------------------------ softmax
    const int i = NT == 1 ? 0 : warp >> 2;  // tile
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + lane_off + i * KEYS;
    const uint32_t t_o = tmem + lane_off + L::O_COL + i * 128;
    const int mi = m0 + i * 128;
    const int grow = mi + row;
    const int wrow = mi + (warp & 3) * 32;  // the warp's first row
    const int cnt = i ? cnt1 : cnt0;
    // last key that this row sees
    const int lim = CAUSAL ? min(n_keys - 1, grow + off) : n_keys - 1;
    const float scale_log2 = pr.scale_log2;
    bool ok = true;
    if (BIAS && cnt > 0) ok = mbar_wait(tab_full, 0, abort_flag, kErrGenFwdSoftmax);
    float m_used = -INFINITY;
    float l = 0.f;
    for (int j = 0; ok && j < cnt; ++j) {
      if (!(ok = mbar_wait(s_full(i), j & 1, abort_flag, kErrGenFwdSoftmax))) break;
      tc_fence_after();
      const int n0 = (t0 + j) * KEYS;
      const bool masked = (n0 + KEYS > n_keys) || (CAUSAL && n0 + KEYS - 1 > wrow + off);
      // relative positions of the warp's part of the tile: all in a last bucket, or looked up
      bool near = false;
      float fb = 0.f;  // the tile's bias
      if (BIAS) {
        const int r_min = n0 - (off + wrow + 31), r_max = n0 + KEYS - 1 - (off + wrow);
        near = r_min < bias.right && r_max > -bias.left;
        fb = tab[r_min >= bias.right ? table_last(bias) : 0];
      }
      // With a bias for each score or a scale that does not keep the order, the scores become
      // scaled scores; masked ones become -inf.  Those that do not stay in registers (the second
      // half of 128) go back to tensor memory.  Without a bias this is rare, and at D = 128 a
      // loop apart keeps the others' shorter (B2 H16 S4096 D128: 273 us against 283).
      const bool scaled = near || scale_log2 <= 0.f;
      const float c = scaled ? 1.f : scale_log2;  // what the scores still have to be multiplied with
      uint32_t sa[32], sb[32];  // 64 scores
      auto adjust = [&](int x) {  // columns x .. x + 63 of the step
        if (scaled) {
          const float* tp = tab + (n0 + x - off - grow + bias.left + kPad);
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            sa[e] = __float_as_uint(fmaf(__uint_as_float(sa[e]), scale_log2, BIAS && near ? tp[e] : fb));
            sb[e] = __float_as_uint(fmaf(__uint_as_float(sb[e]), scale_log2, BIAS && near ? tp[32 + e] : fb));
          }
        }
        if (masked) {
          const int last = lim - n0 - x;
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            if (e > last) sa[e] = 0xff800000u;
            if (32 + e > last) sb[e] = 0xff800000u;
          }
        }
      };
      auto load = [&](int hf) {
        tmem_ld32(t_s + 64 * hf, sa);
        tmem_ld32(t_s + 64 * hf + 32, sb);
        tmem_ld_wait();
      };
      auto store = [&](int hf) {
        tmem_st32(t_s + 64 * hf, sa);
        tmem_st32(t_s + 64 * hf + 32, sb);
        tmem_st_wait();
      };
      constexpr bool APART = HALVES > 1 && !BIAS;
      if (APART && (scaled || masked)) {
#pragma unroll 1
        for (int hf = 0; hf < HALVES; ++hf) {
          load(hf);
          adjust(64 * hf);
          store(hf);
        }
      }
      float tmax = -INFINITY;
#pragma unroll 1
      for (int hf = HALVES - 1; hf >= 0; --hf) {
        load(hf);
        if (!APART) {
          adjust(64 * hf);
          if (hf > 0 && (scaled || masked)) store(hf);
        }
        tmax = max3_nan(tmax, tmax, row_max64(sa, sb));
      }
      if (scaled) fb = 0.f;
      tmax = BIAS ? fmaf(tmax, c, fb) : tmax * c;
      // a visible score that is NaN or +inf makes the row NaN (exp2_fma2 would lose it)
      if (!(tmax < INFINITY)) l = __int_as_float(0x7fffffff);
      const float m_new = fmaxf(m_used, tmax);
      const bool need = m_new > m_used + fwd::RESCALE_THRESHOLD;
      if (__any_sync(0xffffffffu, need)) {
        const float m_safe = (m_new == -INFINITY) ? 0.f : m_new;
        const float alpha = fast_exp2(m_used - m_safe);
        if (j > 0) {
          // O_i(j-1) is complete: S_i(j) was committed after P_i(j-1) V_{j-1}
#pragma unroll 1
          for (int x = 0; x < D; x += 16) {
            uint32_t r[16];
            tmem_ld16(t_o + x, r);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 16; ++e) r[e] = __float_as_uint(__uint_as_float(r[e]) * alpha);
            tmem_st16(t_o + x, r);
          }
        }
        l *= alpha;
        m_used = m_new;
      }
      const float m_safe = (m_used == -INFINITY) ? 0.f : m_used;
      const float shift = BIAS ? fb - m_safe : -m_safe;
      const float2 c2 = make_float2(c, c), nm2 = make_float2(shift, shift);
      // 64 scores -> P -> 32 columns over these scores, and 32 of remainders behind them (the
      // first half's scores are still in registers)
#pragma unroll 1
      for (int hf = 0; hf < HALVES; ++hf) {
        if (hf > 0) load(hf);
        float2 sum2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        uint32_t hi[32], lo[EXACT ? 32 : 1];
#pragma unroll
        for (int u = 0; u < 32; ++u) {
          const uint32_t* src = u < 16 ? sa : sb;
          const int e = 2 * (u & 15);
          const float2 x = fma2(make_float2(__uint_as_float(src[e]), __uint_as_float(src[e + 1])), c2, nm2);
          float p0, p1;
          if ((u & 7) < EMU) {  // EMU of every 8 column pairs on the FMA pipe
            const float2 e2 = exp2_fma2(x);
            p0 = e2.x;
            p1 = e2.y;
          } else {
            p0 = fast_exp2(x.x);
            p1 = fast_exp2(x.y);
          }
          sum2[u & 1] = add2(sum2[u & 1], make_float2(p0, p1));
          hi[u] = pack_bf16x2(p0, p1);
          if (EXACT)
            lo[u] = pack_bf16x2(p0 - __uint_as_float(hi[u] << 16), p1 - __uint_as_float(hi[u] & 0xffff0000u));
        }
        const float2 sv = add2(sum2[0], sum2[1]);
        l += sv.x + sv.y;
        tmem_st32(t_s + 64 * hf, hi);
        if constexpr (EXACT) tmem_st32(t_s + 64 * hf + 32, lo);
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(p_ready(i, hf));
      }
    }
    // Epilogue.  Every thread of the warpgroup reaches the barrier, finished or not.  A row
    // without keys (no max, and none of them NaN) is 0: the sum holds what the polynomial
    // makes of 2^-inf, and tensor memory may hold anything.  Its Q tile, where the output is staged, may still be
    // on its way when the other tile has keys.
    const bool done = ok && (n_kv == 0 || mbar_wait(cnt > 0 ? o_final(i) : q_full, 0, abort_flag, kErrGenFwdSoftmax));
    tc_fence_after();
    const bool valid = done && grow < pr.Sq, none = m_used == -INFINITY && l == l;
    const float inv_l = none ? 0.f : 1.f / l;
    const float lse = none ? -INFINITY : m_used + __log2f(l);
    const uint32_t o_tile = sbase + L::Q_OFF + i * L::Q_TILE;
    const long long ridx = static_cast<long long>(b * pr.Hq + h) * pr.Sq + grow;
    const long long prow = static_cast<long long>(split) * pr.B * pr.Hq * pr.Sq + ridx;
    if (valid) {
      if (n_split > 1)
        part_lse[prow] = lse;
      else if (LSE != nullptr)
        LSE[ridx] = lse;
    }
    __syncwarp();  // tensor memory is loaded by whole warps
    // O, then (EXACT) its remainder, over the Q tile, which is free once every MMA has finished
#pragma unroll 1
    for (int rem = 0; rem < (EXACT && n_split == 1 ? 2 : 1); ++rem) {
      if (done) {
#pragma unroll 1
        for (int x = 0; x < D; x += 32) {
          uint32_t r[32];
          if (cnt > 0) {
            tmem_ld32(t_o + x, r);
            tmem_ld_wait();
          }
          if (none) {
#pragma unroll
            for (int e = 0; e < 32; ++e) r[e] = 0u;
          }
          if (EXACT && rem) {
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              const float y = __uint_as_float(r[e]) * inv_l;
              r[e] = __float_as_uint(y - __bfloat162float(__float2bfloat16_rn(y)));
            }
          }
          if (n_split == 1)
            stage_row32_sw128(o_tile, row, x, r, rem ? 1.f : inv_l);
          else
            write_rows32(o_tile + (warp & 3) * 4096, part + (prow - lane) * pr.D, x, pr.D, pr.Sq - wrow, r, inv_l,
                         lane);
        }
      }
      if (n_split == 1) {  // the store leaves out rows from Sq on
        fence_proxy_async_smem();
        const bool store = whole_barrier_and(1 + i, 128, done);
        if (row == 0 && store && mi < pr.Sq) {
#pragma unroll
          for (int sl = 0; sl < SLABS; ++sl)
            tma_store_4d(rem ? &tm_lo : &tm_o, o_tile + sl * 16384, sl * 64, mi, h, b);
          bulk_commit_group();
          bulk_wait_read();
        }
        if (EXACT) whole_barrier_and(1 + i, 128, true);  // the tile has been read
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == MMA) {
    tc_fence_after();
    tmem_dealloc(tmem, L::TMEM);
  }
}

// Join the splits of a row: O = sum_s w_s O_s / sum_s w_s, w_s = 2^(LSE_s - max LSE).  LANES
// threads a row (D <= 4 LANES), four columns each.  A sequence has as many splits as its
// keys fill; a split whose keys the row does not see (LSE = -inf) weighs nothing.
template <int LANES>
__global__ void __launch_bounds__(256)
    ffa_gen_join_kernel(const __grid_constant__ Problem pr, const float* part, const float* part_lse, const View o,
                        const View o_lo, float* __restrict__ LSE, int keys_per_split, int causal) {
  const long long rows = static_cast<long long>(pr.B) * pr.Hq * pr.Sq;
  const long long r = static_cast<long long>(blockIdx.x) * (256 / LANES) + threadIdx.x / LANES;
  const int c = threadIdx.x % LANES * 4;
  if (r >= rows || c >= pr.D) return;
  const int bh = static_cast<int>(r / pr.Sq), t = static_cast<int>(r % pr.Sq);
  const int b = bh / pr.Hq, h = bh % pr.Hq;
  const int n_keys = pr.keys(b, causal ? pr.offset(b) : 0, causal);
  const int n = max(1, (n_keys + keys_per_split - 1) / keys_per_split);
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the splits have written
  // one pass with a running max: the loads of four splits do not wait for one another
  float m = -INFINITY, total = 0.f;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int s = 0; s < n; ++s) {
    const float lse = part_lse[s * rows + r];
    const float4 x = *reinterpret_cast<const float4*>(part + (s * rows + r) * pr.D + c);
    const float m_new = fmaxf(m, lse), m_safe = m_new == -INFINITY ? 0.f : m_new;
    const float f = exp2f(m - m_safe), w = exp2f(lse - m_safe);
    m = m_new;
    total = fmaf(total, f, w);
    a.x = fmaf(a.x, f, w * x.x);
    a.y = fmaf(a.y, f, w * x.y);
    a.z = fmaf(a.z, f, w * x.z);
    a.w = fmaf(a.w, f, w * x.w);
  }
  const float inv = total == 0.f ? 0.f : 1.f / total;
  const uint2 hi = make_uint2(pack_bf16x2(a.x * inv, a.y * inv), pack_bf16x2(a.z * inv, a.w * inv));
  *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(o.p) + b * o.sb + h * o.sh + t * o.ss + c) = hi;
  if (o_lo.p != nullptr)
    *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(o_lo.p) + b * o_lo.sb + h * o_lo.sh + t * o_lo.ss + c) =
        make_uint2(pack_bf16x2(a.x * inv - __uint_as_float(hi.x << 16), a.y * inv - __uint_as_float(hi.x & 0xffff0000u)),
                   pack_bf16x2(a.z * inv - __uint_as_float(hi.y << 16), a.w * inv - __uint_as_float(hi.y & 0xffff0000u)));
  if (c == 0 && LSE != nullptr) LSE[r] = total == 0.f ? -INFINITY : m + __log2f(total);
}

}  // namespace gen
}  // namespace ffa
