// ffa_gen_bwd.cuh — deterministic backward of general attention (ffa_gen_common.cuh).
//
//   P = exp2(S - LSE)   dP = dO V^T   dS = P o (dP - delta)   delta = rowsum(O o dO)
//   dV = sum_g P_g^T dO_g      dK = scale * sum_g dS_g^T Q_g     (g: query heads of a key head)
//   dQ = scale * dS K          dbias[u, h] = sum of dS over the scores of head h in bucket u
//
// The two kernels of the plain backward (ffa_bwd.cuh), with disjoint output tiles and no
// atomics.  What differs:
//   * delta comes from the dQ kernel, which has dO in hand; dK/dV follows it, launched while it
//     still runs (programmatic dependent launch).  Without a wish for dQ,
//     ffa_gen_prepare_kernel writes delta;
//   * head dims up to 64 walk 64 columns a step instead of 128: 256 columns of tensor memory
//     and two CTAs to an SM, with 32 columns a thread.  The loop of a CTA is a chain of waits
//     (S, exponentials, dP, dS, MMAs); two CTAs and four warps to a scheduler fill each
//     other's;
//   * the dK/dV kernel walks the queries of all heads of its key head, one after another, so
//     a shared key head's gradients are summed in tensor memory;
//   * P = 0 outside the mask, and K / V rows behind the last key are zeroed in shared memory;
//   * dbias rides on the dQ kernel, whose threads hold dS in fp32.  A warp's block of dS (32 rows) far
//     from the diagonal lies in one bucket: a plain sum.  A near block is summed along its
//     diagonals (one shuffle and one add a column: lane l passes its partial sum of a
//     diagonal to lane l + 1), then by bucket; each warp has its own sums, each CTA its own
//     row of the workspace, and ffa_gen_bias_sum_kernel adds the rows in a fixed order;
//   * with few CTAs the streamed dimension is split: the splits write fp32 gradients and
//     ffa_gen_sum_kernel adds them in order.
#pragma once
#include "ffa_bwd.cuh"
#include "ffa_gen_common.cuh"

namespace ffa {
namespace gen {

// Rows of LSE and delta in the workspace, padded to whole tiles.
__host__ __device__ inline int padded_rows(int Sq) { return (Sq + 127) / 128 * 128; }

// delta, and the LSE as the backward reads it: +inf for a row that saw no key and for rows
// behind the last one, which makes their P 0.  TPR threads a row, 16 bytes each.
template <int TPR>
__global__ void __launch_bounds__(256)
    ffa_gen_prepare_kernel(const View o, const View dout, const float* __restrict__ LSE, float* __restrict__ lse_out,
                           float* __restrict__ delta, int H, int Sq, int D) {
  const int rows_p = padded_rows(Sq);  // a multiple of a block's 256 / TPR rows: the grid is exact
  const int sub = threadIdx.x % TPR;
  const long long r = static_cast<long long>(blockIdx.x) * (256 / TPR) + threadIdx.x / TPR;
  const long long bh = r / rows_p;
  const int i = static_cast<int>(r % rows_p);
  float acc = 0.f;
  if (i < Sq && sub * 8 < D) {
    const long long b = bh / H, h = bh % H;
    const uint4 x = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(o.p) + b * o.sb + h * o.sh +
                                                    i * o.ss + sub * 8);
    const uint4 y = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(dout.p) + b * dout.sb +
                                                    h * dout.sh + i * dout.ss + sub * 8);
    const __nv_bfloat162* x2 = reinterpret_cast<const __nv_bfloat162*>(&x);
    const __nv_bfloat162* y2 = reinterpret_cast<const __nv_bfloat162*>(&y);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 a = __bfloat1622float2(x2[e]), c = __bfloat1622float2(y2[e]);
      acc = fmaf(a.x, c.x, acc);
      acc = fmaf(a.y, c.y, acc);
    }
  }
#pragma unroll
  for (int x = TPR / 2; x > 0; x >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, x);
  if (sub == 0) {
    float lse = INFINITY;
    if (i < Sq) {
      lse = LSE[bh * Sq + i];
      if (lse == -INFINITY) lse = INFINITY;
    }
    lse_out[r] = lse;
    delta[r] = acc;
  }
}

// Sum of the splits' fp32 gradients [n_split][B][H][S][D] into a bf16 view; 8 columns a
// thread.  blockIdx.y: the first or the second pair of parts and view (dK and dV).
__global__ void __launch_bounds__(256)
    ffa_gen_sum_kernel(const float* part0, const float* part1, const View out0, const View out1, int n_split, int B,
                       int H, int S, int D) {
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the splits have written
  const float* part = blockIdx.y == 0 ? part0 : part1;
  const View out = blockIdx.y == 0 ? out0 : out1;
  const long long chunks = static_cast<long long>(B) * H * S * (D / 8);
  const long long c = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  if (c >= chunks) return;
  float a[8] = {};
  for (int s = 0; s < n_split; ++s) {
    const float4* src = reinterpret_cast<const float4*>(part + (s * chunks + c) * 8);
    const float4 x = src[0], y = src[1];
    a[0] += x.x, a[1] += x.y, a[2] += x.z, a[3] += x.w;
    a[4] += y.x, a[5] += y.y, a[6] += y.z, a[7] += y.w;
  }
  const int per_row = D / 8;
  const long long r = c / per_row, bh = r / S;
  __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(out.p) + bh / H * out.sb + bh % H * out.sh + r % S * out.ss +
                       c % per_row * 8;
  *reinterpret_cast<uint4*>(dst) = make_uint4(pack_bf16x2(a[0], a[1]), pack_bf16x2(a[2], a[3]),
                                              pack_bf16x2(a[4], a[5]), pack_bf16x2(a[6], a[7]));
}

// dbias[u, h] from the CTAs' rows part[b][h][block][u]: one warp an entry, its lanes take
// every 32nd row, then a fixed tree.
__global__ void __launch_bounds__(128) ffa_gen_bias_sum_kernel(const float* __restrict__ part,
                                                               __nv_bfloat16* __restrict__ dbias, int B, int H,
                                                               int blocks, int buckets) {
  const int lane = threadIdx.x & 31;
  const int e = blockIdx.x * 4 + (threadIdx.x >> 5);
  if (e >= H * buckets) return;
  const int h = e / buckets, u = e % buckets;
  float a = 0.f;
  for (int r = lane; r < B * blocks; r += 32)
    a += part[((static_cast<long long>(r / blocks) * H + h) * blocks + r % blocks) * buckets + u];
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) a += __shfl_xor_sync(0xffffffffu, a, x);
  if (lane == 0) dbias[static_cast<long long>(u) * H + h] = __float2bfloat16_rn(a);
}

// Head h's table (ffa_gen_table_kernel) into shared memory.
__device__ __forceinline__ void copy_table(float* tab, const float* tables, int h, const Bias& bias, int tid, int n) {
  const int units = table_size(bias) / 4;
  const float4* src = reinterpret_cast<const float4*>(tables) + static_cast<long long>(h) * units;
  for (int t = tid; t < units; t += n) reinterpret_cast<float4*>(tab)[t] = src[t];
}

// Give this lane's share of an accumulator (half of the columns for warpgroup g), times
// `mul`, to the staged bf16 tile (128 rows, for a TMA store) or, with `part`, to the warp's
// fp32 rows of `true_d` values, of which `rows` exist.  `empty`: nothing was accumulated, and tensor memory may hold
// anything: zeros.  The whole warp calls it.
template <int D>
__device__ __forceinline__ void give_acc(uint32_t t_acc, int g, uint32_t tile, int row, float* part, int true_d,
                                         bool done, int rows, bool empty, float mul) {
  if (!done) return;
  __syncwarp();  // tensor memory is loaded by whole warps
#pragma unroll 1
  for (int c = g * (D / 2); c < (g + 1) * (D / 2); c += 32) {
    uint32_t r[32];
    if (empty) {
#pragma unroll
      for (int e = 0; e < 32; ++e) r[e] = 0u;
    } else {
      tmem_ld32(t_acc + c, r);
      tmem_ld_wait();
    }
    if (part == nullptr)
      stage_row32_sw128(tile, row, c, r, mul);
    else  // the tile's room is this function's scratch: 4 KB for each of eight warps
      write_rows32(tile + (threadIdx.x >> 5) * 4096, part, c, true_d, rows, r, mul, threadIdx.x & 31);
  }
}

// Barrier of the compute threads, then one TMA store of each staged tile (see
// bwd::store_staged).
template <int D, int NT>
__device__ __forceinline__ void store_staged(bool staged, const CUtensorMap* const (&maps)[NT], uint32_t first_tile,
                                             int row0, int h, int b) {
  fence_proxy_async_smem();
  const bool all = whole_barrier_and(1, 256, staged);
  if (all && threadIdx.x == 0) {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int sl = 0; sl < D / 64; ++sl)
        tma_store_4d(maps[t], first_tile + t * (128 * D * 2) + sl * 16384, sl * 64, row0, h, b);
    bulk_commit_group();
    bulk_wait_read();
  }
}

// ====================================================================================
// dK / dV
// ====================================================================================
// Shape of a CTA: two compute warpgroups, each with CW columns of a step (thread = TMEM lane
// = row), then the control warps.  At D = 128 setmaxnreg moves registers from those to the
// compute warpgroups (see ffa_bwd.cuh); at D = 64 all threads have the same.
template <int D>
struct BwdShape {
  static constexpr int CW = D == 64 ? 32 : 64;
  static constexpr int STEP = 2 * CW;
  static constexpr int CTAS = D == 64 ? 2 : 1;  // of an SM
  static constexpr int TMEM = D == 64 ? 256 : 512;
  static constexpr int THREADS = D == 64 ? 320 : bwd::NTHREADS;
  static constexpr int PRODUCER = 8, MMA = 9, DO_PRODUCER = D == 64 ? -1 : 10;  // warps
};

// TMEM column of the 16-deep K-step `ks` of a packed-bf16 A operand that the two warpgroups
// wrote, CW values each (CW / 2 columns, CW columns apart).
template <int CW>
__device__ __forceinline__ constexpr uint32_t kstep_col(int ks) {
  return (ks / (CW / 16)) * CW + (ks % (CW / 16)) * 8;
}

// Load / store N (16, 32 or 64) consecutive columns of this lane.
__device__ __forceinline__ void ld_cols(uint32_t taddr, float (&v)[64]) { bwd::tmem_ld64(taddr, v); }
__device__ __forceinline__ void ld_cols(uint32_t taddr, float (&v)[32]) {
  uint32_t r[32];
  tmem_ld32(taddr, r);
  tmem_ld_wait();
#pragma unroll
  for (int e = 0; e < 32; ++e) v[e] = __uint_as_float(r[e]);
}
__device__ __forceinline__ void st_cols(uint32_t taddr, const uint32_t (&r)[32]) { tmem_st32(taddr, r); }
__device__ __forceinline__ void st_cols(uint32_t taddr, const uint32_t (&r)[16]) { tmem_st16(taddr, r); }

template <int D, bool BIAS>
struct DkdvLayout {
  static constexpr int STEP = BwdShape<D>::STEP;
  static constexpr int KV_TILE = 128 * D * 2;   // K, V (resident)
  static constexpr int TILE = STEP * D * 2;     // Q, dO (streamed)
  static constexpr int Q_STAGES = 3;
  static constexpr int DO_STAGES = 2;
  static constexpr int K_OFF = 0;
  static constexpr int V_OFF = KV_TILE;
  static constexpr int Q_OFF = 2 * KV_TILE;
  static constexpr int DO_OFF = Q_OFF + Q_STAGES * TILE;
  static constexpr int STAT_BYTES = 2 * STEP * 4;  // lse, delta behind a dO tile
  static constexpr int DO_STAGE_BYTES = TILE + 1024;
  // tensor memory: S^T, dP^T (P and dS are written over it), dV, dK
  static constexpr uint32_t DP_COL = STEP, DV_COL = 2 * STEP, DK_COL = 2 * STEP + D;
  static constexpr int BAR_OFF = DO_OFF + DO_STAGES * DO_STAGE_BYTES;
  // kv_full, q_full[], q_empty[], do_full[2], do_empty[2], s_full, dp_full, p_ready,
  // ds_ready, final, drain, s_free
  static constexpr int NBARS = 1 + 2 * Q_STAGES + 2 * DO_STAGES + 7;
  static constexpr int MISC_OFF = BAR_OFF + NBARS * 8;
  // At D = 128 there is room for the bias table or for a third Q slot.  The slot is worth
  // more, and the steps near the diagonal read the table from L2 (B2 H16 S4096 causal: 257 us
  // against 281 with the table; with all steps near, distance 1024, 262
  // against 284).
  static constexpr bool TAB_SHARED = BIAS && D == 64;
  static constexpr int TAB_OFF = (MISC_OFF + 16 + 15) / 16 * 16;
  static constexpr int MOST = TAB_OFF + (TAB_SHARED ? kTableMax * 4 : 0);
  // no alignment slack (see bwd::DkdvLayout)
  static int smem_bytes(const Bias& bias) { return TAB_OFF + (TAB_SHARED ? table_size(bias) * 4 : 0); }
};

template <int D, bool CAUSAL, bool BIAS>
__global__ void __launch_bounds__(BwdShape<D>::THREADS, BwdShape<D>::CTAS)
    ffa_gen_dkdv_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                        const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_do,
                        const __grid_constant__ CUtensorMap tm_dk, const __grid_constant__ CUtensorMap tm_dv,
                        const __grid_constant__ Problem pr, const __grid_constant__ Bias bias,
                        const float* tables, const float* LSE, const float* DELTA, float* __restrict__ dk_part,
                        float* __restrict__ dv_part, int n_split, int group) {
  using L = DkdvLayout<D, BIAS>;
  using W = BwdShape<D>;
  constexpr int SLABS = D / 64, STEP = W::STEP, CW = W::CW;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw;
  if (smem_u32(smem) & 1023u) {  // the layout has no room to realign: report and leave
    if (threadIdx.x == 0) atomicCAS(&g_status[0], 0u, static_cast<unsigned int>(kErrBwdAlign));
    return;
  }
  const uint32_t sbase = smem_u32(smem);
  const uint32_t bar0 = sbase + L::BAR_OFF;
  constexpr int QS = L::Q_STAGES, DS = L::DO_STAGES;
  const uint32_t kv_full = bar0;
  auto q_full = [&](int s) { return bar0 + 8 * (1 + s); };
  auto q_empty = [&](int s) { return bar0 + 8 * (1 + QS + s); };
  auto do_full = [&](int s) { return bar0 + 8 * (1 + 2 * QS + s); };
  auto do_empty = [&](int s) { return bar0 + 8 * (1 + 2 * QS + DS + s); };
  const uint32_t s_full = bar0 + 8 * (1 + 2 * QS + 2 * DS);
  const uint32_t dp_full = s_full + 8;
  const uint32_t p_ready = s_full + 16;
  const uint32_t ds_ready = s_full + 24;
  const uint32_t final_bar = s_full + 32;
  const uint32_t drain_bar = s_full + 40;
  const uint32_t s_free = s_full + 48;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::MISC_OFF);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::MISC_OFF + 4);
  auto q_addr = [&](int i) { return sbase + L::Q_OFF + (i % QS) * L::TILE; };
  auto do_addr = [&](int i) { return sbase + L::DO_OFF + (i % DS) * L::DO_STAGE_BYTES; };
  auto lse_smem = [&](int i) {
    return reinterpret_cast<const float*>(smem + L::DO_OFF + (i % DS) * L::DO_STAGE_BYTES + L::TILE);
  };

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  // work: (block of 128 keys, split of the steps) of one (sequence, key head); under a causal
  // mask the first key blocks have the most queries and come first
  const CtaWork cw = cta_work((pr.Sk + 127) / 128 * n_split, pr.B * pr.Hkv, group);
  const int split = cw.rank % n_split;
  const int b = pr.seq_at(cw.bh / pr.Hkv), hk = cw.bh % pr.Hkv;
  const int n0 = cw.rank / n_split * 128;
  const int off = (CAUSAL || BIAS) ? pr.offset(b) : 0;
  const int n_keys = pr.keys(b, off, CAUSAL);
  // first query block that sees a key of this block (query i sees key j iff j <= i + off)
  const int q_begin = CAUSAL ? max(0, n0 - off) / STEP * STEP : 0;
  const int nqb = (n0 < n_keys && q_begin < pr.Sq) ? (pr.Sq - q_begin + STEP - 1) / STEP : 0;
  // steps: the query blocks of each head of the group, one head after another
  const int steps = nqb * pr.G;
  const int per_split = (steps + n_split - 1) / n_split;
  const int st0 = min(split * per_split, steps);
  const int ns = min(per_split, steps - st0);
  const int rows_p = padded_rows(pr.Sq);

  if (threadIdx.x == 0) {
    mbar_init(kv_full, 1);
    for (int s = 0; s < QS; ++s) {
      mbar_init(q_full(s), 1);
      mbar_init(q_empty(s), 1);
    }
    for (int s = 0; s < DS; ++s) {
      mbar_init(do_full(s), 1);
      mbar_init(do_empty(s), 1);
    }
    mbar_init(s_full, 1);
    mbar_init(s_free, 256);
    mbar_init(dp_full, 1);
    mbar_init(p_ready, 256);
    mbar_init(ds_ready, 256);
    mbar_init(final_bar, 1);
    mbar_init(drain_bar, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == W::MMA) {
    tmem_alloc(smem_u32(tmem_slot), W::TMEM);
    tmem_relinquish();
  }
  if (warp == W::PRODUCER && lane == 0) {
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_do);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  // LSE and delta are written.  Each warp waits for that itself before its first wait that
  // depends on them: the time limit of a wait on a barrier is for this kernel's own work.
  auto wait_stats = [&]() { asm volatile("griddepcontrol.wait;" ::: "memory"); };
  if (warp >= 8) {
    if constexpr (D == 128) setmaxnreg_dec<bwd::REGS_CONTROL>();
    const uint64_t keep = policy_evict_last();
    auto load_q = [&](int it) -> bool {
      const int s = it % QS;
      if (!mbar_wait(q_empty(s), ((it / QS) & 1) ^ 1, abort_flag, kErrGenDkdvProducer)) return false;
      const int hg = (st0 + it) / nqb, q0 = q_begin + (st0 + it) % nqb * STEP;
      mbar_arrive_expect_tx(q_full(s), L::TILE);
      for (int sl = 0; sl < SLABS; ++sl)
        tma_load_4d(q_addr(it) + sl * (STEP * 128), &tm_q, q_full(s), sl * 64, q0, hk * pr.G + hg, b, keep);
      return true;
    };
    auto load_do = [&](int it) -> bool {  // dO with its LSE and delta
      const int s = it % DS;
      if (!mbar_wait(do_empty(s), ((it / DS) & 1) ^ 1, abort_flag, kErrGenDkdvProducer)) return false;
      const int h = hk * pr.G + (st0 + it) / nqb, q0 = q_begin + (st0 + it) % nqb * STEP;
      mbar_arrive_expect_tx(do_full(s), L::TILE + L::STAT_BYTES);
      for (int sl = 0; sl < SLABS; ++sl)
        tma_load_4d(do_addr(it) + sl * (STEP * 128), &tm_do, do_full(s), sl * 64, q0, h, b, keep);
      const long long r = static_cast<long long>(b * pr.Hq + h) * rows_p + q0;
      bulk_load(do_addr(it) + L::TILE, LSE + r, STEP * 4, do_full(s));
      bulk_load(do_addr(it) + L::TILE + STEP * 4, DELTA + r, STEP * 4, do_full(s));
      return true;
    };
    if (warp == W::PRODUCER) {
      // -------------------------------------------------------------- producer: K, V, Q ring
      if (lane == 0) {
        int n_q = 0, n_do = 0;
        if (ns > 0) {
          mbar_arrive_expect_tx(kv_full, 2 * L::KV_TILE);
          for (int sl = 0; sl < SLABS; ++sl) {
            tma_load_4d(sbase + L::K_OFF + sl * 16384, &tm_k, kv_full, sl * 64, n0, hk, b, keep);
            tma_load_4d(sbase + L::V_OFF + sl * 16384, &tm_v, kv_full, sl * 64, n0, hk, b, keep);
          }
        }
        bool ok = true;
        for (int it = 0; it < ns && ok; ++it) {
          if (W::DO_PRODUCER >= 0 && it == QS) wait_stats();
          if ((ok = load_q(it))) ++n_q;
          if (W::DO_PRODUCER < 0 && ok) {
            if (it == 0) wait_stats();
            if ((ok = load_do(it))) ++n_do;
          }
        }
        if (W::DO_PRODUCER < 0 && ns <= 0) wait_stats();
        if (*abort_flag) {
          if (ns > 0) mbar_wait_drain(kv_full, 0);
          for (int x = max(0, n_q - QS); x < n_q; ++x) mbar_wait_drain(q_full(x % QS), (x / QS) & 1);
          for (int x = max(0, n_do - DS); x < n_do; ++x) mbar_wait_drain(do_full(x % DS), (x / DS) & 1);
        }
      }
    } else if (warp == W::DO_PRODUCER) {
      // -------------------------------------------------------------- producer: dO ring
      if (lane == 0) {
        wait_stats();
        int it = 0;
        while (it < ns && load_do(it)) ++it;
        if (*abort_flag)
          for (int x = max(0, it - DS); x < it; ++x) mbar_wait_drain(do_full(x % DS), (x / DS) & 1);
      }
    } else if (warp == W::MMA) {
      // -------------------------------------------------------------- MMA issuer
      constexpr uint32_t IDESC_SD = idesc_bf16(128, STEP, false, false);  // [128 keys x STEP queries]
      constexpr uint32_t IDESC_G = idesc_bf16(128, D, false, true);      // [128 keys x D]
      const uint64_t kdesc = kmajor_desc(sbase + L::K_OFF, 128, 0), vdesc = kmajor_desc(sbase + L::V_OFF, 128, 0);
      auto issue_s = [&](int i) -> bool {  // S^T = K Q_i^T
        if (!mbar_wait(q_full(i % QS), (i / QS) & 1, abort_flag, kErrGenDkdvMma)) return false;
        tc_fence_after();
        const uint64_t qd = kmajor_desc(q_addr(i), STEP, 0);
        if (elect_one()) {
          mma_ss(tmem, kdesc, qd, IDESC_SD, 0u);
#pragma unroll
          for (int ks = 1; ks < D / 16; ++ks)
            mma_ss_acc(tmem, kdesc + kmajor_step(128, ks), qd + kmajor_step(STEP, ks), IDESC_SD);
          mma_commit(s_full);
        }
        __syncwarp();
        return true;
      };
      auto issue_dp = [&](int i) -> bool {  // dP^T = V dO_i^T
        if (!mbar_wait(do_full(i % DS), (i / DS) & 1, abort_flag, kErrGenDkdvMma)) return false;
        tc_fence_after();
        const uint64_t dd = kmajor_desc(do_addr(i), STEP, 0);
        if (elect_one()) {
          mma_ss(tmem + L::DP_COL, vdesc, dd, IDESC_SD, 0u);
#pragma unroll
          for (int ks = 1; ks < D / 16; ++ks)
            mma_ss_acc(tmem + L::DP_COL, vdesc + kmajor_step(128, ks), dd + kmajor_step(STEP, ks), IDESC_SD);
          mma_commit(dp_full);
        }
        __syncwarp();
        return true;
      };
      auto issue_dv = [&](int i) -> bool {  // dV += P^T dO_i
        if (!mbar_wait(p_ready, i & 1, abort_flag, kErrGenDkdvMma)) return false;
        tc_fence_after();
        const uint64_t dd = mnmajor_desc(do_addr(i), STEP, 0);
        if (elect_one()) {
          mma_ts(tmem + L::DV_COL, tmem + L::DP_COL, dd, IDESC_G, i > 0 ? 1u : 0u);
#pragma unroll
          for (int ks = 1; ks < STEP / 16; ++ks)
            mma_ts_acc(tmem + L::DV_COL, tmem + L::DP_COL + kstep_col<CW>(ks), dd + mnmajor_step(ks), IDESC_G);
        }
        __syncwarp();
        return true;
      };
      auto issue_dk = [&](int i) -> bool {  // dK += dS^T Q_i
        if (!mbar_wait(ds_ready, i & 1, abort_flag, kErrGenDkdvMma)) return false;
        tc_fence_after();
        const uint64_t qd = mnmajor_desc(q_addr(i), STEP, 0);
        if (elect_one()) {
          mma_ts(tmem + L::DK_COL, tmem + L::DP_COL + CW / 2, qd, IDESC_G, i > 0 ? 1u : 0u);
#pragma unroll
          for (int ks = 1; ks < STEP / 16; ++ks)
            mma_ts_acc(tmem + L::DK_COL, tmem + L::DP_COL + CW / 2 + kstep_col<CW>(ks), qd + mnmajor_step(ks), IDESC_G);
          mma_commit(q_empty(i % QS));
          mma_commit(do_empty(i % DS));
        }
        __syncwarp();
        return true;
      };
      bool ok = true;
      if (ns > 0) {
        ok = mbar_wait(kv_full, 0, abort_flag, kErrGenDkdvMma);
        if (ok && n0 + 128 > n_keys && n_keys < pr.Sk) {
          zero_tail(sbase + L::K_OFF, SLABS, n_keys - n0, lane);
          zero_tail(sbase + L::V_OFF, SLABS, n_keys - n0, lane);
        }
        ok = ok && issue_s(0);
        wait_stats();
        ok = ok && issue_dp(0);
      }
      // S(i+1) as soon as the warpgroups have copied S(i) into registers, then dV(i), dK(i)
      // and dP(i+1): P(i) and dS(i) live in the dP columns.
      for (int i = 0; i < ns && ok; ++i) {
        if (i + 1 < ns) {
          if (!(ok = mbar_wait(s_free, i & 1, abort_flag, kErrGenDkdvMma))) break;
          tc_fence_after();
          if (!(ok = issue_s(i + 1))) break;
        }
        if (!(ok = issue_dv(i))) break;
        if (!(ok = issue_dk(i))) break;
        if (i + 1 < ns && !(ok = issue_dp(i + 1))) break;
      }
      if (elect_one()) {
        if (ok) mma_commit(final_bar);
        mma_commit(drain_bar);
      }
      __syncwarp();
      mbar_wait_drain(drain_bar, 0);
    }
    __syncwarp();
  } else {
    if constexpr (D == 128) setmaxnreg_inc<bwd::REGS_COMPUTE>();
    // ---------------------------------------------------------------- compute
    const int g = warp >> 2;                 // warpgroup: query columns [CW g, CW g + CW) of a step
    const int row = (warp & 3) * 32 + lane;  // key row within the block
    const int kg = n0 + row;
    const int kw = n0 + (warp & 3) * 32;  // the warp's first key
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + lane_off + CW * g;
    const uint32_t t_dp = tmem + lane_off + L::DP_COL + CW * g;
    // first query that sees this key (none: past every query)
    const int q_first = kg >= n_keys ? INT_MAX : (CAUSAL ? kg - off : -1);
    const float2 c2 = make_float2(pr.scale_log2, pr.scale_log2);
    bool ok = true;
    int i = 0;
    wait_stats();  // and the bias tables
    // heads of the group; all compute threads pass the barriers of every head
    for (int hg = ns > 0 ? st0 / nqb : 0; i < ns || !ok; ++hg) {
      if (!ok && hg * nqb >= st0 + ns) break;
      float bias_l = 0.f, bias_r = 0.f;
      const float* tab = nullptr;  // the head's table
      if (BIAS) {
        if constexpr (L::TAB_SHARED) {
          float* room = reinterpret_cast<float*>(smem + L::TAB_OFF);
          ok = whole_barrier_and(2, 256, ok);  // everyone is done with the last head's table
          copy_table(room, tables, hk * pr.G + hg, bias, threadIdx.x, 256);
          ok = whole_barrier_and(2, 256, ok);
          tab = room;
        } else {
          tab = tables + static_cast<long long>(hk * pr.G + hg) * table_size(bias);
        }
        bias_l = tab[0];
        bias_r = tab[table_last(bias)];
      }
      const int head_end = min(ns, (hg + 1) * nqb - st0);
      for (; ok && i < head_end; ++i) {
        const int qc = q_begin + (st0 + i - hg * nqb) * STEP + CW * g;  // first query of this thread's columns
        if (!(ok = mbar_wait(do_full(i % DS), (i / DS) & 1, abort_flag, kErrGenDkdvCompute))) break;
        const float* lse_s = lse_smem(i) + CW * g;
        const float* dl_s = lse_s + STEP;
        float p[CW];
        if (!(ok = mbar_wait(s_full, i & 1, abort_flag, kErrGenDkdvCompute))) break;
        tc_fence_after();
        ld_cols(t_s, p);
        tc_fence_before();
        mbar_arrive(s_free);  // S may now be overwritten by S(i+1)
        uint32_t pk[CW / 2];
        {
          const bool masked = kw + 32 > n_keys || (CAUSAL && qc + off < kw + 31);
          bool near = false;
          float fb = 0.f;
          if (BIAS) {
            const int r_min = kw - (off + qc + CW - 1), r_max = kw + 31 - (off + qc);
            near = r_min < bias.right && r_max > -bias.left;
            fb = r_min >= bias.right ? bias_r : bias_l;
          }
          if (BIAS && near) {
            // scores that look their bias up: into the score first, the rest as below
            const float* tp = tab + (kg - off - qc + bias.left + kPad);
#pragma unroll
            for (int e = 0; e < CW; ++e) p[e] = fmaf(p[e], pr.scale_log2, tp[-e]);
          }
          const float2 cc = (BIAS && near) ? make_float2(1.f, 1.f) : c2;
          const float fc = (BIAS && near) ? 0.f : fb;
#pragma unroll
          for (int e = 0; e < CW; e += 4) {
            const float4 l4 = *reinterpret_cast<const float4*>(lse_s + e);
            float2 la = make_float2(-l4.x, -l4.y), lb = make_float2(-l4.z, -l4.w);
            if (BIAS) {
              la = add2(la, make_float2(fc, fc));
              lb = add2(lb, make_float2(fc, fc));
            }
            const float2 xa = fma2(make_float2(p[e], p[e + 1]), cc, la);
            const float2 xb = fma2(make_float2(p[e + 2], p[e + 3]), cc, lb);
            // (a quarter on the FMA pipe, exp2_fma2, changes the time by less than 1 %)
            p[e + 0] = fast_exp2(xa.x);
            p[e + 1] = fast_exp2(xa.y);
            p[e + 2] = fast_exp2(xb.x);
            p[e + 3] = fast_exp2(xb.y);
          }
          if (masked) {  // apart from the loop, so that other steps branch around it
            const int first = q_first - min(qc, 1 << 30);  // column of the first query that sees the key
#pragma unroll
            for (int e = 0; e < CW; ++e)
              if (e < first) p[e] = 0.f;
          }
#pragma unroll
          for (int e = 0; e < CW / 2; ++e) pk[e] = pack_bf16x2(p[2 * e], p[2 * e + 1]);
        }
        if (!(ok = mbar_wait(dp_full, i & 1, abort_flag, kErrGenDkdvCompute))) break;
        tc_fence_after();
        // dP(i) comes into registers 32 columns at a time; P(i) and dS(i) then take its columns
        uint32_t dp[CW / 32][32];
        tmem_ld32(t_dp, dp[0]);
        tmem_ld_wait();
        st_cols(t_dp, pk);
        if constexpr (CW == 64) {
          tmem_ld32(t_dp + 32, dp[1]);
          tmem_ld_wait();
        }
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(p_ready);
        {
          uint32_t dk[CW / 2];
#pragma unroll
          for (int e = 0; e < CW; e += 4) {
            const float4 d4 = *reinterpret_cast<const float4*>(dl_s + e);
            const uint32_t* src = dp[e / 32];
            const int x = e & 31;
            const float2 da = mul2(make_float2(p[e], p[e + 1]),
                                   sub2(make_float2(__uint_as_float(src[x]), __uint_as_float(src[x + 1])),
                                        make_float2(d4.x, d4.y)));
            const float2 db = mul2(make_float2(p[e + 2], p[e + 3]),
                                   sub2(make_float2(__uint_as_float(src[x + 2]), __uint_as_float(src[x + 3])),
                                        make_float2(d4.z, d4.w)));
            dk[e / 2] = pack_bf16x2(da.x, da.y);
            dk[e / 2 + 1] = pack_bf16x2(db.x, db.y);
          }
          st_cols(t_dp + CW / 2, dk);
          tmem_st_wait();
        }
        tc_fence_before();
        mbar_arrive(ds_ready);
      }
    }
    const bool empty = ns <= 0;
    const bool done = ok && (empty || mbar_wait(final_bar, 0, abort_flag, kErrGenDkdvCompute));
    tc_fence_after();
    // every MMA has finished: K's and V's room holds the staged dV and dK tiles
    const long long r = (static_cast<long long>(split) * pr.B * pr.Hkv + b * pr.Hkv + hk) * pr.Sk + kw;
    give_acc<D>(tmem + lane_off + L::DV_COL, g, sbase + L::K_OFF, row, n_split > 1 ? dv_part + r * pr.D : nullptr,
                     pr.D, done, pr.Sk - kw, empty, 1.f);
    give_acc<D>(tmem + lane_off + L::DK_COL, g, n_split > 1 ? sbase + L::K_OFF : sbase + L::V_OFF, row, n_split > 1 ? dk_part + r * pr.D : nullptr,
                     pr.D, done, pr.Sk - kw, empty, pr.scale);
    if (n_split == 1) {
      const CUtensorMap* const maps[2] = {&tm_dv, &tm_dk};
      store_staged<D, 2>(done, maps, sbase + L::K_OFF, n0, hk, b);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == W::MMA) {
    tc_fence_after();
    tmem_dealloc(tmem, W::TMEM);
  }
}

// ====================================================================================
// dQ and dbias
// ====================================================================================
// Floats of scratch of a warp for add_near_block: 47 diagonals of each chain.
template <int CW>
constexpr int kDiagFloats = CW / 16 * 48;

template <int D, bool BIAS>
struct DqLayout {
  static constexpr int STEP = BwdShape<D>::STEP;
  static constexpr int TILE = STEP * D * 2;
  static constexpr int K_STAGES = (BIAS && D == 128) ? 3 : 4;  // the bias part takes one slot's room
  static constexpr int V_STAGES = 3;
  static constexpr int K_OFF = 0;  // also stages the output: 128 rows in two slots at least
  static constexpr int V_OFF = K_OFF + K_STAGES * TILE;
  // tensor memory: S, dP (dS is written over it), dQ, then Q and dO as packed A operands
  static constexpr uint32_t DP = STEP, DQ = 2 * STEP, Q = 2 * STEP + D, DO = 2 * STEP + D + D / 2;
  static constexpr int BAR_OFF = V_OFF + V_STAGES * TILE;
  // qd_ready, k_full[], k_empty[], v_full[3], v_empty[3], s_full, s_free, dp_full, ds_ready,
  // final, drain
  static constexpr int NBARS = 1 + 2 * K_STAGES + 2 * V_STAGES + 6;
  static constexpr int MISC_OFF = BAR_OFF + NBARS * 8;
  static constexpr int DELTA_OFF = (MISC_OFF + 16 + 15) / 16 * 16;  // delta of the block's rows
  // bias: diagonal scratch of each warp, table (fp32 by position), buckets by position,
  // per-warp sums
  static constexpr int DIAG_OFF = DELTA_OFF + 512;
  static constexpr int TAB_OFF = DIAG_OFF + (BIAS ? 8 * kDiagFloats<BwdShape<D>::CW> * 4 : 0);
  static int smem_bytes(const Bias& bias) {
    return TAB_OFF + (BIAS ? table_size(bias) * 4 + lut_size(bias) * 2 + 8 * bias.buckets * 4 : 0) + 1024;
  }
  // at most, with kMaxDistance and kMaxBuckets
  static constexpr int MOST = TAB_OFF + (BIAS ? kTableMax * 4 + (2 * kMaxDistance + 8) * 2 + 8 * kMaxBuckets * 4 : 0) + 1024;
};

// Copy this thread's row of `true_d` bf16 values into D/2 packed TMEM columns (the rest
// zero).  Every lane of the warp calls it.
template <int D>
__device__ __forceinline__ void row_to_tmem(const __nv_bfloat16* __restrict__ src, bool valid, int true_d,
                                            uint32_t taddr) {
#pragma unroll
  for (int c = 0; c < D / 64; ++c) {
    uint32_t w[32];
    const uint4* s4 = reinterpret_cast<const uint4*>(src + 64 * c);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint4 x = (valid && 64 * c + 8 * e < true_d) ? __ldg(s4 + e) : make_uint4(0u, 0u, 0u, 0u);
      w[4 * e + 0] = x.x;
      w[4 * e + 1] = x.y;
      w[4 * e + 2] = x.z;
      w[4 * e + 3] = x.w;
    }
    tmem_st32(taddr + 32 * c, w);
  }
}

// The same, and the row's dot product with `other` and, where given, its remainder `rem`.
template <int D>
__device__ __forceinline__ float row_dot_to_tmem(const __nv_bfloat16* __restrict__ src,
                                                 const __nv_bfloat16* __restrict__ other,
                                                 const __nv_bfloat16* __restrict__ rem, bool valid, int true_d,
                                                 uint32_t taddr) {
  float acc = 0.f;
  auto add = [&](uint32_t x, uint32_t y) {
    const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&x));
    const float2 b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&y));
    acc = fmaf(a.x, b.x, acc);
    acc = fmaf(a.y, b.y, acc);
  };
#pragma unroll
  for (int c = 0; c < D / 64; ++c) {
    uint32_t w[32];
    const uint4 *s4 = reinterpret_cast<const uint4*>(src + 64 * c), *o4 = reinterpret_cast<const uint4*>(other + 64 * c);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const bool in = valid && 64 * c + 8 * e < true_d;
      const uint4 x = in ? __ldg(s4 + e) : make_uint4(0u, 0u, 0u, 0u);
      const uint4 y = in ? __ldg(o4 + e) : make_uint4(0u, 0u, 0u, 0u);
      w[4 * e + 0] = x.x;
      w[4 * e + 1] = x.y;
      w[4 * e + 2] = x.z;
      w[4 * e + 3] = x.w;
      add(x.x, y.x);
      add(x.y, y.y);
      add(x.z, y.z);
      add(x.w, y.w);
    }
    if (rem != nullptr) {  // apart, so that its loads go out together as well
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const bool in = valid && 64 * c + 8 * e < true_d;
        const uint4 z = in ? __ldg(reinterpret_cast<const uint4*>(rem + 64 * c) + e) : make_uint4(0u, 0u, 0u, 0u);
        add(w[4 * e + 0], z.x);
        add(w[4 * e + 1], z.y);
        add(w[4 * e + 2], z.z);
        add(w[4 * e + 3], z.w);
      }
    }
    tmem_st32(taddr + 32 * c, w);
  }
  return acc;
}

// Add the diagonal sums of a warp's 32 x CW block of dS (lane = row, ds[e] = column e) to
// the warp's sums by bucket.  `r0`: relative position of lane 0, column 0; `lut`: bucket of
// position r at r + left; `diag`: scratch of this warp.
//
// A chain takes 16 columns.  Before its column e, lane l holds the sum of diagonal e - l over
// the lanes below it; after it lane 31's diagonal e - 31 is complete, and comes round to
// lane 0.  The chains are independent: one over all columns would wait for 64 shuffles in
// turn.  For the same reason the chunks of diagonals are summed by bucket side by side.  (dQ of
// B2 H16 S4096 D128 causal, distance 256 and 1024: 289 and 365 us with one chain and one
// chunk after another, 267 and 315 so.  Chains of 8 columns: 268 and 317.  As a product with a
// selection matrix, mma.sync, beside the kernel's own: 327 and 370.)
template <int CW>
__device__ __forceinline__ void add_near_block(const float (&ds)[CW], int r0, const Bias& bias,
                                               const unsigned short* lut, float* sums, float* diag, int lane) {
  constexpr int CHAINS = CW / 16;
  float a[CHAINS] = {};
#pragma unroll
  for (int e = 0; e < 16; ++e) {
#pragma unroll
    for (int q = 0; q < CHAINS; ++q) {
      if (e > 0) {
        a[q] = __shfl_sync(0xffffffffu, a[q], (lane + 31) & 31);
        if (lane == 0) {
          diag[q * 48 + e - 1] = a[q];  // diagonal e - 32, kept 31 places on
          a[q] = 0.f;
        }
      }
      a[q] += ds[q * 16 + e];
    }
  }
#pragma unroll
  for (int q = 0; q < CHAINS; ++q) diag[q * 48 + 46 - lane] = a[q];  // diagonal 15 - l
  __syncwarp();
  constexpr int NC = CW / 32 + 1;  // chunks of 32 of the CW + 31 diagonals; the last lane of the last one has none
  float v[NC];
  int u[NC], head[NC];
  bool last[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int x = c * 32 + lane;
    v[c] = 0.f;
#pragma unroll
    for (int q = 0; q < CHAINS; ++q)
      if (x >= q * 16 && x < q * 16 + 47) v[c] += diag[q * 48 + x - q * 16];
    const int r = min(max(r0 + x - 31, -bias.left), bias.right);
    u[c] = lut[r + bias.left];
    // positions of one bucket are neighbours: sums of runs of equal buckets
    const int prev = __shfl_up_sync(0xffffffffu, u[c], 1);
    const uint32_t heads = __ballot_sync(0xffffffffu, lane == 0 || prev != u[c]);
    head[c] = 31 - __clz(heads & (0xffffffffu >> (31 - lane)));
    last[c] = lane == 31 || ((heads >> (lane + 1)) & 1u);  // the run's last lane
  }
#pragma unroll
  for (int k = 1; k < 32; k <<= 1) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const float y = __shfl_up_sync(0xffffffffu, v[c], k);
      if (lane - k >= head[c]) v[c] += y;
    }
  }
#pragma unroll
  for (int c = 0; c < NC; ++c) {  // a chunk's runs differ in bucket, those of two chunks need not
    if (last[c]) sums[u[c]] += v[c];
    __syncwarp();
  }
}

template <int D, bool CAUSAL, bool BIAS>
__global__ void __launch_bounds__(BwdShape<D>::THREADS, BwdShape<D>::CTAS)
    ffa_gen_dq_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                      const __grid_constant__ CUtensorMap tm_dq, const __grid_constant__ Problem pr,
                      const __grid_constant__ Bias bias, const float* tables, const unsigned short* lut_g, const View q,
                      const View o, const View o_lo, const View dout, const float* LSE, float* __restrict__ lse_out,
                      float* __restrict__ delta_out, float* __restrict__ dq_part, float* __restrict__ bias_part,
                      int n_split, int group) {
  using L = DqLayout<D, BIAS>;
  using W = BwdShape<D>;
  constexpr int SLABS = D / 64, STEP = W::STEP, CW = W::CW;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  const uint32_t bar0 = sbase + L::BAR_OFF;
  constexpr int KS = L::K_STAGES, VS = L::V_STAGES;
  const uint32_t qd_ready = bar0;
  auto k_full = [&](int s) { return bar0 + 8 * (1 + s); };
  auto k_empty = [&](int s) { return bar0 + 8 * (1 + KS + s); };
  auto v_full = [&](int s) { return bar0 + 8 * (1 + 2 * KS + s); };
  auto v_empty = [&](int s) { return bar0 + 8 * (1 + 2 * KS + VS + s); };
  const uint32_t s_full = bar0 + 8 * (1 + 2 * KS + 2 * VS);
  const uint32_t s_free = s_full + 8;
  const uint32_t dp_full = s_full + 16;
  const uint32_t ds_ready = s_full + 24;
  const uint32_t final_bar = s_full + 32;
  const uint32_t drain_bar = s_full + 40;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::MISC_OFF);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::MISC_OFF + 4);
  float* delta_s = reinterpret_cast<float*>(smem + L::DELTA_OFF);
  float* tab = reinterpret_cast<float*>(smem + L::TAB_OFF);
  unsigned short* lut = reinterpret_cast<unsigned short*>(tab + (BIAS ? table_size(bias) : 0));
  float* sums_all = reinterpret_cast<float*>(lut + (BIAS ? lut_size(bias) : 0));

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  // work: (block of 128 queries, split of the keys) of one (sequence, query head)
  const int nblk = (pr.Sq + 127) / 128;
  const CtaWork cw = cta_work(nblk * n_split, pr.B * pr.Hq, group);
  const int qblk = CAUSAL ? nblk - 1 - cw.rank / n_split : cw.rank / n_split;
  const int split = cw.rank % n_split;
  const int b = pr.seq_at(cw.bh / pr.Hq), h = cw.bh % pr.Hq, hk = h / pr.G;
  const int bh = b * pr.Hq + h;
  const int m0 = qblk * 128;
  const int off = (CAUSAL || BIAS) ? pr.offset(b) : 0;
  const int n_keys = pr.keys(b, off, CAUSAL);
  const int end = CAUSAL ? min(n_keys, max(off + m0 + 128, 0)) : n_keys;
  const int all = (end + STEP - 1) / STEP;
  const int per_split = (all + n_split - 1) / n_split;
  const int t0 = min(split * per_split, all);
  const int nk = min(per_split, all - t0);

  if (threadIdx.x == 0) {
    mbar_init(qd_ready, 256);
    for (int s = 0; s < KS; ++s) {
      mbar_init(k_full(s), 1);
      mbar_init(k_empty(s), 1);
    }
    for (int s = 0; s < VS; ++s) {
      mbar_init(v_full(s), 1);
      mbar_init(v_empty(s), 1);
    }
    mbar_init(s_full, 1);
    mbar_init(s_free, 256);
    mbar_init(dp_full, 1);
    mbar_init(ds_ready, 256);
    mbar_init(final_bar, 1);
    mbar_init(drain_bar, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == W::MMA) {
    tmem_alloc(smem_u32(tmem_slot), W::TMEM);
    tmem_relinquish();
  }
  if (warp == W::PRODUCER && lane == 0) {
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  asm volatile("griddepcontrol.launch_dependents;");
  if (BIAS && warp < 8)
    for (int t = threadIdx.x; t < 8 * bias.buckets; t += 256) sums_all[t] = 0.f;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp >= 8) {
    if constexpr (D == 128) setmaxnreg_dec<bwd::REGS_CONTROL>();
    if (warp == W::PRODUCER) {
      // -------------------------------------------------------------- producer: K, V rings
      if (lane == 0) {
        const uint64_t keep = policy_evict_last();
        int k_issued = 0, v_issued = 0;
        for (int j = 0; j < nk; ++j) {
          const int sk = j % KS, sv = j % VS;
          if (!mbar_wait(k_empty(sk), ((j / KS) & 1) ^ 1, abort_flag, kErrGenDqProducer)) break;
          mbar_arrive_expect_tx(k_full(sk), L::TILE);
          for (int sl = 0; sl < SLABS; ++sl)
            tma_load_4d(sbase + L::K_OFF + sk * L::TILE + sl * (STEP * 128), &tm_k, k_full(sk), sl * 64, (t0 + j) * STEP, hk, b,
                        keep);
          ++k_issued;
          if (!mbar_wait(v_empty(sv), ((j / VS) & 1) ^ 1, abort_flag, kErrGenDqProducer)) break;
          mbar_arrive_expect_tx(v_full(sv), L::TILE);
          for (int sl = 0; sl < SLABS; ++sl)
            tma_load_4d(sbase + L::V_OFF + sv * L::TILE + sl * (STEP * 128), &tm_v, v_full(sv), sl * 64, (t0 + j) * STEP, hk, b,
                        keep);
          ++v_issued;
        }
        if (*abort_flag) {
          for (int it = max(0, k_issued - KS); it < k_issued; ++it) mbar_wait_drain(k_full(it % KS), (it / KS) & 1);
          for (int it = max(0, v_issued - VS); it < v_issued; ++it) mbar_wait_drain(v_full(it % VS), (it / VS) & 1);
        }
      }
    } else if (warp == W::MMA) {
      // -------------------------------------------------------------- MMA issuer
      constexpr uint32_t IDESC_SD = idesc_bf16(128, STEP, false, false);  // [128 queries x STEP keys]
      constexpr uint32_t IDESC_G = idesc_bf16(128, D, false, true);      // [128 queries x D]
      auto k_addr = [&](int j) { return sbase + L::K_OFF + (j % KS) * L::TILE; };
      auto v_addr = [&](int j) { return sbase + L::V_OFF + (j % VS) * L::TILE; };
      // rows behind the last key are zeroed before the first MMA that reads the tile
      auto fix_tail = [&](uint32_t tile, int j) {
        const int tail = n_keys - (t0 + j) * STEP;
        if (tail < STEP && n_keys < pr.Sk) zero_tail<STEP>(tile, SLABS, tail, lane);
      };
      auto issue_s = [&](int j) -> bool {  // S_j = Q K_j^T  (Q from TMEM)
        if (!mbar_wait(k_full(j % KS), (j / KS) & 1, abort_flag, kErrGenDqMma)) return false;
        fix_tail(k_addr(j), j);
        tc_fence_after();
        const uint64_t kd = kmajor_desc(k_addr(j), STEP, 0);
        if (elect_one()) {
          mma_ts(tmem, tmem + L::Q, kd, IDESC_SD, 0u);
#pragma unroll
          for (int ks = 1; ks < D / 16; ++ks)
            mma_ts_acc(tmem, tmem + L::Q + 8 * ks, kd + kmajor_step(STEP, ks), IDESC_SD);
          mma_commit(s_full);
        }
        __syncwarp();
        return true;
      };
      auto issue_dp = [&](int j) -> bool {  // dP_j = dO V_j^T  (dO from TMEM)
        if (!mbar_wait(v_full(j % VS), (j / VS) & 1, abort_flag, kErrGenDqMma)) return false;
        fix_tail(v_addr(j), j);
        tc_fence_after();
        const uint64_t vd = kmajor_desc(v_addr(j), STEP, 0);
        if (elect_one()) {
          mma_ts(tmem + L::DP, tmem + L::DO, vd, IDESC_SD, 0u);
#pragma unroll
          for (int ks = 1; ks < D / 16; ++ks)
            mma_ts_acc(tmem + L::DP, tmem + L::DO + 8 * ks, vd + kmajor_step(STEP, ks), IDESC_SD);
          mma_commit(dp_full);
          mma_commit(v_empty(j % VS));
        }
        __syncwarp();
        return true;
      };
      auto issue_g = [&](int j) -> bool {  // dQ += dS_j K_j  (dS_j packed in the dP columns)
        if (!mbar_wait(ds_ready, j & 1, abort_flag, kErrGenDqMma)) return false;
        tc_fence_after();
        const uint64_t kd = mnmajor_desc(k_addr(j), 128, 0);
        if (elect_one()) {
          mma_ts(tmem + L::DQ, tmem + L::DP, kd, IDESC_G, j > 0 ? 1u : 0u);
#pragma unroll
          for (int ks = 1; ks < STEP / 16; ++ks)
            mma_ts_acc(tmem + L::DQ, tmem + L::DP + kstep_col<CW>(ks), kd + mnmajor_step(ks), IDESC_G);
          mma_commit(k_empty(j % KS));
        }
        __syncwarp();
        return true;
      };
      bool ok = mbar_wait(qd_ready, 0, abort_flag, kErrGenDqMma);
      tc_fence_after();
      if (ok && nk > 0) ok = issue_s(0) && issue_dp(0);
      // S(j+1) once the warpgroups hold S(j) in registers; dQ(j) once dS(j) is in the dP
      // columns; then dP(j+1) over them
      for (int j = 0; j < nk && ok; ++j) {
        if (j + 1 < nk) {
          if (!(ok = mbar_wait(s_free, j & 1, abort_flag, kErrGenDqMma))) break;
          tc_fence_after();
          if (!(ok = issue_s(j + 1))) break;
        }
        if (!(ok = issue_g(j))) break;
        if (j + 1 < nk && !(ok = issue_dp(j + 1))) break;
      }
      if (elect_one()) {
        if (ok) mma_commit(final_bar);
        mma_commit(drain_bar);
      }
      __syncwarp();
      mbar_wait_drain(drain_bar, 0);
    }
    __syncwarp();
  } else {
    if constexpr (D == 128) setmaxnreg_inc<bwd::REGS_COMPUTE>();
    // ---------------------------------------------------------------- compute
    const int g = warp >> 2;
    const int row = (warp & 3) * 32 + lane;  // query row within the block
    const int qg = m0 + row;
    const int qw = m0 + (warp & 3) * 32;  // the warp's first query
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    // warpgroup 0 puts the Q rows into tensor memory, warpgroup 1 the dO rows, and takes
    // delta = O . dO on the way
    const bool row_in = qg < pr.Sq;
    auto row_of = [&](const View& x) {
      return static_cast<const __nv_bfloat16*>(x.p) + b * x.sb + h * x.sh + static_cast<long long>(row_in ? qg : 0) * x.ss;
    };
    float dl = 0.f;
    if (g == 0)
      row_to_tmem<D>(row_of(q), row_in, pr.D, tmem + lane_off + L::Q);
    else
      dl = row_dot_to_tmem<D>(row_of(dout), row_of(o), o_lo.p ? row_of(o_lo) : nullptr, row_in, pr.D, tmem + lane_off + L::DO);
    tmem_st_wait();
    tc_fence_before();
    mbar_arrive(qd_ready);
    // +inf for a row that saw no key and for rows behind the last one: their P is 0
    float lse = row_in ? LSE[static_cast<long long>(bh) * pr.Sq + qg] : INFINITY;
    if (lse == -INFINITY) lse = INFINITY;
    if (g == 1) {
      delta_s[row] = dl;
      if (split == 0) {
        const long long r = static_cast<long long>(bh) * padded_rows(pr.Sq) + qg;
        lse_out[r] = lse;
        delta_out[r] = dl;
      }
    }
    if (BIAS) {
      asm volatile("griddepcontrol.wait;" ::: "memory");  // the tables are written
      copy_table(tab, tables, h, bias, threadIdx.x, 256);
      for (int t = threadIdx.x; t < lut_size(bias) / 2; t += 256)
        reinterpret_cast<uint32_t*>(lut)[t] = reinterpret_cast<const uint32_t*>(lut_g)[t];
    }
    whole_barrier_and(2, 256, true);
    dl = delta_s[row];
    const int lim = CAUSAL ? min(n_keys - 1, qg + off) : n_keys - 1;  // last visible key
    const uint32_t t_s = tmem + lane_off + CW * g;
    const uint32_t t_dp = tmem + lane_off + L::DP + CW * g;
    float* sums = sums_all + warp * bias.buckets;
    float* diag = reinterpret_cast<float*>(smem + L::DIAG_OFF) + warp * kDiagFloats<CW>;
    float bias_l = 0.f, bias_r = 0.f, sum_l = 0.f, sum_r = 0.f;
    if (BIAS) {
      bias_l = tab[0];
      bias_r = tab[table_last(bias)];
    }
    bool ok = true;
    for (int j = 0; j < nk; ++j) {
      if (!(ok = mbar_wait(s_full, j & 1, abort_flag, kErrGenDqCompute))) break;
      tc_fence_after();
      float p[CW];
      ld_cols(t_s, p);
      tc_fence_before();
      mbar_arrive(s_free);  // S may now be overwritten by S(j+1)
      const int kc = (t0 + j) * STEP + CW * g;  // first key of this thread's columns
      const bool masked = kc + CW > n_keys || (CAUSAL && kc + CW - 1 > qw + off);
      bool near = false, right = false;
      float fb = 0.f;
      if (BIAS) {
        const int r_min = kc - (off + qw + 31), r_max = kc + CW - 1 - (off + qw);
        near = r_min < bias.right && r_max > -bias.left;
        right = r_min >= bias.right;
        fb = right ? bias_r : bias_l;
        if (near) {
          const float* tp = tab + (kc - off - qg + bias.left + kPad);
#pragma unroll
          for (int e = 0; e < CW; ++e) p[e] = fmaf(p[e], pr.scale_log2, tp[e]);
        }
      }
      const bool looked = BIAS && near;
      const float c1 = looked ? 1.f : pr.scale_log2, l1 = looked ? -lse : fb - lse;
      const float2 c2 = make_float2(c1, c1), l2 = make_float2(l1, l1);
#pragma unroll
      for (int e = 0; e < CW; e += 2) {
        const float2 x = fma2(make_float2(p[e], p[e + 1]), c2, l2);
        p[e] = fast_exp2(x.x);
        p[e + 1] = fast_exp2(x.y);
      }
      if (masked) {  // apart from the loop, so that other steps branch around it
        const int last = lim - kc;
#pragma unroll
        for (int e = 0; e < CW; ++e)
          if (e > last) p[e] = 0.f;
      }
      if (!(ok = mbar_wait(dp_full, j & 1, abort_flag, kErrGenDqCompute))) break;
      tc_fence_after();
      float dp[CW];
      ld_cols(t_dp, dp);
      uint32_t dsp[CW / 2];
      const float2 d2 = make_float2(dl, dl);
#pragma unroll
      for (int e = 0; e < CW; e += 2) {
        const float2 ds = mul2(make_float2(p[e], p[e + 1]), sub2(make_float2(dp[e], dp[e + 1]), d2));
        dsp[e >> 1] = pack_bf16x2(ds.x, ds.y);
        if (BIAS) {
          p[e] = ds.x;
          p[e + 1] = ds.y;
        }
      }
      // dS(j) over the first half of this warpgroup's dP columns: the A operand of dQ(j)
      st_cols(t_dp, dsp);
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(ds_ready);
      if (BIAS && bias_part != nullptr) {
        // this step's share of dbias, while the tensor core is at dQ(j)
        if (near) {
          add_near_block<CW>(p, kc - (off + qw), bias, lut, sums, diag, lane);
        } else {
          float2 a = make_float2(0.f, 0.f), c = a;
#pragma unroll
          for (int e = 0; e < CW; e += 4) {
            a = add2(a, make_float2(p[e], p[e + 1]));
            c = add2(c, make_float2(p[e + 2], p[e + 3]));
          }
          const float t = (a.x + a.y) + (c.x + c.y);
          if (right)
            sum_r += t;
          else
            sum_l += t;
        }
      }
    }
    const bool empty = nk <= 0;
    const bool done = ok && (empty || mbar_wait(final_bar, 0, abort_flag, kErrGenDqCompute));
    tc_fence_after();
    if (BIAS && bias_part != nullptr) {
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) {
        sum_l += __shfl_xor_sync(0xffffffffu, sum_l, x);
        sum_r += __shfl_xor_sync(0xffffffffu, sum_r, x);
      }
      if (lane == 0) {
        sums[lut[0]] += sum_l;
        sums[lut[bias.left + bias.right]] += sum_r;
      }
      if (whole_barrier_and(2, 256, done)) {
        float* dst = bias_part + (static_cast<long long>(bh) * nblk * n_split + cw.rank) * bias.buckets;
        for (int u = threadIdx.x; u < bias.buckets; u += 256) {
          float a = 0.f;
#pragma unroll
          for (int w = 0; w < 8; ++w) a += sums_all[w * bias.buckets + u];
          dst[u] = a;
        }
      }
    }
    // every MMA has finished: the K ring is free and holds the staged dQ tile
    const long long r = (static_cast<long long>(split) * pr.B * pr.Hq + bh) * pr.Sq + qw;
    give_acc<D>(tmem + lane_off + L::DQ, g, sbase + L::K_OFF, row, n_split > 1 ? dq_part + r * pr.D : nullptr, pr.D,
                     done, pr.Sq - qw, empty, pr.scale);
    if (n_split == 1) {
      const CUtensorMap* const maps[1] = {&tm_dq};
      store_staged<D, 1>(done, maps, sbase + L::K_OFF, m0, h, b);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == W::MMA) {
    tc_fence_after();
    tmem_dealloc(tmem, W::TMEM);
  }
}

}  // namespace gen
}  // namespace ffa
