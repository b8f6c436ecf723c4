// ffa_gen_step.cuh — general attention (ffa_gen_common.cuh) of a few query rows: a step of
// one or a few tokens over a cache or an encoder's states.
//
// The work is one pass over K and V, so the kernel is bound by HBM.  The G * Sq query rows
// that share a key head (row r = g * Sq + t) form items of 16 RG rows, 16 being the M of
// mma.sync m16n8k16; the tensor cores' rate does not matter here, and a 128-row tcgen05 tile
// would be empty.  Two CTAs to an SM (one with 32 rows), each a TMA warp and four (eight)
// warps that compute:
//   * a CTA takes an item, or, where items are few, a cluster of CTAs shares its keys, and
//     joins its results through distributed shared memory, in the same launch;
//   * few long sequences, or very different ones: all keys of all items, laid end to end, are
//     cut into equal shares (Work), one for each CTA.  The TMA warp walks through its share
//     without a stop: HBM sees no gaps between items.  An item that several CTAs share is
//     joined by ffa_gen_step_join_kernel, launched beside the last CTAs (programmatic
//     dependent launch), which it waits for;
//   * each warp takes 16 rows and a quarter of a tile's keys, and keeps its own running max,
//     sum and O (registers); the four warps of 16 rows are joined in shared memory at the end
//     of a segment.  ROWS8: at most 8 rows, and the softmax of the other 8 is left out.
// 64 sequences, 16 heads, one token on 1500 keys each, D64 (393 MB): 72 us, 5.5 TB/s, its
// launch and end included.
#pragma once
#include "ffa_gen_common.cuh"

namespace ffa {
namespace gen {

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Barrier of all threads of the cluster, with release and acquire of shared memory.  Like the
// barriers of a CTA it wants each warp whole.
__device__ __forceinline__ void cluster_barrier() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Load from the shared memory of the cluster's CTA `rank`, at this CTA's address `addr`.
__device__ __forceinline__ float ld_cluster(uint32_t addr, int rank) {
  float v;
  asm volatile(
      "{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %1, %2;\n\tld.shared::cluster.f32 %0, [a];\n\t}"
      : "=f"(v)
      : "r"(addr), "r"(rank)
      : "memory");
  return v;
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr, int rank) {
  float4 v;
  asm volatile(
      "{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %4, %5;\n\t"
      "ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [a];\n\t}"
      : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
      : "r"(addr), "r"(rank)
      : "memory");
  return v;
}

// ------------------------------------------------------------------------------------
// Work of a CTA
// ------------------------------------------------------------------------------------
// Items: `per_seq` for each sequence (key heads times row tiles), all with as many tiles of
// KEYS keys as the sequence has, at least one (zeros have to be written too).  CTA c of n
// gets the tiles [U c / n, U (c + 1) / n) of all U.  An item that crosses from one CTA into
// the next ones is written in parts, in fp32, normalised, with its LSE: by the CTA in which
// it starts in that CTA's slot 1, by the others in their slot 0.  With `cluster` CTAs for
// each item (one or more) the CTA of rank r takes the r-th equal part of its item.
struct Segment {
  int b, item;    // sequence, item of the sequence
  int keys, off;  // the sequence's visible keys and offset
  int t0, nt;     // first tile and number of tiles
  int tiles;      // tiles of the whole item; 0: there is no segment, the CTA is done
  __device__ __forceinline__ bool whole() const { return t0 == 0 && nt == tiles; }
};
// What the join needs of a CTA: the item that it starts and others finish (parts = 0: none),
// and whether it has a part in slot 0 (with fewer tiles than CTAs some have none).
struct JoinEntry {
  int b, item, parts, slot0;
};

// One thread walks through the CTA's segments (start() is for its whole warp).
template <bool CAUSAL, bool OFFSETS>
struct Work {
  long long left, total, end;  // tiles left to the CTA, all tiles, the tile behind the last segment
  int b, item, t, keys, off, tiles;
  bool shares;

  __device__ __forceinline__ static int tiles_of(int keys, int tile) { return max(1, (keys + tile - 1) / tile); }
  __device__ __forceinline__ void enter(const Problem& pr, int seq, int tile) {
    b = seq;
    off = OFFSETS ? pr.offset(seq) : 0;
    keys = pr.keys(seq, off, CAUSAL);
    tiles = tiles_of(keys, tile);
  }
  __device__ void start(const Problem& pr, int per_seq, int tile, int cluster) {
    shares = cluster == 0;
    if (!shares) {
      const int at = blockIdx.x / cluster, rank = blockIdx.x % cluster;
      enter(pr, at / per_seq, tile);
      item = at % per_seq;
      t = static_cast<int>(static_cast<long long>(tiles) * rank / cluster);
      left = static_cast<long long>(tiles) * (rank + 1) / cluster - t;
      return;
    }
    // tiles of each sequence: a warp takes 32 sequences at a time
    const int lane = threadIdx.x & 31;
    auto seq_tiles = [&](int seq) -> long long {
      if (seq >= pr.B) return 0;
      const int o = OFFSETS ? pr.offset(seq) : 0;
      return static_cast<long long>(per_seq) * tiles_of(pr.keys(seq, o, CAUSAL), tile);
    };
    total = 0;
    for (int s = lane; s < pr.B; s += 32) total += seq_tiles(s);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) total += __shfl_xor_sync(0xffffffffu, total, x);
    end = total * blockIdx.x / gridDim.x;
    left = total * (blockIdx.x + 1LL) / gridDim.x - end;
    long long before = 0;  // tiles of the sequences before the chunk
    for (int s0 = 0; s0 < pr.B; s0 += 32) {
      const long long own = seq_tiles(s0 + lane);
      long long sum = own;
#pragma unroll
      for (int x = 1; x < 32; x <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, sum, x);
        if (lane >= x) sum += y;
      }
      const uint32_t behind = __ballot_sync(0xffffffffu, before + sum > end);
      if (behind) {
        const int l = __ffs(behind) - 1;
        const long long rest = end - before - __shfl_sync(0xffffffffu, sum - own, l);  // tile within the sequence
        enter(pr, s0 + l, tile);
        item = static_cast<int>(rest / tiles);
        t = static_cast<int>(rest % tiles);
        return;
      }
      before += __shfl_sync(0xffffffffu, sum, 31);
    }
  }
  // The next segment.  Notes in `entry` the item that this CTA starts and others finish.
  __device__ void next(const Problem& pr, int per_seq, int tile, Segment& s, JoinEntry& entry) {
    s.tiles = 0;
    if (left <= 0) return;
    s.b = b;
    s.item = item;
    s.keys = keys;
    s.off = off;
    s.tiles = tiles;
    s.t0 = t;
    s.nt = static_cast<int>(min(static_cast<long long>(tiles - t), left));
    left -= s.nt;
    end += s.nt;
    if (left > 0) {  // the item is done, the next one follows
      t = 0;
      if (++item == per_seq) {
        item = 0;
        enter(pr, b + 1, tile);
      }
    } else if (shares && s.t0 == 0 && s.nt < s.tiles) {
      // the CTAs up to the one that holds the item's last tile
      const long long last_tile = end + s.tiles - s.nt - 1;
      int last = static_cast<int>(((last_tile + 1) * gridDim.x - 1) / total);
      while (last + 1 < static_cast<int>(gridDim.x) && total * (last + 1) / gridDim.x <= last_tile) ++last;
      while (total * last / gridDim.x > last_tile) --last;
      entry.b = s.b;
      entry.item = s.item;
      entry.parts = last - static_cast<int>(blockIdx.x) + 1;
    }
  }
};

template <int D, int RG>
struct StepLayout {
  static constexpr int KEYS = D == 64 ? 128 : 64;  // keys of a tile: 32 KB of K and V
  static constexpr int WKEYS = KEYS / 4;           // keys of a warp
  static constexpr int STAGES = RG == 1 ? 3 : 5;
  static constexpr int CTAS = RG == 1 ? 2 : 1;  // of an SM
  static constexpr int SLABS = D / 64;
  static constexpr int TILE = KEYS * D * 2;
  static constexpr int ROWS = 16 * RG;
  static constexpr int WARPS = 4 * RG;  // that compute
  static constexpr int THREADS = 32 * (WARPS + 1);
  static constexpr int RING = STAGES * 2 * TILE;
  // the warps' results are joined JOIN columns at a time: [WARPS][16][JOIN] fp32
  static constexpr int JOIN = 32;
  static constexpr int JOIN_OFF = RING;
  static constexpr int ML_OFF = JOIN_OFF + WARPS * 16 * JOIN * 4;  // max and sum [WARPS][16] each
  static constexpr int SEGS = 4;                                 // segments' ring
  static constexpr int SEG_OFF = ML_OFF + 2 * WARPS * 16 * 4;
  static constexpr int BAR_OFF = SEG_OFF + SEGS * 32;  // full[], empty[], seg_full[], seg_empty[]
  static constexpr int MISC_OFF = BAR_OFF + (2 * STAGES + 2 * SEGS) * 8;
  static constexpr int RES_OFF = MISC_OFF + 16;  // LSE of the CTA's rows, for its cluster
  static_assert(ROWS * D * 4 <= RING, "the CTA's O for its cluster fits in the ring");
  // bias: bucket by position, then entries
  static constexpr int LUT_OFF = RES_OFF + ROWS * 4;
  // bytes of the bias part for `heads` heads
  static int bias_bytes(const Bias& bias, int heads) { return lut_size(bias) * 2 + bias.buckets * heads * 4; }
};

// Heads of the group that a tile of `rows` rows can meet.
__host__ __device__ inline int step_heads(int rows, int Sq, int G) {
  const int n = (rows - 1 + Sq - 1) / Sq + 1;
  return n < G ? n : G;
}

template <int D, int RG, bool ROWS8, bool CAUSAL, bool BIAS>
__global__ void __launch_bounds__(StepLayout<D, RG>::THREADS, StepLayout<D, RG>::CTAS)
    ffa_gen_step_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                        const __grid_constant__ Problem pr, const __grid_constant__ Bias bias, const View q,
                        const View o, float* __restrict__ LSE, float* __restrict__ part, float* __restrict__ part_lse,
                        JoinEntry* __restrict__ entries, int row_tiles, int cluster) {
  using L = StepLayout<D, RG>;
  constexpr int KS = D / 16;          // K-steps of Q K^T
  constexpr int NG = L::WKEYS / 16;   // groups of 16 keys of a warp
  constexpr int NX = ROWS8 ? 1 : 2;   // rows of a thread
  constexpr int ROWS = L::ROWS, JOIN = L::JOIN, STAGES = L::STAGES, NC = 32 * L::WARPS;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sbase = smem_u32(smem);
  const uint32_t bar0 = sbase + L::BAR_OFF;
  auto full = [&](int n) { return bar0 + 8 * (n % STAGES); };
  auto empty = [&](int n) { return bar0 + 8 * (STAGES + n % STAGES); };
  auto seg_full = [&](int n) { return bar0 + 8 * (2 * STAGES + n % L::SEGS); };
  auto seg_empty = [&](int n) { return bar0 + 8 * (2 * STAGES + L::SEGS + n % L::SEGS); };
  auto seg_slot = [&](int n) { return reinterpret_cast<Segment*>(smem + L::SEG_OFF + 32 * (n % L::SEGS)); };
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::MISC_OFF);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rows = pr.G * pr.Sq;
  const int per_seq = pr.Hkv * row_tiles;
  asm volatile("griddepcontrol.launch_dependents;");
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), L::WARPS);
    }
    for (int s = 0; s < L::SEGS; ++s) {
      mbar_init(seg_full(s), 1);
      mbar_init(seg_empty(s), L::WARPS);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  unsigned short* lut = reinterpret_cast<unsigned short*>(smem + L::LUT_OFF);
  float* entry = reinterpret_cast<float*>(smem + L::LUT_OFF + (BIAS ? lut_size(bias) * 2 : 0));
  __syncthreads();

  if (warp == L::WARPS) {
    // ------------------------------------------------------------------ producer
    Work<CAUSAL, CAUSAL || BIAS> work;
    work.start(pr, per_seq, L::KEYS, cluster);
    if (lane == 0) {
      const uint64_t once = policy_evict_first();
      JoinEntry shared{0, 0, 0, work.shares && work.left > 0 && work.t > 0};
      bool ok = true;
      int it = 0;
      for (int n = 0; ok; ++n) {
        Segment s;
        work.next(pr, per_seq, L::KEYS, s, shared);
        if (n >= L::SEGS &&
            !(ok = mbar_wait(seg_empty(n), (n / L::SEGS - 1) & 1, abort_flag, kErrGenStepProducer)))
          break;
        *seg_slot(n) = s;
        mbar_arrive(seg_full(n));
        if (s.tiles == 0) break;
        const int hk = s.item / row_tiles;
        for (int x = 0; x < s.nt; ++x, ++it) {
          if (!(ok = mbar_wait(empty(it), ((it / STAGES) & 1) ^ 1, abort_flag, kErrGenStepProducer))) break;
          const uint32_t dst = sbase + (it % STAGES) * 2 * L::TILE;
          mbar_arrive_expect_tx(full(it), 2 * L::TILE);
#pragma unroll
          for (int sl = 0; sl < L::SLABS; ++sl) {
            tma_load_4d(dst + sl * L::KEYS * 128, &tm_k, full(it), sl * 64, (s.t0 + x) * L::KEYS, hk, s.b, once);
            tma_load_4d(dst + L::TILE + sl * L::KEYS * 128, &tm_v, full(it), sl * 64, (s.t0 + x) * L::KEYS, hk, s.b,
                        once);
          }
        }
      }
      if (entries != nullptr) entries[blockIdx.x] = shared;
      if (*abort_flag)
        for (int x = max(0, it - STAGES); x < it; ++x) mbar_wait_drain(full(x), (x / STAGES) & 1);
    }
    __syncwarp();
    if (cluster > 1) {  // the compute warps' two barriers
      cluster_barrier();
      cluster_barrier();
    }
    return;
  }

  // -------------------------------------------------------------------- compute
  const int quad = lane >> 2, qlane = lane & 3;
  const int rg = warp >> 2;  // the warp's 16 rows of an item
  if (BIAS)
    for (int t = threadIdx.x; t <= bias.left + bias.right; t += NC)
      lut[t] = static_cast<unsigned short>(bias.bucket(t - bias.left));
  // cluster: this CTA's O (the ring's room, once it is read) and LSE, -inf without keys
  float* res = reinterpret_cast<float*>(smem);
  float* res_lse = reinterpret_cast<float*>(smem + L::RES_OFF);
  if (cluster > 1 && threadIdx.x < ROWS) res_lse[threadIdx.x] = -INFINITY;
  bool ok = true;
  int it = 0;  // tile of the CTA
  for (int n = 0;; ++n) {
    // a wait that ran out ends all warps here, at the next segment
    Segment sg{};
    ok = ok && mbar_wait(seg_full(n), (n / L::SEGS) & 1, abort_flag, kErrGenStepCompute);
    if (ok) sg = *seg_slot(n);
    __syncwarp();
    if (lane == 0) mbar_arrive(seg_empty(n));
    ok = whole_barrier_and(1, NC, ok);
    if (!ok || sg.tiles == 0) break;
    const int b = sg.b, n_keys = sg.keys;
    const int hk = sg.item / row_tiles, row0 = sg.item % row_tiles * ROWS;
    // the thread's rows: quad and quad + 8 of the warp's 16; Q as A fragments
    uint32_t qf[KS][4];
    int lim[NX], pos[NX], head[NX];
    const int g0 = row0 / pr.Sq;  // the item's first head of the group
#pragma unroll
    for (int x = 0; x < NX; ++x) {
      const int r = row0 + rg * 16 + x * 8 + quad;
      const bool valid = r < rows;
      const int g = valid ? r / pr.Sq : g0, t = valid ? r % pr.Sq : 0;
      pos[x] = t + sg.off;
      lim[x] = valid ? (CAUSAL ? min(n_keys - 1, t + sg.off) : n_keys - 1) : -1;
      head[x] = (g - g0) * bias.buckets;
      const __nv_bfloat16* src = static_cast<const __nv_bfloat16*>(q.p) + b * q.sb +
                                 static_cast<long long>(hk * pr.G + g) * q.sh + t * q.ss;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const int col = ks * 16 + y * 8 + qlane * 2;
          qf[ks][x + 2 * y] = (valid && col < pr.D) ? *reinterpret_cast<const uint32_t*>(src + col) : 0u;
        }
    }
    if constexpr (ROWS8) {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) qf[ks][1] = qf[ks][3] = 0u;
    }
    if (BIAS) {
      const int heads = step_heads(ROWS, pr.Sq, pr.G);
      for (int t = threadIdx.x; t < heads * bias.buckets; t += NC) {
        const int g = g0 + t / bias.buckets;
        entry[t] = g < pr.G ? bias.entry(t % bias.buckets, hk * pr.G + g, pr.Hq) : 0.f;
      }
      whole_barrier_and(1, NC, true);
    }

    float acc[D / 8][4] = {};
    float mx[NX], sum[NX];
#pragma unroll
    for (int x = 0; x < NX; ++x) {
      mx[x] = -INFINITY;
      sum[x] = 0.f;
    }
    const int w0 = (warp & 3) * L::WKEYS;  // the warp's first key of a tile
    for (int j = 0; j < sg.nt; ++j, ++it) {
      if (!(ok = mbar_wait(full(it), (it / STAGES) & 1, abort_flag, kErrGenStepCompute))) break;
      const uint32_t kt = sbase + (it % STAGES) * 2 * L::TILE, vt = kt + L::TILE;
      const int key0 = (sg.t0 + j) * L::KEYS + w0;
      if (key0 < n_keys) {
        float s[2 * NG][4] = {};
#pragma unroll
        for (int gk = 0; gk < NG; ++gk) {
          const int row = w0 + 16 * gk + (lane & 7) + ((lane >> 4) << 3);
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) {
            uint32_t kf[4];
            ldmatrix4(kf, kt + (ks >> 2) * (L::KEYS * 128) + row * 128 +
                              (((2 * (ks & 3) + ((lane >> 3) & 1)) ^ (row & 7)) << 4));
            mma_16816(s[2 * gk], qf[ks], kf[0], kf[1]);
            mma_16816(s[2 * gk + 1], qf[ks], kf[2], kf[3]);
          }
        }
        if (key0 + L::WKEYS > n_keys) {
          // V rows behind the last key must not reach the product (0 * NaN); this warp is the
          // only one that reads them, and the fence orders its writes before the next copy
          for (int r = n_keys - key0; r < L::WKEYS; ++r)
#pragma unroll
            for (int sl = 0; sl < L::SLABS; ++sl)
              if (lane < 8) st_shared_v4(vt + sl * L::KEYS * 128 + (w0 + r) * 128 + lane * 16, 0u, 0u, 0u, 0u);
          fence_proxy_async_smem();
          __syncwarp();
        }
        uint32_t pf[NG][4];
        if constexpr (ROWS8) {  // rows 8 to 15: P = 0
#pragma unroll
          for (int gk = 0; gk < NG; ++gk) pf[gk][1] = pf[gk][3] = 0u;
        }
#pragma unroll
        for (int x = 0; x < NX; ++x) {
          // the row's scores of this thread: keys key0 + 8 nt + 2 qlane + {0, 1}
          float m = -INFINITY;
#pragma unroll
          for (int nt = 0; nt < 2 * NG; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int key = key0 + 8 * nt + 2 * qlane + e;
              float& y = s[nt][2 * x + e];
              y *= pr.scale_log2;
              if (BIAS) {
                const int r = min(max(key - pos[x], -bias.left), bias.right);
                y += entry[head[x] + lut[r + bias.left]];
              }
              if (key > lim[x]) y = -INFINITY;
              m = fmaxf(m, y);
            }
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
          const float old = mx[x], m_new = fmaxf(old, m);
          const float m_safe = m_new == -INFINITY ? 0.f : m_new;
          if (__any_sync(0xffffffffu, m_new > old)) {
            const float alpha = fast_exp2(old - m_safe);
            mx[x] = m_new;
            sum[x] *= alpha;
#pragma unroll
            for (int d = 0; d < D / 8; ++d) {
              acc[d][2 * x] *= alpha;
              acc[d][2 * x + 1] *= alpha;
            }
          }
          // P goes to the product in bf16, as in the other kernels; its sum stays fp32
#pragma unroll
          for (int nt = 0; nt < 2 * NG; ++nt) {
            const float p0 = fast_exp2(s[nt][2 * x] - m_safe), p1 = fast_exp2(s[nt][2 * x + 1] - m_safe);
            sum[x] += p0 + p1;
            pf[nt >> 1][x + 2 * (nt & 1)] = pack_bf16x2(p0, p1);
          }
        }
#pragma unroll
        for (int gk = 0; gk < NG; ++gk) {
          const int row = w0 + 16 * gk + (lane & 15);
#pragma unroll
          for (int d = 0; d < D / 16; ++d) {
            uint32_t vf[4];
            ldmatrix4_trans(vf, vt + (d >> 2) * (L::KEYS * 128) + row * 128 +
                                    (((2 * (d & 3) + (lane >> 4)) ^ (row & 7)) << 4));
            mma_16816(acc[2 * d], pf[gk], vf[0], vf[1]);
            mma_16816(acc[2 * d + 1], pf[gk], vf[2], vf[3]);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty(it));
    }

    // ------------------------------------------------------------------ join the four warps
    float* so = reinterpret_cast<float*>(smem + L::JOIN_OFF);
    float* sm = reinterpret_cast<float*>(smem + L::ML_OFF);
    float* sl = sm + L::WARPS * 16;
#pragma unroll
    for (int x = 0; x < NX; ++x) {
      float t = sum[x];
      t += __shfl_xor_sync(0xffffffffu, t, 1);
      t += __shfl_xor_sync(0xffffffffu, t, 2);
      if (qlane == 0) {
        sm[warp * 16 + x * 8 + quad] = mx[x];
        sl[warp * 16 + x * 8 + quad] = t;
      }
    }
    // this thread's part of the output: 4 columns of one row in each round; the row's warps
    // are 4 rg .. 4 rg + 3
    const int r = threadIdx.x / (JOIN / 4), c4 = threadIdx.x % (JOIN / 4) * 4;
    const int r16 = (r & 15) + (r >> 4) * 64;
    const bool valid = row0 + r < rows;
    const int t = valid ? (row0 + r) % pr.Sq : 0;
    const long long h = hk * pr.G + (valid ? (row0 + r) / pr.Sq : 0);
    const long long prow = (2LL * blockIdx.x + (sg.t0 == 0 ? 1 : 0)) * ROWS + r;
    float f[4] = {}, m = -INFINITY, total = 0.f;
#pragma unroll
    for (int round = 0; round < D / JOIN; ++round) {
      if (round > 0) whole_barrier_and(1, NC, true);  // the last round has been read
#pragma unroll
      for (int d = 0; d < JOIN / 8; ++d)
#pragma unroll
        for (int x = 0; x < NX; ++x)
          *reinterpret_cast<float2*>(so + (warp * 16 + x * 8 + quad) * JOIN + 8 * d + 2 * qlane) =
              make_float2(acc[round * (JOIN / 8) + d][2 * x], acc[round * (JOIN / 8) + d][2 * x + 1]);
      ok = whole_barrier_and(1, NC, ok);
      if (!valid) continue;
      if (round == 0) {  // the warps' weights, normalised
#pragma unroll
        for (int w = 0; w < 4; ++w) m = fmaxf(m, sm[r16 + w * 16]);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          f[w] = m == -INFINITY ? 0.f : fast_exp2(sm[r16 + w * 16] - m);
          total = fmaf(f[w], sl[r16 + w * 16], total);
        }
        const float inv = total == 0.f ? 0.f : 1.f / total;
#pragma unroll
        for (int w = 0; w < 4; ++w) f[w] *= inv;
      }
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float4 y = *reinterpret_cast<const float4*>(so + (r16 + w * 16) * JOIN + c4);
        a.x = fmaf(f[w], y.x, a.x);
        a.y = fmaf(f[w], y.y, a.y);
        a.z = fmaf(f[w], y.z, a.z);
        a.w = fmaf(f[w], y.w, a.w);
      }
      const int col = round * JOIN + c4;
      if (ok && cluster > 1) {
        *reinterpret_cast<float4*>(res + r * D + col) = a;
      } else if (ok && col < pr.D) {
        if (sg.whole())
          *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(o.p) + b * o.sb + h * o.sh + t * o.ss + col) =
              make_uint2(pack_bf16x2(a.x, a.y), pack_bf16x2(a.z, a.w));
        else
          *reinterpret_cast<float4*>(part + prow * pr.D + col) = a;
      }
    }
    if (ok && valid && c4 == 0) {
      const float lse = total == 0.f ? -INFINITY : m + __log2f(total);
      if (cluster > 1)
        res_lse[r] = lse;
      else if (!sg.whole())
        part_lse[prow] = lse;
      else if (LSE != nullptr)
        LSE[(b * static_cast<long long>(pr.Hq) + h) * pr.Sq + t] = lse;
    }
  }

  if (cluster <= 1) return;
  // -------------------------------------------------------------------- join the cluster
  // Each CTA takes every `cluster`-th group of four columns from all the others' results,
  // weighed with 2^(LSE - max LSE).
  cluster_barrier();
  const int rank = blockIdx.x % cluster, at = blockIdx.x / cluster;
  const int b = at / per_seq, item = at % per_seq;
  const int hk = item / row_tiles, row0 = item % row_tiles * ROWS, n_rows = min(ROWS, rows - row0);
  const int groups = pr.D / 4;
  for (int x = rank * NC + threadIdx.x; x < n_rows * groups; x += cluster * NC) {
    const int r = x / groups, c = x % groups * 4;
    const uint32_t o_at = smem_u32(res + r * D + c), lse_at = smem_u32(res_lse + r);
    float m = -INFINITY, total = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int p = 0; p < cluster; ++p) {  // the loads of four CTAs do not wait for one another
      const float lse = ld_cluster(lse_at, p);
      const float4 y = ld_cluster4(o_at, p);
      const float m_new = fmaxf(m, lse), m_safe = m_new == -INFINITY ? 0.f : m_new;
      const float f = fast_exp2(m - m_safe), w = lse == -INFINITY ? 0.f : fast_exp2(lse - m_safe);
      m = m_new;
      total = fmaf(total, f, w);
      // a CTA without keys has left the ring's contents here
      a.x = fmaf(a.x, f, w == 0.f ? 0.f : w * y.x);
      a.y = fmaf(a.y, f, w == 0.f ? 0.f : w * y.y);
      a.z = fmaf(a.z, f, w == 0.f ? 0.f : w * y.z);
      a.w = fmaf(a.w, f, w == 0.f ? 0.f : w * y.w);
    }
    const float inv = total == 0.f ? 0.f : 1.f / total;
    const long long h = hk * pr.G + (row0 + r) / pr.Sq;
    const int t = (row0 + r) % pr.Sq;
    *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(o.p) + b * o.sb + h * o.sh + t * o.ss + c) =
        make_uint2(pack_bf16x2(a.x * inv, a.y * inv), pack_bf16x2(a.z * inv, a.w * inv));
    if (c == 0 && LSE != nullptr)
      LSE[(b * static_cast<long long>(pr.Hq) + h) * pr.Sq + t] = total == 0.f ? -INFINITY : m + __log2f(total);
  }
  cluster_barrier();  // nobody leaves while another reads its shared memory
}

// Join the parts of the items that cross CTAs: O = sum_p w_p O_p / sum_p w_p with
// w_p = 2^(LSE_p - max LSE).  blockIdx.x: the CTA in which an item starts; a warp takes one
// row, four columns a lane.  A part whose keys the row does not see (LSE = -inf) is not read,
// nor is the slot of a CTA that has none.
__global__ void __launch_bounds__(128)
    ffa_gen_step_join_kernel(const __grid_constant__ Problem pr, const float* part, const float* part_lse,
                             const JoinEntry* entries, const View o, float* __restrict__ LSE, int row_tiles, int rows) {
  const int lane = threadIdx.x & 31;
  const int row = blockIdx.y * 4 + (threadIdx.x >> 5);  // of the item
  asm volatile("griddepcontrol.wait;" ::: "memory");    // the parts are written
  // Row of part p: slot 1 of the first CTA, slot 0 of the next ones.  A lane takes the LSE of
  // one part of 32; its loads do not wait for one another (a slot that was not written is
  // inside the workspace, and its value is dropped), nor do those of the parts themselves.
  auto at = [&](int p) { return (2LL * (blockIdx.x + p) + (p == 0 ? 1 : 0)) * rows + row; };
  const int left = gridDim.x - blockIdx.x;  // parts there can be
  const JoinEntry e = entries[blockIdx.x];
  const int item_row = e.item % row_tiles * rows + row;
  float m = -INFINITY, total = 0.f;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  const int c = lane * 4;
  for (int p0 = 0; p0 < left; p0 += 32) {
    float lse = -INFINITY;
    if (p0 + lane < left) {
      const bool written = p0 + lane == 0 || entries[blockIdx.x + p0 + lane].slot0;
      const float y = part_lse[at(p0 + lane)];
      if (written && p0 + lane < e.parts) lse = y;
    }
    if (p0 >= e.parts || item_row >= pr.G * pr.Sq) break;  // the same for the whole warp
    const float m_old = m;
    float top = lse;
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
    m = fmaxf(m_old, top);
    const float m_safe = m == -INFINITY ? 0.f : m;
    const float f = exp2f(m_old - m_safe), w = exp2f(lse - m_safe);  // NaN where the part is
    float sum = w;
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
    total = fmaf(total, f, sum);
    a.x *= f;
    a.y *= f;
    a.z *= f;
    a.w *= f;
    const int n = min(32, e.parts - p0);
    for (int q0 = 0; q0 < n; q0 += 8) {
      float4 x[8];
      float wq[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        wq[q] = __shfl_sync(0xffffffffu, w, q0 + q);  // 0 for a part that there is not
        x[q] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (wq[q] > 0.f && c < pr.D) x[q] = *reinterpret_cast<const float4*>(part + at(p0 + q0 + q) * pr.D + c);
      }
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        a.x = fmaf(wq[q], x[q].x, a.x);
        a.y = fmaf(wq[q], x[q].y, a.y);
        a.z = fmaf(wq[q], x[q].z, a.z);
        a.w = fmaf(wq[q], x[q].w, a.w);
      }
    }
  }
  if (e.parts == 0 || item_row >= pr.G * pr.Sq) return;
  const int h = e.item / row_tiles * pr.G + item_row / pr.Sq, t = item_row % pr.Sq;
  const float inv = total == 0.f ? 0.f : 1.f / total;
  if (c < pr.D) {
    __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(o.p) + e.b * o.sb + h * o.sh + t * o.ss + c;
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16x2(a.x * inv, a.y * inv), pack_bf16x2(a.z * inv, a.w * inv));
  }
  if (lane == 0 && LSE != nullptr)
    LSE[(static_cast<long long>(e.b) * pr.Hq + h) * pr.Sq + t] = total == 0.f ? -INFINITY : m + __log2f(total);
}

}  // namespace gen
}  // namespace ffa
