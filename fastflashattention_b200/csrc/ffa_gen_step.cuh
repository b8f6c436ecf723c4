// ffa_gen_step.cuh — general attention (ffa_gen_common.cuh) of a few query rows: a step of
// one or a few tokens over a cache or an encoder's states.
//
// The work is one pass over K and V, so the kernel is bound by HBM.  The G * Sq query rows
// that share a key head (row r = g * Sq + t) form tiles of 16 MT rows, the M of mma.sync
// m16n8k16; the tensor cores' rate does not matter here, and a 128-row tcgen05 tile would
// be empty.  A CTA of four warps takes one row tile and one split of the keys:
//   * stages of 64 keys (K and V) come through a cp.async ring, 16 bytes a copy, zero-filled
//     behind the last key (which also keeps what a cache holds there out of the products);
//   * each warp takes 16 keys of a stage and keeps its own running max, sum and O
//     (registers); the four are joined in shared memory at the end;
//   * splits write their normalised O (fp32) and LSE; ffa_gen_join_kernel weighs them.
#pragma once
#include "ffa_gen_common.cuh"

namespace ffa {
namespace gen {

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
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

template <int D, int MT>
struct StepLayout {
  static constexpr int KEYS = 64;  // keys of a stage, 16 for each warp
  static constexpr int STAGES = D == 64 ? 4 : 3;
  static constexpr int TILE = KEYS * D * 2;
  static constexpr int ROWS = 16 * MT;
  static constexpr int RING = STAGES * 2 * TILE;
  // the join of the four warps reuses the ring: O [4][ROWS][D] fp32
  static_assert(4 * ROWS * D * 4 <= RING, "the warps' results fit in the ring");
  static constexpr int ML_OFF = RING;                       // max and sum [4][ROWS] each
  static constexpr int LUT_OFF = ML_OFF + 2 * 4 * ROWS * 4; // bias: bucket by position, then entries
  // bytes of the bias part for `heads` heads
  static int bias_bytes(const Bias& bias, int heads) {
    return (bias.left + bias.right + 2) / 2 * 4 + bias.buckets * heads * 4;
  }
};

// Heads of the group that a tile of `rows` rows can meet.
__host__ __device__ inline int step_heads(int rows, int Sq, int G) {
  const int n = (rows - 1 + Sq - 1) / Sq + 1;
  return n < G ? n : G;
}

template <int D, int MT, bool CAUSAL, bool BIAS>
__global__ void __launch_bounds__(128)
    ffa_gen_step_kernel(const __grid_constant__ Problem pr, const __grid_constant__ Bias bias, const View q,
                        const View k, const View v, const View o, float* __restrict__ LSE, float* __restrict__ part,
                        float* __restrict__ part_lse, int n_split, int row_tiles) {
  using L = StepLayout<D, MT>;
  constexpr int KS = D / 16;       // K-steps of Q K^T
  constexpr int CHUNKS = D / 8;    // 16-byte chunks of a row
  constexpr int ROWS = L::ROWS;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sbase = smem_u32(smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int quad = lane >> 2, qlane = lane & 3;

  const int split = blockIdx.x % n_split;
  const int row0 = (blockIdx.x / n_split) % row_tiles * ROWS;
  const int hk = blockIdx.x / (n_split * row_tiles) % pr.Hkv;
  const int b = blockIdx.x / (n_split * row_tiles) / pr.Hkv;
  const int rows = pr.G * pr.Sq;
  const int off = (CAUSAL || BIAS) ? pr.offset(b) : 0;
  const int n_keys = pr.keys(b, off, CAUSAL);
  const int stages_all = (n_keys + L::KEYS - 1) / L::KEYS;
  const int per_split = (stages_all + n_split - 1) / n_split;
  const int s0 = split * per_split;
  const int ns = max(0, min(stages_all - s0, per_split));

  // ------------------------------------------------------------------ K/V ring
  const __nv_bfloat16* kb = static_cast<const __nv_bfloat16*>(k.p) + b * k.sb + hk * k.sh;
  const __nv_bfloat16* vb = static_cast<const __nv_bfloat16*>(v.p) + b * v.sb + hk * v.sh;
  auto load = [&](int n) {  // stage n of this split; a commit group even when there is none
    if (n < ns) {
      const uint32_t dst = sbase + (n % L::STAGES) * 2 * L::TILE;
      const int key0 = (s0 + n) * L::KEYS;
#pragma unroll
      for (int e = 0; e < L::KEYS * CHUNKS / 128; ++e) {
        const int c = threadIdx.x + e * 128;
        const int row = c / CHUNKS, ch = c % CHUNKS;
        const bool ok = key0 + row < n_keys && ch * 8 < pr.D;
        const uint32_t at = dst + row * (D * 2) + ((ch ^ (row & 7)) << 4);
        const long long key = ok ? key0 + row : 0, col = ok ? ch * 8 : 0;
        cp_async16(at, kb + key * k.ss + col, ok);
        cp_async16(at + L::TILE, vb + key * v.ss + col, ok);
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int n = 0; n < L::STAGES - 1; ++n) load(n);

  // ------------------------------------------------------------------ Q, and each row's limits
  // the thread's rows: quad and quad + 8 of each 16-row tile
  uint32_t qf[MT][KS][4];
  int lim[MT][2], pos[MT][2], head[MT][2];
  const int g0 = row0 / pr.Sq;  // the tile's first head of the group
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int r = row0 + mt * 16 + x * 8 + quad;
      const bool ok = r < rows;
      const int g = ok ? r / pr.Sq : g0, t = ok ? r % pr.Sq : 0;
      pos[mt][x] = t + off;
      lim[mt][x] = ok ? (CAUSAL ? min(n_keys - 1, t + off) : n_keys - 1) : -1;
      head[mt][x] = g - g0;
      const __nv_bfloat16* src = static_cast<const __nv_bfloat16*>(q.p) + b * q.sb +
                                 static_cast<long long>(hk * pr.G + g) * q.sh + t * q.ss;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const int col = ks * 16 + y * 8 + qlane * 2;
          qf[mt][ks][x + 2 * y] = (ok && col < pr.D) ? *reinterpret_cast<const uint32_t*>(src + col) : 0u;
        }
    }
  // bias: bucket of each position in [-left, right], entries [head][bucket]
  const unsigned short* lut = reinterpret_cast<const unsigned short*>(smem + L::LUT_OFF);
  const float* entries = nullptr;
  if (BIAS) {
    unsigned short* w = reinterpret_cast<unsigned short*>(smem + L::LUT_OFF);
    float* ew = reinterpret_cast<float*>(smem + L::LUT_OFF + (bias.left + bias.right + 2) / 2 * 4);
    entries = ew;
    const int heads = step_heads(ROWS, pr.Sq, pr.G);
    for (int t = threadIdx.x; t <= bias.left + bias.right; t += 128)
      w[t] = static_cast<unsigned short>(bias.bucket(t - bias.left));
    for (int t = threadIdx.x; t < heads * bias.buckets; t += 128) {
      const int g = g0 + t / bias.buckets;
      ew[t] = g < pr.G ? bias.entry(t % bias.buckets, hk * pr.G + g, pr.Hq) : 0.f;
    }
    __syncthreads();
  }

  // ------------------------------------------------------------------ the keys
  float acc[MT][D / 8][4];
  float mx[MT][2], sum[MT][2];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      mx[mt][x] = -INFINITY;
      sum[mt][x] = 0.f;
    }
#pragma unroll
    for (int n = 0; n < D / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[mt][n][e] = 0.f;
  }
  const int w16 = warp * 16;
  for (int n = 0; n < ns; ++n) {
    cp_async_wait<L::STAGES - 2>();
    __syncthreads();  // stage n has landed; everyone is done with stage n - 1
    load(n + L::STAGES - 1);
    const uint32_t kt = sbase + (n % L::STAGES) * 2 * L::TILE, vt = kt + L::TILE;
    const int key0 = (s0 + n) * L::KEYS + w16;
    if (key0 >= n_keys) continue;  // the warp's keys are all behind the last one
    float s[MT][2][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int nt = 0; nt < 2; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[mt][nt][e] = 0.f;
    {
      const int row = w16 + (lane & 7) + ((lane >> 4) << 3);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        uint32_t kf[4];
        ldmatrix4(kf, kt + row * (D * 2) + (((2 * ks + ((lane >> 3) & 1)) ^ (row & 7)) << 4));
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          mma_16816(s[mt][0], qf[mt][ks], kf[0], kf[1]);
          mma_16816(s[mt][1], qf[mt][ks], kf[2], kf[3]);
        }
      }
    }
    uint32_t pf[MT][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        // the row's 4 scores of this thread: s[mt][nt][2x], s[mt][nt][2x + 1], keys
        // key0 + 8 nt + 2 qlane + {0, 1}
        float m = -INFINITY;
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int key = key0 + 8 * nt + 2 * qlane + e;
            float& y = s[mt][nt][2 * x + e];
            y *= pr.scale_log2;
            if (BIAS) {
              const int r = min(max(key - pos[mt][x], -bias.left), bias.right);
              y += entries[head[mt][x] * bias.buckets + lut[r + bias.left]];
            }
            if (key > lim[mt][x]) y = -INFINITY;
            m = fmaxf(m, y);
          }
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
        const float m_new = fmaxf(mx[mt][x], m);
        const float m_safe = m_new == -INFINITY ? 0.f : m_new;
        const float alpha = fast_exp2(mx[mt][x] - m_safe);
        mx[mt][x] = m_new;
        float t = 0.f;
        float p[2][2];
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            p[nt][e] = fast_exp2(s[mt][nt][2 * x + e] - m_safe);
            t += p[nt][e];
          }
        sum[mt][x] = fmaf(sum[mt][x], alpha, t);
        // P goes to the product in bf16, as in the other kernels; its sum stays fp32
        pf[mt][x] = pack_bf16x2(p[0][0], p[0][1]);
        pf[mt][2 + x] = pack_bf16x2(p[1][0], p[1][1]);
#pragma unroll
        for (int d = 0; d < D / 8; ++d) {
          acc[mt][d][2 * x] *= alpha;
          acc[mt][d][2 * x + 1] *= alpha;
        }
      }
    {
      const int row = w16 + (lane & 15);
#pragma unroll
      for (int d = 0; d < D / 16; ++d) {
        uint32_t vf[4];
        ldmatrix4_trans(vf, vt + row * (D * 2) + (((2 * d + (lane >> 4)) ^ (row & 7)) << 4));
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          mma_16816(acc[mt][2 * d], pf[mt], vf[0], vf[1]);
          mma_16816(acc[mt][2 * d + 1], pf[mt], vf[2], vf[3]);
        }
      }
    }
  }
  cp_async_wait<0>();
  __syncthreads();  // the ring is free

  // ------------------------------------------------------------------ join the four warps
  float* so = reinterpret_cast<float*>(smem);
  float* sm = reinterpret_cast<float*>(smem + L::ML_OFF);
  float* sl = sm + 4 * ROWS;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int r = mt * 16 + x * 8 + quad;
      float t = sum[mt][x];
      t += __shfl_xor_sync(0xffffffffu, t, 1);
      t += __shfl_xor_sync(0xffffffffu, t, 2);
      if (qlane == 0) {
        sm[warp * ROWS + r] = mx[mt][x];
        sl[warp * ROWS + r] = t;
      }
      float* dst = so + (warp * ROWS + r) * D + 2 * qlane;
#pragma unroll
      for (int d = 0; d < D / 8; ++d)
        *reinterpret_cast<float2*>(dst + 8 * d) = make_float2(acc[mt][d][2 * x], acc[mt][d][2 * x + 1]);
    }
  __syncthreads();
  for (int c = threadIdx.x; c < ROWS * CHUNKS; c += 128) {
    const int r = c / CHUNKS, col = c % CHUNKS * 8;
    if (row0 + r >= rows) break;
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; ++w) m = fmaxf(m, sm[w * ROWS + r]);
    float total = 0.f, out[8] = {};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = m == -INFINITY ? 0.f : fast_exp2(sm[w * ROWS + r] - m);
      total = fmaf(f, sl[w * ROWS + r], total);
      const float* src = so + (w * ROWS + r) * D + col;
#pragma unroll
      for (int e = 0; e < 8; ++e) out[e] = fmaf(f, src[e], out[e]);
    }
    const float inv = total == 0.f ? 0.f : 1.f / total;
    const int g = (row0 + r) / pr.Sq, t = (row0 + r) % pr.Sq;
    const long long h = hk * pr.G + g;
    const long long ridx = (b * static_cast<long long>(pr.Hq) + h) * pr.Sq + t;
    const float lse = total == 0.f ? -INFINITY : m + __log2f(total);
#pragma unroll
    for (int e = 0; e < 8; ++e) out[e] *= inv;
    if (n_split > 1) {
      const long long idx = static_cast<long long>(split) * pr.B * pr.Hq * pr.Sq + ridx;
      if (col == 0) part_lse[idx] = lse;
      if (col < pr.D) {
        float4* dst = reinterpret_cast<float4*>(part + idx * pr.D + col);
        dst[0] = make_float4(out[0], out[1], out[2], out[3]);
        dst[1] = make_float4(out[4], out[5], out[6], out[7]);
      }
    } else {
      if (col == 0 && LSE != nullptr) LSE[ridx] = lse;
      if (col < pr.D) {
        __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(o.p) + b * o.sb + h * o.sh + t * o.ss + col;
        *reinterpret_cast<uint4*>(dst) = make_uint4(pack_bf16x2(out[0], out[1]), pack_bf16x2(out[2], out[3]),
                                                    pack_bf16x2(out[4], out[5]), pack_bf16x2(out[6], out[7]));
      }
    }
  }
}

// Join the splits of a row: O = sum_s w_s O_s / sum_s w_s, w_s = 2^(LSE_s - max LSE).  One
// warp a row, four columns a lane; a split without keys (LSE = -inf) is not read.
__global__ void __launch_bounds__(128)
    ffa_gen_join_kernel(const float* __restrict__ part, const float* __restrict__ part_lse, const View o,
                        float* __restrict__ LSE, int n_split, int B, int H, int Sq, int D) {
  const int lane = threadIdx.x & 31;
  const long long rows = static_cast<long long>(B) * H * Sq;
  const long long r = static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (r >= rows) return;
  float m = -INFINITY;
  for (int s = lane; s < n_split; s += 32) m = fmaxf(m, part_lse[s * rows + r]);
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
  float total = 0.f;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  const int c = lane * 4;
  if (m > -INFINITY) {
#pragma unroll 4
    for (int s = 0; s < n_split; ++s) {
      const float lse = part_lse[s * rows + r];
      if (lse == -INFINITY) continue;
      const float w = exp2f(lse - m);
      total += w;
      if (c < D) {
        const float4 x = *reinterpret_cast<const float4*>(part + (s * rows + r) * D + c);
        a.x = fmaf(w, x.x, a.x);
        a.y = fmaf(w, x.y, a.y);
        a.z = fmaf(w, x.z, a.z);
        a.w = fmaf(w, x.w, a.w);
      }
    }
  }
  const float inv = total == 0.f ? 0.f : 1.f / total;
  if (c < D) {
    const long long bh = r / Sq, t = r % Sq;
    __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(o.p) + bh / H * o.sb + bh % H * o.sh + t * o.ss + c;
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16x2(a.x * inv, a.y * inv), pack_bf16x2(a.z * inv, a.w * inv));
  }
  if (lane == 0 && LSE != nullptr) LSE[r] = total == 0.f ? -INFINITY : m + __log2f(total);
}

}  // namespace gen
}  // namespace ffa
