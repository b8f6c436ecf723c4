// ffa_gen_common.cuh — what the kernels of general attention share.
//
// General attention is the family behind ffa_gen_* (include/ffa.h): queries and keys of
// different lengths, key heads shared by groups of query heads, a key length per sequence,
// queries that start at an offset, a causal mask and a bias learned by relative position:
//
//   S_ij = scale * q_i . k_j + bias[bucket(j - (i + off_b)), h]      P = softmax_j(S)
//   key j is visible to query i of sequence b iff  j < len_b  and (causal) j <= i + off_b
//
// Everything below works in base 2: scores and bias entries are multiplied by log2(e).
#pragma once
#include "ffa_common.cuh"

namespace ffa {
namespace gen {

constexpr int kMaxBuckets = 256;    // buckets of the position bias
constexpr int kMaxDistance = 1024;  // largest border between two buckets
constexpr int kOffsetLimit = 1 << 29;  // of lengths and offsets: sums of two stay in 32 bits

// Sizes and masks of a problem, as the kernels get them.
struct Problem {
  int B, Hq, Hkv, G, Sq, Sk, D;  // G = Hq / Hkv query heads for each key head; D = true head dim
  const int* key_lengths;        // [B] or null: all Sk keys
  const int* query_offsets;      // [B] or null: query_offset for all
  int query_offset;
  float scale_log2, scale;

  // Keys that some query of sequence b can see.  Keys behind them are read by nobody, so a
  // cache may hold anything there, NaN included.
  __device__ __forceinline__ int keys(int b, int off, bool causal) const {
    int n = key_lengths ? min(max(key_lengths[b], 0), Sk) : Sk;
    if (causal) n = min(n, max(off + Sq, 0));
    return n;
  }
  // The sequence whose CTAs come at place `pos`.  Where lengths differ, each 32 sequences
  // are taken longest first, so that the launch does not end on a long one (B4 H32 over
  // 8 heads, 2048 queries on 1000 to 4001 keys, D128: forward 325 us against 337 in their own
  // order, though each CTA of the backward starts later for it: 1020 us against 1009).  The
  // whole warp calls it.
  __device__ __forceinline__ int seq_at(int pos) const {
    if (key_lengths == nullptr || B == 1) return pos;
    const int lane = threadIdx.x & 31, first = pos & ~31;
    const int n = first + lane < B ? min(max(key_lengths[first + lane], 0), Sk) : -1;  // -1: behind them all
    const int count = min(B - first, 32);
    int rank = 0;  // sequences of the 32 that come before this lane's
#pragma unroll 4
    for (int x = 0; x < count; ++x) {
      const int y = __shfl_sync(0xffffffffu, n, x);
      rank += y > n || (y == n && x < lane);
    }
    return first + __ffs(__ballot_sync(0xffffffffu, rank == pos - first)) - 1;
  }
  __device__ __forceinline__ int offset(int b) const {
    return query_offsets ? min(max(query_offsets[b], -kOffsetLimit), kOffsetLimit) : query_offset;
  }
};

// The position bias.  Buckets are given by borders: on each side, bucket u holds the
// distances in [borders[u], borders[u + 1]), the last one all from borders[side - 1] on.
// A relative position r = key - query with r > 0 is in the second half of the buckets when
// `both`; else it counts as distance 0.
// From -left down and from right up the bucket, and so the bias, is constant.
struct Bias {
  const __nv_bfloat16* table;  // [buckets, Hq]
  int side, both, buckets;
  int left, right;
  short borders[kMaxBuckets];

  __device__ __forceinline__ int bucket(int r) const {
    const int d = both ? abs(r) : max(-r, 0);
    int lo = 0, hi = side;  // borders[lo] <= d < borders[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (borders[mid] <= d)
        lo = mid;
      else
        hi = mid;
    }
    return lo + ((both && r > 0) ? side : 0);
  }
  // Entry times log2(e).  Entries, +inf too, are clamped to +-2^14 (times log2 e): beyond that one key
  // outweighs any other by more than fp32 can hold, and the sum of a score and a bias of
  // the type's lowest value would lose the score.  -inf (the bucket is masked) and NaN stay.
  __device__ __forceinline__ float entry(int u, int h, int Hq) const {
    const float v = __bfloat162float(table[static_cast<long long>(u) * Hq + h]);
    const float lim = 16384.f;
    const float c = v > lim ? lim : ((v < -lim && v > -INFINITY) ? -lim : v);
    return c * static_cast<float>(kLog2e);
  }
};

// The bias of one head by relative position: entry r + left + kPad for r in [-left - kPad,
// right + kPad].  A tile of at most 128 x 128 scores that meets a position in (-left, right)
// lies inside; the others have one bias for all their scores (the first or the last entry).
// ffa_gen_table_kernel writes the tables of all heads once a call, and a CTA brings its
// head's into shared memory with one bulk copy.  Neighbouring lanes read neighbouring
// positions: no bank conflicts.
constexpr int kPad = 256;
constexpr int kTableMax = 2 * kMaxDistance + 2 * kPad + 4;
// entries of a table, rounded up to whole 16-byte units
__host__ __device__ __forceinline__ int table_size(const Bias& bias) {
  return (bias.left + bias.right + 2 * kPad + 1 + 3) / 4 * 4;
}
__device__ __forceinline__ int table_last(const Bias& bias) { return bias.left + bias.right + 2 * kPad; }
// Bucket by position, entry r + left, behind the tables (16-bit, whole 16-byte units).
__host__ __device__ __forceinline__ int lut_size(const Bias& bias) { return (bias.left + bias.right + 1 + 7) / 8 * 8; }

__global__ void __launch_bounds__(256)
    ffa_gen_table_kernel(const __grid_constant__ Bias bias, float* __restrict__ tables,
                         unsigned short* __restrict__ lut, int Hq) {
  asm volatile("griddepcontrol.launch_dependents;");
  const int size = table_size(bias), t = blockIdx.x * 256 + threadIdx.x;
  if (t >= size) return;
  const int r = t - bias.left - kPad, u = bias.bucket(r);
  for (int h = blockIdx.y; h < Hq; h += gridDim.y) tables[static_cast<long long>(h) * size + t] = bias.entry(u, h, Hq);
  if (lut != nullptr && blockIdx.y == 0 && r >= -bias.left && r + bias.left < lut_size(bias))
    lut[r + bias.left] = static_cast<unsigned short>(u);
}

// A device tensor [B, H, S, D] with contiguous D, as the C ABI describes it.
struct View {
  void* p;
  long long sb, sh, ss;
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* m, uint32_t bar, int c0, int c1, int c2,
                                            int c3, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%3, %4, %5, %6}], [%2], %7;" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "l"(policy)
      : "memory");
}
__device__ __forceinline__ void tma_store_4d(const CUtensorMap* m, uint32_t src, int c0, int c1, int c2, int c3) {
  asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%2, %3, %4, %5}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(m)),
               "r"(src), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
               : "memory");
}
// Untiled copy of `bytes` (a multiple of 16; both addresses 16-byte aligned).
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(bar)
               : "memory");
}

// 32 lanes x 16 columns of 32-bit (tmem_ld32 with half the columns).
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}

// named_barrier_and, for warps whose lanes may have come apart (loops and branches by lane in
// front of it): the hardware barrier is an aligned one, which wants each warp whole.
__device__ __forceinline__ bool whole_barrier_and(int id, int n, bool pred) {
  __syncwarp();
  return named_barrier_and(id, n, pred);
}

// Zero the rows from `row` on of a tile of ROWS rows in shared memory (64-column slabs, 128
// bytes a row; the swizzle moves nothing between rows).  The whole warp calls it,
// before it issues MMAs that read the tile.  A probability of 0 does not undo a NaN in the
// value it is multiplied with, so rows behind the last key must not reach an MMA.
template <int ROWS = 128>
__device__ __forceinline__ void zero_tail(uint32_t tile, int slabs, int row, int lane) {
  for (int sl = 0; sl < slabs; ++sl)
    for (int o = row * 128 + lane * 16; o < ROWS * 128; o += 512) st_shared_v4(tile + sl * ROWS * 128 + o, 0u, 0u, 0u, 0u);
  fence_proxy_async_smem();
  __syncwarp();
}

// Write a warp's 32 rows x 32 fp32 accumulator columns (lane = row), times `mul`, to columns
// [c0, c0 + 32) of the fp32 rows dst, dst + D, ... of which `rows` exist.  D is a multiple
// of 8.  The values change places in `scratch` (4 KB of shared memory of this warp), so that
// eight lanes write 128 bytes of a row: lanes that wrote a row each would leave 32 pieces of
// 16 bytes for every store.
__device__ __forceinline__ void write_rows32(uint32_t scratch, float* dst, int c0, int D, int rows,
                                             const uint32_t (&r)[32], float mul, int lane) {
  __syncwarp();  // the last call's values have been read
#pragma unroll
  for (int e = 0; e < 8; ++e)
    st_shared_v4(scratch + lane * 128 + ((e ^ (lane & 7)) << 4), __float_as_uint(__uint_as_float(r[4 * e]) * mul),
                 __float_as_uint(__uint_as_float(r[4 * e + 1]) * mul),
                 __float_as_uint(__uint_as_float(r[4 * e + 2]) * mul),
                 __float_as_uint(__uint_as_float(r[4 * e + 3]) * mul));
  __syncwarp();
  const int col = c0 + 4 * (lane & 7);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int row = 4 * e + (lane >> 3);
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(scratch + row * 128 + (((lane & 7) ^ (row & 7)) << 4))
                 : "memory");
    if (row < rows && col < D) *reinterpret_cast<float4*>(dst + static_cast<long long>(row) * D + col) = v;
  }
}

// 4-D tensor map over a [B, H, S, D] bf16 tensor: boxes of 64 columns x `rows` rows, 128-byte
// swizzle.  Columns from D on and rows from S on read as zero and are not written, so head
// dims below the kernel's 64 or 128 need no padding in memory.
int make_map(CUtensorMap* map, const View& t, int B, int H, int S, int D, int rows = 128);

}  // namespace gen
}  // namespace ffa
