// ffa_gen_api.cuh — host side of general attention: argument checks, how a problem is split,
// tensor maps, launches and the ffa_gen_* entry points (include/ffa.h).
#pragma once
#include <climits>
#include <cmath>

#include "ffa_gen_bwd.cuh"
#include "ffa_gen_fwd.cuh"
#include "ffa_gen_step.cuh"

namespace ffa {

int make_map4(CUtensorMap* map, const void* base, const cuuint64_t (&dims)[4], const cuuint64_t (&strides)[3], int rows);

namespace gen {

constexpr int kSMs = 148;

inline long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

int make_map(CUtensorMap* map, const View& t, int B, int H, int S, int D, int rows) {
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(S), static_cast<cuuint64_t>(H),
                              static_cast<cuuint64_t>(B)};
  const cuuint64_t strides[3] = {static_cast<cuuint64_t>(t.ss) * 2, static_cast<cuuint64_t>(t.sh) * 2,
                                 static_cast<cuuint64_t>(t.sb) * 2};
  return make_map4(map, t.p, dims, strides, rows);
}

// ------------------------------------------------------------------------------------
// arguments
// ------------------------------------------------------------------------------------
inline int check_problem(const ffa_gen_problem* p) {
  if (!p) return set_error(FFA_ERR_INVALID, "null problem");
  if (p->batch < 0 || p->q_heads < 0 || p->kv_heads < 0 || p->q_len < 0 || p->k_len < 0)
    return set_error(FFA_ERR_INVALID, "sizes must be non-negative");
  if (p->head_dim < 8 || p->head_dim > 128 || p->head_dim % 8 != 0)
    return set_error(FFA_ERR_UNSUPPORTED, "head_dim must be a multiple of 8 in [8, 128]");
  if (p->kv_heads == 0 ? p->q_heads != 0 : p->q_heads % p->kv_heads != 0)
    return set_error(FFA_ERR_INVALID, "q_heads must be a multiple of kv_heads");
  if (p->q_len >= kOffsetLimit || p->k_len >= kOffsetLimit)
    return set_error(FFA_ERR_UNSUPPORTED, "lengths must be below 2^29");
  if (p->query_offset > kOffsetLimit || p->query_offset < -kOffsetLimit)
    return set_error(FFA_ERR_UNSUPPORTED, "query_offset must be within +-2^29");
  if (!std::isfinite(p->scale)) return set_error(FFA_ERR_INVALID, "scale must be finite");
  if (p->causal && !p->bias && p->q_heads > 0)  // (the bias of no heads has no data)
    return set_error(FFA_ERR_UNSUPPORTED, "general attention is causal only with a position bias (see ffa_fwd)");
  if (p->bias) {
    if (p->buckets < 1 || p->buckets > kMaxBuckets || (p->both && p->buckets % 2 != 0) || !p->borders)
      return set_error(FFA_ERR_UNSUPPORTED, "buckets must be in [1, 256], and even for both directions");
    const int side = p->both ? p->buckets / 2 : p->buckets;
    if (p->borders[0] != 0) return set_error(FFA_ERR_INVALID, "the first bucket border must be 0");
    for (int u = 1; u < side; ++u)
      if (p->borders[u] < p->borders[u - 1] || p->borders[u] > kMaxDistance)
        return set_error(FFA_ERR_UNSUPPORTED, "bucket borders must ascend, up to 1024");
  }
  // one CTA for each 16 rows of a head, at the most
  const long long heads = static_cast<long long>(p->batch) * p->q_heads;
  const long long len = p->q_len > p->k_len ? p->q_len : p->k_len;
  if (heads > INT_MAX || heads * (len > 0 ? len : 1) > 16LL * INT_MAX)
    return set_error(FFA_ERR_UNSUPPORTED, "the problem exceeds the grid limit of 2^31-1 CTAs");
  return FFA_OK;
}

inline int check_tensor(const ffa_gen_tensor* t, bool needed) {
  if (!t || (needed && !t->data)) return set_error(FFA_ERR_INVALID, "null tensor pointer");
  if (!needed) return FFA_OK;
  if (reinterpret_cast<uintptr_t>(t->data) & 15u)
    return set_error(FFA_ERR_INVALID, "tensor pointers must be 16-byte aligned");
  for (const long long s : {t->stride_b, t->stride_h, t->stride_s})
    if (s <= 0 || s % 8 != 0 || s >= (1LL << 39))
      return set_error(FFA_ERR_INVALID, "strides must be positive multiples of 8 elements below 2^39");
  return FFA_OK;
}

inline View view(const ffa_gen_tensor* t) { return {t->data, t->stride_b, t->stride_h, t->stride_s}; }

inline Problem device_problem(const ffa_gen_problem* p) {
  Problem d;
  d.B = p->batch;
  d.Hq = p->q_heads;
  d.Hkv = p->kv_heads;
  d.G = p->kv_heads ? p->q_heads / p->kv_heads : 1;
  d.Sq = p->q_len;
  d.Sk = p->k_len;
  d.D = p->head_dim;
  d.key_lengths = p->key_lengths;
  d.query_offsets = p->query_offsets;
  d.query_offset = p->query_offset;
  d.scale_log2 = static_cast<float>(p->scale * kLog2e);
  d.scale = static_cast<float>(p->scale);
  return d;
}

inline Bias device_bias(const ffa_gen_problem* p) {
  Bias b{};
  if (!p->bias) return b;
  b.table = static_cast<const __nv_bfloat16*>(p->bias);
  b.buckets = p->buckets;
  b.both = p->both ? 1 : 0;
  b.side = b.both ? p->buckets / 2 : p->buckets;
  for (int u = 0; u < b.side; ++u) b.borders[u] = static_cast<short>(p->borders[u]);
  const int last = b.borders[b.side - 1];
  b.left = last;
  b.right = b.both ? (last > 1 ? last : 1) : 0;
  return b;
}

// ------------------------------------------------------------------------------------
// how a problem is split
// ------------------------------------------------------------------------------------
// The backward: parts that the streamed dimension (`units` tiles) is cut into when `ctas`
// CTAs leave SMs idle: as many as one wave of `slots` CTAs holds, each with at least `least`
// tiles.
inline int split_of(long long ctas, long long slots, long long units, long long least) {
  if (ctas <= 0 || ctas * 2 > slots) return 1;
  const long long n = slots / ctas, most = units / least;
  return static_cast<int>(n < most ? n : (most > 1 ? most : 1));
}

// The forward: steps of a split when `ctas` CTAs, `slots` at a time, each walk up to `units`
// steps, `mean` on average, of `step_us` microseconds.  The estimate of a split's size, in
// steps: where all CTAs are alike, waves times (a split's steps + `fixed`, a CTA's start and
// end); else (a causal mask, lengths that differ; the longest come first) one longest split
// where a single wave holds them all, or the mean load and a part of a split at the end.
// Joining costs `join`, and for each split the traffic of `rows` fp32 rows of O.  The
// smallest estimate wins.  (B200, B2 H32 over 8 heads, 500 tokens on 8192 keys, D128: 142 us
// in one split, 132 in two, 124 in three, 146 in four.)
inline long long split_steps(long long ctas, long long slots, long long units, double mean, long long rows, int D,
                             double step_us, double fixed, double join) {
  const double traffic = static_cast<double>(rows) * D * 8 / 6.5e6 / step_us;
  long long best = units > 0 ? units : 1;
  double least = 1e300;
  for (long long n = 1; n <= 64 && n <= (units + 1) / 2; ++n) {
    const long long per = ceil_div(units, n);
    if (ceil_div(units, per) != n) continue;
    const double load = static_cast<double>(ctas) / slots;
    double cost;
    if (mean > 0.99 * units) {
      cost = std::ceil(load * n) * (per + fixed);
    } else {
      const double splits = std::max(1.0, mean / per + (n > 1 ? 0.5 : 0.0));  // of a CTA's steps, on average
      cost = load * splits <= 1.0 ? per + fixed
                                  : std::max(per + fixed, load * (mean + splits * fixed)) +
                                        (n > 1 ? 0.5 : 0.15) * (per + fixed);
    }
    if (n > 1) cost += join + n * traffic;
    if (cost < least) {
      least = cost;
      best = per;
    }
  }
  return best;
}

struct FwdPlan {
  bool step;  // ffa_gen_step_kernel (few query rows for each key head), else ffa_gen_fwd_kernel
  // step: groups of 16 rows of an item, items of a key head, CTAs, and of those for each item
  // (0: equal shares of all keys)
  int rg, row_tiles, grid, cluster;
  // else: splits of the keys and their steps
  int n_split, per_split, keys_per_split;
  // workspace, offsets in floats (tables) and of the parts: O, LSE, entries (bytes)
  long long table_floats, part_off, lse_off, entry_off, bytes;
  bool join;
};

inline FwdPlan fwd_plan(const ffa_gen_problem* p, const Bias& bias, bool exact) {
  FwdPlan f{};
  const long long heads = static_cast<long long>(p->batch) * p->q_heads;
  const long long group_rows = p->kv_heads ? static_cast<long long>(p->q_heads / p->kv_heads) * p->q_len : 0;
  const bool small_d = p->head_dim <= 64;
  f.step = group_rows <= 64 && !exact;  // the step kernel has no form with remainders
  if (heads * p->q_len == 0) return f;
  if (f.step) {
    f.rg = group_rows <= 16 ? 1 : 2;
    f.row_tiles = static_cast<int>(ceil_div(group_rows, 16 * f.rg));
    const long long items = static_cast<long long>(p->batch) * p->kv_heads * f.row_tiles;
    const long long units = std::max<long long>(1, ceil_div(p->k_len, small_d ? 128 : 64));  // tiles of an item, at most
    const long long slots = kSMs * (f.rg == 1 ? 2 : 1);
    // Clusters of up to 16 CTAs for each item, as many as fit at once, at least two tiles for
    // each CTA (many items: one CTA each), or equal shares of all items' tiles and a join.
    // The estimate of time decides: all tiles (32 KB) through HBM, or a CTA's tiles at 0.7 us
    // (0.85 with 32 rows), and 12 us more for shares and their join.  Shares win where few
    // items leave SMs without work, or sequences of different lengths do (B2 H32 over 4 heads,
    // 3 tokens on 50001 keys, D128: 58 us against 89; B2 H32 over 4 heads, 1 token on 50001
    // keys: 54 against 46; B64 H16, 1 token on 375 to 1500 keys, D64: 60 against 53).  With
    // very many sequences shares would look through them for too long.
    // The lengths are on the device, so with key_lengths the mean load is a guess, two thirds of
    // the longest.  Where all are full it costs nothing here (B64 H16, 1 token on 1500 keys, D64:
    // 65 us with and without the tensor; B8 H32 over 8, 1 on 8192, D128: 44), where all are a
    // tenth of Sk little (24 against 21 for keys of that shape; 12 against 12).
    // A cluster lies inside one GPC, whose SMs it may not fill: `fit` holds how many clusters
    // of 1, 2, .. 16 CTAs run at once (a B200 with 148 SMs says 296, 148, 71, 33, 14 with two
    // CTAs to an SM and 148, 74, 33, 15, 7 with one; a little less here, as a GPU's SMs may lie
    // in other GPCs).  One cluster too many costs a second wave (B1 H16, 1 token on 4000 keys,
    // D64: 20 us with clusters of 16, 15 with clusters of 8).
    constexpr int fit[2][5] = {{296, 148, 64, 32, 12}, {148, 74, 32, 14, 6}};
    f.cluster = 1;
    int at_once = fit[f.rg - 1][0];
    for (int x = 1; x < 5 && items <= fit[f.rg - 1][x] && units >= f.cluster * 4; ++x) {
      f.cluster *= 2;
      at_once = fit[f.rg - 1][x];
    }
    const long long share_ctas = std::max<long long>(1, std::min(slots, items * units / 2));
    const double mean = p->batch > 1 && p->key_lengths ? 0.67 : 1.0;
    const double tile_us = f.rg == 1 ? 0.7 : 0.85, hbm = 0.005 * mean * items * units;
    const double by_cluster = std::max(tile_us * units / f.cluster * std::max(1.0, mean * items / at_once), hbm);
    const double by_share = std::max(tile_us * mean * items * units / share_ctas, hbm) + 12.0;
    if (units > 2 && p->batch <= 1024 && by_share < by_cluster) f.cluster = 0;
    f.grid = static_cast<int>(f.cluster ? items * f.cluster : std::min(slots, items * units / 2));
    f.join = f.cluster == 0;
    if (f.join) {
      const long long rows = 2LL * f.grid * 16 * f.rg;
      f.lse_off = rows * p->head_dim;
      f.entry_off = (f.lse_off + rows) * 4;
      f.bytes = f.entry_off + static_cast<long long>(f.grid) * sizeof(JoinEntry);
    }
    return f;
  }
  const int rows = small_d ? 128 : 256, keys = small_d ? 64 : 128;
  const long long units = std::max<long long>(1, ceil_div(p->k_len, keys));
  // steps of a block of queries on average: lengths that differ are taken as two thirds of
  // the longest; under a causal mask the blocks see more and more keys.  The guess serves lengths
  // that are spread; where all are full it may choose one split too few or too many (B2 H32 over
  // 8, 500 on 8192, D128: 163 us against 125 without the tensor; B4 H32 over 8, 2048 on 4001: 530
  // against 462; B16 H20, 224 on 1500, D64: 66 and 66)
  double mean = static_cast<double>(units);
  if (p->batch > 1 && p->key_lengths) mean *= 0.67;
  if (p->causal) {
    const double off = p->query_offsets ? std::max(0, p->k_len - p->q_len) : p->query_offset;
    const double seen = std::min<double>(p->k_len, std::max(0.0, off + 0.5 * p->q_len)) / std::max(1, p->k_len);
    mean = std::max(1.0, mean * seen);
  }
  // a step of one CTA: up to four of them share an SM at head dims up to 64
  const long long slots = kSMs * (small_d ? FwdLayout<64>::ctas(exact) : FwdLayout<128>::ctas(exact));
  f.per_split = static_cast<int>(split_steps(heads * ceil_div(p->q_len, rows), slots, units, mean,
                                             heads * p->q_len, p->head_dim, small_d ? 1.0 : 2.2, small_d ? 5.0 : 2.7,
                                             small_d ? 11.0 : 4.5));
  f.n_split = static_cast<int>(ceil_div(units, f.per_split));
  f.keys_per_split = f.per_split * keys;
  f.join = f.n_split > 1;
  if (p->bias) f.table_floats = static_cast<long long>(p->q_heads) * table_size(bias);
  f.part_off = f.table_floats;
  f.lse_off = f.part_off + (f.join ? f.n_split * heads * p->q_len * p->head_dim : 0);
  f.bytes = (f.lse_off + (f.join ? f.n_split * heads * p->q_len : 0)) * 4;
  return f;
}

struct BwdPlan {
  int dq_split, dkdv_split;
  long long stat_floats;              // LSE and delta, each
  long long dq_off, dk_off, dv_off;   // offsets in floats; all regions start 256-byte aligned
  long long table_off, lut_off, bias_off, bytes;
};

inline BwdPlan bwd_plan(const ffa_gen_problem* p, const Bias& bias) {
  BwdPlan w{};
  const long long hq = static_cast<long long>(p->batch) * p->q_heads, hk = static_cast<long long>(p->batch) * p->kv_heads;
  const long long qb = ceil_div(p->q_len, 128), kb = ceil_div(p->k_len, 128);
  const long long g = p->kv_heads ? p->q_heads / p->kv_heads : 1;
  const int slots = p->head_dim <= 64 ? 2 * kSMs : kSMs;
  w.dq_split = split_of(hq * qb, slots, kb, 4);
  w.dkdv_split = split_of(hk * kb, slots, g * qb, 4);
  auto round64 = [](long long n) { return (n + 63) / 64 * 64; };
  w.stat_floats = round64(hq * padded_rows(p->q_len));
  long long at = 2 * w.stat_floats;
  w.dq_off = at;
  if (w.dq_split > 1) at += round64(w.dq_split * hq * p->q_len * p->head_dim);
  w.dk_off = at;
  if (w.dkdv_split > 1) at += round64(w.dkdv_split * hk * p->k_len * p->head_dim);
  w.dv_off = at;
  if (w.dkdv_split > 1) at += round64(w.dkdv_split * hk * p->k_len * p->head_dim);
  w.table_off = at;
  if (p->bias) at += round64(static_cast<long long>(p->q_heads) * table_size(bias));
  w.lut_off = at;
  if (p->bias) at += round64(lut_size(bias) / 2);
  w.bias_off = at;
  if (p->bias) at += round64(hq * qb * w.dq_split * p->buckets);
  w.bytes = at * 4;
  return w;
}

// ------------------------------------------------------------------------------------
// launches
// ------------------------------------------------------------------------------------
inline int launched() {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? FFA_OK : set_error(FFA_ERR_LAUNCH, cudaGetErrorString(e));
}

// check_launch_regs, asked once for each kernel (the answer is a property of the build).
inline int check_regs_once(const void* kernel, int needed, bool* done) {
  if (__atomic_load_n(done, __ATOMIC_ACQUIRE)) return FFA_OK;
  const int rc = check_launch_regs(kernel, needed);
  if (rc == FFA_OK) __atomic_store_n(done, true, __ATOMIC_RELEASE);
  return rc;
}

// Clusters of 16 CTAs for `kernel`, once for each device.
inline int allow_clusters_once(const void* kernel, unsigned long long* done) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return set_error(FFA_ERR_LAUNCH, "cudaGetDevice failed");
  const unsigned long long bit = 1ull << (dev & 63);
  if (__atomic_load_n(done, __ATOMIC_ACQUIRE) & bit) return FFA_OK;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
    return set_error(FFA_ERR_LAUNCH, "cudaFuncSetAttribute(NonPortableClusterSizeAllowed) failed");
  __atomic_fetch_or(done, bit, __ATOMIC_ACQ_REL);
  return FFA_OK;
}

struct Call {
  Problem pr;
  Bias bias;
  View q, k, v, o, o_lo, dout, dq, dk, dv;
  float* lse;
  bool want_dbias;
  cudaStream_t stream;
};

// A launch that may start before the kernel in front of it ends (it waits itself, where it
// needs that kernel's results), so that its launch costs nothing.  What the kernel in front
// writes is not constant while this one runs: its pointers are not `const __restrict__`, which
// would let the compiler take the loads for constant ones and move them above the wait.
template <typename... P, typename... A>
static int launch_early(void (*kern)(P...), dim3 grid, int threads, int smem, cudaStream_t stream, A... args) {
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, P(args)...);
  return e == cudaSuccess ? FFA_OK : set_error(FFA_ERR_LAUNCH, cudaGetErrorString(e));
}

static int launch_tables(const Call& c, float* tables, unsigned short* lut) {
  const dim3 grid(static_cast<unsigned>(ceil_div(table_size(c.bias), 256)), std::min(c.pr.Hq, 256));
  ffa_gen_table_kernel<<<grid, 256, 0, c.stream>>>(c.bias, tables, lut, c.pr.Hq);
  return launched();
}

template <int D, bool CAUSAL, bool BIAS, bool EXACT>
static int launch_gen_fwd(const Call& c, const FwdPlan& f, float* ws) {
  using L = FwdLayout<D>;
  const Problem& pr = c.pr;
  CUtensorMap tq, tk, tv, to, tlo;
  int rc;
  if ((rc = make_map(&tq, c.q, pr.B, pr.Hq, pr.Sq, pr.D))) return rc;
  if ((rc = make_map(&to, c.o, pr.B, pr.Hq, pr.Sq, pr.D))) return rc;
  tlo = to;
  if (EXACT && (rc = make_map(&tlo, c.o_lo, pr.B, pr.Hq, pr.Sq, pr.D))) return rc;
  tk = tv = tq;  // without keys nothing is loaded through them
  if (pr.Sk > 0) {
    if ((rc = make_map(&tk, c.k, pr.B, pr.Hkv, pr.Sk, pr.D, L::KEYS))) return rc;
    if ((rc = make_map(&tv, c.v, pr.B, pr.Hkv, pr.Sk, pr.D, L::KEYS))) return rc;
  }
  auto kern = ffa_gen_fwd_kernel<D, CAUSAL, BIAS, EXACT>;
  static unsigned long long configured = 0;
  constexpr int most = L::TAB_OFF + (BIAS ? kTableMax * 4 : 0) + 1024;
  if ((rc = set_smem_once(reinterpret_cast<const void*>(kern), most, &configured))) return rc;
  if constexpr (D == 128) {
    static bool configured_regs = false;
    if ((rc = check_regs_once(reinterpret_cast<const void*>(kern), fwd::LAUNCH_REGS_NEEDED, &configured_regs)))
      return rc;
  }
  if (BIAS && (rc = launch_tables(c, ws, nullptr))) return rc;
  const dim3 grid(static_cast<unsigned>(ceil_div(pr.Sq, L::ROWS) * f.n_split * pr.B * pr.Hq));
  const int group = work_group(pr.B * pr.Hq, pr.Sk, pr.D, CAUSAL), smem = L::smem_bytes(c.bias);
  const float* tables = ws;
  float *part = ws ? ws + f.part_off : nullptr, *part_lse = ws ? ws + f.lse_off : nullptr;
  if (BIAS)
    return launch_early(kern, grid, L::THREADS, smem, c.stream, tq, tk, tv, to, tlo, pr, c.bias, tables, c.lse, part,
                        part_lse, f.n_split, f.per_split, group);
  kern<<<grid, L::THREADS, smem, c.stream>>>(tq, tk, tv, to, tlo, pr, c.bias, tables, c.lse, part, part_lse, f.n_split,
                                             f.per_split, group);
  return launched();
}

template <int D, int RG, bool ROWS8, bool CAUSAL, bool BIAS>
static int launch_gen_step_rg(const Call& c, const FwdPlan& f, float* ws) {
  using L = StepLayout<D, RG>;
  const Problem& pr = c.pr;
  int rc;
  CUtensorMap tk{}, tv{};
  if (pr.Sk > 0) {
    if ((rc = make_map(&tk, c.k, pr.B, pr.Hkv, pr.Sk, pr.D, L::KEYS))) return rc;
    if ((rc = make_map(&tv, c.v, pr.B, pr.Hkv, pr.Sk, pr.D, L::KEYS))) return rc;
  } else {  // the one tile of an item without keys is loaded all the same, and not used
    if ((rc = make_map(&tk, c.q, pr.B, pr.Hq, pr.Sq, pr.D, L::KEYS))) return rc;
    tv = tk;
  }
  int smem = L::LUT_OFF;
  if (BIAS) smem += L::bias_bytes(c.bias, step_heads(L::ROWS, pr.Sq, pr.G));
  auto kern = ffa_gen_step_kernel<D, RG, ROWS8, CAUSAL, BIAS>;
  constexpr int most = L::LUT_OFF + (BIAS ? (2 * kMaxDistance + 8) * 2 + kMaxBuckets * L::ROWS * 4 : 0);
  static unsigned long long configured = 0;
  if ((rc = set_smem_once(reinterpret_cast<const void*>(kern), most, &configured))) return rc;
  JoinEntry* entries = ws ? reinterpret_cast<JoinEntry*>(reinterpret_cast<uintptr_t>(ws) + f.entry_off) : nullptr;
  float* part_lse = ws ? ws + f.lse_off : nullptr;
  if (f.cluster > 8) {
    static unsigned long long sixteen = 0;
    if ((rc = allow_clusters_once(reinterpret_cast<const void*>(kern), &sixteen))) return rc;
  }
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = static_cast<unsigned>(f.cluster > 1 ? f.cluster : 1);
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(f.grid);
  cfg.blockDim = dim3(L::THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = c.stream;
  cfg.attrs = &attr;
  cfg.numAttrs = f.cluster > 1 ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, tk, tv, pr, c.bias, c.q, c.o, c.lse, ws, part_lse, entries,
                                           f.row_tiles, f.cluster);
  if (e != cudaSuccess) return set_error(FFA_ERR_LAUNCH, cudaGetErrorString(e));
  if (!f.join) return FFA_OK;
  const int rows = std::min(L::ROWS, pr.G * pr.Sq);
  return launch_early(ffa_gen_step_join_kernel, dim3(f.grid, static_cast<unsigned>(ceil_div(rows, 4))), 128, 0,
                      c.stream, pr, ws, part_lse, entries, c.o, c.lse, f.row_tiles, L::ROWS);
}

template <int D, bool CAUSAL, bool BIAS>
static int launch_gen_step(const Call& c, const FwdPlan& f, float* ws) {
  if (f.rg == 2) return launch_gen_step_rg<D, 2, false, CAUSAL, BIAS>(c, f, ws);
  return c.pr.G * c.pr.Sq <= 8 ? launch_gen_step_rg<D, 1, true, CAUSAL, BIAS>(c, f, ws)
                               : launch_gen_step_rg<D, 1, false, CAUSAL, BIAS>(c, f, ws);
}

template <int D, bool CAUSAL, bool BIAS>
static int launch_gen_dkdv(const Call& c, const BwdPlan& w, float* ws) {
  using L = DkdvLayout<D, BIAS>;
  using W = BwdShape<D>;
  const Problem& pr = c.pr;
  CUtensorMap tk, tv, tq, tdo, tdk, tdv;
  int rc;
  if ((rc = make_map(&tk, c.k, pr.B, pr.Hkv, pr.Sk, pr.D))) return rc;
  if ((rc = make_map(&tv, c.v, pr.B, pr.Hkv, pr.Sk, pr.D))) return rc;
  if ((rc = make_map(&tdk, c.dk, pr.B, pr.Hkv, pr.Sk, pr.D))) return rc;
  if ((rc = make_map(&tdv, c.dv, pr.B, pr.Hkv, pr.Sk, pr.D))) return rc;
  const bool queries = pr.Hq > 0 && pr.Sq > 0;
  tq = tdo = tk;  // without queries nothing is loaded through them
  if (queries) {
    if ((rc = make_map(&tq, c.q, pr.B, pr.Hq, pr.Sq, pr.D, W::STEP))) return rc;
    if ((rc = make_map(&tdo, c.dout, pr.B, pr.Hq, pr.Sq, pr.D, W::STEP))) return rc;
  }
  auto kern = ffa_gen_dkdv_kernel<D, CAUSAL, BIAS>;
  static unsigned long long configured = 0;
  if ((rc = set_smem_once(reinterpret_cast<const void*>(kern), L::MOST, &configured))) return rc;
  if constexpr (D == 128) {
    static bool configured_regs = false;
    if ((rc = check_regs_once(reinterpret_cast<const void*>(kern), bwd::LAUNCH_REGS_NEEDED, &configured_regs)))
      return rc;
  }
  const dim3 grid(static_cast<unsigned>(ceil_div(pr.Sk, 128) * w.dkdv_split * pr.B * pr.Hkv));
  const int rows = static_cast<int>(std::min<long long>(1LL * pr.Sq * pr.G, INT_MAX));
  const float* tables = ws + w.table_off;
  const float *lse = ws, *delta = ws + w.stat_floats;
  const int smem = L::smem_bytes(c.bias), group = work_group(pr.B * pr.Hkv, rows, pr.D, CAUSAL);
  if (queries)  // behind the kernel that writes delta
    return launch_early(kern, grid, W::THREADS, smem, c.stream, tk, tv, tq, tdo, tdk, tdv, pr, c.bias, tables, lse,
                        delta, ws + w.dk_off, ws + w.dv_off, w.dkdv_split, group);
  kern<<<grid, W::THREADS, smem, c.stream>>>(tk, tv, tq, tdo, tdk, tdv, pr, c.bias, tables, lse, delta, ws + w.dk_off,
                                             ws + w.dv_off, w.dkdv_split, group);
  return launched();
}

template <int D, bool CAUSAL, bool BIAS>
static int launch_gen_dq(const Call& c, const BwdPlan& w, float* ws) {
  using L = DqLayout<D, BIAS>;
  using W = BwdShape<D>;
  const Problem& pr = c.pr;
  CUtensorMap tk, tv, tdq;
  int rc;
  if ((rc = make_map(&tdq, c.dq, pr.B, pr.Hq, pr.Sq, pr.D))) return rc;
  tk = tv = tdq;  // without keys nothing is loaded through them
  if (pr.Sk > 0) {
    if ((rc = make_map(&tk, c.k, pr.B, pr.Hkv, pr.Sk, pr.D, W::STEP))) return rc;
    if ((rc = make_map(&tv, c.v, pr.B, pr.Hkv, pr.Sk, pr.D, W::STEP))) return rc;
  }
  auto kern = ffa_gen_dq_kernel<D, CAUSAL, BIAS>;
  static unsigned long long configured = 0;
  if ((rc = set_smem_once(reinterpret_cast<const void*>(kern), L::MOST, &configured))) return rc;
  if constexpr (D == 128) {
    static bool configured_regs = false;
    if ((rc = check_regs_once(reinterpret_cast<const void*>(kern), bwd::LAUNCH_REGS_NEEDED, &configured_regs)))
      return rc;
  }
  const dim3 grid(static_cast<unsigned>(ceil_div(pr.Sq, 128) * w.dq_split * pr.B * pr.Hq));
  const int smem = L::smem_bytes(c.bias), group = work_group(pr.B * pr.Hq, pr.Sk, pr.D, CAUSAL);
  const float* tables = ws + w.table_off;
  const unsigned short* lut = reinterpret_cast<const unsigned short*>(ws + w.lut_off);
  const float* lse = c.lse;
  float* bias_part = c.want_dbias ? ws + w.bias_off : nullptr;
  if (BIAS)
    return launch_early(kern, grid, W::THREADS, smem, c.stream, tk, tv, tdq, pr, c.bias, tables, lut, c.q, c.o, c.o_lo, c.dout,
                        lse, ws, ws + w.stat_floats, ws + w.dq_off, bias_part, w.dq_split, group);
  kern<<<grid, W::THREADS, smem, c.stream>>>(tk, tv, tdq, pr, c.bias, tables, lut, c.q, c.o, c.o_lo, c.dout, lse, ws,
                                             ws + w.stat_floats, ws + w.dq_off, bias_part, w.dq_split, group);
  return launched();
}

// The instantiation for the problem's head dim, mask and bias (check_problem: causal only
// with a bias).
template <template <int, bool, bool> class F, typename... A>
static int dispatch(const Call& c, bool causal, A&&... a) {
  const bool bias = c.bias.table != nullptr;
  if (c.pr.D <= 64) {
    if (!bias) return F<64, false, false>::run(c, a...);
    return causal ? F<64, true, true>::run(c, a...) : F<64, false, true>::run(c, a...);
  }
  if (!bias) return F<128, false, false>::run(c, a...);
  return causal ? F<128, true, true>::run(c, a...) : F<128, false, true>::run(c, a...);
}
template <int D, bool C, bool B>
struct RunFwd {
  static int run(const Call& c, const FwdPlan& f, float* ws) {
    if constexpr (B)
      if (c.o_lo.p) return launch_gen_fwd<D, C, B, true>(c, f, ws);
    return launch_gen_fwd<D, C, B, false>(c, f, ws);
  }
};
template <int D, bool C, bool B>
struct RunStep {
  static int run(const Call& c, const FwdPlan& f, float* ws) { return launch_gen_step<D, C, B>(c, f, ws); }
};
template <int D, bool C, bool B>
struct RunDkdv {
  static int run(const Call& c, const BwdPlan& w, float* ws) { return launch_gen_dkdv<D, C, B>(c, w, ws); }
};
template <int D, bool C, bool B>
struct RunDq {
  static int run(const Call& c, const BwdPlan& w, float* ws) { return launch_gen_dq<D, C, B>(c, w, ws); }
};

}  // namespace gen
}  // namespace ffa

extern "C" {

long long ffa_gen_fwd_workspace(const ffa_gen_problem* p, int with_o_lo) {
  if (ffa::gen::check_problem(p)) return -1;
  return ffa::gen::fwd_plan(p, ffa::gen::device_bias(p), with_o_lo != 0).bytes;
}

long long ffa_gen_bwd_workspace(const ffa_gen_problem* p) {
  if (ffa::gen::check_problem(p)) return -1;
  return ffa::gen::bwd_plan(p, ffa::gen::device_bias(p)).bytes;
}

int ffa_gen_fwd(const ffa_gen_problem* p, const ffa_gen_tensor* q, const ffa_gen_tensor* k, const ffa_gen_tensor* v,
                const ffa_gen_tensor* o, const ffa_gen_tensor* o_lo, float* lse, void* workspace,
                long long workspace_bytes, void* stream) {
  using namespace ffa::gen;
  int rc = check_problem(p);
  if (rc) return rc;
  if (static_cast<long long>(p->batch) * p->q_heads * p->q_len == 0) return FFA_OK;
  const bool keys = p->k_len > 0;
  if ((rc = check_tensor(q, true)) || (rc = check_tensor(o, true)) || (rc = check_tensor(k, keys)) ||
      (rc = check_tensor(v, keys)))
    return rc;
  const Bias bias = device_bias(p);
  if (o_lo && !p->bias) return ffa::set_error(FFA_ERR_INVALID, "o_lo comes with a bias");
  if (o_lo && (rc = check_tensor(o_lo, true))) return rc;
  const FwdPlan f = fwd_plan(p, bias, o_lo != nullptr);
  if (f.bytes > 0 && (!workspace || workspace_bytes < f.bytes || (reinterpret_cast<uintptr_t>(workspace) & 15u)))
    return ffa::set_error(FFA_ERR_INVALID, "workspace missing, too small or not 16-byte aligned");
  if ((rc = ffa::ensure_context()) != FFA_OK) return rc;
  Call c{};
  c.pr = device_problem(p);
  c.bias = bias;
  c.q = view(q);
  c.k = view(k);
  c.v = view(v);
  c.o = view(o);
  if (o_lo) c.o_lo = view(o_lo);
  c.lse = lse;
  c.stream = static_cast<cudaStream_t>(stream);
  float* ws = f.bytes > 0 ? static_cast<float*>(workspace) : nullptr;
  if (f.step) return dispatch<RunStep>(c, p->causal, f, ws);
  rc = dispatch<RunFwd>(c, p->causal, f, ws);
  if (rc || !f.join) return rc;
  const long long rows = static_cast<long long>(p->batch) * p->q_heads * p->q_len;
  auto join = [&](auto kern, int lanes) {
    return launch_early(kern, dim3(static_cast<unsigned>(ceil_div(rows * lanes, 256))), 256, 0, c.stream, c.pr,
                        ws + f.part_off, ws + f.lse_off, c.o, c.o_lo, lse, f.keys_per_split, p->causal ? 1 : 0);
  };
  return p->head_dim <= 64 ? join(ffa_gen_join_kernel<16>, 16) : join(ffa_gen_join_kernel<32>, 32);
}

int ffa_gen_bwd(const ffa_gen_problem* p, const ffa_gen_tensor* q, const ffa_gen_tensor* k, const ffa_gen_tensor* v,
                const ffa_gen_tensor* o, const ffa_gen_tensor* o_lo, const ffa_gen_tensor* dout, const float* lse,
                const ffa_gen_tensor* dq, const ffa_gen_tensor* dk, const ffa_gen_tensor* dv, void* dbias, void* workspace,
                long long workspace_bytes, void* stream) {
  using namespace ffa::gen;
  int rc = check_problem(p);
  if (rc) return rc;
  const long long hq = static_cast<long long>(p->batch) * p->q_heads;
  const bool queries = hq * p->q_len > 0, keys = static_cast<long long>(p->batch) * p->kv_heads * p->k_len > 0;
  const bool want_dq = dq != nullptr, want_dkdv = dk != nullptr;
  if (want_dkdv != (dv != nullptr)) return ffa::set_error(FFA_ERR_INVALID, "dk and dv are wanted together");
  if (dbias && (!p->bias || !want_dq)) return ffa::set_error(FFA_ERR_INVALID, "dbias needs a bias, and comes with dq");
  if ((rc = check_tensor(q, queries)) || (rc = check_tensor(o, queries)) || (rc = check_tensor(dout, queries)) ||
      (rc = check_tensor(k, keys)) || (rc = check_tensor(v, keys)))
    return rc;
  if (o_lo && (rc = check_tensor(o_lo, queries))) return rc;
  if (queries && !lse) return ffa::set_error(FFA_ERR_INVALID, "null tensor pointer");
  if (want_dq && (rc = check_tensor(dq, queries))) return rc;
  if (want_dkdv && ((rc = check_tensor(dk, keys)) || (rc = check_tensor(dv, keys)))) return rc;
  const Bias bias = device_bias(p);
  const BwdPlan w = bwd_plan(p, bias);
  if (w.bytes > 0 && (!workspace || workspace_bytes < w.bytes || (reinterpret_cast<uintptr_t>(workspace) & 15u)))
    return ffa::set_error(FFA_ERR_INVALID, "workspace missing, too small or not 16-byte aligned");
  if ((rc = ffa::ensure_context()) != FFA_OK) return rc;
  Call c{};
  c.pr = device_problem(p);
  c.bias = bias;
  c.q = view(q);
  c.k = view(k);
  c.v = view(v);
  c.o = view(o);
  if (o_lo) c.o_lo = view(o_lo);
  c.dout = view(dout);
  c.lse = const_cast<float*>(lse);
  c.stream = static_cast<cudaStream_t>(stream);
  float* ws = static_cast<float*>(workspace);
  if (p->bias && queries && (rc = launch_tables(c, ws + w.table_off, reinterpret_cast<unsigned short*>(ws + w.lut_off))))
    return rc;
  if (queries && !want_dq) {
    const long long rows = hq * padded_rows(p->q_len);
    if (p->head_dim <= 64)
      ffa_gen_prepare_kernel<8><<<static_cast<unsigned>(rows / 32), 256, 0, c.stream>>>(
          c.o, c.dout, lse, ws, ws + w.stat_floats, p->q_heads, p->q_len, p->head_dim);
    else
      ffa_gen_prepare_kernel<16><<<static_cast<unsigned>(rows / 16), 256, 0, c.stream>>>(
          c.o, c.dout, lse, ws, ws + w.stat_floats, p->q_heads, p->q_len, p->head_dim);
    if ((rc = launched())) return rc;
  }
  // `n` (one or two) gradients of the same shape from their splits, behind the kernel that wrote them
  auto sum = [&](int n, const float* part0, const View& out0, const float* part1, const View& out1, int n_split, int H,
                 int S) {
    const long long chunks = static_cast<long long>(p->batch) * H * S * (p->head_dim / 8);
    return launch_early(ffa_gen_sum_kernel, dim3(static_cast<unsigned>(ceil_div(chunks, 256)), n), 256, 0, c.stream, part0,
                        part1, out0, out1, n_split, p->batch, H, S, p->head_dim);
  };
  if (want_dq && queries) {
    c.dq = view(dq);
    c.want_dbias = dbias != nullptr;
    if ((rc = dispatch<RunDq>(c, p->causal, w, ws))) return rc;
  }
  if (want_dkdv && keys) {
    c.dk = view(dk);
    c.dv = view(dv);
    if ((rc = dispatch<RunDkdv>(c, p->causal, w, ws))) return rc;
    if (w.dkdv_split > 1 &&
        (rc = sum(2, ws + w.dk_off, c.dk, ws + w.dv_off, c.dv, w.dkdv_split, p->kv_heads, p->k_len)))
      return rc;
  }
  if (want_dq && queries && w.dq_split > 1 &&
      (rc = sum(1, ws + w.dq_off, c.dq, ws + w.dq_off, c.dq, w.dq_split, p->q_heads, p->q_len)))
    return rc;
  if (dbias && p->q_heads > 0) {
    const int blocks = queries ? static_cast<int>(ceil_div(p->q_len, 128)) * w.dq_split : 0;
    ffa_gen_bias_sum_kernel<<<static_cast<unsigned>(ceil_div(static_cast<long long>(p->q_heads) * p->buckets, 4)), 128,
                              0, c.stream>>>(ws + w.bias_off, static_cast<__nv_bfloat16*>(dbias), p->batch, p->q_heads,
                                             blocks, p->buckets);
    if ((rc = launched())) return rc;
  }
  return FFA_OK;
}

}  // extern "C"
