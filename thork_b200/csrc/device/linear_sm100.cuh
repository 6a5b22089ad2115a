// linear_sm100.cuh — the linear-layer kernels for sm_100a: matrix products
// with bias, activation and residual in the epilogue, and the same products
// grouped by expert with ragged sizes, forward and backward.
//
//   rows_kernel   persistent CTA pairs (tcgen05 cta_group::2), tiles of 256
//                 columns by up to 256 rows: products of many rows
//   outer_kernel  the same for a product over rows: the weights' gradient
//   swap_kernel   one 128 x BN tile per cluster with the weights as the MMA's
//                 128 rows, the contraction split over the cluster and summed
//                 through distributed shared memory: few rows, bound by the
//                 bytes of the weights
//   slope_kernel  dpre = dout * act'(preact) and the bias gradient's column
//                 sums: bound by its three passes over [M, N]
//
// Operand layouts in shared memory are the 128-byte-swizzled canonical ones
// that TMA writes (sm100.cuh).  A grouped product takes the expert's row
// ranges from `offsets` in device memory; every offset is clamped into the
// row buffer and made non-decreasing, so no value of it reads or writes
// outside the arrays.
#pragma once
#include "sm100.cuh"

namespace thork {
namespace lin {

using namespace thork::dev;

enum : int { KIND_BF16 = 0, KIND_E4M3 = 1 };
enum : int { ACT_NONE = 0, ACT_RELU = 1, ACT_GELU = 2, ACT_GELU_TANH = 3, ACT_SILU = 4 };

constexpr int kMaxGroups = 1024;

// Every kernel here may start before the kernel that writes its inputs has
// ended (programmatic dependent launch), and out may be the residual itself.
// So ordinary loads go past L1 (ld.global.cg): neither a read-only load, whose
// data may not change while the kernel lives, nor a line that this SM cached
// before the wait can return an old value.

// What happens to an accumulator on its way to the output:
//   z = acc * alpha [* group_scale[g]] + bias;  preact = z;
//   out = act(z) + residual
// in fp32, each output rounded once to bf16.
struct Epilogue {
  unsigned short *out;             // bf16 [rows, cols]
  unsigned short *preact;          // bf16 [rows, cols] or null
  const unsigned short *bias;      // bf16 [cols] or null
  const unsigned short *residual;  // bf16 [rows, cols] or null
  const float *group_scale;        // fp32 [groups] or null
  float alpha;
  int act;
  int cols;
  u32 *status;
};

struct GemmArgs {
  Epilogue epi;
  int GM, GN, GK;      // extents of the (per-group) product; grouped rows: GM = buffer rows
  const int *offsets;  // [groups + 1] row offsets, or null
  int groups, rows;    // groups, rows of the buffer that the offsets divide
  int w_static;        // swap_kernel: no earlier launch writes the weights
  // Two products of one call that do not read each other's output overlap: the
  // first (trigger_late) lets the second start only once everything before the
  // first has completed, so that the second (wait_last) needs no wait of its
  // own before it reads; it waits for the first before it ends, so whatever
  // follows it follows both.
  int trigger_late, wait_last;
};

// ---------------------------------------------------------------- small PTX
__device__ __forceinline__ void tma_load_3d(u32 dst, const TensorMap *m, u32 bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<u64>(m)), "r"(bar), "r"(x), "r"(y), "r"(z)
      : "memory");
}

// Completion may be counted on the other CTA's barrier of a pair.
__device__ __forceinline__ void tma_load_3d_pair(u32 dst, const TensorMap *m, u32 bar_cluster, int x,
                                                 int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<u64>(m)), "r"(bar_cluster), "r"(x), "r"(y), "r"(z)
      : "memory");
}

__device__ __forceinline__ void tma_store_3d(const TensorMap *m, u32 src, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(
          reinterpret_cast<u64>(m)),
      "r"(src), "r"(x), "r"(y), "r"(z)
      : "memory");
}

// Arrive on `bar`, at the same shared-memory offset in both CTAs of a pair,
// when the tcgen05 operations issued so far by this thread are complete.
__device__ __forceinline__ void tc_commit_pair(u32 bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          bar),
      "h"(static_cast<unsigned short>(3))
      : "memory");
}

// An epilogue warp hands its accumulator columns back to the MMA thread of the
// pair's leader (`bar_cluster` in its shared memory).  What is ordered are the
// tensor-memory loads, which have completed and which
// tcgen05.fence::before_thread_sync orders before this arrival, so it need not
// release memory: as a release of cluster scope it waited for every store in
// flight (outer_kernel: 2000 of 4500 cycles between short tiles).
__device__ __forceinline__ void arrive_tmem_free(u32 bar_cluster) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar_cluster) : "memory");
}

// One lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  u32 p;
  asm volatile(
      "{\n\t.reg .pred P;\n\t"
      "elect.sync _|P, 0xffffffff;\n\t"
      "selp.b32 %0, 1, 0, P;\n\t}"
      : "=r"(p));
  return p != 0;
}

__device__ __forceinline__ u32 cluster_nctarank() {
  u32 r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}

__device__ __forceinline__ float4 ld_cluster_v4(u32 addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

__device__ __forceinline__ float ld_cluster_f32(u32 addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

__device__ __forceinline__ void st_cluster_u32(u32 addr, u32 v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

__device__ __forceinline__ float bf16_lo(u32 w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(u32 w) { return __uint_as_float(w & 0xFFFF0000u); }

// ---------------------------------------------------------------- activations
// silu is z * sigmoid(z) and gelu_tanh z * sigmoid(2u): one exponential and one
// reciprocal each.  The normal distribution function of gelu is written as its
// lower tail, Phi(-|z|) = exp(-z^2 / 2) t P(t) with t = 1 / (1 + p |z|), the form
// of Hastings' approximations of erf; p and the six coefficients of P were fitted
// here to the tail itself, for the smallest larger one of its relative error over
// 1e-4 and its absolute error over 1.5e-7 (Lawson's iteration on [0, 13.5]).  Its
// exponential is the density's, which the slope needs as well.  Both tails stay
// relatively accurate, which the bf16 rounding of a small result needs: evaluated
// in fp32 Phi(-|z|) is within 5e-5 of its value (a fit of erf's absolute error
// was off by 0.9 half-steps of bf16 at -6, by 5 at -10) and within 3e-7 in all; the
// others within 2e-5, where the exponent is large, and 2^-21 elsewhere.  An
// exponential or a sigmoid below 2^-126 counts as 0.  A NaN stays a NaN (relu
// included).
//
// Two values at a time, in the packed fp32 instructions: slope_kernel has
// about as many instructions to issue as bytes to move (4096 x 14336, gelu:
// 126 us with erff and expf, 73 with an approximation of its own, 62-70 packed;
// its traffic takes 54).
struct F2 {
  u64 v;
};
__device__ __forceinline__ F2 f2(float lo, float hi) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ F2 f2(float x) { return f2(x, x); }
__device__ __forceinline__ void split(F2 a, float &lo, float &hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(a.v));
}
__device__ __forceinline__ F2 operator*(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 operator+(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ F2 exp2_2(F2 a) {
  float x, y;
  split(a, x, y);
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(x));
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(y));
  return f2(x, y);
}
__device__ __forceinline__ F2 reciprocal2(F2 a) {  // 0 for infinity
  float x, y;
  split(a, x, y);
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(x));
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(y));
  return f2(x, y);
}

constexpr float kLog2e = 1.4426950408889634f;

// 1 / (1 + 2^-a)
__device__ __forceinline__ F2 sigmoid_exp2(F2 minus_a) { return reciprocal2(f2(1.0f) + exp2_2(minus_a)); }

// Phi(z), and bell = exp(-z^2 / 2).
__device__ __forceinline__ F2 normal_cdf(F2 z, F2 &bell) {
  bell = exp2_2(z * z * f2(-0.5f * kLog2e));
  float x, y, tx, ty;
  split(z, x, y);
  const F2 t = reciprocal2(fma2(f2(0.29219924f), f2(fabsf(x), fabsf(y)), f2(1.0f)));
  F2 poly = fma2(t, f2(-0.0865463706f), f2(0.2694105702f));
  poly = fma2(t, poly, f2(-0.0747055592f));
  poly = fma2(t, poly, f2(0.1701724730f));
  poly = fma2(t, poly, f2(0.1041578453f));
  poly = fma2(t, poly, f2(0.1175109787f));
  split(t * poly * bell, tx, ty);  // Phi(-|z|)
  return f2(x < 0.0f ? tx : 1.0f - tx, y < 0.0f ? ty : 1.0f - ty);
}

// -2u log2(e) = z (c0 + c1 z^2) for gelu_tanh's 2u = 2 sqrt(2/pi) (z + 0.044715 z^3)
constexpr float kTanh0 = 1.5957691216057308f, kTanh1 = kTanh0 * 0.044715f;

__device__ __forceinline__ F2 act_value(F2 z, int act) {
  F2 bell;
  switch (act) {
    case ACT_GELU: return z * normal_cdf(z, bell);
    case ACT_GELU_TANH:
      return z * sigmoid_exp2(z * fma2(z * z, f2(-kTanh1 * kLog2e), f2(-kTanh0 * kLog2e)));
    default: return z * sigmoid_exp2(z * f2(-kLog2e));  // silu
  }
}

// Derivative of the activation at z.
__device__ __forceinline__ F2 act_slope(F2 z, int act) {
  if (act == ACT_GELU) {
    F2 bell;
    const F2 cdf = normal_cdf(z, bell);
    return fma2(z * f2(0.3989422804014327f), bell, cdf);
  }
  if (act == ACT_GELU_TANH) {
    const F2 zz = z * z;
    const F2 p = sigmoid_exp2(z * fma2(zz, f2(-kTanh1 * kLog2e), f2(-kTanh0 * kLog2e)));
    const F2 q = fma2(p, p * f2(-1.0f), p);  // p (1 - p)
    // z q first, which is 0 for large |z|, where z^2 overflows (0 times infinity)
    const F2 w = z * q;
    return fma2(w * z * z, f2(3.0f * kTanh1), fma2(w, f2(kTanh0), p));
  }
  const F2 p = sigmoid_exp2(z * f2(-kLog2e));
  const F2 q = fma2(p, p * f2(-1.0f), p);
  return fma2(z, q, p);
}

template <int ACT, int N>
__device__ __forceinline__ void act_forward_as(float (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N; i += 2) split(act_value(f2(v[i], v[i + 1]), ACT), v[i], v[i + 1]);
}

template <int N>
__device__ __forceinline__ void act_forward(float (&v)[N], int act) {
  if (act == ACT_RELU) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = v[i] <= 0.0f ? 0.0f : v[i];
  } else if (act == ACT_GELU) {
    act_forward_as<ACT_GELU>(v);
  } else if (act == ACT_GELU_TANH) {
    act_forward_as<ACT_GELU_TANH>(v);
  } else if (act == ACT_SILU) {
    act_forward_as<ACT_SILU>(v);
  }
}

template <int ACT, int N>
__device__ __forceinline__ void act_backward_as(float (&v)[N], const float (&z)[N]) {
#pragma unroll
  for (int i = 0; i < N; i += 2)
    split(f2(v[i], v[i + 1]) * act_slope(f2(z[i], z[i + 1]), ACT), v[i], v[i + 1]);
}

// v[i] *= derivative of the activation at z[i].
template <int N>
__device__ __forceinline__ void act_backward(float (&v)[N], const float (&z)[N], int act) {
  if (act == ACT_RELU) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] *= z[i] > 0.0f ? 1.0f : 0.0f;
  } else if (act == ACT_GELU) {
    act_backward_as<ACT_GELU>(v, z);
  } else if (act == ACT_GELU_TANH) {
    act_backward_as<ACT_GELU_TANH>(v, z);
  } else if (act == ACT_SILU) {
    act_backward_as<ACT_SILU>(v, z);
  }
}

// ---------------------------------------------------------------- groups
// off[i] clamped into [0, rows] and made non-decreasing, and the running
// count of row tiles of `tile` rows, by one warp (all lanes call).
// tab_off has groups + 1 entries, tab_tile (may be null) too.
__device__ __forceinline__ void scan_groups(const int *offsets, int groups, int rows, int tile,
                                            int *tab_off, int *tab_tile, u32 *status) {
  const int lane = static_cast<int>(lane_id());
  int top = 0, count = 0;  // running maximum of the offsets, running tile count
  bool bad = false;
  for (int base = 0; base <= groups; base += 32) {
    const int i = base + lane;
    const int raw = i <= groups ? __ldcg(offsets + i) : 0;
    int v = max(0, min(raw, rows));
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, v, d);
      if (lane >= d) v = max(v, o);
    }
    v = max(v, top);
    bad |= i <= groups && v != raw;
    int prev = __shfl_up_sync(0xffffffffu, v, 1);
    if (lane == 0) prev = base == 0 ? v : top;
    // tiles of group i - 1, whose rows are [prev, v)
    int n = (i >= 1 && i <= groups) ? (v - prev + tile - 1) / tile : 0;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, n, d);
      if (lane >= d) n += o;
    }
    n += count;
    if (i <= groups) {
      tab_off[i] = v;
      if (tab_tile) tab_tile[i] = n;
    }
    top = __shfl_sync(0xffffffffu, v, 31);
    count = __shfl_sync(0xffffffffu, n, 31);
  }
  if (bad) report_status(status, STATUS_BAD_CONFIG, 0x40);
}

// ===========================================================================
// rows_kernel
// ===========================================================================
// out[m, n] = act(sum_k X[m, k] W[k, n] ...) for many rows.  A cluster of two
// CTAs computes tiles of 256 columns n by up to 256 rows m, as the transpose:
// the weights are the MMA's M dimension (CTA r holds columns
// [128 r, 128 r + 128)), the rows its N dimension (CTA r holds one half of the
// tile's rows).  The N dimension of an instruction may be any multiple of 32,
// so a tile has as many rows as there are, in units of 64: a group's rows, or
// a product's, fill tiles of four units and leave the rest to a last, shorter
// one, and no multiplication is spent on rows of another group.  With rows as the M
// dimension every group would round up to 256 rows.
//
// Persistent: pair i takes tiles i, i + pairs, ...; the tiles of the last,
// partial wave are split by rows into as many pieces as there are pairs for
// (4096^3: 256 tiles are 3.46 waves; the last 34 become 68 halves).
//
// Warps: 0 TMA producer, 1 MMA issuer (leader only), 2..9 epilogue: two warps
// per TMEM lane quadrant, taking the tile's 32-row slices in turn.
//
// Bound by the tensor pipe (90 % of active cycles at 4096 x 4096 x 14336), and
// back to back by the power cap.  Ten calls after a pause / 1.5 s back to back:
// 4096^3 94 us (1460 TFLOP/s) / 110 (1248), with gelu, bias, residual and saved
// pre-activation 103 (1337) / 122 (1130); 8192^3 732 (1502) / 829 (1326); e4m3
// 8192^3 with bias, relu and residual 396 (2776) / 443 (2484); 8 experts of 14336
// x 4096 with 8192 rows and silu 655 (1468) / 736 (1307), 725 / 826 with the rows
// dealt out unevenly.  Where tiles are fewer than pairs, splitting them by rows
// fills the pairs but shortens no tile's contraction, of which a block takes 0.2
// to 0.3 us however few its rows: 256 x 4096 x 4096 22 us of 5.8.  Six stages of
// 32 KiB per CTA; 512-column tiles of four 48 KiB stages gained 1 % at 8192^3
// and lost 3 % at 4096^3.
template <int KIND_, bool W_MN_, bool GROUPED_>
struct RowsCfg {
  static constexpr int KIND = KIND_, STAGES = 6;
  static constexpr bool W_MN = W_MN_, GROUPED = GROUPED_;
  static constexpr int ELEM = KIND == KIND_BF16 ? 2 : 1;
  static constexpr int BNC = 128;  // columns per CTA
  static constexpr int UNIT = 64, MAX_UNITS = 4;
  static constexpr int BOX_ROWS = UNIT / 2;  // a CTA's half of a unit, one TMA box
  static constexpr int BK = 128 / ELEM;
  static constexpr int CHUNK = 128 / ELEM;
  static constexpr int UMMA_K = 32 / ELEM;
  static constexpr int W_BYTES = BNC * 128, BOX_BYTES = BOX_ROWS * 128;
  static constexpr int STAGE_BYTES = W_BYTES + MAX_UNITS * BOX_BYTES;
  static constexpr int TMEM_COLS = 2 * UNIT * MAX_UNITS;
  static constexpr int EPI_WARPS = 8;
  static constexpr int THREADS = 32 * (2 + EPI_WARPS);
  static constexpr int RASTER = 8;  // row tiles walked column by column
  static constexpr int STG_OFF = STAGES * STAGE_BYTES;
  static constexpr int BAR_OFF = STG_OFF + EPI_WARPS * 2048;
  static constexpr int NBARS = 2 * STAGES + 5;
  static constexpr int TAB_OFF = BAR_OFF + NBARS * 8 + 16;
  static constexpr int TAB_BYTES = GROUPED ? (kMaxGroups + 1) * 8 : 0;
  static constexpr int SMEM_BYTES = 1024 + TAB_OFF + TAB_BYTES;
  // without the N field, which is the tile's
  static constexpr u32 IDESC =
      make_idesc(KIND == KIND_BF16 ? 1u : 0u, KIND == KIND_BF16 ? 1u : 0u, W_MN, false, 256, 0);
  static_assert(SMEM_BYTES <= 232448, "shared memory budget exceeded");
};

// n / d for 0 <= n < 2^31 by a multiplication: every role of a persistent
// kernel finds its tiles with a few of these, and a division instruction
// sequence is long enough to show between short tiles.
struct Divisor {
  u32 d, m;
  __device__ __forceinline__ explicit Divisor(int d_) : d(d_), m(0xFFFFFFFFu / static_cast<u32>(d_)) {}
  // floor(n m / 2^32) is the quotient or one less, as n < 2^31
  __device__ __forceinline__ int operator()(int n, int &rest) const {
    u32 q = __umulhi(static_cast<u32>(n), m), r = static_cast<u32>(n) - q * d;
    if (r >= d) {
      ++q;
      r -= d;
    }
    rest = static_cast<int>(r);
    return static_cast<int>(q);
  }
};

// Tile t of an ntm x ntn grid of tiles: bands of BAND tile rows are walked
// column by column, so that the tiles in flight share operand panels in L2.
template <int BAND>
struct Raster {
  Divisor band;  // tiles of a whole band
  int ntn;
  __device__ __forceinline__ explicit Raster(int ntn_) : band(BAND * ntn_), ntn(ntn_) {}
  __device__ __forceinline__ void operator()(int t, int ntm, int &tm, int &tn) const {
    int r;
    const int q = band(t, r), first = q * BAND, rows = ntm - first;
    if (rows >= BAND) {
      tn = r / BAND;
      tm = first + r % BAND;
    } else {
      tn = r / rows;
      tm = first + r - tn * rows;
    }
  }
};

template <int N>
struct Const {
  static constexpr int value = N;
};

struct RowTile {
  int m0, row_end;  // first row; rows from here on belong to another tile or group
  int n0;           // first column (of the pair)
  int units;        // 64-row units
  int grp;
};

// The pair's tiles in order; every role walks the same sequence.
template <class C>
struct RowWalk {
  const GemmArgs &g;
  const int *tab_off, *tab_tile;
  int i, step, whole, pieces, items, grp, ntn;
  Raster<C::RASTER> raster;

  __device__ __forceinline__ RowWalk(const GemmArgs &g_, const int *o, const int *tl)
      : g(g_), tab_off(o), tab_tile(tl), i(blockIdx.x / 2), step(gridDim.x / 2), grp(0),
        ntn((g_.GN + 2 * C::BNC - 1) / (2 * C::BNC)), raster(ntn) {
    const int total = (C::GROUPED ? tab_tile[g.groups] : row_tiles(g.GM)) * ntn;
    const int rest = total % step;
    whole = total - rest;
    pieces = rest ? min(C::MAX_UNITS, step / rest) : 1;
    items = whole + rest * pieces;
    more = find(ahead);
  }
  static __device__ __forceinline__ int row_tiles(int rows) {
    return (rows + C::UNIT * C::MAX_UNITS - 1) / (C::UNIT * C::MAX_UNITS);
  }

  // The next tile; the one after it is worked out here as well, while the
  // caller's first wait would still be pending, so that the arithmetic stays
  // off the path from one tile's end to the next one's start.
  RowTile ahead;
  bool more;
  __device__ __forceinline__ bool next(RowTile &x) {
    if (!more) return false;
    x = ahead;
    more = find(ahead);
    return true;
  }

  __device__ __forceinline__ bool find(RowTile &x) {
    for (; i < items; i += step) {
      int t = i, piece = 0, parts = 1;
      if (i >= whole && pieces > 1) {
        const int r = i - whole;
        t = whole + r / pieces;
        piece = r - r / pieces * pieces;
        parts = pieces;
      }
      int first = 0, base = 0, rows = g.GM, ntm;
      if (C::GROUPED) {
        while (t >= tab_tile[grp + 1] * ntn) ++grp;
        first = tab_tile[grp];
        ntm = tab_tile[grp + 1] - first;
        base = tab_off[grp];
        rows = tab_off[grp + 1] - base;
      } else {
        ntm = row_tiles(rows);
      }
      int tm, tn;
      raster(t - first * ntn, ntm, tm, tn);
      // the row tile's units, and of those the piece's
      const int units = min((rows - tm * (C::UNIT * C::MAX_UNITS) + C::UNIT - 1) / C::UNIT, C::MAX_UNITS);
      const int p0 = units * piece / parts, p1 = units * (piece + 1) / parts;
      if (p1 == p0) continue;
      const int row = tm * (C::UNIT * C::MAX_UNITS);
      x.m0 = base + row + p0 * C::UNIT;
      x.row_end = base + min(rows, row + p1 * C::UNIT);
      x.n0 = tn * 2 * C::BNC;
      x.units = p1 - p0;
      x.grp = C::GROUPED ? grp : 0;
      i += step;
      return true;
    }
    return false;
  }
};

// A warp's block of the output: 32 columns n (TMEM lanes) by 32 rows m (TMEM
// columns).  tcgen05.ld.16x256b delivers it as 8 x 8 fragments of (n, m), and
// stmatrix.trans writes such fragments as (m, n): one instruction per four
// fragments turns the accumulator's columns into the output's rows.
//
// Fragment values: f[h][4 j + 2 e + i] is column n = 16 h + 8 e + lane / 4,
// row m = 8 j + 2 (lane % 4) + i.  The staging block is 32 rows of 64 bytes;
// 16-byte chunk c of row r lies at chunk c ^ (r / 2 % 4), which spreads the
// eight rows of a fragment over all banks.
__device__ __forceinline__ void tmem_ld_16x256b_x4(u32 taddr, u32 (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}

// Address that this lane gives a matrix instruction over the four column
// blocks (chunks) of rows [8 j, 8 j + 8): row 8 j + lane % 8, chunk lane / 8.
__device__ __forceinline__ u32 block_addr(u32 stg, int j, int lane) {
  const int r = 8 * j + (lane & 7);
  return stg + r * 64 + (((lane >> 3) ^ ((r >> 1) & 3)) * 16);
}

__device__ __forceinline__ void put_block(const float (&f)[2][16], u32 stg, int lane) {
#pragma unroll
  for (int j = 0; j < 4; ++j)
    asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(
                     block_addr(stg, j, lane)),
                 "r"(pack_bf16x2(f[0][4 * j], f[0][4 * j + 1])), "r"(pack_bf16x2(f[0][4 * j + 2], f[0][4 * j + 3])),
                 "r"(pack_bf16x2(f[1][4 * j], f[1][4 * j + 1])), "r"(pack_bf16x2(f[1][4 * j + 2], f[1][4 * j + 3]))
                 : "memory");
}

__device__ __forceinline__ void add_block(float (&f)[2][16], u32 stg, int lane) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    u32 w[4];
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                 : "r"(block_addr(stg, j, lane))
                 : "memory");
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        f[h][4 * j + 2 * e] += bf16_lo(w[2 * h + e]);
        f[h][4 * j + 2 * e + 1] += bf16_hi(w[2 * h + e]);
      }
  }
}

// The block's rows in global memory, 16 bytes per lane and step: lane covers
// chunk lane % 4 of row 8 it + lane / 4.
__device__ __forceinline__ void load_block(uint4 (&v)[4], const unsigned short *src, int cols, int row0,
                                           int row_end, int col0, int lane) {
  const int col = col0 + (lane & 3) * 8;
#pragma unroll
  for (int it = 0; it < 4; ++it) {
    const int row = row0 + 8 * it + (lane >> 2);
    v[it] = make_uint4(0, 0, 0, 0);
    if (row < row_end && col < cols)
      v[it] = __ldcg(reinterpret_cast<const uint4 *>(src + static_cast<long long>(row) * cols + col));
  }
}

__device__ __forceinline__ uint4 *staged(unsigned char *stg, int it, int lane) {
  const int r = 8 * it + (lane >> 2);
  return reinterpret_cast<uint4 *>(stg + r * 64 + (((lane & 3) ^ ((r >> 1) & 3)) * 16));
}

__device__ __forceinline__ void store_block(unsigned char *stg, unsigned short *dst, int cols, int row0,
                                            int row_end, int col0, int lane) {
  const int col = col0 + (lane & 3) * 8;
#pragma unroll
  for (int it = 0; it < 4; ++it) {
    const int row = row0 + 8 * it + (lane >> 2);
    const uint4 v = *staged(stg, it, lane);
    // cols is a multiple of 8, so a 16-byte chunk is wholly in or out
    if (row < row_end && col < cols)
      st_global_v4(dst + static_cast<long long>(row) * cols + col, v.x, v.y, v.z, v.w);
  }
}

template <class C>
__global__ void __launch_bounds__(C::THREADS, 1)
    rows_kernel(const __grid_constant__ TensorMap tmap_w, const __grid_constant__ TensorMap tmap_x,
                const __grid_constant__ TensorMap tmap_xu, const GemmArgs g) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  const u32 raw = smem_u32(smem_raw);
  const u32 base = (raw + 1023u) & ~1023u;
  unsigned char *smem = smem_raw + (base - raw);
  const u32 bars = base + C::BAR_OFF;
  auto full_bar = [&](int s) { return bars + 8u * s; };
  auto empty_bar = [&](int s) { return bars + 8u * (C::STAGES + s); };
  auto tfull_bar = [&](int a) { return bars + 8u * (2 * C::STAGES + a); };
  auto tempty_bar = [&](int a) { return bars + 8u * (2 * C::STAGES + 2 + a); };
  const u32 drain_bar = bars + 8u * (2 * C::STAGES + 4);
  u32 *tmem_slot = reinterpret_cast<u32 *>(smem + C::BAR_OFF + C::NBARS * 8);
  volatile u32 *abort_flag = tmem_slot + 1;
  int *tab_off = reinterpret_cast<int *>(smem + C::TAB_OFF);
  int *tab_tile = tab_off + kMaxGroups + 1;
  u32 *status = g.epi.status;

  const int warp = threadIdx.x / 32;
  const int lane = threadIdx.x % 32;
  const u32 rank = cluster_ctarank();

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(tfull_bar(a), 1);
      mbar_init(tempty_bar(a), 2 * C::EPI_WARPS);  // both CTAs' epilogue warps, on the leader's
    }
    mbar_init(drain_bar, 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmap_w);
    tma_prefetch_desc(&tmap_x);
    tma_prefetch_desc(&tmap_xu);
  }
  if (warp == 1) {
    tmem_alloc<2>(smem_u32(tmem_slot), C::TMEM_COLS);
    tmem_relinquish<2>();
  }
  if (C::GROUPED && warp == 2) {
    pdl_wait();  // the offsets may come from the previous kernel of the stream
    scan_groups(g.offsets, g.groups, g.rows, C::UNIT * C::MAX_UNITS, tab_off, tab_tile,
                blockIdx.x == 0 ? status : nullptr);
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // both CTAs' barriers are initialised before any remote use
  tc_fence_after();
  if (!g.trigger_late) pdl_launch_dependents();
  const u32 tmem_base = *tmem_slot;
  const int nkb = (g.GK + C::BK - 1) / C::BK;
  pdl_wait();  // the previous kernel of the stream is complete from here on
  if (g.trigger_late && threadIdx.x == 0) pdl_launch_dependents();

  if (warp == 0) {
    // ------------------------------------------------ TMA producer (both CTAs)
    if (elect_one()) {
      RowWalk<C> walk(g, tab_off, tab_tile);
      RowTile x;
      const u32 leader_full = mapa_cluster(full_bar(0), 0);
      int s = 0;
      u32 ph = 0;
      while (!*abort_flag && walk.next(x)) {
        const int n = x.n0 + rank * C::BNC, m = x.m0 + rank * x.units * C::BOX_ROWS;
        const u32 bytes = 2 * (C::W_BYTES + x.units * C::BOX_BYTES);
        for (int kb = 0; kb < nkb; ++kb) {
          if (!mbar_wait(empty_bar(s), ph ^ 1u, status, 0x61)) {
            *abort_flag = 1;
            break;
          }
          const u32 sw = base + s * C::STAGE_BYTES, sx = sw + C::W_BYTES;
          const u32 fb = leader_full + 8u * s;
          if (rank == 0) mbar_arrive_expect_tx(full_bar(s), bytes);
          if (C::W_MN) {
#pragma unroll
            for (int c = 0; c < C::BNC / C::CHUNK; ++c)
              tma_load_3d_pair(sw + c * C::BK * 128, &tmap_w, fb, n + c * C::CHUNK, kb * C::BK, x.grp);
          } else {
            tma_load_3d_pair(sw, &tmap_w, fb, kb * C::BK, n, x.grp);
          }
          // a whole tile's rows in one box: a box more costs the TMA unit as
          // much as eight rows (4096 x 14336 x 4096: 411 us with four boxes
          // of 32 rows, 389 with one of 128)
          if (x.units == C::MAX_UNITS)
            tma_load_3d_pair(sx, &tmap_x, fb, kb * C::BK, m, 0);
          else
            for (int u = 0; u < x.units; ++u)
              tma_load_3d_pair(sx + u * C::BOX_BYTES, &tmap_xu, fb, kb * C::BK, m + u * C::BOX_ROWS, 0);
          if (++s == C::STAGES) {
            s = 0;
            ph ^= 1u;
          }
        }
      }
      // drain: every issued load has landed and been read before the CTA exits
      for (int i = 0; i < C::STAGES; ++i) {
        if (!mbar_wait(empty_bar(s), ph ^ 1u, status, 0x62)) break;
        if (++s == C::STAGES) {
          s = 0;
          ph ^= 1u;
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------ MMA issuer (leader CTA)
    // all of it in lane 0: a warp-wide step per k-block idles the tensor pipe
    if (rank == 0 && elect_one()) {
      RowWalk<C> walk(g, tab_off, tab_tile);
      RowTile x;
      int s = 0, it = 0;
      u32 ph = 0;
      while (!*abort_flag && walk.next(x)) {
        const int acc = it & 1;
        const u32 d_tmem = tmem_base + acc * (C::TMEM_COLS / 2);
        if (!mbar_wait(tempty_bar(acc), ((it >> 1) & 1) ^ 1u, status, 0x63)) {
          *abort_flag = 1;
          break;
        }
        tc_fence_after();
        bool ok = true;
        // the instruction descriptor as a constant: one that varies at run time
        // is moved to uniform registers for every instruction
        auto run = [&](auto units) {
          constexpr u32 idesc = C::IDESC | (decltype(units)::value * C::UNIT >> 3) << 17;
          for (int kb = 0; kb < nkb; ++kb) {
            if (!mbar_wait(full_bar(s), ph, status, 0x64)) {
              *abort_flag = 1;
              ok = false;
              break;
            }
            tc_fence_after();
            const u32 sw = base + s * C::STAGE_BYTES, sx = sw + C::W_BYTES;
#pragma unroll
            for (int k = 0; k < C::BK / C::UMMA_K; ++k) {
              const u64 ad = C::W_MN ? smem_desc_sw128(sw + k * C::UMMA_K * 128, C::BK * 128, 1024)
                                     : smem_desc_sw128(sw + k * 32, 16, 1024);
              const u64 bd = smem_desc_sw128(sx + k * 32, 16, 1024);
              const u32 accum = (kb > 0 || k > 0) ? 1u : 0u;
              if (C::KIND == KIND_BF16)
                mma2_f16_ss(d_tmem, ad, bd, idesc, accum);
              else
                mma2_f8f6f4_ss(d_tmem, ad, bd, idesc, accum);
            }
            tc_commit_pair(empty_bar(s));
            if (++s == C::STAGES) {
              s = 0;
              ph ^= 1u;
            }
          }
        };
        if (x.units == 4)
          run(Const<4>());
        else if (x.units == 3)
          run(Const<3>());
        else if (x.units == 2)
          run(Const<2>());
        else
          run(Const<1>());
        if (!ok || *abort_flag) break;
        tc_commit_pair(tfull_bar(acc));
        ++it;
      }
      tc_commit2(mapa_cluster(drain_bar, 0));
      mbar_wait(drain_bar, 0, status, 0x65);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------ epilogue (both CTAs)
    const int q = warp & 3;            // TMEM lane quadrant this warp may access
    const int half = (warp - 2) >> 2;  // takes slices half, half + 2, ...
    const Epilogue &p = g.epi;
    unsigned char *stg = smem + C::STG_OFF + (warp - 2) * 2048;
    const u32 stg_at = base + C::STG_OFF + (warp - 2) * 2048;
    const u32 leader_tempty = mapa_cluster(tempty_bar(0), 0);
    RowWalk<C> walk(g, tab_off, tab_tile);
    RowTile x;
    int it = 0;
    while (!*abort_flag && walk.next(x)) {
      const float alpha = p.group_scale ? p.alpha * __ldcg(p.group_scale + x.grp) : p.alpha;
      const int col0 = x.n0 + rank * C::BNC + q * 32;  // the warp's columns, one per lane
      const bool live = col0 < p.cols;
      float bias[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // of columns lane / 4 + 8 i
      if (p.bias) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int col = col0 + 8 * i + (lane >> 2);
          if (col < p.cols) bias[i] = __uint_as_float(static_cast<u32>(__ldcg(p.bias + col)) << 16);
        }
      }
      uint4 res[4];
      if (p.residual && live) load_block(res, p.residual, p.cols, x.m0 + half * 32, x.row_end, col0, lane);
      const int acc = it & 1;
      bool ok = true;
      if (lane == 0) ok = mbar_wait(tfull_bar(acc), (it >> 1) & 1, status, 0x66);
      if (!__shfl_sync(0xffffffffu, ok ? 1 : 0, 0)) {
        *abort_flag = 1;
        break;
      }
      tc_fence_after();
      const u32 t_lane = tmem_base + (static_cast<u32>(q * 32) << 16) + acc * (C::TMEM_COLS / 2);
      const int slices = live ? x.units * 2 : 0;
#pragma unroll 1
      for (int i = half; i < slices; i += 2) {
        const int row0 = x.m0 + i * 32;
        if (row0 >= x.row_end) break;
        u32 lo[16], hi[16];
        tmem_ld_16x256b_x4(t_lane + i * 32, lo);
        tmem_ld_16x256b_x4(t_lane + (16u << 16) + i * 32, hi);
        tmem_wait_ld();
        float v[2][16];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          v[0][j] = fmaf(__uint_as_float(lo[j]), alpha, bias[j >> 1 & 1]);
          v[1][j] = fmaf(__uint_as_float(hi[j]), alpha, bias[2 + (j >> 1 & 1)]);
        }
        if (p.preact) {
          put_block(v, stg_at, lane);
          __syncwarp();
          store_block(stg, p.preact, p.cols, row0, x.row_end, col0, lane);
          __syncwarp();
        }
        act_forward(v[0], p.act);
        act_forward(v[1], p.act);
        if (p.residual) {
#pragma unroll
          for (int k = 0; k < 4; ++k) *staged(stg, k, lane) = res[k];
          __syncwarp();
          add_block(v, stg_at, lane);
          __syncwarp();
          load_block(res, p.residual, p.cols, row0 + 64, x.row_end, col0, lane);
        }
        put_block(v, stg_at, lane);
        __syncwarp();
        store_block(stg, p.out, p.cols, row0, x.row_end, col0, lane);
        __syncwarp();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        arrive_tmem_free(leader_tempty + 8u * acc);
      }
      ++it;
    }
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // the leader's MMAs into both TMEMs are complete
  tc_fence_after();
  if (warp == 1) tmem_dealloc<2>(tmem_base, C::TMEM_COLS);
}

// ===========================================================================
// outer_kernel
// ===========================================================================
// The weights' gradient dW[k, n] = sum over rows of X[row, k] dY[row, n], for
// all rows or per group.  A cluster of two CTAs computes 256 x 256 tiles of
// dW; CTA r holds rows k [128 r, 128 r + 128) and columns n
// [128 r, 128 r + 128) of the operands, both MN-major as they are stored, and
// owns its half's accumulator rows.  Persistent, like rows_kernel; the tiles
// of the last wave are halved in n where that fills the pairs.  Warps: 0 TMA
// producer, 1 MMA issuer (leader only), 2..9 epilogue (two warps per TMEM lane
// quadrant, each half of the tile's 64-column slices), 10 (grouped only)
// clears the rows behind a group's end.
//
// The contraction runs over a group's rows, whose count is any number, and a
// block of 64 rows that crosses the group's end also loads rows of the next
// group, or rows behind the last one, whose values (NaN among them) must not
// count.  An instruction takes 16 rows.  So the whole sixteens of the last
// block are an ordinary block of which fewer instructions are issued, and the
// last rows, fewer than 16, are a block of their own: its loads complete on a
// barrier of the CTA's own, warp 10 zeroes the lines behind the group's end in
// both operands and, once both CTAs have, releases it to the MMA thread.
// These short blocks have two slots beside the ring, are fetched first and
// used last, so that the round trip hides behind the tile's other blocks
// (8 x [500, 4096]^T [500, 4096]: 158 us with the zeroing in the ring's order,
// 128 without a remainder).
//
// A warp's 32 rows x 64 columns of the result leave through shared memory by
// TMA, in whole 128-byte lines; it clips what lies outside dW.
//
// Bound by the tensor pipe for many rows (4096 x 4096 x 14336: 95 % of active
// cycles, 328 us or 1465 TFLOP/s after a pause, 377 or 1277 back to back), by the
// operands' latency for groups of a few hundred (8 x 512 rows of 4096 x 4096: 120
// us) and by the writes of dW below (64 x 64 rows of 4096 x 1024: 117 us, 4.6
// TB/s; 16-byte stores took 286).
template <bool GROUPED_>
struct OuterCfg {
  static constexpr bool GROUPED = GROUPED_;
  static constexpr int STAGES = GROUPED ? 5 : 6;
  static constexpr int BM = 128;  // rows (k) and columns (n) per CTA
  static constexpr int BK = 64, CHUNK = 64, UMMA_K = 16;
  static constexpr int CHUNK_BYTES = BK * 128;  // 64 values by 64 rows
  static constexpr int A_BYTES = BM * 128;
  static constexpr int STAGE_BYTES = 2 * A_BYTES;
  static constexpr int SHORT_CHUNK = UMMA_K * 128;  // 64 values by 16 rows
  static constexpr int SHORT_BYTES = 4 * SHORT_CHUNK;
  static constexpr int TMEM_COLS = 512;
  static constexpr int EPI_WARPS = 8;
  static constexpr int THREADS = 32 * (2 + EPI_WARPS + (GROUPED ? 1 : 0));
  static constexpr int RASTER = 8;  // tile rows walked column by column
  static constexpr int SHORT_OFF = STAGES * STAGE_BYTES;
  static constexpr int STG_OFF = SHORT_OFF + (GROUPED ? 2 * SHORT_BYTES : 0);
  static constexpr int BAR_OFF = STG_OFF + EPI_WARPS * 4096;
  static constexpr int NBARS = 2 * STAGES + 5 + (GROUPED ? 8 : 0);
  static constexpr int TAB_OFF = BAR_OFF + NBARS * 8 + 16;
  static constexpr int TAB_BYTES = GROUPED ? (kMaxGroups + 1) * 4 : 0;
  static constexpr int SMEM_BYTES = 1024 + TAB_OFF + TAB_BYTES;
  // without the N field, which is the tile's
  static constexpr u32 IDESC = make_idesc(1u, 1u, true, true, 256, 0);
  static_assert(SMEM_BYTES <= 232448, "shared memory budget exceeded");
};

struct OuterTile {
  int m0, n0;        // first row k and column n of the tile
  int chunks;        // 64-column chunks per CTA: 2, or 1 for half a tile
  int grp;           // group, 0 when dense
  int r0;            // first row of the contraction
  int blocks, last;  // 64-row blocks, and the instructions (16 rows) of the last one
  int rest;          // rows behind them, fewer than 16 (grouped)
};

template <class C>
struct OuterWalk {
  const GemmArgs &g;
  const int *tab_off;
  int i, step, whole, items, ntm, ntn;
  bool halves;
  Raster<C::RASTER> raster;
  Divisor per_group;

  __device__ __forceinline__ OuterWalk(const GemmArgs &g_, const int *o)
      : g(g_), tab_off(o), i(blockIdx.x / 2), step(gridDim.x / 2), ntm((g_.GM + 255) / 256),
        ntn((g_.GN + 255) / 256), raster(ntn), per_group(ntm * ntn) {
    const int total = ntm * ntn * (C::GROUPED ? g.groups : 1);
    const int rest = total % step;
    whole = total - rest;
    halves = 2 * rest <= step;
    items = whole + rest * (halves ? 2 : 1);
    more = find(ahead);
  }

  OuterTile ahead;  // worked out one tile early, as in RowWalk
  bool more;
  __device__ __forceinline__ bool next(OuterTile &x) {
    if (!more) return false;
    x = ahead;
    more = find(ahead);
    return true;
  }

  __device__ __forceinline__ bool find(OuterTile &x) {
    for (; i < items; i += step) {
      int t = i, part = 0;
      x.chunks = 2;
      if (i >= whole && halves) {
        t = whole + (i - whole) / 2;
        part = (i - whole) & 1;
        x.chunks = 1;
      }
      int local = t, tm, tn;
      x.grp = C::GROUPED ? per_group(t, local) : 0;
      raster(local, ntm, tm, tn);
      x.m0 = tm * 256;
      x.n0 = tn * 256 + part * 128;
      if (x.n0 >= g.GN) continue;  // the second half of a tile that has only one
      if (x.n0 + 128 >= g.GN) x.chunks = 1;
      const int len = C::GROUPED ? tab_off[x.grp + 1] - tab_off[x.grp] : g.GK;
      x.r0 = C::GROUPED ? tab_off[x.grp] : 0;
      // dense: TMA fills the rows behind the last with zeros
      const int steps = C::GROUPED ? len / C::UMMA_K : (len + C::UMMA_K - 1) / C::UMMA_K;
      x.rest = C::GROUPED ? len % C::UMMA_K : 0;
      x.blocks = (steps + 3) / 4;
      x.last = steps - 4 * (x.blocks - 1);
      i += step;
      return true;
    }
    return false;
  }
};

template <class C>
__global__ void __launch_bounds__(C::THREADS, 1)
    outer_kernel(const __grid_constant__ TensorMap tmap_x, const __grid_constant__ TensorMap tmap_y,
                 const __grid_constant__ TensorMap tmap_x16, const __grid_constant__ TensorMap tmap_y16,
                 const __grid_constant__ TensorMap tmap_out, const GemmArgs g) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  const u32 raw = smem_u32(smem_raw);
  const u32 base = (raw + 1023u) & ~1023u;
  unsigned char *smem = smem_raw + (base - raw);
  const u32 bars = base + C::BAR_OFF;
  auto full_bar = [&](int s) { return bars + 8u * s; };
  auto empty_bar = [&](int s) { return bars + 8u * (C::STAGES + s); };
  auto tfull_bar = [&](int a) { return bars + 8u * (2 * C::STAGES + a); };
  auto tempty_bar = [&](int a) { return bars + 8u * (2 * C::STAGES + 2 + a); };
  const u32 drain_bar = bars + 8u * (2 * C::STAGES + 4);
  // of the short blocks' two slots: this CTA's loads have landed; the peer has
  // zeroed (leader's copy); both have (leader's); the MMA has read the slot
  auto short_full = [&](int b) { return bars + 8u * (2 * C::STAGES + 5 + b); };
  auto short_peer = [&](int b) { return bars + 8u * (2 * C::STAGES + 7 + b); };
  auto short_ready = [&](int b) { return bars + 8u * (2 * C::STAGES + 9 + b); };
  auto short_empty = [&](int b) { return bars + 8u * (2 * C::STAGES + 11 + b); };
  u32 *tmem_slot = reinterpret_cast<u32 *>(smem + C::BAR_OFF + C::NBARS * 8);
  volatile u32 *abort_flag = tmem_slot + 1;
  int *tab_off = reinterpret_cast<int *>(smem + C::TAB_OFF);
  u32 *status = g.epi.status;

  const int warp = threadIdx.x / 32;
  const int lane = threadIdx.x % 32;
  const u32 rank = cluster_ctarank();

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    if (C::GROUPED) {
      for (int b = 0; b < 2; ++b) {
        mbar_init(short_full(b), 1);
        mbar_init(short_peer(b), 1);
        mbar_init(short_ready(b), 1);
        mbar_init(short_empty(b), 1);
      }
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(tfull_bar(a), 1);
      mbar_init(tempty_bar(a), 2 * C::EPI_WARPS);  // both CTAs' epilogue warps, on the leader's
    }
    mbar_init(drain_bar, 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmap_x);
    tma_prefetch_desc(&tmap_y);
  }
  if (warp == 1) {
    tmem_alloc<2>(smem_u32(tmem_slot), C::TMEM_COLS);
    tmem_relinquish<2>();
  }
  if (C::GROUPED && warp == 2) {
    if (!g.wait_last) pdl_wait();  // the offsets may come from the previous kernel of the stream
    scan_groups(g.offsets, g.groups, g.rows, 256, tab_off, nullptr, blockIdx.x == 0 ? status : nullptr);
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // both CTAs' barriers are initialised before any remote use
  tc_fence_after();
  pdl_launch_dependents();
  const u32 tmem_base = *tmem_slot;
  if (!g.wait_last) pdl_wait();  // the previous kernel of the stream is complete from here on

  if (warp == 0) {
    // ------------------------------------------------ TMA producer (both CTAs)
    if (elect_one()) {
      OuterWalk<C> walk(g, tab_off);
      OuterTile x;
      const u32 leader_full = mapa_cluster(full_bar(0), 0);
      int s = 0, shorts = 0;
      u32 ph = 0;
      while (!*abort_flag && walk.next(x)) {
        const int m = x.m0 + rank * C::BM, n = x.n0 + rank * x.chunks * C::CHUNK;
        if (x.rest) {
          const int b = shorts & 1, row = x.r0 + x.blocks * C::BK - (x.blocks ? (4 - x.last) * C::UMMA_K : 0);
          if (!mbar_wait(short_empty(b), ((shorts >> 1) & 1) ^ 1u, status, 0x40)) {
            *abort_flag = 1;
            break;
          }
          ++shorts;
          const u32 sx = base + C::SHORT_OFF + b * C::SHORT_BYTES, sy = sx + 2 * C::SHORT_CHUNK;
          mbar_arrive_expect_tx(short_full(b), (2 + x.chunks) * C::SHORT_CHUNK);
          const u32 fb = mapa_cluster(short_full(b), rank);
          tma_load_3d_pair(sx, &tmap_x16, fb, m, row, 0);
          tma_load_3d_pair(sx + C::SHORT_CHUNK, &tmap_x16, fb, m + C::CHUNK, row, 0);
          tma_load_3d_pair(sy, &tmap_y16, fb, n, row, 0);
          if (x.chunks == 2) tma_load_3d_pair(sy + C::SHORT_CHUNK, &tmap_y16, fb, n + C::CHUNK, row, 0);
        }
        const u32 bytes = 2 * (C::A_BYTES + x.chunks * C::CHUNK_BYTES);
        for (int kb = 0; kb < x.blocks; ++kb) {
          if (!mbar_wait(empty_bar(s), ph ^ 1u, status, 0x41)) {
            *abort_flag = 1;
            break;
          }
          const u32 sx = base + s * C::STAGE_BYTES, sy = sx + C::A_BYTES;
          if (rank == 0) mbar_arrive_expect_tx(full_bar(s), bytes);
          const u32 fb = leader_full + 8u * s;
          const int row = x.r0 + kb * C::BK;
          tma_load_3d_pair(sx, &tmap_x, fb, m, row, 0);
          tma_load_3d_pair(sx + C::CHUNK_BYTES, &tmap_x, fb, m + C::CHUNK, row, 0);
          tma_load_3d_pair(sy, &tmap_y, fb, n, row, 0);
          if (x.chunks == 2) tma_load_3d_pair(sy + C::CHUNK_BYTES, &tmap_y, fb, n + C::CHUNK, row, 0);
          if (++s == C::STAGES) {
            s = 0;
            ph ^= 1u;
          }
        }
      }
      // drain: every issued load has landed and been read before the CTA exits
      for (int i = 0; i < C::STAGES; ++i) {
        if (!mbar_wait(empty_bar(s), ph ^ 1u, status, 0x42)) break;
        if (++s == C::STAGES) {
          s = 0;
          ph ^= 1u;
        }
      }
      for (int i = 0; C::GROUPED && i < 2; ++i, ++shorts)
        if (!mbar_wait(short_empty(shorts & 1), ((shorts >> 1) & 1) ^ 1u, status, 0x42)) break;
    }
  } else if (warp == 1) {
    // ------------------------------------------------ MMA issuer (leader CTA)
    // all of it in lane 0: a warp-wide step per k-block idles the tensor pipe
    if (rank == 0 && elect_one()) {
      OuterWalk<C> walk(g, tab_off);
      OuterTile x;
      int s = 0, it = 0, shorts = 0;
      u32 ph = 0;
      while (!*abort_flag && walk.next(x)) {
        if (x.blocks == 0 && x.rest == 0) continue;  // an empty group: the epilogue writes zeros
        const int acc = it & 1;
        const u32 d_tmem = tmem_base + acc * (C::TMEM_COLS / 2);
        if (!mbar_wait(tempty_bar(acc), ((it >> 1) & 1) ^ 1u, status, 0x43)) {
          *abort_flag = 1;
          break;
        }
        tc_fence_after();
        bool ok = true;
        auto run = [&](auto chunks) {
          constexpr u32 idesc = C::IDESC | (decltype(chunks)::value * 128 >> 3) << 17;
          for (int kb = 0; kb < x.blocks; ++kb) {
            if (!mbar_wait(full_bar(s), ph, status, 0x44)) {
              *abort_flag = 1;
              ok = false;
              return;
            }
            tc_fence_after();
            const u32 sx = base + s * C::STAGE_BYTES, sy = sx + C::A_BYTES;
            const auto mma = [&](int k) {
              mma2_f16_ss(d_tmem, smem_desc_sw128(sx + k * C::UMMA_K * 128, C::CHUNK_BYTES, 1024),
                          smem_desc_sw128(sy + k * C::UMMA_K * 128, C::CHUNK_BYTES, 1024), idesc,
                          (kb > 0 || k > 0) ? 1u : 0u);
            };
            if (kb < x.blocks - 1 || x.last == 4) {
#pragma unroll
              for (int k = 0; k < 4; ++k) mma(k);
            } else {
              for (int k = 0; k < x.last; ++k) mma(k);
            }
            tc_commit_pair(empty_bar(s));
            if (++s == C::STAGES) {
              s = 0;
              ph ^= 1u;
            }
          }
          if (x.rest) {
            const int b = shorts & 1;
            if (!mbar_wait(short_ready(b), (shorts >> 1) & 1, status, 0x49)) {
              *abort_flag = 1;
              ok = false;
              return;
            }
            ++shorts;
            tc_fence_after();
            const u32 sx = base + C::SHORT_OFF + b * C::SHORT_BYTES;
            mma2_f16_ss(d_tmem, smem_desc_sw128(sx, C::SHORT_CHUNK, 1024),
                        smem_desc_sw128(sx + 2 * C::SHORT_CHUNK, C::SHORT_CHUNK, 1024), idesc,
                        x.blocks ? 1u : 0u);
            tc_commit_pair(short_empty(b));
          }
        };
        if (x.chunks == 2)
          run(Const<2>());
        else
          run(Const<1>());
        if (!ok || *abort_flag) break;
        tc_commit_pair(tfull_bar(acc));
        ++it;
      }
      tc_commit2(mapa_cluster(drain_bar, 0));
      mbar_wait(drain_bar, 0, status, 0x45);
    }
    __syncwarp();
  } else if (C::GROUPED && warp == 2 + C::EPI_WARPS) {
    // ------------------------------------------------ rows behind a group's end
    OuterWalk<C> walk(g, tab_off);
    OuterTile x;
    int shorts = 0;
    while (!*abort_flag && walk.next(x)) {
      if (!x.rest) continue;
      const int b = shorts & 1;
      const u32 par = (shorts >> 1) & 1;
      ++shorts;
      bool ok = true;
      if (lane == 0) ok = mbar_wait(short_full(b), par, status, 0x46);
      if (!__shfl_sync(0xffffffffu, ok ? 1 : 0, 0)) {
        *abort_flag = 1;
        break;
      }
      unsigned char *at = smem + C::SHORT_OFF + b * C::SHORT_BYTES;
      for (int i = x.rest * 8 + lane; i < C::UMMA_K * 8; i += 32)
        for (int c = 0; c < 2 + x.chunks; ++c)
          *reinterpret_cast<uint4 *>(at + c * C::SHORT_CHUNK + i * 16) = make_uint4(0, 0, 0, 0);
      fence_proxy_async_smem();  // the MMA reads through the async proxy
      __syncwarp();
      if (lane == 0) {
        if (rank != 0) {
          mbar_arrive_cluster(short_peer(b), 0);
        } else {
          if (!mbar_wait(short_peer(b), par, status, 0x47)) *abort_flag = 1;
          fence_proxy_async_smem();
          mbar_arrive(short_ready(b));
        }
      }
      __syncwarp();
    }
  } else {
    // ------------------------------------------------ epilogue (both CTAs)
    const int q = warp & 3;            // TMEM lane quadrant this warp may access
    const int half = (warp - 2) >> 2;  // takes 32-column slices half, half + 2, ...
    unsigned char *stg = smem + C::STG_OFF + (warp - 2) * 4096;
    const u32 stg_at = base + C::STG_OFF + (warp - 2) * 4096;
    const u32 leader_tempty = mapa_cluster(tempty_bar(0), 0);
    OuterWalk<C> walk(g, tab_off);
    OuterTile x;
    int it = 0;
    while (!*abort_flag && walk.next(x)) {
      const bool some = x.blocks || x.rest;
      const int row0 = x.m0 + rank * C::BM + q * 32;
      const int acc = it & 1;
      if (some) {
        bool ok = true;
        if (lane == 0) ok = mbar_wait(tfull_bar(acc), (it >> 1) & 1, status, 0x48);
        if (!__shfl_sync(0xffffffffu, ok ? 1 : 0, 0)) {
          *abort_flag = 1;
          break;
        }
        tc_fence_after();
      }
      const u32 t_row = tmem_base + (static_cast<u32>(q * 32) << 16) + acc * (C::TMEM_COLS / 2);
#pragma unroll 1
      for (int i = half; i < 2 * x.chunks; i += 2) {
        const int col0 = x.n0 + 64 * i;
        if (row0 >= g.GM || col0 >= g.GN) break;
        u32 w[32];  // thread = row: 64 columns as bf16
        if (some) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            u32 r[32];
            tmem_ld_32x32b_x32(t_row + 64 * i + 32 * h, r);
            tmem_wait_ld();
#pragma unroll
            for (int j = 0; j < 16; ++j)
              w[16 * h + j] = pack_bf16x2(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1]));
          }
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) w[j] = 0u;
        }
        if (lane == 0) bulk_wait_read<0>();  // the slice before has left the staging block
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 8; ++j)
          *reinterpret_cast<uint4 *>(stg + lane * 128 + ((j ^ (lane & 7)) * 16)) =
              make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          tma_store_3d(&tmap_out, stg_at, col0, row0, x.grp);
          bulk_commit();
        }
      }
      if (some) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          arrive_tmem_free(leader_tempty + 8u * acc);
        }
        ++it;
      }
    }
    if (lane == 0) bulk_wait<0>();
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (g.wait_last) pdl_wait();
  cluster_sync();  // the leader's MMAs into both TMEMs are complete
  tc_fence_after();
  if (warp == 1) tmem_dealloc<2>(tmem_base, C::TMEM_COLS);
}

// ===========================================================================
// swap_kernel
// ===========================================================================
// out[m, n] for up to BN rows m and 128 columns n per cluster, computed as
// the transpose: the weights' 128 columns are the MMA's M dimension, the rows
// its N dimension, so a tile of few rows wastes no weight traffic.  The S
// CTAs of the cluster take equal shares of the k-blocks, which puts every SM
// (two CTAs each) on the weights' stream however few tiles there are; their
// fp32 accumulators go to their own shared memory, [row][128] floats over the
// finished pipeline stages, and each CTA sums every S-th row over the cluster
// in rank order (deterministic, no workspace in global memory) and stores it.
//
// Bound by the weights' bytes: 1 x 14336 x 4096 21.0 us (5.6 TB/s, S=2), 16 x
// 4096 x 14336 21.7 us (5.4 TB/s, S=8).  Of narrower weights by some 5 us that
// are fixed (launch, first loads, sum): 1 x 4096 x 4096 9.2 us of 5.1, 128 x
// 4096 x 4096 14.4 of 5.5.  5 to 6 stages leave room for two CTAs an SM and hold 190 KiB of loads in flight.
//
// X_MN: X is given as its transpose, [k, m] row-major.  That is the weights'
// gradient, out[k, n] = sum over rows X[row, k] dY[row, n], where it has few
// tiles and many rows to sum over.
//
// A wait that expires in one CTA (an accumulator that is not complete) is told
// to the whole cluster, which then stores nothing.
template <int KIND_, int BN_, int STAGES_, bool W_MN_, bool X_MN_, bool GROUPED_>
struct SwapCfg {
  static constexpr int KIND = KIND_, BN = BN_, STAGES = STAGES_;
  static constexpr bool W_MN = W_MN_, X_MN = X_MN_, GROUPED = GROUPED_;
  static constexpr int ELEM = KIND == KIND_BF16 ? 2 : 1;
  static constexpr int BM = 128;
  static constexpr int BK = 128 / ELEM;
  static constexpr int CHUNK = 128 / ELEM;
  static constexpr int UMMA_K = 32 / ELEM;
  static constexpr int W_BYTES = BM * 128, X_BYTES = BN * 128;
  static constexpr int STAGE_BYTES = W_BYTES + X_BYTES;
  static constexpr int TMEM_COLS = BN < 32 ? 32 : BN;
  static constexpr int THREADS = 192;
  static constexpr int BAR_OFF = STAGES * STAGE_BYTES;
  static constexpr int NBARS = 2 * STAGES + 1;
  static constexpr int TAB_OFF = BAR_OFF + NBARS * 8 + 32;
  static constexpr int TAB_BYTES = GROUPED ? (kMaxGroups + 1) * 8 : 0;
  static constexpr int SMEM_BYTES = 1024 + TAB_OFF + TAB_BYTES;
  static constexpr u32 IDESC =
      make_idesc(KIND == KIND_BF16 ? 1u : 0u, KIND == KIND_BF16 ? 1u : 0u, W_MN, X_MN, BM, BN);
  static_assert(!X_MN || BN % CHUNK == 0, "an MN-major operand is whole 128-byte lines");
  static_assert(BN * BM * 4 <= STAGES * STAGE_BYTES, "the fp32 tile overlays the stages");
  static_assert(BN % 16 == 0 && BN <= 128, "tile rows");
  // two CTAs share an SM; a third never does (tensor memory: 3 x 128 columns would still fit)
  static_assert(SMEM_BYTES <= 232448 && 3 * SMEM_BYTES > 232448, "two CTAs per SM");
};

template <class C>
__global__ void __launch_bounds__(C::THREADS)
    swap_kernel(const __grid_constant__ TensorMap tmap_w, const __grid_constant__ TensorMap tmap_x,
                const GemmArgs g) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  const u32 raw = smem_u32(smem_raw);
  const u32 base = (raw + 1023u) & ~1023u;
  unsigned char *smem = smem_raw + (base - raw);
  const u32 bars = base + C::BAR_OFF;
  auto full_bar = [&](int s) { return bars + 8u * s; };
  auto empty_bar = [&](int s) { return bars + 8u * (C::STAGES + s); };
  const u32 done_bar = bars + 8u * (2 * C::STAGES);
  u32 *tmem_slot = reinterpret_cast<u32 *>(smem + C::BAR_OFF + C::NBARS * 8);
  volatile u32 *failed = tmem_slot + 1;
  u32 *status = g.epi.status;
  int *tab_off = reinterpret_cast<int *>(smem + C::TAB_OFF);
  int *tab_tile = tab_off + kMaxGroups + 1;

  const int warp = threadIdx.x / 32;
  const int lane = threadIdx.x % 32;
  const int S = static_cast<int>(cluster_nctarank()), rank = static_cast<int>(cluster_ctarank());
  const int ntn = (g.GN + C::BM - 1) / C::BM;
  const int item = blockIdx.x / S;
  const int rt = item / ntn, n0 = (item - rt * ntn) * C::BM;  // row tile; a tile row's weights are walked in order

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    mbar_init(done_bar, 1);
    *failed = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmap_w);
    tma_prefetch_desc(&tmap_x);
  }
  if (warp == 1) {
    tmem_alloc<1>(smem_u32(tmem_slot), C::TMEM_COLS);
    tmem_relinquish<1>();
  }
  if (C::GROUPED && warp == 2) {
    pdl_wait();  // the offsets may come from the previous kernel of the stream
    scan_groups(g.offsets, g.groups, g.rows, C::BN, tab_off, tab_tile, blockIdx.x == 0 ? status : nullptr);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (!g.trigger_late) pdl_launch_dependents();
  const u32 tmem_base = *tmem_slot;

  int m0 = rt * C::BN, row_end = g.GM, grp = 0;
  bool live = true;
  if (C::GROUPED) {
    // the last group whose first tile is at or before rt (tab_tile is non-decreasing)
    live = rt < tab_tile[g.groups];
    if (live) {
      int lo = 0, hi = g.groups;  // tab_tile[lo] <= rt < tab_tile[hi]
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (tab_tile[mid] <= rt)
          lo = mid;
        else
          hi = mid;
      }
      grp = lo;
      m0 = tab_off[grp] + (rt - tab_tile[grp]) * C::BN;
      row_end = tab_off[grp + 1];
    }
  }
  const int nkb = (g.GK + C::BK - 1) / C::BK;
  const int kb0 = static_cast<int>(static_cast<long long>(nkb) * rank / S);
  const int kb1 = static_cast<int>(static_cast<long long>(nkb) * (rank + 1) / S);
  const int rows = min(C::BN, row_end - m0);

  // one thread, before the cluster meets
  auto fail = [&] {
    for (int c = 0; c < S; ++c) st_cluster_u32(mapa_cluster(smem_u32(tmem_slot + 1), c), 1);
  };

  auto load_w = [&](int s, int kb) {
    const u32 sw = base + s * C::STAGE_BYTES;
    if (C::W_MN) {
#pragma unroll
      for (int c = 0; c < C::BM / C::CHUNK; ++c)
        tma_load_3d(sw + c * C::BK * 128, &tmap_w, full_bar(s), n0 + c * C::CHUNK, kb * C::BK, grp);
    } else {
      tma_load_3d(sw, &tmap_w, full_bar(s), kb * C::BK, n0, grp);
    }
  };

  if (live) {
    if (warp == 0) {
      if (elect_one()) {
        // weights that no earlier kernel writes are fetched for the opening
        // stages while the previous kernel of the stream still runs
        int pre = 0;
        if (!C::GROUPED && g.w_static) {
          for (; pre < C::STAGES && kb0 + pre < kb1; ++pre) {
            mbar_arrive_expect_tx(full_bar(pre), C::STAGE_BYTES);
            load_w(pre, kb0 + pre);
          }
        }
        if (!g.wait_last) pdl_wait();
        if (g.trigger_late) pdl_launch_dependents();
        int s = 0;
        u32 ph = 0;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (kb - kb0 >= pre) {
            if (!mbar_wait(empty_bar(s), ph ^ 1u, status, 0x51)) break;
            mbar_arrive_expect_tx(full_bar(s), C::STAGE_BYTES);
            load_w(s, kb);
          }
          const u32 sx = base + s * C::STAGE_BYTES + C::W_BYTES;
          if (C::X_MN) {
#pragma unroll
            for (int c = 0; c < C::BN / C::CHUNK; ++c)
              tma_load_3d(sx + c * C::BK * 128, &tmap_x, full_bar(s), m0 + c * C::CHUNK, kb * C::BK, 0);
          } else {
            tma_load_3d(sx, &tmap_x, full_bar(s), kb * C::BK, m0, 0);
          }
          if (++s == C::STAGES) {
            s = 0;
            ph ^= 1u;
          }
        }
        // drain: every issued load has landed and been read before the CTA exits
        for (int i = 0; i < C::STAGES; ++i) {
          if (!mbar_wait(empty_bar(s), ph ^ 1u, status, 0x54)) break;
          if (++s == C::STAGES) {
            s = 0;
            ph ^= 1u;
          }
        }
      }
    } else if (warp == 1) {
      if (elect_one()) {
        // X comes behind the previous kernel, which may take any time: the
        // bounded wait begins only when that has ended
        if (!g.wait_last) pdl_wait();
        int s = 0;
        u32 ph = 0;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!mbar_wait(full_bar(s), ph, status, 0x52)) {
            fail();
            break;
          }
          tc_fence_after();
          const u32 sw = base + s * C::STAGE_BYTES, sx = sw + C::W_BYTES;
#pragma unroll
          for (int k = 0; k < C::BK / C::UMMA_K; ++k) {
            const u64 ad = C::W_MN ? smem_desc_sw128(sw + k * C::UMMA_K * 128, C::BK * 128, 1024)
                                   : smem_desc_sw128(sw + k * 32, 16, 1024);
            const u64 bd = C::X_MN ? smem_desc_sw128(sx + k * C::UMMA_K * 128, C::BK * 128, 1024)
                                   : smem_desc_sw128(sx + k * 32, 16, 1024);
            const u32 accum = (kb > kb0 || k > 0) ? 1u : 0u;
            if (C::KIND == KIND_BF16)
              mma_f16_ss(tmem_base, ad, bd, C::IDESC, accum);
            else
              mma_f8f6f4_ss(tmem_base, ad, bd, C::IDESC, accum);
          }
          tc_commit(empty_bar(s));
          if (++s == C::STAGES) {
            s = 0;
            ph ^= 1u;
          }
        }
        tc_commit(done_bar);
      }
    } else {
      if (!g.wait_last) pdl_wait();  // bias, residual and outputs are ordered after the previous kernel
      const int q = warp & 3;
      bool ok = true;
      if (lane == 0) {
        ok = mbar_wait(done_bar, 0, status, 0x53);
        if (!ok) fail();
      }
      ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
      tc_fence_after();
      if (ok) {
        // every load has landed and been read: the stages are free
        float *acc = reinterpret_cast<float *>(smem) + q * 32 + lane;
        const u32 t_row = tmem_base + (static_cast<u32>(q * 32) << 16);
        constexpr int CH = C::BN < 32 ? 16 : 32;
#pragma unroll 1
        for (int r0 = 0; r0 < rows; r0 += CH) {
          u32 r[CH];
          if constexpr (CH == 32)
            tmem_ld_32x32b_x32(t_row + r0, r);
          else
            tmem_ld_32x32b_x16(t_row + r0, r);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < CH; ++i)
            if (r0 + i < rows) acc[(r0 + i) * C::BM] = __uint_as_float(r[i]);
        }
      }
    }
    __syncwarp();
    tc_fence_before();
    if (S > 1)
      cluster_sync();
    else
      __syncthreads();

    if (warp >= 2 && !*failed) {
      const Epilogue &p = g.epi;
      const int col = n0 + 4 * lane;
      const float alpha = p.group_scale ? p.alpha * __ldcg(p.group_scale + grp) : p.alpha;
      float4 bias = make_float4(0.f, 0.f, 0.f, 0.f);
      if (p.bias && col < p.cols) {
        const uint2 w = __ldcg(reinterpret_cast<const uint2 *>(p.bias + col));
        bias = make_float4(bf16_lo(w.x), bf16_hi(w.x), bf16_lo(w.y), bf16_hi(w.y));
      }
      for (int r = rank + S * (warp - 2); r < rows; r += 4 * S) {
        const long long off = static_cast<long long>(m0 + r) * p.cols + col;
        const u32 at = base + (r * C::BM + 4 * lane) * 4;
        uint2 res = make_uint2(0, 0);
        if (p.residual && col < p.cols) res = __ldcg(reinterpret_cast<const uint2 *>(p.residual + off));
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        if (S > 1) {
          for (int c = 0; c < S; ++c) {
            const float4 w = ld_cluster_v4(mapa_cluster(at, c));
            v[0] += w.x;
            v[1] += w.y;
            v[2] += w.z;
            v[3] += w.w;
          }
        } else {
          const float4 w = *reinterpret_cast<const float4 *>(smem + (r * C::BM + 4 * lane) * 4);
          v[0] = w.x;
          v[1] = w.y;
          v[2] = w.z;
          v[3] = w.w;
        }
        v[0] = v[0] * alpha + bias.x;
        v[1] = v[1] * alpha + bias.y;
        v[2] = v[2] * alpha + bias.z;
        v[3] = v[3] * alpha + bias.w;
        if (p.preact && col < p.cols)
          *reinterpret_cast<uint2 *>(p.preact + off) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
        act_forward(v, p.act);
        v[0] += bf16_lo(res.x);
        v[1] += bf16_hi(res.x);
        v[2] += bf16_lo(res.y);
        v[3] += bf16_hi(res.y);
        if (col < p.cols)
          *reinterpret_cast<uint2 *>(p.out + off) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
      }
    }
    __syncwarp();
    if (S > 1) cluster_sync();  // no CTA leaves while another still reads its tile
  }
  __syncthreads();
  tc_fence_after();
  if (g.wait_last) pdl_wait();
  if (warp == 1) tmem_dealloc<1>(tmem_base, C::TMEM_COLS);
}

// ===========================================================================
// slope_kernel
// ===========================================================================
// dpre = dout * act'(preact), and/or the column sums of dpre (before its
// rounding) over all rows.  A block owns 8 LANES columns and every `split`-th
// block of rows: LANES threads cover a row's 16 LANES bytes.  For the sums the
// `split` blocks of a column stripe are a cluster, of at most eight: a
// thread's eight column sums meet in shared memory and then over the cluster,
// in a fixed order.  The fewer columns there are, the narrower the stripes, so
// that the blocks fill the GPU.
//
// Bound by its traffic, with about as many instructions to issue: 4096 x 14336
// with gelu and the sums 62-70 us (5.0-5.6 TB/s), 4096 x 4096 with silu 18-20 us
// (5.1-5.6 TB/s).
struct SlopeArgs {
  const unsigned short *dout, *preact;
  unsigned short *dpre;
  float *dbias;
  int rows, cols, act, split;
  const int *offsets;  // grouped: rows [offsets[0], offsets[groups]) only
  int groups;
};

constexpr int kSlopeThreads = 256;

// BENT: there is an activation, and dpre is written.
template <int LANES, bool BENT>
__global__ void __launch_bounds__(kSlopeThreads, 4) slope_kernel(const SlopeArgs a) {
  constexpr int ROWS = kSlopeThreads / LANES, COLS = 8 * LANES;
  constexpr int U = BENT ? 2 : 4;  // rows in flight per thread: 64 bytes either way
  __shared__ float part[kSlopeThreads / 32][COLS];
  __shared__ int last;
  const int tid = threadIdx.x, lane = tid % LANES;
  const int stripe = blockIdx.x / a.split, rank = blockIdx.x - stripe * a.split;
  const int col = stripe * COLS + lane * 8;
  pdl_launch_dependents();
  pdl_wait();
  int lo = 0, hi = a.rows;
  if (a.offsets) {
    // the last group ends at the largest clamped offset
    if (tid == 0) last = 0;
    __syncthreads();
    for (int i = tid; i <= a.groups; i += kSlopeThreads) atomicMax(&last, min(__ldcg(a.offsets + i), a.rows));
    __syncthreads();
    lo = max(0, min(__ldcg(a.offsets), a.rows));
    hi = last;
  }
  float acc[8] = {};
  if (col < a.cols) {
    const int stride = ROWS * a.split;
    for (int row = lo + rank * ROWS + tid / LANES; row < hi; row += U * stride) {
      uint4 d[U], z[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int r = row + u * stride;
        const long long off = static_cast<long long>(r) * a.cols + col;
        d[u] = z[u] = make_uint4(0, 0, 0, 0);
        if (r < hi) {
          d[u] = __ldcg(reinterpret_cast<const uint4 *>(a.dout + off));
          if (BENT) z[u] = __ldcg(reinterpret_cast<const uint4 *>(a.preact + off));
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int r = row + u * stride;
        if (r >= hi) break;
        const u32 dw[4] = {d[u].x, d[u].y, d[u].z, d[u].w}, zw[4] = {z[u].x, z[u].y, z[u].z, z[u].w};
        float x[8], y[8];
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          x[2 * h] = bf16_lo(dw[h]);
          x[2 * h + 1] = bf16_hi(dw[h]);
          y[2 * h] = bf16_lo(zw[h]);
          y[2 * h + 1] = bf16_hi(zw[h]);
        }
        if (BENT) {
          act_backward(x, y, a.act);
          st_global_v4(a.dpre + static_cast<long long>(r) * a.cols + col, pack_bf16x2(x[0], x[1]),
                       pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] += x[i];
      }
    }
  }
  if (!a.dbias) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
#pragma unroll
    for (int m = LANES; m < 32; m <<= 1) acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], m);  // the warp's rows
    if ((tid & 31) < LANES) part[tid >> 5][lane * 8 + i] = acc[i];
  }
  __syncthreads();
  if (tid < COLS) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < kSlopeThreads / 32; ++i) s += part[i][tid];
    part[0][tid] = s;
  }
  __syncthreads();
  if (a.split > 1) cluster_sync();
  if (rank == 0 && tid < COLS) {
    float s = part[0][tid];
    for (int c = 1; c < a.split; ++c) s += ld_cluster_f32(mapa_cluster(smem_u32(&part[0][tid]), c));
    const int n = stripe * COLS + tid;
    if (n < a.cols) a.dbias[n] = s;
  }
  __syncwarp();
  if (a.split > 1) cluster_sync();
}

}  // namespace lin
}  // namespace thork
