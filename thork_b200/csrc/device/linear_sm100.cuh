// linear_sm100.cuh — the linear-layer kernels for sm_100a: matrix products
// with bias, activation and residual in the epilogue, and the same products
// grouped by expert with ragged sizes, forward and backward.
//
//   pair_kernel   persistent CTA pairs (tcgen05 cta_group::2), 256 x BN tiles:
//                 the tensor-bound products (many rows; both gradients)
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
// what the product's groups divide: nothing, the output's rows, or the contraction
enum : int { DENSE = 0, GROUP_ROWS = 1, GROUP_K = 2 };

constexpr int kMaxGroups = 1024;

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
  int GM, GN, GK;      // extents of the (per-group) product; GROUP_ROWS: GM = buffer rows
  const int *offsets;  // [groups + 1] row offsets, or null
  int groups, rows;    // groups, rows of the buffer that the offsets divide
  int w_static;        // swap_kernel: no earlier launch writes the weights
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

__device__ __forceinline__ float bf16_lo(u32 w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(u32 w) { return __uint_as_float(w & 0xFFFF0000u); }

// ---------------------------------------------------------------- activations
// gelu_tanh is written z * sigmoid(2u), silu z * sigmoid(z): one exponential
// and one division each, with a relative error of a few 2^-22, far below the
// bf16 rounding of the output.  A NaN stays a NaN (relu included).
__device__ __forceinline__ float gelu_tanh_2u(float z) {
  return 1.5957691216057308f * z * (1.0f + 0.044715f * z * z);
}

template <int N>
__device__ __forceinline__ void act_forward(float (&v)[N], int act) {
  if (act == ACT_RELU) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = v[i] <= 0.0f ? 0.0f : v[i];
  } else if (act == ACT_GELU) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = 0.5f * v[i] * (1.0f + erff(v[i] * 0.7071067811865476f));
  } else if (act == ACT_GELU_TANH) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = __fdividef(v[i], 1.0f + __expf(-gelu_tanh_2u(v[i])));
  } else if (act == ACT_SILU) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = __fdividef(v[i], 1.0f + __expf(-v[i]));
  }
}

// Derivative of the activation at z.
__device__ __forceinline__ float act_slope(float z, int act) {
  if (act == ACT_RELU) return z > 0.0f ? 1.0f : 0.0f;
  if (act == ACT_GELU) {
    const float cdf = 0.5f * (1.0f + erff(z * 0.7071067811865476f));
    return cdf + z * 0.3989422804014327f * expf(-0.5f * z * z);
  }
  if (act == ACT_GELU_TANH) {
    const float p = 1.0f / (1.0f + expf(-gelu_tanh_2u(z)));
    // d(2u)/dz = 2 sqrt(2/pi) (1 + 3 * 0.044715 z^2)
    return p + z * p * (1.0f - p) * 1.5957691216057308f * (1.0f + 0.134145f * z * z);
  }
  if (act == ACT_SILU) {
    const float p = 1.0f / (1.0f + expf(-z));
    return p * (1.0f + z * (1.0f - p));
  }
  return 1.0f;
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
    const int raw = i <= groups ? offsets[i] : 0;
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
// pair_kernel
// ===========================================================================
// A cluster of two CTAs computes 256 x BN tiles; CTA r holds rows
// [128 r, 128 r + 128) of the A tile and columns [BN/2 r, BN/2 (r + 1)) of the
// B tile, and owns the tile's accumulator rows of its half.  Warps: 0 TMA
// producer, 1 MMA issuer (leader only), 2..9 epilogue (two warps per TMEM
// lane quadrant, each half of the tile's 64-column slices), 10 (GROUP_K
// only) zeroes the rows behind a group's end in its last k-block.
//
// GROUP_K needs that because the contraction runs over a group's rows, whose
// count is any number: the last k-block also loads rows of the next group, or
// rows behind the last one, whose values (NaN among them) must not count.
// Those rows are whole 128-byte lines of both MN-major operands.  Such a
// block's loads complete on a barrier of the CTA's own; warp 10 zeroes the
// lines and, once both CTAs have, releases the block to the MMA thread.
template <int KIND_, int BN_, int STAGES_, bool A_MN_, bool B_MN_, int MODE_>
struct PairCfg {
  static constexpr int KIND = KIND_, BN = BN_, STAGES = STAGES_, MODE = MODE_;
  static constexpr bool A_MN = A_MN_, B_MN = B_MN_;
  static constexpr int ELEM = KIND == KIND_BF16 ? 2 : 1;
  static constexpr int BM = 128;  // rows per CTA
  static constexpr int BNH = BN / 2;
  static constexpr int BK = 128 / ELEM;
  static constexpr int CHUNK = 128 / ELEM;  // MN elements per 128-byte line
  static constexpr int UMMA_K = 32 / ELEM;
  static constexpr int A_BYTES = BM * 128, B_BYTES = BNH * 128;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int TMEM_COLS = 2 * BN;
  static constexpr int EPI_WARPS = 8;
  static constexpr int THREADS = 32 * (2 + EPI_WARPS + (MODE == GROUP_K ? 1 : 0));
  static constexpr int GROUP_M = 8;  // pair-tile rows per raster group
  // shared memory: stages | staging (4 KiB per epilogue warp) | barriers | group table
  static constexpr int STG_OFF = STAGES * STAGE_BYTES;
  static constexpr int BAR_OFF = STG_OFF + EPI_WARPS * 4096;
  static constexpr int NBARS = 2 * STAGES + 5 + (MODE == GROUP_K ? 2 * STAGES : 0);
  static constexpr int TAB_OFF = BAR_OFF + NBARS * 8 + 16;
  static constexpr int TAB_BYTES =
      MODE == DENSE ? 0 : (kMaxGroups + 1) * 4 * (MODE == GROUP_ROWS ? 2 : 1);
  static constexpr int SMEM_BYTES = 1024 + TAB_OFF + TAB_BYTES;
  static constexpr u32 IDESC =
      make_idesc(KIND == KIND_BF16 ? 1u : 0u, KIND == KIND_BF16 ? 1u : 0u, A_MN, B_MN, 256, BN);
  static_assert(BN == 256 || BN == 128, "whole 64-column slices for both epilogue halves");
  static_assert(!B_MN || BNH % CHUNK == 0, "per-CTA B columns are whole 128-byte lines");
  static_assert(SMEM_BYTES <= 232448, "shared memory budget exceeded");
};

struct Tile {
  int m0, n0;     // first output row (of the pair) and column
  int row_end;    // rows from here on belong to another group
  int grp;        // group, 0 when dense
  int k0;         // GROUP_K: first row of the contraction
  int nkb, tail;  // k-blocks; GROUP_K: valid rows of the last one, 0 when whole
};

// The pair's tiles in order; every role walks the same sequence.
template <class C>
struct Walk {
  const GemmArgs &g;
  const int *tab_off, *tab_tile;
  int t, step, total, grp, ntn;

  __device__ __forceinline__ Walk(const GemmArgs &g_, const int *o, const int *tl)
      : g(g_), tab_off(o), tab_tile(tl), t(blockIdx.x / 2), step(gridDim.x / 2), grp(0) {
    ntn = (g.GN + C::BN - 1) / C::BN;
    const int ntm = (g.GM + 255) / 256;
    total = C::MODE == GROUP_ROWS ? tab_tile[g.groups] * ntn
                                  : ntm * ntn * (C::MODE == GROUP_K ? g.groups : 1);
  }

  // raster: groups of GROUP_M tile rows walked column by column, so that the
  // tiles in flight share operand panels in L2
  __device__ __forceinline__ void raster(int local, int ntm, Tile &x) const {
    const int per = C::GROUP_M * ntn;
    const int q = local / per, first = q * C::GROUP_M, r = local - q * per;
    const int rows = min(ntm - first, C::GROUP_M);
    x.m0 = (first + r % rows) * 256;
    x.n0 = r / rows * C::BN;
  }

  __device__ __forceinline__ bool next(Tile &x) {
    if (t >= total) return false;
    if (C::MODE == GROUP_ROWS) {
      while (t >= tab_tile[grp + 1] * ntn) ++grp;
      const int first = tab_tile[grp];
      raster(t - first * ntn, tab_tile[grp + 1] - first, x);
      x.m0 += tab_off[grp];
      x.row_end = tab_off[grp + 1];
      x.grp = grp;
    } else {
      const int ntm = (g.GM + 255) / 256;
      x.grp = C::MODE == GROUP_K ? t / (ntm * ntn) : 0;
      raster(t - x.grp * ntm * ntn, ntm, x);
      x.row_end = g.GM;
    }
    if (C::MODE == GROUP_K) {
      x.k0 = tab_off[x.grp];
      const int len = tab_off[x.grp + 1] - x.k0;
      x.nkb = (len + C::BK - 1) / C::BK;
      x.tail = len % C::BK;
    } else {
      x.k0 = 0;
      x.nkb = (g.GK + C::BK - 1) / C::BK;
      x.tail = 0;
    }
    t += step;
    return true;
  }
};

// One warp's 32 accumulator rows x 64 columns of residual, 16 bytes per lane
// and step: lane covers chunk lane % 8 of row 4 it + lane / 8.
__device__ __forceinline__ void load_residual(uint4 (&res)[8], const Epilogue &p, int row0, int row_end,
                                              int col0, int lane) {
  const int col = col0 + (lane & 7) * 8;
#pragma unroll
  for (int it = 0; it < 8; ++it) {
    const int row = row0 + 4 * it + (lane >> 3);
    res[it] = make_uint4(0, 0, 0, 0);
    if (row < row_end && col < p.cols)
      // an ordinary load: out may be the residual itself
      res[it] = *reinterpret_cast<const uint4 *>(p.residual + static_cast<long long>(row) * p.cols + col);
  }
}

__device__ __forceinline__ void store_slice(const unsigned char *stg, unsigned short *out, int cols,
                                            int row0, int row_end, int col0, int lane) {
  const int chunk = lane & 7, col = col0 + chunk * 8;
#pragma unroll
  for (int it = 0; it < 8; ++it) {
    const int r = 4 * it + (lane >> 3), row = row0 + r;
    const uint4 v = *reinterpret_cast<const uint4 *>(stg + r * 128 + ((chunk ^ (r & 7)) * 16));
    if (row < row_end && col < cols)
      st_global_v4(out + static_cast<long long>(row) * cols + col, v.x, v.y, v.z, v.w);
  }
}

// Epilogue of 32 rows x 64 columns (TMEM lanes of t_row, or zeros).  Thread =
// row: the accumulator arrives with a row's columns in one thread, and leaves
// through this warp's 4 KiB staging slice (row = lane, 16-byte chunks XOR the
// row, so both directions are free of bank conflicts) as whole 128-byte
// lines.  The residual takes the same way in: loaded in whole lines, laid
// into the slice, picked up by the row's thread and added in fp32.
__device__ __forceinline__ void epilogue_slice(const Epilogue &p, u32 t_row, bool zero, float alpha,
                                               int row0, int row_end, int col0,
                                               const uint4 (&res)[8], unsigned char *stg, int lane) {
  float v[64];
  if (zero) {
#pragma unroll
    for (int i = 0; i < 64; ++i) v[i] = 0.0f;
  } else {
    u32 a[32], b[32];
    tmem_ld_32x32b_x32(t_row, a);
    tmem_ld_32x32b_x32(t_row + 32, b);
    tmem_wait_ld();
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      v[i] = __uint_as_float(a[i]) * alpha;
      v[32 + i] = __uint_as_float(b[i]) * alpha;
    }
  }
  if (p.bias) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      // cols is a multiple of 8, so an 8-column piece is wholly in or out
      const int col = col0 + 8 * j;
      if (col < p.cols) {
        const uint4 w = __ldg(reinterpret_cast<const uint4 *>(p.bias + col));
        const u32 x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          v[8 * j + 2 * h] += bf16_lo(x[h]);
          v[8 * j + 2 * h + 1] += bf16_hi(x[h]);
        }
      }
    }
  }
  auto slot = [&](int j) { return reinterpret_cast<uint4 *>(stg + lane * 128 + ((j ^ (lane & 7)) * 16)); };
  auto put = [&] {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      *slot(j) = make_uint4(pack_bf16x2(v[8 * j], v[8 * j + 1]), pack_bf16x2(v[8 * j + 2], v[8 * j + 3]),
                            pack_bf16x2(v[8 * j + 4], v[8 * j + 5]), pack_bf16x2(v[8 * j + 6], v[8 * j + 7]));
  };
  if (p.preact) {
    put();
    __syncwarp();
    store_slice(stg, p.preact, p.cols, row0, row_end, col0, lane);
    __syncwarp();
  }
  if (p.residual) {
#pragma unroll
    for (int it = 0; it < 8; ++it) {
      const int r = 4 * it + (lane >> 3);
      *reinterpret_cast<uint4 *>(stg + r * 128 + (((lane & 7) ^ (r & 7)) * 16)) = res[it];
    }
  }
  act_forward(v, p.act);
  if (p.residual) {
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint4 w = *slot(j);
      const u32 x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        v[8 * j + 2 * h] += bf16_lo(x[h]);
        v[8 * j + 2 * h + 1] += bf16_hi(x[h]);
      }
    }
  }
  put();  // a row's chunks are read and written by its own thread alone
  __syncwarp();
  store_slice(stg, p.out, p.cols, row0, row_end, col0, lane);
  __syncwarp();
}

template <class C>
__global__ void __launch_bounds__(C::THREADS, 1)
    pair_kernel(const __grid_constant__ TensorMap tmap_a, const __grid_constant__ TensorMap tmap_b,
                const GemmArgs g) {
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
  auto tail_bar = [&](int s) { return bars + 8u * (2 * C::STAGES + 5 + s); };   // this CTA's loads landed
  auto fixed_bar = [&](int s) { return bars + 8u * (3 * C::STAGES + 5 + s); };  // leader: the peer has zeroed
  u32 *tmem_slot = reinterpret_cast<u32 *>(smem + C::BAR_OFF + C::NBARS * 8);
  volatile u32 *abort_flag = tmem_slot + 1;
  int *tab_off = reinterpret_cast<int *>(smem + C::TAB_OFF);
  int *tab_tile = C::MODE == GROUP_ROWS ? tab_off + kMaxGroups + 1 : nullptr;
  u32 *status = g.epi.status;

  const int warp = threadIdx.x / 32;
  const int lane = threadIdx.x % 32;
  const u32 rank = cluster_ctarank();

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
      if (C::MODE == GROUP_K) {
        mbar_init(tail_bar(s), 1);
        mbar_init(fixed_bar(s), 1);
      }
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(tfull_bar(a), 1);
      mbar_init(tempty_bar(a), 2 * C::EPI_WARPS);  // both CTAs' epilogue warps, on the leader's
    }
    mbar_init(drain_bar, 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmap_a);
    tma_prefetch_desc(&tmap_b);
  }
  if (warp == 1) {
    tmem_alloc<2>(smem_u32(tmem_slot), C::TMEM_COLS);
    tmem_relinquish<2>();
  }
  if (C::MODE != DENSE && warp == 2) {
    pdl_wait();  // the offsets may come from the previous kernel of the stream
    scan_groups(g.offsets, g.groups, g.rows, 256, tab_off, tab_tile, blockIdx.x == 0 ? status : nullptr);
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // both CTAs' barriers are initialised before any remote use
  tc_fence_after();
  pdl_launch_dependents();
  const u32 tmem_base = *tmem_slot;
  pdl_wait();  // the previous kernel of the stream is complete from here on

  if (warp == 0) {
    // ------------------------------------------------ TMA producer (both CTAs)
    if (lane == 0) {
      Walk<C> walk(g, tab_off, tab_tile);
      Tile x;
      int s = 0;
      u32 ph = 0;
      while (!*abort_flag && walk.next(x)) {
        const int am = x.m0 + rank * C::BM, bn = x.n0 + rank * C::BNH;
        for (int kb = 0; kb < x.nkb; ++kb) {
          if (!mbar_wait(empty_bar(s), ph ^ 1u, status, 0x41)) {
            *abort_flag = 1;
            break;
          }
          const u32 sa = base + s * C::STAGE_BYTES, sb = sa + C::A_BYTES;
          u32 fb;
          if (C::MODE == GROUP_K && x.tail && kb == x.nkb - 1) {
            fb = tail_bar(s);
            mbar_arrive_expect_tx(fb, C::STAGE_BYTES);
            fb = mapa_cluster(fb, rank);
          } else {
            if (rank == 0) mbar_arrive_expect_tx(full_bar(s), 2 * C::STAGE_BYTES);
            fb = mapa_cluster(full_bar(s), 0);
          }
          const int k = x.k0 + kb * C::BK;
          if (C::A_MN) {
#pragma unroll
            for (int c = 0; c < C::BM / C::CHUNK; ++c)
              tma_load_3d_pair(sa + c * C::BK * 128, &tmap_a, fb, am + c * C::CHUNK, k, 0);
          } else {
            tma_load_3d_pair(sa, &tmap_a, fb, k, am, 0);
          }
          const int z = C::MODE == GROUP_ROWS ? x.grp : 0;
          if (C::B_MN) {
#pragma unroll
            for (int c = 0; c < C::BNH / C::CHUNK; ++c)
              tma_load_3d_pair(sb + c * C::BK * 128, &tmap_b, fb, bn + c * C::CHUNK, k, z);
          } else {
            tma_load_3d_pair(sb, &tmap_b, fb, k, bn, z);
          }
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
    }
  } else if (warp == 1) {
    // ------------------------------------------------ MMA issuer (leader CTA)
    // all of it in lane 0: a warp-wide step per k-block idles the tensor pipe
    if (rank == 0 && lane == 0) {
      Walk<C> walk(g, tab_off, tab_tile);
      Tile x;
      int s = 0, it = 0;
      u32 ph = 0;
      while (!*abort_flag && walk.next(x)) {
        if (x.nkb == 0) continue;  // an empty group's gradient: the epilogue writes zeros
        const int acc = it & 1;
        const u32 d_tmem = tmem_base + acc * C::BN;
        if (!mbar_wait(tempty_bar(acc), ((it >> 1) & 1) ^ 1u, status, 0x43)) {
          *abort_flag = 1;
          break;
        }
        tc_fence_after();
        bool ok = true;
        for (int kb = 0; kb < x.nkb; ++kb) {
          if (!mbar_wait(full_bar(s), ph, status, 0x44)) {
            *abort_flag = 1;
            ok = false;
            break;
          }
          tc_fence_after();
          const u32 sa = base + s * C::STAGE_BYTES, sb = sa + C::A_BYTES;
#pragma unroll
          for (int k = 0; k < C::BK / C::UMMA_K; ++k) {
            const u64 ad = C::A_MN ? smem_desc_sw128(sa + k * C::UMMA_K * 128, C::BK * 128, 1024)
                                   : smem_desc_sw128(sa + k * 32, 16, 1024);
            const u64 bd = C::B_MN ? smem_desc_sw128(sb + k * C::UMMA_K * 128, C::BK * 128, 1024)
                                   : smem_desc_sw128(sb + k * 32, 16, 1024);
            const u32 accum = (kb > 0 || k > 0) ? 1u : 0u;
            if (C::KIND == KIND_BF16)
              mma2_f16_ss(d_tmem, ad, bd, C::IDESC, accum);
            else
              mma2_f8f6f4_ss(d_tmem, ad, bd, C::IDESC, accum);
          }
          tc_commit2(mapa_cluster(empty_bar(s), 0));
          tc_commit2(mapa_cluster(empty_bar(s), 1));
          if (++s == C::STAGES) {
            s = 0;
            ph ^= 1u;
          }
        }
        if (!ok || *abort_flag) break;
        tc_commit2(mapa_cluster(tfull_bar(acc), 0));
        tc_commit2(mapa_cluster(tfull_bar(acc), 1));
        ++it;
      }
      tc_commit2(mapa_cluster(drain_bar, 0));
      mbar_wait(drain_bar, 0, status, 0x45);
    }
    __syncwarp();
  } else if (C::MODE == GROUP_K && warp == 2 + C::EPI_WARPS) {
    // ------------------------------------------------ rows behind a group's end
    Walk<C> walk(g, tab_off, tab_tile);
    Tile x;
    int s = 0;
    u32 uses = 0;  // bit s: parity of the next use of stage s's tail barriers
    while (!*abort_flag && walk.next(x)) {
      if (x.nkb == 0) continue;
      s = (s + x.nkb - 1) % C::STAGES;  // the last k-block's stage
      if (x.tail) {
        const u32 par = (uses >> s) & 1u;
        uses ^= 1u << s;
        bool ok = true;
        if (lane == 0) ok = mbar_wait(tail_bar(s), par, status, 0x46);
        if (!__shfl_sync(0xffffffffu, ok ? 1 : 0, 0)) {
          *abort_flag = 1;
          break;
        }
        constexpr int LINES = C::STAGE_BYTES / 128 / C::BK;  // 128-byte columns of A and B
        unsigned char *st = smem + s * C::STAGE_BYTES;
        for (int i = x.tail * 8 + lane; i < C::BK * 8; i += 32) {
#pragma unroll
          for (int c = 0; c < LINES; ++c)
            *reinterpret_cast<uint4 *>(st + c * C::BK * 128 + i * 16) = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_smem();  // the MMA reads through the async proxy
        __syncwarp();
        if (lane == 0) {
          if (rank != 0) {
            mbar_arrive_cluster(fixed_bar(s), 0);
          } else {
            if (!mbar_wait(fixed_bar(s), par, status, 0x47)) *abort_flag = 1;
            fence_proxy_async_smem();
            mbar_arrive(full_bar(s));
          }
        }
        __syncwarp();
      }
      s = (s + 1) % C::STAGES;
    }
  } else {
    // ------------------------------------------------ epilogue (both CTAs)
    const int q = warp & 3;            // TMEM lane quadrant this warp may access
    const int half = (warp - 2) >> 2;  // which half of the tile's columns
    constexpr int SLICES = C::BN / 128;
    unsigned char *stg = smem + C::STG_OFF + (warp - 2) * 4096;
    Walk<C> walk(g, tab_off, tab_tile);
    Tile x;
    int it = 0;
    while (!*abort_flag && walk.next(x)) {
      Epilogue p = g.epi;
      if (C::MODE == GROUP_K) p.out += static_cast<long long>(x.grp) * g.GM * g.GN;
      const float alpha = p.group_scale ? p.alpha * __ldg(p.group_scale + x.grp) : p.alpha;
      const int row0 = x.m0 + rank * C::BM + q * 32;
      const int c0 = half * SLICES * 64;
      uint4 res[8];
      if (p.residual) load_residual(res, p, row0, x.row_end, x.n0 + c0, lane);
      const int acc = it & 1;
      if (x.nkb) {
        bool ok = true;
        if (lane == 0) ok = mbar_wait(tfull_bar(acc), (it >> 1) & 1, status, 0x48);
        if (!__shfl_sync(0xffffffffu, ok ? 1 : 0, 0)) {
          *abort_flag = 1;
          break;
        }
        tc_fence_after();
      }
      const u32 t_row = tmem_base + (static_cast<u32>(q * 32) << 16) + acc * C::BN + c0;
#pragma unroll 1
      for (int i = 0; i < SLICES; ++i) {
        if (row0 < x.row_end && x.n0 + c0 + 64 * i < p.cols)
          epilogue_slice(p, t_row + 64 * i, x.nkb == 0, alpha, row0, x.row_end, x.n0 + c0 + 64 * i, res,
                         stg, lane);
        if (p.residual && i + 1 < SLICES)
          load_residual(res, p, row0, x.row_end, x.n0 + c0 + 64 * (i + 1), lane);
      }
      if (x.nkb) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (rank == 0)
            mbar_arrive(tempty_bar(acc));
          else
            mbar_arrive_cluster(tempty_bar(acc), 0);
        }
        ++it;
      }
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
template <int KIND_, int BN_, int STAGES_, bool W_MN_, bool GROUPED_>
struct SwapCfg {
  static constexpr int KIND = KIND_, BN = BN_, STAGES = STAGES_;
  static constexpr bool W_MN = W_MN_, GROUPED = GROUPED_;
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
      make_idesc(KIND == KIND_BF16 ? 1u : 0u, KIND == KIND_BF16 ? 1u : 0u, W_MN, false, BM, BN);
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
  pdl_launch_dependents();
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
      if (lane == 0) {
        // weights that no earlier kernel writes are fetched for the opening
        // stages while the previous kernel of the stream still runs
        int pre = 0;
        if (!C::GROUPED && g.w_static) {
          for (; pre < C::STAGES && kb0 + pre < kb1; ++pre) {
            mbar_arrive_expect_tx(full_bar(pre), C::STAGE_BYTES);
            load_w(pre, kb0 + pre);
          }
        }
        pdl_wait();
        int s = 0;
        u32 ph = 0;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (kb - kb0 >= pre) {
            if (!mbar_wait(empty_bar(s), ph ^ 1u, status, 0x51)) break;
            mbar_arrive_expect_tx(full_bar(s), C::STAGE_BYTES);
            load_w(s, kb);
          }
          tma_load_3d(base + s * C::STAGE_BYTES + C::W_BYTES, &tmap_x, full_bar(s), kb * C::BK, m0, 0);
          if (++s == C::STAGES) {
            s = 0;
            ph ^= 1u;
          }
        }
      }
    } else if (warp == 1) {
      if (lane == 0) {
        int s = 0;
        u32 ph = 0;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!mbar_wait(full_bar(s), ph, status, 0x52)) break;
          tc_fence_after();
          const u32 sw = base + s * C::STAGE_BYTES, sx = sw + C::W_BYTES;
#pragma unroll
          for (int k = 0; k < C::BK / C::UMMA_K; ++k) {
            const u64 ad = C::W_MN ? smem_desc_sw128(sw + k * C::UMMA_K * 128, C::BK * 128, 1024)
                                   : smem_desc_sw128(sw + k * 32, 16, 1024);
            const u64 bd = smem_desc_sw128(sx + k * 32, 16, 1024);
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
      pdl_wait();  // bias, residual and outputs are ordered after the previous kernel
      const int q = warp & 3;
      bool ok = true;
      if (lane == 0) ok = mbar_wait(done_bar, 0, status, 0x53);
      ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
      tc_fence_after();
      if (ok) {
        // every load has landed and been read: the stages are free
        float *acc = reinterpret_cast<float *>(smem) + q * 32 + lane;
        const u32 t_row = tmem_base + (static_cast<u32>(q * 32) << 16);
#pragma unroll 1
        for (int r0 = 0; r0 < rows; r0 += 16) {
          u32 r[16];
          tmem_ld_32x32b_x16(t_row + r0, r);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 16; ++i)
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

    if (warp >= 2) {
      const Epilogue &p = g.epi;
      const int col = n0 + 4 * lane;
      const float alpha = p.group_scale ? p.alpha * __ldg(p.group_scale + grp) : p.alpha;
      float4 bias = make_float4(0.f, 0.f, 0.f, 0.f);
      if (p.bias && col < p.cols) {
        const uint2 w = __ldg(reinterpret_cast<const uint2 *>(p.bias + col));
        bias = make_float4(bf16_lo(w.x), bf16_hi(w.x), bf16_lo(w.y), bf16_hi(w.y));
      }
      for (int r = rank + S * (warp - 2); r < rows; r += 4 * S) {
        const long long off = static_cast<long long>(m0 + r) * p.cols + col;
        const u32 at = base + (r * C::BM + 4 * lane) * 4;
        uint2 res = make_uint2(0, 0);
        if (p.residual && col < p.cols) res = *reinterpret_cast<const uint2 *>(p.residual + off);
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
  if (warp == 1) tmem_dealloc<1>(tmem_base, C::TMEM_COLS);
}

// ===========================================================================
// slope_kernel
// ===========================================================================
// dpre = dout * act'(preact), and/or the column sums of dpre (before its
// rounding) over all rows.  A cluster of CTAs owns 128 columns: 16 threads
// cover a row's 256 bytes, each CTA every R-th block of 16 rows; a thread's
// eight column sums meet in shared memory and then over the cluster, in a
// fixed order.
struct SlopeArgs {
  const unsigned short *dout, *preact;
  unsigned short *dpre;
  float *dbias;
  int rows, cols, act;
  const int *offsets;  // grouped: rows [offsets[0], offsets[groups]) only
  int groups;
};

__global__ void __launch_bounds__(256) slope_kernel(const SlopeArgs a) {
  __shared__ float part[16][128];
  __shared__ float sum[128];
  __shared__ int last;
  const int tid = threadIdx.x;
  const int R = static_cast<int>(cluster_nctarank()), rank = static_cast<int>(cluster_ctarank());
  const int col = blockIdx.x / R * 128 + (tid & 15) * 8;
  const bool in = col < a.cols;
  pdl_launch_dependents();
  pdl_wait();
  int lo = 0, hi = a.rows;
  if (a.offsets) {
    // the last group ends at the largest clamped offset
    if (tid == 0) last = 0;
    __syncthreads();
    for (int i = tid; i <= a.groups; i += 256) atomicMax(&last, min(a.offsets[i], a.rows));
    __syncthreads();
    lo = max(0, min(a.offsets[0], a.rows));
    hi = last;
  }
  float acc[8] = {};
  if (in) {
    constexpr int U = 4;  // rows in flight per thread
    for (int row = lo + rank * 16 + (tid >> 4); row < hi; row += U * 16 * R) {
      uint4 d[U], z[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int r = row + u * 16 * R;
        const long long off = static_cast<long long>(r) * a.cols + col;
        d[u] = z[u] = make_uint4(0, 0, 0, 0);
        if (r < hi) {
          d[u] = __ldg(reinterpret_cast<const uint4 *>(a.dout + off));
          if (a.preact) z[u] = __ldg(reinterpret_cast<const uint4 *>(a.preact + off));
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int r = row + u * 16 * R;
        if (r >= hi) break;
        const u32 dw[4] = {d[u].x, d[u].y, d[u].z, d[u].w}, zw[4] = {z[u].x, z[u].y, z[u].z, z[u].w};
        u32 o[4];
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          float x = bf16_lo(dw[h]), y = bf16_hi(dw[h]);
          if (a.preact) {
            x *= act_slope(bf16_lo(zw[h]), a.act);
            y *= act_slope(bf16_hi(zw[h]), a.act);
          }
          acc[2 * h] += x;
          acc[2 * h + 1] += y;
          o[h] = pack_bf16x2(x, y);
        }
        if (a.dpre)
          st_global_v4(a.dpre + static_cast<long long>(r) * a.cols + col, o[0], o[1], o[2], o[3]);
      }
    }
  }
  if (!a.dbias) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) part[tid >> 4][(tid & 15) * 8 + i] = acc[i];
  __syncthreads();
  if (tid < 128) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) s += part[i][tid];
    sum[tid] = s;
  }
  __syncthreads();
  if (R > 1) cluster_sync();
  if (rank == 0 && tid < 128) {
    float s = sum[tid];
    for (int c = 1; c < R; ++c) s += ld_cluster_f32(mapa_cluster(smem_u32(&sum[tid]), c));
    const int n = blockIdx.x / R * 128 + tid;
    if (n < a.cols) a.dbias[n] = s;
  }
  __syncwarp();
  if (R > 1) cluster_sync();
}

}  // namespace lin
}  // namespace thork
