// linear.cu — the linear-layer operators of libthork_rt.so and their C-ABI
// entry points (declared in include/thork_rt.h):
//   thork_linear_{bf16,e4m3}             product + bias + activation + residual
//   thork_linear_backward_bf16           its gradients
//   thork_grouped_gemm_{bf16,e4m3}       products grouped by expert, ragged sizes
//   thork_grouped_gemm_backward_bf16     their gradients
// Kernels: device/linear_sm100.cuh.  No call allocates memory or keeps a
// workspace, so calls on different streams, and graphs that captured them,
// share nothing but the status word.
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

#include "device/linear_sm100.cuh"
#include "thork_internal.h"
#include "thork_rt.h"

using thork::dev::TensorMap;

namespace {
using namespace thork::lin;

// ---------------------------------------------------------------- launching
// Opt in to a kernel's dynamic shared memory, once per kernel and device.
int allow_smem(const void *kernel, int bytes, std::atomic<uint64_t> &done) {
  int dev;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return thork_cuda_error(e, "cudaGetDevice");
  const uint64_t bit = 1ull << (dev & 63);
  if (done.load(std::memory_order_acquire) & bit) return THORK_OK;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return thork_cuda_error(e, "cudaFuncSetAttribute(max dynamic smem)");
  done.fetch_or(bit, std::memory_order_release);
  return THORK_OK;
}

// Launch in clusters of `cluster` CTAs, with programmatic stream
// serialisation: the kernels wait for the previous one before they touch
// memory that it may write.
template <class... KArgs, class... Args>
int launch(void (*kern)(KArgs...), unsigned grid, int threads, int smem, int cluster, cudaStream_t s,
           const char *what, const Args &...args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid, 1, 1);
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, args...);
  return e == cudaSuccess ? THORK_OK : thork_cuda_error(e, what);
}

template <class C>
int run_swap(const TensorMap &tw, const TensorMap &tx, const GemmArgs &g, long long items, int split,
             cudaStream_t s, const char *what) {
  static std::atomic<uint64_t> done{0};
  int rc;
  auto kern = swap_kernel<C>;
  if ((rc = allow_smem(reinterpret_cast<const void *>(kern), C::SMEM_BYTES, done))) return rc;
  if (items * split > 0x7fffffffll)
    return thork_set_error(THORK_ERR_INVALID, "%s: %lld tiles are more than a launch can hold", what, items);
  return launch(kern, static_cast<unsigned>(items * split), C::THREADS, C::SMEM_BYTES, split, s, what, tw,
                tx, g);
}

// ---------------------------------------------------------------- a product
// One (grouped) product in GEMM terms: out[m, n] = sum_k X[m, k] W[k, n], X
// row-major [rows, k], W either as stored ([k, n] row-major, W_MN) or its
// transpose ([n, k] row-major).
struct Product {
  const void *x, *w;
  int rows, n, k;  // rows of X (of the buffer when grouped)
  int groups;      // 0: dense
};

template <int KIND, bool W_MN>
int map_w(TensorMap &t, const Product &p, int box_n) {
  const int elem = KIND == KIND_BF16 ? 2 : 1;
  const int dt = KIND == KIND_BF16 ? THORK_DT_BF16 : THORK_DT_E4M3;
  const uint64_t e = p.groups ? p.groups : 1;
  if (W_MN)
    return thork_encode_tmap_3d(&t, dt, p.w, p.n, p.k, e, 128 / elem, 128 / elem);
  return thork_encode_tmap_3d(&t, dt, p.w, p.k, p.n, e, 128 / elem, box_n);
}

template <int KIND>
int map_x(TensorMap &t, const Product &p, int box_rows) {
  const int elem = KIND == KIND_BF16 ? 2 : 1;
  return thork_encode_tmap_3d(&t, KIND == KIND_BF16 ? THORK_DT_BF16 : THORK_DT_E4M3, p.x, p.k, p.rows, 1,
                              128 / elem, box_rows);
}

template <int KIND, int BN, int STAGES, bool W_MN, bool GROUPED>
int swap_product(const Product &p, const GemmArgs &g, int split, cudaStream_t s, const char *what) {
  using C = SwapCfg<KIND, BN, STAGES, W_MN, false, GROUPED>;
  int rc;
  alignas(64) TensorMap tw, tx;
  if ((rc = map_w<KIND, W_MN>(tw, p, C::BM))) return rc;
  if ((rc = map_x<KIND>(tx, p, BN))) return rc;
  const long long ntn = (p.n + C::BM - 1) / C::BM;
  long long rt = (p.rows + BN - 1) / BN;
  if (GROUPED) {
    // at most one partial tile per group that has rows
    const long long most = (static_cast<long long>(p.rows) + static_cast<long long>(p.groups) * (BN - 1)) / BN;
    rt = most < p.rows ? most : p.rows;
  }
  return run_swap<C>(tw, tx, g, rt * ntn, split, s, what);
}

template <int KIND, bool W_MN, bool GROUPED>
int rows_product(const Product &p, const GemmArgs &g, cudaStream_t s, const char *what) {
  using C = RowsCfg<KIND, W_MN, GROUPED>;
  static std::atomic<uint64_t> done{0};
  int rc, sms;
  alignas(64) TensorMap tw, tx, txu;
  if ((rc = map_w<KIND, W_MN>(tw, p, C::BNC))) return rc;
  if ((rc = map_x<KIND>(tx, p, C::MAX_UNITS * C::BOX_ROWS))) return rc;
  if ((rc = map_x<KIND>(txu, p, C::BOX_ROWS))) return rc;
  auto kern = rows_kernel<C>;
  if ((rc = allow_smem(reinterpret_cast<const void *>(kern), C::SMEM_BYTES, done))) return rc;
  if ((rc = thork_sm_count(&sms))) return rc;
  // one pair per unit of 64 rows and 256 columns at most
  long long units = (static_cast<long long>(p.rows) + C::UNIT - 1) / C::UNIT;
  if (GROUPED) units += p.groups < p.rows ? p.groups : p.rows;
  const long long most = units * ((p.n + 2 * C::BNC - 1) / (2 * C::BNC));
  const int pairs = static_cast<int>(most < sms / 2 ? most : sms / 2);
  return launch(kern, 2 * pairs, C::THREADS, C::SMEM_BYTES, 2, s, what, tw, tx, txu, g);
}

// ---------------------------------------------------------------- choice of kernel
// Microseconds of one dense product by each kernel, estimated.  The forms and
// constants were fitted to timings of 4050 bf16 products on B200 (M 1 to 1600, N
// and K 128 to 14336), each with the choices that looked possible: on the 3537
// whose choice by the estimates was among them it is 1.9 % (mean) from the best,
// on 6.7 % of them by more than 10 %, at worst 1.68 times.  e4m3 products take
// the same estimates with their own blocks and bytes.  Both sides, every choice
// timed (us; floor: bytes or operations at the measured rates; swap_kernel's best
// with BN rows a tile and the contraction split in S, behind it the rule's):
//                        bf16                                  e4m3
//     M    N     K   floor  rows  swap  (BN/S)  rule     floor  rows  swap  (BN/S)  rule
//     1  4096  4096   5.1   19.1   9.1   32/8   16/8      2.6   11.6   7.1   16/8   16/8
//    64  4096  4096   5.3   19.6  11.7   64/8   64/8      2.7   12.0   8.8   32/4   64/8
//   128  4096  4096   5.5   21.1  14.0   64/4  128/8      2.8   12.4  10.3   64/4   64/4
//   256  4096  4096   5.8   22.0  18.0  128/4   rows      3.0   12.8  13.4   64/2   rows
//    64 14336  4096  18.3   23.3  25.2   64/2   rows      9.3   14.0  16.7   32/1   rows
//   256 14336  4096  19.4   29.7  41.1  128/1   rows     10.3   18.5  25.8  128/1   rows
//    64  4096 14336  18.3   55.3  24.1   64/8   64/8      9.2   29.7  15.5   64/8   64/8
//   256  4096 14336  19.4   58.5  36.3  128/4  128/4      9.9   31.5  22.6  128/4  128/4
//   400  4096 14336  28.7   64.4  60.5  128/2   rows     14.4   34.7  36.0  128/2   rows
//   128  1552  1040   0.6    8.9   6.8   32/4   32/4      0.3    6.9   5.5   16/1   32/4
//   777  1552  1040   1.5   10.0  13.1   64/1   rows      0.8    8.1  10.6   64/1   rows
// Of 28 products of either type (these and their neighbours at 1 to 777 rows) the
// rule is within 10 % of the best on all but 256 x 4096 x 4096 in bf16.
constexpr int ceil_div(long long a, int b) { return static_cast<int>((a + b - 1) / b); }

double rows_us(int nkb, int m, int n, double mbytes, int pairs) {
  int units = ceil_div(m, 64);
  if (units > 4) units = 4;
  const long long tiles = static_cast<long long>(ceil_div(m, 256)) * ceil_div(n, 256);
  double waves = 1.0;
  if (tiles < pairs) {
    const int pieces = static_cast<int>(pairs / tiles < 4 ? pairs / tiles : 4);
    units = ceil_div(units, pieces);
  } else {
    const int rest = static_cast<int>(tiles % pairs);
    const int pieces = rest ? (pairs / rest < 4 ? pairs / rest : 4) : 1;
    waves = static_cast<double>(tiles / pairs) + (rest ? (pieces > 1 ? 0.7 : 1.0) : 0.0);
  }
  const double block = 0.07 * units > 0.3 ? 0.07 * units : 0.3;
  const double math = waves * (nkb * block + 0.2), memory = mbytes / 7.0;
  return 5.2 + (math > memory ? math : memory);
}

double swap_us(int nkb, int m, int n, double mbytes, int sms, int bn, int split) {
  const double ctas = static_cast<double>(ceil_div(m, bn)) * ceil_div(n, 128) * split;
  double waves = static_cast<double>(static_cast<long long>(ctas / (2 * sms) + 0.95));
  if (waves < 1.0) waves = 1.0;
  // two CTAs of an SM share its feed: a stage is 16 KiB of weights and 128 bytes a row
  const double shared = ctas > 2 * sms ? 2.0 : ctas > sms ? ctas / sms : 1.0;
  const double feed = 0.6 * (16 + bn / 8) / 32 * shared;
  const double math = waves * (ceil_div(nkb, split) * (feed > 0.26 ? feed : 0.26) + 0.15), memory = mbytes / 6.3;
  const double height = (m < bn ? m : bn) / 16.0;
  return 5.1 + height * (0.32 * (split > 1 ? 1.3 : 1.0) + 0.02 * split) + (math > memory ? math : memory);
}

// A kernel and how it cuts the work: bn rows a tile and the contraction split
// in `split` for swap_kernel, bn = 0 for rows_kernel or outer_kernel.
struct Choice {
  int bn, split;
};

// out[m, n] over nkb blocks of a contraction that moves mbytes.
Choice by_estimate(int nkb, int m, int n, double mbytes, int sms, int least_bn) {
  double best = rows_us(nkb, m, n, mbytes, sms / 2);
  Choice choice = {0, 0};
  for (int bn = least_bn; bn <= 128; bn *= 2)
    for (int split = 1; split <= 8 && 2 * split <= nkb + 1; split *= 2) {
      const double us = swap_us(nkb, m, n, mbytes, sms, bn, split);
      if (us < best) {
        best = us;
        choice = {bn, split};
      }
    }
  return choice;
}

Choice choose_dense(int elem, int m, int n, int k, int sms) {
  const double mbytes =
      (elem * (static_cast<double>(n) * k + static_cast<double>(m) * k) + 2.0 * m * n) * 1e-6;
  return by_estimate(ceil_div(k, 128 / elem), m, n, mbytes, sms, 16);
}

template <int KIND, bool W_MN>
int dense_product(const Product &p, const GemmArgs &g, cudaStream_t s, const char *what) {
  int rc, sms;
  if ((rc = thork_sm_count(&sms))) return rc;
  const Choice c = choose_dense(KIND == KIND_BF16 ? 2 : 1, p.rows, p.n, p.k, sms);
  const int bn = c.bn, split = c.split;
  switch (bn) {
    case 16: return swap_product<KIND, 16, 6, W_MN, false>(p, g, split, s, what);
    case 32: return swap_product<KIND, 32, 5, W_MN, false>(p, g, split, s, what);
    case 64: return swap_product<KIND, 64, 4, W_MN, false>(p, g, split, s, what);
    case 128: return swap_product<KIND, 128, 3, W_MN, false>(p, g, split, s, what);
    default: return rows_product<KIND, W_MN, false>(p, g, s, what);
  }
}

// The groups' sizes are on the device, so the rule goes by their mean and their
// sum.  Few rows a group: swap_kernel, whose tiles waste no instruction on
// rows that are not there; more, or so many in all that one group alone may
// hold many: rows_kernel (us, mean rows 2 / 3 / 8 / 31 / 63: E=8 of 14336 x
// 4096 126 against 131 with rows_kernel; E=52 of 1432 x 2416 50 / 55; E=64 of
// 2048 x 2048 86 / 85; E=37 of 760 x 1304 28.6 / 22.3; e4m3 E=64 of 2048 x
// 1024 48 / 35).
Choice choose_grouped(int elem, int groups, int rows, int n, int k, int sms) {
  const int mean = ceil_div(rows, groups);
  if (mean > 24 || rows > 512) return {0, 0};
  // two CTAs fit on an SM: split the contraction until they are all in use
  const long long held = groups < rows ? groups : rows;
  const int nkb = ceil_div(k, 128 / elem);
  int split = 1;
  while (split < 8 && 2 * split * held * ceil_div(n, 128) <= 2 * sms && 4 * split <= nkb) split *= 2;
  return {mean <= 4 ? 16 : 32, split};
}

template <int KIND, bool W_MN>
int grouped_product(const Product &p, const GemmArgs &g, cudaStream_t s, const char *what) {
  int rc, sms;
  if ((rc = thork_sm_count(&sms))) return rc;
  const Choice c = choose_grouped(KIND == KIND_BF16 ? 2 : 1, p.groups, p.rows, p.n, p.k, sms);
  if (c.bn == 16) return swap_product<KIND, 16, 5, W_MN, true>(p, g, c.split, s, what);
  if (c.bn == 32) return swap_product<KIND, 32, 5, W_MN, true>(p, g, c.split, s, what);
  return rows_product<KIND, W_MN, true>(p, g, s, what);
}

// The dense weight gradient by swap_kernel: 128 columns n by BN rows k a
// cluster, the rows of X and dY split over it.
template <int BN, int STAGES>
int swap_gradient(const void *x, const void *dy, int rows, int n, int k, const GemmArgs &args, int split,
                  cudaStream_t s, const char *what) {
  using C = SwapCfg<KIND_BF16, BN, STAGES, true, true, false>;
  int rc;
  alignas(64) TensorMap tx, ty;
  if ((rc = thork_encode_tmap_3d(&ty, THORK_DT_BF16, dy, n, rows, 1, C::CHUNK, C::BK))) return rc;
  if ((rc = thork_encode_tmap_3d(&tx, THORK_DT_BF16, x, k, rows, 1, C::CHUNK, C::BK))) return rc;
  GemmArgs g = args;
  g.w_static = 0;
  return run_swap<C>(ty, tx, g, static_cast<long long>(ceil_div(k, BN)) * ceil_div(n, C::BM), split, s, what);
}

// dW[k, n] = sum over rows X[m, k] dY[m, n], of each group's rows when grouped.
template <bool GROUPED>
int weight_gradient(const void *x, const void *dy, int rows, int n, int k, const GemmArgs &g,
                    cudaStream_t s, const char *what) {
  using C = OuterCfg<GROUPED>;
  static std::atomic<uint64_t> done{0};
  int rc, sms;
  alignas(64) TensorMap tx, ty, tx16, ty16, tout;
  const auto map = [&](TensorMap &t, const void *p, int cols, int box_rows) {
    return thork_encode_tmap_3d(&t, THORK_DT_BF16, p, cols, rows, 1, C::CHUNK, box_rows);
  };
  if ((rc = map(tx, x, k, C::BK)) || (rc = map(ty, dy, n, C::BK))) return rc;
  if (GROUPED) {
    if ((rc = map(tx16, x, k, C::UMMA_K)) || (rc = map(ty16, dy, n, C::UMMA_K))) return rc;
  } else {
    tx16 = tx;  // no short blocks
    ty16 = ty;
  }
  if ((rc = thork_encode_tmap_3d(&tout, THORK_DT_BF16, g.epi.out, n, k, GROUPED ? g.groups : 1, C::CHUNK, 32)))
    return rc;
  auto kern = outer_kernel<C>;
  if ((rc = allow_smem(reinterpret_cast<const void *>(kern), C::SMEM_BYTES, done))) return rc;
  if ((rc = thork_sm_count(&sms))) return rc;
  // one pair per half of a tile at most
  const long long most = 2ll * ((k + 255) / 256) * ((n + 255) / 256) * (GROUPED ? g.groups : 1);
  const int pairs = static_cast<int>(most < sms / 2 ? most : sms / 2);
  return launch(kern, 2 * pairs, C::THREADS, C::SMEM_BYTES, 2, s, what, tx, ty, tx16, ty16, tout, g);
}

// Few tiles with many rows to sum over: split the rows over clusters, by the
// same estimates (us, outer_kernel / swap_kernel: 2604 rows of 184 x 152 17.0 /
// 7.7, 8054 of 256 x 536 33.6 / 12.9, 8192 of 1024 x 1024 33.7 / 22.9; 637 of
// 1800 x 488 8.7 / 10.9, 7008 of 2168 x 1384 56 / 90; of those timed the rule
// missed one, 1000 of 776 x 520, with 9.8 / 8.9).
Choice choose_gradient(int rows, int n, int k, int sms) {
  const double mbytes = 2e-6 * (static_cast<double>(n) * k + static_cast<double>(rows) * (n + k));
  return by_estimate(ceil_div(rows, 64), k, n, mbytes, sms, 64);
}

int dense_gradient(const void *x, const void *dy, int rows, int n, int k, const GemmArgs &g, cudaStream_t s,
                   const char *what) {
  int rc, sms;
  if ((rc = thork_sm_count(&sms))) return rc;
  const Choice c = choose_gradient(rows, n, k, sms);
  if (c.bn == 64) return swap_gradient<64, 4>(x, dy, rows, n, k, g, c.split, s, what);
  if (c.bn == 128) return swap_gradient<128, 3>(x, dy, rows, n, k, g, c.split, s, what);
  return weight_gradient<false>(x, dy, rows, n, k, g, s, what);
}

template <int LANES>
int run_slope(const SlopeArgs &a, int cluster, cudaStream_t s, const char *what) {
  const unsigned grid = static_cast<unsigned>(ceil_div(a.cols, 8 * LANES)) * a.split;
  return a.preact ? launch(slope_kernel<LANES, true>, grid, kSlopeThreads, 0, cluster, s, what, a)
                  : launch(slope_kernel<LANES, false>, grid, kSlopeThreads, 0, cluster, s, what, a);
}

int slope(SlopeArgs a, cudaStream_t s, const char *what) {
  int rc, sms;
  if ((rc = thork_sm_count(&sms))) return rc;
  const int wave = 4 * sms;  // one wave of four blocks per SM
  // the widest stripes whose blocks, at most eight a stripe where they are
  // summed, come near one wave
  int lanes = 16;
  while (a.dbias && lanes > 4 && 8ll * ceil_div(a.cols, 8 * lanes) * 4 < 3ll * wave) lanes /= 2;
  int split = wave / ceil_div(a.cols, 8 * lanes);
  // no more than leave a block two passes over its rows
  const int most = ceil_div(a.rows, 2 * kSlopeThreads / lanes);
  if (split > most) split = most;
  if (a.dbias && split > 8) split = 8;
  if (split < 1) split = 1;
  a.split = split;
  const int cluster = a.dbias ? split : 1;
  return lanes == 16 ? run_slope<16>(a, cluster, s, what)
         : lanes == 8 ? run_slope<8>(a, cluster, s, what)
                      : run_slope<4>(a, cluster, s, what);
}

// ---------------------------------------------------------------- checks
// Row and column numbers, rounded up to whole tiles and passes, are ints.
constexpr int kMaxDim = 1 << 30;

int check_sizes(int rows, int n, int k, int align, const char *what) {
  if (rows <= 0 || n <= 0 || k <= 0)
    return thork_set_error(THORK_ERR_INVALID, "%s: dimensions must be positive (M=%d N=%d K=%d)", what,
                           rows, n, k);
  if (rows > kMaxDim || n > kMaxDim || k > kMaxDim)
    return thork_set_error(THORK_ERR_INVALID, "%s: dimensions must be at most 2^30 (M=%d N=%d K=%d)", what,
                           rows, n, k);
  if (n % align || k % align)
    return thork_set_error(THORK_ERR_INVALID,
                           "%s: K and N must be multiples of %d for 16-byte TMA row strides (M=%d N=%d K=%d)",
                           what, align, rows, n, k);
  return THORK_OK;
}

// An epilogue waits for the whole contraction of its tile, at most
// THORK_WAIT_TIMEOUT_NS (1 s).  A block of the contraction is 64 values (e4m3:
// 128) and takes 0.3 us of a tile at the tensor pipe's rate and at most 1.5 us
// where every CTA's operands come from HBM, so 2^23 values stay below 0.2 s.
constexpr int kMaxContraction = 1 << 23;

int check_contraction(int len, const char *name, const char *what) {
  if (len > kMaxContraction)
    return thork_set_error(THORK_ERR_INVALID, "%s: a contraction over %s=%d is more than 2^23", what, name, len);
  return THORK_OK;
}

int check_groups(int groups, const void *offsets, const char *what) {
  if (groups < 1 || groups > kMaxGroups)
    return thork_set_error(THORK_ERR_INVALID, "%s: E=%d must be 1..%d", what, groups, kMaxGroups);
  if (!offsets || (reinterpret_cast<uintptr_t>(offsets) & 3u))
    return thork_set_error(THORK_ERR_INVALID, "%s: offsets are NULL or not 4-byte aligned", what);
  return THORK_OK;
}

int check_act(int act, const char *what) {
  if (act < THORK_ACT_NONE || act > THORK_ACT_SILU)
    return thork_set_error(THORK_ERR_INVALID, "%s: unknown activation %d", what, act);
  return THORK_OK;
}

// One array argument: required ones may not be NULL, all are 16-byte aligned.
struct Arg {
  const void *p;
  const char *name;
  bool required, output;
};

template <size_t N>
int check_args(const Arg (&args)[N], const char *what) {
  for (const Arg &a : args) {
    if (a.required && !a.p) return thork_set_error(THORK_ERR_INVALID, "%s: %s is NULL", what, a.name);
    if (reinterpret_cast<uintptr_t>(a.p) & 15u)
      return thork_set_error(THORK_ERR_INVALID, "%s: %s must be 16-byte aligned", what, a.name);
  }
  for (const Arg &o : args)
    for (const Arg &i : args)
      if (o.output && o.p && o.p == i.p && &o != &i)
        return thork_set_error(THORK_ERR_INVALID, "%s: %s and %s are the same array", what, o.name, i.name);
  return THORK_OK;
}

template <int KIND>
int linear(const void *a, const void *b, void *c, const void *bias, const void *residual, void *preact,
           int M, int N, int K, float alpha, int act, int flags, void *stream, const char *what) {
  int rc;
  if ((rc = check_sizes(M, N, K, KIND == KIND_BF16 ? 8 : 16, what))) return rc;
  if ((rc = check_contraction(K, "K", what))) return rc;
  if ((rc = check_act(act, what))) return rc;
  if (flags & ~THORK_LINEAR_W_STATIC)
    return thork_set_error(THORK_ERR_INVALID, "%s: unknown flags 0x%x", what, flags);
  const Arg args[] = {{a, "A", true, false}, {b, "B", true, false}, {bias, "bias", false, false},
                      {c, "out", true, true}, {preact, "preact", false, true}};
  if ((rc = check_args(args, what))) return rc;
  const Arg inplace[] = {{residual, "residual", false, false}, {preact, "preact", false, true}};
  if ((rc = check_args(inplace, what))) return rc;  // out may be the residual itself
  GemmArgs g = {};
  g.epi = {static_cast<unsigned short *>(c), static_cast<unsigned short *>(preact),
           static_cast<const unsigned short *>(bias), static_cast<const unsigned short *>(residual),
           nullptr, alpha, act, N, nullptr};
  if ((rc = thork_host_status_word(&g.epi.status))) return rc;
  g.GM = g.rows = M;
  g.GN = N;
  g.GK = K;
  g.w_static = flags & THORK_LINEAR_W_STATIC;
  return dense_product<KIND, true>({a, b, M, N, K, 0}, g, static_cast<cudaStream_t>(stream), what);
}

template <int KIND>
int grouped(const void *a, const void *b, void *c, const int *offsets, void *preact, int E, int T, int N,
            int K, float alpha, const float *group_scale, int act, int flags, void *stream,
            const char *what) {
  int rc;
  if ((rc = check_sizes(T, N, K, KIND == KIND_BF16 ? 8 : 16, what))) return rc;
  if ((rc = check_contraction(K, "K", what))) return rc;
  if ((rc = check_groups(E, offsets, what))) return rc;
  if ((rc = check_act(act, what))) return rc;
  if (flags & ~THORK_LINEAR_W_STATIC)
    return thork_set_error(THORK_ERR_INVALID, "%s: unknown flags 0x%x", what, flags);
  const Arg args[] = {{a, "A", true, false}, {b, "B", true, false}, {c, "out", true, true},
                      {preact, "preact", false, true}};
  if ((rc = check_args(args, what))) return rc;
  if (reinterpret_cast<uintptr_t>(group_scale) & 3u)
    return thork_set_error(THORK_ERR_INVALID, "%s: scale_b is not 4-byte aligned", what);
  GemmArgs g = {};
  g.epi = {static_cast<unsigned short *>(c), static_cast<unsigned short *>(preact), nullptr, nullptr,
           group_scale, alpha, act, N, nullptr};
  if ((rc = thork_host_status_word(&g.epi.status))) return rc;
  g.GM = g.rows = T;
  g.GN = N;
  g.GK = K;
  g.offsets = offsets;
  g.groups = E;
  return grouped_product<KIND, true>({a, b, T, N, K, E}, g, static_cast<cudaStream_t>(stream), what);
}

// Gradients of a (grouped) linear layer from dout and, with an activation,
// the pre-activation; groups == 0 is the dense layer.
int backward(void *da, void *db, float *dbias, const void *dout, const void *a, const void *b,
             const void *preact, void *dpre, const int *offsets, int groups, int rows, int N, int K,
             int act, void *stream, const char *what) {
  int rc;
  if ((rc = check_sizes(rows, N, K, 8, what))) return rc;
  if (da && (rc = check_contraction(N, "N", what))) return rc;
  if (db && (rc = check_contraction(rows, groups ? "T" : "M", what))) return rc;
  if ((rc = check_act(act, what))) return rc;
  const bool bent = act != THORK_ACT_NONE;
  if (bent != (preact != nullptr) || bent != (dpre != nullptr))
    return thork_set_error(THORK_ERR_INVALID,
                           "%s: preact and dpre go with an activation, and with one only", what);
  const Arg args[] = {{dout, "dout", true, false}, {a, "A", db != nullptr, false},
                      {b, "B", da != nullptr, false}, {preact, "preact", false, false},
                      {dpre, "dpre", false, true}, {da, "dA", false, true}, {db, "dB", false, true},
                      {dbias, "dbias", false, true}};
  if ((rc = check_args(args, what))) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (bent || dbias) {
    const SlopeArgs sl = {static_cast<const unsigned short *>(dout),
                          static_cast<const unsigned short *>(preact), static_cast<unsigned short *>(dpre),
                          dbias, rows, N, act, 1, offsets, groups};
    if ((rc = slope(sl, s, what))) return rc;
  }
  const void *dz = bent ? dpre : dout;
  GemmArgs g = {};
  g.epi.alpha = 1.0f;
  if ((rc = thork_host_status_word(&g.epi.status))) return rc;
  g.rows = rows;
  g.offsets = offsets;
  g.groups = groups;
  if (da) {
    GemmArgs d = g;
    d.epi.out = static_cast<unsigned short *>(da);
    d.epi.cols = K;
    d.GM = rows;
    d.GN = K;
    d.GK = N;
    d.trigger_late = db != nullptr;
    const Product p = {dz, b, rows, K, N, groups};
    rc = groups ? grouped_product<KIND_BF16, false>(p, d, s, what) : dense_product<KIND_BF16, false>(p, d, s, what);
    if (rc) return rc;
  }
  if (db) {
    GemmArgs w = g;
    w.epi.out = static_cast<unsigned short *>(db);
    w.epi.cols = N;
    w.GM = K;
    w.GN = N;
    w.GK = rows;
    w.wait_last = da != nullptr;
    rc = groups ? weight_gradient<true>(a, dz, rows, N, K, w, s, what)
                : dense_gradient(a, dz, rows, N, K, w, s, what);
    if (rc) return rc;
  }
  return THORK_OK;
}
}  // namespace

extern "C" int thork_linear_choice(int form, int M, int N, int K, int E, int sms, int *tile_rows,
                                   int *split) {
  const char *what = "linear_choice";
  int rc;
  if (!tile_rows || !split) return thork_set_error(THORK_ERR_INVALID, "%s: NULL output", what);
  if ((rc = check_sizes(M, N, K, 8, what))) return rc;
  if (sms < 2 || E < 1) return thork_set_error(THORK_ERR_INVALID, "%s: sms=%d E=%d", what, sms, E);
  Choice c;
  switch (form) {
    case THORK_CHOICE_BF16: c = choose_dense(2, M, N, K, sms); break;
    case THORK_CHOICE_E4M3: c = choose_dense(1, M, N, K, sms); break;
    case THORK_CHOICE_GRADIENT: c = choose_gradient(M, N, K, sms); break;
    case THORK_CHOICE_GROUPED_BF16: c = choose_grouped(2, E, M, N, K, sms); break;
    case THORK_CHOICE_GROUPED_E4M3: c = choose_grouped(1, E, M, N, K, sms); break;
    default: return thork_set_error(THORK_ERR_INVALID, "%s: unknown form %d", what, form);
  }
  *tile_rows = c.bn;
  *split = c.split;
  return THORK_OK;
}

extern "C" int thork_linear_bf16(const void *d_a, const void *d_b, void *d_out, const void *d_bias,
                                 const void *d_residual, void *d_preact, int M, int N, int K,
                                 int activation, int flags, void *stream) {
  return linear<KIND_BF16>(d_a, d_b, d_out, d_bias, d_residual, d_preact, M, N, K, 1.0f, activation, flags,
                           stream, "linear_bf16");
}

extern "C" int thork_linear_e4m3(const void *d_a, const void *d_b, void *d_out, const void *d_bias,
                                 const void *d_residual, void *d_preact, int M, int N, int K,
                                 float scale_a, float scale_b, int activation, int flags, void *stream) {
  return linear<KIND_E4M3>(d_a, d_b, d_out, d_bias, d_residual, d_preact, M, N, K, scale_a * scale_b,
                           activation, flags, stream, "linear_e4m3");
}

extern "C" int thork_linear_backward_bf16(void *d_da, void *d_db, float *d_dbias, const void *d_dout,
                                          const void *d_a, const void *d_b, const void *d_preact,
                                          void *d_dpre, int M, int N, int K, int activation, void *stream) {
  return backward(d_da, d_db, d_dbias, d_dout, d_a, d_b, d_preact, d_dpre, nullptr, 0, M, N, K, activation,
                  stream, "linear_backward_bf16");
}

extern "C" int thork_grouped_gemm_bf16(const void *d_a, const void *d_b, void *d_out, const int *d_offsets,
                                       void *d_preact, int E, int T, int N, int K, int activation,
                                       int flags, void *stream) {
  return grouped<KIND_BF16>(d_a, d_b, d_out, d_offsets, d_preact, E, T, N, K, 1.0f, nullptr, activation,
                            flags, stream, "grouped_gemm_bf16");
}

extern "C" int thork_grouped_gemm_e4m3(const void *d_a, const void *d_b, void *d_out, const int *d_offsets,
                                       void *d_preact, int E, int T, int N, int K, float scale_a,
                                       const float *d_scale_b, int activation, int flags, void *stream) {
  return grouped<KIND_E4M3>(d_a, d_b, d_out, d_offsets, d_preact, E, T, N, K, scale_a, d_scale_b,
                            activation, flags, stream, "grouped_gemm_e4m3");
}

extern "C" int thork_grouped_gemm_backward_bf16(void *d_da, void *d_db, const void *d_dout, const void *d_a,
                                                const void *d_b, const int *d_offsets, const void *d_preact,
                                                void *d_dpre, int E, int T, int N, int K, int activation,
                                                void *stream) {
  int rc;
  if ((rc = check_groups(E, d_offsets, "grouped_gemm_backward_bf16"))) return rc;
  return backward(d_da, d_db, nullptr, d_dout, d_a, d_b, d_preact, d_dpre, d_offsets, E, T, N, K,
                  activation, stream, "grouped_gemm_backward_bf16");
}
