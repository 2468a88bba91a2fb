// Products grouped by expert (bf16, both gradients, block-scaled e4m3) and the
// dense block-scaled e4m3 products, which are the same with a single group.
#include <atomic>
#include <cmath>
#include <cstring>

#include "gemm_fp8_sm100.cuh"
#include "gemm_grouped_simt.cuh"
#include "gemm_grouped_sm100.cuh"
#include "gemm_host.cuh"

namespace {

using col::simt::GroupedSimtParams;
using col::sm100::GroupedCfg;
using col::sm100::GroupedParams;
using col::sm100::kForward;
using col::sm100::kGradW;
using col::sm100::kGradX;

constexpr std::uint64_t kIntMax = 0x7fffffffull;

// Sizes every entry point shares: rows and widths below 2^31 (rounded up to
// whole tiles), at most kMaxGroups groups.
inline bool sizes_ok(std::uint64_t rows, std::uint64_t k, std::uint64_t columns,
                     std::uint64_t groups) {
  return rows <= kIntMax - 1024 && k != 0 && k <= kIntMax - 1024 && columns <= kIntMax - 1024 &&
         groups <= static_cast<std::uint64_t>(col::kMaxGroups);
}

GroupedSimtParams simt_params(const void* a, const void* b, const std::int32_t* offsets, void* out,
                              std::uint64_t rows, std::uint64_t k, std::uint64_t n,
                              std::uint64_t w_rows, std::uint64_t groups) {
  GroupedSimtParams p = {};
  p.a = a;
  p.b = b;
  p.offsets = offsets;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.rows = static_cast<int>(rows);
  p.k = static_cast<int>(k);
  p.n = static_cast<int>(n);
  p.w_rows = static_cast<int>(w_rows);
  p.groups = static_cast<int>(groups);
  return p;
}

// ---------------------------------------------------------------- tensor maps

// A tensor map is a pure function of these; the calling thread keeps the last
// few, since a call on the same weights or reused buffers needs the same map
// (as gemm.cu does for the dense products).
struct MapKey {
  const void* base;
  std::uint64_t cols;     // contiguous elements
  std::uint64_t rows;
  std::uint64_t experts;  // 0: two-dimensional
  std::uint32_t box_rows;
  std::uint32_t elem;     // bytes
};

// Map over row-major [experts][rows][cols]; box = 128 bytes of columns (the
// swizzle span) x box_rows rows.  Out-of-range boxes read zeros.
int encode_map(CUtensorMap* map, const MapKey& key) {
  struct Entry {
    CUtensorMap map;
    MapKey key;
    bool valid;
  };
  constexpr int kEntries = 32;
  thread_local Entry cache[kEntries] = {};
  const std::uintptr_t h = (reinterpret_cast<std::uintptr_t>(key.base) >> 7) ^ (key.rows * 31u) ^
                           (key.cols * 131u) ^ (key.experts * 7u) ^
                           (static_cast<std::uintptr_t>(key.box_rows) * 13u);
  Entry& e = cache[(h ^ (h >> 5) ^ (h >> 10)) % kEntries];
  if (e.valid && e.key.base == key.base && e.key.cols == key.cols && e.key.rows == key.rows &&
      e.key.experts == key.experts && e.key.box_rows == key.box_rows && e.key.elem == key.elem) {
    std::memcpy(map, &e.map, sizeof(CUtensorMap));
    return 0;
  }
  auto enc = col::tensor_map_encoder();
  if (!enc) return col::kErrNoTensorMapEncoder;
  const cuuint64_t dims[3] = {key.cols, key.rows, key.experts};
  const cuuint64_t strides[2] = {key.cols * key.elem, key.cols * key.rows * key.elem};
  const cuuint32_t box[3] = {128 / key.elem, key.box_rows, 1};
  const cuuint32_t estrides[3] = {1, 1, 1};
  const CUresult r = enc(
      map, key.elem == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8,
      key.experts == 0 ? 2 : 3, const_cast<void*>(key.base), dims, strides, box, estrides,
      CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return col::kErrTensorMapEncode;
  std::memcpy(&e.map, map, sizeof(CUtensorMap));
  e.key = key;
  e.valid = true;
  return 0;
}

// Whether TMA can address rows of `cols` elements from `base`.
inline bool tma_ok(const void* base, std::uint64_t cols, std::uint32_t elem) {
  return col::aligned16(base) && (cols * elem) % 16 == 0;
}

// ---------------------------------------------------------------- launches

// Dynamic shared memory of a kernel, set once per device.
template <typename Kernel>
int allow_smem(Kernel kernel, std::uint32_t bytes, int dev, std::atomic<std::uint64_t>& done) {
  const std::uint64_t bit = 1ull << (dev & 63);
  if (done.load(std::memory_order_acquire) & bit) return 0;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             static_cast<int>(bytes));
  if (e != cudaSuccess) return static_cast<int>(e);
  done.fetch_or(bit, std::memory_order_release);
  return 0;
}

// Workers (CTAs or CTA pairs) that can be resident at once.
// (every kernel here takes over half of an SM's shared memory, so one answer a
// device serves them all)
template <typename Kernel>
int resident_pairs(Kernel kernel, std::uint32_t smem, int dev) {
  static std::atomic<int> cached[64] = {};
  int pairs = cached[dev & 63].load(std::memory_order_acquire);
  if (pairs != 0) return pairs;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2, 1, 1);
  cfg.blockDim = dim3(col::sm100::kCtaThreads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = 2;
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if (cudaOccupancyMaxActiveClusters(&pairs, kernel, &cfg) != cudaSuccess || pairs <= 0) {
    cudaGetLastError();
    pairs = -1;
  }
  cached[dev & 63].store(pairs, std::memory_order_release);
  return pairs;
}

// ---------------------------------------------------------------- choice of tiles

// A tensor-core variant: CTAs of a tile, accumulator columns, rows of a CTA,
// CTAs that share a tile's sum.
struct Variant {
  int cg;
  int bn;
  int rows;
  int split;
};

// What a variant takes, measured under load on a B200 (148 SMs), in us: a
// k-block of a tile, the same where the tile alone reads its rows of w so that
// DRAM bounds it, and a tile's share that does not overlap (most of it storing).
struct VariantCost {
  Variant v;
  double block;
  double block_dram;
  double tile;
};

// bf16 (k-blocks of 64); fastest of 12 runs of ten launches back to back on the same
// inputs: 16384 rows over 8 experts, 4096 x 4096: pairs 376 us, single CTAs with 256
// columns 476, with 128 columns 561.  256 rows over 64 experts, gate/up 2048 x
// 4096: 32-row tiles 156 us, 128 columns 172, 256 columns 170, pairs 195.  Over 27
// drawn sizes (512-16384 rows, 1-32 experts, widths 512-8192) the choice takes
// 1.06 (forward), 1.08 (by x) and 1.06 (by W) times the best variant in the
// geometric mean, at worst 1.5; pairs alone 1.09, 1.08 and 1.05, single CTAs 1.15
// and more.  Below 128 rows a group pairs are not considered.
constexpr VariantCost kBf16Costs[] = {
    {{2, 256, 128, 1}, 0.44, 0.53, 1.8},
    {{1, 256, 128, 1}, 0.48, 0.72, 1.4},
    {{1, 128, 128, 1}, 0.285, 0.38, 0.8},
    {{1, 128, 32, 1}, 0.285, 0.34, 0.8},
};
constexpr int kSingle128 = 2;

// e4m3 (k-blocks of 128), measured the same way: 8192 x 4096 x 4096: pairs 156 us,
// 256 columns 192, 128 columns 205; the decode shape above: 128 columns 103 us,
// 256 columns 112, pairs 161.  Tiles of 32 rows took as long as those of 128 there,
// so they serve only sums that a cluster shares.
constexpr VariantCost kFp8Costs[] = {
    {{2, 256, 128, 1}, 0.60, 0.66, 1.5},
    {{1, 256, 128, 1}, 0.79, 0.80, 1.5},
    {{1, 128, 128, 1}, 0.435, 0.435, 0.8},
};

// Row tiles of `rows` rows over `groups` groups whose sizes the host does not
// know: groups without rows have none, the others at least one, and on average
// half a tile more than their rows fill.
double expected_row_tiles(std::uint64_t rows, std::uint64_t groups, bool known, int tile_rows) {
  const double fill = static_cast<double>(rows) / tile_rows;
  if (known) return static_cast<double>((rows + tile_rows - 1) / tile_rows);
  const double used = static_cast<double>(rows < groups ? rows : groups);
  return fill + 0.5 * used > used ? fill + 0.5 * used : used;
}

// The most row tiles there can be: each has at least one row, each group at most
// one that is not full.
std::uint64_t most_row_tiles(std::uint64_t rows, std::uint64_t groups, bool known, int tile_rows) {
  if (known) return (rows + tile_rows - 1) / tile_rows;
  const std::uint64_t tiles = rows / tile_rows + groups;
  return tiles < rows ? tiles : rows;
}

// The variant whose waves of tiles take least.  `row_tiles(tile_rows)` and
// `columns` (accumulator columns) span the tiles, `k_blocks` the sum of one.
template <int COUNT, typename RowTiles>
Variant choose_variant(const VariantCost (&costs)[COUNT], RowTiles row_tiles, double columns,
                       double k_blocks, double rows_per_group, int sm_count, bool rows32 = true,
                       double* us_out = nullptr) {
  Variant best = costs[0].v;
  double best_us = -1.0;
  for (const VariantCost& c : costs) {
    if (c.v.rows == 32 && !rows32) continue;
    const int tile_rows = c.v.cg * c.v.rows;
    // a pair's tile that is not half full is two CTAs' time for one's work
    if (c.v.cg == 2 && rows_per_group < 128.0) continue;
    const double tiles = row_tiles(tile_rows) * std::ceil(columns / c.v.bn);
    const double waves = std::ceil(tiles / (sm_count / c.v.cg));
    const double block = rows_per_group <= tile_rows ? c.block_dram : c.block;
    const double us = waves * (k_blocks * block + c.tile);
    if (best_us < 0.0 || us < best_us) {
      best = c.v;
      best_us = us;
    }
  }
  if (us_out) *us_out = best_us;
  return best;
}

template <int MODE, bool SWIGLU, int CG, int BN, int ROWS, int SPLIT = 1>
int launch_grouped_bf16(GroupedParams& p, std::uint64_t most_tiles, int dev, int sm_count,
                        cudaStream_t s) {
  using Cfg = GroupedCfg<CG, BN, ROWS, SPLIT>;
  auto kernel = col::sm100::grouped_bf16_kernel<MODE, SWIGLU, CG, BN, ROWS, SPLIT>;
  static std::atomic<std::uint64_t> done{0};
  if (int rc = allow_smem(kernel, Cfg::kSmemBytes, dev, done)) return rc;
  int workers = sm_count;
  if constexpr (CG == 2) {
    workers = resident_pairs(kernel, Cfg::kSmemBytes, dev);
    if (workers <= 0) return static_cast<int>(cudaErrorInvalidConfiguration);
  }
  // clusters that share a tile's sum take one tile each
  if (SPLIT > 1 || most_tiles < static_cast<std::uint64_t>(workers)) {
    workers = static_cast<int>(most_tiles);
  }
  return col::launch_serialised(kernel, dim3(static_cast<unsigned>(workers * CG * SPLIT)),
                                dim3(col::sm100::kCtaThreads), Cfg::kSmemBytes, s, p);
}

// The variant of a bf16 product by waves of tiles, and its time.
Variant waves_bf16(int mode, std::uint64_t t, std::uint64_t k, std::uint64_t n,
                   std::uint64_t experts, std::uint64_t columns, int sm_count,
                   double* us_out = nullptr) {
  // Rows a group: of the operand that a tile's rows come from (kGradW: of w, the
  // same for every group, and the sums have T rows over the groups).
  const double group_rows = static_cast<double>(t) / static_cast<double>(t < experts ? t : experts);
  const double k_blocks = mode == kGradW   ? std::ceil(group_rows / 64.0)
                          : mode == kGradX ? std::ceil(static_cast<double>(n) / 64.0)
                                           : std::ceil(static_cast<double>(k) / 64.0);
  return choose_variant(
      kBf16Costs,
      [&](int tile_rows) {
        if (mode == kGradW) return static_cast<double>(experts * ((n + tile_rows - 1) / tile_rows));
        return expected_row_tiles(t, experts, false, tile_rows);
      },
      static_cast<double>(columns), k_blocks, mode == kGradW ? 1e9 : group_rows, sm_count,
      mode != kGradW, us_out);
}

// The variant that a bf16 product runs.
Variant choose_bf16(int mode, bool swiglu, std::uint64_t t, std::uint64_t k, std::uint64_t n,
                    std::uint64_t experts, int sm_count) {
  const std::uint64_t columns = mode != kForward ? k : swiglu ? 2 * n : n;
  Variant v = waves_bf16(mode, t, k, n, experts, columns, sm_count);
  if (mode == kGradW) return v;
  // A few tiles of few rows: four or two CTAs share each sum while there are SMs
  // for them, with at least four k-blocks apiece.
  const std::uint64_t tiles = most_row_tiles(t, experts, false, 32) * ((columns + 127) / 128);
  const std::uint64_t k_blocks = ((mode == kForward ? k : n) + 63) / 64;
  for (const int split : {4, 2}) {
    if (v.split == 1 && tiles * split <= static_cast<std::uint64_t>(sm_count) &&
        k_blocks >= 4u * split) {
      v = Variant{1, 128, 32, split};
    }
  }
  return v;
}

// Whether 32 bits count the scales.
inline bool scales_ok(std::uint64_t t, std::uint64_t k, std::uint64_t w_rows, std::uint64_t experts) {
  const std::uint64_t k_blocks = (k + 127) / 128;
  return t * k_blocks <= kIntMax && experts * ((w_rows + 127) / 128) * k_blocks <= kIntMax;
}

// The variant that an e4m3 product runs; `known`: all rows are one group's.
Variant choose_fp8(std::uint64_t t, std::uint64_t k, std::uint64_t w_rows, std::uint64_t experts,
                   bool known, int sm_count) {
  const std::uint64_t k_blocks = (k + 127) / 128;
  const double used = static_cast<double>(t < experts ? t : experts);
  Variant v = choose_variant(
      kFp8Costs, [&](int tile_rows) { return expected_row_tiles(t, experts, known, tile_rows); },
      static_cast<double>(w_rows), static_cast<double>(k_blocks), static_cast<double>(t) / used,
      sm_count);
  // A few tiles of few rows: four or two CTAs share each sum while there are
  // SMs for them, with at least two k-blocks apiece.  One row by 4096 x 4096:
  // 12.5 us with one CTA a tile, 9.1 with two, 8.1 with four; one row by 1024 x
  // 4096: 12.2, 8.2, 6.9, and 6.2 with four and 64 columns.
  const std::uint64_t tiles32 = most_row_tiles(t, experts, known, 32);
  double best_blocks = 0.0;
  for (const int bn : {64, 128}) {
    for (const int split : {2, 4}) {
      const std::uint64_t ctas = tiles32 * ((w_rows + bn - 1) / bn) * split;
      if (ctas > static_cast<std::uint64_t>(sm_count) || k_blocks < 2u * split) continue;
      // k-blocks of a CTA, those of 64 columns at 0.7 of the others' time
      const double blocks = std::ceil(static_cast<double>(k_blocks) / split) * (bn == 64 ? 0.7 : 1.0);
      if (best_blocks == 0.0 || blocks < best_blocks) {
        best_blocks = blocks;
        v = Variant{1, bn, 32, split};
      }
    }
  }
  return v;
}

// What a product's kernel gets, but for its tiles; -1 where TMA cannot address the
// operands.
template <int MODE, bool SWIGLU>
int grouped_params(GroupedParams& p, const void* a, const void* b, const std::int32_t* offsets,
                   void* out, std::uint64_t t, std::uint64_t k, std::uint64_t n,
                   std::uint64_t experts, int dev, const col::DeviceInfo& info) {
  if (!tma_ok(a, MODE == kForward ? k : n, 2) || !tma_ok(b, k, 2)) return -1;
  if (info.cc_major != 10) return col::kErrDeviceNotSupported;
  std::memset(&p, 0, sizeof(p));
  p.status = col::gemm_status_ptr(dev);
  if (!p.status) return static_cast<int>(cudaErrorInvalidDevice);
  const std::uint64_t out_cols = MODE == kForward ? n : k;
  p.offsets = offsets;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.rows = static_cast<int>(t);
  p.groups = static_cast<int>(experts);
  p.out_cols = static_cast<int>(out_cols);
  p.out_rows = static_cast<int>(n);
  p.num_k_blocks = static_cast<int>(((MODE == kForward ? k : n) + 63) / 64);
  p.up_offset = static_cast<int>(n);
  p.out_vec_ok = col::aligned16(out) && out_cols % 8 == 0;
  return 0;
}

// The column tiles and tensor maps of a variant.
template <int MODE, bool SWIGLU>
int grouped_maps(GroupedParams& p, const Variant& v, const void* a, const void* b, std::uint64_t t,
                 std::uint64_t k, std::uint64_t n, std::uint64_t experts) {
  const std::uint64_t a_cols = MODE == kForward ? k : n;
  p.num_n_blocks = (p.out_cols * (SWIGLU ? 2 : 1) + v.bn - 1) / v.bn;
  int rc = encode_map(&p.map_a, {a, a_cols, t, 0, MODE == kGradW ? 64u : 128u, 2});
  if (rc == 0 && MODE != kGradW && v.cg == 1) rc = encode_map(&p.map_a32, {a, a_cols, t, 0, 32, 2});
  if (rc != 0) return rc;
  const std::uint32_t b_box =
      MODE == kForward ? static_cast<std::uint32_t>(col::sm100::b_box_rows(SWIGLU, v.cg, v.bn)) : 64u;
  return MODE == kGradW
             ? encode_map(&p.map_b, {b, k, t, 0, b_box, 2})
             : encode_map(&p.map_b, {b, k, SWIGLU ? 2 * n : n, experts, b_box, 2});
}

// Tensor-core product; -1 where TMA cannot address the operands.
template <int MODE, bool SWIGLU>
int grouped_bf16_tc(const void* a, const void* b, const std::int32_t* offsets, void* out,
                    std::uint64_t t, std::uint64_t k, std::uint64_t n, std::uint64_t experts,
                    cudaStream_t s) {
  int dev = 0;
  const col::DeviceInfo& info = col::device_info(&dev);
  GroupedParams p;
  int rc = grouped_params<MODE, SWIGLU>(p, a, b, offsets, out, t, k, n, experts, dev, info);
  if (rc != 0) return rc;
  const Variant v = choose_bf16(MODE, SWIGLU, t, k, n, experts, info.sm_count);
  rc = grouped_maps<MODE, SWIGLU>(p, v, a, b, t, k, n, experts);
  if (rc != 0) return rc;
  const int tile_rows = v.cg * v.rows;
  const std::uint64_t m_tiles = MODE == kGradW ? experts * ((n + tile_rows - 1) / tile_rows)
                                               : most_row_tiles(t, experts, false, tile_rows);
  const std::uint64_t most_tiles = m_tiles * p.num_n_blocks;
  if (most_tiles > kIntMax) return static_cast<int>(cudaErrorInvalidValue);
  const int sms = info.sm_count;
  if (v.cg == 2) return launch_grouped_bf16<MODE, SWIGLU, 2, 256, 128>(p, most_tiles, dev, sms, s);
  if constexpr (MODE != kGradW) {
    if (v.split == 4) return launch_grouped_bf16<MODE, SWIGLU, 1, 128, 32, 4>(p, most_tiles, dev, sms, s);
    if (v.split == 2) return launch_grouped_bf16<MODE, SWIGLU, 1, 128, 32, 2>(p, most_tiles, dev, sms, s);
    if (v.rows == 32) return launch_grouped_bf16<MODE, SWIGLU, 1, 128, 32>(p, most_tiles, dev, sms, s);
  }
  if (v.bn == 256) return launch_grouped_bf16<MODE, SWIGLU, 1, 256, 128>(p, most_tiles, dev, sms, s);
  return launch_grouped_bf16<MODE, SWIGLU, 1, 128, 128>(p, most_tiles, dev, sms, s);
}

template <int ROWS>
int launch_backward(const GroupedParams& by_x, const GroupedParams& by_w, int input_ctas,
                    int weight_ctas, int dev, cudaStream_t s) {
  constexpr std::uint32_t kX = GroupedCfg<1, 128, ROWS, 1>::kSmemBytes;
  constexpr std::uint32_t kW = GroupedCfg<1, 128, 128, 1>::kSmemBytes;
  constexpr std::uint32_t kSmem = kX > kW ? kX : kW;
  auto kernel = col::sm100::grouped_bf16_backward_kernel<ROWS>;
  static std::atomic<std::uint64_t> done{0};
  if (int rc = allow_smem(kernel, kSmem, dev, done)) return rc;
  return col::launch_serialised(kernel, dim3(static_cast<unsigned>(input_ctas + weight_ctas)),
                                dim3(col::sm100::kCtaThreads), kSmem, s, by_x, by_w, input_ctas);
}

// Both gradients in one launch, each on its share of the SMs, where that takes
// less than two launches after one another; -1 where it does not, or TMA cannot
// address the operands.  A second launch costs kSecondLaunchUs on the GPU (its
// start, and the first one's last wave), and ~6 us of the caller's time.
// The margin is for shares that uneven groups unbalance: without it 3519 rows over
// 5, 2264 x 568, took 50.6 us instead of 39.6.  Over 70 drawn sizes (8-6000 rows,
// 1-64 experts, widths 64-3000, three spreads of the groups; back to back) the
// choice takes 1.006 times the faster form in the geometric mean, at worst 1.20;
// always two launches 1.43, at worst 2.04.
constexpr double kSecondLaunchUs = 4.0;
constexpr double kBothMargin = 1.2;
constexpr double kInputBlockUs = 0.3;

// The CTAs of either gradient in one launch; rows == 0: two launches take less.
struct BothGradients {
  int rows;  // of a tile of the gradient by x
  int input_ctas;
  int weight_ctas;
};

BothGradients plan_both(std::uint64_t t, std::uint64_t k, std::uint64_t n, std::uint64_t experts,
                        int sm_count) {
  const std::uint64_t columns = (k + 127) / 128;
  const int rows = t <= 32 * experts ? 32 : 128;
  const double group_rows = static_cast<double>(t) / static_cast<double>(t < experts ? t : experts);
  const double input_tiles = expected_row_tiles(t, experts, false, rows) * static_cast<double>(columns);
  const double weight_tiles = static_cast<double>(experts * ((n + 127) / 128) * columns);
  // a tile's time in either: of the single CTAs with 128 columns, whose blocks by x
  // take between the two figures of the table, as part of the SMs read w
  const VariantCost& cost = kBf16Costs[kSingle128];
  const double input_us = std::ceil(static_cast<double>(n) / 64.0) * kInputBlockUs + cost.tile;
  const double weight_us = std::ceil(group_rows / 64.0) * cost.block + cost.tile;
  double input_share = input_tiles;
  double weight_share = weight_tiles;
  if (input_tiles + weight_tiles > sm_count) {
    const double part = input_tiles * input_us / (input_tiles * input_us + weight_tiles * weight_us);
    input_share = std::fmin(std::fmax(std::round(part * sm_count), 1.0), sm_count - 1.0);
    weight_share = sm_count - input_share;
  }
  const double both_us = std::fmax(std::ceil(input_tiles / input_share) * input_us,
                                   std::ceil(weight_tiles / weight_share) * weight_us);
  double first_us = 0.0;
  double second_us = 0.0;
  waves_bf16(kGradX, t, k, n, experts, k, sm_count, &first_us);
  waves_bf16(kGradW, t, k, n, experts, k, sm_count, &second_us);
  if (both_us * kBothMargin >= first_us + second_us + kSecondLaunchUs) return {0, 0, 0};
  return {rows, static_cast<int>(std::ceil(input_share)), static_cast<int>(weight_share)};
}

int backward_tc(const void* grad, const void* x, const void* w, const std::int32_t* offsets,
                void* dx, void* dw, std::uint64_t t, std::uint64_t k, std::uint64_t n,
                std::uint64_t experts, cudaStream_t s) {
  int dev = 0;
  const col::DeviceInfo& info = col::device_info(&dev);
  const BothGradients plan = plan_both(t, k, n, experts, info.sm_count);
  const int rows = plan.rows;
  if (rows == 0) return -1;
  GroupedParams by_x, by_w;
  int rc = grouped_params<kGradX, false>(by_x, grad, w, offsets, dx, t, k, n, experts, dev, info);
  if (rc == 0) rc = grouped_params<kGradW, false>(by_w, grad, x, offsets, dw, t, k, n, experts, dev, info);
  if (rc == 0) rc = grouped_maps<kGradX, false>(by_x, {1, 128, rows, 1}, grad, w, t, k, n, experts);
  if (rc == 0) rc = grouped_maps<kGradW, false>(by_w, {1, 128, 128, 1}, grad, x, t, k, n, experts);
  if (rc != 0) return rc;
  if (rows == 32) return launch_backward<32>(by_x, by_w, plan.input_ctas, plan.weight_ctas, dev, s);
  return launch_backward<128>(by_x, by_w, plan.input_ctas, plan.weight_ctas, dev, s);
}

template <bool SWIGLU, int CG, int BN, int ROWS, int SPLIT>
int launch_fp8(col::sm100::Fp8Params& p, std::uint64_t most_tiles, int dev, int sm_count,
               cudaStream_t s) {
  using Cfg = col::sm100::Fp8Cfg<CG, BN, ROWS, SPLIT>;
  auto kernel = col::sm100::fp8_kernel<SWIGLU, CG, BN, ROWS, SPLIT>;
  static std::atomic<std::uint64_t> done{0};
  if (int rc = allow_smem(kernel, Cfg::kSmemBytes, dev, done)) return rc;
  if constexpr (col::sm100::fp8_split_regs(BN)) {
    // The warps that take registers over wait until they are free, so the
    // kernel must have been compiled to start with enough of them.
    static const bool covered = [kernel]() {
      cudaFuncAttributes attr;
      return cudaFuncGetAttributes(&attr, kernel) == cudaSuccess &&
             attr.numRegs >= col::sm100::kFp8RegsLaunch;
    }();
    if (!covered) return static_cast<int>(cudaErrorInvalidConfiguration);
  }
  int workers = sm_count;
  if constexpr (CG == 2) {
    workers = resident_pairs(kernel, Cfg::kSmemBytes, dev);
    if (workers <= 0) return static_cast<int>(cudaErrorInvalidConfiguration);
  }
  // clusters that share a tile's sum take one tile each
  if (SPLIT > 1 || most_tiles < static_cast<std::uint64_t>(workers)) {
    workers = static_cast<int>(most_tiles);
  }
  return col::launch_serialised(kernel, dim3(static_cast<unsigned>(workers * CG * SPLIT)),
                                dim3(col::sm100::kCtaThreads), Cfg::kSmemBytes, s, p);
}

// Tensor-core product; -1 where TMA cannot address the operands or 32 bits do
// not count the scales.
template <bool SWIGLU>
int fp8_tc(const void* x, const float* xs, const void* w, const float* ws,
           const std::int32_t* offsets, void* out, std::uint64_t t, std::uint64_t k,
           std::uint64_t n, std::uint64_t experts, cudaStream_t s) {
  const std::uint64_t w_rows = SWIGLU ? 2 * n : n;
  const std::uint64_t k_blocks = (k + 127) / 128;
  const std::uint64_t scale_rows = (w_rows + 127) / 128;
  if (!tma_ok(x, k, 1) || !tma_ok(w, k, 1)) return -1;
  if (!scales_ok(t, k, w_rows, experts)) return -1;
  int dev = 0;
  const col::DeviceInfo& info = col::device_info(&dev);
  if (info.cc_major != 10) return col::kErrDeviceNotSupported;
  col::sm100::Fp8Params fp;
  std::memset(&fp, 0, sizeof(fp));
  GroupedParams& p = fp.g;
  p.status = col::gemm_status_ptr(dev);
  if (!p.status) return static_cast<int>(cudaErrorInvalidDevice);
  p.offsets = offsets;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.rows = static_cast<int>(t);
  p.groups = static_cast<int>(experts);
  p.out_cols = static_cast<int>(n);
  p.num_k_blocks = static_cast<int>(k_blocks);
  p.up_offset = static_cast<int>(n);
  p.out_vec_ok = col::aligned16(out) && n % 8 == 0;
  fp.a_scale = xs;
  fp.b_scale = ws;
  fp.b_scale_rows = static_cast<int>(scale_rows);

  const Variant v = choose_fp8(t, k, w_rows, experts, offsets == nullptr, info.sm_count);
  p.num_n_blocks = static_cast<int>((w_rows + v.bn - 1) / v.bn);
  const std::uint64_t most_tiles =
      most_row_tiles(t, experts, offsets == nullptr, v.cg * v.rows) * p.num_n_blocks;
  if (most_tiles * v.split > kIntMax) return static_cast<int>(cudaErrorInvalidValue);
  int rc = encode_map(&p.map_a, {x, k, t, 0, 128, 1});
  if (rc == 0 && v.cg == 1) rc = encode_map(&p.map_a32, {x, k, t, 0, 32, 1});
  if (rc == 0) {
    rc = encode_map(&p.map_b, {w, k, w_rows, experts,
                               static_cast<std::uint32_t>(col::sm100::b_box_rows(SWIGLU, v.cg, v.bn)), 1});
  }
  if (rc != 0) return rc;
  const int sms = info.sm_count;
  if (v.cg == 2) return launch_fp8<SWIGLU, 2, 256, 128, 1>(fp, most_tiles, dev, sms, s);
  if (v.rows == 32) {
    if (v.bn == 128) {
      return v.split == 4 ? launch_fp8<SWIGLU, 1, 128, 32, 4>(fp, most_tiles, dev, sms, s)
                          : launch_fp8<SWIGLU, 1, 128, 32, 2>(fp, most_tiles, dev, sms, s);
    }
    return v.split == 4 ? launch_fp8<SWIGLU, 1, 64, 32, 4>(fp, most_tiles, dev, sms, s)
                        : launch_fp8<SWIGLU, 1, 64, 32, 2>(fp, most_tiles, dev, sms, s);
  }
  if (v.bn == 256) return launch_fp8<SWIGLU, 1, 256, 128, 1>(fp, most_tiles, dev, sms, s);
  return launch_fp8<SWIGLU, 1, 128, 128, 1>(fp, most_tiles, dev, sms, s);
}

template <bool SWIGLU>
int grouped_forward_bf16(const void* x, const void* w, const std::int32_t* offsets, void* out,
                         std::uint64_t t, std::uint64_t k, std::uint64_t n, std::uint64_t experts,
                         void* stream) {
  if (t == 0 || n == 0 || experts == 0) return 0;
  const std::uint64_t w_rows = SWIGLU ? 2 * n : n;
  if (!x || !w || !offsets || !out || !sizes_ok(t, k, n, experts) || w_rows > kIntMax - 1024) {
    return static_cast<int>(cudaErrorInvalidValue);
  }
  const cudaStream_t s = col::as_stream(stream);
  const int rc = grouped_bf16_tc<kForward, SWIGLU>(x, w, offsets, out, t, k, n, experts, s);
  if (rc != -1) return rc;
  const GroupedSimtParams p = simt_params(x, w, offsets, out, t, k, n, w_rows, experts);
  return col::simt::launch_grouped_simt<__nv_bfloat16, col::simt::kForward, SWIGLU>(p, s);
}

template <bool SWIGLU>
int forward_fp8(const void* x, const float* xs, const void* w, const float* ws,
                const std::int32_t* offsets, void* out, std::uint64_t t, std::uint64_t k,
                std::uint64_t n, std::uint64_t experts, void* stream) {
  const std::uint64_t w_rows = SWIGLU ? 2 * n : n;
  if (!x || !xs || !w || !ws || !out || !sizes_ok(t, k, n, experts) || w_rows > kIntMax - 1024) {
    return static_cast<int>(cudaErrorInvalidValue);
  }
  // A tile of scales must not span gate and up rows.
  if (SWIGLU && n % 128 != 0) return static_cast<int>(cudaErrorInvalidValue);
  const cudaStream_t s = col::as_stream(stream);
  const int rc = fp8_tc<SWIGLU>(x, xs, w, ws, offsets, out, t, k, n, experts, s);
  if (rc != -1) return rc;
  GroupedSimtParams p = simt_params(x, w, offsets, out, t, k, n, w_rows, experts);
  p.a_scale = xs;
  p.b_scale = ws;
  return col::simt::launch_grouped_simt<__nv_fp8_e4m3, col::simt::kForward, SWIGLU>(p, s);
}

}  // namespace

COL_API int cuda_operator_gemm_grouped_bf16(const void* input_bf16, const void* weight_bf16,
                                            const int32_t* offsets, void* output_bf16, uint64_t t,
                                            uint64_t k, uint64_t n, uint64_t experts,
                                            void* stream) {
  return grouped_forward_bf16<false>(input_bf16, weight_bf16, offsets, output_bf16, t, k, n,
                                     experts, stream);
}

COL_API int cuda_operator_gemm_grouped_swiglu_bf16(const void* input_bf16,
                                                   const void* packed_weight_bf16,
                                                   const int32_t* offsets, void* output_bf16,
                                                   uint64_t t, uint64_t k, uint64_t n,
                                                   uint64_t experts, void* stream) {
  return grouped_forward_bf16<true>(input_bf16, packed_weight_bf16, offsets, output_bf16, t, k, n,
                                    experts, stream);
}

COL_API int cuda_operator_gemm_grouped_bf16_grad_input(const void* grad_bf16,
                                                       const void* weight_bf16,
                                                       const int32_t* offsets,
                                                       void* grad_input_bf16, uint64_t t,
                                                       uint64_t k, uint64_t n, uint64_t experts,
                                                       void* stream) {
  if (t == 0 || k == 0 || experts == 0) return 0;
  if (!grad_bf16 || !weight_bf16 || !offsets || !grad_input_bf16 || n == 0 ||
      !sizes_ok(t, k, n, experts)) {
    return static_cast<int>(cudaErrorInvalidValue);
  }
  const cudaStream_t s = col::as_stream(stream);
  const int rc = grouped_bf16_tc<kGradX, false>(grad_bf16, weight_bf16, offsets, grad_input_bf16, t,
                                                k, n, experts, s);
  if (rc != -1) return rc;
  const GroupedSimtParams p =
      simt_params(grad_bf16, weight_bf16, offsets, grad_input_bf16, t, k, n, n, experts);
  return col::simt::launch_grouped_simt<__nv_bfloat16, col::simt::kGradX, false>(p, s);
}

COL_API int cuda_operator_gemm_grouped_bf16_grad_weight(const void* grad_bf16,
                                                        const void* input_bf16,
                                                        const int32_t* offsets,
                                                        void* grad_weight_bf16, uint64_t t,
                                                        uint64_t k, uint64_t n, uint64_t experts,
                                                        void* stream) {
  if (k == 0 || n == 0 || experts == 0) return 0;
  if (!offsets || !grad_weight_bf16 || (t != 0 && (!grad_bf16 || !input_bf16)) ||
      !sizes_ok(t, k, n, experts)) {
    return static_cast<int>(cudaErrorInvalidValue);
  }
  const cudaStream_t s = col::as_stream(stream);
  int rc = -1;
  if (t != 0) {
    rc = grouped_bf16_tc<kGradW, false>(grad_bf16, input_bf16, offsets, grad_weight_bf16, t, k, n,
                                        experts, s);
  }
  if (rc != -1) return rc;
  // also t == 0 (there is nothing to address): every sum is empty, all zeros
  const GroupedSimtParams p =
      simt_params(grad_bf16, input_bf16, offsets, grad_weight_bf16, t, k, n, n, experts);
  return col::simt::launch_grouped_simt<__nv_bfloat16, col::simt::kGradW, false>(p, s);
}

COL_API int cuda_operator_gemm_grouped_bf16_backward(const void* grad_bf16, const void* input_bf16,
                                                     const void* weight_bf16,
                                                     const int32_t* offsets, void* grad_input_bf16,
                                                     void* grad_weight_bf16, uint64_t t, uint64_t k,
                                                     uint64_t n, uint64_t experts, void* stream) {
  if (t != 0 && k != 0 && n != 0 && experts != 0) {
    if (!grad_bf16 || !input_bf16 || !weight_bf16 || !offsets || !grad_input_bf16 ||
        !grad_weight_bf16 || !sizes_ok(t, k, n, experts)) {
      return static_cast<int>(cudaErrorInvalidValue);
    }
    const int rc = backward_tc(grad_bf16, input_bf16, weight_bf16, offsets, grad_input_bf16,
                               grad_weight_bf16, t, k, n, experts, col::as_stream(stream));
    if (rc != -1) return rc;
  }
  const int rc = cuda_operator_gemm_grouped_bf16_grad_input(
      grad_bf16, weight_bf16, offsets, grad_input_bf16, t, k, n, experts, stream);
  if (rc != 0) return rc;
  return cuda_operator_gemm_grouped_bf16_grad_weight(grad_bf16, input_bf16, offsets,
                                                     grad_weight_bf16, t, k, n, experts, stream);
}

COL_API int cuda_operator_gemm_fp8_block128(const void* input_fp8, const float* input_scale,
                                            const void* weight_fp8, const float* weight_scale,
                                            void* output_bf16, uint64_t m, uint64_t k, uint64_t n,
                                            void* stream) {
  if (m == 0 || n == 0) return 0;
  return forward_fp8<false>(input_fp8, input_scale, weight_fp8, weight_scale, nullptr, output_bf16,
                            m, k, n, 1, stream);
}

COL_API int cuda_operator_gemm_swiglu_fp8_block128(const void* input_fp8, const float* input_scale,
                                                   const void* packed_weight_fp8,
                                                   const float* weight_scale, void* output_bf16,
                                                   uint64_t m, uint64_t k, uint64_t n,
                                                   void* stream) {
  if (m == 0 || n == 0) return 0;
  return forward_fp8<true>(input_fp8, input_scale, packed_weight_fp8, weight_scale, nullptr,
                           output_bf16, m, k, n, 1, stream);
}

COL_API int cuda_operator_gemm_grouped_fp8_block128(const void* input_fp8,
                                                    const float* input_scale,
                                                    const void* weight_fp8,
                                                    const float* weight_scale,
                                                    const int32_t* offsets, void* output_bf16,
                                                    uint64_t t, uint64_t k, uint64_t n,
                                                    uint64_t experts, void* stream) {
  if (t == 0 || n == 0 || experts == 0) return 0;
  if (!offsets) return static_cast<int>(cudaErrorInvalidValue);
  return forward_fp8<false>(input_fp8, input_scale, weight_fp8, weight_scale, offsets, output_bf16,
                            t, k, n, experts, stream);
}

COL_API int cuda_operator_gemm_grouped_swiglu_fp8_block128(
    const void* input_fp8, const float* input_scale, const void* packed_weight_fp8,
    const float* weight_scale, const int32_t* offsets, void* output_bf16, uint64_t t, uint64_t k,
    uint64_t n, uint64_t experts, void* stream) {
  if (t == 0 || n == 0 || experts == 0) return 0;
  if (!offsets) return static_cast<int>(cudaErrorInvalidValue);
  return forward_fp8<true>(input_fp8, input_scale, packed_weight_fp8, weight_scale, offsets,
                           output_bf16, t, k, n, experts, stream);
}

COL_API int cuda_operator_lab_expert_tiles(int product, uint64_t t, uint64_t k, uint64_t n,
                                           uint64_t experts, int sm_count, int* tiles) {
  if (!tiles || sm_count < 2 || t == 0 || n == 0 || experts == 0 || !sizes_ok(t, k, n, experts)) {
    return static_cast<int>(cudaErrorInvalidValue);
  }
  Variant v = {0, 0, 0, 0};
  const bool k8 = k % 8 == 0;
  const bool n8 = n % 8 == 0;
  const std::uint64_t w_rows =
      product == COL_EXPERT_SWIGLU_FP8 || product == COL_DENSE_SWIGLU_FP8 ? 2 * n : n;
  const bool fp8 = k % 16 == 0 && scales_ok(t, k, w_rows, experts);
  switch (product) {
    case COL_EXPERT_BF16:
    case COL_EXPERT_SWIGLU_BF16:
      if (k8) v = choose_bf16(kForward, product == COL_EXPERT_SWIGLU_BF16, t, k, n, experts, sm_count);
      break;
    case COL_EXPERT_GRAD_INPUT:
      if (k8 && n8) v = choose_bf16(kGradX, false, t, k, n, experts, sm_count);
      break;
    case COL_EXPERT_GRAD_WEIGHT:
      if (k8 && n8) v = choose_bf16(kGradW, false, t, k, n, experts, sm_count);
      break;
    case COL_EXPERT_BOTH_GRADS:
      if (k8 && n8) {
        const int rows = plan_both(t, k, n, experts, sm_count).rows;
        if (rows != 0) v = {1, 128, rows, 1};
      }
      break;
    case COL_EXPERT_FP8:
    case COL_EXPERT_SWIGLU_FP8:
      if (fp8) v = choose_fp8(t, k, w_rows, experts, false, sm_count);
      break;
    case COL_DENSE_FP8:
    case COL_DENSE_SWIGLU_FP8:
      if (experts != 1) return static_cast<int>(cudaErrorInvalidValue);
      if (fp8) v = choose_fp8(t, k, w_rows, 1, true, sm_count);
      break;
    default:
      return static_cast<int>(cudaErrorInvalidValue);
  }
  tiles[0] = v.cg;
  tiles[1] = v.bn;
  tiles[2] = v.rows;
  tiles[3] = v.split;
  return 0;
}
